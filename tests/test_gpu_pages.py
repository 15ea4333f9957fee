"""The exact paged cache on the GPU against 64-bit torch: write, decode, ledger, observe, evict."""

import math
import random

import pytest
import torch

from tests import pages_oracle as O
from turboquant_b200 import AttentionLedger, CompressedKVStore, ExactCacheSpec, PagedKVCache, compute_hybrid_attention

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
RANGE = -7


class Setup:
    """A cache whose sequences have pages of their own in random order; every row that belongs to no token is NaN."""

    def __init__(self, lens, H, D, page=16, dtype=BF16, seed=0, layout="plain", spare=2, sharp=1.0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.H, self.D, self.page, self.dtype = lens, H, D, page, dtype
        self.longest = max(max(lens), 1)
        width = -(-self.longest // page)
        blocks = len(lens) * width + spare
        self.table = torch.randperm(blocks, generator=g)[: len(lens) * width].int().view(len(lens), width)
        shape = {"plain": (2, blocks, page, H, D), "heads": (2, blocks, H, page, D), "pairs": (blocks, 2, page, H, D),
                 "padded": (2, blocks, page, H, D + 8)}[layout]
        planes = torch.full(shape, math.nan, dtype=dtype)
        views = {"plain": lambda p: (p[0], p[1]), "heads": lambda p: (p[0].transpose(1, 2), p[1].transpose(1, 2)),
                 "pairs": lambda p: (p[:, 0], p[:, 1]), "padded": lambda p: (p[0, ..., :D], p[1, ..., :D])}[layout]
        self.k, self.v = views(planes)
        for b, n in enumerate(lens):
            t = torch.arange(n)
            at = self.table[b, t // page].long(), t % page
            self.k[at] = (torch.randn(n, H, D, generator=g) * sharp * torch.exp(0.5 * torch.randn(D, generator=g))).to(dtype)
            self.v[at] = torch.randn(n, H, D, generator=g).to(dtype)
        self.spec = ExactCacheSpec(D, H, block_size=page, dtype=dtype)
        dev = planes.cuda()
        self.cache = PagedKVCache(self.spec, *views(dev))
        self.dtable, self.dlens = self.table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
        self.gen = g

    def query(self, *lead, heads):
        return torch.randn(*lead, heads, self.D, generator=self.gen).to(self.dtype)

    def rows(self, b):
        """(n, H, D) doubles of sequence b."""
        n = self.lens[b]
        t = torch.arange(n)
        at = self.table[b, t // self.page].long(), t % self.page
        return self.k[at].double(), self.v[at].double()


def weight_error(q, k, scale):
    """Relative error of a softmax weight: scores are sums of exact products held in 32 bits, at most D / 16 <= 16 additions that
    lose 2^-22 of the largest partial sum each, once in the score and once in the reference of the normalisation; exponentials
    and sums lose some 2^-20."""
    size = (q.abs().amax() * k.abs().sum(-1).amax()).item() * scale if k.numel() else 0.0
    return 2 * 16 * 2.0 ** -22 * size + 2.0 ** -19


def check_out(got, ref, p, v, dtype, rel):
    """Half a step of the type for the output's rounding; the weights' own error, and 2^-16 for the two 16-bit parts they are
    multiplied in, on the sum of the weighted magnitudes.  Numbers below the type's normal range round absolutely."""
    bound = torch.einsum("rhgn,nhd->rhgd", p, v.abs()) * (rel + 2.0 ** -16)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    allowed = ref.abs() * torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -6) + bound + tiny
    assert not torch.isnan(got).any()
    over = ((got - ref).abs() - allowed).max().item()
    assert over <= 0, over


def ledger_of(s, seed=1, batch=None, slots=None):
    g = torch.Generator().manual_seed(seed)
    led = AttentionLedger(batch or len(s.lens), s.H, slots or s.longest, "cuda")
    led.mass.copy_(torch.rand(led.mass.shape, generator=g))
    return led


CASES = [  # lens, H, G, D, page, dtype, layout
    ([1], 1, 1, 128, 16, BF16, "plain"),
    ([17, 0, 15, 16, 1], 2, 4, 128, 16, BF16, "plain"),
    ([300], 8, 4, 128, 16, BF16, "heads"),
    ([5000, 3, 0, 777, 128], 2, 8, 128, 16, BF16, "pairs"),
    ([2049], 1, 5, 64, 32, FP16, "padded"),
    ([1000, 31, 2], 3, 7, 64, 7, BF16, "plain"),
    ([1234, 64], 2, 16, 128, 128, FP16, "plain"),
    ([999, 40], 1, 33, 128, 16, BF16, "plain"),
    ([4097], 4, 4, 256, 16, BF16, "plain"),
    ([513, 0, 90], 2, 12, 256, 24, FP16, "heads"),
    ([100] * 70, 2, 2, 64, 1, BF16, "plain"),
    ([0, 0], 2, 2, 128, 16, BF16, "plain"),
    ([20000], 1, 1, 128, 64, FP16, "plain"),
]


@pytest.mark.parametrize("lens,H,G,D,page,dtype,layout", CASES)
def test_decode(lens, H, G, D, page, dtype, layout):
    s = Setup(lens, H, D, page, dtype, seed=3, layout=layout)
    q = s.query(len(lens), heads=H * G)
    led = ledger_of(s, slots=s.longest + 5)
    before = led.mass.cpu().double()
    out = s.cache.decode(q.cuda(), s.dtable, s.dlens, s.longest, ledger=led)
    plain = s.cache.decode(q.cuda(), s.dtable, s.dlens, s.longest)
    assert torch.equal(out, plain)                       # the ledger does not change the output, and the same call gives the same bits
    out, mass = out.cpu().double(), led.mass.cpu().double()
    for b, n in enumerate(lens):
        k, v = s.rows(b)
        qb = q[b].double().view(1, H, G, D)
        ref, p = O.attention(qb, k, v)
        rel = weight_error(qb, k, D ** -0.5)
        check_out(out[b].view(1, H, G, D), ref, p, v, dtype, rel)
        add = p[0].sum(1)
        assert torch.equal(mass[b, :, n:], before[b, :, n:])
        # the increment's error, and one rounding of the sum
        assert ((mass[b, :, :n] - before[b, :, :n] - add).abs() <= add * rel + mass[b, :, :n] * 2.0 ** -23).all()
    assert s.cache.status() == 0


def test_decode_joins_many_pieces_and_large_scores():
    """One long sequence over every CTA, with scores so large that one token has nearly all the weight; scale given."""
    s = Setup([30011], 2, 128, 16, BF16, seed=5, sharp=4.0)
    q = s.query(1, heads=8)
    out = s.cache.decode(q.cuda(), s.dtable, s.dlens, s.longest, scale=0.5).cpu().double()
    k, v = s.rows(0)
    ref, p = O.attention(q[0].double().view(1, 2, 4, 128), k, v, scale=0.5)
    check_out(out.view(1, 2, 4, 128), ref, p, v, BF16, weight_error(q.double(), k, 0.5))


def test_decode_into_a_buffer_from_strided_views():
    s = Setup([90, 33, 250], 2, 128, seed=8)
    q = s.query(3, heads=8)
    wide = torch.zeros(3, 16, 128, dtype=BF16, device="cuda")
    wide[:, 4:12] = q.cuda()
    table = torch.full((5, 40), 10 ** 6, dtype=torch.int32, device="cuda")      # wider, more rows, bad entries behind
    table[:3, : s.table.shape[1]] = s.dtable
    lens = torch.tensor([90, 33, 250, 7, 9], dtype=torch.int32, device="cuda")
    out = torch.full((3, 8, 128), 7.0, dtype=BF16, device="cuda")
    got = s.cache.decode(wide[:, 4:12], table, lens, 640, out=out)
    assert got is out and torch.equal(out, s.cache.decode(q.cuda(), s.dtable, s.dlens, s.longest))
    every_other = torch.zeros(3, 2 * s.table.shape[1], dtype=torch.int32, device="cuda")
    every_other[:, ::2] = s.dtable
    assert torch.equal(out, s.cache.decode(q.cuda(), every_other[:, ::2], s.dlens, s.longest))
    assert s.cache.status() == 0


def test_no_tokens_at_all():
    s = Setup([0, 0, 0], 2, 128)
    q = s.query(3, heads=4).cuda()
    led = ledger_of(s)
    before = led.mass.clone()
    assert not s.cache.decode(q, s.dtable, s.dlens, 0, ledger=led).any()
    assert s.cache.decode(q[:0], s.dtable, s.dlens, 5).shape == (0, 4, 128)
    s.cache.observe(q[:, None], s.dtable, s.dlens, 1, led)
    s.cache.observe(q[:, None][:, :0], s.dtable, s.dlens, 1, led)
    assert s.cache.evict(s.dtable, s.dlens, 0, led, 4).tolist() == [0, 0, 0]
    s.cache.write(q[:0, :2], q[:0, :2], torch.zeros(0, dtype=torch.int64, device="cuda"))
    assert (led.mass == 0).all() and before.any() and s.cache.status() == 0


@pytest.mark.parametrize("page", [16, 7])
def test_bad_pages_and_lengths_are_left_out_and_reported(page):
    """A table entry outside the pages: its tokens are as if they were not there; a length out of range is clamped."""
    s = Setup([200, 150, 40], 2, 128, page, seed=2)
    table = s.table.clone()
    table[0, 1], table[0, 3], table[2, :] = -1, 10 ** 9, s.cache.num_blocks
    there = torch.ones(3, 200, dtype=torch.bool)
    for b in range(3):
        for t in range(200):
            there[b, t] = 0 <= table[b, t // page] < s.cache.num_blocks
    q, win = s.query(3, heads=8), s.query(3, 5, heads=8)
    led, led2 = ledger_of(s), ledger_of(s)
    before = led.mass.cpu().double()
    out = s.cache.decode(q.cuda(), table.cuda(), s.dlens, 200, ledger=led).cpu().double()
    assert s.cache.status() == RANGE and s.cache.status() == 0
    s.cache.observe(win.cuda(), table.cuda(), s.dlens, 200, led2)
    assert s.cache.status() == RANGE
    for b, n in enumerate(s.lens):
        k, v = s.rows(b)
        ref, p = O.attention(q[b].double().view(1, 2, 4, 128), k, v, there=there[b, :n])
        rel = weight_error(q.double(), k, 128 ** -0.5)
        check_out(out[b].view(1, 2, 4, 128), ref, p, v, BF16, rel)
        last = torch.arange(n - 5, n)
        _, pw = O.attention(win[b].double().view(5, 2, 4, 128), k, v, last=last, there=there[b, :n])
        for m, add in ((led.mass, p[0].sum(1)), (led2.mass, pw.sum((0, 2)))):
            m = m[b, :, :n].cpu().double()
            assert ((m - before[b, :, :n] - add).abs() <= add * rel + m * 2.0 ** -22).all()
    wrong = torch.tensor([200, 10 ** 6, -5], dtype=torch.int32, device="cuda")
    right = torch.tensor([200, 200, 0], dtype=torch.int32, device="cuda")
    table[0] = s.table[0]
    table[1] = s.table[0]
    a = s.cache.decode(q.cuda(), table.cuda(), wrong, 200)
    assert s.cache.status() == RANGE
    assert torch.equal(a, s.cache.decode(q.cuda(), table.cuda(), right, 200)) and s.cache.status() == 0


@pytest.mark.parametrize("D,H,page,dtype,layout,T", [(128, 8, 16, BF16, "plain", 64), (64, 3, 7, FP16, "pairs", 33), (256, 1, 1, BF16, "heads", 1),
                                                     (128, 2, 32, FP16, "padded", 1501)])
def test_write(D, H, page, dtype, layout, T):
    s = Setup([max(1, T + 40)], H, D, page, dtype, layout=layout)
    g = torch.Generator().manual_seed(1)
    fused = torch.randn(T, 3, H, D, generator=g).to(dtype)           # key and value inside a wider row
    k, v = fused[:, 1], fused[:, 2]
    slots = torch.randperm(s.cache.num_blocks * page, generator=g)[:T]
    slots[T // 2:T // 2 + 3] = -1 if T > 3 else slots[T // 2:T // 2 + 3]
    want_k, want_v = s.k.clone(), s.v.clone()
    for t, slot in enumerate(slots.tolist()):
        if slot >= 0:
            want_k[slot // page, slot % page], want_v[slot // page, slot % page] = k[t], v[t]
    dev = fused.cuda()
    s.cache.write(dev[:, 1], dev[:, 2], slots.cuda())
    bits = lambda t: t.contiguous().view(torch.int16)  # noqa: E731  NaN rows included: nothing else was touched
    assert torch.equal(bits(s.cache.key_cache.cpu()), bits(want_k)) and torch.equal(bits(s.cache.value_cache.cpu()), bits(want_v))
    assert s.cache.status() == 0
    if T > 3:      # rows that lie between 16-byte boundaries are copied first; key and value of other strides
        odd = torch.zeros(T * H * D + 1, dtype=dtype, device="cuda")[1:].view(T, H, D)
        odd.copy_(dev[:, 2])
        s.cache.write(odd, dev[:, 1], slots.cuda())
        assert torch.equal(s.cache.key_cache.cpu()[slots[0] // page, slots[0] % page], v[0])
        assert torch.equal(s.cache.value_cache.cpu()[slots[0] // page, slots[0] % page], k[0])
        bad = slots.clone()
        bad[0], bad[1] = s.cache.num_blocks * page, 2 ** 62
        s.cache.write(dev[:, 1], dev[:, 2], bad.cuda())
        assert s.cache.status() == RANGE


@pytest.mark.parametrize("lens,W,H,G,D,page,dtype", [
    ([1], 1, 1, 1, 128, 16, BF16), ([127, 128, 129, 0, 5], 16, 2, 4, 128, 16, BF16), ([1000], 32, 2, 4, 128, 16, BF16),
    ([700, 20], 33, 1, 5, 64, 7, FP16), ([300, 4], 70, 2, 8, 64, 32, BF16), ([2000], 8, 1, 8, 256, 24, BF16),
    ([6001, 3000], 64, 2, 2, 128, 128, FP16), ([513], 300, 1, 1, 256, 1, FP16),
])
def test_observe(lens, W, H, G, D, page, dtype):
    s = Setup(lens, H, D, page, dtype, seed=11)
    q = s.query(len(lens), W, heads=H * G)
    led = ledger_of(s, slots=s.longest + 3)
    before = led.mass.cpu().double()
    s.cache.observe(q.cuda(), s.dtable, s.dlens, s.longest, led)
    mass = led.mass.cpu().double()
    assert s.cache.status() == 0
    for b, n in enumerate(lens):
        assert torch.equal(mass[b, :, n:], before[b, :, n:])
        if n == 0:
            continue
        k, v = s.rows(b)
        qb = q[b].double().view(W, H, G, D)
        _, p = O.attention(qb, k, v, last=torch.arange(n - W, n))
        add, rel = p.sum((0, 2)), weight_error(qb, k, D ** -0.5)
        # sums of up to W G weights in 32 bits, one addition per row tile to the mass
        many = (W * G + 2 + W * G // 128) * 2.0 ** -24
        assert ((mass[b, :, :n] - before[b, :, :n] - add).abs() <= add * (rel + many) + (mass[b, :, :n]) * 2.0 ** -23 * (1 + W * G // 128)).all()


@pytest.mark.parametrize("scale", [0.0, -0.05, 0.3])
def test_scales_of_either_sign(scale):
    """No scale at all (equal weights), a negative one, a large one; the last tile is a partial one and has a bad page."""
    s = Setup([300, 129], 2, 128, seed=14)
    table = s.table.clone()
    table[0, 3] = -1
    there = torch.ones(300, dtype=torch.bool)
    there[48:64] = False
    q = s.query(2, 4, heads=8)
    a, b = AttentionLedger(2, 2, s.longest, "cuda"), AttentionLedger(2, 2, s.longest, "cuda")
    s.cache.observe(q.cuda(), table.cuda(), s.dlens, s.longest, a, scale=scale)
    out = s.cache.decode(q[:, 3].cuda(), table.cuda(), s.dlens, s.longest, scale=scale, ledger=b).cpu().double()
    for i, n in enumerate(s.lens):
        k, v = s.rows(i)
        ok = there[:n] if i == 0 else torch.ones(n, dtype=torch.bool)
        rel = weight_error(q.double(), k, abs(scale))
        _, p = O.attention(q[i].double().view(4, 2, 4, 128), k, v, scale=scale, last=torch.arange(n - 4, n), there=ok)
        ref, p1 = O.attention(q[i, 3].double().view(1, 2, 4, 128), k, v, scale=scale, there=ok)
        check_out(out[i].view(1, 2, 4, 128), ref, p1, v, BF16, rel)
        for led, add in ((a, p.sum((0, 2))), (b, p1[0].sum(1))):
            assert ((led.mass[i, :, :n].cpu().double() - add).abs() <= add * (rel + 2.0 ** -19)).all()
    assert s.cache.status() == RANGE


def test_observing_one_query_is_what_decode_adds():
    s = Setup([400, 77], 2, 128, seed=4)
    q = s.query(2, heads=8).cuda()
    a, b = ledger_of(s), ledger_of(s)
    s.cache.decode(q, s.dtable, s.dlens, s.longest, ledger=a)
    s.cache.observe(q[:, None], s.dtable, s.dlens, s.longest, b)
    # two ways of adding the same products: the bound of either, twice
    rel = 2 * weight_error(q.cpu().double(), s.rows(0)[0], 128 ** -0.5)
    assert ((a.mass - b.mass).abs() <= 8 * rel + a.mass * 2.0 ** -22).all()


def _evict_reference(s, led, lens, budget, recent):
    """Planes, mass, positions, held and seen after the rule, from the state before."""
    k, v = s.cache.key_cache.cpu().clone(), s.cache.value_cache.cpu().clone()
    mass, pos = led.mass.cpu(), led.positions.cpu()
    held, seen = led.held.tolist(), led.seen.tolist()
    new_mass, new_pos = torch.zeros_like(mass), torch.full_like(pos, -1)
    new_lens, new_seen = [], []
    for b, n in enumerate(lens):
        r = O.rows(s.table[b], n, s.page)
        for h in range(s.H):
            source, at = O.evict(mass[b, h, :n].tolist(), pos[b, h, :n].tolist(), held[b], seen[b], n, budget, recent)
            m = len(source)
            new_mass[b, h, :m], new_pos[b, h, :m] = mass[b, h, source], torch.tensor(at, dtype=torch.int32)
            for plane in (k, v):
                to = [t for t in range(m) if source[t] != t]
                if to:
                    rt, rf = r[to], r[[source[t] for t in to]]
                    plane[rt // s.page, rt % s.page, h] = plane[rf // s.page, rf % s.page, h]
        new_lens.append(min(n, budget))
        new_seen.append(seen[b] + n - held[b])
    return k, v, new_mass, new_pos, new_lens, new_seen


def same_bits(a, b):
    view = {2: torch.int16, 4: torch.int32}[a.element_size()]
    return torch.equal(a.contiguous().cpu().view(view), b.contiguous().cpu().view(view))


@pytest.mark.parametrize("lens,budget,recent,D,H,page,slots", [
    ([300], 256, 32, 128, 2, 16, 300), ([40, 0, 5, 64, 65], 64, 64, 64, 3, 7, 70), ([100, 90], 1, 1, 128, 1, 16, 128),
    ([100, 3], 0, 0, 128, 2, 16, 100), ([33, 2048, 2049, 1500], 1000, 0, 64, 1, 16, 2049), ([5000, 8192], 700, 100, 64, 1, 32, 8192),
    ([8193, 9000, 20], 4096, 300, 64, 1, 16, 9001), ([20011], 19000, 19000, 64, 1, 64, 20011), ([40000, 1500], 1000, 64, 64, 1, 128, 40000),
    ([70001], 3000, 100, 64, 1, 128, 70100), ([50, 60], 500, 20, 256, 2, 24, 60),
])
@pytest.mark.parametrize("in_place", [True, False])
def test_evict(lens, budget, recent, D, H, page, slots, in_place):
    """Three rounds, with tokens appended between them, so that positions of all kinds occur; ties and zeros among the masses."""
    s = Setup(lens, H, D, page, seed=6)
    led, now = AttentionLedger(len(lens), H, slots, "cuda"), list(lens)
    g = torch.Generator().manual_seed(9)
    for turn in range(3):
        mass = torch.rand(led.mass.shape, generator=g)
        mass = torch.where(torch.rand(mass.shape, generator=g) < 0.2, (mass * 4).round() / 4, mass)
        for b, n in enumerate(now):
            mass[b, :, n:] = 0
        led.mass.copy_(mass)
        dl = torch.tensor(now, dtype=torch.int32, device="cuda")
        k, v, nm, np_, nl, ns = _evict_reference(s, led, now, budget, recent)
        other = None if in_place else AttentionLedger(len(lens), H, slots, "cuda")
        if other is not None:
            other.mass.fill_(5.0), other.positions.fill_(77)
        kept = [t.clone() for t in led._tensors]
        got = s.cache.evict(s.dtable, dl, s.longest, led, budget, recent, out=other)
        if other is not None:
            assert all(torch.equal(a, c) for a, c in zip(kept, led._tensors))
            led = other
        assert got.tolist() == nl == led.held.tolist() and led.seen.tolist() == ns and dl.tolist() == now
        assert torch.equal(led.positions.cpu(), np_) and same_bits(led.mass, nm)
        assert same_bits(s.cache.key_cache, k) and same_bits(s.cache.value_cache, v)
        now = [min(n, m + 1 + 7 * turn) for n, m in zip(lens, nl)]     # tokens arrive in the slots behind (their rows are there)
    assert s.cache.status() == 0


def test_evict_orders_masses_of_every_kind():
    """NaN above infinity above numbers, -0 equal to 0, ties to the lower slot, and the latest whatever they have."""
    s = Setup([12], 1, 64)
    led = AttentionLedger(1, 1, 12, "cuda")
    inf, nan = math.inf, math.nan
    led.mass.copy_(torch.tensor([0.0, -0.0, 3.0, nan, -1.0, inf, 3.0, -inf, 0.0, 3.0, 1e-40, -5.0]).view(1, 1, 12))
    k, v, nm, np_, nl, ns = _evict_reference(s, led, [12], 6, 1)
    s.cache.evict(s.dtable, s.dlens, 12, led, 6, 1)
    assert sorted(led.positions[0, 0, :6].tolist()) == [2, 3, 5, 6, 9, 11]
    assert torch.equal(led.positions.cpu(), np_) and same_bits(led.mass, nm) and same_bits(s.cache.key_cache, k)


def test_evict_when_more_are_recent_than_fit_the_rule():
    """Positions that a caller wrote: more of them count as recent than the budget holds; then the masses decide among those."""
    s = Setup([64], 1, 64)
    led = AttentionLedger(1, 1, 64, "cuda")
    led.held.fill_(64), led.seen.fill_(1000), led.positions.fill_(999)
    led.mass.copy_(torch.rand(1, 1, 64, generator=torch.Generator().manual_seed(0)))
    want = _evict_reference(s, led, [64], 10, 3)
    s.cache.evict(s.dtable, s.dlens, 64, led, 10, 3)
    assert same_bits(led.mass, want[2]) and same_bits(s.cache.key_cache, want[0])


def test_evict_reports_a_bad_page_and_moves_the_rest():
    s = Setup([64], 1, 64)
    led = AttentionLedger(1, 1, 64, "cuda")
    led.mass.copy_(torch.arange(64.0).view(1, 1, 64))           # the last 32 stay and move to the first 32 slots
    table = s.table.clone()
    table[0, 3] = -1                                            # slots 48..63
    before = s.cache.key_cache.clone()
    s.cache.evict(table.cuda(), s.dlens, 64, led, 32)
    assert s.cache.status() == RANGE
    rows = lambda plane: plane.flatten(0, 1)[O.rows(s.table[0], 64, 16).cuda()]  # noqa: E731
    assert torch.equal(rows(s.cache.key_cache)[:16], rows(before)[32:48]) and torch.equal(rows(s.cache.key_cache)[16:], rows(before)[16:])


def test_every_token_is_counted_once():
    """Lengths that put the borders of shares, warps and sequences in all places to each other: a step's weights sum to the
    number of query heads, and the outputs follow for values that are all ones."""
    rng = random.Random(17)
    for i in range(60):
        D, H, G = rng.choice((64, 128, 256)), rng.randint(1, 3), rng.choice((1, 4, 8, 11))
        top = rng.choice((60, 400, 3000, 20000))
        lens = [rng.randint(1, top) for _ in range(rng.choice((1, 2, 3, 9, 33)))]
        while sum(lens) > 60000:
            lens.pop()
        s = Setup(lens, H, D, rng.choice((16, 64)), seed=i)
        ones = torch.ones_like(s.cache.value_cache)
        cache = PagedKVCache(s.spec, s.cache.key_cache, ones)
        led = AttentionLedger(len(lens), H, s.longest, "cuda")
        out = cache.decode(s.query(len(lens), heads=H * G).cuda(), s.dtable, s.dlens, s.longest, ledger=led)
        # weights are off by 2^-20 or so each, sums of up to 20000 of them in 64 bits
        assert ((led.mass.double().sum(-1) - G).abs() <= G * 2.0 ** -15).all(), (i, lens)
        assert ((out.double() - 1).abs() <= 2.0 ** -8).all() and cache.status() == 0


def test_two_captured_graphs_and_an_eager_stream_at_once():
    """Calls captured twice and replayed at the same time, beside eager calls on a third stream: each has memory of its own."""
    s = Setup([9000, 4000], 2, 128, seed=12)
    qs = [s.query(2, heads=8).cuda() for _ in range(3)]
    want = [s.cache.decode(q, s.dtable, s.dlens, s.longest) for q in qs]
    graphs, outs, masses = [], [], []
    for q in qs[:2]:
        led = AttentionLedger(2, 2, s.longest, "cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(s.cache.decode(q, s.dtable, s.dlens, s.longest, ledger=led))
        graphs.append(graph)
        masses.append(led.mass)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            third = s.cache.decode(qs[2], s.dtable, s.dlens, s.longest)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(third, want[2])
    for m in masses:      # twenty steps' weights of four query heads: additions in 32 bits
        assert ((m.double().sum(-1) - 80).abs() <= 80 * 2.0 ** -13).all()


def test_a_captured_step_follows_the_lengths():
    """Write, decode with the ledger and evict captured once, replayed as the sequence grows: lengths are read on the device."""
    H, D, n, budget = 2, 128, 40, 32
    s = Setup([64], H, D, seed=13)
    led = AttentionLedger(1, H, 64, "cuda")
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    k, v, q = (torch.empty(1, h, D, dtype=BF16, device="cuda") for h in (H, H, 4 * H))
    slot = torch.zeros(1, dtype=torch.int64, device="cuda")

    def step():
        lens.add_(1)
        slot.copy_(s.dtable[0].gather(0, ((lens - 1) // 16).long()) * 16 + (lens - 1) % 16)
        s.cache.write(k, v, slot)
        out = s.cache.decode(q, s.dtable, lens, 64, ledger=led)
        lens.copy_(s.cache.evict(s.dtable, lens, 64, led, budget, 8))
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for t in (k, v, q):
            t.normal_()
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(5):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=s.gen).to(BF16))
        rows = O.rows(s.table[0], 33, 16)
        keys, values = (p.cpu().flatten(0, 1)[rows[:32]].double() for p in (s.cache.key_cache, s.cache.value_cache))
        keys, values = torch.cat([keys, k.cpu().double()]), torch.cat([values, v.cpu().double()])
        graph.replay()
        ref, p = O.attention(q.cpu().double().view(1, H, 4, D), keys, values)
        check_out(out.cpu().double().view(1, H, 4, D), ref, p, values, BF16, weight_error(q.cpu().double(), keys, D ** -0.5))
        assert lens.item() == 32 and led.seen.item() == 40 + 1 + i + 1
        assert (led.positions[0, :, :32] >= led.seen.item() - 8).sum(-1).tolist() == [8, 8]
    assert s.cache.status() == 0


def test_a_prompt_evicted_then_compressed():
    """The calls together: a prompt written, observed, evicted; steps with the ledger; another eviction; what is left compressed
    from the same pages - and attention over it as over the kept rows compressed by hand."""
    H, G, D, n, page = 2, 4, 128, 700, 16
    dev = torch.device("cuda")
    g = torch.Generator().manual_seed(21)
    cache = PagedKVCache.allocate(ExactCacheSpec(D, H), 64, dev)
    table = torch.randperm(64, generator=g)[:50].int().view(1, 50).cuda()
    rnd = lambda *shape: torch.randn(*shape, generator=g).to(BF16)  # noqa: E731
    all_k, all_v = rnd(n + 40, H, D), rnd(n + 40, H, D)
    led = AttentionLedger(1, H, 800, dev)

    def put(first, count, at):
        t = torch.arange(at, at + count, device=dev)
        cache.write(all_k[first:first + count].cuda(), all_v[first:first + count].cuda(), table[0, t // page].long() * page + t % page)

    put(0, n, 0)
    lens = torch.tensor([n], dtype=torch.int32, device=dev)
    cache.observe(rnd(1, 16, H * G, D).cuda(), table, lens, n, led)
    assert ((led.mass.double().sum(-1) - 16 * G).abs() < 16 * G * 2.0 ** -13).all()
    lens = cache.evict(table, lens, n, led, 256, 32)
    for i in range(40):
        put(n + i, 1, 256 + i)
        lens += 1
        q = rnd(1, H * G, D)
        out = cache.decode(q.cuda(), table, lens, 300, ledger=led)
    lens = cache.evict(table, lens, 300, led, 250, 32)
    assert lens.tolist() == [250] and led.seen.tolist() == [740] and cache.status() == 0
    pos = led.positions[0, :, :250].cpu().long()
    for h in range(H):
        assert len(set(pos[h].tolist())) == 250 and set(range(708, 740)) <= set(pos[h].tolist())
    kept_k = torch.stack([all_k[pos[h], h] for h in range(H)], 1)
    kept_v = torch.stack([all_v[pos[h], h] for h in range(H)], 1)
    rows = O.rows(table[0].cpu(), 250, page)
    assert torch.equal(cache.key_cache.flatten(0, 1).cpu()[rows], kept_k) and torch.equal(cache.value_cache.flatten(0, 1).cpu()[rows], kept_v)
    ref, p = O.attention(q[0].double().view(1, H, G, D), kept_k.double(), kept_v.double())
    out = cache.decode(q.cuda(), table, lens, 250)
    check_out(out.cpu().double().view(1, H, G, D), ref, p, kept_v.double(), BF16, weight_error(q.double(), kept_k.double(), D ** -0.5))
    a, b = (CompressedKVStore(D, H, device=dev) for _ in range(2))
    a.append_from_paged(cache.key_cache, cache.value_cache, table[0], 250)
    b.append_chunk(kept_k.cuda(), kept_v.cuda())
    assert torch.equal(compute_hybrid_attention(q.cuda(), a, None, None, H * G), compute_hybrid_attention(q.cuda(), b, None, None, H * G))


def test_more_sequences_than_a_cta_has_threads():
    """Lengths are looked at 256 at a time; every third sequence is empty."""
    rng = random.Random(3)
    lens = [0 if i % 3 == 0 else rng.randint(1, 70) for i in range(700)]
    s = Setup(lens, 2, 64, 16, FP16, seed=30)
    led, led2 = AttentionLedger(700, 2, s.longest, "cuda"), AttentionLedger(700, 2, s.longest, "cuda")
    q, win = s.query(700, heads=4), s.query(700, 3, heads=4)
    out = s.cache.decode(q.cuda(), s.dtable, s.dlens, s.longest, ledger=led).cpu().double()
    s.cache.observe(win.cuda(), s.dtable, s.dlens, s.longest, led2)
    for b in range(0, 700):
        k, v = s.rows(b)
        qb = q[b].double().view(1, 2, 2, 64)
        ref, p = O.attention(qb, k, v)
        rel = weight_error(qb, k, 64 ** -0.5)
        check_out(out[b].view(1, 2, 2, 64), ref, p, v, FP16, rel)
        if lens[b]:
            _, pw = O.attention(win[b].double().view(3, 2, 2, 64), k, v, last=torch.arange(lens[b] - 3, lens[b]))
            for m, add in ((led.mass, p[0].sum(1)), (led2.mass, pw.sum((0, 2)))):
                assert ((m[b, :, :lens[b]].cpu().double() - add).abs() <= add * (rel + 2.0 ** -20)).all()
    for m in (led, led2):
        m.mass.copy_(torch.rand(m.mass.shape, generator=s.gen))
    want = _evict_reference(s, led, lens, 20, 5)
    got = s.cache.evict(s.dtable, s.dlens, s.longest, led, 20, 5)
    assert got.tolist() == want[4] and same_bits(led.mass, want[2]) and same_bits(s.cache.key_cache, want[0]) and s.cache.status() == 0


def test_planes_beyond_four_gigabytes():
    """Pages at the end of planes of 2^32 bytes and more each: every kernel's offsets pass 32 bits."""
    H, D, page = 8, 128, 16
    blocks = (2 ** 32 + 2 ** 27) // (page * H * D * 2)
    planes = torch.zeros(2, blocks, page, H, D, dtype=BF16, device="cuda")
    cache = PagedKVCache(ExactCacheSpec(D, H), planes[0], planes[1])
    n, g = 100, torch.Generator().manual_seed(2)
    table = torch.arange(blocks - 7, blocks, dtype=torch.int32, device="cuda").flip(0).view(1, 7)
    t = torch.arange(n, device="cuda")
    k, v = (torch.randn(n, H, D, generator=g).to(BF16) for _ in range(2))
    cache.write(k.cuda(), v.cuda(), table[0, t // page].long() * page + t % page)
    lens, led, led2 = torch.tensor([n], dtype=torch.int32, device="cuda"), AttentionLedger(1, H, n, "cuda"), AttentionLedger(1, H, n, "cuda")
    q = torch.randn(1, 4 * H, D, generator=g).to(BF16)
    out = cache.decode(q.cuda(), table, lens, n, ledger=led)
    cache.observe(q[:, None].cuda(), table, lens, n, led2)
    ref, p = O.attention(q[0].double().view(1, H, 4, D), k.double(), v.double())
    rel = weight_error(q.double(), k.double(), D ** -0.5)
    check_out(out.cpu().double().view(1, H, 4, D), ref, p, v.double(), BF16, rel)
    for m in (led, led2):
        assert ((m.mass[0].cpu().double() - p[0].sum(1)).abs() <= p[0].sum(1) * (rel + 2.0 ** -20)).all()
    kept = torch.sort(torch.argsort(led.mass[0].cpu(), dim=-1, descending=True, stable=True)[:, :50], dim=-1).values
    cache.evict(table, lens, n, led, 50)
    assert torch.equal(torch.sort(led.positions[0, :, :50].cpu().long(), dim=-1).values, kept) and cache.status() == 0
    rows = planes[0].flatten(0, 1)[table[0, t // page].long() * page + t % page].cpu()
    for h in range(H):
        assert torch.equal(rows[:50, h], k[led.positions[0, h, :50].cpu().long(), h])
    assert not planes[0][:64].any()


def test_layouts_of_small_tensors():
    """Lengths and tables as views, a table shared by all rows, more rows of lengths than sequences."""
    s = Setup([70, 70, 70], 2, 128, seed=31)
    q = s.query(3, heads=8).cuda()
    want = s.cache.decode(q, s.dtable, s.dlens, 70)
    lens = torch.tensor([[70, 1], [70, 2], [70, 3], [5, 5]], dtype=torch.int32, device="cuda")[:, 0]
    assert torch.equal(s.cache.decode(q, s.dtable, lens, 70), want)
    shared = s.dtable[:1].expand(3, -1)
    a = s.cache.decode(q, shared, s.dlens, 70)
    assert torch.equal(a[0], want[0]) and not torch.equal(a[1], want[1])
    window = s.query(6, 5, heads=8).cuda()[::2]
    x, y = AttentionLedger(3, 2, 70, "cuda"), AttentionLedger(3, 2, 70, "cuda")
    s.cache.observe(window, shared, s.dlens, 70, x)
    s.cache.observe(window.contiguous(), shared.contiguous(), s.dlens, 70, y)
    assert torch.equal(x.mass, y.mass) and s.cache.status() == 0


def test_a_cache_made_and_used_on_another_stream():
    side = torch.cuda.Stream()
    s = Setup([500, 30], 2, 128, seed=32)
    q = s.query(2, heads=8).cuda()
    want = s.cache.decode(q, s.dtable, s.dlens, 500)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        cache = PagedKVCache(s.spec, s.cache.key_cache, s.cache.value_cache)
        outs = [cache.decode(q, s.dtable, s.dlens, 500) for _ in range(5)]
    side.synchronize()
    assert all(torch.equal(o, want) for o in outs) and cache.status() == 0


def test_a_long_trim_captured():
    """A cluster of CTAs a row, replayed: the same trim each time, since the ledger it reads is left alone."""
    s = Setup([20000, 100], 1, 64, 128, seed=33)
    led, out = AttentionLedger(2, 1, 20000, "cuda"), AttentionLedger(2, 1, 20000, "cuda")
    led.mass.copy_(torch.rand(led.mass.shape, generator=s.gen))
    want = _evict_reference(s, led, s.lens, 3000, 50)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lens = s.cache.evict(s.dtable, s.dlens, 20000, led, 3000, 50, out=out)
    for _ in range(3):
        out.mass.fill_(3.0)
        graph.replay()
    torch.cuda.synchronize()
    assert lens.tolist() == want[4] and same_bits(out.mass, want[2]) and torch.equal(out.positions.cpu(), want[3])
    assert same_bits(s.cache.key_cache, want[0]) and same_bits(s.cache.value_cache, want[1])


def test_random_batches():
    """Lengths, heads, pages and types at random: decode with a ledger against 64 bits."""
    rng = random.Random(5)
    for i in range(12):
        D, H, G = rng.choice((64, 128, 256)), rng.randint(1, 4), rng.choice((1, 3, 4, 8, 9, 16, 20))
        lens = [rng.choice((0, rng.randint(1, 40), rng.randint(1, 1500))) for _ in range(rng.randint(1, 30))]
        s = Setup(lens, H, D, rng.choice((1, 5, 16, 16, 48)), rng.choice((BF16, FP16)), seed=100 + i)
        q = s.query(len(lens), heads=H * G)
        led = AttentionLedger(len(lens), H, s.longest, "cuda")
        out = s.cache.decode(q.cuda(), s.dtable, s.dlens, s.longest, ledger=led).cpu().double()
        for b, n in enumerate(lens):
            k, v = s.rows(b)
            qb = q[b].double().view(1, H, G, D)
            ref, p = O.attention(qb, k, v)
            rel = weight_error(qb, k, D ** -0.5)
            check_out(out[b].view(1, H, G, D), ref, p, v, s.dtype, rel)
            assert ((led.mass[b, :, :n].cpu().double() - p[0].sum(1)).abs() <= p[0].sum(1) * (rel + G * 2.0 ** -23)).all()
        assert s.cache.status() == 0
