"""The exact paged cache on the GPU where its numbers, lengths and layouts come to their ends, against 64-bit torch."""

import math

import pytest
import torch

from tests import pages_oracle as O
from turboquant_b200 import AttentionLedger, CompressedCacheSpec, CompressedPagedKVCache, ExactCacheSpec, PagedKVCache

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
RANGE = -7


def cache_over(k, v, page, seed=0):
    """A cache that holds k / v (batch, n, H, D) in pages in random order -> cache, table, lengths (all n)."""
    b, n, h, d = k.shape
    width = -(-n // page)
    cache = PagedKVCache.allocate(ExactCacheSpec(d, h, block_size=page, dtype=k.dtype), b * width, "cuda")
    table = torch.randperm(b * width, generator=torch.Generator().manual_seed(seed)).int().view(b, width)
    for plane, x in ((cache.key_cache, k), (cache.value_cache, v)):
        padded = torch.zeros(b, width * page, h, d, dtype=k.dtype)
        padded[:, :n] = x
        plane[table.flatten().long().cuda()] = padded.view(b * width, page, h, d).cuda()
    return cache, table.cuda(), torch.full((b,), n, dtype=torch.int32, device="cuda")


def score_error(q, k, scale):
    """Relative error of a softmax weight: a score is a sum of exact products held in 32 bits, at most D / 16 <= 16 additions that
    lose 2^-22 of the largest partial sum each, once in the score and once in the reference of the normalisation; exponentials
    and sums lose some 2^-20."""
    size = (q.abs().amax() * k.abs().sum(-1).amax()).item() * scale
    return 2 * 16 * 2.0 ** -22 * size + 2.0 ** -19


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("D,H,G,b,n", [(128, 4, 4, 300, 200), (64, 2, 16, 280, 330), (256, 2, 1, 200, 250), (128, 1, 2, 1, 20011)])
def test_small_weights_under_a_large_one_with_no_value(D, H, G, b, n, dtype):
    """The first token of sequence b lies b % 28 octaves above the others and has a value of zeros: what is left of the output are
    the small weights."""
    g = torch.Generator().manual_seed(D + n)
    q, k = torch.zeros(b, H * G, D), torch.zeros(b, n, H, D)
    q[..., 1:], k[..., 1:] = 0.5 * torch.randn(b, H * G, D - 1, generator=g), 0.3 * torch.randn(b, n, H, D - 1, generator=g)
    q[..., 0] = 8.0
    octaves = torch.arange(b) % 28 if b > 1 else torch.tensor([24])
    k[:, 0, :, 0] = (octaves * math.log(2.0) * math.sqrt(D) / 8.0)[:, None]
    v = 0.5 + torch.randn(b, n, H, D, generator=g)
    v[:, 0] = 0.0
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    cache, table, lens = cache_over(k, v, 16)
    led = AttentionLedger(b, H, n, "cuda")
    out = cache.decode(q.cuda(), table, lens, n).cpu().double().view(b, H, G, D)
    assert torch.equal(cache.decode(q.cuda(), table, lens, n, ledger=led).cpu().double().view(b, H, G, D), out)
    p = torch.softmax(torch.einsum("bhgd,bnhd->bhgn", q.double().view(b, H, G, D), k.double()) / math.sqrt(D), -1)
    ref, size = torch.einsum("bhgn,bnhd->bhgd", p, v.double()), torch.einsum("bhgn,bnhd->bhgd", p, v.double().abs())
    rel = score_error(q.double(), k.double(), D ** -0.5)
    # The output's rounding is half a step; a weight of two 16-bit numbers is off by 2^-18 (bf16) or 2^-22 (fp16) of itself, or
    # where fp16 ends, 2^-15 2^-25 = 2^-40 of the largest weight, which is at most 1; sums of 32 bits, at most n / 16 times two
    # additions in a chain that lose 2^-22 of the magnitudes each.
    lost = size * (rel + 2.0 ** -18 + n / 8 * 2.0 ** -22) + (2.0 ** -40 if dtype is FP16 else 0.0) * v.double().abs().sum(1).view(b, H, 1, D)
    half = ref.abs() * torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -6) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    over = ((out - ref).abs() - lost - half).amax((1, 2, 3))
    assert (over <= 0).all(), (over.max().item(), octaves[over > 0].unique().tolist())
    added = p.sum(2)
    assert ((led.mass.cpu().double() - added).abs() <= added * (rel + (G + 1) * 2.0 ** -24)).all() and cache.status() == 0


@pytest.mark.parametrize("which", ["returned", "held"])
def test_lengths_of_an_eviction_go_straight_into_the_compressed_cache(which):
    """The lengths that an eviction writes, read by the launch behind it: the same bits as with lengths that lay there before."""
    b, h, n = 40, 2, 600
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(b, n, h, 128, generator=g).to(BF16) for _ in range(2))
    exact, table, lens = cache_over(k, v, 16)
    packed = CompressedPagedKVCache.allocate(CompressedCacheSpec(128, h, 3, 2), b * 40, "cuda")
    slots = torch.cat([torch.arange(n) + 640 * i for i in range(b)]).cuda()
    packed.write(k.view(-1, h, 128).cuda(), v.view(-1, h, 128).cuda(), slots)
    tables = torch.arange(b * 40, dtype=torch.int32, device="cuda").view(b, 40)
    q = torch.randn(b, 4 * h, 128, generator=g).to(BF16).cuda()
    led = AttentionLedger(b, h, n, "cuda")
    wants = {}
    for budget in (500, 17, 333):
        wants[budget] = packed.decode(q, tables, torch.full((b,), budget, dtype=torch.int32, device="cuda"), n).clone()
    assert not torch.equal(wants[500], wants[17])
    for i in range(30):
        budget = (500, 17, 333)[i % 3]
        led.reset()
        torch.full((b,), 10 ** 6 + i, dtype=torch.int32, device="cuda")       # what the new lengths' memory held before
        new = exact.evict(table, lens, n, led, budget)
        got = packed.decode(q, tables, new if which == "returned" else led.held, n)
        assert torch.equal(got, wants[budget]) and packed.workspace.status() == 0


def test_observing_after_an_eviction():
    """A second prompt of a chat: windows of the tokens that came after the eviction see all that is held and each other up to their
    own; queries further back give nothing and are reported.  A sequence that nothing was evicted from stays as it was."""
    H, G, D, W = 2, 4, 128, 12
    n = torch.tensor([400, 90, 300, 64])
    g = torch.Generator().manual_seed(8)
    k, v = torch.randn(4, 400, H, D, generator=g).to(BF16), torch.randn(4, 400, H, D, generator=g).to(BF16)
    cache, table, _ = cache_over(k, v, 16)
    led = AttentionLedger(4, H, 400, "cuda")
    led.mass.copy_(torch.rand(4, H, 400, generator=g))
    lens = cache.evict(table, n.int().cuda(), 400, led, 100, 10)      # 100 of 400, 90 as they are, 100 of 300, 64 as they are
    assert lens.tolist() == [100, 90, 100, 64]
    for more, early in (([12, 0, 40, 3], False), ([5, 1, 0, 12], True)):
        now = lens + torch.tensor(more, dtype=torch.int32, device="cuda")      # slots behind hold rows already
        led.mass.zero_()
        q = torch.randn(4, W, H * G, D, generator=g).to(BF16)
        cache.observe(q.cuda(), table, now, 400, led)
        assert cache.status() == (RANGE if early else 0)
        for b, m in enumerate(now.tolist()):
            rows = [O.gather(plane.cpu(), table[b].cpu(), m, 16) for plane in (cache.key_cache, cache.value_cache)]
            last = torch.arange(m - W, m)
            if b % 2 == 0:
                last = torch.where(last < 100, -1, last)
            qb = q[b].double().view(W, H, G, D)
            _, p = O.attention(qb, *rows, last=last)
            add, rel = p.sum((0, 2)), score_error(qb, rows[0], D ** -0.5)
            got = led.mass[b].cpu().double()
            assert ((got[:, :m] - add).abs() <= add * (rel + (W * G + 2) * 2.0 ** -24)).all() and not got[:, m:].any()
            assert abs(got.sum().item() - H * G * (last >= 0).sum().item()) <= 1e-3 * W * H * G


def test_observing_after_an_eviction_with_many_rows():
    """Windows of several row tiles, of which the first lie wholly in the part that is in no order."""
    H, G, D, W, n = 1, 8, 64, 70, 513
    g = torch.Generator().manual_seed(9)
    k, v = torch.randn(1, n, H, D, generator=g).to(FP16), torch.randn(1, n, H, D, generator=g).to(FP16)
    cache, table, lens = cache_over(k, v, 32)
    for held, seen in ((480, 481), (500, 2000), (513, 600), (600, 700), (480, 480), (0, 0)):
        led = AttentionLedger(1, H, n, "cuda")
        led.held.fill_(held), led.seen.fill_(seen)
        q = torch.randn(1, W, H * G, D, generator=g).to(FP16)
        cache.observe(q.cuda(), table, lens, n, led)
        evicted = seen != held
        assert cache.status() == (RANGE if evicted and held > n - W else 0)
        last = torch.arange(n - W, n)
        if evicted:
            last = torch.where(last < held, -1, last)
        _, p = O.attention(q[0].double().view(W, H, G, D), k[0].double(), v[0].double(), last=last)
        add, rel = p.sum((0, 2)), score_error(q.double(), k.double(), D ** -0.5)
        assert ((led.mass[0].cpu().double() - add).abs() <= add * (rel + (W * G + W * G // 128 + 2) * 2.0 ** -24)).all()


@pytest.mark.parametrize("W,G", [(4, 4), (40, 4), (1, 1)])
def test_a_key_that_is_not_a_number(W, G):
    """Every weight of a query that sees it is NaN, in whatever part of the sequence it lies; other sequences and rows are not touched."""
    H, D, n = 2, 128, 5000
    g = torch.Generator().manual_seed(W)
    k, v = torch.randn(3, n, H, D, generator=g).to(BF16), torch.randn(3, n, H, D, generator=g).to(BF16)
    k[0, 1024:1152, 1] = math.nan             # a tile of the product
    k[1, 4000, 0, 7] = math.nan
    cache, table, lens = cache_over(k, v, 16)
    q = torch.randn(3, W, H * G, D, generator=g).to(BF16)
    seen, step = AttentionLedger(3, H, n, "cuda"), AttentionLedger(3, H, n, "cuda")
    cache.observe(q.cuda(), table, lens, n, seen)
    out = cache.decode(q[:, -1].cuda(), table, lens, n, ledger=step).cpu().view(3, H, G, D)
    whole = torch.tensor([[0, 1], [1, 0], [0, 0]], dtype=torch.bool)
    for mass in (seen.mass.cpu(), step.mass.cpu()):
        nan = torch.isnan(mass)
        nan[:, :, n - W:] |= whole[..., None]      # a window's own tokens: not all queries see them, the last one does
        assert torch.equal(nan.all(-1), whole) and torch.equal(nan.any(-1), whole)
    assert torch.equal(torch.isnan(out).all(-1).all(-1), whole) and torch.equal(torch.isnan(out).any(-1).any(-1), whole)
    assert cache.status() == 0


def test_a_ledgers_scratch_memory_is_bounded():
    """Lengths of a few hundred under a bound of 2^20 tokens, as a captured step has it: 64 query heads would keep 268 MB of scores a
    sequence.  The batch goes through in slices; a slice may be one sequence, and sequences may be empty."""
    H, G, D, most = 2, 32, 64, 2 ** 20
    g = torch.Generator().manual_seed(11)
    k, v = torch.randn(7, 700, H, D, generator=g).to(BF16), torch.randn(7, 700, H, D, generator=g).to(BF16)
    cache, table, _ = cache_over(k, v, 16)
    wide = torch.full((7, most // 16), -1, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    n = [500, 0, 33, 1, 700, 16, 257]
    lens = torch.tensor(n, dtype=torch.int32, device="cuda")
    q = torch.randn(7, H * G, D, generator=g).to(BF16)
    led = AttentionLedger(7, H, most, "cuda")
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = cache.decode(q.cuda(), wide, lens, most, ledger=led)
    assert torch.cuda.max_memory_allocated() - before < 2 ** 29 + 2 ** 26
    assert cache.status() == 0
    for b, m in enumerate(n):
        rows = k[b, :m].double(), v[b, :m].double()
        qb = q[b].double().view(1, H, G, D)
        ref, p = O.attention(qb, *rows)
        add, rel = p[0].sum(1), score_error(qb, k.double(), D ** -0.5)
        assert ((led.mass[b, :, :m].cpu().double() - add).abs() <= add * (rel + (G + 1) * 2.0 ** -24)).all() and not led.mass[b, :, m:].any()
        size = torch.einsum("rhgn,nhd->rhgd", p, rows[1].abs())
        bound = ref.abs() * torch.finfo(BF16).eps / 2 * (1 + 2.0 ** -6) + size * (rel + 2.0 ** -18 + (m / 8 + 2) * 2.0 ** -22)
        assert ((out[b].cpu().double().view(1, H, G, D) - ref).abs() <= bound).all()


def test_tensors_with_a_dimension_of_one():
    """One token of padded rows, one kv head, one page, one sequence's table as a column: torch lets such a dimension have any
    stride, and calls the tensor contiguous."""
    g = torch.Generator().manual_seed(3)
    odd = torch.randn(5, 260, generator=g).to(BF16).cuda()
    rows = odd[:, :256].unflatten(1, (2, 128))                    # (5, 2, 128), strides (260, 128, 1)
    cache = PagedKVCache.allocate(ExactCacheSpec(128, 2), 3, "cuda")
    for t in (1, 2, 5):
        slots = torch.arange(t, device="cuda") + 7 * t
        cache.write(rows[:t], rows[:t].flip(1), slots)
        flat = cache.key_cache.flatten(0, 1)[slots], cache.value_cache.flatten(0, 1)[slots]
        assert torch.equal(flat[0], rows[:t]) and torch.equal(flat[1], rows[:t].flip(1))
    planes = torch.zeros(4099, dtype=BF16, device="cuda")[:4096].as_strided((2, 16, 1, 128), (2048, 128, 1, 1))
    single = PagedKVCache(ExactCacheSpec(128, 1), planes, torch.zeros_like(planes))
    one = torch.randn(3, 129, generator=g).to(BF16).cuda().as_strided((3, 1, 128), (128, 131, 1))
    single.write(one, one, torch.tensor([4, 30, 9], device="cuda"))
    assert torch.equal(planes.flatten(0, 1)[[4, 30, 9]], one)
    lens = torch.tensor([9], dtype=torch.int32, device="cuda")
    column = torch.tensor([[1, 5], [7, 7]], dtype=torch.int32, device="cuda").t()[:1, :1]      # (1, 1), strides (1, 2)
    q = torch.randn(1, 4, 128, generator=g).to(BF16).cuda()
    plain = torch.tensor([[1]], dtype=torch.int32, device="cuda")
    assert column.stride(1) != 1 and torch.equal(single.decode(q, column, lens, 16), single.decode(q, plain, lens, 16))
    led = AttentionLedger(1, 1, 16, "cuda")
    single.observe(q[:, None], column, lens, 16, led)
    assert single.evict(column, lens, 16, led, 5).tolist() == [5] and single.status() == 0 and cache.status() == 0


def test_a_bound_of_no_tokens():
    """Lengths beyond it are clamped to nothing and reported by every call, and an empty table will do."""
    k = torch.randn(3, 40, 2, 128, generator=torch.Generator().manual_seed(0)).to(BF16)
    cache, table, lens = cache_over(k, k, 16)
    q, none, empty = torch.ones(3, 8, 128, dtype=BF16, device="cuda"), torch.zeros_like(lens), table[:, :0]
    before = cache.key_cache.clone()
    for now, code in ((none, 0), (lens, RANGE), (torch.tensor([0, 0, -1], dtype=torch.int32, device="cuda"), RANGE)):
        for t in (table, empty):
            led = AttentionLedger(3, 2, 40, "cuda")
            led.mass.fill_(2.0)
            assert not cache.decode(q, t, now, 0, ledger=led).any() and cache.status() == code
            cache.observe(q[:, None], t, now, 0, led)
            assert cache.status() == code and (led.mass == 2.0).all()
            assert cache.evict(t, now, 0, led, 5, 2).tolist() == [0, 0, 0] and cache.status() == code
            assert not led.mass.any() and (led.positions == -1).all() and not led.held.any() and not led.seen.any()
    assert torch.equal(cache.key_cache, before)
    assert not cache.decode(q, empty, lens, 0, out=torch.ones_like(q)).any() and cache.status() == RANGE


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_one_query_observed_adds_what_its_decode_adds(dtype):
    """From no mass at all, every increment against the other's: two ways of adding the same products, each within its bound."""
    H, G, D, n = 2, 4, 128, 900
    g = torch.Generator().manual_seed(17)
    k, v = torch.randn(3, n, H, D, generator=g).to(dtype), torch.randn(3, n, H, D, generator=g).to(dtype)
    cache, table, lens = cache_over(k, v, 16)
    lens[1], lens[2] = 77, 1
    q = torch.randn(3, H * G, D, generator=g).to(dtype)
    a, b = AttentionLedger(3, H, n, "cuda"), AttentionLedger(3, H, n, "cuda")
    cache.decode(q.cuda(), table, lens, n, ledger=a)
    cache.observe(q[:, None].cuda(), table, lens, n, b)
    rel = score_error(q.double(), k.double(), D ** -0.5) + (G + 1) * 2.0 ** -24
    a, b = a.mass.cpu().double(), b.mass.cpu().double()
    assert ((a - b).abs() <= 2 * rel * torch.minimum(a, b) * (1 + 2.0 ** -6)).all()
    assert (a[0] > 0).all() and (a[1, :, :77] > 0).all() and not a[1, :, 77:].any() and cache.status() == 0
    assert ((a.sum(-1) - G).abs() <= G * rel).all()
