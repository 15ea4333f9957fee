"""What the exact paged cache has a GPU do, as cases that can be timed and compared.

Four operators over pages of 16-bit keys and values, (num_blocks, block_size, kv_heads, head_dim) planes:

write     new tokens into the slots an engine chose: a decode step's (one per sequence) or a prompt's.
decode    attention of one new token per sequence over its pages, any mix of lengths; with a ledger, the
          weight every cached token received is added to what it has received before.
observe   the weights of a prompt's last queries alone (no output): what a ledger holds when a prompt is done.
evict     a cache brought down to `budget` tokens: the `recent` latest stay, then those with the largest
          accumulated weight (ties: the lower slot); tokens kept behind the budget move into the holes before it.

`own` false: elementary torch operations in 32 bits on padded batches.  `own` true: the package's calls.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one decode step's new tokens of a batch, scattered: the smallest call, latency alone
        dict(name="write_step_64", op="write", batch=64, lo=1, hi=1, kv_heads=8, head_dim=128, page=16, dtype="bf16"),
        # the tokens of a long prompt
        dict(name="write_prompt_32k", op="write", batch=1, lo=32768, hi=32768, kv_heads=8, head_dim=128, page=16, dtype="bf16"),
        # a handful of short sequences, an empty one possible: launches and latency
        dict(name="decode_5_short", op="decode", batch=5, lo=0, hi=500, kv_heads=8, q_heads=32, head_dim=128, page=16,
             dtype="bf16", ledger=False),
        # one long sequence with wide heads: work split along the sequence and joined
        dict(name="decode_one_32k_d256", op="decode", batch=1, lo=32768, hi=32768, kv_heads=4, q_heads=16, head_dim=256, page=16,
             dtype="bf16", ledger=False),
        # a large batch of short chats, sixteen query heads on each of two kv heads, larger pages
        dict(name="decode_256_chats_fp16", op="decode", batch=256, lo=1, hi=1500, kv_heads=2, q_heads=32, head_dim=128, page=32,
             dtype="fp16", ledger=False),
        # a serving batch of mixed lengths, 64 query heads: the largest call
        dict(name="decode_64_mixed", op="decode", batch=64, lo=1024, hi=32768, kv_heads=8, q_heads=64, head_dim=128, page=16,
             dtype="bf16", ledger=False),
        # a batch whose caches are to be evicted from: the weights are accumulated
        dict(name="decode_ledger_16x8k", op="decode", batch=16, lo=4001, hi=8192, kv_heads=8, q_heads=32, head_dim=128, page=16,
             dtype="bf16", ledger=True),
        # the last 32 queries of one prompt, ragged
        dict(name="observe_5003", op="observe", batch=1, lo=5003, hi=5003, kv_heads=8, q_heads=32, head_dim=128, page=16,
             dtype="bf16", window=32),
        # the last 16 of a batch of long prompts
        dict(name="observe_8_long", op="observe", batch=8, lo=4096, hi=32768, kv_heads=8, q_heads=32, head_dim=128, page=16,
             dtype="bf16", window=16),
        # one short sequence trimmed
        dict(name="evict_300", op="evict", batch=1, lo=300, hi=300, kv_heads=8, head_dim=128, page=16, dtype="bf16", budget=256,
             recent=32, held=256),
        # the usual trim of a batch: 64 tokens have come in since the last one
        dict(name="evict_64_steady", op="evict", batch=64, lo=2112, hi=2112, kv_heads=8, head_dim=128, page=16, dtype="bf16",
             budget=2048, recent=64, held=2048),
        # long prompts cut to an eighth
        dict(name="evict_4_prompts", op="evict", batch=4, lo=20001, hi=32768, kv_heads=8, head_dim=128, page=16, dtype="bf16",
             budget=4096, recent=128, held=0),
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("write", "decode", "decode", "decode", "observe", "evict", "evict"))
    d = rng.choice((64, 128, 128, 256))
    h = rng.choice((1, 2, 3, 4, 8))
    c = dict(op=op, kv_heads=h, head_dim=d, page=rng.choice((16, 16, 32, 64, 128, 1, 7, 24)), dtype=rng.choice(("bf16", "bf16", "fp16")))
    if op == "write":
        if rng.random() < 0.5:
            return dict(c, batch=_log(rng, 1, 512), lo=1, hi=1)
        n = _log(rng, 16, 30000)
        return dict(c, batch=1, lo=n, hi=n)
    hi = _log(rng, 1, 32000)
    batch = _log(rng, 1, 256)
    while batch * hi * h * d > (200_000_000 if op == "decode" else 60_000_000):
        batch, hi = (batch // 2, hi) if batch > 1 else (batch, hi // 2)
    lo = rng.randint(0 if batch >= 4 and hi >= 4 else 1, hi)
    if op == "decode":
        g = rng.choice((1, 2, 4, 4, 5, 7, 8, 16))
        return dict(c, batch=batch, lo=lo, hi=hi, q_heads=h * g, ledger=rng.random() < 0.4)
    if op == "observe":
        g, w = rng.choice((1, 2, 4, 8)), rng.choice((1, 8, 16, 32, 33))
        while batch * hi * h * g * w > 400_000_000:
            batch, hi = (batch // 2, hi) if batch > 1 else (batch, hi // 2)
        return dict(c, batch=batch, lo=max(1, min(lo, hi)), hi=hi, q_heads=h * g, window=w)
    budget = _log(rng, 1, max(1, hi))
    return dict(c, batch=batch, lo=lo, hi=hi, budget=budget, recent=rng.randint(0, budget), held=rng.choice((0, budget)))


def _lengths(c):
    """Lengths of the sequences of a batch: the same for every seed, so that the work is."""
    rng = random.Random(1000003 * c["batch"] + 17 * c["lo"] + c["hi"])
    return [rng.randint(c["lo"], c["hi"]) for _ in range(c["batch"])]


# ---------------------------------------------------------------------------- inputs

def prepare(case, seed):
    c, dt = case, DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    b, h, d, page, lens = c["batch"], c["kv_heads"], c["head_dim"], c["page"], _lengths(c)
    longest = max(max(lens), 1)
    per = -(-longest // page)

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)

    # every sequence has pages of its own, in random order; channels of the keys differ in size
    blocks = b * per
    table = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32).view(b, per)
    spread = torch.exp(0.5 * normal(d, dtype=torch.float32)).to(dt)
    s = dict(case=c, table=table, longest=longest, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    if c["op"] == "write":
        s["key_cache"], s["value_cache"] = (torch.zeros(blocks, page, h, d, dtype=dt, device="cuda") for _ in range(2))
        pos = torch.cat([torch.arange(n, device="cuda") for n in lens])
        seq = torch.repeat_interleave(torch.arange(b, device="cuda"), s["lens"].long())
        if longest == 1:      # a step's token goes anywhere in its page
            pos = torch.randint(0, page, (b,), generator=gen, device="cuda")
        s["slots"] = table[seq, pos // page].long() * page + pos % page
        s["k"], s["v"] = normal(sum(lens), h, d) * spread, normal(sum(lens), h, d)
    else:
        s["key_cache"], s["value_cache"] = normal(blocks, page, h, d).mul_(spread), normal(blocks, page, h, d)
    if c["op"] == "decode":
        s["q"] = normal(b, c["q_heads"], d)
    if c["op"] == "observe":
        s["q"] = normal(b, c["window"], c["q_heads"], d)
    if c["op"] == "evict" or c["op"] == "observe" or c.get("ledger"):
        # weights received so far: a few tokens have most of it, some none at all
        used = torch.arange(longest, device="cuda") < s["lens"][:, None, None]
        weight = torch.exp(2.0 * normal(b, h, longest, dtype=torch.float32))
        if c["op"] != "evict":      # what a few steps leave: of the size of what this one adds
            weight *= c["q_heads"] / h / longest
        some = torch.rand(b, h, longest, generator=gen, device="cuda") > 0.1
        s["mass"] = torch.where(used & some, weight, torch.zeros_like(weight))
        held = torch.clamp(s["lens"], max=c.get("held", 0))
        s["held"], s["seen"] = held, held + 1000 * (held > 0).int()
        # what an eviction leaves: distinct positions below `seen` in some order, -1 behind them
        order = torch.argsort(torch.rand(b, h, longest, generator=gen, device="cuda"), dim=-1).to(torch.int32)
        known = torch.arange(longest, device="cuda") < held[:, None, None]
        rank = torch.argsort(torch.argsort(torch.where(known, order, order + longest), dim=-1), dim=-1).to(torch.int32)
        s["positions"] = torch.where(known, rank, torch.full_like(rank, -1))
        if c["op"] == "evict":
            s["after"] = [torch.empty_like(s[k]) for k in ("mass", "positions", "held", "seen")]
    _handles(s)
    return s


def _handles(s):
    """The cache and the ledger objects that a program keeps over its tensors."""
    if own:
        from turboquant_b200 import AttentionLedger, ExactCacheSpec, PagedKVCache
        c = s["case"]
        spec = ExactCacheSpec(c["head_dim"], c["kv_heads"], block_size=c["page"], dtype=DTYPES[c["dtype"]])
        s["cache"] = PagedKVCache(spec, s["key_cache"], s["value_cache"])
        s["ledger"] = AttentionLedger.over(s["mass"], s["positions"], s["held"], s["seen"]) if "mass" in s else None
        if "after" in s:
            s["ledger_after"] = AttentionLedger.over(*s["after"])


# ---------------------------------------------------------------------------- one pass

def run(s):
    op = s["case"]["op"]
    if op == "write":
        if own:
            s["cache"].write(s["k"], s["v"], s["slots"])
        else:
            _plain_write(s)
        return {"keys": s["key_cache"], "values": s["value_cache"]}
    if op == "decode":
        if own:
            out = s["cache"].decode(s["q"], s["table"], s["lens"], s["longest"], ledger=s["ledger"])
        else:
            out = _plain_decode(s)
        return {"out": out, "mass": s["mass"]} if s["case"]["ledger"] else {"out": out}
    if op == "observe":
        if own:
            s["cache"].observe(s["q"], s["table"], s["lens"], s["longest"], s["ledger"])
        else:
            _plain_observe(s)
        return {"mass": s["mass"]}
    if own:
        lens = s["cache"].evict(s["table"], s["lens"], s["longest"], s["ledger"], s["case"]["budget"], s["case"]["recent"],
                                out=s["ledger_after"])
    else:
        lens = _plain_evict(s)
    mass, positions, held, seen = s["after"]
    return {"lens": lens, "mass": mass, "positions": positions, "held": held, "seen": seen, "keys": s["key_cache"],
            "values": s["value_cache"]}


def _plain_write(s):
    s["key_cache"].flatten(0, 1)[s["slots"]] = s["k"]
    s["value_cache"].flatten(0, 1)[s["slots"]] = s["v"]


def _rows(s):
    """(batch, longest) index of every slot in the planes' rows."""
    page = s["case"]["page"]
    t = torch.arange(s["longest"], device="cuda")
    return s["table"][:, t // page].long() * page + t % page


def _weights(s, query):
    """Softmax weights (batch, kv head, queries x heads, slot) of query (batch, window, q_heads, d) over the cached keys."""
    c = s["case"]
    h, d, w = c["kv_heads"], c["head_dim"], query.shape[1]
    g = c["q_heads"] // h
    keys = s["key_cache"].flatten(0, 1)[_rows(s)].float().permute(0, 2, 3, 1)                  # (b, h, d, t)
    q = query.float().view(-1, w, h, g, d).permute(0, 2, 1, 3, 4).reshape(-1, h, w * g, d)
    scores = torch.matmul(q, keys) / math.sqrt(d)
    t = torch.arange(s["longest"], device="cuda")
    last = s["lens"][:, None] - w + torch.arange(w, device="cuda")                              # (b, w) last slot a query sees
    seen = (t <= last[..., None]).repeat_interleave(g, dim=1)[:, None]                         # (b, 1, w g, t)
    top = torch.where(seen, scores, torch.full_like(scores, -math.inf)).amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top)) * seen
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _plain_decode(s):
    c = s["case"]
    p = _weights(s, s["q"][:, None])
    values = s["value_cache"].flatten(0, 1)[_rows(s)].float().permute(0, 2, 1, 3)              # (b, h, t, d)
    out = torch.matmul(p, values).reshape(c["batch"], c["q_heads"], c["head_dim"]).to(s["q"].dtype)
    if c["ledger"]:
        s["mass"] += p.sum(2)
    return out


def _plain_observe(s):
    s["mass"] += _weights(s, s["q"]).sum(2)


def _plain_evict(s):
    c, n = s["case"], s["lens"][:, None, None]
    budget, held, seen = c["budget"], s["held"][:, None, None], s["seen"][:, None, None]
    slot = torch.arange(s["longest"], device="cuda")
    positions = torch.where(slot < held, s["positions"], seen + slot.int() - held)
    total = seen + n - held
    cached = slot < n
    rank = torch.where(cached, s["mass"], torch.full_like(s["mass"], -1.0))
    order = torch.argsort(rank, dim=-1, descending=True, stable=True)
    late = (cached & (positions >= total - c["recent"])).int()
    order = order.gather(-1, torch.argsort(late.gather(-1, order), dim=-1, descending=True, stable=True))
    kept = torch.zeros_like(cached.expand_as(late)).scatter_(-1, order[..., :budget], True) & cached
    after = torch.clamp(n, max=budget)
    hole, mover = ~kept & (slot < after), kept & (slot >= after)
    movers = torch.argsort(mover.int(), dim=-1, descending=True, stable=True)
    source = torch.where(hole, movers.gather(-1, (hole.long().cumsum(-1) - 1).clamp(min=0)), slot.expand_as(movers))
    out_mass, out_positions, out_held, out_seen = s["after"]
    inside = slot < after
    out_mass.copy_(torch.where(inside, s["mass"].gather(-1, source), torch.zeros_like(s["mass"])))
    out_positions.copy_(torch.where(inside, positions.gather(-1, source), torch.full_like(positions, -1)))
    out_held.copy_(after[:, 0, 0])
    out_seen.copy_(total[:, 0, 0])
    row = _rows(s)
    seq, head, to = torch.nonzero(hole, as_tuple=True)
    at = source[seq, head, to]
    s["key_cache"].flatten(0, 1)[row[seq, to], head] = s["key_cache"].flatten(0, 1)[row[seq, at], head]
    s["value_cache"].flatten(0, 1)[row[seq, to], head] = s["value_cache"].flatten(0, 1)[row[seq, at], head]
    return after[:, 0, 0].contiguous()


# ---------------------------------------------------------------------------- the definition, in 64 bits

def exact(case, seed):
    """One sequence at a time, one kv head's group of queries at a time, in float64."""
    s, c = prepare(case, seed), case
    if c["op"] == "write":
        got = {}
        for name, plane, rows in (("keys", s["key_cache"], s["k"]), ("values", s["value_cache"], s["v"])):
            full = plane.double().reshape(-1, c["kv_heads"], c["head_dim"])
            full.index_copy_(0, s["slots"], rows.double())
            got[name] = full.view(plane.shape)
        return got
    lens, page, h, d = _lengths(c), c["page"], c["kv_heads"], c["head_dim"]
    if c["op"] == "evict":
        return _exact_evict(s, lens)
    g, w = c["q_heads"] // h, c.get("window", 1)
    query = s["q"].double().view(c["batch"], w, h, g, d)
    out = torch.zeros(c["batch"], h, g, d, dtype=torch.float64, device="cuda")
    mass = s["mass"].double() if "mass" in s else None
    for b, n in enumerate(lens):
        if n == 0:
            continue
        blocks = s["table"][b, : -(-n // page)].long()
        keys = s["key_cache"][blocks].reshape(-1, h, d)[:n].double()
        values = s["value_cache"][blocks].reshape(-1, h, d)[:n].double()
        for i in range(h):
            z = torch.einsum("wgd,td->wgt", query[b, :, i], keys[:, i]) * d ** -0.5
            for j in range(w):                     # query j of the window sees the first n - w + j + 1 tokens
                m = n - w + j + 1
                if m < 1:
                    continue
                p = torch.softmax(z[j, :, :m], dim=-1)
                if c["op"] == "decode":
                    out[b, i] = p @ values[:m, i]
                if mass is not None:
                    mass[b, i, :m] += p.sum(0)
    if c["op"] == "observe":
        return {"mass": mass}
    got = {"out": out.view(c["batch"], c["q_heads"], d)}
    if c["ledger"]:
        got["mass"] = mass
    return got


def _exact_evict(s, lens):
    """Straight from the rule: sort the tokens of a head, keep the first `budget`, fill the holes in order."""
    c, page = s["case"], s["case"]["page"]
    if sum(lens) * c["kv_heads"] > 1_500_000:      # tokens sorted one by one on the host
        return None
    keys, values = s["key_cache"].double().cpu(), s["value_cache"].double().cpu()
    mass, positions, table = s["mass"].double().cpu(), s["positions"].cpu(), s["table"].cpu().tolist()
    held, seen = s["held"].tolist(), s["seen"].tolist()
    new_mass, new_positions, new_lens, new_seen = torch.zeros_like(mass), torch.full_like(positions, -1), [], []
    for b, n in enumerate(lens):
        total, m = seen[b] + n - held[b], min(n, c["budget"])
        new_lens.append(m)
        new_seen.append(total)
        row = [table[b][t // page] * page + t % page for t in range(n)]
        for i in range(c["kv_heads"]):
            weight, pos = mass[b, i].tolist(), positions[b, i].tolist()
            pos = [pos[t] if t < held[b] else seen[b] + t - held[b] for t in range(n)]
            first = sorted(range(n), key=lambda t: (pos[t] < total - c["recent"], -weight[t], t))[:m]
            kept = set(first)
            source, movers = list(range(m)), iter(sorted(t for t in kept if t >= m))
            for t in range(m):
                if t not in kept:
                    source[t] = next(movers)
            if m == 0:
                continue
            new_mass[b, i, :m] = mass[b, i, source]
            new_positions[b, i, :m] = torch.tensor([pos[t] for t in source], dtype=torch.int32)
            moved = [t for t in range(m) if source[t] != t]
            to, at = [row[t] for t in moved], [row[source[t]] for t in moved]
            for plane in (keys, values):
                flat = plane.view(-1, c["kv_heads"], c["head_dim"])
                flat[to, i] = flat[at, i]
    ints = lambda v: torch.tensor(v, dtype=torch.int32)
    return {"lens": ints(new_lens), "mass": new_mass, "positions": new_positions, "held": ints(new_lens), "seen": ints(new_seen),
            "keys": keys, "values": values}


# ---------------------------------------------------------------------------- work

def work(case):
    c, lens = case, _lengths(case)
    n, h, d, b = sum(lens), c["kv_heads"], c["head_dim"], c["batch"]
    if c["op"] == "write":       # both rows of a token read and written, its slot
        return {"bytes": n * (h * 8 * d + 8), "flops": 0}
    pages = sum(-(-x // c["page"]) for x in lens) * 4 + 4 * b
    if c["op"] == "decode":      # keys and values once, query in, output out; the ledger's weights read and written
        return {"bytes": n * h * 4 * d + pages + b * c["q_heads"] * 4 * d + (8 * n * h if c["ledger"] else 0),
                "flops": n * c["q_heads"] * 4 * d}
    if c["op"] == "observe":     # keys once, one product with the window's queries
        w = c["window"]
        return {"bytes": n * h * 2 * d + pages + b * w * c["q_heads"] * 2 * d + 8 * n * h, "flops": n * w * c["q_heads"] * 2 * d}
    moved, recent = 0.0, c["recent"]
    for x in lens:
        m = min(x, c["budget"])
        behind, free, old = x - m, m - recent, x - recent
        late = min(recent, behind)      # the latest tokens lie behind the budget
        moved += late + (behind - late) * (free / old if old > 0 else 0.0) if behind else 0.0
    known = sum(min(x, c["held"]) for x in lens)
    return {"bytes": h * (4 * n + 4 * known + 8 * b * max(max(lens), 1) + moved * 8 * d) + pages, "flops": n * h}
