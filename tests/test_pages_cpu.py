"""The exact paged cache without a GPU: what the C ABI and the classes refuse before anything is launched."""

import ctypes as C

import pytest
import torch

from turboquant_b200 import AttentionLedger, ExactCacheSpec, PagedKVCache, _lib
from turboquant_b200 import exact_cache as X

NULL, SHAPE, ALIGN, UNSUPPORTED, WORKSPACE, RANGE = -1, -2, -3, -4, -6, -7


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


@pytest.fixture
def call():
    """Addresses that are only looked at: nothing gets as far as a launch."""
    page = (C.c_uint8 * 4096)()
    base = (C.addressof(page) + 255) // 256 * 256
    pages = _lib.tq_pages(base, base, _lib.TQ_BF16, 16, 8, 2, 128, 16 * 2 * 128, 2 * 128, 128)
    batch = _lib.tq_pages_batch(base, 4, 4, base, 3, 64)
    ledger = _lib.tq_pages_ledger(base, base, base, base, 64)
    return type("Call", (), dict(page=page, base=base, pages=pages, batch=batch, ledger=ledger))


def decode(lib, c, q_heads=8, query=None, out=None, mass=None, stride=64, bytes=0, scratch=None):
    base = c.base
    pick = lambda x: base if x is None else x  # noqa: E731
    return lib.tq_pages_decode(C.byref(c.pages), C.byref(c.batch), pick(query), q_heads, 1.0, pick(out), mass, stride, pick(scratch), bytes,
                               base, base, None)


@pytest.mark.parametrize("field,value,code", [
    ("key", None, NULL), ("value", None, NULL), ("dtype", _lib.TQ_F32, UNSUPPORTED), ("block_size", 0, SHAPE), ("num_blocks", 0, SHAPE),
    ("num_blocks", 1 << 31, SHAPE), ("num_kv_heads", 0, SHAPE), ("head_dim", 96, UNSUPPORTED), ("stride_block", 4, ALIGN), ("stride_token", 12, ALIGN),
    ("stride_head", 1, ALIGN), ("stride_head", -8, SHAPE)])
def test_pages_are_checked(lib, call, field, value, code):
    assert decode(lib, call) == WORKSPACE          # all is well but the scratch memory
    setattr(call.pages, field, value)
    size = C.c_size_t(0)
    assert decode(lib, call) == code
    assert lib.tq_pages_write(C.byref(call.pages), call.base, call.base, 4, 256, 128, 256, 128, call.base, call.base, None) == code
    assert lib.tq_pages_observe_scratch_bytes(C.byref(call.pages), C.byref(call.batch), 4, 8, C.byref(size)) == code
    assert lib.tq_pages_evict_scratch_bytes(C.byref(call.pages), C.byref(call.batch), 4, C.byref(size)) == code


@pytest.mark.parametrize("field,value,code", [
    ("block_tables", None, NULL), ("seq_lens", None, NULL), ("batch", 0, SHAPE), ("max_seq_len", 0, SHAPE), ("max_seq_len", 65, RANGE),
    ("table_width", 3, RANGE), ("table_stride", 3, SHAPE), ("table_width", 0, SHAPE)])
def test_batches_are_checked(lib, call, field, value, code):
    setattr(call.batch, field, value)
    size = C.c_size_t(0)
    assert decode(lib, call) == code
    assert lib.tq_pages_observe_scratch_bytes(C.byref(call.pages), C.byref(call.batch), 4, 8, C.byref(size)) == code
    assert lib.tq_pages_evict_scratch_bytes(C.byref(call.pages), C.byref(call.batch), 4, C.byref(size)) == code


def test_calls_are_checked(lib, call):
    c, base = call, call.base
    assert decode(lib, c, q_heads=7) == SHAPE and decode(lib, c, q_heads=0) == SHAPE
    assert decode(lib, c, query=base + 2) == ALIGN and decode(lib, c, out=base + 8) == ALIGN and decode(lib, c, scratch=base + 4) == ALIGN
    assert decode(lib, c, mass=base, stride=63) == RANGE and decode(lib, c, mass=base) == WORKSPACE
    assert lib.tq_pages_decode(C.byref(c.pages), C.byref(c.batch), base, 8, 1.0, base, None, 0, base, 1 << 30, None, base, None) == NULL
    assert lib.tq_pages_decode(C.byref(c.pages), C.byref(c.batch), base, 8, 1.0, base, None, 0, base, 1 << 30, base, None, None) == NULL
    write = lambda n=4, k=base, strides=(256, 128, 256, 128): lib.tq_pages_write(  # noqa: E731
        C.byref(c.pages), k, base, n, *strides, base, base, None)
    assert write(n=-1) == SHAPE and write(n=0) == 0 and write(k=base + 2) == ALIGN and write(k=None) == NULL
    assert write(strides=(256, 128, 260, 128)) == ALIGN
    size = C.c_size_t(0)
    observe = lambda window=4, heads=8, q=base, stride=64, n=0: lib.tq_pages_observe(  # noqa: E731
        C.byref(c.pages), C.byref(c.batch), q, window, heads, 1.0, base, stride, base, n, base, None)
    assert observe() == WORKSPACE and observe(window=0) == SHAPE and observe(heads=9) == SHAPE and observe(q=base + 2) == ALIGN
    assert observe(stride=60) == RANGE and observe(q=None) == NULL
    assert lib.tq_pages_observe_scratch_bytes(C.byref(c.pages), C.byref(c.batch), 4, 8, None) == NULL
    evict = lambda budget=8, recent=2, led=c.ledger, n=0: lib.tq_pages_evict(  # noqa: E731
        C.byref(c.pages), C.byref(c.batch), C.byref(led), C.byref(c.ledger), budget, recent, base, base, n, base, None)
    assert evict() == WORKSPACE and evict(budget=-1) == SHAPE and evict(recent=9) == SHAPE and evict(recent=-1) == SHAPE
    short = _lib.tq_pages_ledger(base, base, base, base, 63)
    missing = _lib.tq_pages_ledger(base, None, base, base, 64)
    assert evict(led=short) == RANGE and evict(led=missing) == NULL
    assert lib.tq_pages_evict_scratch_bytes(C.byref(c.pages), C.byref(c.batch), 8, C.byref(size)) == 0 and size.value == 6 * 4 + 6 * 8 * 16
    assert lib.tq_pages_evict_scratch_bytes(C.byref(c.pages), C.byref(c.batch), 60, C.byref(size)) == 0 and size.value == 6 * 4 + 6 * 4 * 16
    assert lib.tq_pages_evict_scratch_bytes(C.byref(c.pages), C.byref(c.batch), 100, C.byref(size)) == 0 and size.value == 6 * 4


def test_the_list_of_units_stays_in_32_bits(lib, call):
    call.batch.table_width = call.batch.table_stride = 1 << 26
    call.batch.max_seq_len, call.batch.batch = 1 << 30, 16
    assert decode(lib, call) == SHAPE
    call.batch.batch = 15
    assert decode(lib, call) == WORKSPACE


def test_spec():
    spec = ExactCacheSpec(128, 8)
    assert spec.bytes_per_token == 512 and spec.page_size_bytes == 16 * 8 * 512
    assert spec.num_blocks_for(10 * spec.page_size_bytes + 5) == 10 and spec.max_memory_usage_bytes(17) == 2 * spec.page_size_bytes
    for bad in (dict(head_dim=96), dict(head_dim=128, block_size=0), dict(head_dim=128, num_kv_heads=0)):
        with pytest.raises(ValueError):
            ExactCacheSpec(**{"num_kv_heads": 2, **bad})
    with pytest.raises(TypeError):
        ExactCacheSpec(128, 2, dtype=torch.float32)


def test_the_cache_needs_planes_of_one_layout_on_the_gpu():
    with pytest.raises(RuntimeError):
        PagedKVCache(ExactCacheSpec(128, 2), torch.zeros(4, 16, 2, 128, dtype=torch.bfloat16), torch.zeros(4, 16, 2, 128, dtype=torch.bfloat16))


def test_ledger():
    led = AttentionLedger(3, 2, 10, "cpu")
    led.mass += 1
    led.held += 4
    led.seen += 5
    led.positions += 9
    led.reset([1])
    assert led.mass[1].sum() == 0 and led.mass[0].sum() == 20 and led.held.tolist() == [4, 0, 4] and led.seen.tolist() == [5, 0, 5]
    assert (led.positions[1] == -1).all() and (led.positions[2] == 8).all()
    led.reset()
    assert led.mass.sum() == 0 and (led.positions == -1).all() and not led.held.any()
    assert AttentionLedger.over(*led._tensors).mass is led.mass and led.batch == 3 and led.max_tokens == 10
    for bad in ((0, 2, 10), (3, 0, 10), (3, 2, 0)):
        with pytest.raises(ValueError):
            AttentionLedger(*bad, "cpu")
    mass, positions, held, seen = led._tensors
    for wrong in ((mass.double(), positions, held, seen), (mass, positions.long(), held, seen), (mass, positions[:, :, :9], held, seen),
                  (mass, positions, held[:2], seen), (mass, positions, held, seen.long()), (mass[:, :, ::2], positions[:, :, ::2], held, seen),
                  (mass, positions.to("meta"), held, seen)):
        with pytest.raises(ValueError):
            AttentionLedger.over(*wrong)


class Host:
    """Stands in for the native calls: takes nothing, so that the Python checks run."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *args: self.calls.append(name)


@pytest.fixture
def cache(monkeypatch):
    """A cache on the CPU whose native calls refuse everything."""
    host = Host()
    monkeypatch.setattr(X.E, "host", lambda: host)
    monkeypatch.setattr(X.E, "require_cuda", lambda t, name: None)
    c = PagedKVCache.allocate(ExactCacheSpec(128, 2), 8, "cpu")
    c.host = host
    return c


def test_planes_are_checked(cache):
    bf, spec = torch.bfloat16, cache.spec
    good = torch.zeros(8, 16, 2, 128, dtype=bf)
    PagedKVCache(spec, good, good.clone())
    for bad in (good[:, :8], good[..., :64], good.flatten(0, 1), good[:7], torch.zeros(8, 16, 2, 256, dtype=bf)[..., ::2],
                torch.zeros(8, 16, 2, 132, dtype=bf)[..., :128], torch.zeros(8 * 16 * 2 * 128 + 1, dtype=bf)[1:].view(8, 16, 2, 128)):
        with pytest.raises(ValueError):
            PagedKVCache(spec, good, bad)
    with pytest.raises(TypeError):
        PagedKVCache(spec, good.half(), good.half())


def test_refusals_of_the_class(cache):
    bf = torch.bfloat16
    table, lens = torch.zeros(3, 4, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    q, k = torch.zeros(3, 8, 128, dtype=bf), torch.zeros(3, 2, 128, dtype=bf)
    led = AttentionLedger(3, 2, 64, "cpu")
    slots = torch.arange(3)
    for args in ((k.half(), k.half(), slots), (k, k.half(), slots)):
        with pytest.raises(TypeError):
            cache.write(*args)
    for args in ((k[:, :1], k[:, :1], slots), (k, k[:2], slots), (k, k, slots[:2]), (k, k, slots.int()), (k[0], k[0], slots), (k, k, slots[None])):
        with pytest.raises(ValueError):
            cache.write(*args)
    with pytest.raises(TypeError):
        cache.decode(q.half(), table, lens, 64)
    with pytest.raises(TypeError):
        cache.decode(q, table, lens, 64, ledger=led.mass)
    for args in ((q[:, :3], table, lens, 64), (q[..., :64], table, lens, 64), (q[0], table, lens, 64), (q, table.long(), lens, 64), (q, table[:2], lens, 64),
                 (q, table[0], lens, 64), (q, table, lens[:2], 64), (q, table, lens.long(), 64), (q, table, lens, 65), (q, table, lens, -1), (q, table, lens, 2 ** 30)):
        with pytest.raises(ValueError):
            cache.decode(*args)
    for out in (torch.zeros(3, 8, 64, dtype=bf), torch.zeros(3, 8, 128), torch.zeros(3, 8, 256, dtype=bf)[..., ::2]):
        with pytest.raises(ValueError):
            cache.decode(q, table, lens, 64, out=out)
    small = [AttentionLedger(2, 2, 64, "cpu"), AttentionLedger(3, 1, 64, "cpu"), AttentionLedger(3, 2, 63, "cpu")]
    window = q[:, None]
    for bad in small:
        with pytest.raises(ValueError):
            cache.decode(q, table, lens, 64, ledger=bad)
        with pytest.raises(ValueError):
            cache.observe(window, table, lens, 64, bad)
        with pytest.raises(ValueError):
            cache.evict(table, lens, 64, bad, 8)
        with pytest.raises(ValueError):
            cache.evict(table, lens, 64, led, 8, out=bad)
    for args in ((q, table, lens, 64, led), (window[:, :, :3], table, lens, 64, led), (window, table, lens, 65, led)):
        with pytest.raises(ValueError):
            cache.observe(*args)
    with pytest.raises(TypeError):
        cache.observe(window.half(), table, lens, 64, led)
    for budget, recent in ((8, 9), (8, -1), (-1, 0), (2 ** 31, 0)):
        with pytest.raises(ValueError):
            cache.evict(table, lens, 64, led, budget, recent)
    assert cache.status() == 0


@pytest.mark.parametrize("batch,tokens,code", [(16, (1 << 30) - 32, SHAPE), (16, (1 << 30) - (1 << 19), 0), (15, 1 << 30, 0)])
def test_a_list_rounded_up_to_shares_stays_in_32_bits(lib, call, batch, tokens, code):
    """2^31 - 64 units of 16 tokens and head fit, but not once every CTA's share is rounded up."""
    call.batch.max_seq_len, call.batch.batch = tokens, batch
    call.batch.table_width = call.batch.table_stride = 1 << 26
    size = C.c_size_t(0)
    assert lib.tq_pages_decode_scratch_bytes(C.byref(call.pages), C.byref(call.batch), 8, 0, C.byref(size)) == code
