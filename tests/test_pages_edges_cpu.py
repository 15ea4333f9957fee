"""The exact paged cache without a GPU, beyond test_pages_cpu.py: what is refused, and what small tensors pass for."""

import ctypes as C

import pytest
import torch

from tests.test_pages_cpu import NULL, SHAPE, WORKSPACE, cache, call, lib  # noqa: F401  fixtures
from turboquant_b200 import AttentionLedger, ExactCacheSpec, PagedKVCache, _lib


def test_what_a_ledger_holds_comes_in_a_pair(lib, call):  # noqa: F811
    size = C.c_size_t(0)
    ask = lambda: lib.tq_pages_observe_scratch_bytes(C.byref(call.pages), C.byref(call.batch), 4, 8, C.byref(size))  # noqa: E731
    assert ask() == 0
    call.batch.held = call.base
    assert ask() == NULL
    call.batch.seen = call.base
    assert ask() == 0
    call.batch.held = None
    assert ask() == NULL


def test_scratch_of_a_ledger_is_bounded(lib, call):  # noqa: F811
    """What the scores take beside the rest: 4 bytes a query head and token of the bound, 512 MB or one sequence at most."""
    def scores(batch, tokens, heads=64):
        call.batch.batch, call.batch.max_seq_len, call.batch.table_width, call.batch.table_stride = batch, tokens, 1 << 26, 1 << 26
        got = []
        for mass in (0, 1):
            size = C.c_size_t(0)
            assert lib.tq_pages_decode_scratch_bytes(C.byref(call.pages), C.byref(call.batch), heads, mass, C.byref(size)) == 0
            got.append(size.value)
        return got[1] - got[0]
    sums = lambda rows: (rows * 64 * 4 + 255) // 256 * 256  # noqa: E731
    assert scores(4, 1000) == 4 * 64 * 1008 * 4 + sums(4)
    assert scores(16, 131072) == 2 ** 29 + sums(16)
    for batch in (17, 64, 256):
        assert scores(batch, 131072) == 2 ** 29 + sums(16)
    assert scores(3, 1 << 22) == 2 ** 30 + sums(1) and scores(1000, 100000) == 20 * 64 * 100000 * 4 + sums(20)


def test_planes_with_a_dimension_of_one(cache):  # noqa: F811
    """The stride of a dimension of one, odd or different between the planes, is nobody's business; that of a larger one is."""
    bf = torch.bfloat16
    odd = lambda shape, strides: torch.zeros(8192, dtype=bf).as_strided(shape, strides)  # noqa: E731
    for shape, a, b in (((1, 2, 2, 64), (777, 128, 64, 1), (1030, 128, 64, 1)), ((2, 1, 2, 64), (1024, 3, 64, 1), (1024, 64, 64, 1)),
                        ((2, 2, 1, 64), (512, 64, 100, 1), (512, 64, 64, 1)), ((1, 1, 1, 64), (1, 3, 5, 1), (64, 64, 64, 1))):
        spec = ExactCacheSpec(64, shape[2], block_size=shape[1])
        made = PagedKVCache(spec, odd(shape, a), odd(shape, b)).c
        for n, got, want in zip(shape, (made.stride_block, made.stride_token, made.stride_head), a):
            assert got == (want if n > 1 else 0)
    spec = ExactCacheSpec(64, 2, block_size=2)
    with pytest.raises(ValueError):
        PagedKVCache(spec, odd((2, 2, 2, 64), (516, 128, 64, 1)), odd((2, 2, 2, 64), (516, 128, 64, 1)))
    with pytest.raises(ValueError):
        PagedKVCache(spec, odd((2, 2, 2, 64), (512, 128, 64, 1)), odd((2, 2, 2, 64), (256, 128, 64, 1)))
    with pytest.raises(ValueError):
        PagedKVCache(spec, odd((1, 2, 2, 64), (512, 128, 64, 1)), odd((1, 2, 2, 64), (512, 256, 128, 2)))


def test_a_ledger_is_what_its_attributes_are(cache):  # noqa: F811
    """A tensor put in the place of another counts for every call, not for some."""
    taken = []
    cache.host.pages_decode = cache.host.pages_observe = cache.host.pages_evict = lambda *args: taken.append(args)
    table, lens, q = torch.zeros(3, 4, dtype=torch.int32), torch.ones(3, dtype=torch.int32), torch.zeros(3, 8, 128, dtype=torch.bfloat16)
    led = AttentionLedger(3, 2, 64, "cpu")
    led.mass, led.held = led.mass.clone(), led.held.clone()
    for call_it in (lambda: cache.decode(q, table, lens, 64, ledger=led), lambda: cache.observe(q[:, None], table, lens, 64, led),
                    lambda: cache.evict(table, lens, 64, led, 8)):
        with pytest.raises(RuntimeError):          # nothing native answers
            call_it()
        assert any(a is led.mass for a in taken[-1])
    assert sum(a is led.held for a in taken[-1]) == 2          # evict: the ledger that is read and the one that is written


@pytest.mark.parametrize("array", ["mass", "positions", "held", "seen"])
def test_a_ledger_half_over_another_is_refused(lib, call, array):  # noqa: F811
    base = call.base
    evict = lambda out: lib.tq_pages_evict(C.byref(call.pages), C.byref(call.batch), C.byref(call.ledger), C.byref(out), 8, 2, base, base, 0,  # noqa: E731
                                           base, None)
    words = 3 if array in ("held", "seen") else 3 * 2 * 64
    fields = dict(mass=base, positions=base, held=base, seen=base, max_tokens=64)
    for shift, code in ((0, WORKSPACE), (4, SHAPE), (-4, SHAPE), ((words - 1) * 4, SHAPE), (words * 4, WORKSPACE), (-words * 4, WORKSPACE)):
        assert evict(_lib.tq_pages_ledger(**{**fields, array: base + shift})) == code
    wider = {**fields, "max_tokens": 65}
    assert evict(_lib.tq_pages_ledger(**wider)) == SHAPE                # the same memory with rows of another length
    apart = {**wider, "mass": base + 8 * 1024, "positions": base + 8 * 1024}
    assert evict(_lib.tq_pages_ledger(**apart)) == WORKSPACE
