"""The exact paged cache without a GPU, beyond test_pages_cpu.py: what is refused, and what small tensors pass for."""

import ctypes as C

from tests.test_pages_cpu import NULL, cache, call, lib  # noqa: F401  fixtures


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
