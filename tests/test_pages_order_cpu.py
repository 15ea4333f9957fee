"""What may begin before an eviction has written its lengths (csrc/tq_stream_order.h), stepped through on the CPU.

The launches and the model are those of test_stream_order_cpu.py with the exact paged cache's among them, and with lengths beside
the pool and rows as what a launch writes and a later one may read in front of its wait: the decode family reads lengths at its
entry, whether or not it then waits for its first record.
"""

import ctypes as C
import itertools
import os
import re
import subprocess

import pytest

from tests.test_stream_order_cpu import CSRC, GLUE, LAUNCHES, UNKNOWN, DECODE, STORE_EARLY, NEUTRAL, PREP_BEHIND_STORE, WAITED, STORE_PLAIN, _launch

LENGTHS = 7
PAGES = ("pages write", "pages decode", "pages observe", "pages evict")
MORE = 'extern "C" int prep_may_overlap(int k) { return tq_prep_may_overlap(k); }\n'


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("pages_order")
    (d / "glue.cpp").write_text(GLUE + MORE)
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O1", "-shared", "-fPIC", "-I", CSRC, "-o", str(d / "glue.so"), str(d / "glue.cpp")],
                   check=True)
    lib = C.CDLL(str(d / "glue.so"))
    lib.notes_new.restype = C.c_void_p
    lib.notes_free.argtypes = [C.c_void_p]
    lib.note.argtypes = [C.c_void_p, C.c_ulong, C.c_int]
    lib.last.argtypes = [C.c_void_p, C.c_ulong]
    return lib


def _grids(r, name, ahead, evict_note, plain_prep):
    """The grids of a call: (programmatic, lets others begin, writes, reads early), and its note."""
    if name == "pages write":
        return [(True, "waited", {"rows"}, set())], WAITED
    if name == "pages decode":
        return [(True, "waited", set(), set())] * 2, WAITED
    if name == "pages observe":        # the second launch reads lengths, tables and keys before its wait
        return [(True, "waited", set(), set()), (True, "waited", set(), {"rows", "lengths"})], WAITED
    if name == "pages evict":
        return [(True, "waited", set(), set()), (True, "waited", {"rows", "lengths"}, set())], evict_note
    prog, begin, writes, early, kind = _launch(r, name, ahead)
    early = {early} if early else set()
    if name == "prepare":
        prog = bool(r.prep_may_overlap(ahead)) if plain_prep else True
    if name == "decode" and prog:
        early = early | {"lengths"}
    return [(prog, begin, {writes} if writes else set(), early)], kind


def _run(r, steps, evict_note=LENGTHS, plain_prep=True):
    notes, loose = r.notes_new(), set()
    try:
        for name in steps:
            if name == "others":              # eight other streams launch something
                for st in range(100, 108):
                    r.note(notes, st, DECODE)
                continue
            grids, kind = _grids(r, name, r.last(notes, 7), evict_note, plain_prep)
            for prog, begin, writes, early in grids:
                if prog and early & loose:
                    return "%s reads %s that may not be written" % (name, sorted(early & loose))
                loose = (loose if prog and begin == "entry" else set()) | writes
            if kind is not None:
                r.note(notes, 7, kind)
    finally:
        r.notes_free(notes)
    return None


def test_nobody_reads_early_what_may_not_be_written(rules):
    wrong = [(steps, bad) for n in range(1, 5) for steps in itertools.product(LAUNCHES + PAGES + ("others",), repeat=n)
             for bad in (_run(rules, steps),) if bad]
    assert not wrong, wrong[:4]


@pytest.mark.parametrize("steps", [("pages evict", "decode"), ("pages evict", "prepare", "decode"), ("pages evict", "others", "prepare", "decode"),
                                   ("pages evict", "prepare", "prepare", "decode")])
def test_the_model_sees_lengths_that_are_read_too_early(rules, steps):
    """An eviction noted like a launch that writes rows only, or a preparation that begins under it."""
    assert _run(rules, steps) is None
    assert "lengths" in _run(rules, steps, evict_note=WAITED, plain_prep=False)
    if "prepare" in steps:
        assert "lengths" in _run(rules, steps, plain_prep=False)


def test_what_an_eviction_costs_the_launches_behind(rules):
    """Rows behind it are late, the pool is late, and after any launch that has waited the usual overlaps are back."""
    assert not rules.rows_at_rest(LENGTHS) and not rules.may_overlap(LENGTHS) and not rules.prep_may_overlap(LENGTHS)
    for ahead in (DECODE, STORE_EARLY, NEUTRAL, PREP_BEHIND_STORE, WAITED, STORE_PLAIN):
        assert rules.prep_may_overlap(ahead)
    assert not rules.prep_may_overlap(UNKNOWN)      # the eviction's note may be the one that is gone


def test_the_places_that_launch_follow_the_rules():
    """Read from the source: what lets its dependents begin at entry is launched by the rule, and an eviction leaves its note."""
    preps = 0
    for name in sorted(os.listdir(CSRC)):
        if name.endswith(".cu"):
            text = open(os.path.join(CSRC, name)).read()
            for m in re.finditer(r"tq_note_prep_launch\(st\);", text):
                before = text[:m.start()]
                assert re.search(r"numAttrs = tq_prep_may_overlap\(tq_last_launch\(st\)\) \? 1 : 0;[^\n]*\n\s*$", before), name
                preps += 1
    assert preps >= 3
    text = open(os.path.join(CSRC, "tq_pages_cache.cu")).read()
    evict = text[text.index('extern "C" int tq_pages_evict('):]
    assert re.findall(r"tq_note_launch\(st, (\w+)\)", evict) == ["TQ_LAUNCH_LENGTHS"]
