"""The ring of notes of csrc/attention_tc.cu's packed form, gone through on the CPU with the roles' order of test_attention_order: the warps that look through V clear the
place of the next item, note an item's numbers that are none when they find them, and the warps of the rows' way out read an item's note behind its sums and once more
behind their word that the next item may have them. Read must be what this item's warps wrote."""
from __future__ import annotations

import random

import pytest

from test_attention_order import Hazard, Memory, WARPS, _rows_form, _run

RING = 8
# (row tiles, key tiles) of a CTA's items: more than two times round, items without a second tile, long ones among short ones
RUNS = [[(1, 1)] * 18, [(2, 1)] * 18, [(2, 1), (1, 1)] * 9, [(1, 1), (1, 1), (2, 1)] * 6, [(2, 3)] + [(1, 1)] * 9 + [(1, 4)] + [(2, 1)] * 8]


def _noted(i):
    return i % 3 != 1


def _with_ring(items, ring=RING, clear=True):
    actors, counts = _rows_form(items)
    mem = Memory()
    for w in range(WARPS):
        mem["found", w, 0] = ("clear", 0)
        ops, at = [], 0
        for i, (_, n) in enumerate(items):
            if clear:
                ops.append(mem.put(("found", w, (i + 1) % ring), ("clear", i + 1)))
            for j in range(n):
                look = actors[f"hidden rows {w}"][at:at + 4]             # wait for V, two reads, the arrival
                at += 4
                note = [mem.put(("found", w, i % ring), ("note", i))] if _noted(i) and j == n - 1 else []
                ops += look[:-1] + note + look[-1:]
        assert at == len(actors[f"hidden rows {w}"])
        actors[f"hidden rows {w}"] = ops
    for w in range(WARPS):
        ops, at = [], 0
        for i, (tiles, _) in enumerate(items):
            read = [mem.get(("found", v, i % ring), ("note" if _noted(i) else "clear", i)) for v in range(WARPS)]
            for _ in range(tiles):
                out = actors[f"rows out {w}"][at:at + 4]                 # wait for the sums, two reads, "O is free"
                at += 4
                ops += out[:1] + read + out[1:] + read
        assert at == len(actors[f"rows out {w}"])
        actors[f"rows out {w}"] = ops
    return actors, counts


def _go_through(items, every=12, **kw):
    for held, ops in _with_ring(items, **kw)[0].items():
        if held in ("rows out 0", "hidden rows 1", "loads"):
            for stop in range(0, len(ops), every // 4 if held == "rows out 0" else every):
                _run(*_with_ring(items, **kw), held, stop)
    rng = random.Random(0)
    for _ in range(10):
        _run(*_with_ring(items, **kw), rng=rng)


@pytest.mark.parametrize("items", RUNS)
def test_a_note_is_its_items(items):
    _go_through(items)


def test_six_places_would_do():
    """At the start of item n a warp has seen V of n - 1, which is loaded behind the sums of n - 3; those begin when the rows' way out has begun its last reads of n - 4, so that it is
    through with n - 5 for certain. The place cleared there is that of n + 1: with six, n - 5 had it before. Eight leave room."""
    for items in RUNS[:3]:
        _go_through(items, ring=6)


@pytest.mark.parametrize("ring", [2, 5])
def test_too_short_a_ring_is_found_out(ring):
    with pytest.raises(Hazard, match="found"):
        _go_through(RUNS[0], every=4, ring=ring)


def test_a_place_never_cleared_is_found_out():
    with pytest.raises(Hazard, match="found"):
        _go_through(RUNS[0], clear=False)
