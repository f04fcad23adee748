"""The order of the roles of csrc/attention_tc.cu, gone through on the CPU: each role's waits, arrivals and accesses as the kernel issues them,
run against one another while one warp at a time is held back as long as anybody else can go on, and in random orders. Checked are what
waits by parity rest on (nobody is two completions of a barrier behind) and what is read (the item and key tile that it was meant to be).

An item has one or two tiles of 128 rows and some key tiles. A barrier completes when its count of arrivals is there; a wait is for the
n-th completion, as the kernel's parity stands for it. Products execute in the order in which they were issued, some time later."""
from __future__ import annotations

import random

import pytest

# (row tiles, key tiles) of the items that one CTA serves
RUNS = [[(2, 1)] * 4, [(2, 1), (1, 1), (2, 1), (1, 1), (2, 1)], [(1, 1)] * 4, [(2, 3), (1, 2), (2, 1)], [(1, 4), (2, 1), (1, 1), (2, 2)]]


class Hazard(Exception):
    pass


class Barriers:
    def __init__(self, counts):
        self.count, self.here, self.done, self.seen = dict(counts), dict.fromkeys(counts, 0), dict.fromkeys(counts, 0), {}

    def arrive(self, bar):
        self.here[bar] += 1
        if self.here[bar] == self.count[bar]:
            self.here[bar], self.done[bar] = 0, self.done[bar] + 1
            for (b, who), n in self.seen.items():
                if b == bar and self.done[bar] > n + 1:
                    raise Hazard(f"{bar} completed again before {who} saw the completion before")


def _run(actors, counts, held=None, stop=0, rng=None):
    """actors: name -> list of ("wait", bar, n-th completion), ("arrive", bar) or ("do", callable). n = 0 passes at once. Everybody who ever waits for
    a barrier has to see each of its completions that it waits for in turn. `held` stands at its stop-th step until nobody else can go on;
    with `rng` who goes next, and how far, is drawn."""
    bars = Barriers(counts)
    waits = {}
    for name, ops in actors.items():
        for op in ops:
            if op[0] == "wait" and op[2] > 0:
                waits.setdefault((op[1], name), []).append(op[2])
    for key, ns in waits.items():
        assert ns == list(range(1, len(ns) + 1)), key      # a role that waits for a barrier waits for every completion up to its last
    bars.seen = {key: 0 for key in waits}
    at = dict.fromkeys(actors, 0)

    def step(name):
        """False when it has to wait or is through."""
        if at[name] == len(actors[name]):
            return False
        op = actors[name][at[name]]
        if op[0] == "wait":
            if bars.done[op[1]] < op[2]:
                return False
            if op[2] > 0:
                bars.seen[op[1], name] = op[2]
                if op[2] == len(waits[op[1], name]):
                    del bars.seen[op[1], name]             # it waits for this barrier no more
        elif op[0] == "arrive":
            bars.arrive(op[1])
        else:
            op[1]()
        at[name] += 1
        return True

    if rng is not None:
        names = list(actors)
        for _ in range(300):
            rng.shuffle(names)
            for name in names:
                for _ in range(rng.choice((0, 0, 1, 3, 40))):
                    if not step(name):
                        break
    going = True
    while going:
        going = False
        for name in actors:
            while not (name == held and at[name] == stop) and step(name):
                going = True
        if not going and held is not None:
            held, going = None, True
    stuck = [name for name in actors if at[name] < len(actors[name])]
    if stuck:
        raise Hazard(f"nobody can go on: {stuck}")


class Memory(dict):
    def put(self, at, what):
        def f():
            self[at] = what
        return "do", f

    def get(self, at, what):
        def f():
            if self.get_(at) != what:
                raise Hazard(f"{at} holds {self.get_(at)} where {what} is read")
        return "do", f

    def get_(self, at):
        return dict.get(self, at)


WARPS = 2      # of each role that has several: enough for one of them to be behind


def _tensor_core(queue, issued):
    """The products and completions in the order of issue; what is not issued yet is waited for."""
    ops = []
    for i, op in enumerate(queue):
        ops += [("wait", f"issued{i}", 1), op]
        issued[f"issued{i}"] = 1
    return ops


def _cache_form(items, own_o_full=True):
    """Warps 0-7 softmax and rows out, 8 products, 12-15 operands."""
    mem, queue = Memory(), []
    counts = {**{("kv_full", s): WARPS for s in range(4)}, **{("kv_empty", s): 1 for s in range(4)}}
    for t in (0, 1):
        counts.update({("q_full", t): WARPS, ("q_empty", t): 1, ("s_full", t): 2, ("p_early", t): WARPS, ("p_full", t): WARPS, ("o_full", t): 2})
    o_bar = "o_full" if own_o_full else "s_full"
    actors = {f"softmax {t}.{w}": [] for t in (0, 1) for w in range(WARPS)}
    # ---- softmax
    for t in (0, 1):
        for w in range(WARPS):
            ops, seen, tile_no, mine = actors[f"softmax {t}.{w}"], {"s_full": 0, "o_full": 0}, 0, 0
            for i, (tiles, n) in enumerate(items):
                if t >= tiles:
                    tile_no += n
                    continue
                for j in range(n):
                    seen["s_full"] += 1
                    ops += [("wait", ("s_full", t), seen["s_full"]), mem.get(("info", tile_no % 4, w), tile_no), mem.get(("s", t), (i, j))]
                    if j == 0:
                        ops.append(mem.get(("power", mine % 2, t, w), i))
                    else:
                        ops.append(mem.get(("o", t), (i, j - 1)))
                    ops += [mem.put(("p early", t, w), (i, j)), ("arrive", ("p_early", t)), mem.put(("p", t, w), (i, j)), ("arrive", ("p_full", t))]
                    tile_no += 1
                seen[o_bar] += 1
                mine += 1
                ops += [("wait", (o_bar, t), seen[o_bar]), mem.get(("o", t), (i, n - 1))]
    # ---- products, and what the tensor cores do with them
    issue, seen = [], {}

    def wait(bar):
        seen[bar] = seen.get(bar, 0) + 1
        issue.append(("wait", bar, seen[bar]))

    def push(*ops):
        for op in ops:
            issue.append(("arrive", f"issued{len(queue)}"))
            queue.append(op)

    def issue_s(t, i, j, slot, tile):
        push(mem.get(("q", t), i), mem.get(("ring", slot), ("k", tile)), mem.put(("s", t), (i, j)))

    def ready(t):
        push(("arrive", ("s_full", t)))
        issue.append(("arrive", ("s_full", t)))
    kv_no = tile_no = 0
    for i, (tiles, n) in enumerate(items):
        wait(("kv_full", kv_no % 4))
        for t in range(tiles):
            wait(("q_full", t))
            issue_s(t, i, 0, kv_no % 4, tile_no)
            if n == 1:
                push(("arrive", ("q_empty", t)))
            ready(t)
        push(("arrive", ("kv_empty", kv_no % 4)))
        for j in range(n):
            vs, ks, more = (kv_no + 1) % 4, (kv_no + 2) % 4, j + 1 < n
            wait(("kv_full", vs))
            for t in range(tiles):
                wait(("p_early", t))
                push(mem.get(("ring", vs), ("v", tile_no)), *(mem.get(("p early", t, w), (i, j)) for w in range(WARPS)))
                wait(("p_full", t))
                if more and t == 0:
                    wait(("kv_full", ks))
                push(*(mem.get(("p", t, w), (i, j)) for w in range(WARPS)), mem.put(("o", t), (i, j)))
                if more:
                    issue_s(t, i, j + 1, ks, tile_no + 1)
                    if j + 2 == n:
                        push(("arrive", ("q_empty", t)))
                if more or not own_o_full:
                    ready(t)
                else:
                    push(("arrive", ("o_full", t)))
                    issue.append(("arrive", ("o_full", t)))
            push(("arrive", ("kv_empty", vs)))
            if more:
                push(("arrive", ("kv_empty", ks)))
            kv_no, tile_no = kv_no + 2, tile_no + 1
    actors["products"] = issue
    actors["tensor cores"] = _tensor_core(queue, counts)
    # ---- operands
    for w in range(WARPS):
        ops, kv_no, tile_no, q_no = [], 0, 0, [0, 0]
        for i, (tiles, n) in enumerate(items):
            for t in range(tiles):
                ops.append(("wait", ("q_empty", t), q_no[t]))
                q_no[t] += 1
                ops += [mem.put(("power", (q_no[t] - 1) % 2, t, w), i), mem.put(("q", t), i), ("arrive", ("q_full", t))]
            for j in range(n):
                for kind in "kv":
                    ops.append(("wait", ("kv_empty", kv_no % 4), kv_no // 4))
                    if kind == "k":
                        ops.append(mem.put(("info", tile_no % 4, w), tile_no))
                    ops += [mem.put(("ring", kv_no % 4), (kind, tile_no)), ("arrive", ("kv_full", kv_no % 4))]
                    kv_no += 1
                tile_no += 1
        actors[f"operands {w}"] = ops
    return actors, counts


def _rows_form(items, slot_by_tile=True, with_p=True):
    """Warps 0-7 softmax, 8 products, 9 loads, 10 and 11 hidden rows of V, 12-15 rows out."""
    mem, queue = Memory(), []
    counts = {**{("kv_full", s): 1 for s in range(4)}, **{("kv_empty", s): 1 for s in range(4)}}
    for t in (0, 1):
        counts.update({("q_full", t): 1, ("q_empty", t): 1, ("s_full", t): 2, ("p_early", t): WARPS, ("p_full", t): WARPS, ("o_full", t): 2 if with_p else WARPS + 1,
                       ("o_empty", t): WARPS, ("v_ready", t): WARPS})
    actors = {}
    # ---- softmax, and l of its rows
    for t in (0, 1):
        for w in range(WARPS):
            ops, s_seen, tile_no, mine = [], 0, 0, 0
            for i, (tiles, n) in enumerate(items):
                if t >= tiles:
                    tile_no += n
                    mine += not slot_by_tile
                    continue
                for j in range(n):
                    s_seen += 1
                    ops += [("wait", ("s_full", t), s_seen), mem.get(("info", tile_no % 4), tile_no), mem.get(("s", t), (i, j))]
                    if j > 0:
                        ops.append(mem.get(("o", t), (i, j - 1)))
                    ops += [mem.put(("p early", t, w), (i, j)), ("arrive", ("p_early", t)), mem.put(("p", t, w), (i, j))]
                    if with_p and j + 1 == n:
                        ops.append(mem.put(("l", mine % 2, t, w), i))
                    ops.append(("arrive", ("p_full", t)))
                    tile_no += 1
                if not with_p:
                    ops += [mem.put(("l", mine % 2, t, w), i), ("arrive", ("o_full", t))]
                mine += 1
            actors[f"softmax {t}.{w}"] = ops
    # ---- products
    issue, seen = [], {}

    def wait(bar):
        seen[bar] = seen.get(bar, 0) + 1
        issue.append(("wait", bar, seen[bar]))

    def push(*ops):
        for op in ops:
            issue.append(("arrive", f"issued{len(queue)}"))
            queue.append(op)

    def issue_s(t, i, j, slot, tile):
        push(mem.get(("q", t), i), mem.get(("ring", slot), ("k", tile)), mem.put(("s", t), (i, j)))

    def ready(t):
        push(("arrive", ("s_full", t)))
        issue.append(("arrive", ("s_full", t)))
    kv_no, tile_no, o_no = 0, 0, [0, 0]
    for i, (tiles, n) in enumerate(items):
        wait(("kv_full", kv_no % 4))
        for t in range(tiles):
            wait(("q_full", t))
            issue_s(t, i, 0, kv_no % 4, tile_no)
            if n == 1:
                push(("arrive", ("q_empty", t)))
            ready(t)
        push(("arrive", ("kv_empty", kv_no % 4)))
        for j in range(n):
            vs, ks, more = (kv_no + 1) % 4, (kv_no + 2) % 4, j + 1 < n
            wait(("kv_full", vs))
            wait(("v_ready", vs // 2))
            for t in range(tiles):
                wait(("p_early", t))
                if j == 0:
                    issue.append(("wait", ("o_empty", t), o_no[t]))
                    o_no[t] += 1
                push(mem.get(("ring", vs), ("v", tile_no)), *(mem.get(("p early", t, w), (i, j)) for w in range(WARPS)), mem.put(("o", t), "being added to"))
                wait(("p_full", t))
                if more and t == 0:
                    wait(("kv_full", ks))
                push(*(mem.get(("p", t, w), (i, j)) for w in range(WARPS)), mem.put(("o", t), (i, j)))
                if more:
                    issue_s(t, i, j + 1, ks, tile_no + 1)
                    if j + 2 == n:
                        push(("arrive", ("q_empty", t)))
                    ready(t)
                else:
                    push(("arrive", ("o_full", t)))
                    if with_p:
                        issue.append(("arrive", ("o_full", t)))
            push(("arrive", ("kv_empty", vs)))
            if more:
                push(("arrive", ("kv_empty", ks)))
            kv_no, tile_no = kv_no + 2, tile_no + 1
    actors["products"] = issue
    actors["tensor cores"] = _tensor_core(queue, counts)
    # ---- loads
    ops, q_no, state = [], [0, 0], {"kv": 0, "tile": 0}

    def load(kind):
        slot = state["kv"] % 4
        ops.append(("wait", ("kv_empty", slot), state["kv"] // 4))
        if kind == "k":
            ops.append(mem.put(("info", state["tile"] % 4), state["tile"]))
        ops.extend([mem.put(("ring", slot), (kind, state["tile"])), ("arrive", ("kv_full", slot))])
        state["kv"] += 1
    for i, (tiles, n) in enumerate(items):
        load("k")
        for t in range(tiles):
            ops += [("wait", ("q_empty", t), q_no[t]), mem.put(("q", t), i), ("arrive", ("q_full", t))]
            q_no[t] += 1
        load("v")
        state["tile"] += 1
        for j in range(1, n):
            load("k")
            load("v")
            state["tile"] += 1
    actors["loads"] = ops
    # ---- hidden rows of V
    for w in range(WARPS):
        ops, v_no, tile_no = [], {1: 0, 3: 0}, 0
        for i, (tiles, n) in enumerate(items):
            for j in range(n):
                slot = (2 * tile_no + 1) % 4
                v_no[slot] += 1
                ops += [("wait", ("kv_full", slot), v_no[slot]), mem.get(("info", tile_no % 4), tile_no), mem.get(("ring", slot), ("v", tile_no)), ("arrive", ("v_ready", slot // 2))]
                tile_no += 1
        actors[f"hidden rows {w}"] = ops
    # ---- rows out
    for w in range(WARPS):
        ops, o_seen, mine = [], [0, 0], [0, 0]
        for i, (tiles, n) in enumerate(items):
            for t in range(tiles):
                o_seen[t] += 1
                at = mine[t] if slot_by_tile else i
                ops += [("wait", ("o_full", t), o_seen[t]), mem.get(("l", at % 2, t, w), i), mem.get(("o", t), (i, n - 1)), ("arrive", ("o_empty", t))]
                mine[t] += 1
        actors[f"rows out {w}"] = ops
    return actors, counts


def _go_through(build, items, **kw):
    for held, ops in build(items, **kw)[0].items():
        if held != "tensor cores":
            for stop in range(len(ops)):
                _run(*build(items, **kw), held, stop)
    rng = random.Random(0)
    for _ in range(20):
        _run(*build(items, **kw), rng=rng)


@pytest.mark.parametrize("items", RUNS)
def test_cache_form(items):
    _go_through(_cache_form, items)


@pytest.mark.parametrize("items", RUNS)
def test_rows_form(items):
    _go_through(_rows_form, items)


def test_a_slot_by_items_of_the_cta_is_found_out():
    """l of a second tile, its slot taken by the number of the CTA's item: an item without a second tile lets the next but one overwrite it."""
    with pytest.raises(Hazard, match="l"):
        _go_through(_rows_form, RUNS[1], slot_by_tile=False)


def test_an_arrival_of_its_own_for_the_sums_is_found_out():
    """l announced by its writers' arrivals behind p: a warp of one item later arrives in place of one that is late."""
    with pytest.raises(Hazard, match="l"):
        _go_through(_rows_form, RUNS[0], with_p=False)


@pytest.mark.parametrize("items", RUNS[:3])
def test_one_barrier_for_logits_and_sums_is_found_out(items):
    """With "O is done" and the next item's first logits on one barrier, the issuing warp's arrivals for both complete it before either product is
    done, and a softmax warp that is late misses a completion."""
    with pytest.raises(Hazard):
        _go_through(_cache_form, items, own_o_full=False)
