"""The barriers of the short polynomial (csrc/muon.cu, iterate and iterate_small: up to 16 rows), simulated on the host under
random interleavings of a block's warps.

Every warp reads the trace from G's diagonal. Then the chain warps (one for each tile) make S, V and the next G of every
step, the P warps follow with P' = S P, and all warps scale P by the factor that they took from the trace. Each tile of a
matrix carries the step that wrote it; the check is that every read finds the step that it means and that every schedule
runs to its end. A named barrier completes when its number of warps have arrived, whether they wait or not."""
import os
import random
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "smel-ft_b200", "csrc", "muon.cu")
WARPS = 8


def warp(w, nt, steps, trace_barrier):
    """The operations of warp w, in the order of the device code."""
    T = nt * nt
    diagonal = [("G", i * nt + i) for i in range(nt)]
    whole = lambda m: [(m, n) for n in range(T)]  # noqa: E731
    yield ("read", diagonal, 0)
    if trace_barrier:
        yield ("sync", "block", WARPS)
    if w < T:  # chain
        yield ("read", [("G", w)], 0)
        for k in range(steps):
            s = f"S{k & 1}"
            yield ("read", whole("G"), k)
            if k >= 2:
                yield ("sync", 5 + (k & 1), 2 * T)
            yield ("write", (s, w), k)
            yield ("arrive", 3 + (k & 1), 2 * T)
            if k + 1 == steps:
                break
            yield ("sync", 1, T)
            yield ("read", whole(s), k)
            yield ("read", whole("G"), k)
            yield ("write", ("V", w), k)
            yield ("sync", 1, T)
            yield ("read", whole(s), k)
            yield ("read", whole("V"), k)
            yield ("write", ("G", w), k + 1)
            yield ("sync", 1, T)
    elif w < 2 * T:  # P
        for k in range(steps):
            s, to, frm = f"S{k & 1}", f"M{k & 1}", f"M{(k + 1) & 1}"
            yield ("sync", 3 + (k & 1), 2 * T)
            if k:
                yield ("read", whole(s), k)
                yield ("read", whole(frm), k - 1)
            else:
                yield ("read", [(s, w - T)], k)
            yield ("write", (to, w - T), k)
            if k + 2 < steps:
                yield ("arrive", 5 + (k & 1), 2 * T)
            yield ("sync", 2, T)
    yield ("sync", "block", WARPS)
    yield ("read", [(f"M{(steps - 1) & 1}", n) for n in range(T) if n % WARPS == w], steps - 1)


def run(nt, steps, seed, trace_barrier=True):
    """A random schedule; the reads that found another step's tile."""
    rng = random.Random(seed)
    weight = [rng.choice((1, 1, 20)) for _ in range(WARPS)]  # some warps are late
    memory = {("G", n): 0 for n in range(nt * nt)}
    warps = {w: warp(w, nt, steps, trace_barrier) for w in range(WARPS)}
    ready, arrived, waiting, wrong = dict.fromkeys(range(WARPS)), {}, {}, []
    while warps:
        assert ready, f"no warp can go on: {waiting}"
        w = rng.choices(list(ready), [weight[v] for v in ready])[0]
        op = next(warps[w], None)
        if op is None:
            del warps[w], ready[w]
        elif op[0] == "write":
            memory[op[1]] = op[2]
        elif op[0] == "read":
            wrong += [(w, at, op[2], memory.get(at)) for at in op[1] if memory.get(at) != op[2]]
        else:
            kind, bar, count = op
            arrived[bar] = arrived.get(bar, 0) + 1
            if kind == "sync":
                waiting.setdefault(bar, []).append(w)
                del ready[w]
            if arrived[bar] == count:
                arrived[bar] = 0
                ready.update(dict.fromkeys(waiting.pop(bar, ())))
    assert not any(arrived.values())
    return wrong


@pytest.mark.parametrize("nt", [1, 2])
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 5, 8])
def test_every_read_finds_its_step(nt, steps):
    for seed in range(150):
        assert run(nt, steps, seed) == []


def test_the_trace_needs_its_barrier():
    """Without a barrier behind the trace a late warp reads the diagonal of a later step's G."""
    for nt in (1, 2):
        wrong = [x for seed in range(300) for x in run(nt, 5, seed, trace_barrier=False)]
        assert wrong and all(at[0] == "G" and meant == 0 and found > 0 for _, at, meant, found in wrong)


def test_the_kernel_has_the_barrier():
    with open(SOURCE) as f:
        text = f.read()
    body = text[text.index("__device__ double* iterate("):]
    trace = body[body.index("tr +="):body.index("iterate_small<NT>(")]
    assert re.search(r"__shfl_xor_sync.*__syncthreads\(\);", trace, re.S)


def cluster(blocks, seed, give_up=True):
    """The exchange of the Gram parts (ortho_kernel) with pushes that take any time and waits that may give up: per block
    whether it stored, and what landed in a block that had left."""
    rng = random.Random(seed)
    landed, left, stored, lost = [0] * blocks, [False] * blocks, [False] * blocks, []
    arrivals = {"up": 0, "exit": 0}
    flying = []  # receivers of pushes under way

    def block(r):
        arrivals["up"] += 1
        yield lambda: arrivals["up"] == blocks
        flying.extend(range(blocks))
        there = True
        if give_up and rng.random() < 0.3:
            there = landed[r] == blocks  # the wait's limit, whatever has come by now
        else:
            yield lambda: landed[r] == blocks
        arrivals["exit"] += 1
        if there:
            stored[r] = landed[r] == blocks
            assert stored[r]
        yield lambda: arrivals["exit"] == blocks
        if not there:
            yield lambda: landed[r] == blocks
        left[r] = True

    runs = {r: block(r) for r in range(blocks)}
    until = {r: lambda: True for r in range(blocks)}
    while runs or flying:
        can = [r for r in runs if until[r]()]
        assert can or flying
        if flying and (not can or rng.random() < 0.2):
            to = flying.pop(rng.randrange(len(flying)))
            landed[to] += 1
            lost += [to] if left[to] else []
        else:
            r = rng.choice(can)
            until[r] = next(runs[r], None)
            if until[r] is None:
                del runs[r]
    return stored, lost


@pytest.mark.parametrize("blocks", [2, 4, 8])
def test_pushes_land_in_blocks_that_are_still_there(blocks):
    """A block whose wait gives up stores nothing and stays until the others' parts have landed; the rest is not disturbed."""
    some = 0
    for seed in range(400):
        stored, lost = cluster(blocks, seed)
        assert lost == []
        some += not all(stored)
        assert cluster(blocks, seed, give_up=False) == ([True] * blocks, [])
    assert some


def test_the_kernel_heeds_the_wait():
    with open(SOURCE) as f:
        text = f.read()
    body = text[text.index(" ortho_kernel(const"):]
    body = body[:body.index("\n}\n")]
    waits = re.findall(r"(\w+ = )?mbar_wait\(", body)
    assert len(waits) == 2 and waits[0]
    assert body.index("__syncthreads_and(") < body.index("iterate<") < body.index("store_slice<")
