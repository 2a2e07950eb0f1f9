"""The barriers at the end of a strip's tile (block_gemm_strip_kernel in csrc/fp8_block_gemm.cu), walked through every
interleaving on the CPU: timing on a GPU shows one order of events, this shows all of them.

A cluster of ranks shares the blocks of K of a tile.  In each rank an issuing warp fills accumulators and adding warps
drain them; at the end of a tile every adding warp pushes its sums into the ranks that own them, waits on its own rank's
`ready` (one arrival with the bytes to come, made by the first adding warp, and those bytes), adds, and arrives on every
rank's `released`, which is waited for before the next tile's pushes.  A wait knows a phase by its parity alone, so it
must not be overtaken by two phases; that depends on where the arrival on `ready` stands.  The order that the walk takes
for the kernel is read from the kernel's source."""
import os
import re
from collections import namedtuple

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = os.path.join(ROOT, "qwen3x-orin_b200", "csrc", "fp8_block_gemm.cu")

RANKS, WARPS, TILES = 2, 2, 3

# a barrier: completed phases, arrivals still missing in the phase at hand, bytes still to come (counted in pushes)
Barrier = namedtuple("Barrier", "completed missing bytes")
# issued blocks of K, accumulators filled and drained, the two barriers of a tile's end, pushes on their way, pushes landed,
# and for each adding warp the number of its program's steps that are behind it
Rank = namedtuple("Rank", "issued filled drained ready released coming landed at")


def settle(b, arrivals):
    return Barrier(b.completed + 1, arrivals, 0) if b.missing == 0 and b.bytes == 0 else b


def passed(completed, phase):
    """What a wait with this phase's parity answers: whether the barrier's phase at hand has the other parity."""
    return completed % 2 != phase % 2


def program(warp, blocks, order):
    steps = []
    for tile in range(TILES):
        steps += [("drain", tile, b) for b in range(blocks)]
        steps += [(what, tile, 0) for what in order if (what != "expect" or warp == 0) and (what != "await_released" or tile > 0)]
        steps += [("push", tile, 0), ("await_ready", tile, 0), ("release", tile, 0)]
    return steps


def walk(blocks, accumulators, owners, order):
    """None if every interleaving ends with all warps through their programs, else what goes wrong."""
    programs = [program(w, blocks, order) for w in range(WARPS)]
    ends = [len(p) for p in programs]
    # when a warp has released its tile: steps behind it
    released_at = [[i + 1 for i, s in enumerate(p) if s[0] == "release"] for p in programs]

    def issue(r):  # the issuing warp never waits for anything but `drained`: it goes as far as it can
        while r.issued < TILES * blocks:
            buffer, turn = r.issued % accumulators, r.issued // accumulators
            if turn > 0 and not passed(r.drained[buffer][0], turn - 1):
                break
            filled = list(r.filled)
            filled[buffer] += 1
            r = r._replace(issued=r.issued + 1, filled=tuple(filled))
        return r

    def step(state, rank, warp):
        """The state after the next step of a warp, None if it has to wait, or a text: a fault."""
        r = state[rank]
        what, tile, block = programs[warp][r.at[warp]]
        new = list(state)
        if what == "drain":
            n = tile * blocks + block
            buffer = n % accumulators
            if not passed(r.filled[buffer], n // accumulators):
                return None
            drained = list(r.drained)
            done, missing = drained[buffer]
            drained[buffer] = (done + 1, WARPS) if missing == 1 else (done, missing - 1)
            r = r._replace(drained=tuple(drained))
        elif what == "expect":
            b = Barrier(r.ready.completed, r.ready.missing - 1, r.ready.bytes + (RANKS * WARPS if owners[rank] else 0))
            if b.missing < 0:
                return "a second arrival in one phase of `ready`"
            r = r._replace(ready=settle(b, 1))
        elif what == "await_released":
            if not passed(r.released.completed, tile - 1):
                return None
        elif what == "push":
            for other in range(RANKS):
                if owners[other]:
                    o = new[other]
                    if tile > 0 and any(o.at[w] < released_at[w][tile - 1] for w in range(WARPS)):
                        return "sums pushed over ones that are still to be read"
                    new[other] = o._replace(coming=o.coming + 1)
            r = new[rank]
        elif what == "await_ready":
            if not passed(r.ready.completed, tile):
                return None
            if owners[rank] and r.landed < (tile + 1) * RANKS * WARPS:
                return "sums read before they came"
        else:
            for other in range(RANKS):
                o = new[other]
                b = Barrier(o.released.completed, o.released.missing - 1, 0)
                new[other] = o._replace(released=settle(b, RANKS * WARPS))
            r = new[rank]
        at = list(r.at)
        at[warp] += 1
        new[rank] = issue(r._replace(at=tuple(at)))
        return tuple(new)

    def land(state, rank):
        r = state[rank]
        ready = settle(Barrier(r.ready.completed, r.ready.missing, r.ready.bytes - 1), 1)
        return state[:rank] + (r._replace(coming=r.coming - 1, landed=r.landed + 1, ready=ready),) + state[rank + 1:]

    fresh = Rank(0, (0,) * accumulators, ((0, WARPS),) * accumulators, Barrier(0, 1, 0), Barrier(0, RANKS * WARPS, 0), 0, 0, (0,) * WARPS)
    start = (issue(fresh),) * RANKS
    seen, todo = {start}, [start]
    while todo:
        state = todo.pop()
        following, running = [], False
        for rank in range(RANKS):
            if state[rank].coming:
                following.append(land(state, rank))
            for warp in range(WARPS):
                if state[rank].at[warp] < ends[warp]:
                    running = True
                    new = step(state, rank, warp)
                    if isinstance(new, str):
                        return new
                    if new is not None:
                        following.append(new)
        if running and not following:
            return "stuck"
        for new in following:
            if new not in seen:
                seen.add(new)
                todo.append(new)
    return None


RIGHT = ("await_released", "expect")
WRONG = ("expect", "await_released")


def order_in_source():
    with open(SOURCE) as f:
        text = f.read()
    kernel = text[text.index("block_gemm_strip_kernel("):]
    expects = [m.start() for m in re.finditer(r"barrier_expect\(ready,", kernel)]
    waits = [m.start() for m in re.finditer(r"wait_warp\(released,", kernel)]
    pushes = [m.start() for m in re.finditer(r"\bpush\(at_rank", kernel)]
    assert len(expects) == len(waits) == len(pushes) == 1
    assert waits[0] < pushes[0] and expects[0] < pushes[0]
    return RIGHT if waits[0] < expects[0] else WRONG


# (owners: whether a rank owns tokens whose sums it adds; with few tokens the last ranks own none)
@pytest.mark.parametrize("owners", [(True, True), (True, False)])
@pytest.mark.parametrize("blocks,accumulators", [(1, 4), (2, 4), (3, 4), (4, 4), (5, 4), (1, 2), (2, 2), (3, 2)])
def test_every_interleaving_of_the_kernels_order_ends(blocks, accumulators, owners):
    assert walk(blocks, accumulators, owners, order_in_source()) is None


def test_the_walk_sees_an_arrival_that_overtakes_a_sister_warp():
    """With the arrival on `ready` in front of the wait on `released`, a rank without tokens completes a phase alone, and
    with as many accumulators as blocks nothing holds its first warp to the others."""
    assert walk(4, 4, (True, False), WRONG) == "stuck"
    assert walk(3, 4, (True, False), WRONG) == "stuck"
    # what hid it: every rank owns tokens, or the accumulators come round within a tile
    assert walk(4, 4, (True, True), WRONG) is None
    assert walk(3, 2, (True, False), WRONG) is None


def test_the_walk_sees_pushes_that_do_not_wait():
    assert walk(2, 4, (True, True), ("expect",)) == "sums pushed over ones that are still to be read"
