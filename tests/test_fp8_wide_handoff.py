"""The named barriers by which the wide fp8 product hands a block's sums over, simulated on the host: nobody waits for good, even where
the memory barriers' limited waits run out.

Which role syncs or only arrives on which barrier is read from the kernel's source. A barrier completes with its ninth warp (eight that
add the sums up and one beside them); its count and its waiting warps then begin anew.
"""

import os
import random
import re

import pytest

from qr_v2_b200_kernel_b200 import build

WARPS = 8


def _calls():
    source = open(os.path.join(build.CSRC, "fp8_linear.cuh")).read()
    source = source[source.index("fp8_wide_kernel(") :]

    def one(barrier, index):
        found = re.findall(rf"named_(sync|arrive)\({barrier} \+ {index}, kFp8Hand\)", source)
        assert len(found) == 1
        return found[0]

    return {"tell": one(1, r"\(j & 1\)"), "told": one(1, "buf"), "take": one(3, "buf"), "taken": one(3, r"\(j & 1\)")}


def _simulate(calls, blocks, stop, rng):
    """Runs the roles in random order; the product of block `stop` never ends. Returns whether all of them come to their end."""
    done, freed = [0], [0]  # blocks multiplied; accumulators given back
    ran_out = [False]

    def adds():
        for j in range(blocks):
            yield calls["told"], 1 + j % 2
            yield calls["take"], 3 + j % 2

    def tells():
        for j in range(blocks):
            if not ran_out[0]:
                while done[0] <= j and j < stop:
                    yield "wait", None
                if j >= stop:  # the limit
                    ran_out[0] = True
            yield calls["tell"], 1 + j % 2

    def takes():
        for j in range(blocks):
            yield calls["taken"], 3 + j % 2
            freed[0] += 1

    def multiplies():
        for j in range(min(stop, blocks)):
            while freed[0] < j - 1:
                yield "wait", None
            done[0] += 1
            yield "wait", None

    roles = [adds() for _ in range(WARPS)] + [tells(), takes(), multiplies()]
    state = ["run"] * len(roles)
    count, waiting = [0] * 5, [[] for _ in range(5)]
    idle = 0
    while any(s != "end" for s in state):
        able = [i for i, s in enumerate(state) if s == "run"]
        if not able or idle > 50 * len(roles):
            return False
        i = rng.choice(able)
        try:
            what, barrier = next(roles[i])
        except StopIteration:
            state[i] = "end"
            idle = 0
            continue
        if what == "wait":
            idle += 1
            continue
        idle = 0
        count[barrier] += 1
        if what == "sync":
            waiting[barrier].append(i)
            state[i] = "blocked"
        if count[barrier] == WARPS + 1:
            for w in waiting[barrier]:
                state[w] = "run"
            count[barrier], waiting[barrier] = 0, []
    return True


@pytest.mark.parametrize("blocks", [1, 2, 3, 32, 65])
def test_every_role_comes_to_its_end(blocks):
    calls = _calls()
    for seed in range(200):
        rng = random.Random(seed)
        stop = rng.choice([blocks, rng.randrange(blocks + 1)])
        assert _simulate(calls, blocks, stop, rng), (seed, stop)


def test_the_simulation_finds_a_hand_over_that_stalls():
    # the signals not waited for: fine as long as the products hold them back, not where those end
    calls = {"tell": "arrive", "told": "sync", "take": "arrive", "taken": "sync"}
    assert all(_simulate(calls, 32, 32, random.Random(seed)) for seed in range(50))
    assert not all(_simulate(calls, 32, 3, random.Random(seed)) for seed in range(50))
