"""What the chunked gated-delta kernel does when a wait runs out, on the host: no GPU is made to stall.

The roles are those of test_gated_delta_protocol, with waits that give up: a role whose wait has run out waits for no
mbarrier any more and goes through its code to the end, the MMA and load warps without issuing anything. Named barriers
count arrivals, as the hardware does. The chain's warps, which otherwise only arrive at them, join them once they have
given up (``hand_over`` in the kernel).
"""

import random
import re
from pathlib import Path

import pytest

from test_gated_delta_protocol import _roles

CSRC = Path(__file__).resolve().parents[1] / "memt-1.0_b200" / "csrc"
NAMED = ("barS", "barR", "barW", "barEnd")


class _Stuck(Exception):
    pass


def _run(ns, n, seed, alias, out, lose=None, gives_up=None, joins=True):
    """Runs until every role has ended, or raises _Stuck. lose: ("tile" or "batch", k), the k-th never
    lands or completes, nor do the batches behind it; gives_up: (role, i), that role's i-th wait runs out at once.
    joins: whether the chain's warps join named barriers once they have given up. Returns the roles that gave up."""
    rng = random.Random(seed)
    bars, roles = _roles(ns, n, alias, out)
    at = {name: next(role, None) for name, role in roles.items()}
    dead, last, waits = set(), {}, dict.fromkeys(at, 0)
    batches, tiles, issued = [], [], {"tile": 0, "batch": 0}
    weight = {name: rng.choice([1, 1, 5, 30]) for name in [*at, "tensor pipe", "tma"]}

    def reach(name, bar):  # an arrival at a named barrier: at most one of a warp in a phase
        if last.get((name, bar)) == bars[bar].done:
            raise _Stuck(f"{name} arrives twice in phase {bars[bar].done} of {bar}")
        last[name, bar] = bars[bar].done
        bars[bar].arrive()

    while True:
        ready, waiting = [], []
        for name, op in at.items():
            if op is None or op[0] == "joined" and bars[op[1]].done == op[2]:
                continue
            if op[0] == "wait" and name not in dead and bars[op[1]].done % 2 == op[2] % 2:
                waiting.append(name)
                if (name, waits[name]) == gives_up:
                    dead.add(name)
                else:
                    continue
            ready.append(name)
        ready += ["tensor pipe"] * bool(batches) + ["tma"] * bool(tiles)
        if not ready:
            if not waiting:
                left = {name: op for name, op in at.items() if op is not None}
                if left:
                    raise _Stuck(str(left))
                return dead
            dead.add(rng.choice(waiting))  # half a second later
            continue
        name = rng.choices(ready, [weight[r] for r in ready])[0]
        if name == "tensor pipe":
            for b in batches.pop(0):
                bars[b].arrive()
            continue
        if name == "tma":
            bars[tiles.pop(rng.randrange(len(tiles)))].arrive()
            continue
        kind, what, more = at[name]
        if kind == "wait":
            waits[name] += 1
        elif kind == "sync" or kind == "arrive" and what[0] in NAMED and name in dead and joins:
            at[name] = "joined", what, bars[what].done
            reach(name, what)
            continue
        elif kind == "arrive":
            if what[0] in NAMED:
                reach(name, what)
            else:
                bars[what].arrive()
        elif kind in ("issue", "load") and name not in dead:
            queue, sort = (batches, "batch") if kind == "issue" else (tiles, "tile")
            if lose is None or lose[0] != sort or issued[sort] < lose[1] or sort == "tile" and issued[sort] > lose[1]:
                queue.append(what)
            issued[sort] += 1
        at[name] = next(roles[name], None)


SHAPES = [(3, False), (2, True)]


@pytest.mark.parametrize("stages,alias", SHAPES)
@pytest.mark.parametrize("out", [True, False])
def test_every_role_ends_when_nothing_is_lost(stages, alias, out):
    for seed in range(20):
        assert _run(stages, 9, seed, alias, out) == set()


@pytest.mark.parametrize("stages,alias", SHAPES)
@pytest.mark.parametrize("out", [True, False])
@pytest.mark.parametrize("lose", [("tile", 0), ("tile", 3), ("tile", 8), ("batch", 0), ("batch", 10), ("batch", 33)])
def test_every_role_ends_when_something_is_lost(stages, alias, out, lose):
    for seed in range(15):
        assert _run(stages, 9, seed, alias, out, lose=lose)


@pytest.mark.parametrize("stages,alias", SHAPES)
@pytest.mark.parametrize("out", [True, False])
@pytest.mark.parametrize("role", ["mma", "loads", "table 0", "table 1", "outputs 2", "chain 0", "chain 7", "chain 12"])
def test_every_role_ends_when_one_gives_up(stages, alias, out, role):
    """Alone, with nothing lost: the others are still waiting for it."""
    for seed in range(4):
        for i in (0, 1, 2, 5, 8, 20):
            _run(stages, 9, seed, alias, out, gives_up=(role, i))


def test_passing_a_barrier_after_giving_up_gets_stuck():
    """What hand_over is for."""
    stuck = 0
    for seed in range(40):
        try:
            _run(3, 9, seed, False, True, lose=("tile", 3), joins=False)
        except _Stuck:
            stuck += 1
    assert stuck == 40


def _code(name):
    return re.sub(r"//.*", "", (CSRC / name).read_text())


def test_the_chain_joins_named_barriers_once_it_has_given_up():
    code = _code("delta_tc.cuh")
    body = re.search(r"auto hand_over = \[&\]\(int id\) \{(.*?)\};", code, re.S).group(1)
    assert re.sub(r"\s+", " ", body).strip() == "if (alive) bar_arrive<288>(id); else bar_sync<288>(id);"
    assert code.count("bar_arrive<288>") == 1  # nowhere else
    for bar in ("kBarS", "kBarR", "kBarW"):
        assert f"hand_over({bar} + half)" in code and f"bar_sync<288>({bar})" in code
    # a warp of the chain has given up as a whole: behind both places where it waits
    assert code.count("alive = __all_sync(~0u, alive);") == 2
