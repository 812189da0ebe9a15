"""The barrier protocol of the chunked linear-attention kernel, run on the host in random orders.

Each role of the kernel is a generator of its waits and arrivals, in the order of its code; MMA batches
complete in the order of their issue and tiles land in any. A wait names the phase it means. The barriers
only carry a phase's parity, so a wait must meet its barrier no more than one phase off: a later phase
that completes before the wait is made (overrun) would hang, an earlier one still open (underrun) would let it pass.
"""

import random

import pytest


class _Barrier:
    def __init__(self, count):
        self.count = self.pending = count
        self.done = 0

    def arrive(self):
        self.pending -= 1
        if self.pending == 0:
            self.done += 1
            self.pending = self.count


def _roles(D, OUT, n, ragged):
    """(barriers, role name -> generator) of one CTA with n chunks. The names are the kernel's."""
    units, alias, stages, tables = (2 if D == 256 else 1), D == 256, {256: 2, 128: 3, 64: 4}[D], 4
    bars = {}

    def add(names, number, count):
        for name in names.split():
            for i in range(number):
                bars[name, i] = _Barrier(count)

    add("QF KF VF QE KE VE", stages, 1)
    add("TF", tables, 1)
    add("TE", tables, 16)
    add("BU", units, 1)
    add("UE", units, 8 if units == 1 else 4)
    add("VW BP SB OE", 1, 8)
    add("SC XD XY", 1, 1)

    def wait(name, i, phase):
        return "wait", (name, i), phase

    def arrive(name, i=0):
        return "arrive", (name, i), None

    def issue(*barriers):  # a batch of MMAs and the barriers its commits arrive on
        return "issue", barriers, None

    def mma():
        def scores(c):
            yield wait("QF", c % stages, c // stages)
            yield wait("KF", c % stages, c // stages)
            yield issue(("SC", 0))

        def state_sums(c, u):
            if u == 0:
                if not OUT:
                    yield wait("KF", c % stages, c // stages)
                yield wait("VW", 0, c)
            if u > 0:
                yield wait("UE", 0, c)
            elif c > 0:
                yield wait("UE", units - 1, c - 1)
            last = u == units - 1
            yield issue(("BU", u), *([("KE", c % stages)] if last else []),
                        *([("VE", c % stages)] if last and not OUT else []))

        def outputs(c):
            yield wait("SB", 0, c)
            if not alias and c > 0:
                yield wait("OE", 0, c - 1)
            yield issue(("XD", 0), ("QE", c % stages))
            yield wait("BP", 0, c)
            yield issue(("XY", 0), ("VE", c % stages))

        if OUT and n:
            yield from scores(0)
        for c in range(n):
            yield from state_sums(c, 0)
            if OUT:
                yield from outputs(c)
            if units == 2:
                yield from state_sums(c, 1)
            if OUT and c + 1 < n:
                if alias:
                    yield wait("OE", 0, c)
                yield from scores(c + 1)

    def loads():
        for c in range(n):
            for full, free in (("VF", "VE"), ("QF", "QE"), ("KF", "KE")):
                if full == "QF" and not OUT:
                    continue
                if c >= stages:
                    yield wait(free, c % stages, c // stages - 1)
                yield "load", (full, c % stages), None

    def table(first):
        for c in range(first, n, 2):
            if c >= tables:
                yield wait("TE", c % tables, c // tables - 1)
            yield arrive("TF", c % tables)

    def work():
        def split(c):
            yield wait("VF", c % stages, c // stages)
            if ragged and c == n - 1:
                yield wait("KF", c % stages, c // stages)
            yield wait("TF", c % tables, c // tables)
            if c > 0:
                yield wait("BU", units - 1, c - 1)
            yield arrive("VW")
            if not OUT:
                yield arrive("TE", c % tables)

        def write(c):
            yield wait("XY", 0, c)
            yield arrive("OE")
            yield arrive("TE", c % tables)

        for c in range(n):
            yield from split(c)
            if OUT and (alias or c > 0):
                yield from write(c if alias else c - 1)
        if OUT and not alias and n:
            yield from write(n - 1)

    def state(half):
        for c in range(n):
            if OUT:
                if c > 0:
                    yield wait("XD", 0, c - 1)
                yield arrive("SB")
            yield wait("TF", c % tables, c // tables)
            if OUT:
                yield wait("SC", 0, c)
                yield arrive("BP")
            u = half if units == 2 else 0
            yield arrive("TE", c % tables)
            yield wait("BU", u, c)
            yield arrive("UE", u)

    roles = {"mma": mma(), "loads": loads(), "table 0": table(0), "table 1": table(1)}
    roles.update({f"work {i}": work() for i in range(8)})
    roles.update({f"state {i}": state(i // 4) for i in range(8)})
    return bars, roles


def _run(D, OUT, n, seed, edit=None):
    rng = random.Random(seed)
    bars, roles = _roles(D, OUT, n, ragged=seed % 2 == 0)
    if edit is not None:
        edit(bars, roles)
    at = {name: next(role, None) for name, role in roles.items()}
    batches, tiles = [], []
    weight = {name: rng.choice([1, 1, 5, 30]) for name in [*at, "tensor pipe", "tma"]}  # slow and fast ones
    while True:
        ready = []
        for name, op in at.items():
            if op is None:
                continue
            if op[0] == "wait":
                done = bars[op[1]].done
                assert done <= op[2] + 1, f"overrun: {name} waits for phase {op[2]} of {op[1]}, {done} are done"
                assert done >= op[2], f"underrun: {name} waits for phase {op[2]} of {op[1]}, {done} are done"
                if done == op[2]:
                    continue
            ready.append(name)
        ready += ["tensor pipe"] * bool(batches) + ["tma"] * bool(tiles)
        if not ready:
            stuck = {name: op for name, op in at.items() if op is not None}
            assert not stuck, f"deadlock: {stuck}"
            return
        name = rng.choices(ready, [weight[r] for r in ready])[0]
        if name == "tensor pipe":
            for b in batches.pop(0):
                bars[b].arrive()
        elif name == "tma":
            bars[tiles.pop(rng.randrange(len(tiles)))].arrive()
        else:
            kind, what, _ = at[name]
            if kind == "arrive":
                bars[what].arrive()
            elif kind == "issue":
                batches.append(what)
            elif kind == "load":
                tiles.append(what)
            at[name] = next(roles[name], None)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("OUT", [True, False])
@pytest.mark.parametrize("chunks", [0, 1, 2, 3, 4, 5, 9, 14])
def test_no_order_stalls_or_overtakes(D, OUT, chunks):
    for seed in range(8):
        _run(D, OUT, chunks, seed)


def test_a_planted_mistake_is_found():
    """State warps that do not wait for the products that read their copy write it a phase early."""
    def edit(bars, roles):
        for i in range(8):
            role = roles[f"state {i}"]
            roles[f"state {i}"] = (op for op in role if op[:2] != ("wait", ("XD", 0)))
        bars["SB", 0].count = bars["SB", 0].pending = 1

    with pytest.raises(AssertionError, match="overrun|underrun|deadlock"):
        for seed in range(40):
            _run(128, True, 9, seed, edit)
