"""The barrier protocol of the chunked gated-delta kernel, run on the host in random orders.

Each role of the kernel is a generator of its waits and arrivals, in the order of its code; MMA batches complete in
the order of their issue and tiles land in any. A wait names the phase it means. The barriers only carry a phase's
parity, so a wait must meet its barrier no more than one phase off: a later phase that completes before the wait is
made (overrun) would hang, an earlier one still open (underrun) would let it pass. What the barriers guard is followed
too: every read of a buffer must find the chunk that it means there, and nothing may be overwritten that is
still to be read.
"""

import random

import pytest

STAGES, TABLES = {64: 4, 128: 3}, 4
READERS = {"KQ": 1, "V": 8, "table": 12, "scores": 4, "A": 4, "T": 1, "B": 1, "S": 1, "X": 8, "R": 1, "U": 8, "W": 1,
           "P": 8, "out": 4}


class _Barrier:
    def __init__(self, count):
        self.count = self.pending = count
        self.done = 0

    def arrive(self):
        self.pending -= 1
        if self.pending == 0:
            self.done += 1
            self.pending = self.count


def _roles(D, n):
    """(barriers, role name -> generator) of one CTA with n chunks. The names are the kernel's."""
    ns, bars = STAGES[D], {}

    def add(names, number, count):
        for name in names.split():
            for i in range(number):
                bars[name, i] = _Barrier(count)

    add("KF VF KE", ns, 1)
    add("VE", ns, 8)
    add("TF", TABLES, 1)
    add("TE", TABLES, 12)
    add("SC XD UD PD OD", 1, 1)
    add("SR AE TW OE", 1, 4)
    add("AW BW", 1, 2)
    add("SB RW WW", 1, 8)

    def wait(name, phase, i=0):
        return "wait", (name, i), phase

    def arrive(name, i=0):
        return "arrive", (name, i), None

    def issue(reads, writes, *barriers):  # a batch of MMAs: what it reads and writes, the barriers it arrives on
        return "issue", barriers, (reads, writes)

    def reads(*what):
        return "reads", what, None

    def writes(*what):
        return "writes", what, None

    def mma():
        def scores(c):
            yield wait("KF", c // ns, c % ns)
            if c > 0:
                yield wait("SR", c - 1)
            yield issue([("KQ", c % ns, c, 0)], [("scores", 0, c)], ("SC", 0))

        if n:
            yield from scores(0)
        for c in range(n):
            s = c % ns
            yield wait("SB", c)
            yield issue([("KQ", s, c, 0), ("S", 0, c, 0)], [("X", 0, c)], ("XD", 0))
            if c + 1 < n:
                yield from scores(c + 1)
            yield wait("RW", c)
            yield wait("TW", c)
            yield issue([("R", 0, c, 1), ("T", 0, c, 1)], [("U", 0, c)], ("UD", 0))
            if c > 0:
                yield wait("OE", c - 1)
            yield issue([("KQ", s, c, 0), ("S", 0, c, 1)], [("out", 0, c)])
            yield wait("WW", c)
            yield issue([("KQ", s, c, 1), ("W", 0, c, 0)], [("P", 0, c)], ("PD", 0), ("KE", s))
            yield wait("BW", c)
            yield issue([("B", 0, c, 1), ("W", 0, c, 1)], [], ("OD", 0))

    def loads():
        for c in range(n):
            s = c % ns
            for full, free, what in (("KF", "KE", "KQ"), ("VF", "VE", "V")):
                if c >= ns:
                    yield wait(free, c // ns - 1, s)
                yield "load", (full, s), (what, s, c)

    def table(first):
        for c in range(first, n, 2):
            if c >= TABLES:
                yield wait("TE", c // TABLES - 1, c % TABLES)
            yield writes(("table", c % TABLES, c))
            yield arrive("TF", c % TABLES)

    def invert(i):
        for c in range(n):
            yield wait("AW", c)
            yield reads(("A", 0, c, 1))
            if c > 0:
                yield wait("UD", c - 1)
            if i == 0:
                yield writes(("T", 0, c))
            yield arrive("TW")
            yield arrive("AE")

    def outputs(quad):
        b = quad >= 2

        def prepare(c):
            yield wait("TF", c // TABLES, c % TABLES)
            yield wait("SC", c)
            if c > 0:
                yield wait("OD" if b else "AE", c - 1)
            yield reads(("scores", 0, c, 1))
            if quad == 1 or quad == 3:
                yield writes(("B" if b else "A", 0, c))
            yield arrive("SR")
            yield arrive("BW" if b else "AW")

        def write_out(c):
            yield wait("OD", c)
            yield reads(("out", 0, c, 1))
            yield arrive("OE")
            yield reads(("table", c % TABLES, c, 1))
            yield arrive("TE", c % TABLES)

        for c in range(n):
            yield from prepare(c)
            if c > 0:
                yield from write_out(c - 1)
        if n:
            yield from write_out(n - 1)

    def chain(i):
        for c in range(n):
            s = c % ns
            if c > 0:
                yield reads(("P", 0, c - 1, 1))
            if i == 0:
                yield writes(("S", 0, c))
            yield arrive("SB")
            yield wait("VF", c // ns, s)
            yield wait("TF", c // TABLES, c % TABLES)
            yield reads(("V", s, c, 1))
            yield arrive("VE", s)
            yield wait("XD", c)
            yield reads(("X", 0, c, 1))
            if i == 0:
                yield writes(("R", 0, c))
            yield arrive("RW")
            yield wait("UD", c)
            yield reads(("U", 0, c, 1), ("table", c % TABLES, c, 1))
            if i == 0:
                yield writes(("W", 0, c))
            yield arrive("WW")
            yield arrive("TE", c % TABLES)
            yield wait("PD", c)
        if n:
            yield reads(("P", 0, n - 1, 1))

    roles = {"mma": mma(), "loads": loads(), "table 0": table(0), "table 1": table(1)}
    roles.update({f"invert {i}": invert(i) for i in range(4)})
    roles.update({f"outputs {i}": outputs(i) for i in range(4)})
    roles.update({f"chain {i}": chain(i) for i in range(8)})
    return bars, roles


class _Buffers:
    """name, place -> the chunk in it and how many last reads of it are still to come."""

    def __init__(self):
        self.held = {}

    def write(self, name, place, chunk):
        old = self.held.get((name, place))
        assert old is None or old[1] <= 0, f"{name} {place}: chunk {chunk} over {old[0]}, of which {old[1]} reads are open"
        self.held[name, place] = [chunk, READERS[name]]

    def read(self, name, place, chunk, last):
        old = self.held.get((name, place))
        if name == "W" and old is None and chunk == 0:
            return
        assert old is not None and old[0] == chunk, f"{name} {place}: chunk {old and old[0]} read as {chunk}"
        old[1] -= last


def _run(D, n, seed, edit=None):
    rng = random.Random(seed)
    bars, roles = _roles(D, n)
    if edit is not None:
        edit(bars, roles)
    buffers = _Buffers()
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
        if name == "tensor pipe":  # the oldest batch runs and completes
            barriers, (reads, writes) = batches.pop(0)
            for r in reads:
                buffers.read(*r)
            for w in writes:
                buffers.write(*w)
            for b in barriers:
                bars[b].arrive()
        elif name == "tma":
            barrier, what = tiles.pop(rng.randrange(len(tiles)))
            buffers.write(*what)
            bars[barrier].arrive()
        else:
            kind, what, more = at[name]
            if kind == "arrive":
                bars[what].arrive()
            elif kind == "issue":
                batches.append((what, more))
            elif kind == "load":
                tiles.append((what, more))
            elif kind == "reads":
                for r in what:
                    buffers.read(*r)
            elif kind == "writes":
                for w in what:
                    buffers.write(*w)
            at[name] = next(roles[name], None)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("chunks", [0, 1, 2, 3, 4, 5, 9, 14])
def test_no_order_stalls_or_overtakes(D, chunks):
    for seed in range(12):
        _run(D, chunks, seed)


@pytest.mark.parametrize("name,role", [("UD", "invert"), ("OD", "outputs"), ("KE", "loads"), ("TE", "table"),
                                       ("SR", "mma"), ("AE", "outputs"), ("RW", "mma"), ("SB", "mma"), ("PD", "chain")])
def test_a_wait_left_out_is_seen(name, role):
    def edit(bars, roles):
        for r in [r for r in roles if r.startswith(role)]:
            roles[r] = (op for op in list(roles[r]) if not (op[0] == "wait" and op[1][0] == name))

    with pytest.raises(AssertionError):
        for seed in range(40):
            _run(128, 9, seed, edit)
