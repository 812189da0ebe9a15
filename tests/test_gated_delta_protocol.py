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

TABLES = 4
READERS = {"KQ": 1, "V": 16, "TB": 1, "table": 20, "S": 1, "X": 8, "R": 1, "U": 8, "W": 1, "P": 8, "out": 4,
           "xq": 4, "over": 4}


class _Barrier:
    def __init__(self, count):
        self.count = self.pending = count
        self.done = 0

    def arrive(self):
        self.pending -= 1
        if self.pending == 0:
            self.done += 1
            self.pending = self.count


def _roles(ns, n, alias, out=True):
    """(barriers, role name -> generator) of one CTA with n chunks, ns stages; alias: O lies on
    U (D = 256); out: outputs are made (not in a first pass over segments). The names are the kernel's."""
    bars = {}

    def add(names, number, count):
        for name in names.split():
            for i in range(number):
                bars[name, i] = _Barrier(count)

    add("LF LE", ns, 1)
    add("TF", TABLES, 1)
    add("TE", TABLES, 20 if out else 16)
    add("XD UD PD", 2, 1)
    add("OD", 1, 1)
    add("OE", 1, 4)
    # named barriers, in warps; those in pairs are of the chain's halves
    add("barS barR barW", 2, 9)
    add("barEnd", 1, 20)

    def wait(name, phase, i=0):
        return "wait", (name, i), phase

    def arrive(name, i=0):
        return "arrive", (name, i), None

    def sync(name, i=0):
        return "sync", (name, i), None

    def issue(reads, writes, *barriers):  # a batch of MMAs: what it reads and writes, the barriers it arrives on
        return "issue", barriers, (reads, writes)

    def reads(*what):
        return "reads", what, None

    def writes(*what):
        return "writes", what, None

    def mma():
        for c in range(n):
            s = c % ns
            yield wait("LF", c // ns, s)
            yield sync("barS", 0)
            yield issue([("KQ", s, c, 0), ("S", 0, c, not out)], [])
            yield sync("barS", 1)
            yield issue([("KQ", s, c, 0), ("S", 1, c, not out)], [("X", 0, c), ("X", 1, c)], ("XD", 0), ("XD", 1))
            if out and alias and c > 0:
                yield wait("OE", c - 1)
            if out:
                yield issue([("KQ", s, c, 0), ("S", 0, c, 1), ("S", 1, c, 1)], [("xq", 0 if alias else c & 1, c)])
            yield sync("barR", 0)
            yield issue([("R", 0, c, 0), ("TB", s, c, 0)], [("U", 0, c)] + [("over", 0, c)] * (alias and out), ("UD", 0))
            yield sync("barR", 1)
            yield issue([("R", 0, c, 1), ("R", 1, c, 1), ("TB", s, c, 0)], [("U", 1, c)], ("UD", 1))
            yield sync("barW", 0)
            yield issue([("KQ", s, c, 0), ("W", 0, c, 0)], [])
            yield sync("barW", 1)
            yield issue([("KQ", s, c, 1), ("W", 1, c, 0)], [("P", 0, c), ("P", 1, c)], ("PD", 0), ("PD", 1))
            if out and not alias and c > 0:
                yield wait("OE", c - 1)
            yield issue([("TB", s, c, 1), ("W", 0, c, 1), ("W", 1, c, 1)], [("out", 0, c)] * out, ("OD", 0), ("LE", s))
        if n:
            yield wait("OD", n - 1)
            yield wait("LE", (n - 1) // ns, (n - 1) % ns)

    def loads():
        for c in range(n):
            if c >= ns:
                yield wait("LE", c // ns - 1, c % ns)
            yield "load", ("LF", c % ns), [(what, c % ns, c) for what in ("KQ", "V", "TB")]

    def table(first):
        for c in range(first, n, 2):
            if c >= TABLES:
                yield wait("TE", c // TABLES - 1, c % TABLES)
            yield writes(("table", c % TABLES, c))
            yield arrive("TF", c % TABLES)

    def outputs(i):
        for c in range(n if out else 0):
            yield wait("TF", c // TABLES, c % TABLES)
            yield wait("OD", c)
            for _ in range(30):  # (they take their time)
                yield reads()
            yield reads(("out", 0, c, 1), ("xq", 0 if alias else c & 1, c, 1), *[("over", 0, c, 1)] * alias)
            yield arrive("OE")
            yield reads(("table", c % TABLES, c, 1))
            yield arrive("TE", c % TABLES)
        yield sync("barEnd")

    def chain(i):
        half = i // 8

        def fetch(c):
            yield wait("LF", c // ns, c % ns)
            yield wait("TF", c // TABLES, c % TABLES)
            yield reads(("V", c % ns, c, 1), ("table", c % TABLES, c, 0))

        if n:
            yield from fetch(0)
        for c in range(n):
            if i % 8 == 0:
                yield writes(("S", half, c))
            yield arrive("barS", half)
            yield wait("XD", c, half)
            yield reads(("X", half, c, 1))
            if i % 8 == 0:
                yield writes(("R", half, c))
            yield arrive("barR", half)
            yield reads(("table", c % TABLES, c, 0))
            yield wait("UD", c, half)
            yield reads(("U", half, c, 1))
            if i % 8 == 0:
                yield writes(("W", half, c))
            yield arrive("barW", half)
            yield reads(("table", c % TABLES, c, 1))
            yield arrive("TE", c % TABLES)
            if c + 1 < n:
                yield from fetch(c + 1)
            yield wait("PD", c, half)
            yield reads(("P", half, c, 1))
        yield sync("barEnd")

    roles = {"mma": mma(), "loads": loads(), "table 0": table(0), "table 1": table(1)}
    roles.update({f"outputs {i}": outputs(i) for i in range(4)})
    roles.update({f"chain {i}": chain(i) for i in range(16)})
    return bars, roles


class _Buffers:
    """name, place -> the chunk in it and how many last reads of it are still to come."""

    def __init__(self, readers):
        self.held, self.readers = {}, readers

    def write(self, name, place, chunk):
        old = self.held.get((name, place))
        assert old is None or old[1] <= 0, f"{name} {place}: chunk {chunk} over {old[0]}, of which {old[1]} reads are open"
        self.held[name, place] = [chunk, self.readers[name]]

    def read(self, name, place, chunk, last):
        old = self.held.get((name, place))
        assert old is not None and old[0] == chunk, f"{name} {place}: chunk {old and old[0]} read as {chunk}"
        old[1] -= last


def _run(ns, n, seed, edit=None, alias=False, out=True):
    rng = random.Random(seed)
    bars, roles = _roles(ns, n, alias, out)
    if edit is not None:
        edit(bars, roles)
    buffers = _Buffers(READERS if out else {**READERS, "table": 16})
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
            if op[0] == "joined" and bars[op[1]].done == op[2]:
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
            for w in what:
                buffers.write(*w)
            bars[barrier].arrive()
        else:
            kind, what, more = at[name]
            if kind == "sync":  # arrives, and waits for the others
                at[name] = "joined", what, bars[what].done
                bars[what].arrive()
                continue
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


@pytest.mark.parametrize("stages,alias", [(3, False), (2, True)])
@pytest.mark.parametrize("out", [True, False])
@pytest.mark.parametrize("chunks", [0, 1, 2, 3, 4, 5, 9, 14])
def test_no_order_stalls_or_overtakes(stages, alias, chunks, out):
    for seed in range(20):
        _run(stages, chunks, seed, alias=alias, out=out)


@pytest.mark.parametrize("name,role", [("LE", "loads"), ("TE", "table"), ("barR", "mma"),
                                       ("barS", "mma"), ("PD", "chain"), ("OD", "outputs"),
                                       ("OE", "mma")])
def test_a_wait_left_out_is_seen(name, role):
    def edit(bars, roles):
        for r in [r for r in roles if r.startswith(role)]:
            roles[r] = (op for op in list(roles[r]) if not (op[0] in ("wait", "sync") and op[1][0] == name))

    for alias in (False, True):
        with pytest.raises(AssertionError):
            for seed in range(40):
                _run(3, 9, seed, edit, alias)


@pytest.mark.parametrize("name,role", [("XD", "chain"), ("UD", "chain"), ("barW", "mma"), ("LF", "chain"),
                                       ("TF", "chain")])
def test_any_wait_left_out_is_seen(name, role):
    """The waits that order X -> R, U -> w U and w U -> P, and those for tiles and tables."""
    def edit(bars, roles):
        for r in [r for r in roles if r.startswith(role)]:
            roles[r] = (op for op in list(roles[r]) if not (op[0] in ("wait", "sync") and op[1][0] == name))

    for alias in (False, True):
        with pytest.raises(AssertionError):
            for seed in range(40):
                _run(3, 9, seed, edit, alias)
