"""The chunked gated-delta kernel's order of products and hand-overs, run on the host in random orders: test_gated_delta_protocol's
machine with the roles as they are where U's terms for the outputs have a hand-over of their own, and with tensor memory
followed column block by column block, as its pieces hold one thing after another within a chunk:

    X's columns of 16 tokens     X, then U's two terms
    R's                          R's two terms
    U's (D = 256: then O)        U, then w U's two terms
    S's                          S's terms, then P
"""

import pytest

import test_gated_delta_protocol as P

TABLES = P.TABLES
# how many reads each thing sees before its place is written again (a batch of products reads once)
READERS = {"KQ": 1, "V": 16, "TB": 1, "table": 20, "X": 1, "R": 1, "U": 1, "W": 1, "Uo": 1, "S": 1, "Pp": 1, "P": 1, "xq": 4,
           "O": 4}


class _Cells(P._Buffers):
    """Places hold (thing, chunk)."""

    def write(self, place, _, what):
        old = self.held.get(place)
        assert old is None or old[1] <= 0, f"{place}: {what} over {old[0]}, of which {old[1]} reads are open"
        self.held[place] = [what, self.readers[what[0]]]

    def read(self, place, _, what, last):
        old = self.held.get(place)
        assert old is not None and old[0] == what, f"{place}: {old and old[0]} read as {what}"
        old[1] -= last


def roles(ns, n, alias, out=True):
    """As test_gated_delta_protocol._roles."""
    bars = {}

    def add(names, number, count):
        for name in names.split():
            for i in range(number):
                bars[name, i] = P._Barrier(count)

    add("LF LE", ns, 1)
    add("TF", TABLES, 1)
    add("TE", TABLES, 20 if out else 16)
    add("XD UD PD", 2, 1)
    add("OD", 1, 1)
    add("OE", 1, 4)
    add("barS barR barW barU", 2, 9)
    add("barEnd", 1, 20)

    def wait(name, phase, i=0):
        return "wait", (name, i), phase

    def arrive(name, i=0):
        return "arrive", (name, i), None

    def sync(name, i=0):
        return "sync", (name, i), None

    def issue(reads, writes, *barriers):
        return "issue", barriers, (reads, writes)

    def reads(*what):
        return "reads", what, None

    def writes(*what):
        return "writes", what, None

    def r(place, thing, c, last=1):  # of a read
        return place, 0, (thing, c), last

    def w(place, thing, c):
        return place, 0, (thing, c)

    def cells(name, h):  # of the chain's warps of one half: each has tensor-memory lanes and columns of its own
        return [(name, i) for i in range(8 * h, 8 * h + 8)]

    def both(name):
        return cells(name, 0) + cells(name, 1)

    def mma():
        for c in range(n):
            s = c % ns
            kq, tb = ("KQ", s), ("TB", s)
            xq = ("xq", 0 if alias else c & 1)
            yield wait("LF", c // ns, s)
            yield sync("barS", 0)
            yield issue([r(kq, "KQ", c, 0)] + [r(x, "S", c, not out) for x in cells("s", 0)], [])
            yield sync("barS", 1)
            yield issue([r(kq, "KQ", c, 0)] + [r(x, "S", c, not out) for x in cells("s", 1)],
                        [w(x, "X", c) for x in both("x")], ("XD", 0), ("XD", 1))
            if out and alias and c > 0:
                yield wait("OE", c - 1)
            if out:
                yield issue([r(kq, "KQ", c, 0)] + [r(x, "S", c) for x in both("s")], [w(xq, "xq", c)])
            yield sync("barR", 0)
            yield issue([r(tb, "TB", c, 0)] + [r(x, "R", c, 0) for x in cells("r", 0)], [w(x, "U", c) for x in cells("u", 0)],
                        ("UD", 0))
            yield sync("barR", 1)
            yield issue([r(tb, "TB", c, 0)] + [r(x, "R", c) for x in both("r")], [w(x, "U", c) for x in cells("u", 1)], ("UD", 1))
            yield sync("barW", 0)
            yield issue([r(kq, "KQ", c, 0)] + [r(x, "W", c) for x in cells("u", 0)], [w(x, "Pp", c) for x in both("s")])
            yield sync("barW", 1)
            yield issue([r(kq, "KQ", c)] + [r(x, "W", c) for x in cells("u", 1)] + [r(x, "Pp", c) for x in both("s")],
                        [w(x, "P", c) for x in both("s")], ("PD", 0), ("PD", 1))
            if out:
                yield sync("barU", 0)
                yield sync("barU", 1)
                if not alias and c > 0:
                    yield wait("OE", c - 1)
            yield issue([r(tb, "TB", c)] + [r(x, "Uo", c) for x in both("x") if out],
                        [w(x, "O", c) for x in (both("u") if alias else [("o", 0)]) if out], ("OD", 0), ("LE", s))
        if n:
            yield wait("OD", n - 1)
            yield wait("LE", (n - 1) // ns, (n - 1) % ns)

    def loads():
        for c in range(n):
            if c >= ns:
                yield wait("LE", c // ns - 1, c % ns)
            yield "load", ("LF", c % ns), [w((what, c % ns), what, c) for what in ("KQ", "V", "TB")]

    def table(first):
        for c in range(first, n, 2):
            if c >= TABLES:
                yield wait("TE", c // TABLES - 1, c % TABLES)
            yield writes(w(("table", c % TABLES), "table", c))
            yield arrive("TF", c % TABLES)

    def outputs(i):
        for c in range(n if out else 0):
            yield wait("TF", c // TABLES, c % TABLES)
            yield wait("OD", c)
            for _ in range(30):  # (they take their time)
                yield reads()
            yield reads(r(("xq", 0 if alias else c & 1), "xq", c),
                        *[r(x, "O", c) for x in (both("u") if alias else [("o", 0)])])
            yield arrive("OE")
            yield reads(r(("table", c % TABLES), "table", c))
            yield arrive("TE", c % TABLES)
        yield sync("barEnd")

    def chain(i):
        h = i // 8

        def fetch(c):
            yield wait("LF", c // ns, c % ns)
            yield wait("TF", c // TABLES, c % TABLES)
            yield reads(r(("V", c % ns), "V", c), r(("table", c % TABLES), "table", c, 0))

        if n:
            yield from fetch(0)
        for c in range(n):
            yield writes(w(("s", i), "S", c))
            yield arrive("barS", h)
            yield wait("XD", c, h)
            yield reads(r(("x", i), "X", c))
            yield writes(w(("r", i), "R", c))
            yield arrive("barR", h)
            yield reads(r(("table", c % TABLES), "table", c, 0))
            yield wait("UD", c, h)
            yield reads(r(("u", i), "U", c))
            yield writes(w(("u", i), "W", c))
            yield arrive("barW", h)
            if out:
                yield writes(w(("x", i), "Uo", c))
                yield arrive("barU", h)
            yield reads(r(("table", c % TABLES), "table", c))
            yield arrive("TE", c % TABLES)
            if c + 1 < n:
                yield from fetch(c + 1)
            yield wait("PD", c, h)
            yield reads(r(("s", i), "P", c))
        yield sync("barEnd")

    every = {"mma": mma(), "loads": loads(), "table 0": table(0), "table 1": table(1)}
    every.update({f"outputs {i}": outputs(i) for i in range(4)})
    every.update({f"chain {i}": chain(i) for i in range(16)})
    return bars, every


@pytest.fixture
def run(monkeypatch):
    monkeypatch.setattr(P, "_roles", roles)
    monkeypatch.setattr(P, "_Buffers", _Cells)
    monkeypatch.setattr(P, "READERS", READERS)
    return P._run


@pytest.mark.parametrize("stages,alias", [(3, False), (2, True)])
@pytest.mark.parametrize("out", [True, False])
@pytest.mark.parametrize("chunks", [0, 1, 2, 3, 4, 5, 9, 14])
def test_no_order_stalls_or_overtakes(run, stages, alias, chunks, out):
    for seed in range(12):
        run(stages, chunks, seed, alias=alias, out=out)


@pytest.mark.parametrize("name,role", [("LE", "loads"), ("TE", "table"), ("barS", "mma"), ("barR", "mma"), ("barW", "mma"),
                                       ("barU", "mma"), ("XD", "chain"), ("UD", "chain"), ("PD", "chain"), ("LF", "chain"),
                                       ("TF", "chain"), ("OD", "outputs"), ("OE", "mma")])
def test_a_wait_left_out_is_seen(run, name, role):
    def edit(bars, every):
        for r in [r for r in every if r.startswith(role)]:
            every[r] = (op for op in list(every[r]) if not (op[0] in ("wait", "sync") and op[1][0] == name))

    for alias in (False, True):
        with pytest.raises(AssertionError):
            for seed in range(40):
                run(3, 9, seed, edit, alias)
