"""The hand-overs between the warp roles of the tensor-core linear-attention scan (csrc/gdn_linear_attn_tc.cu), replayed on
the CPU under random schedules: a model of the roles' waits, arrivals, loads and products with mbarriers that count phases.

Checked in every run: a wait by parity succeeds only for its own phase; no barrier gets an arrival that it does not expect;
no buffer is written while a product or a load may use it; a product, and whatever is stored, finds the operands it was
meant to; every role ends; nothing is in flight when the block gives its memory back. The runs with failures let roles give
up (their bounded wait runs out) at random places, or lose a load or a product's completion for good."""
import random
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "sorernn_b200" / "csrc"
ARRIVALS = dict(FULL_A=1, FULL_B=1, FULL_C0=1, FULL_C1=1, QK=1, U=1, AX=1, AH=1, O=1, HL=4, XR=4, X2=4, UR=4, P0=8, P1=8,
                E=8, D16=1, D18=1, D19=1)
STATES_ONLY = dict(U_ODD=1, HL=8, HL_ODD=8, UR=8, UR_ODD=8)


class Barrier:
    def __init__(self, name, count):
        self.name, self.count, self.pending, self.tx, self.phase = name, count, count, 0, 0

    def _turn(self):
        if self.pending == 0 and self.tx == 0:
            self.phase, self.pending = self.phase + 1, self.count

    def arrive(self, tx=0):
        assert self.pending > 0, f"unexpected arrival at {self.name}"
        self.pending, self.tx = self.pending - 1, self.tx + tx
        self._turn()

    def land(self):
        self.tx -= 1
        self._turn()

    def passed(self, k):  # what the hardware sees: the parity of the phase it is in
        seen = (self.phase & 1) != (k & 1)
        assert seen == (self.phase > k) or not seen, f"{self.name}: wait for phase {k} passes in phase {self.phase}"
        return seen


class Block:
    """One CTA. outputs: the form with outputs, else states only; turns: the halves of X take turns."""

    def __init__(self, seed, nch, wants_state, has_x, outputs, turns, give_up=0.0, lose=0.0, run_on=False, no_drain=False):
        self.rnd = random.Random(seed)
        self.nch, self.has_x, self.outputs, self.turns = nch, has_x, outputs, turns
        self.n_u = nch if wants_state or not outputs else nch - 1
        self.give_up, self.lose, self.run_on, self.no_drain = give_up, lose, run_on, no_drain
        self.bars = {n: Barrier(n, c) for n, c in {**ARRIVALS, **({} if outputs else STATES_ONLY)}.items()}
        self.holds, self.readers = {}, {}       # buffer: what it holds, the products that read it
        self.loads, self.products = [], {16: [], 18: [], 19: []}
        self.dead, self.failed, self.met, self.round = set(), False, 0, 0
        self.stored = []

    # ---- operations --------------------------------------------------------------------------------------------
    def arrive(self, who, bar):
        if who not in self.dead or self.run_on:
            self.bars[bar].arrive()

    def write(self, buf, what):
        assert not self.readers.get(buf), f"{buf} written while {self.readers[buf]} read it"
        assert self.holds.get(buf) not in ("load", "product"), f"{buf} written under a {self.holds[buf]}"
        self.holds[buf] = what

    def read(self, buf, what):
        assert self.holds.get(buf) == what, f"{buf} holds {self.holds.get(buf)}, {what} expected"

    def load(self, buf, bar, what):
        assert not self.readers.get(buf), f"load over {buf}"
        self.holds[buf] = "load"
        self.bars[bar].arrive(1)
        if self.rnd.random() >= self.lose:
            self.loads.append((buf, bar, what))

    def product(self, warp, operands, dst, what):
        for buf, content in operands:
            self.read(buf, content)
            self.readers.setdefault(buf, []).append((warp, what))
        self.holds[dst] = "product"
        self.products[warp].append(("product", operands, dst, what))

    def commit(self, warp, bar):
        lost = self.rnd.random() < self.lose and not bar.startswith("D")
        self.products[warp].append(("commit", None if lost else bar))

    def advance_load(self):
        buf, bar, what = self.loads.pop(self.rnd.randrange(len(self.loads)))
        self.holds[buf] = what
        self.bars[bar].land()

    def advance_product(self, warp):
        kind, *rest = self.products[warp].pop(0)
        if kind == "commit":
            if rest[0]:
                self.bars[rest[0]].arrive()
            return
        operands, dst, what = rest
        for buf, content in operands:
            self.read(buf, content)
            self.readers[buf].remove((warp, what))
        self.holds[dst] = what

    # ---- names and phases of chunk c -----------------------------------------------------------------------------
    def odd(self, c):
        return "_ODD" if not self.outputs and c % 2 else ""

    def turn(self, c):
        return c if self.outputs else c // 2

    def u(self, c):
        return "U" + self.odd(c), self.turn(c)

    def ur(self, c):
        return "UR" + self.odd(c), self.turn(c)

    def full_c(self, c):
        return ("FULL_C0", c) if self.outputs else (f"FULL_C{c % 2}", c // 2)

    def c_buf(self, c):
        return "C0" if self.outputs else f"C{c % 2}"

    # ---- roles: each yields the (barrier, phase) it waits for, or None to let others run ----------------------------
    def loader(self):
        me, loaded = "load", dict(FULL_A=0, FULL_B=0, FULL_C0=0, FULL_C1=0)
        out = lambda: me in self.dead and not self.run_on  # noqa: E731

        def load(buf, bar, c):
            self.load(buf, bar, c)
            loaded[bar] += 1

        for c in range(self.nch):
            if self.outputs:
                if c:
                    yield "QK", c - 1
                if out():
                    break
                load("B", "FULL_B", c)
                if c:
                    yield "AX", c - 1
                if out():
                    break
                load("A", "FULL_A", c)
                if c:
                    yield self.u(c - 1)
                    yield "O", c - 1
            elif c > 1:
                yield self.u(c - 2)
            if out():
                break
            load(self.c_buf(c), self.full_c(c)[0], c)
            yield None
        if not self.no_drain:
            for bar, n in loaded.items():
                if n:
                    yield bar, n - 1, "fresh"

    def drain(self, warp):
        if not self.no_drain:
            self.commit(warp, f"D{warp}")
            yield f"D{warp}", 0, "fresh"

    def issue_p(self):
        me = 16
        out = lambda: me in self.dead and not self.run_on  # noqa: E731
        for c in range(self.nch):
            yield "FULL_A", c
            yield "FULL_B", c
            if c:
                yield "O", c - 1
            if out():
                break
            self.product(16, [("A", c), ("B", c)], "P", ("P", c))
            self.commit(16, "QK")
            yield self.full_c(c)
            if c:
                yield "E", c - 1
            for half in (0, 1):
                yield f"P{half}", c
                if out():
                    break
                self.product(16, [(f"W{half}{q}", c) for q in range(4)] + [("C0", c)], "OA", ("OA", c, half))
            if out():
                break
            self.commit(16, "O")
        yield from self.drain(16)

    def issue_u(self):
        me, ahead = 18, 1 if self.outputs else 2
        for c in range(self.nch):
            yield self.full_c(c)
            yield "HL" + self.odd(c), self.turn(c)
            if c >= ahead:
                yield self.ur(c - ahead)
            if me in self.dead and not self.run_on:
                break
            if c < self.n_u:
                rows = [(f"HL{self.odd(c)}{w}", c) for w in range(4 if self.outputs else 8)]
                self.product(18, rows + [(self.c_buf(c), c)], "TU" + self.odd(c), ("U", c))
            self.commit(18, self.u(c)[0])
        yield from self.drain(18)

    def issue_x(self):
        me = 19
        out = lambda: me in self.dead and not self.run_on  # noqa: E731
        for c in range(self.nch):
            yield "FULL_A", c
            yield "XR", c
            if c:
                yield "E", c - 1
            for half in (0, 1):
                if self.turns and half:
                    self.commit(19, "AH")
                    yield "X2", c
                if out():
                    break
                if c or self.has_x:
                    rows = [(f"X{0 if self.turns else half}{w}", (c, half)) for w in range(4)]
                    self.product(19, [("A", c)] + rows, "OI", ("OI", c, half))
            if out():
                break
            self.commit(19, "AX")
        yield from self.drain(19)

    def state(self, w):
        me = f"state{w}"
        out = lambda: me in self.dead and not self.run_on  # noqa: E731

        def rest():
            for c in range(-1, self.n_u):
                if c >= 0:
                    yield self.u(c)
                    if out():
                        return
                    self.read("TU" + self.odd(c), ("U", c))
                    yield None
                    self.read("TU" + self.odd(c), ("U", c))
                    self.arrive(me, self.ur(c)[0])
                if not self.outputs or c + 1 >= self.nch:
                    continue
                if c >= 0:
                    yield "AX", c
                if out():
                    return
                self.write(f"X0{w}", (c + 1, 0))
                if self.turns:
                    self.arrive(me, "XR")
                    yield "AH", c + 1
                    if out():
                        continue
                    self.write(f"X0{w}", (c + 1, 1))
                    self.arrive(me, "X2")
                else:
                    self.write(f"X1{w}", (c + 1, 1))
                    self.arrive(me, "XR")

        yield from rest()
        if not out():
            self.stored.append((me, self.n_u))  # every product it took was the right one: read() checked them

    def split(self, w):
        me, ahead = f"split{w}", 1 if self.outputs else 2
        for c in range(self.nch):
            if c >= ahead:
                yield self.u(c - ahead)
            if not self.outputs or c == self.nch - 1:  # the last chunk's rows past the end
                yield self.full_c(c)
            if me not in self.dead or self.run_on:
                self.write(f"HL{self.odd(c)}{w}", c)
                yield None
            self.arrive(me, "HL" + self.odd(c))

    def output(self, w):
        me = f"out{w}"
        good = lambda: me not in self.dead  # noqa: E731
        for c in range(self.nch):
            yield "QK", c
            if c == self.nch - 1:
                yield self.full_c(c)
            if good():
                self.read("P", ("P", c))
            for half in (0, 1):
                yield None
                if w < 4:
                    self.holds[f"W{half}{w}"] = c if good() else "garbage"
                self.arrive(me, f"P{half}")
            if c:
                yield "meet"
            inter = c > 0 or self.has_x
            if inter:
                yield "AX", c
            yield "O", c
            if good():
                for _ in range(2):
                    if inter:
                        self.read("OI", ("OI", c, 1))
                    self.read("OA", ("OA", c, 1))
                    yield None
            else:
                self.failed = True
            self.arrive(me, "E")
            yield "meet"
            if w == 0 and not self.failed:
                assert good()
                self.stored.append(("tile", c))

    def run(self):
        roles = {"load": self.loader(), 18: self.issue_u()}
        if self.outputs:
            roles.update({16: self.issue_p(), 19: self.issue_x()})
            roles.update({f"state{w}": self.state(w) for w in range(4)})
            roles.update({f"split{w}": self.split(w) for w in range(4)})
            roles.update({f"out{w}": self.output(w) for w in range(8)})
        else:
            roles.update({f"state{w}": self.state(w) for w in range(8)})
            roles.update({f"split{w}": self.split(w) for w in range(8)})
        waits = {n: None for n in roles}
        speed = {n: self.rnd.random() ** 3 + 1e-3 for n in list(roles) + ["land", 16, 18, 19]}

        def ready(n):
            w = waits[n]
            if w is None:
                return True
            if w == "meet" or w[0] == "meet":
                return w[0] == "meet" and self.round > w[1]
            if n in self.dead and len(w) == 2:  # it looks once
                return True
            return self.bars[w[0]].passed(w[1])

        while roles:
            blocked = [n for n in roles if waits[n] is not None and waits[n][0] != "meet" and n not in self.dead]
            acts = [("role", n) for n in roles if ready(n)] + [("product", w) for w in self.products if self.products[w]]
            acts += [("land", "land")] if self.loads else []
            if not acts or self.rnd.random() < self.give_up:
                if not acts:
                    assert self.give_up or self.lose, f"no role can go on: {waits}"
                    stuck = [n for n in roles if waits[n] is not None and waits[n][0] != "meet"]
                    assert stuck, f"no role can go on: {waits}"
                    n = self.rnd.choice(stuck)
                    if len(waits[n]) == 3:  # a drain's own wait runs out
                        waits[n] = None
                    else:
                        self.dead.add(n)
                    continue
                if blocked:
                    n = self.rnd.choice(blocked)
                    if len(waits[n]) == 2 and not self.bars[waits[n][0]].passed(waits[n][1]):
                        self.dead.add(n)
                continue
            kind, n = self.rnd.choices(acts, [speed[a[1]] for a in acts])[0]
            if kind == "land":
                self.advance_load()
            elif kind == "product":
                self.advance_product(n)
            else:
                try:
                    waits[n] = next(roles[n])
                except StopIteration:
                    del roles[n]
                    continue
                if waits[n] == "meet":
                    waits[n] = ("meet", self.round)
                    self.met += 1
                    if self.met == 8:
                        self.met, self.round = 0, self.round + 1
        assert not self.loads and not any(self.products.values()), "in flight at the end"
        return self


def blocks(seed, **kw):
    r = random.Random(seed)
    return Block(seed, nch=r.randint(0, 6), wants_state=r.random() < 0.5, has_x=r.random() < 0.5, outputs=r.random() < 0.7,
                 turns=r.random() < 0.5, **kw)


def test_barriers_are_the_kernels():
    text = (CSRC / "gdn_linear_attn_tc.cu").read_text()
    names = re.search(r"enum Bar \{([^}]*)\}", text).group(1).replace(" ", "").split(",")
    assert names == list(ARRIVALS) + ["NBAR"]
    assert re.search(r"enum Bar2 \{ U_ODD = AX, HL_ODD = XR, UR_ODD = P0 \}", text)
    init = re.search(r"mbar_init\(&bar\[i\], (.*)\);", text).group(1)
    assert init == "i >= D16 ? 1 : i >= P0 || (!OUT && i >= HL) ? 8 : i >= HL ? 4 : 1"
    at = {n: i for i, n in enumerate(ARRIVALS)}
    for n, i in at.items():
        assert ARRIVALS[n] == (1 if i >= at["D16"] else 8 if i >= at["P0"] else 4 if i >= at["HL"] else 1)


def test_every_schedule_ends_with_all_outputs():
    for seed in range(400):
        b = blocks(seed).run()
        if b.outputs:
            assert [c for n, c in b.stored if n == "tile"] == list(range(b.nch))
        assert len([n for n, _ in b.stored if n != "tile"]) == (4 if b.outputs else 8)


@pytest.mark.parametrize("kw", [dict(give_up=0.6), dict(give_up=0.02), dict(give_up=0.002), dict(lose=0.05),
                                dict(give_up=0.005, lose=0.02)])
def test_roles_that_give_up(kw):
    gave_up = 0
    for seed in range(400):
        b = blocks(seed, **kw).run()
        gave_up += bool(b.dead)
        tiles = [c for n, c in b.stored if n == "tile"]
        assert tiles == list(range(len(tiles)))
    assert gave_up > 50


@pytest.mark.parametrize("rule,give_up", [("run_on", 0.01), ("no_drain", 0.6)])
def test_the_checks_find_a_broken_rule(rule, give_up):
    """Roles that hand over after giving up, or that leave without their loads and products: some schedule shows it."""
    found = 0
    for seed in range(200):
        try:
            blocks(seed, give_up=give_up, **{rule: True}).run()
        except AssertionError:
            found += 1
    assert found
