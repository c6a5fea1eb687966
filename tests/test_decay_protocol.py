"""The order of the tensor-core walk of decayed linear attention (flare_decay_tc.cu), on the CPU.

Its roles hand tiles to one another through mbarriers.  The model below runs the same waits, arrivals and copies as the kernel's
roles, each at a speed of its own, and looks at two things that no run on a GPU can show to be excluded: that whoever reads a tile
reads what it is meant to (the chunk's own load, weighted, cleared), and that no wait tests the parity of a phase which is not the
barrier's last or next one (it would pass too early, or wait for a phase that has gone by).

A role is one process here; what a thread issues in order completes in order; two issuing warps are not ordered with one another.
"""
import heapq
import random

import pytest

KL = 128


class Fault(AssertionError):
    pass


class Barrier:
    def __init__(self, name, count):
        self.name, self.count, self.left, self.done = name, count, count, 0

    def arrive(self):
        self.left -= 1
        if self.left == 0:
            self.left = self.count
            self.done += 1

    def passes(self, phase):
        """What a wait for the parity of this phase returns now."""
        if (self.done & 1) == (phase & 1):
            if self.done > phase:
                raise Fault(f"{self.name}: phase {phase} went by unseen")
            return False
        if self.done != phase + 1:
            raise Fault(f"{self.name}: a wait for phase {phase} passed while {self.done} were over")
        return True


class Sim:
    def __init__(self, seed):
        self.rng, self.now, self.queue, self.n, self.waiting = random.Random(seed), 0.0, [], 0, {}

    def at(self, delay, fn):
        self.n += 1
        heapq.heappush(self.queue, (self.now + delay, self.n, fn))

    def some(self, slow=0.05):
        """A duration: mostly about one, now and then a long one."""
        return self.rng.expovariate(1.0) * (30.0 if self.rng.random() < slow else 1.0)

    def start(self, name, gen):
        def step():
            try:
                want = next(gen)
            except StopIteration:
                self.waiting.pop(name, None)
                return
            if want is None:
                self.at(self.some(), step)
                return
            bar, phase = want
            self.waiting[name] = f"{bar.name} phase {phase}"

            def poll():
                if bar.passes(phase):
                    self.at(self.some() * 0.1, step)
                else:
                    self.at(self.some(0.02) * 0.3, poll)

            self.at(self.some(0.02) * 0.1, poll)

        self.waiting[name] = "start"
        self.at(self.some(), step)

    def run(self, limit=200_000):
        while self.queue and self.waiting:
            self.now, _, fn = heapq.heappop(self.queue)
            fn()
            if self.n > limit:
                raise Fault(f"no end: {self.waiting}")


class Pipe:
    """What one thread issues: operations that complete in order, some time after their issue."""

    def __init__(self, sim):
        self.sim, self.free = sim, 0.0

    def issue(self, check, done=lambda: None):
        begins = max(self.sim.now, self.free) + self.sim.some() * 0.3
        ends = self.free = begins + self.sim.some() * 0.3

        def end():
            check()
            done()

        def begin():
            check()
            self.sim.at(max(0.0, ends - self.sim.now), end)

        self.sim.at(begins - self.sim.now, begin)

    def commit(self, bar):
        self.free += 1e-6
        self.sim.at(self.free - self.sim.now, bar.arrive)


class Cta:
    """One CTA of a walk.  chunks: those it takes; terms[c], cnt[c]: the terms and the live tokens of chunk c of the sequence."""

    def __init__(self, sim, wide, rank, size, terms, cnt, plus=False, wait_c=True, own_clear=True):
        self.sim, self.rank, self.size, self.terms, self.cnt, self.plus, self.wait_c, self.own_clear = \
            sim, rank, size, terms, cnt, plus, wait_c, own_clear
        self.wide, self.total = wide, len(terms)
        self.chunks = list(range(rank, self.total, size))
        self.kA, self.kB, self.kC = (2, 1, 2) if wide else (3, 3, 3)
        B = lambda name, count: Barrier(f"cta {rank} {name}", count)
        self.full = [B(f"bFull{i}", 1) for i in range(self.kA)]
        self.fullC = [B(f"bFullC{i}", 1) for i in range(self.kC)]
        self.free = [B(f"bFree{i}", 2) for i in range(self.kA)]
        self.freeB, self.clear, self.yx = B("bFreeB", 2), B("bClear", 1), B("bYx", 1)
        self.S, self.P, self.X = ([B(f"{n}{i}", 1) for i in range(2)] for n in ("bS", "bP", "bX"))
        self.W, self.Ev = ([B(f"{n}{i}", 1) for i in range(2)] for n in ("bW", "bEv"))
        self.kvFree, self.yFree, self.inn = B("bKvFree", 1), B("bYFree", 1), B("bIn", 1)
        self.a, self.b, self.c = [None] * self.kA, [None] * self.kB, [None] * self.kC
        self.w, self.s = [None] * 2, [None] * 2
        self.unit, self.pow = [None] * 4, [None] * 4       # fp16: powers of two of the weighted c and of P
        self.kv = self.y = self.yx_v = self.packed = self.state = None
        self.pend = {}
        self.out = []

    # -- what a reader must find ---------------------------------------------------------------------------------------
    def raw(self, i):
        return (i, "loaded")

    def ready(self, i):
        """A tile of b or c as products may read it: behind the length cleared."""
        return (i, "cleared") if self.cnt[self.chunks[i]] < KL else (i, "loaded")

    def see(self, what, got, want):
        if got != want:
            raise Fault(f"cta {self.rank} {what}: found {got}, not {want}")

    # -- loads -----------------------------------------------------------------------------------------------------------
    def load(self, tiles, at, i, done):
        tiles[at] = (i, "on its way")

        def land():
            tiles[at] = (i, "loaded")
            done()

        self.sim.at(self.sim.some(), land)

    def load_ab(self, tiles, at, i):
        bar = self.full[i % self.kA]

        def landed():
            self.pend[i] = self.pend.get(i, 0) + 1
            if self.pend[i] == 2:                  # both tiles' bytes: the phase ends
                bar.arrive()

        self.load(tiles, at, i, landed)

    def load_c(self, i):
        self.load(self.c, i % self.kC, i, self.fullC[i % self.kC].arrive)

    def roles(self):
        return {"load": self.r_load, "S PC": self.r_spc, "BC AX": self.r_bcax, "weigh": self.r_weigh, "P": self.r_p, "state": self.r_state,
                "out": self.r_out}

    def t(self, i):
        return self.terms[self.chunks[i]]

    def r_load(self):
        n = len(self.chunks)
        for i in range(n):
            if self.wide and i + 1 < n:
                yield self.freeB, i
                self.load_ab(self.b, 0, i + 1)
            if i + self.kA < n:
                yield self.free[i % self.kA], i // self.kA
                self.load_c(i + self.kA)
                if not self.wide:
                    self.load_ab(self.b, i % self.kB, i + self.kA)
                self.load_ab(self.a, i % self.kA, i + self.kA)
        yield None

    def first_loads(self):
        for i in range(min(len(self.chunks), 3)):
            if i < self.kC:
                self.load_c(i)
            if i < self.kB:
                self.load_ab(self.b, i, i)
            if i < self.kA:
                self.load_ab(self.a, i, i)

    # -- products --------------------------------------------------------------------------------------------------------
    def r_spc(self):
        pipe, n = Pipe(self.sim), len(self.chunks)
        ahead, ev = 0 if self.wide else 1, 0
        for j in range(n + ahead):
            if j < n:
                yield self.full[j % self.kA], j // self.kA
                if self.cnt[self.chunks[j]] < KL:
                    yield (self.clear, 0) if self.own_clear else (self.W[ev & 1], ev >> 1)
                ev += 2 if self.t(j) == 3 else 1

                def read(j=j):
                    self.see("S reads a", self.a[j % self.kA], self.raw(j))
                    self.see("S reads b", self.b[j % self.kB], self.ready(j))

                def wrote(j=j):
                    self.s[j & 1] = ("S", j)

                pipe.issue(read, wrote)
                pipe.commit(self.S[j & 1])
                if self.wide:
                    pipe.commit(self.freeB)
            i = j - ahead
            if i < 0:
                continue
            if self.wait_c:
                yield self.fullC[i % self.kC], i // self.kC
            yield self.P[i & 1], i >> 1
            if i > 0:
                yield self.yFree, i - 1

            def read_p(i=i):
                self.see("P C reads P", self.s[i & 1], ("P", i))
                self.see("P C reads c", self.c[i % self.kC], self.ready(i))

            def wrote_y(i=i):
                self.y = i

            pipe.issue(read_p, wrote_y)
            pipe.commit(self.free[i % self.kA])

    def r_bcax(self):
        pipe, n = Pipe(self.sim), len(self.chunks)
        ev = i = j = 0
        while i < n:
            if j < n and (j == i or (j == i + 1 and (not self.wide or (self.W[ev & 1].done & 1) != ((ev >> 1) & 1)))):
                yield self.full[j % self.kA], j // self.kA
                yield self.W[ev & 1], ev >> 1
                if j > 0:
                    yield self.kvFree, j - 1
                t = self.t(j)
                last = 1 if t == 3 or (self.plus and t == 2) else 0
                for k in range(last + 1):
                    own_c = k > 0 and self.plus and t == 2

                    def read(j=j, ev=ev, t=t, k=k, own_c=own_c):
                        self.see("B^T C reads b", self.b[j % self.kB], self.ready(j))
                        if own_c:
                            self.see("B^T C reads c", self.c[j % self.kC], self.ready(j))
                            return
                        tiles = (ev & 1,) if t == 1 else (0,) if k else (0, 1)
                        for x in tiles:
                            self.see("B^T C reads its terms", self.w[x], ev)

                    def wrote(j=j, k=k, last=last):
                        if k == last:
                            self.kv = j

                    pipe.issue(read, wrote)
                    if t == 3 or k == last:
                        pipe.commit(self.Ev[ev & 1])
                    if k < last and t == 3:
                        ev += 1
                        yield self.W[ev & 1], ev >> 1
                if self.wide:
                    pipe.commit(self.freeB)
                ev += 1
                j += 1
                continue
            yield self.X[i & 1], i >> 1
            if i > 0:
                yield self.yFree, i - 1

            def read_x(i=i):
                self.see("A X reads a", self.a[i % self.kA], self.raw(i))
                self.see("A X reads X", self.packed, i)

            def wrote_yx(i=i):
                self.yx_v = i

            pipe.issue(read_x, wrote_yx)
            pipe.commit(self.yx)
            pipe.commit(self.free[i % self.kA])
            i += 1

    # -- the roles of threads --------------------------------------------------------------------------------------------
    def r_weigh(self):
        ev, before = 0, 1
        for i in range(len(self.chunks)):
            short = self.cnt[self.chunks[i]] < KL
            t = self.t(i)
            yield self.fullC[i % self.kC], i // self.kC
            if short:
                yield self.full[i % self.kA], i // self.kA
            for part in range(2 if t == 3 else 1):
                back = 1 if t > 1 or before > 1 else 2
                if ev >= back:
                    yield self.Ev[(ev - back) & 1], (ev - back) >> 1
                self.see("weights read c", self.c[i % self.kC], self.ready(i) if part else self.raw(i))
                yield None
                if short and part == 0:
                    self.see("clearing b", self.b[i % self.kB], self.raw(i))
                    self.b[i % self.kB] = self.c[i % self.kC] = (i, "cleared")
                for x in ((ev & 1,) if t == 1 else (0,) if part else (0, 1)):
                    self.w[x] = ev
                self.unit[i & 3] = i
                if short and part == 0:
                    self.clear.arrive()
                self.W[ev & 1].arrive()
                before = t
                ev += 1

    def r_p(self):
        for i in range(len(self.chunks)):
            yield self.S[i & 1], i >> 1
            self.see("weights read S", self.s[i & 1], ("S", i))
            yield None
            self.see("weights read S", self.s[i & 1], ("S", i))
            self.s[i & 1], self.pow[i & 3] = ("P", i), i
            self.P[i & 1].arrive()

    def r_state(self):
        ev = 0
        for i, c in enumerate(self.chunks):
            if self.t(i) == 3:
                ev += 1
            yield self.Ev[ev & 1], ev >> 1
            self.see("the state reads B^T C", self.kv, i)
            self.see("the state reads its unit", self.unit[i & 3], i)
            yield None
            self.see("the state reads B^T C", self.kv, i)
            if not self.wide:
                self.kvFree.arrive()
            if self.wide and i > 0:
                yield self.yx, i - 1
            if self.size > 1 and c > 0:
                yield self.inn, i - 1 if self.rank == 0 else i
            if c > 0:
                self.see("the state arrives", self.state, c - 1)
            self.state = c
            yield None
            if self.size > 1 and c + 1 < self.total:
                to = self.peers[(self.rank + 1) % self.size]

                def land(c=c, to=to):
                    self.see("the state leaves", self.state, c)
                    to.state = c
                    to.inn.arrive()

                self.sim.at(self.sim.some(), land)
            if self.wide:
                self.kvFree.arrive()
            elif i > 0:
                yield self.yx, i - 1
            self.packed = i
            yield None
            self.X[i & 1].arrive()
            ev += 1

    def r_out(self):
        for i in range(len(self.chunks)):
            yield self.free[i % self.kA], i // self.kA
            self.see("outputs read P C", self.y, i)
            self.see("outputs read A X", self.yx_v, i)
            self.see("outputs read P's power", self.pow[i & 3], i)
            yield None
            self.see("outputs read P C", self.y, i)
            self.see("outputs read A X", self.yx_v, i)
            self.yFree.arrive()
            self.out.append(i)


def walk(seed, wide, size, terms, last=KL, rev=False, **kw):
    """A walk of len(terms) chunks, the sequence's last one `last` tokens long; raises Fault where the order is not kept."""
    sim = Sim(seed)
    cnt = [KL] * len(terms)
    cnt[0 if rev else -1] = last
    ctas = [Cta(sim, wide, r, size, terms, cnt, **kw) for r in range(size)]
    for cta in ctas:
        cta.peers = ctas
        cta.first_loads()
        for name, role in cta.roles().items():
            sim.start(f"{name} of {cta.rank}", role())
    sim.run()
    if sim.waiting:
        raise Fault(f"stuck: {sim.waiting}")
    for cta in ctas:
        assert cta.out == list(range(len(cta.chunks)))


TERMS = [[1] * 7, [1, 1, 2, 2, 3, 3, 3, 3], [3] * 6, [2] * 6, [1, 2, 3], [1], [3], [1, 3, 3], [1, 1, 3], [2, 3, 3, 3]]
SEEDS = range(20)


@pytest.mark.parametrize("size", [1, 2, 3, 4])
@pytest.mark.parametrize("wide", [False, True], ids=["64", "128"])
@pytest.mark.parametrize("terms", TERMS, ids=str)
def test_whole_chunks(terms, wide, size):
    for seed in SEEDS:
        walk(seed, wide, size, terms)
        walk(seed, wide, size, [min(t, 2) for t in terms], plus=True)


@pytest.mark.parametrize("size", [1, 2, 3, 4])
@pytest.mark.parametrize("wide", [False, True], ids=["64", "128"])
@pytest.mark.parametrize("terms", TERMS, ids=str)
def test_a_chunk_that_ends_early(terms, wide, size):
    """The sequence's last chunk, or its mirror image's first; the mirror image returns no state, so its chunks take one term."""
    for seed in SEEDS:
        walk(seed, wide, size, terms, last=50)
        walk(seed, wide, size, [min(t, 2) for t in terms], last=1, plus=True)
        walk(seed, wide, size, [1] * len(terms), last=72, rev=True)


@pytest.mark.parametrize("terms,rev,how", [([1] * 7, True, "went by unseen"), ([3, 3], False, "a wait for phase 1 passed while 0")])
def test_the_model_notices_phases_that_are_not_followed(terms, rev, how):
    with pytest.raises(Fault, match=how):
        for seed in range(4000):
            walk(seed, False, 1, terms, last=72, rev=rev, own_clear=False)


@pytest.mark.parametrize("wide", [False, True], ids=["64", "128"])
def test_the_model_notices_products_that_do_not_wait_for_c(wide):
    with pytest.raises(Fault, match="P C reads c"):
        for seed in range(400):
            walk(seed, wide, 1, [1] * 7, wait_c=False)
