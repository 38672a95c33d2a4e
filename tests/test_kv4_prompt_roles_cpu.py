"""CPU: the roles and barriers of k_kv4_prompt (csrc/fn_kv4_prompt.cu) as coroutines under random schedules: every wait ends, and every
shared place holds the tile that its reader expects, when it starts to read it and when it is done.

NB: operand buffers (1: fp32 rows of 256 dims), FAR: the long form of the kernel, in which some tiles' P V is added by the workers."""

import random

import pytest


class Barrier:
    def __init__(self, count):
        self.count = self.left = count
        self.phase = 0

    def arrive(self, k=1):
        assert self.left >= k
        self.left -= k
        if self.left == 0:
            self.phase, self.left = self.phase + 1, self.count

    def done(self, phase):  # what a wait by parity can tell
        return (self.phase & 1) != (phase & 1)


class Cta:
    def __init__(self, seed, nb, long_form, tiles, share, first=2):
        """tiles: of each row tile; share of tiles that the workers add; first: the tile of a row tile from which S waits for the tile two
        before it to be added."""
        self.rng, self.nb, self.long_form, self.tiles, self.first = random.Random(seed), nb, long_form, tiles, first
        self.far = [long_form and self.rng.random() < share for _ in range(sum(tiles))]
        self.rk, self.rv = 2, nb
        n = lambda count, places=2: [Barrier(count) for _ in range(places)]  # noqa: E731
        self.rkf, self.rke, self.rvf, self.rve = n(1), n(5 if long_form else 4), n(1), n(8)
        self.kf, self.ke, self.vf, self.sf, self.pf, self.xf = n(4), n(1), n(4), n(1), n(4), n(1, 8)
        self.of, self.oe, self.qf, self.qe, self.lf = Barrier(1), Barrier(8), Barrier(8), Barrier(1), Barrier(4)
        # which tile a place holds; four warps each where four fill it
        self.raw_k, self.raw_v, self.s = [None] * 2, [None] * 2, [None] * 2
        self.k, self.v, self.p = ([[None] * 4 for _ in range(2)] for _ in range(3))
        self.valid, self.scales, self.f, self.o = [None] * 8, [None] * 8, [[None] * 4 for _ in range(4)], None
        self.issued, self.at_barrier, self.barrier_gen = [], 0, 0

    def wait(self, bar, phase):
        while not bar.done(phase):
            yield

    def known(self, g):
        return self.valid[g & 7] == g and (not self.long_form or self.scales[g & 7] == g)

    def copies(self):
        for g in range(sum(self.tiles)):
            for raw, full, empty, r in ((self.raw_k, self.rkf, self.rke, self.rk), (self.raw_v, self.rvf, self.rve, self.rv)):
                if g >= r:
                    yield from self.wait(empty[g % r], g // r - 1)
                if raw is self.raw_k:
                    self.valid[g & 7] = g
                raw[g % r] = g
                yield
                full[g % r].arrive()

    def looks(self):
        for g in range(sum(self.tiles)):
            yield from self.wait(self.rkf[g % self.rk], g // self.rk)
            assert self.raw_k[g % self.rk] == g and self.valid[g & 7] == g
            self.scales[g & 7] = g
            yield
            self.xf[g & 7].arrive()
            self.rke[g % self.rk].arrive()

    def products(self):
        g0 = 0
        for i, n in enumerate(self.tiles):
            yield from self.wait(self.qf, i)
            for j in range(n + 1):
                g = g0 + j
                if j < n:
                    yield from self.wait(self.kf[g % self.nb], g // self.nb)
                    if g >= 2 and j >= self.first and self.far[g - 2]:
                        yield from self.wait(self.oe, g - 2)
                    self.issued += [("S", g), self.sf[g & 1], self.ke[g % self.nb]] + [self.qe] * (j == n - 1)
                    yield
                if j > 0:
                    g -= 1
                    yield from self.wait(self.pf[g & 1], g >> 1)
                    yield from self.wait(self.vf[g % self.nb], g // self.nb)
                    if g > 0:
                        yield from self.wait(self.oe, g - 1)
                    self.issued += [("O", g)] * (not self.far[g]) + [self.of]
                    yield
            g0 += n

    def tensor_core(self):  # what was issued, in order, some time later
        if not self.issued:
            return
        x = self.issued.pop(0)
        if isinstance(x, Barrier):
            x.arrive()
        elif x[0] == "S":
            assert self.k[x[1] % self.nb] == [x[1]] * 4
            self.s[x[1] & 1], self.p[x[1] & 1] = x[1], [None] * 4
        else:
            assert self.p[x[1] & 1] == [x[1]] * 4 and self.v[x[1] % self.nb] == [x[1]] * 4
            self.o = x[1]

    def softmax(self, me):
        g = 0
        for n in self.tiles:
            for _ in range(n):
                yield from self.wait(self.sf[g & 1], g >> 1)
                assert self.s[g & 1] == g and self.known(g)
                yield
                self.f[g & 3][me] = self.p[g & 1][me] = g
                yield
                assert self.s[g & 1] == g
                self.pf[g & 1].arrive()
                g += 1
            self.lf.arrive()

    def workers_barrier(self):
        self.at_barrier, gen = self.at_barrier + 1, self.barrier_gen
        if self.at_barrier == 8:
            self.at_barrier, self.barrier_gen = 0, gen + 1
        while self.barrier_gen == gen:
            yield

    def make(self, g, me, raw, r, full, operand, filled):
        yield from self.wait(full[g % r], g // r)
        if self.long_form:
            yield from self.wait(self.xf[g & 7], g >> 3)
        if operand is self.k and g >= self.nb:
            yield from self.wait(self.ke[g % self.nb], g // self.nb - 1)
        assert raw[g % r] == g and self.known(g)
        yield
        if operand is self.k or not self.far[g]:
            operand[g % self.nb][me] = g
        assert raw[g % r] == g
        filled[g % self.nb].arrive()
        if operand is self.k:
            self.rke[g % r].arrive()
        elif not self.far[g]:
            self.rve[g % r].arrive(2)

    def worker(self, x):
        half, me, g0 = x >> 2, x & 3, 0
        for i, n in enumerate(self.tiles):
            if i > 0:
                yield from self.wait(self.qe, i - 1)
            for _ in range(3):
                yield from self.workers_barrier()
            self.qf.arrive()
            for j in range(-1, n + 1):
                g, adds, last = g0 + j, j > 0, g0 + j - 1
                far = adds and self.far[last]
                if far:
                    yield from self.wait(self.rvf[last % self.rv], last // self.rv)
                    yield from self.wait(self.pf[last & 1], last >> 1)
                    for _ in range(2):
                        assert self.raw_v[last % self.rv] == last and self.p[last & 1][me] == last and self.s[last & 1] == last
                        assert self.f[last & 3][me] == last and self.known(last)
                        yield
                    self.rve[last % self.rv].arrive()
                v = self.make(g, me, self.raw_v, self.rv, self.rvf, self.v, self.vf)
                if half == 0 and j + 1 < n:
                    yield from self.make(g + 1, me, self.raw_k, self.rk, self.rkf, self.k, self.kf)
                if half == 1 and 0 <= j < n and self.nb == 2:
                    yield from v
                if adds:
                    yield from self.wait(self.of, last)
                if half == 1 and 0 <= j < n and self.nb == 1:
                    yield from v
                if adds:
                    for _ in range(2):
                        assert self.f[last & 3][me] == last and (far or self.o == last) and self.known(last)
                        yield
                    self.oe.arrive()
            g0 += n
            yield from self.wait(self.lf, i)

    def run(self, limit=200_000):
        roles = [self.copies(), self.products()] + [self.looks()] * self.long_form
        roles += [self.softmax(x) for x in range(4)] + [self.worker(x) for x in range(8)]
        slow = {id(r): self.rng.choice([1, 1, 1, 5, 30]) for r in roles}
        for _ in range(limit):
            if not roles:
                return True
            if self.rng.random() < 0.3:
                self.tensor_core()
            r = self.rng.choice(roles)
            if self.rng.random() * slow[id(r)] < 1:
                try:
                    next(r)
                except StopIteration:
                    roles.remove(r)
        return False


@pytest.mark.parametrize("nb", [1, 2])
@pytest.mark.parametrize("long_form, share", [(False, 0.0), (True, 0.1), (True, 0.6), (True, 1.0)])
def test_every_wait_ends_and_every_place_is_read_in_time(nb, long_form, share):
    for seed in range(25):
        rng = random.Random(seed)
        tiles = [rng.randint(1, 6) for _ in range(rng.randint(1, 6))]
        assert Cta(seed, nb, long_form, tiles, share).run(), (seed, tiles)


def test_waiting_for_a_tile_of_the_row_tile_before_would_not_end():
    """Its phase is two ago by then, and a wait by parity takes it for the one to come."""
    assert not Cta(1, 1, True, [4, 4], 1.0, first=0).run()
