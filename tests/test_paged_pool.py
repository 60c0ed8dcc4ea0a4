"""The page pool's bookkeeping (host only): against a plain model of it over
random runs of its calls, and its refusals."""
import random

import numpy as np
import pytest

from autoresearch_amd import engine


def code_of(f, *a):
    with pytest.raises(engine.FgptError) as e:
        f(*a)
    return e.value.code


class Model:
    """Sequences as lists of (token, page, slot): what a pool has to keep true."""

    def __init__(self, pool):
        self.p = pool
        self.rows = {s: [] for s in range(pool.max_seq)}  # a row's content, by position
        self.mem = {}                                      # (page, slot) -> content
        self.n = 0

    def extend(self, s, n):
        before = self.p.free, self.p.need(s, n)
        c = self.p.extend(s, n)
        assert self.p.free == before[0] - before[1]
        if c is not None:
            for slot in range(self.p.page_size):
                if (c[0], slot) in self.mem:
                    self.mem[c[1], slot] = self.mem[c[0], slot]
        t = self.p.table(s)
        for _ in range(n):
            pos = len(self.rows[s])
            self.n += 1
            self.rows[s].append(self.n)
            self.mem[int(t[pos // self.p.page_size]), pos % self.p.page_size] = self.n

    def check(self):
        held = set()
        for s, rows in self.rows.items():
            assert self.p.len(s) == len(rows)
            t = self.p.table(s)
            assert len(t) == -(-len(rows) // self.p.page_size)
            for pos, want in enumerate(rows):
                pg = int(t[pos // self.p.page_size])
                if pg >= 0:
                    assert self.mem[pg, pos % self.p.page_size] == want, (s, pos)
            held |= {int(x) for x in t if x >= 0}
        assert self.p.free == self.p.n_pages - len(held)
        return held


@pytest.mark.parametrize("seed", range(12))
def test_random_runs(seed):
    r = random.Random(seed)
    P = r.choice([16, 32])
    p = engine.Pool(r.choice([5, 40, 300]), P, 6)
    m = Model(p)
    for _ in range(300):
        s = r.randrange(6)
        do = r.choice(["extend", "extend", "extend", "fork", "trim", "compact", "end"])
        if do == "extend":
            n = r.choice([0, 1, 1, 2, P - 1, P, 3 * P + 1])
            if p.need(s, n) <= p.free:
                m.extend(s, n)
            else:
                assert code_of(p.extend, s, n) == -5
        elif do == "fork":
            d = r.randrange(6)
            n = r.randint(0, p.len(s))
            if d == s or p.len(d):
                assert code_of(p.fork, s, d, n) == -1
            else:
                p.fork(s, d, n)
                m.rows[d] = m.rows[s][:n]
        elif do == "trim":
            n = r.randint(0, p.len(s))
            p.trim(s, n)
            m.rows[s] = m.rows[s][:n]
        elif do == "end":
            p.trim(s)
            m.rows[s] = []
        else:
            src, dst = p.compact()
            assert not set(src) & set(dst)
            old = dict(m.mem)
            for a, b in zip(src, dst):
                for slot in range(P):
                    if (int(a), slot) in old:
                        m.mem[int(b), slot] = old[int(a), slot]
            held = m.check()
            assert held == set(range(len(held)))
        m.check()
    p.close()


def test_slide_gives_pages_back():
    p = engine.Pool(100, 16, 3)
    m = Model(p)
    m.extend(0, 200)  # 13 pages
    p.slide(0, window=40, sinks=4)
    # the next token, at 200, sees 161..: pages 1..9 (16..159) go, page 0 holds the sinks
    t = p.table(0)
    assert [i for i, g in enumerate(t) if g < 0] == list(range(1, 10))
    assert p.free == 100 - 4
    m.check()
    m.extend(0, 30)
    p.slide(0, window=40, sinks=4)
    assert [i for i, g in enumerate(p.table(0)) if g < 0] == list(range(1, 11))  # 191.. seen
    m.check()
    # shortened so far that a given-back page would be seen: refused, nothing changed
    for n in (17, 100, 214):
        assert code_of(p.trim, 0, n) == -1 and code_of(p.fork, 0, 1, n) == -1
    assert p.len(0) == 230
    p.fork(0, 1, 215)  # 215 sees 176..
    assert code_of(p.trim, 1, 214) == -1
    p.fork(0, 2, 16)
    p.trim(0, 12)
    assert p.len(0) == 12 and list(p.table(0)) == list(p.table(2))
    p.trim(1)
    p.trim(0)
    p.trim(2)
    assert p.free == 100


def test_shared_pages_live_until_the_last_holder():
    p = engine.Pool(10, 16, 4)
    m = Model(p)
    m.extend(0, 40)
    for d in (1, 2):
        p.fork(0, d, 40)
        m.rows[d] = list(m.rows[0])
    assert p.free == 7
    for s in (0, 1):  # a copy of the last page each; the last holder keeps it
        assert p.need(s, 1) == 1
        m.extend(s, 1)
    assert p.need(2, 1) == 0 and p.extend(2, 1) is None
    assert p.free == 5
    p.trim(0)
    p.trim(1)
    assert p.free == 7
    assert code_of(p.extend, 0, 8 * 16) == -5 and p.len(0) == 0 and p.free == 7


def test_compact_room():
    import ctypes as C
    lib = engine.load_library()
    p = engine.Pool(8, 16, 3)
    p.extend(0, 64)
    p.extend(1, 64)
    p.trim(0)
    n = C.c_int32()
    a = (C.c_int32 * 8)()
    assert lib.fg_pool_compact(p._h, a, a, 3, C.byref(n)) == -1 and n.value == 4
    assert list(p.table(1)) == [4, 5, 6, 7]
    src, dst = p.compact()
    assert sorted(src) == [4, 5, 6, 7] and sorted(dst) == [0, 1, 2, 3]
    assert len(p.compact()[0]) == 0


@pytest.mark.parametrize("args", [(0, 16, 1), (4, 16, 0), (4, 8, 1), (4, 24, 1), (4, 512, 1)])
def test_bad_pools(args):
    assert code_of(engine.Pool, *args) == -1


def test_bad_calls():
    p = engine.Pool(4, 16, 2)
    p.extend(0, 20)
    for f, a in [(p.len, (2,)), (p.len, (-1,)), (p.table, (9,)), (p.need, (0, -1)), (p.extend, (0, -1)),
                 (p.extend, (5, 1)), (p.fork, (0, 0, 5)), (p.fork, (0, 1, 21)), (p.fork, (0, 1, -1)),
                 (p.fork, (0, 7, 1)), (p.trim, (0, 21)), (p.trim, (0, -1)), (p.slide, (0, 0, 0)),
                 (p.slide, (0, 4, -1)), (p.need, (0, (1 << 30)))]:
        assert code_of(f, *a) == -1, (f, a)
    assert p.len(0) == 20 and p.free == 2
    lib = engine.load_library()
    assert lib.fg_pool_len(None, 0, None) == -1 and lib.fg_pool_free(None, None) == -1
    assert lib.fg_pool_create(4, 16, 2, None) == -1 and lib.fg_pool_destroy(None) == 0
    assert lib.fg_pool_compact(p._h, None, None, 0, None) == -1
    assert np.array_equal(p.table(0), [0, 1])
