"""Paged KV cache, host side: page bookkeeping against a token-by-token model, the
coverage of attention plans, and refusals (no GPU)."""
import ctypes as C

import numpy as np
import pytest

from flarellm_amd import _lib as L

INVALID, UNSUPPORTED, STATE, OOM = -1, -2, -4, -5


class Pages:
    """fl_pages without a device."""

    def __init__(self, pages=32, page_size=64, seqs=8, max_len=1000, kv_heads=2, fmt=L.FL_KV_F16, head_dim=64, layers=1):
        self.lib = L.load()
        self.P, self.seqs, self.max_len, self.kv_heads = page_size, seqs, max_len, kv_heads
        cfg = L.PagesConfig(layers, kv_heads, head_dim, fmt, pages, page_size, seqs, max_len)
        self.h = C.c_void_p()
        self.rc = self.lib.fl_pages_create(None, C.byref(cfg), None, None, None, None, C.byref(self.h))

    def __del__(self):
        self.lib.fl_pages_destroy(self.h)

    def call(self, name, *lists):
        arrays = [None if x is None else np.ascontiguousarray(x, np.int32) for x in lists]
        return getattr(self.lib, "fl_pages_" + name)(self.h, *(None if a is None else a.ctypes.data for a in arrays),
                                                      len(lists[0]))

    def fork(self, src, dst, lens=None):
        return self.call("fork", src, dst, lens)

    def compact(self):
        n = C.c_int(-1)
        assert self.lib.fl_pages_compact(self.h, C.byref(n)) == 0
        return n.value

    def tables(self):
        t = np.empty((self.seqs, -(-self.max_len // self.P)), np.int32)
        n = np.empty(self.seqs, np.int32)
        assert self.lib.fl_pages_tables(self.h, t.ctypes.data, n.ctypes.data) == 0
        return t, n

    def copies(self):
        n = self.lib.fl_pages_copies(self.h, None, 0)
        c = np.empty((n, 3), np.int32)
        assert self.lib.fl_pages_copies(self.h, c.ctypes.data, n) == n
        return c

    def plan(self, seqs, seen, heads):
        a, b = np.ascontiguousarray(seqs, np.int32), np.ascontiguousarray(seen, np.int32)
        n = self.lib.fl_pages_plan(self.h, a.ctypes.data, b.ctypes.data, len(a), heads, None, 0)
        if n < 0:
            return n
        items = np.empty((n, 6), np.int32)
        assert self.lib.fl_pages_plan(self.h, a.ctypes.data, b.ctypes.data, len(a), heads, items.ctypes.data, n) == n
        return items

    def free_count(self):
        return self.lib.fl_pages_free_count(self.h)

    def error(self):
        return self.lib.fl_last_error(None).decode()


class Model:
    """What each slot holds, and what each sequence should."""

    def __init__(self, p, pages):
        self.p = p
        self.slots = np.zeros((pages, p.P), np.int64)
        self.want = [[] for _ in range(p.seqs)]
        self.next = 1

    def moved(self):
        """The last call's copies, on the slots (all read before any is written)."""
        c, before = self.p.copies(), self.slots.copy()
        assert len(set(c[:, 1])) == len(c)
        for src, dst, blocks in c:
            self.slots[dst, : 32 * blocks] = before[src, : 32 * blocks]

    def extend(self, seqs, counts):
        self.moved()
        t, n = self.p.tables()
        for s, c in zip(seqs, counts):
            for j in range(n[s] - c, n[s]):
                self.slots[t[s, j // self.p.P], j % self.p.P] = self.next
                self.want[s].append(self.next)
                self.next += 1

    def check(self, pages):
        t, n = self.p.tables()
        used = set()
        for s in range(self.p.seqs):
            assert n[s] == len(self.want[s]) == self.p.lib.fl_pages_len(self.p.h, s)
            held = -(-n[s] // self.p.P)
            assert (t[s, held:] == -1).all() and (t[s, :held] >= 0).all()
            used |= set(t[s, :held].tolist())
            got = [self.slots[t[s, j // self.p.P], j % self.p.P] for j in range(n[s])]
            assert got == self.want[s], s
        assert self.p.free_count() == pages - len(used)
        return used


@pytest.mark.parametrize("seed,page,pages,seqs", [(0, 32, 40, 6), (1, 64, 23, 9), (2, 96, 130, 20), (3, 32, 65, 3)])
def test_random_operations_keep_every_sequence(seed, page, pages, seqs):
    rng = np.random.default_rng(seed)
    p = Pages(pages, page, seqs, 400)
    assert p.rc == 0
    m = Model(p, pages)
    for step in range(400):
        op = rng.choice(["extend", "extend", "extend", "fork", "copy", "free", "truncate", "compact"])
        t0, n0 = p.tables()
        free0 = p.free_count()
        some = rng.permutation(seqs)[: rng.integers(1, seqs + 1)]
        if op == "extend":
            counts = rng.choice([0, 1, 1, 2, int(rng.integers(1, 90))], len(some))
            rc = p.call("extend", some, counts)
            if any(n0[s] + c > 400 for s, c in zip(some, counts)):
                assert rc == INVALID
            elif rc == 0:
                m.extend(some, counts)
        elif op in ("fork", "copy"):
            empty = [s for s in range(seqs) if n0[s] == 0]
            full = [s for s in range(seqs) if n0[s] > 0]
            if not empty or not full:
                continue
            dst = rng.permutation(empty)[: rng.integers(1, len(empty) + 1)]
            src = rng.choice(full, len(dst))
            if op == "fork":
                lens = [int(rng.integers(0, n0[s] + 1)) for s in src] if rng.random() < 0.5 else None
                rc = p.fork(src, dst, lens)
                assert rc == 0 and p.free_count() == free0 and len(p.copies()) == 0
            else:
                lens = None
                rc = p.call("copy", src, dst)
                need = sum(-(-n0[s] // page) for s in src)
                assert (rc == OOM) == (need > free0)
            if rc == 0:
                m.moved()
                for i, (s, d) in enumerate(zip(src, dst)):
                    m.want[d] = m.want[s][: None if lens is None else lens[i]]
        elif op == "free":
            some = some[: 1 + len(some) // 3]
            rc = p.call("free", some)
            assert rc == 0
            for s in some:
                m.want[s] = []
        elif op == "truncate":
            lens = [int(rng.integers(0, n0[s] + 1)) for s in some]
            rc = p.call("truncate", some, lens)
            assert rc == 0
            for s, n in zip(some, lens):
                m.want[s] = m.want[s][:n]
        else:
            rc, moved = 0, p.compact()
            assert moved == len(p.copies())
            m.moved()
        if rc:
            t1, n1 = p.tables()
            assert (t0 == t1).all() and (n0 == n1).all() and p.free_count() == free0
        used = m.check(pages)
        if op == "compact":
            assert used == set(range(len(used)))


def test_new_pages_are_the_lowest_free_ones():
    p = Pages(pages=200, page_size=32, seqs=4, max_len=5000)
    assert p.call("extend", [0, 1], [100, 70]) == 0
    assert p.tables()[0][:2, :4].tolist() == [[0, 1, 2, 3], [4, 5, 6, -1]]
    assert p.call("free", [0]) == 0
    assert p.call("extend", [2, 1], [40, 200]) == 0
    t = p.tables()[0]
    assert t[2, :2].tolist() == [0, 1] and t[1, :9].tolist() == [4, 5, 6, 2, 3, 7, 8, 9, 10]


def test_only_a_shared_page_is_copied_and_the_last_holder_keeps_it():
    p = Pages(pages=16, page_size=64, seqs=4)
    assert p.call("extend", [0], [70]) == 0
    assert p.fork([0, 0, 0], [1, 2, 3], [70, 65, 64]) == 0
    assert p.free_count() == 14
    # 1 and 0 hold page 1 with 2; 3 ends at a page's end and shares nothing that it writes to
    assert p.call("extend", [1, 3, 0, 2], [1, 1, 0, 1]) == 0
    assert p.copies().tolist() == [[1, 2, 1], [1, 4, 1]]
    t = p.tables()[0]
    assert t[:, :2].tolist() == [[0, 1], [0, 2], [0, 4], [0, 3]]
    assert p.call("extend", [0], [1]) == 0 and len(p.copies()) == 0  # its page is its own now


def test_refusals_leave_everything_as_it_was():
    p = Pages(pages=4, page_size=32, seqs=4, max_len=128)
    assert p.call("extend", [0], [40]) == 0
    t0, n0 = p.tables()
    bad = [
        ("extend", INVALID, [4], [1]), ("extend", INVALID, [-1], [1]), ("extend", INVALID, [1, 1], [1, 1]),
        ("extend", INVALID, [0], [-1]), ("extend", INVALID, [0], [89]), ("extend", INVALID, [1], [2**31 - 1]),
        ("extend", OOM, [1, 2], [32, 33]), ("extend", INVALID, [0], None),
        ("copy", STATE, [0], [0]), ("copy", INVALID, [1], [1]), ("copy", INVALID, [0, 0], [1, 1]), ("copy", OOM, [0, 0], [1, 2]),
        ("copy", INVALID, [0], [7]), ("copy", INVALID, [9], [1]),
        ("free", INVALID, [5]), ("free", INVALID, [-2]),
        ("truncate", INVALID, [0], [41]), ("truncate", INVALID, [0], [-1]), ("truncate", INVALID, [0, 0], [3, 4]),
    ]
    for name, code, *lists in bad:
        assert p.call(name, *lists) == code, (name, lists)
        assert p.error()
        t1, n1 = p.tables()
        assert (t0 == t1).all() and (n0 == n1).all() and p.free_count() == 2
    forks = [(INVALID, [0], [1], [41]), (INVALID, [0], [1], [-1]), (STATE, [0], [0], None), (INVALID, [0, 1], [1, 2], None),
             (INVALID, [0, 0], [1, 1], None), (INVALID, [4], [1], None), (INVALID, [0], [4], None)]
    for code, src, dst, lens in forks:
        assert p.fork(src, dst, lens) == code, (src, dst, lens)
    assert p.lib.fl_pages_extend(p.h, None, None, 1) == INVALID
    assert p.lib.fl_pages_extend(p.h, None, None, -1) == INVALID
    assert p.lib.fl_pages_free(None, None, 0) == INVALID
    assert p.lib.fl_pages_len(p.h, 4) == -1 and p.lib.fl_pages_len(None, 0) == -1 and p.lib.fl_pages_free_count(None) == -1
    assert p.plan([0], [41], 2) == INVALID and p.plan([0], [-1], 2) == INVALID and p.plan([4], [0], 2) == INVALID
    assert p.plan([0], [1], 3) == INVALID
    # work needs a device
    x = np.zeros(1 << 12, np.float32)
    one = np.array([0], np.int32)
    assert p.lib.fl_pages_write(p.h, 0, 1, x.ctypes.data, x.ctypes.data, 128) == STATE
    assert p.lib.fl_pages_attention(p.h, 0, x.ctypes.data, 128, one.ctypes.data, one.ctypes.data, 1, 2, x.ctypes.data) == STATE
    assert p.lib.fl_pages_read(p.h, 0, one.ctypes.data, one.ctypes.data, one.ctypes.data, 1, x.ctypes.data, None) == STATE
    assert p.call("free", [0, 0]) == 0 and p.free_count() == 4  # emptied twice is emptied


@pytest.mark.parametrize("change,code", [
    (dict(head_dim=96), UNSUPPORTED), (dict(fmt=L.FL_KV_KIVI2), UNSUPPORTED), (dict(fmt=9), UNSUPPORTED),
    (dict(page_size=48), INVALID), (dict(page_size=0), INVALID), (dict(page_size=8192), INVALID), (dict(pages=0), INVALID),
    (dict(pages=1 << 26, page_size=64), INVALID), (dict(pages=1 << 24, page_size=32), INVALID), (dict(seqs=0), INVALID), (dict(max_len=0), INVALID),
    (dict(layers=0), INVALID), (dict(kv_heads=0), INVALID), (dict(layers=1 << 12, kv_heads=16), INVALID),
    (dict(seqs=1 << 30), INVALID)])
def test_bad_configurations(change, code):
    p = Pages(**change)
    assert p.rc == code and not p.h.value


def test_bytes():
    lib = L.load()
    kv, sc = C.c_size_t(), C.c_size_t()
    for fmt, size, scale in ((L.FL_KV_F32, 4, 0), (L.FL_KV_F16, 2, 0), (L.FL_KV_Q8, 1, 2)):
        cfg = L.PagesConfig(3, 5, 128, fmt, 7, 96, 2, 100)
        assert lib.fl_pages_bytes(C.byref(cfg), C.byref(kv), C.byref(sc)) == 0
        assert kv.value == 3 * 5 * 128 * 7 * 96 * size and sc.value == 3 * 5 * 4 * 7 * 96 * scale
    assert lib.fl_pages_bytes(None, C.byref(kv), C.byref(sc)) == INVALID


def grown(rng, p, system, groups, forks, prefix, tails):
    """Sequences with a common beginning, prompts behind it and tails; returns their ids."""
    assert p.call("extend", [0], [system]) == 0
    heads = [g * forks for g in range(groups)]
    assert p.fork([0] * (groups - 1), heads[1:]) == 0
    assert p.call("extend", heads, [prefix] * groups) == 0
    assert p.fork([g * forks for g in range(groups) for _ in range(1, forks)],
                  [g * forks + f for g in range(groups) for f in range(1, forks)]) == 0
    ids = list(range(groups * forks))
    for s in ids:
        assert p.call("extend", [s], [int(tails[s])]) == 0
    return ids


@pytest.mark.parametrize("page,system,groups,forks,prefix,heads,kv_heads", [
    (32, 100, 3, 4, 77, 8, 2), (64, 0, 1, 1, 0, 2, 2), (64, 0, 5, 3, 300, 12, 1), (96, 500, 1, 9, 0, 64, 2), (32, 64, 2, 2, 64, 6, 2)])
@pytest.mark.parametrize("queries", [1, 3, 40])
def test_plans_cover_every_token_once(page, system, groups, forks, prefix, heads, kv_heads, queries):
    rng = np.random.default_rng(page + groups + queries)
    p = Pages(400, page, 32, 2000, kv_heads=kv_heads)
    tails = rng.integers(1, 200, groups * forks)
    ids = grown(rng, p, system, groups, forks, prefix, tails)
    t, n = p.tables()
    seqs = np.repeat(ids + [31], queries)  # (31 is empty)
    seen = np.array([rng.integers(0, n[s] + 1) if rng.random() < 0.4 else n[s] for s in seqs])
    order = rng.permutation(len(seqs))
    seqs, seen = seqs[order], seen[order]
    items = p.plan(seqs, seen, heads)
    covered = [np.zeros(m, int) for m in seen]
    parts, units = {}, {}
    read = {}
    for q, lo, hi, page0, form, unit in items.tolist():
        assert lo % 32 == 0 and lo < hi and lo < seen[q]
        assert t[seqs[q], lo // page] == page0
        covered[q][lo:hi] += 1
        parts.setdefault(q, []).append(unit)
        if unit >= 0:
            assert unit not in units
            units[unit] = q
    assert all((c == 1).all() for c in covered)
    # one part alone is written as the result; several have a place each
    for q, u in parts.items():
        assert u == [-1] or -1 not in u
    assert sorted(units) == list(range(len(units)))


def test_shared_pages_are_read_once():
    """Eight sequences of one prompt: its pages are in items of all eight, not in eight items."""
    p = Pages(200, 64, 8, 4000, kv_heads=2)
    grown(None, p, 0, 1, 8, 2000, np.full(8, 30))
    n = p.tables()[1]
    items = p.plan(range(8), n, 8)  # 4 heads a kv head: 32 rows
    full = 2000 // 64 * 64
    shared = [r for r in items.tolist() if r[1] < full]
    spans = {(r[1], r[2]) for r in shared}
    assert all(r[2] <= full for r in shared)
    assert len(shared) == 8 * len(spans) and sum(hi - lo for lo, hi in spans) == full
    own = [r for r in items.tolist() if r[1] >= full]
    assert sorted(r[0] for r in own) == list(range(8)) and all(r[1] == full and r[2] == 2030 for r in own)
