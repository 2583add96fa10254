"""Paged KV cache on the GPU: attention, stores, copies and reads against float64
computations on the host.

Attention's tolerance, per value: a score s_j = sum_d q_d k_jd / sqrt(D) is formed from
q in two binary16 parts (22 bits, truncated: off by 2^-21) and D products summed in
f32, so it is off by at most A (2^-21 + (D + 2) 2^-23), A = max_j sum_d |q_d k_jd| /
sqrt(D) (a part of the sum may be any half); the exponent's argument is rounded again
(2^-23 of its size, at most 2 A) and exp2 is good to 2^-22.  The weights are then off by
E = A (2^-21 + (D + 6) 2^-23) + 2^-21 each, relative, the result by 2 E sum_j p_j |v_j|
(once through the weights, once through their sum), to which summing adds a rounding of
2^-23 per 32-token block, wave and part, and p's own parts 2^-21: (T / 32 + 80) 2^-23.
"""
import numpy as np
import pytest
import torch

from flarellm_amd import FL_KV_F16, FL_KV_F32, FL_KV_Q8, FlareError
from flarellm_amd.pages import PagedKv

pytestmark = pytest.mark.gpu
FORMS = {"f32": FL_KV_F32, "f16": FL_KV_F16, "q8": FL_KV_Q8}


def stored(fmt, x):
    """What a cache of this form holds of f32 rows x [.., D]."""
    if fmt == "f32":
        return x
    if fmt == "f16":
        return x.astype(np.float16).astype(np.float32)
    b = x.reshape(-1, 32)
    amax = np.abs(b).max(1, keepdims=True)
    inv = np.where(amax > 0, np.float32(1) / np.where(amax > 0, amax, np.float32(1)) * np.float32(127), np.float32(0))
    y = (b * inv).astype(np.float32)
    code = np.trunc(y + np.copysign(np.float32(0.49999997), y))
    scale = (amax * (np.float32(1) / np.float32(127))).astype(np.float16).astype(np.float32)
    return (code * scale).astype(np.float32).reshape(x.shape)


class Twin:
    """A PagedKv and what its sequences should hold, as rows on the host."""

    def __init__(self, backend, fmt, heads, kv_heads, D, page, pages, seqs=16, layers=1, max_len=0, fill=None, seed=0):
        self.fmt, self.heads, self.nkv, self.D, self.layers = fmt, heads, kv_heads, D, layers
        self.kv = PagedKv(backend, layers, pages, page, kv_heads, D, FORMS[fmt], seqs, max_len)
        self.rng = np.random.default_rng(seed)
        for t in (self.kv.k, self.kv.v, self.kv.k_scale, self.kv.v_scale):
            if t is not None and fill is not None:
                t.fill_(fill if t.is_floating_point() else 77)
        none = np.zeros((layers, 0, kv_heads, D), np.float32)
        self.rows = {s: (none, none) for s in range(seqs)}

    def extend(self, seqs, counts, values=None):
        n = int(sum(counts))
        k, v = values or (self.rng.standard_normal((self.layers, n, self.nkv, self.D)).astype(np.float32) for _ in "kv")
        self.kv.extend(seqs, counts)
        self.kv.write(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
        at = 0
        for s, c in zip(seqs, counts):
            old = self.rows[s]
            self.rows[s] = tuple(np.concatenate([o, stored(self.fmt, x[:, at: at + c])], 1) for o, x in zip(old, (k, v)))
            at += c

    def fork(self, src, dst, lens=None, deep=False):
        if deep:
            self.kv.copy(src, dst)
        else:
            self.kv.fork(src, dst, lens)
        for i, (s, d) in enumerate(zip(src, dst)):
            n = self.rows[s][0].shape[1] if lens is None else lens[i]
            self.rows[d] = tuple(x[:, :n] for x in self.rows[s])

    def truncate(self, seqs, lens):
        self.kv.truncate(seqs, lens)
        for s, n in zip(seqs, lens):
            self.rows[s] = tuple(x[:, :n] for x in self.rows[s])

    def free(self, seqs):
        self.kv.free(seqs)
        for s in seqs:
            self.rows[s] = tuple(x[:, :0] for x in self.rows[s])

    def check_rows(self):
        ids = [s for s in self.rows if self.rows[s][0].shape[1]]
        lens = [self.rows[s][0].shape[1] for s in ids]
        assert [self.kv.length(s) for s in ids] == lens
        for l in range(self.layers):
            k, v = self.kv.read(ids, [0] * len(ids), lens, layer=l)
            assert np.array_equal(k.cpu().numpy(), np.concatenate([self.rows[s][0][l] for s in ids])), l
            assert np.array_equal(v.cpu().numpy(), np.concatenate([self.rows[s][1][l] for s in ids])), l

    def want(self, q, seqs, seen, layer):
        """(result, tolerance) in float64."""
        G, D = self.heads // self.nkv, self.D
        out, tol = np.zeros(q.shape), np.zeros(q.shape)
        for i, (s, n) in enumerate(zip(seqs, seen)):
            if n == 0:
                continue
            k, v = (x[layer][:n].astype(np.float64) for x in self.rows[s])
            for h in range(self.heads):
                a, b, c = q[i, h].astype(np.float64), k[:, h // G], v[:, h // G]
                with np.errstate(invalid="ignore", over="ignore"):
                    x = b @ a / np.sqrt(D)
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    out[i, h] = p @ c
                    big = (np.abs(b) @ np.abs(a)).max() / np.sqrt(D)
                    e = big * (2.0**-21 + (D + 6) * 2.0**-23) + 2.0**-21
                    tol[i, h] = (2 * e + (n / 32 + 80) * 2.0**-23) * (p @ np.abs(c))
        return out, tol

    def attend(self, seqs, seen=None, layer=0, q=None, **kw):
        if q is None:
            q = self.rng.standard_normal((len(seqs), self.heads, self.D)).astype(np.float32)
        got = self.kv.attention(torch.from_numpy(q).cuda(), seqs, seen, layer=layer, **kw).cpu().numpy()
        n = [self.rows[s][0].shape[1] for s in seqs] if seen is None else seen
        return got, *self.want(q, seqs, n, layer)

    def check(self, *a, **kw):
        got, want, tol = self.attend(*a, **kw)
        off = np.abs(got - want)
        assert (off <= tol).all(), (off / np.maximum(tol, 1e-300)).max()
        return got


@pytest.mark.parametrize("fmt", ["f32", "f16", "q8"])
@pytest.mark.parametrize("page", [32, 96])
def test_rows_come_back(backend, fmt, page):
    """Stores, forks that write to a shared page, deep copies, truncation and compaction keep every row."""
    t = Twin(backend, fmt, 4, 2, 64 if page == 32 else 128, page, 70, layers=2, max_len=600, fill=float("nan"))
    t.extend([0, 3], [75, 1])
    t.check_rows()
    t.fork([0, 0, 3], [1, 2, 4], [75, 33, 1])
    t.extend([1, 0, 4, 2], [1, 40, 2, 70])
    t.check_rows()
    t.fork([1, 2], [5, 6], deep=True)
    t.extend([6, 5], [3, 130])
    t.free([0, 3])
    t.check_rows()
    assert t.kv.compact() > 0
    t.check_rows()
    t.truncate([5, 6], [64, 0])
    t.extend([5], [1])
    t.check_rows()
    assert t.kv.compact() >= 0
    t.check_rows()


@pytest.mark.parametrize("fmt", ["f32", "f16", "q8"])
@pytest.mark.parametrize("heads,kv_heads,D", [(32, 8, 64), (32, 8, 128), (9, 3, 64), (4, 4, 128), (14, 2, 64), (40, 8, 128),
                                              (32, 1, 64), (6, 6, 64)])
def test_single_queries(backend, fmt, heads, kv_heads, D):
    """Sequences of 1 to a few hundred tokens, some sharing a beginning, one slot empty."""
    t = Twin(backend, fmt, heads, kv_heads, D, 64, 90, fill=float("nan"), seed=heads)
    t.extend([0, 1, 2, 3, 4], [1, 31, 64, 65, 300])
    t.fork([4, 4, 2, 4], [5, 6, 7, 8], [300, 150, 64, 256])
    t.extend([5, 6, 4, 8, 7], [1, 70, 9, 1, 2])
    t.check(list(range(9)))
    t.check([8, 15, 5, 4, 0, 6])
    got = t.check([15, 14])
    assert not got.any()


@pytest.mark.parametrize("fmt", ["f32", "f16", "q8"])
@pytest.mark.parametrize("page", [32, 64, 128, 160])
def test_long_shared_prefix(backend, fmt, page):
    """Many queries behind a prefix that is cut over workgroups; prompts with prompts of their own."""
    t = Twin(backend, fmt, 8, 2, 128, page, 9000 // page + 60, seqs=24, seed=page)
    t.extend([0], [3001])
    t.fork([0, 0], [8, 16])
    t.extend([0, 8, 16], [700, 33, 1])
    t.fork([0] * 7 + [8] * 7 + [16] * 3, list(range(1, 8)) + list(range(9, 16)) + [17, 18, 19])
    ids = list(range(20))
    t.extend(ids, [1 + 13 * (i % 5) for i in ids])
    t.check(ids)
    t.check(ids[::-1])
    t.check([3])


@pytest.mark.parametrize("fmt", ["f32", "f16", "q8"])
@pytest.mark.parametrize("queries", [2, 5, 17, 70])
def test_several_queries_of_a_sequence(backend, fmt, queries):
    """Drafts and the prefill of a suffix: query t sees the tokens up to its own."""
    t = Twin(backend, fmt, 6, 2, 64, 32, 200, seqs=8, seed=queries)
    t.extend([0], [333])
    t.fork([0, 0], [1, 2], [333, 100])
    t.extend([0, 1, 2, 3], [queries, queries + 1, queries, queries])
    n = t.kv.lens()
    seqs = [s for s in (2, 0, 3, 1) for _ in range(queries)]
    seen = [int(n[s]) - queries + 1 + i for s in (2, 0, 3, 1) for i in range(queries)]
    t.check(seqs, seen)
    # any subset of any order, some that see little or nothing
    rng = np.random.default_rng(queries)
    seqs = rng.integers(0, 5, 40)
    t.check([int(s) for s in seqs], [int(rng.integers(0, n[s] + 1)) for s in seqs])


@pytest.mark.parametrize("fmt", ["f32", "f16", "q8"])
@pytest.mark.parametrize("heads,kv_heads,D,forks", [(8, 2, 64, 1), (8, 2, 64, 8), (16, 2, 128, 20), (4, 2, 128, 8)])
@pytest.mark.parametrize("size", [1.0, 1e-3, 300.0])
def test_nothing_is_lost_on_the_whole(backend, fmt, heads, kv_heads, D, forks, size):
    """The error of all values together: roundings of 2^-24 each, independent of each
    other, D of them in a score of size 1 (16 x 2^-24 at most), as many again of its
    weight and of the sum: 2^-19 of the result's 2-norm.  For V of any size."""
    t = Twin(backend, fmt, heads, kv_heads, D, 64, 80, seqs=32, seed=forks)
    for n in (300, 2500):
        k, v = (t.rng.standard_normal((1, n, kv_heads, D)).astype(np.float32) for _ in "kv")
        t.extend([0], [n], (k, (v * size).astype(np.float32)))
    t.fork([0] * (forks - 1), range(1, forks))
    got, want, _ = t.attend(list(range(forks)))
    assert np.linalg.norm(got - want) <= 2.0**-19 * np.linalg.norm(want)


def test_the_same_as_the_contiguous_cache(backend):
    """One sequence: the attention of fl_gqa_from_cache over the same rows."""
    from flarellm_amd.synth import ModelSpec
    from flarellm_amd import FL_Q8_0

    spec = ModelSpec("t", 256, 1, 8, 2, 64, 256, 64, 512, FL_Q8_0, FL_Q8_0, None)
    rng = np.random.default_rng(3)
    k, v = (rng.standard_normal((1, 300, 2, 64)).astype(np.float32) for _ in "kv")
    q = rng.standard_normal((1, 8, 64)).astype(np.float32)
    for fmt in FORMS:
        backend.init_gpu_kv_cache(spec, FORMS[fmt])
        backend.gpu_kv_write_batch(0, 0, k[0].reshape(300, -1), v[0].reshape(300, -1))
        one = backend.grouped_query_attention_from_gpu_cache(q.reshape(-1), 0, 300).reshape(1, 8, 64)
        t = Twin(backend, fmt, 8, 2, 64, 64, 8)
        t.extend([2], [300], (k, v))
        assert np.abs(t.check([2], q=q) - one).max() < 2e-3  # (the other's cache path rounds p to binary16)


@pytest.mark.parametrize("fmt", ["f32", "f16", "q8"])
def test_values_that_are_not_finite_stay_with_those_that_see_them(backend, fmt):
    t = Twin(backend, fmt, 4, 2, 64, 32, 60, seqs=6, fill=float("nan"), seed=9)
    k, v = (t.rng.standard_normal((1, 90, 2, 64)).astype(np.float32) for _ in "kv")
    if fmt == "q8":  # a block with such a value has no codes: the scale is what it leaves
        k[0, 70, 0, :32], v[0, 75, 1, :32] = 1e30, 1e30
    else:
        k[0, 70, 0, 5], v[0, 75, 1, 7], v[0, 80, 0, 9] = np.nan, np.inf, np.nan
    t.extend([0], [90], (k, v))
    t.fork([0, 0], [1, 2], [90, 70])
    t.extend([1, 2], [5, 5])
    seqs, seen = [0] * 5 + [1, 2, 2], [64, 70, 75, 76, 90, 95, 75, 3]
    got, want, tol = t.attend(seqs, seen)
    ok = np.isfinite(want)
    assert ok[[0, 1, 6, 7]].all() and not ok[4].all()
    assert (np.isnan(want) == np.isnan(got)).all()
    assert (got[~ok & ~np.isnan(want)] == want[~ok & ~np.isnan(want)]).all()
    assert (np.abs(got - want)[ok] <= tol[ok]).all()
    # large finite ones, and queries of any size
    q = (t.rng.standard_normal((3, 4, 64)) * np.array([1e-30, 1e4, 0.0])[:, None, None]).astype(np.float32)
    t.check([2, 2, 2], [75, 40, 64], q=q)


def test_rows_of_wider_tensors(backend):
    """Keys, values and queries that are slices of one fused projection's output."""
    t = Twin(backend, "f16", 8, 2, 64, 64, 20, seed=4)
    n, W = 70, (8 + 2 + 2) * 64 + 4
    x = torch.randn(n, W, device="cuda")
    q, k, v = x[:, :512].view(n, 8, 64), x[:, 512:640].view(n, 2, 64), x[:, 640:768].view(n, 2, 64)
    t.kv.extend([5], [n])
    t.kv.write(k, v)
    t.rows[5] = tuple(stored("f16", a.cpu().numpy()[None]) for a in (k, v))
    seen = list(range(1, n + 1))
    got = t.kv.attention(q, [5] * n, seen).cpu().numpy()
    want, tol = t.want(q.cpu().numpy(), [5] * n, seen, 0)
    assert (np.abs(got - want) <= tol).all()
    # an unaligned slice, and the caller's own result tensor
    y = torch.zeros(n * 512 + 1, device="cuda")[1:].view(n, 8, 64)
    y.copy_(q)
    out = torch.empty(n, 8, 64, device="cuda")
    assert t.kv.attention(y, [5] * n, seen, out=out) is out
    assert np.array_equal(out.cpu().numpy(), got)


def test_other_streams(backend):
    """Tensors made on a side stream right before the call, used there right after."""
    t = Twin(backend, "f16", 8, 2, 128, 64, 80, seed=5)
    k, v = (t.rng.standard_normal((1, 2000, 2, 128)).astype(np.float32) for _ in "kv")
    q = t.rng.standard_normal((1, 8, 128)).astype(np.float32)
    ck, cv, cq = (torch.from_numpy(x).cuda() for x in (k, v, q))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for stream in (side, t.kv.stream, torch.cuda.default_stream()):
        with torch.cuda.stream(stream):
            slow = torch.randn(4096, 4096, device="cuda")
            for _ in range(8):
                slow = slow @ slow * 1e-2
            keep = (slow[0, 0] * 0).nan_to_num()
            t.kv.extend([1], [2000])
            t.kv.write(ck + keep, cv + keep)
            got = t.kv.attention(cq + keep, [1]) * 1.0
        stream.synchronize()
        t.rows[1] = tuple(stored("f16", x) for x in (k, v))
        want, tol = t.want(q, [1], [2000], 0)
        assert (np.abs(got.cpu().numpy() - want) <= tol).all()
        t.free([1])


def test_plans_follow_the_tables(backend):
    """The same call again after each change of the sequences, and calls between that have other queries."""
    t = Twin(backend, "f16", 8, 2, 64, 32, 100, seqs=6, seed=6)
    t.extend([0, 1], [200, 10])
    for step in range(6):
        t.check([0, 1, 5])
        t.check([1])
        if step == 1:
            t.fork([0], [5])
        if step == 2:
            t.extend([5, 1], [40, 3])
        if step == 3:
            t.free([0])
            t.extend([0], [7])
        if step == 4:
            t.truncate([5], [100])
            assert t.kv.compact() > 0
        t.extend([1], [1])
    # other head counts over the same pages
    t.heads = 4
    t.check([0, 1, 5])


def test_a_batch_from_prompt_to_answers(backend):
    """As a serving program uses it: a system prompt, two prompts behind it with a
    causal prefill, three answers each, steps of one token in every layer; one
    answer ends, the pool is made dense, the others go on."""
    L, H, N, D = 3, 6, 2, 64
    t = Twin(backend, "f16", H, N, D, 32, 64, seqs=8, layers=L, max_len=400, fill=float("nan"), seed=8)
    t.extend([0], [97])
    t.fork([0], [3])
    t.extend([0, 3], [40, 29])
    for l in range(L):  # the prompts' own tokens, after the shared ones
        seqs = [0] * 40 + [3] * 29
        t.check(seqs, list(range(98, 138)) + list(range(98, 127)), layer=l)
    t.fork([0, 0, 3, 3], [1, 2, 4, 5])
    live = [0, 1, 2, 3, 4, 5]
    for step in range(40):
        t.extend(live, [1] * len(live))
        for l in range(L):
            t.check(live, layer=l)
        if step == 20:
            t.free([1, 3])
            live = [0, 2, 4, 5]
            t.kv.compact()
            t.check_rows()
    t.check_rows()
    used = 64 - t.kv.free_pages
    t.free(live)
    assert t.kv.free_pages == 64 and used < 4 * (137 + 40) // 32


@pytest.mark.parametrize("fmt,heads,kv_heads,page", [("q8", 32, 1, 4096), ("f32", 64, 2, 128), ("f16", 64, 2, 4096)])
def test_the_largest_groups_and_pages(backend, fmt, heads, kv_heads, page):
    t = Twin(backend, fmt, heads, kv_heads, 64, page, 8 if page > 1000 else 40, seqs=5, max_len=4200, fill=float("nan"), seed=page)
    t.extend([0, 1], [700, 3])
    t.fork([0], [2])
    t.extend([2, 0], [1, 2])
    t.check([0, 1, 2, 2, 3], [702, 3, 701, 65, 0])
    t.check_rows()


def test_an_extend_that_fails_leaves_the_one_before(backend):
    """Its tokens, in more blocks than go with a launch, may still be stored."""
    t = Twin(backend, "f16", 4, 1, 64, 32, 300, seqs=8, max_len=9600)
    x = [torch.randn(5000, 1, 64, device="cuda") for _ in "kv"]
    t.kv.extend([0, 1], [4500, 500])
    with pytest.raises(FlareError, match="needed"):
        t.kv.extend([0, 2], [4800, 9600])
    with pytest.raises(FlareError):
        t.kv.extend([2, 2], [9600, 1])
    t.kv.write(*x)
    t.rows[0], t.rows[1] = ([stored("f16", r[None, s].cpu().numpy()) for r in x] for s in (slice(0, 4500), slice(4500, 5000)))
    t.check_rows()
    t.check([0, 1])
    t.extend([1, 2], [100, 4300])  # one that outgrows its memory and does not
    t.check_rows()


@pytest.mark.parametrize("fmt,heads,kv_heads,D", [("f32", 9, 3, 64), ("f16", 32, 8, 128), ("q8", 8, 8, 64), ("f16", 14, 2, 64)])
def test_joined_where_the_last_part_arrives(backend, fmt, heads, kv_heads, D):
    """A few parts a query, joined in the launch: in the same order whichever arrives last, call after
    call with one plan (its counts start from zero again) and with others between; queries that see nothing."""
    t = Twin(backend, fmt, heads, kv_heads, D, 32, 200, seqs=12, max_len=2000, seed=heads)
    t.extend([0], [700])
    t.fork([0] * 5, [1, 2, 3, 4, 5], [700, 690, 512, 100, 700])
    t.extend([0, 1, 2, 3, 6], [9, 60, 33, 1, 400])
    seqs, seen = [0, 1, 2, 3, 4, 5, 6, 7, 5, 1, 8], [709, 760, 723, 513, 100, 0, 400, 0, 31, 650, 0]
    q = t.rng.standard_normal((len(seqs), heads, D)).astype(np.float32)
    first = t.check(seqs, seen, q=q)
    for i in range(20):
        got = t.check(seqs, seen, q=q)
        assert np.array_equal(got, first)
        if i % 5 == 0:
            t.check([1, 6], [760, 399])
    many = [s for s in range(7) for _ in range(40)]  # joined by a launch of its own
    t.check(many, [100 - i % 40 for i in range(len(many))])
    t.check(many, [t.rows[s][0].shape[1] - i % 40 for i, s in enumerate(many)])
    assert np.array_equal(t.check(seqs, seen, q=q), first)


@pytest.mark.parametrize("idle", [1, 64, 65, 3000])
def test_queries_that_see_nothing(backend, idle):
    """Rows of empty sequences among others are zeros, wherever and however many they are."""
    t = Twin(backend, "f16", 4, 2, 64, 32, 40, seqs=8)
    t.extend([0, 1], [500, 3])
    for rest in ([0], [1], [0, 1, 1], []):
        seqs = [2] * (idle // 2) + rest + [3] * (idle - idle // 2)
        out = torch.full((len(seqs), 4, 64), float("nan"), device="cuda")
        q = t.rng.standard_normal((len(seqs), 4, 64)).astype(np.float32)
        t.check(seqs, q=q, out=out)
        empty = [i for i, s in enumerate(seqs) if s > 1]
        assert not out[empty].any()


def test_values_not_finite_in_a_part(backend):
    """An infinity in one part of a query that others do not see."""
    t = Twin(backend, "f16", 8, 2, 64, 32, 60, seqs=4)
    k, v = (t.rng.standard_normal((1, 600, 2, 64)).astype(np.float32) for _ in "kv")
    v[0, 300, 1, 5] = np.inf
    t.extend([0], [600], (k, v))
    t.fork([0], [1], [290])
    t.extend([1], [50])
    q = t.rng.standard_normal((3, 8, 64)).astype(np.float32)
    got, want, tol = t.attend([0, 1, 0], [600, 340, 300], q=q)
    assert np.isposinf(got[0, 4:, 5]).all()
    got[0, 4:, 5] = want[0, 4:, 5] = tol[0, 4:, 5] = 0
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("new", [1, 70])
def test_long_lists(backend, new):
    """More copies and runs of one call than go with its launch, and the two lists together."""
    t = Twin(backend, "f16", 2, 1, 64, 64, 700, seqs=130, max_len=12000, layers=2)
    t.extend([0], [9 * 64 + 20])
    t.fork([0] * 129, list(range(1, 130)))
    t.extend(list(range(130)), [new] * 130)
    t.check_rows()
    t.check(list(range(0, 130, 9)), layer=1)
    t.truncate(list(range(130)), [9 * 64] * 130)
    t.free(list(range(1, 129)))
    t.extend([0], [7000])
    t.fork([0, 129], [1, 2], deep=True)
    t.free([0])
    assert t.kv.compact() > 96
    t.check_rows()
    t.check([1, 2, 129], layer=1)


def test_one_token_of_many_layers(backend):
    """A token of a [layers, tokens, ..] buffer; a page's last slots."""
    t = Twin(backend, "f32", 4, 2, 64, 32, 20, layers=4)
    k, v = (torch.randn(4, 40, 2, 64, device="cuda") for _ in "kv")
    for i in range(40):
        t.kv.extend([5], [1])
        t.kv.write(k[:, i: i + 1], v[:, i: i + 1])
    t.rows[5] = (k.cpu().numpy(), v.cpu().numpy())
    t.check_rows()
    for l in range(4):
        t.check([5, 5], [40, 33], layer=l)


def test_odd_strides(backend):
    """Rows of odd widths, several layers at once."""
    t = Twin(backend, "q8", 4, 2, 64, 32, 20, layers=3)
    k, v = (torch.randn(3, 37, 131, device="cuda")[:, :, 2:130].view(3, 37, 2, 64) for _ in "kv")
    t.kv.extend([1, 2], [30, 7])
    t.kv.write(k[1:], v[1:], layer=1)
    t.kv.write(k[0], v[0])
    t.rows[1], t.rows[2] = ([stored("q8", x[:, s].cpu().numpy().copy()) for x in (k, v)] for s in (slice(0, 30), slice(30, 37)))
    t.check_rows()
    q = torch.randn(5, 259, device="cuda")[:, 1:257].view(5, 4, 64)
    seqs, seen = [1, 2, 1, 2, 1], [30, 7, 1, 2, 29]
    for l in range(3):
        want, tol = t.want(q.cpu().numpy(), seqs, seen, l)
        assert (np.abs(t.kv.attention(q, seqs, seen, layer=l).cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize("fmt", ["f16", "q8"])
def test_offsets_past_32_bits(backend, fmt):
    """Pages whose elements begin past 2^32."""
    page, nkv, D = 128, 8, 128
    high = (1 << 32) // (page * nkv * D) + 50
    t = Twin(backend, fmt, 16, nkv, D, page, high + 8, seqs=4, max_len=high * page)
    t.kv.extend([3], [high * page])  # (its rows are not looked at)
    t.extend([0], [200])
    assert t.kv.tables()[0][0] == high
    t.fork([0], [1])
    t.extend([1, 0], [3, 70])
    t.check([0, 1, 0], [270, 203, 5])
    t.check_rows()
    del t
    torch.cuda.empty_cache()


def test_two_pools_at_once(backend):
    """Pools share the backend's stream, not their workspaces or plans."""
    a = Twin(backend, "f16", 8, 2, 64, 64, 60, seed=1)
    b = Twin(backend, "q8", 8, 2, 64, 32, 90, seed=2)
    a.extend([0, 1], [1500, 20])
    b.extend([0, 1], [900, 700])
    q = np.random.default_rng(0).standard_normal((2, 8, 64)).astype(np.float32)
    d = torch.from_numpy(q).cuda()
    outs = [(a.kv.attention(d, [0, 1]), b.kv.attention(d, [1, 0])) for _ in range(3)]
    for x, y in outs:
        for t, got, seqs in ((a, x, [0, 1]), (b, y, [1, 0])):
            want, tol = t.want(q, seqs, [t.rows[s][0].shape[1] for s in seqs], 0)
            assert (np.abs(got.cpu().numpy() - want) <= tol).all()


def test_refusals(backend):
    t = Twin(backend, "f16", 8, 2, 64, 32, 10, seqs=4, max_len=100)
    kv = t.kv
    t.extend([0], [40])
    q = torch.randn(1, 8, 64, device="cuda")
    row = torch.randn(1, 2, 64, device="cuda")
    with pytest.raises(FlareError, match="sees 41"):
        kv.attention(q, [0], [41])
    with pytest.raises(FlareError):
        kv.attention(q, [4], [0])
    with pytest.raises(FlareError, match="layers"):
        kv.attention(q, [0], layer=1)
    with pytest.raises(FlareError, match="heads"):
        kv.attention(torch.randn(1, 7, 64, device="cuda"), [0])
    with pytest.raises(FlareError, match="query heads"):
        kv.attention(torch.randn(1, 66, 64, device="cuda"), [0])
    for bad in (q.half(), q.cpu(), torch.randn(1, 64, 8, device="cuda").transpose(1, 2), q[0], torch.randn(1, 8, 32, device="cuda")):
        with pytest.raises(ValueError):
            kv.attention(bad, [0])
    with pytest.raises(ValueError):
        kv.attention(q, [0, 1])
    with pytest.raises(ValueError):
        kv.attention(q, [0.5])
    with pytest.raises(ValueError):
        kv.attention(q, [0], out=torch.empty(1, 8, 128, device="cuda")[:, :, :64])
    with pytest.raises(ValueError, match="room for 40"):
        kv.write(row, row)
    kv.extend([1], [1])
    kv.fork([0], [2])
    with pytest.raises(FlareError, match="follows"):
        kv.write(row, row)
    with pytest.raises(FlareError, match="pages needed"):
        kv.extend([1, 3], [99, 100])
        kv.extend([0], [60])
    with pytest.raises(FlareError):
        kv.read([0], [30], [11])
    with pytest.raises(FlareError):
        kv.read([0], [-1], [2])
    assert kv.attention(q[:0], []).shape == (0, 8, 64)
    kv.extend([], [])
    kv.write(row[:0], row[:0])
    with pytest.raises(FlareError):
        PagedKv(backend, 1, 4, 40, 2, 64)
    kv.close()
    with pytest.raises(FlareError, match="closed"):
        kv.attention(q, [0], [1])


def test_queries_and_result_apart(backend):
    t = Twin(backend, "f16", 8, 2, 64, 32, 10, seqs=4, max_len=100)
    t.extend([0], [40])
    x = torch.randn(5, 8, 64, device="cuda")
    before = x.clone()
    for q, out in ((x[:2], x[:2]), (x[:2], x[1:3]), (x[1:3], x[:2]), (x[::2], x[2:5])):
        with pytest.raises(FlareError, match="overlap"):
            t.kv.attention(q, [0] * q.shape[0], [40] * q.shape[0], out=out)
    assert torch.equal(x, before)
    t.kv.attention(x[:2], [0, 0], [40, 7], out=x[2:4])  # side by side
    want, tol = t.want(before[:2].cpu().numpy(), [0, 0], [40, 7], 0)
    assert (np.abs(x[2:4].cpu().numpy() - want) <= tol).all() and torch.equal(x[4], before[4])
    with pytest.raises(FlareError, match="layers"):
        t.kv.read([0], [0], [1], layer=1)
    t.kv.close()
    for call in (lambda: t.kv.free_pages, lambda: t.kv.length(0), t.kv.tables, t.kv.compact):
        with pytest.raises(FlareError, match="closed"):
            call()


def test_capture_is_refused(backend):
    """A call under capture is an error and leaves the sequences alone; the capture goes on."""
    t = Twin(backend, "f16", 8, 2, 64, 32, 20)
    t.extend([0], [70])
    q = torch.randn(1, 8, 64, device="cuda")
    out = torch.empty(1, 8, 64, device="cuda")
    x = torch.zeros(4, device="cuda")
    t.kv.attention(q, [0], out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=t.kv.stream):
        x += 1
        with pytest.raises(FlareError, match="captured"):
            t.kv.attention(q, [0], out=out)
        with pytest.raises(FlareError, match="captured"):
            t.kv.extend([0], [1])
        with pytest.raises(FlareError, match="captured"):
            t.kv.compact()
    g.replay()
    torch.cuda.synchronize()
    assert x.tolist() == [1.0] * 4 and t.kv.length(0) == 70
    t.check([0])
    # the capture of another stream, which the backend's joins
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        x += 1
        with pytest.raises(FlareError, match="captured"):
            t.kv.attention(q, [0], out=out)
        x += 1
    for i in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert x.tolist() == [3.0 + 2 * i] * 4
        t.check([0])
