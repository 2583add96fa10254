"""Operators of the paged KV cache, case by case.

A case is one pass through an operator of `flarellm_amd.pages.PagedKv` on what a
serving program already holds:

  attend    attention of a batch of queries over the pages of their sequences.
            All sequences begin with the same `root` tokens, the `forks`
            sequences of each of `groups` prompts share `prefix` more, and each
            has a tail of its own; `queries` tokens of each sequence are queries
            (1: a decode step), the last of them sees the whole sequence.  `idle`
            more batch slots hold no sequence.
  append    a step that gives each of `rows` sequences some new tokens: slots are
            reserved, keys and values stored, and the step is taken back
  fork      one sequence is forked, and each of the sequences gets a token: the
            page that the forks would write to is copied for each; then the forks
            are freed
  compact   sequences are copied twice, the first copies freed and the others
            moved down into the hole; then these are freed too

Head counts and sizes are those of `flarellm_amd.synth` (SmolLM2-135M,
Llama-3.2-1B and Llama-3-8B) or generic.  Queries, keys and values are N(0, 1),
which is what N(0, 0.02) weights make of a normalized row.

The plain form of each operator computes in 32 bits on the page layout that
`PagedKv` documents:

  K [layer][page][kv head][slot][D],  V [layer][page][kv head][slot / 32][D][32]

with, for the 8-bit form, a binary16 scale per (slot, 32 channels) beside each.
"""
import math

import numpy as np
import torch

own = False

FORMATS = {"f32": torch.float32, "f16": torch.float16, "q8": torch.int8}
BYTES = {"f32": 4.0, "f16": 2.0, "q8": 1.0 + 2.0 / 32}


def _shape(heads, kv_heads, head_dim):
    return dict(heads=heads, kv_heads=kv_heads, head_dim=head_dim)


SMOL_135M, LLAMA_1B, LLAMA_8B = _shape(9, 3, 64), _shape(32, 8, 64), _shape(32, 8, 128)


def _attend(fmt, shape, page, groups, forks, root=0, prefix=0, tail=(1, 1), queries=1, idle=0, **more):
    return dict(op="attend", fmt=fmt, page=page, root=root, groups=groups, prefix=prefix, forks=forks,
                tail_lo=tail[0], tail_hi=tail[1], queries=queries, idle=idle, **shape, **more)


def _cache(op, fmt, shape, page, layers, **more):
    return dict(op=op, fmt=fmt, page=page, layers=layers, kv_heads=shape["kv_heads"], head_dim=shape["head_dim"], **more)


def listed():
    return [
        # the first tokens of a single chat: all latency
        _attend("f16", LLAMA_1B, 64, 1, 1, tail=(37, 37), name="attend_1x37"),
        # eight answers to one prompt of ordinary length, a few tokens in
        _attend("f16", LLAMA_1B, 64, 1, 8, prefix=785, tail=(1, 60), name="attend_8_answers_785"),
        # a batch of unrelated chats of very different lengths
        _attend("f16", LLAMA_8B, 64, 16, 1, tail=(40, 8000), name="attend_16_chats_ragged"),
        # many questions about one long document
        _attend("f16", LLAMA_8B, 128, 1, 64, prefix=32768, tail=(1, 500), name="attend_64_document_32k"),
        # a system prompt, four prompts behind it, eight answers to each
        _attend("q8", LLAMA_8B, 64, 4, 8, root=2050, prefix=1500, tail=(1, 300), name="attend_tree_q8"),
        # eight prompts of 129 tokens behind a shared system prompt: their prefill
        _attend("f16", LLAMA_8B, 64, 1, 8, prefix=4000, tail=(129, 129), queries=129, name="attend_suffix_8x129"),
        # drafts of a speculative step on the smallest model, two slots empty
        _attend("f32", SMOL_135M, 32, 5, 1, tail=(9, 700), queries=4, idle=2, name="attend_drafts_f32"),
        # one decoded token for each of 64 sequences
        _cache("append", "f16", LLAMA_8B, 64, 1, rows=64, have_lo=3, have_hi=900, new_lo=1, new_hi=1,
               name="append_64x1"),
        # prompts that enter an 8-bit cache, odd lengths
        _cache("append", "q8", LLAMA_8B, 64, 1, rows=3, have_lo=0, have_hi=90, new_lo=309, new_hi=1201,
               name="append_prompts_q8"),
        # a prompt forked for four answers, the page at its end half full
        _cache("fork", "f16", LLAMA_1B, 64, 16, forks=3, have=741, name="fork_4_answers"),
        # a wide beam search's fork, all layers of the 8B shape
        _cache("fork", "f16", LLAMA_8B, 128, 32, forks=63, have=2135, name="fork_64_beams"),
        # a fragmented pool made dense again
        _cache("compact", "f16", LLAMA_8B, 64, 8, rows=12, lo=5, hi=2500, name="compact_12_rows"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    shape = rng.choice([SMOL_135M, LLAMA_1B, LLAMA_8B, _shape(8, 8, 128), _shape(14, 2, 64), _shape(40, 8, 128)])
    page = rng.choice([32, 64, 96, 128, 256])
    kind = rng.choice(["attend"] * 6 + ["append", "append", "fork", "compact"])
    if kind == "attend":
        fmt = rng.choice(["f16", "f16", "q8", "f32"])
        groups, forks = log(1, 12), log(1, 24)
        seqs = groups * forks
        queries = rng.choice([1, 1, 1, 2, log(2, 16), log(16, 160)])
        while groups * forks * queries > 1200:
            queries = max(1, queries // 2)
        root, prefix = rng.choice([0, log(20, 4000)]), rng.choice([0, log(20, 12000)])
        lo = log(queries, max(queries + 1, 400))
        hi = lo + log(1, 2000)
        # not over the largest listed case's reads or products
        while (groups * prefix + seqs * hi + root) * shape["kv_heads"] * shape["head_dim"] > 32 << 20 or \
                seqs * queries * (root + prefix + hi) * shape["heads"] * shape["head_dim"] > 8 << 30:
            root, prefix, hi = root // 2, prefix // 2, max(lo, hi // 2)
            if root + prefix == 0 and hi == lo:
                queries = max(1, queries // 2)
                lo = hi = max(queries, lo // 2)
        return _attend(fmt, shape, page, groups, forks, root=root, prefix=prefix, tail=(lo, hi), queries=queries,
                       idle=rng.choice([0, 0, rng.randint(1, 5)]))
    if kind == "append":
        rows, lo = log(1, 96), log(1, 60)
        hi = lo + log(1, max(2, 3000 // rows))
        return _cache(kind, rng.choice(["f16", "q8", "f32"]), shape, page, 1, rows=rows, have_lo=0, have_hi=log(1, 500),
                      new_lo=lo, new_hi=hi)
    fmt = rng.choice(["f16", "f32"])
    layers = log(1, 16)
    if kind == "fork":
        have = log(1, 1500)  # (at a page's end there would be nothing to copy)
        return _cache(kind, fmt, shape, page, layers, forks=log(1, 32), have=have + (have % page == 0))
    lo = log(1, 300)
    return _cache(kind, fmt, shape, page, min(layers, 8), rows=log(1, 12), lo=lo, hi=lo + log(1, 900))


# ---- sizes ----------------------------------------------------------------------


def _spread(i, lo, hi):
    """The i-th of some lengths between lo and hi, ragged and the same for every seed."""
    return lo + (i * 40503 + 977 * (i % 7)) % (hi - lo + 1)


def _tails(c):
    return [_spread(i + 1, max(c["tail_lo"], c["queries"]), max(c["tail_hi"], c["queries"]))
            for i in range(c["groups"] * c["forks"])]


def _append_sizes(c):
    have = [_spread(i + 1, c["have_lo"], c["have_hi"]) for i in range(c["rows"])]
    new = [_spread(i + 3, c["new_lo"], c["new_hi"]) for i in range(c["rows"])]
    return have, new


def _compact_lens(c):
    return [_spread(i + 1, c["lo"], c["hi"]) for i in range(c["rows"])]


def work(case):
    c = case
    token = 2 * c["kv_heads"] * c["head_dim"]  # keys and values of a token in one layer
    if c["op"] == "attend":
        tails = _tails(c)
        n = c["root"] + c["groups"] * c["prefix"] + sum(tails)
        rows = len(tails) * c["queries"] + c["idle"]
        seen = sum(c["root"] + c["prefix"] + t for t in tails) * c["queries"]
        seen -= len(tails) * c["queries"] * (c["queries"] - 1) // 2
        return {"bytes": n * token * BYTES[c["fmt"]] + 8.0 * rows * c["heads"] * c["head_dim"],
                "flops": 4.0 * seen * c["heads"] * c["head_dim"]}
    each = token * BYTES[c["fmt"]] * c["layers"]
    if c["op"] == "append":
        n = sum(_append_sizes(c)[1])
        back = n * token * (BYTES["q8"] + 4.0) if c["fmt"] == "q8" else 0.0  # read back as values
        return {"bytes": n * (each + 4.0 * token * c["layers"]) + back, "flops": 0.0}
    if c["op"] == "fork":
        return {"bytes": 2.0 * c["forks"] * max(1, c["have"] % c["page"]) * each, "flops": 0.0}
    return {"bytes": 6.0 * sum(_compact_lens(c)) * each, "flops": 0.0}


# ---- inputs ---------------------------------------------------------------------


def _normal(seed, k, *shape):
    """The k-th input of a seed."""
    g = torch.Generator("cuda")
    g.manual_seed(seed * 64 + k)
    return torch.randn(*shape, generator=g, device="cuda")


def _attend_inputs(c, seed):
    """Keys and values of the root, the prompts and the tails, and the queries."""
    nkv, D = c["kv_heads"], c["head_dim"]
    S, T = c["groups"] * c["forks"], max(_tails(c))
    kv = [(_normal(seed, 4 * n, *lead, nkv, D), _normal(seed, 4 * n + 1, *lead, nkv, D))
          for n, lead in enumerate([(c["root"],), (c["groups"], c["prefix"]), (S, T)])]
    return kv, _normal(seed, 63, S * c["queries"] + c["idle"], c["heads"], D)


def _append_inputs(c, seed):
    n = sum(_append_sizes(c)[1])
    return tuple(_normal(seed, i, c["layers"], n, c["kv_heads"], c["head_dim"]) for i in (0, 1))


def _round(x, d):
    return -(-x // d)


def _pool_pages(c):
    if c["op"] == "append":
        return sum(_round(h + n, c["page"]) for h, n in zip(*_append_sizes(c))) + 2
    if c["op"] == "fork":
        return _round(c["have"] + 1, c["page"]) + c["forks"] + 2
    return 3 * sum(_round(n, c["page"]) for n in _compact_lens(c))


def _seqs(c):
    return {"append": c.get("rows"), "fork": c.get("forks", 0) + 1, "compact": 3 * c.get("rows", 0)}[c["op"]]


def _max_len(c):
    return {"append": c.get("have_hi", 0) + c.get("new_hi", 0), "fork": c.get("have", 0) + 1, "compact": c.get("hi")}[c["op"]]


def _pool_fill(c, seed):
    """What a pool holds before a fork or a compaction."""
    nkv, D, P, N = c["kv_heads"], c["head_dim"], c["page"], _pool_pages(c)
    t = FORMATS[c["fmt"]]
    return (_normal(seed, 0, c["layers"], N, nkv, P, D).to(t), _normal(seed, 1, c["layers"], N, nkv, P // 32, D, 32).to(t))


# ---- plain forms: page layout -----------------------------------------------------


def _quantize(x):
    """32 channels to 8 bits with a binary16 scale: code = x * 127 / amax, halves away from zero."""
    b = x.unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    y = b * torch.where(amax > 0, 127.0 / amax, torch.zeros_like(amax))
    # (the largest number below a half: adding a half itself would round 0.49999997 up)
    code = torch.trunc(y + torch.copysign(torch.full_like(y, 0.49999997), y)).clamp(-127, 127)
    return code.reshape(x.shape).to(torch.int8), (amax / 127.0).squeeze(-1).to(torch.float16)


def _values(x, scale):
    if scale is None:
        return x.float()
    return (x.float().unflatten(-1, (-1, 32)) * scale.float().unsqueeze(-1)).flatten(-2)


def _v_rows(v):
    """[..., slot / 32, D, 32] to [..., slot, D]."""
    return v.transpose(-1, -2).flatten(-3, -2)


def _v_blocks(v):
    """[..., slot, D] to [..., slot / 32, D, 32]."""
    return v.unflatten(-2, (-1, 32)).transpose(-1, -2).contiguous()


def _pages_of(x, page):
    """[..., tokens, kv head, D] to [..., pages, kv head, slot, D], padded with zeros."""
    n = _round(x.shape[-3], page)
    x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, n * page - x.shape[-3]))
    return x.reshape(*x.shape[:-3], n, page, *x.shape[-2:]).transpose(-2, -3)


# ---- attention --------------------------------------------------------------------


def _attend_pool(c, seed):
    """The pages of all sequences, in shuffled order, and which hold what: the
    full pages of the root, the further full pages of each prompt, the rest of each
    sequence (the tables of the sequences differ from there on)."""
    P = c["page"]
    (kv_root, kv_group, kv_tail), q = _attend_inputs(c, seed)
    r, g = c["root"] // P, (c["root"] + c["prefix"]) // P - c["root"] // P
    lens = torch.tensor([c["root"] + c["prefix"] + t for t in _tails(c)], device="cuda")
    parts = []
    for root, group, tail in zip(kv_root, kv_group, kv_tail):
        group = torch.cat([root[r * P:].expand(c["groups"], *root[r * P:].shape), group], 1)
        tail = torch.cat([group[:, g * P:].repeat_interleave(c["forks"], 0), tail], 1)
        parts.append([_pages_of(x, P) for x in (root[: r * P], group[:, : g * P], tail)])
    shapes = [x.shape[:-3] for x in parts[0]]
    n = [math.prod(s) for s in shapes]
    order = torch.from_numpy(np.random.default_rng(seed).permutation(sum(n))).cuda()
    state = {"tables": [order[sum(n[:i]): sum(n[: i + 1])].reshape(s) for i, s in enumerate(shapes)], "q": q}
    for name, x in zip("kv", parts):
        flat = torch.cat([y.flatten(0, -4) for y in x])
        if c["fmt"] == "q8":
            code, scale = _quantize(flat)
        else:
            code, scale = flat.to(FORMATS[c["fmt"]]), None
        code = code if name == "k" else _v_blocks(code)
        state[name] = torch.empty_like(code).index_copy_(0, order, code)
        state[name + "s"] = None if scale is None else torch.empty_like(scale).index_copy_(0, order, scale)
    # tokens of the last segment that query t of a sequence sees
    back = torch.arange(c["queries"] - 1, -1, -1, device="cuda")
    state["seen"] = (lens - (r + g) * P)[:, None] - back[None, :]
    return state


def _attend_plain(c, s):
    nkv, D, G, nq = c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"], c["queries"]
    S = c["groups"] * c["forks"]
    q = s["q"][: S * nq].reshape(S, nq, nkv, G, D).permute(0, 2, 1, 3, 4).reshape(S, nkv, nq * G, D) / math.sqrt(D)

    def gather(name, table, n):
        # [n, kv head, tokens, D]
        t = table.reshape(n, table.shape[-1])
        x = s[name][t] if name == "k" else _v_rows(s[name][t])
        return _values(x, None if s[name + "s"] is None else s[name + "s"][t]).transpose(1, 2).flatten(2, 3)

    def by(x, n):
        # the queries of n groups of sequences, each group as one batch: [n, kv head, rows, D]
        return x.unflatten(0, (n, S // n)).transpose(1, 2).flatten(2, 3)

    def back(x):
        return x.unflatten(2, (S // x.shape[0], nq * G)).transpose(1, 2).flatten(0, 1)

    scores = [back(torch.matmul(by(q, n), gather("k", t, n).transpose(2, 3)))
              for n, t in zip((1, c["groups"], S), s["tables"])]
    width = [x.shape[-1] for x in scores]
    hidden = torch.arange(width[2], device="cuda")[None, None, :] >= s["seen"][:, :, None]
    scores[2] = scores[2].masked_fill(hidden.repeat_interleave(G, 1)[:, None], -math.inf)
    p = torch.cat(scores, -1)
    p = torch.exp(p - p.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = sum(back(torch.matmul(by(x, n), gather("v", t, n)))
            for n, t, x in zip((1, c["groups"], S), s["tables"], p.split(width, -1)))
    o = o.reshape(S, nkv, nq, G, D).permute(0, 2, 1, 3, 4).reshape(S * nq, c["heads"], D)
    return torch.cat([o, o.new_zeros(c["idle"], c["heads"], D)])


def _stored(fmt, x):
    """What a cache holds of x, in 64 bits (the codes of the 8-bit form are defined by 32-bit arithmetic)."""
    if fmt == "f32":
        return x.double()
    if fmt == "f16":
        return x.half().double()
    b = x.reshape(-1, 32)
    top = b.abs().max(1, keepdim=True).values
    y = b * (127.0 / top)
    code = torch.sign(y) * torch.floor(y.abs() + 0.5)
    return (code.double() * (top / 127.0).half().double()).reshape(x.shape)


def _attend_exact(c, seed):
    """Sequence by sequence in 64 bits, from the tokens themselves."""
    kv, q = _attend_inputs(c, seed)
    nkv, D, nq = c["kv_heads"], c["head_dim"], c["queries"]
    G = c["heads"] // nkv

    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for i, tail in enumerate(_tails(c)):
        k, v = (_stored(c["fmt"], torch.cat([kv[0][j], kv[1][j][i // c["forks"]], kv[2][j][i, :tail]])) for j in (0, 1))
        n = k.shape[0]
        rows = q[i * nq: (i + 1) * nq].double().reshape(nq, nkv, G, D)
        for h in range(nkv):
            a = torch.matmul(rows[:, h].reshape(nq * G, D), k[:, h].T.contiguous()) * D ** -0.5
            last = torch.arange(n - nq + 1, n + 1, device="cuda").repeat_interleave(G)
            a[torch.arange(n, device="cuda")[None] >= last[:, None]] = -math.inf
            o = torch.matmul(torch.softmax(a, 1), v[:, h].contiguous())
            out[i * nq: (i + 1) * nq].view(nq, nkv, G, D)[:, h] = o.reshape(nq, G, D)
    return out


# ---- append, fork, compact ----------------------------------------------------------


def _new_pages(held, first, last, page, taken):
    """Tables of sequences that grow from `first` to `last` tokens: each takes the
    free pages of lowest index in turn.  held: int32 [seqs, pages], -1 where none."""
    count = _ceil(last, page) - _ceil(first, page)
    free = np.flatnonzero(~taken)[: count.sum()]
    row = np.repeat(np.arange(len(count)), count)
    at = np.arange(count.sum()) - np.repeat(np.cumsum(count) - count, count) + np.repeat(_ceil(first, page), count)
    held = held.copy()
    held[row, at] = free
    return held


def _ceil(a, b):
    return -(-np.asarray(a) // b)


def _taken(table, pages):
    t = np.zeros(pages, bool)
    t[table[table >= 0]] = True
    return t


def _append_plain(c, s):
    P, nkv, D, N = c["page"], c["kv_heads"], c["head_dim"], _pool_pages(c)
    have, new = s["have"], s["new"]
    table = _new_pages(s["table"], have, have + new, P, _taken(s["table"], N))
    row = np.repeat(np.arange(len(new)), new)
    pos = np.arange(new.sum()) - np.repeat(np.cumsum(new) - new, new) + np.repeat(have, new)
    page = torch.from_numpy(table[row, pos // P].astype(np.int64)).cuda()
    slot = torch.from_numpy(pos % P).cuda()
    k, v = s["new_k"], s["new_v"]
    if c["fmt"] == "q8":
        (k, ks), (v, vs) = _quantize(k), _quantize(v)
        s["ks"][:, page, :, slot] = ks.transpose(0, 1)
        s["vs"][:, page, :, slot] = vs.transpose(0, 1)
    t = FORMATS[c["fmt"]]
    s["k"][:, page, :, slot] = k.transpose(0, 1).to(t)
    s["v"][:, page, :, slot // 32, :, slot % 32] = v.transpose(0, 1).to(t)
    out = {"table": torch.from_numpy(table), "len": torch.from_numpy((have + new).astype(np.int32))}
    if c["fmt"] == "q8":
        k = _values(s["k"][0, page, :, slot], s["ks"][0, page, :, slot])
        v = _values(s["v"][0, page, :, slot // 32, :, slot % 32], s["vs"][0, page, :, slot])
        return out | {"k": k, "v": v}
    return out | {"k": s["k"], "v": s["v"]}


def _blocks_plain(c, s, src, dst, blocks):
    """Copies the first blocks[i] 32-slot blocks of page src[i] to page dst[i], in all layers."""
    B = c["page"] // 32
    i = np.repeat(np.arange(len(blocks)), blocks)
    b = torch.from_numpy(np.arange(len(i)) - np.repeat(np.cumsum(blocks) - blocks, blocks)).cuda()
    at = [torch.from_numpy(np.asarray(x)[i].astype(np.int64)).cuda() for x in (src, dst)]
    for x in (s["k"].view(*s["k"].shape[:3], B, -1), s["v"].view(*s["v"].shape[:3], B, -1)):
        x[:, at[1], :, b] = x[:, at[0], :, b]


def _fork_plain(c, s):
    P, n, have = c["page"], c["forks"] + 1, c["have"]
    full, used = have // P, have % P
    table = np.full((n, _round(have + 1, P)), -1, np.int32)
    table[:, : _round(have, P)] = np.arange(_round(have, P))
    free = np.arange(_round(have, P), _round(have, P) + n, dtype=np.int32)
    if used:  # the forks take a page of their own each, the first sequence keeps the page
        table[1:, full] = free[:-1]
        _blocks_plain(c, s, np.full(n - 1, full), free[:-1], np.full(n - 1, _round(used, 32)))
    else:
        table[1:, full], table[0, full] = free[:-1], free[-1]
    return {"k": s["k"], "v": s["v"], "table": torch.from_numpy(table),
            "len": torch.from_numpy(np.full(n, have + 1, np.int32))}


def _compact_plain(c, s):
    P, lens = c["page"], np.array(_compact_lens(c))
    pages = _ceil(lens, P)
    U, first = pages.sum(), np.cumsum(pages) - pages
    row = np.repeat(np.arange(len(lens)), pages)
    at = np.arange(U) - first[row]
    blocks = _ceil(np.minimum(P, lens[row] - at * P), 32)
    # the second copies are made in reverse order
    order = np.argsort(-row, kind="stable")
    _blocks_plain(c, s, np.arange(U), U + np.arange(U), blocks)
    _blocks_plain(c, s, order, 2 * U + np.arange(U), blocks[order])
    _blocks_plain(c, s, 2 * U + np.arange(U), U + np.arange(U), blocks[order])
    n = len(lens)
    table = np.full((3 * n, _round(_max_len(c), P)), -1, np.int32)
    table[row, at] = np.arange(U)
    table[2 * n + row[order], at[order]] = U + np.arange(U)
    return {"k": s["k"], "v": s["v"], "table": torch.from_numpy(table),
            "len": torch.from_numpy(np.concatenate([lens, 0 * lens, lens]).astype(np.int32))}


def _cache_exact(c, seed):
    """The pages after the pass, page by page, in 64 bits."""
    P, D = c["page"], c["head_dim"]
    if c["op"] == "append":
        have, new = _append_sizes(c)
        if c["fmt"] == "q8":
            k, v = (_stored("q8", x[0]) for x in _append_inputs(c, seed))
            return {"k": k, "v": v, "table": None, "len": None}
        k, v = (x.double() for x in _append_inputs(c, seed))
        N = _pool_pages(c)
        out = {"k": k.new_zeros(c["layers"], N, c["kv_heads"], P, D),
               "v": k.new_zeros(c["layers"], N, c["kv_heads"], P // 32, D, 32)}
        free = sum(_round(h, P) for h in have)
        first, t = 0, 0
        for h, n in zip(have, new):
            held = list(range(first, first + _round(h, P)))
            first += len(held)
            for j in range(h, h + n):
                if j // P == len(held):
                    held.append(free)
                    free += 1
                out["k"][:, held[j // P], :, j % P] = k[:, t]
                out["v"][:, held[j // P], :, j % P // 32, :, j % 32] = v[:, t]
                t += 1
        return out | {"table": None, "len": None}
    k, v = (x.double() for x in _pool_fill(c, seed))

    def copy(a, b, slots):
        B = -(-slots // 32)
        k[:, b, :, : 32 * B] = k[:, a, :, : 32 * B]
        v[:, b, :, :B] = v[:, a, :, :B]

    if c["op"] == "fork":
        if c["have"] % P:
            for i in range(c["forks"]):
                copy(c["have"] // P, c["have"] // P + 1 + i, c["have"] % P)
    else:
        lens = _compact_lens(c)
        slots = [[min(P, n - P * i) for i in range(_round(n, P))] for n in lens]
        U = sum(map(len, slots))
        start = [sum(map(len, slots[:i])) for i in range(len(slots))]
        flat = [x for s in slots for x in s]
        for i in range(U):
            copy(i, U + i, flat[i])
        back = [(start[r] + i, slots[r][i]) for r in reversed(range(len(lens))) for i in range(len(slots[r]))]
        for to, (a, n) in enumerate(back):
            copy(a, 2 * U + to, n)
            copy(2 * U + to, U + to, n)
    return {"k": k, "v": v, "table": None, "len": None}


def exact(case, seed):
    if case["op"] == "attend":
        return _attend_exact(case, seed)
    return _cache_exact(case, seed)


# ---- the framework's operators --------------------------------------------------------


_held = {}


def _backend():
    from flarellm_amd.backend import HipBackend

    if "backend" not in _held:
        _held["backend"] = HipBackend(0)
    return _held["backend"]


def _paged(c, layers, pages, seqs, max_len):
    from flarellm_amd import FL_KV_F16, FL_KV_F32, FL_KV_Q8
    from flarellm_amd.pages import PagedKv

    fmt = {"f32": FL_KV_F32, "f16": FL_KV_F16, "q8": FL_KV_Q8}[c["fmt"]]
    return PagedKv(_backend(), layers=layers, pages=pages, page_size=c["page"], kv_heads=c["kv_heads"],
                   head_dim=c["head_dim"], kv_format=fmt, max_seqs=seqs, max_len=max_len)


def _attend_own(c, seed):
    """The sequences as a serving program makes them: root, forks, prompts, forks, tails."""
    (root, group, tail), q = _attend_inputs(c, seed)
    G, F, P, tails = c["groups"], c["forks"], c["page"], _tails(c)
    S = G * F
    longest = c["root"] + c["prefix"] + max(tails)
    pages = _round(c["root"], P) + G * (_round(c["prefix"], P) + 1) + sum(_round(t, P) + 1 for t in tails)
    kv = _paged(c, 1, pages, S + c["idle"], longest)
    if c["root"]:
        kv.extend([0], [c["root"]])
        kv.write(root[0], root[1])
    heads = [g * F for g in range(G)]
    kv.fork([0] * (G - 1), heads[1:])
    if c["prefix"]:
        kv.extend(heads, [c["prefix"]] * G)
        kv.write(*(x.flatten(0, 1) for x in group))
    kv.fork([g * F for g in range(G) for _ in range(1, F)], [g * F + f for g in range(G) for f in range(1, F)])
    kv.extend(list(range(S)), tails)
    kv.write(*(torch.cat([x[i, :t] for i, t in enumerate(tails)]) for x in tail))
    lens = np.array([c["root"] + c["prefix"] + t for t in tails], np.int32)
    back = np.arange(c["queries"] - 1, -1, -1, dtype=np.int32)
    seqs = np.concatenate([np.repeat(np.arange(S), c["queries"]), np.arange(S, S + c["idle"])]).astype(np.int32)
    seen = np.concatenate([(lens[:, None] - back[None]).ravel(), np.zeros(c["idle"])]).astype(np.int32)
    return {"kv": kv, "q": q, "seqs": seqs, "seen": seen}


def _cache_own(c, seed):
    kv = _paged(c, c["layers"], _pool_pages(c), _seqs(c), _max_len(c))
    s = {"kv": kv}
    if c["op"] == "append":
        have, new = _append_sizes(c)
        kv.k.zero_(), kv.v.zero_()
        rows = np.arange(c["rows"], dtype=np.int32)
        kv.extend(rows, np.array(have, np.int32))
        s |= dict(zip(("new_k", "new_v"), _append_inputs(c, seed)), rows=rows, have=np.array(have, np.int32),
                  new=np.array(new, np.int32))
        return s
    k, v = _pool_fill(c, seed)
    kv.k.copy_(k), kv.v.copy_(v)
    if c["op"] == "fork":
        kv.extend([0], [c["have"]])
        n = c["forks"] + 1
        ids = np.arange(n, dtype=np.int32)
        return s | {"src": 0 * ids[1:], "dst": ids[1:], "all": np.roll(ids, -1), "one": np.ones(n, np.int32)}
    n = c["rows"]
    kv.extend(np.arange(n, dtype=np.int32), _compact_lens(c))
    ids = np.arange(3 * n, dtype=np.int32).reshape(3, n)
    return s | {"src": ids[0], "one": ids[1], "two": ids[2], "back": np.ascontiguousarray(ids[0, ::-1]),
                "two_back": np.ascontiguousarray(ids[2, ::-1])}


def _run_own(c, s):
    kv = s["kv"]
    with torch.cuda.stream(kv.stream):  # the program's work is on the backend's stream
        if c["op"] == "attend":
            return kv.attention(s["q"], s["seqs"], s["seen"])
        if c["op"] == "append":
            kv.extend(s["rows"], s["new"])
            kv.write(s["new_k"], s["new_v"])
            out = {"table": torch.from_numpy(kv.tables()), "len": torch.from_numpy(kv.lens())}
            if c["fmt"] == "q8":
                out["k"], out["v"] = kv.read(s["rows"], s["have"], s["new"])
            else:
                out["k"], out["v"] = kv.k, kv.v
            kv.truncate(s["rows"], s["have"])
            return out
        if c["op"] == "fork":
            kv.fork(s["src"], s["dst"])
            kv.extend(s["all"], s["one"])
            out = {"table": torch.from_numpy(kv.tables()), "len": torch.from_numpy(kv.lens()), "k": kv.k, "v": kv.v}
            kv.free(s["dst"])
            kv.truncate([0], [c["have"]])
            return out
        kv.copy(s["src"], s["one"])
        kv.copy(s["back"], s["two_back"])
        kv.free(s["one"])
        kv.compact()
        out = {"table": torch.from_numpy(kv.tables()), "len": torch.from_numpy(kv.lens()), "k": kv.k, "v": kv.v}
        kv.free(s["two"])
        return out


# ---- what the tools call ------------------------------------------------------------------


def prepare(case, seed):
    c = case
    if own:
        return {"case": c} | (_attend_own(c, seed) if c["op"] == "attend" else _cache_own(c, seed))
    if c["op"] == "attend":
        return {"case": c} | _attend_pool(c, seed)
    s = {"case": c}
    if c["op"] != "append":
        s["k"], s["v"] = _pool_fill(c, seed)
        return s
    P, N, nkv, D = c["page"], _pool_pages(c), c["kv_heads"], c["head_dim"]
    have, new = (np.array(x) for x in _append_sizes(c))
    empty = np.full((c["rows"], _round(_max_len(c), P)), -1, np.int32)
    s |= {"have": have, "new": new, "table": _new_pages(empty, 0 * have, have, P, np.zeros(N, bool))}
    s["new_k"], s["new_v"] = _append_inputs(c, seed)
    t = FORMATS[c["fmt"]]
    s["k"] = torch.zeros(c["layers"], N, nkv, P, D, dtype=t, device="cuda")
    s["v"] = torch.zeros(c["layers"], N, nkv, P // 32, D, 32, dtype=t, device="cuda")
    if c["fmt"] == "q8":
        s["ks"], s["vs"] = (torch.zeros(c["layers"], N, nkv, P, D // 32, dtype=torch.float16, device="cuda") for _ in "kv")
    return s


def run(state):
    c = state["case"]
    if own:
        return _run_own(c, state)
    return {"attend": _attend_plain, "append": _append_plain, "fork": _fork_plain, "compact": _compact_plain}[c["op"]](c, state)
