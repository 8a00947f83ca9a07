"""The operators over several sequences behind page tables, as they are measured: the rows' norm, rotary and append, the
attention of prompts, single tokens and draft trees over the cache, the bookkeeping of the cache's pages, and the log
probabilities of given tokens.

A case is a dict of plain values; "lens" and "ctx" are the sequences' new rows and the positions they hold already.
`prepare` makes what a program has in hand (activations, caches, tables, logits; on the GPU, from the seed), `run` is one
pass: elementary torch operations, or the library's entry points where `own` is true.
"""
import math

import numpy as np
import torch

own = False

PAGE = 64   # cache rows a page
NROT, ROPE_BASE, EPS = 64, 1e7, 1e-6
BIG = {"nq": 24, "nkv": 4, "hd": 256}     # the benchmark configurations' attention heads
SMALL = {"nq": 8, "nkv": 2, "hd": 128}    # the narrower heads of the tests
EVEN = {"nq": 16, "nkv": 2, "hd": 256}
HEADS = [BIG, BIG, SMALL, EVEN]
VOCAB = 151936
MOST_FLOPS = 4 * 24 * 256 * 8192 * 8193 // 2
MOST_SCORES = 8192 * 8192 * 24
MOST_BYTES = 4 * 2000 * VOCAB
DEV = "cuda"


# ---------------------------------------------------------------- the cases
def listed():
    many = lambda v: ",".join(str(x) for x in v)   # noqa: E731
    return [
        # six conversations' draft trees of 16 nodes enter the cache: the smallest of the attention path's calls
        {"name": "append_6_trees", "op": "append", "tree": True, **BIG, "lens": many([16] * 6), "ctx": "4000,129,16383,800,12288,7001", "twist": 1},
        # a batch of prompts, one of them long
        {"name": "append_prompts_5301", "op": "append", "tree": False, **BIG, "lens": "37,4096,1,1167", "ctx": "0,0,511,64", "twist": 0},
        # one long prompt from its first token
        {"name": "prompt_8192", "op": "prompt", **BIG, "lens": "8192", "ctx": "0"},
        # short prompts of very different lengths in one call, the narrower heads
        {"name": "prompts_packed_ragged", "op": "prompt", **SMALL, "lens": "1,17,1500,130,777,300,1029,64", "ctx": "0,0,0,0,0,0,0,0"},
        # a chunk of a long prompt after 31 000 positions that are in the cache
        {"name": "prompt_chunk_1000_after_31k", "op": "prompt", **BIG, "lens": "1000", "ctx": "31000"},
        # plain decoding: one new token for each of twelve conversations
        {"name": "decode_12_sequences", "op": "prompt", **BIG, "lens": many([1] * 12),
         "ctx": "517,30011,4096,12000,63,8191,20000,1025,16384,2500,9999,28000"},
        # one conversation's tree of 16 drafts
        {"name": "tree_16_at_3000", "op": "tree", **BIG, "lens": "16", "ctx": "3000", "twist": 1},
        # six conversations, trees of different sizes over long contexts
        {"name": "trees_6_at_16k", "op": "tree", **BIG, "lens": "40,24,64,33,9,63", "ctx": "16384,20001,9000,30000,16000,12345", "twist": 2},
        # eight samples of one prompt: the tables are shared, the page that they go on in is copied
        {"name": "pages_fork_8", "op": "pages", "fork": True, **BIG, "planes": 24, "lens": "24,24,24,24,24,24,24,24", "ctx": "4130,0,0,0,0,0,0,0", "twist": 0},
        # after a tree window: the accepted path's rows move together, the pages behind them are free again
        {"name": "pages_keep_paths_32", "op": "pages", "fork": False, **BIG, "planes": 4, "lens": many([48] * 32),
         "ctx": many([(997 * i * i) % 2000 + 1 for i in range(32)]), "twist": 3},
        # a window's rows at the whole vocabulary, twenty alternatives each
        {"name": "logprobs_16_rows", "op": "logprobs", "rows": 16, "vocab": VOCAB, "k": 20, "masked": 0.0},
        # a prompt is scored: every row's token, five alternatives, part of the vocabulary masked out
        {"name": "logprobs_prompt_2000", "op": "logprobs", "rows": 2000, "vocab": VOCAB, "k": 5, "masked": 0.3},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _fits(c):
    lens, ctx = _ints(c["lens"]), _ints(c["ctx"])
    scores = len(lens) * max(lens) * max(a + b for a, b in zip(lens, ctx)) * c["nq"]
    w = work(c)
    return scores <= MOST_SCORES and w["flops"] <= MOST_FLOPS and w["bytes"] <= MOST_BYTES and sum(lens) + sum(ctx) <= 300000


def draw(rng):
    op = rng.choice(["append", "prompt", "prompt", "prompt", "tree", "tree", "pages", "logprobs"])
    many = lambda v: ",".join(str(x) for x in v)   # noqa: E731
    if op == "logprobs":
        return {"op": op, "rows": _log(rng, 1, 2000), "vocab": rng.choice([VOCAB, 32768, rng.randrange(20000, 150000)]), "k": rng.choice([0, 1, 5, 20, 64]),
                "masked": rng.choice([0.0, 0.3, 0.95])}
    heads = rng.choice(HEADS)
    if op == "pages":
        n, fork = _log(rng, 2, 64), rng.random() < 0.5
        lens = [rng.randrange(1, 65) for _ in range(n)]
        ctx = [_log(rng, 1, 6000)] + [0] * (n - 1) if fork else [_log(rng, 1, 3000) for _ in range(n)]
        return {"op": op, "fork": fork, **heads, "planes": rng.choice([2, 4, 8]), "lens": many(lens), "ctx": many(ctx), "twist": rng.randrange(1, 6)}
    while True:
        n = _log(rng, 1, 24)
        if op == "tree":
            lens, ctx = [rng.randrange(1, 65) for _ in range(n)], [_log(rng, 1, 40000) for _ in range(n)]
        elif op == "append":
            lens, ctx = [_log(rng, 1, 4000) for _ in range(n)], [rng.choice([0, _log(rng, 1, 30000)]) for _ in range(n)]
        elif rng.random() < 0.4:
            lens, ctx = [1] * n, [_log(rng, 1, 60000) for _ in range(n)]
        else:
            lens, ctx = [_log(rng, 1, 6000) for _ in range(n)], [rng.choice([0, 0, _log(rng, 1, 30000)]) for _ in range(n)]
        c = {"op": op, **heads, "lens": many(lens), "ctx": many(ctx)}
        if op == "append":
            c["tree"] = rng.random() < 0.3
            if c["tree"]:
                c["lens"] = many([min(x, 64) for x in lens])
        if op in ("append", "tree"):
            c["twist"] = rng.randrange(1, 6)
        if _fits(c):
            return c


def _ints(text):
    return [int(x) for x in text.split(",")]


def _parents(n, twist):
    """A draft tree of n nodes in the order of their making: node 0 is the committed token."""
    return [-1] + [max(0, i - 1 - (i * i + 3 * i * twist) % 6) for i in range(1, n)]


def _depths(parent):
    d = []
    for p in parent:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def _path(parent):
    """The accepted path: from the root to the newest node."""
    path, i = [], len(parent) - 1
    while i >= 0:
        path.append(i)
        i = parent[i]
    return path[::-1]


def work(case):
    if case["op"] == "logprobs":
        T, n, k = case["rows"], case["vocab"], case["k"]
        return {"bytes": 4 * T * n + T * (4 + 12) + 8 * T * k, "flops": 5 * T * n}
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    lens, ctx = _ints(case["lens"]), _ints(case["ctx"])
    rows = sum(lens)
    if case["op"] == "append":
        return {"bytes": rows * (4 * nq * hd + 8 * nkv * hd + 2 * nq * hd + 4 * nkv * hd), "flops": rows * 6 * (nq + nkv) * hd}
    if case["op"] == "pages":
        row, n = 2 * nkv * hd, len(lens)
        if case["fork"]:   # one of the holders keeps the page
            moved = (ctx[0] % PAGE) * (n - 1)
            tables = 2 * n * -(-ctx[0] // PAGE)
        else:
            moved = sum(sum(1 for i, x in enumerate(_path(_parents(m, case["twist"]))) if x != i) for m in lens)
            tables = 2 * sum(-(-(a + b) // PAGE) for a, b in zip(lens, ctx))
        return {"bytes": 2 * moved * row * case["planes"] + 4 * tables, "flops": 0}
    if case["op"] == "tree":
        seen = sum(m * x + sum(d + 1 for d in _depths(_parents(m, case["twist"]))) for m, x in zip(lens, ctx))
    else:
        seen = sum(m * x + m * (m + 1) // 2 for m, x in zip(lens, ctx))
    kv = sum(m + x for m, x in zip(lens, ctx))
    return {"bytes": rows * nq * hd * (2 + 4 + 2) + kv * nkv * hd * 4, "flops": 4 * nq * hd * seen}


# ---------------------------------------------------------------- what a program has in hand
def _dev(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    normal = lambda *shape, dtype=torch.float32: torch.randn(*shape, device=DEV, dtype=dtype, generator=g)   # noqa: E731
    s = {"case": dict(case)}
    if case["op"] == "logprobs":
        T, n, k = case["rows"], case["vocab"], case["k"]
        x = normal(T, n) * 3.0
        pick = torch.argmax(x - torch.log(-torch.log(torch.rand(T, n, device=DEV, generator=g).clamp_(1e-6, 1 - 1e-6))), dim=1)
        if case["masked"]:   # a grammar leaves part of the vocabulary out, never the token that was taken
            out = torch.rand(n, device=DEV, generator=g) < case["masked"]
            keep = x.gather(1, pick[:, None])
            x.masked_fill_(out[None, :], -math.inf)
            x.scatter_(1, pick[:, None], keep)
        s.update(logits=x, tok=pick.to(torch.int32)[:, None].contiguous())
        s["out"] = {"lse": torch.empty(T, device=DEV), "entropy": torch.empty(T, device=DEV), "lp": torch.empty(T, 1, device=DEV),
                    "top_lp": torch.empty(T, k, device=DEV), "top_i": torch.empty(T, k, dtype=torch.int32, device=DEV)}
        s["err"] = torch.zeros(1, dtype=torch.int32, device=DEV)
        return s
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    lens, ctx = _ints(case["lens"]), _ints(case["ctx"])
    n, rows = len(lens), sum(lens)
    if case["op"] == "pages":
        ends = [(ctx[0] if case["fork"] else x) + m for m, x in zip(lens, ctx)]
        width = max(-(-e // PAGE) for e in ends) + 1
        held = [-(-x // PAGE) for x in ctx]
        npages = (held[0] + sum(-(-m // PAGE) + 1 for m in lens) if case["fork"] else sum(-(-e // PAGE) for e in ends)) + 9
    else:
        ends = [m + x for m, x in zip(lens, ctx)]
        width = max(-(-e // PAGE) for e in ends)
        held = [-(-e // PAGE) for e in ends]
        npages = sum(held) + 3
    ids = torch.randperm(npages, device=DEV, generator=g).to(torch.int32)   # pages lie in no order
    pt, at = torch.full((n, width), -1, dtype=torch.int32, device=DEV), 0
    for i, h in enumerate(held):
        pt[i, :h] = ids[at:at + h]
        at += h
    s.update(rows=rows, pt=pt, npages=npages, max_pos=max(ends), max_len=max(lens), err=torch.zeros(1, dtype=torch.int32, device=DEV))
    if case["op"] == "pages":
        ref = torch.zeros(npages, dtype=torch.int32, device=DEV)
        ref[ids[:at].long()] = 1
        paths = [_path(_parents(m, case["twist"])) for m in lens]
        wide = max(len(p) for p in paths)
        s.update(ref=ref, len=_dev(ctx), add=_dev(lens), pos0=torch.zeros(n, dtype=torch.int32, device=DEV),
                 row0=torch.zeros(n + 1, dtype=torch.int32, device=DEV), lim=_dev([ctx[0]] * n if case["fork"] else ctx),
                 source=_dev([0] * n if case["fork"] else list(range(n))), keep=_dev([p + [0] * (wide - len(p)) for p in paths]),
                 nkeep=_dev([len(p) for p in paths]), planes=normal(case["planes"], npages + 1, PAGE, nkv * hd, dtype=torch.float16))
        s["bases"] = _dev([s["planes"][i].data_ptr() for i in range(case["planes"])], torch.int64)
        return s
    s.update(row0=_dev([0] + list(np.cumsum(lens))), pos0=_dev(ctx), qg=normal(rows, nq, 2 * hd),
             kc=normal(npages, PAGE, nkv * hd, dtype=torch.float16), vc=normal(npages, PAGE, nkv * hd, dtype=torch.float16))
    if case["op"] == "append":
        s.update(k=normal(rows, nkv, hd) * 2.0, v=normal(rows, nkv, hd), qn=1.0 + 0.1 * normal(hd), kn=1.0 + 0.1 * normal(hd),
                 q16=torch.empty(rows, nq, hd, dtype=torch.float16, device=DEV))
    else:
        s.update(q16=normal(rows, nq, hd).to(torch.float16), out=torch.empty(rows, nq, hd, dtype=torch.float16, device=DEV))
    if case.get("tree", case["op"] == "tree"):
        words = -(-max(lens) // 32)
        parents = [_parents(m, case["twist"]) for m in lens]
        s["parent"] = _dev([p for t in parents for p in t])
        s["words"] = words
        if case["op"] == "tree":   # masks are made once for a window's layers
            bits = np.zeros((rows, words), np.uint32)
            for r0, t in zip([0] + list(np.cumsum(lens)), parents):
                for i, p in enumerate(t):
                    if p >= 0:
                        bits[r0 + i] = bits[r0 + p]
                    bits[r0 + i, i // 32] |= np.uint32(1 << (i % 32))
            s["anc"] = torch.from_numpy(bits.view(np.int32)).to(DEV)
        else:
            s.update(anc=torch.empty(rows, words, dtype=torch.int32, device=DEV), depth=torch.empty(rows, dtype=torch.int32, device=DEV))
    return s


# ---------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "prompt": _own_attn, "tree": _own_attn, "pages": _own_pages, "logprobs": _own_logprobs}[op](state)
    return {"append": _append, "prompt": _attn, "tree": _attn, "pages": _pages, "logprobs": _logprobs}[op](state)


def _slots(s):
    """Every row's sequence, its place in it, and the cache row where its position lies."""
    t = torch.arange(s["rows"], device=DEV)
    seq = torch.searchsorted(s["row0"].long()[1:].contiguous(), t, right=True)
    i = t - s["row0"].long()[seq]
    pos = s["pos0"].long()[seq] + i
    return seq, i, s["pt"].long()[seq, pos // PAGE] * PAGE + pos % PAGE


def _masks(s, seq, i):
    """Ancestor bits and depths of the trees: the closure of the parents' relation by repeated products."""
    n, rows, words = int(s["row0"].numel()) - 1, s["rows"], s["words"]
    A = torch.zeros(n, 32 * words, 32 * words, device=DEV)
    own_row = torch.arange(32 * words, device=DEV)
    A[:, own_row, own_row] = 1.0
    par = s["parent"].long()
    A[seq, i, torch.where(par >= 0, par, i)] = 1.0
    for _ in range(max(1, (s["max_len"] - 1).bit_length())):
        A = (torch.matmul(A, A) > 0).float()
    seen = A[seq, i]
    bits = (seen.long().view(rows, words, 32) << torch.arange(32, device=DEV)).sum(2)
    return torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).to(torch.int32), seen.sum(1).to(torch.int32) - 1


def _append(s):
    c = s["case"]
    nq, nkv, hd = c["nq"], c["nkv"], c["hd"]
    seq, i, slot = _slots(s)
    got = {}
    step = i
    if c["tree"]:
        got["anc"], got["depth"] = _masks(s, seq, i)
        step = got["depth"].long()
    # the angle is the product of the position and the pair's frequency in 32 bits, as the cache's other rows have it
    freq = torch.pow(torch.tensor(ROPE_BASE, dtype=torch.float64, device=DEV), -2.0 * torch.arange(NROT // 2, device=DEV, dtype=torch.float64) / NROT).float()
    theta = ((s["pos0"].long()[seq] + step).float()[:, None] * freq).double()
    cs, sn = torch.cos(theta).float()[:, None], torch.sin(theta).float()[:, None]

    def norm_rope(x, w):
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        a, b = y[..., :NROT // 2], y[..., NROT // 2:NROT]
        return torch.cat([a * cs - b * sn, b * cs + a * sn, y[..., NROT:]], dim=-1)

    s["q16"].copy_(norm_rope(s["qg"][..., :hd], s["qn"]))
    s["kc"].view(-1, nkv * hd)[slot] = norm_rope(s["k"], s["kn"]).view(-1, nkv * hd).to(torch.float16)
    s["vc"].view(-1, nkv * hd)[slot] = s["v"].view(-1, nkv * hd).to(torch.float16)
    got.update(q16=s["q16"], kc=s["kc"], vc=s["vc"])
    return got


def _attn(s):
    """The sequences side by side, each filled up to the longest."""
    c = s["case"]
    nq, nkv, hd = c["nq"], c["nkv"], c["hd"]
    n, most, top = int(s["pos0"].numel()), s["max_len"], s["max_pos"]
    row0, pos0 = s["row0"].long(), s["pos0"].long()
    have = row0[1:] - row0[:-1]
    i = torch.arange(most, device=DEV)
    rows = torch.clamp(row0[:-1, None] + i, max=s["rows"] - 1)
    p = torch.arange(top, device=DEV)
    live = p[None, :] < (pos0 + have)[:, None]
    cells = torch.where(live, s["pt"].long()[:, torch.div(p, PAGE, rounding_mode="floor")] * PAGE + p % PAGE, 0)
    k = s["kc"].view(-1, nkv, hd)[cells].float()
    v = torch.where(live[:, :, None, None], s["vc"].view(-1, nkv, hd)[cells].float(), 0.0)
    q = s["q16"][rows].float().view(n, most, nkv, nq // nkv, hd)
    x = torch.einsum("nthqd,nphd->nhqtp", q, k)
    x *= 1.0 / math.sqrt(hd)
    rel = p[None, None, :] - pos0[:, None, None]
    if c["op"] == "tree":
        at = rel.clamp(0, 32 * s["words"] - 1)
        word = torch.gather(s["anc"][rows].long(), 2, (at // 32).expand(n, most, top))
        seen = (rel < 0) | (((word >> (at % 32)) & 1) == 1)
    else:
        seen = rel <= i[None, :, None]
    seen = seen & live[:, None, :]
    x.masked_fill_(~seen[:, None, None], -math.inf)
    x -= x.amax(-1, keepdim=True)
    x.exp_()
    z = x.sum(-1)
    o = torch.einsum("nhqtp,nphd->nthqd", x, v) / z.permute(0, 3, 1, 2)[..., None]
    seq = torch.repeat_interleave(torch.arange(n, device=DEV), have, output_size=s["rows"])
    mine = torch.arange(s["rows"], device=DEV) - row0[seq]
    gate = s["qg"][..., hd:]
    s["out"].copy_(o.reshape(n, most, nq, hd)[seq, mine] / (1.0 + torch.exp(-gate)))
    return s["out"]


def _held(length):
    return torch.div(length + PAGE - 1, PAGE, rounding_mode="floor")


def _count(s, pt, used):
    """How many entries of the tables name each page."""
    at = torch.where(used, pt.long(), s["npages"]).view(-1)
    return torch.zeros(s["npages"] + 1, dtype=torch.int64, device=DEV).scatter_add_(0, at, torch.ones_like(at))[:-1].to(torch.int32)


def _pages(s):
    c = s["case"]
    n, width = s["pt"].shape
    col = torch.arange(width, device=DEV)
    rows_w = c["nkv"] * c["hd"]
    planes = s["planes"]
    # the tables of the sequences that are gone on from, cut to their lengths
    source = s["source"].long()
    new_len = torch.minimum(s["len"].long()[source], s["lim"].long())
    used = col < _held(new_len)[:, None]
    pt = torch.where(used, s["pt"][source], -1)
    ref = s["ref"] + _count(s, pt, used) - _count(s, s["pt"], s["pt"] >= 0)
    # room for the new rows: a shared page that is gone on in is copied, unless all its holders go on and this is the first
    add = s["add"].long()
    pos0 = new_len
    end = pos0 + add
    tail = (pos0 % PAGE != 0) & (add > 0)
    at = torch.clamp(torch.div(pos0, PAGE, rounding_mode="floor"), max=width - 1)
    page = torch.where(tail, pt.long().gather(1, at[:, None])[:, 0], -1)
    same = (page[:, None] == page[None, :]) & tail[:, None] & tail[None, :]
    rank = torch.tril(same, -1).sum(1)
    copy = tail & ((ref.long()[page.clamp(min=0)] > same.sum(1)) | (rank > 0))
    h0, h1 = _held(pos0), _held(end)
    want = h1 - h0 + copy.long()
    off = torch.cumsum(want, 0) - want
    free = torch.sort(torch.where(ref == 0, torch.arange(s["npages"], device=DEV), s["npages"])).values
    fresh = (col >= h0[:, None]) & (col < h1[:, None])
    mine = (off + copy.long())[:, None] + col - h0[:, None]
    pt = torch.where(fresh, free[mine.clamp(0, s["npages"] - 1)].to(torch.int32), pt)
    dst = torch.where(copy, free[off.clamp(max=s["npages"] - 1)], s["npages"])
    moved = (col == at[:, None]) & copy[:, None]
    pt = torch.where(moved, dst[:, None].to(torch.int32), pt)
    dump = torch.where(copy, page, s["npages"])
    ref = ref + _count(s, pt, fresh | moved) - torch.zeros(s["npages"] + 1, dtype=torch.int64, device=DEV).scatter_add_(
        0, dump, torch.ones_like(dump))[:-1].to(torch.int32)
    below = torch.arange(PAGE, device=DEV)[None, :, None] < (pos0 % PAGE)[:, None, None]
    planes[:, dst] = torch.where(below, planes[:, dump], planes[:, dst])
    if not c["fork"]:   # the accepted paths' rows move together; the pages behind them go
        keep, nkeep = s["keep"].long(), s["nkeep"].long()
        i = torch.arange(keep.shape[1], device=DEV)
        ok = i < nkeep[:, None]
        a, b = pos0[:, None] + keep, pos0[:, None] + i
        cell = lambda p: torch.where(ok, pt.long().gather(1, (p // PAGE).clamp(max=width - 1)) * PAGE + p % PAGE, s["npages"] * PAGE)   # noqa: E731
        flat = planes.view(planes.shape[0], -1, rows_w)
        flat[:, cell(b)] = flat[:, cell(a)]
        end = pos0 + nkeep
        gone = (col >= _held(end)[:, None]) & (pt >= 0)
        ref = ref - _count(s, pt, gone)
        pt = torch.where(gone, -1, pt)
    s["pt"].copy_(pt)
    s["ref"].copy_(ref)
    s["len"].copy_(end)
    s["pos0"].copy_(pos0)
    s["row0"][1:].copy_(torch.cumsum(add, 0))
    return _page_outputs(s)


def _page_outputs(s):
    return {"pt": s["pt"], "ref": s["ref"], "len": s["len"], "pos0": s["pos0"], "row0": s["row0"], "planes": s["planes"][:, :s["npages"]]}


def _logprobs(s):
    x, k = s["logits"], s["case"]["k"]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(1)
    lse = m[:, 0] + torch.log(z)
    ent = torch.log(z) - torch.where(e > 0, e * (x - m), 0.0).sum(1) / z
    o = s["out"]
    o["lse"].copy_(lse)
    o["entropy"].copy_(ent)
    o["lp"].copy_(x.gather(1, s["tok"].long()) - lse[:, None])
    if k:   # ties to the lowest index: an order-preserving key of the value above the index's complement
        b = (x + 0.0).view(torch.int32).long()
        key = torch.where(b < 0, -(b & 0x7FFFFFFF) - 1, b) * 2 ** 32 + (2 ** 32 - 1 - torch.arange(x.shape[1], device=DEV))
        top = torch.topk(key, k, dim=1).values
        at = 2 ** 32 - 1 - (top & 0xFFFFFFFF)
        o["top_i"].copy_(at)
        o["top_lp"].copy_(x.gather(1, at) - lse[:, None])
    return o


# ---------------------------------------------------------------- the library's calls
def _lib():
    from sfnx_b200 import lib as L

    return L


def _seqs(s, L):
    """The sequences' struct, the pages' geometry and the workspace, made once."""
    if "seqs" not in s:
        c = s["case"]
        s["seqs"] = L.Seqs(int(s["pos0"].numel()), s["rows"], s["row0"].data_ptr(), s["pos0"].data_ptr(), s["pt"].data_ptr(), s["pt"].shape[1],
                           s["npages"], None, s["max_pos"])
        s["pages"] = L.KvPages(None, PAGE * c["nkv"] * c["hd"], PAGE, 0, 0)
        if c["op"] != "append":
            size = L.load().fnx_attn_seqs_scratch_bytes(L.byref(s["seqs"]), c["nq"], c["nkv"], c["hd"])
            s["scratch"] = torch.empty(max(1, size), dtype=torch.uint8, device=DEV)
    return s["seqs"], s["pages"]


def _own_append(s):
    L, c = _lib(), s["case"]
    sq, g = _seqs(s, L)
    got, st = {}, L.stream()
    if c["tree"]:
        L.call("fnx_tree_masks", s["parent"].data_ptr(), L.byref(sq), s["anc"].data_ptr(), s["words"], s["depth"].data_ptr(), s["err"].data_ptr(), st)
        got.update(anc=s["anc"], depth=s["depth"])
    L.call("fnx_attn_seqs_append", s["qg"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["qn"].data_ptr(), s["kn"].data_ptr(), s["kc"].data_ptr(),
           s["vc"].data_ptr(), g, L.byref(sq), L.ptr(s.get("depth")), s["q16"].data_ptr(), EPS, L.Rope(ROPE_BASE, NROT), c["nq"], c["nkv"], c["hd"],
           s["err"].data_ptr(), st)
    got.update(q16=s["q16"], kc=s["kc"], vc=s["vc"])
    return got


def _own_attn(s):
    L, c = _lib(), s["case"]
    sq, g = _seqs(s, L)
    nq, nkv, hd = c["nq"], c["nkv"], c["hd"]
    if c["op"] == "tree":
        L.call("fnx_attn_tree", s["q16"].data_ptr(), nq * hd, s["qg"].data_ptr(), s["kc"].data_ptr(), s["vc"].data_ptr(), g, L.byref(sq), s["anc"].data_ptr(),
               s["words"], s["out"].data_ptr(), nq * hd, nq, nkv, hd, s["scratch"].data_ptr(), L.stream())
    else:
        L.call("fnx_attn_prompt", s["q16"].data_ptr(), nq * hd, s["qg"].data_ptr(), s["kc"].data_ptr(), s["vc"].data_ptr(), g, L.byref(sq),
               s["out"].data_ptr(), nq * hd, nq, nkv, hd, s["scratch"].data_ptr(), L.stream())
    return s["out"]


def _own_pages(s):
    L, c = _lib(), s["case"]
    n, width = s["pt"].shape
    if "pool" not in s:
        s["pool"] = L.PagePool(s["npages"], PAGE, s["ref"].data_ptr(), n, s["pt"].data_ptr(), width, s["len"].data_ptr())
        s["pages"] = L.KvPages(None, PAGE * c["nkv"] * c["hd"], PAGE, 0, 0)
        s["scratch"] = torch.zeros(L.load().fnx_pages_scratch_bytes(L.byref(s["pool"])), dtype=torch.uint8, device=DEV)
    pool, g, scratch, err, st = L.byref(s["pool"]), s["pages"], s["scratch"].data_ptr(), s["err"].data_ptr(), L.stream()
    L.call("fnx_pages_fork", pool, s["source"].data_ptr(), s["lim"].data_ptr(), scratch, err, st)
    L.call("fnx_pages_reserve", pool, s["add"].data_ptr(), s["pos0"].data_ptr(), s["row0"].data_ptr(), s["bases"].data_ptr(), c["planes"], g, c["nkv"], c["hd"],
           scratch, err, st)
    if not c["fork"]:
        L.call("fnx_pages_keep", pool, s["pos0"].data_ptr(), s["keep"].data_ptr(), s["keep"].shape[1], s["nkeep"].data_ptr(), s["bases"].data_ptr(), c["planes"],
               g, c["nkv"], c["hd"], scratch, err, st)
    return _page_outputs(s)


def _own_logprobs(s):
    L, c, o = _lib(), s["case"], s["out"]
    T, n = s["logits"].shape
    if "scratch" not in s:
        s["scratch"] = torch.zeros(L.load().fnx_logprobs_scratch_bytes(n, T, c["k"]), dtype=torch.uint8, device=DEV)
    L.call("fnx_logprobs", s["logits"].data_ptr(), n, n, T, 0, s["tok"].data_ptr(), 1, c["k"], o["lse"].data_ptr(), o["entropy"].data_ptr(), o["lp"].data_ptr(),
           o["top_lp"].data_ptr(), o["top_i"].data_ptr(), s["scratch"].data_ptr(), s["err"].data_ptr(), L.stream())
    return o


# ---------------------------------------------------------------- the definitions in 64 bits, sequence by sequence
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "prompt": _exact_attn, "tree": _exact_attn, "pages": _exact_pages, "logprobs": _exact_logprobs}[case["op"]](s)


def _exact_append(s):
    c = s["case"]
    nq, nkv, hd = c["nq"], c["nkv"], c["hd"]
    kc, vc, q16 = s["kc"].double(), s["vc"].double(), torch.empty(s["rows"], nq, hd, dtype=torch.float64, device=DEV)
    got, r0 = {}, 0
    anc, depth = [], []
    f = np.float32(np.power(np.float64(np.float32(ROPE_BASE)), -2.0 * np.arange(NROT // 2) / NROT))
    pt = s["pt"].cpu().numpy()
    for n, (m, x) in enumerate(zip(_ints(c["lens"]), _ints(c["ctx"]))):
        step = np.arange(m)
        if c["tree"]:
            par = _parents(m, c["twist"])
            step = np.array(_depths(par))
            for i in range(m):
                word, j = [0] * s["words"], i
                while j >= 0:
                    word[j // 32] |= 1 << (j % 32)
                    j = par[j]
                anc.append([w - 2 ** 32 if w >= 2 ** 31 else w for w in word])
            depth += step.tolist()
        theta = np.float64(np.float32(x + step)[:, None] * f[None, :])
        sn, cs = (torch.from_numpy(t).to(DEV)[:, None] for t in (np.sin(theta), np.cos(theta)))
        pos = x + np.arange(m)
        cell = torch.from_numpy(pt[n, pos // PAGE].astype(np.int64) * PAGE + pos % PAGE).to(DEV)

        def turned(y, w):
            y = y.double()
            y = y / torch.sqrt(torch.mean(y ** 2, -1, keepdim=True) + EPS) * w.double()
            h = NROT // 2
            z = y.clone()
            z[..., :h] = y[..., :h] * cs - y[..., h:NROT] * sn
            z[..., h:NROT] = y[..., :h] * sn + y[..., h:NROT] * cs
            return z

        q16[r0:r0 + m] = turned(s["qg"][r0:r0 + m, :, :hd], s["qn"])
        kc.view(-1, nkv, hd)[cell] = turned(s["k"][r0:r0 + m], s["kn"])
        vc.view(-1, nkv, hd)[cell] = s["v"][r0:r0 + m].double()
        r0 += m
    if c["tree"]:
        got.update(anc=torch.tensor(anc, dtype=torch.int32), depth=torch.tensor(depth, dtype=torch.int32))
    got.update(q16=q16, kc=kc, vc=vc)
    return got


def _exact_attn(s):
    c = s["case"]
    nq, nkv, hd = c["nq"], c["nkv"], c["hd"]
    out, r0 = torch.empty(s["rows"], nq, hd, dtype=torch.float64, device=DEV), 0
    for n, (m, x) in enumerate(zip(_ints(c["lens"]), _ints(c["ctx"]))):
        pages = s["pt"][n, :-(-(m + x) // PAGE)].long()
        K, V = (t[pages].reshape(-1, nkv, hd)[:m + x].double() for t in (s["kc"], s["vc"]))
        if c["op"] == "tree":
            par = _parents(m, c["twist"])
            tail = np.zeros((m, m), bool)
            for i in range(m):
                j = i
                while j >= 0:
                    tail[i, j] = True
                    j = par[j]
            tail = torch.from_numpy(tail).to(DEV)
        else:
            tail = torch.ones(m, m, dtype=torch.bool, device=DEV).tril()
        for h in range(nq):
            w = s["q16"][r0:r0 + m, h].double() @ K[:, h // (nq // nkv)].T / math.sqrt(hd)
            w[:, x:].masked_fill_(~tail, -math.inf)
            out[r0:r0 + m, h] = torch.softmax(w, dim=1) @ V[:, h // (nq // nkv)]
        out[r0:r0 + m] *= torch.sigmoid(s["qg"][r0:r0 + m, :, hd:].double())
        r0 += m
    return out


def _exact_pages(s):
    c = s["case"]
    lens, ctx, npages = _ints(c["lens"]), _ints(c["ctx"]), s["npages"]
    n, width = s["pt"].shape
    pt, planes = s["pt"].cpu().numpy(), s["planes"]
    up = lambda x: -(-x // PAGE)   # noqa: E731
    tables = [list(pt[0][:up(ctx[0])]) if c["fork"] else list(pt[i][:up(ctx[i])]) for i in range(n)]
    pos0 = [ctx[0]] * n if c["fork"] else list(ctx)
    ref = np.zeros(npages, np.int64)
    for t in tables:
        for p in t:
            ref[p] += 1
    free = [p for p in range(npages) if ref[p] == 0]
    tails = [(i, tables[i][-1]) for i in range(n) if pos0[i] % PAGE and lens[i]]
    for i in range(n):
        if (i, tables[i][-1] if tables[i] else -1) in tails:
            p = tables[i][-1]
            holders = [j for j, q in tails if q == p]
            if ref[p] > 1 and (i != holders[0] or sum(p in t for t in tables) > len(holders)):
                new = free.pop(0)
                planes[:, new, :pos0[i] % PAGE] = planes[:, p, :pos0[i] % PAGE]
                tables[i] = tables[i][:-1] + [new]
                ref[new] = 1
        while len(tables[i]) < up(pos0[i] + lens[i]):
            new = free.pop(0)
            ref[new] = 1
            tables[i].append(new)
    end = [a + b for a, b in zip(pos0, lens)]
    if not c["fork"]:
        for i in range(n):
            path = _path(_parents(lens[i], c["twist"]))
            for j, x in enumerate(path):
                a, b = pos0[i] + x, pos0[i] + j
                planes[:, tables[i][b // PAGE], b % PAGE] = planes[:, tables[i][a // PAGE], a % PAGE]
            end[i] = pos0[i] + len(path)
            tables[i] = tables[i][:up(end[i])]
    ref = np.zeros(npages, np.int32)
    for t in tables:
        for p in t:
            ref[p] += 1
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)   # noqa: E731
    return {"pt": i32([[int(p) for p in t] + [-1] * (width - len(t)) for t in tables]), "ref": torch.from_numpy(ref), "len": i32(end), "pos0": i32(pos0),
            "row0": i32([0] + [int(x) for x in np.cumsum(lens)]), "planes": planes[:, :npages]}


def _exact_logprobs(s):
    T, k = s["case"]["rows"], s["case"]["k"]
    got = {name: torch.empty(T, w, dtype=torch.float64, device=DEV) for name, w in (("lse", 1), ("entropy", 1), ("lp", 1), ("top_lp", k))}
    top_i = torch.empty(T, k, dtype=torch.int32, device=DEV)
    for t0 in range(0, T, 64):
        x = s["logits"][t0:t0 + 64].double()
        lse = torch.logsumexp(x, 1, keepdim=True)
        p = torch.exp(x - lse)
        got["lse"][t0:t0 + 64] = lse
        got["entropy"][t0:t0 + 64] = -torch.where(p > 0, p * (x - lse), 0.0).sum(1, keepdim=True)
        got["lp"][t0:t0 + 64] = x.gather(1, s["tok"][t0:t0 + 64].long()) - lse
        if k:
            v, i = torch.sort(x, dim=1, descending=True, stable=True)
            got["top_lp"][t0:t0 + 64] = v[:, :k] - lse
            top_i[t0:t0 + 64] = i[:, :k].to(torch.int32)
    return {"lse": got["lse"][:, 0], "entropy": got["entropy"][:, 0], "lp": got["lp"], "top_lp": got["top_lp"], "top_i": top_i}
