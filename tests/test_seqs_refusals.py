"""What the calls over several sequences refuse on the host (no launch is reached, so no GPU is needed), the walk down a draft tree
and the merge of slices' log probabilities."""
import ctypes as C

import numpy as np
import pytest

P = 4096   # stands for a device address, 16-byte aligned; never read


def _seqs(fnx, **kw):
    v = dict(nseq=2, rows=8, row0=P, pos0=P, pt=P, pt_stride=4, npages=9, kv0=None, max_pos=100)
    v.update(kw)
    return fnx.Seqs(*v.values())


def _geometry(fnx, page=64 * 2 * 128, rows=64, cap=0, q8=0):
    return fnx.KvPages(None, page, rows, cap, q8)


BAD_SEQS = [(dict(row0=None), {}, "null buffer"), (dict(nseq=0), {}, "0 sequences"), (dict(rows=0), {}, "0 rows"), (dict(max_pos=-1), {}, "max_pos -1"),
            (dict(pt_stride=0), {}, "tables of 0"), (dict(npages=0), {}, "0 pages"), (dict(pt=None), {}, "row count"), ({}, dict(rows=0), "pages of 0 rows"),
            ({}, dict(page=64 * 256 - 8), "a page of"), ({}, dict(page=64 * 256 + 4), "a multiple of 8"), ({}, dict(q8=1), "int8"),
            (dict(pt_stride=1 << 26), {}, "2\\^31")]


@pytest.mark.parametrize("seqs,geometry,text", BAD_SEQS)
def test_sequences_that_make_no_sense(fnx, seqs, geometry, text):
    sq, g = _seqs(fnx, **seqs), _geometry(fnx, **geometry)
    with pytest.raises(fnx.FnxError, match=text):
        fnx.call("fnx_attn_prompt", P, 1024, None, P, P, g, fnx.byref(sq), P, 1024, 8, 2, 128, P, None)
    with pytest.raises(fnx.FnxError, match=text):
        fnx.call("fnx_attn_tree", P, 1024, None, P, P, g, fnx.byref(sq), P, 1, P, 1024, 8, 2, 128, P, None)
    with pytest.raises(fnx.FnxError, match=text):
        fnx.call("fnx_attn_seqs_append", P, P, P, P, P, P, P, g, fnx.byref(sq), None, P, 1e-6, fnx.Rope(1e4, 64), 8, 2, 128, P, None)


@pytest.mark.parametrize("change,text", [
    (dict(hd=64), "head dim 64"), (dict(nq=9), "9 query heads"), (dict(nq=34), "34 query heads"), (dict(nkv=0), "0 KV heads"), (dict(q=P + 2), "aligned"),
    (dict(kc=P + 8), "aligned"), (dict(out=P + 8), "aligned"), (dict(qg=P + 4), "aligned"), (dict(scratch=None), "null"), (dict(out=None), "null"), (dict(q=None), "null"),
    (dict(q_stride=1016), "apart"), (dict(q_stride=1028), "apart"), (dict(out_stride=0), "apart"), (dict(anc=None), "ancestor"), (dict(words=0), "ancestor")])
def test_attention_arguments(fnx, change, text):
    v = dict(q=P, q_stride=1024, qg=None, kc=P, vc=P, out=P, out_stride=1024, nq=8, nkv=2, hd=128, scratch=P, anc=P, words=1)
    v.update(change)
    sq, g = _seqs(fnx), _geometry(fnx)
    head, tail = (v["q"], v["q_stride"], v["qg"], v["kc"], v["vc"], g, fnx.byref(sq)), (v["out"], v["out_stride"], v["nq"], v["nkv"], v["hd"], v["scratch"], None)
    if "anc" not in change and "words" not in change:
        with pytest.raises(fnx.FnxError, match=text):
            fnx.call("fnx_attn_prompt", *head, *tail)
    with pytest.raises(fnx.FnxError, match=text):
        fnx.call("fnx_attn_tree", *head, v["anc"], v["words"], *tail)


def test_attention_takes_pages_of_whole_groups_of_8_rows(fnx):
    sq = _seqs(fnx)
    with pytest.raises(fnx.FnxError, match="a multiple of 8"):
        fnx.call("fnx_attn_prompt", P, 1024, None, P, P, _geometry(fnx, page=12 * 256, rows=12), fnx.byref(sq), P, 1024, 8, 2, 128, P, None)


@pytest.mark.parametrize("change,text", [(dict(nrot=0), "rotary"), (dict(nrot=63), "rotary"), (dict(nrot=130), "rotary"), (dict(k=P + 4), "aligned"), (dict(q16=P + 8), "aligned"),
                                         (dict(err=None), "null"), (dict(qn=None), "null")])
def test_append_arguments(fnx, change, text):
    v = dict(qg=P, k=P, v=P, qn=P, kn=P, kc=P, vc=P, q16=P, nrot=64, err=P)
    v.update(change)
    with pytest.raises(fnx.FnxError, match=text):
        fnx.call("fnx_attn_seqs_append", v["qg"], v["k"], v["v"], v["qn"], v["kn"], v["kc"], v["vc"], _geometry(fnx), fnx.byref(_seqs(fnx)), None, v["q16"], 1e-6,
                 fnx.Rope(1e4, v["nrot"]), 8, 2, 128, v["err"], None)


@pytest.mark.parametrize("change,text", [(dict(parent=None), "null"), (dict(anc=None), "null"), (dict(err=None), "null"), (dict(words=0), "words"), (dict(words=33), "words")])
def test_tree_mask_arguments(fnx, change, text):
    v = dict(parent=P, anc=P, words=1, err=P)
    v.update(change)
    with pytest.raises(fnx.FnxError, match=text):
        fnx.call("fnx_tree_masks", v["parent"], fnx.byref(_seqs(fnx)), v["anc"], v["words"], None, v["err"], None)
    with pytest.raises(fnx.FnxError, match="sequences"):
        fnx.call("fnx_tree_masks", P, fnx.byref(_seqs(fnx, nseq=0)), P, 1, None, P, None)


def _pool(fnx, **kw):
    v = dict(npages=8, rows=64, ref=P, nseq=2, pt=P, pt_stride=4, len=P)
    v.update(kw)
    return fnx.PagePool(*v.values())


@pytest.mark.parametrize("pool,text", [(dict(ref=None), "null"), (dict(pt=None), "null"), (dict(len=None), "null"), (dict(npages=0), "0 pages"), (dict(rows=0), "of 0 rows"),
                                       (dict(pt_stride=0), "tables of 0"), (dict(nseq=0), "0 sequences"), (dict(nseq=4097), "4097 sequences"),
                                       (dict(pt_stride=1 << 25), "2\\^31")])
def test_pools_that_make_no_sense(fnx, pool, text):
    p = _pool(fnx, **pool)
    g = fnx.KvPages(None, 64 * 256, p.rows, 0, 0)
    with pytest.raises(fnx.FnxError, match=text):
        fnx.call("fnx_pages_fork", fnx.byref(p), P, None, P, P, None)
    with pytest.raises(fnx.FnxError, match=text):
        fnx.call("fnx_pages_reserve", fnx.byref(p), P, P, P, P, 2, g, 2, 128, P, P, None)
    with pytest.raises(fnx.FnxError, match=text):
        fnx.call("fnx_pages_keep", fnx.byref(p), P, P, 4, P, P, 2, g, 2, 128, P, P, None)


@pytest.mark.parametrize("pool", [dict(npages=(1 << 30) + 1), dict(rows=1, pt_stride=(1 << 30) + 1)])
def test_pools_past_2_to_30(fnx, pool):
    with pytest.raises(fnx.FnxError, match="2\\^30 at most"):
        fnx.call("fnx_pages_fork", fnx.byref(_pool(fnx, **pool)), P, None, P, P, None)


@pytest.mark.parametrize("change,text", [(dict(planes=None), "planes"), (dict(nplanes=0), "0 planes"), (dict(nplanes=65536), "planes"), (dict(hd=96), "of 96"), (dict(nkv=0), "0 KV"),
                                         (dict(rows=32), "pages of 32"), (dict(page=64 * 256 - 8), "a page of"), (dict(page=64 * 256 + 2), "multiple of 8"),
                                         (dict(page=64 * 136 - 8, q8=1), "a page of"), (dict(add=None), "null")])
def test_page_arguments(fnx, change, text):
    v = dict(planes=P, nplanes=2, page=64 * 256, rows=64, q8=0, nkv=2, hd=128, add=P)
    v.update(change)
    g = fnx.KvPages(None, v["page"], v["rows"], 0, v["q8"])
    with pytest.raises(fnx.FnxError, match=text):
        fnx.call("fnx_pages_reserve", fnx.byref(_pool(fnx)), v["add"], P, P, v["planes"], v["nplanes"], g, v["nkv"], v["hd"], P, P, None)
    with pytest.raises(fnx.FnxError, match=text):
        fnx.call("fnx_pages_keep", fnx.byref(_pool(fnx)), P, v["add"], 4, P, v["planes"], v["nplanes"], g, v["nkv"], v["hd"], P, P, None)


@pytest.mark.parametrize("change,text", [(dict(n=0), "rows of 0"), (dict(T=0), "0 rows"), (dict(stride=99), "99 apart"), (dict(k=65), "65 alternatives"), (dict(n=3, k=4), "of 3"),
                                         (dict(v0=-1), "token -1"), (dict(tok=None), "given tokens"), (dict(logits=None), "null"), (dict(top=None), "null"),
                                         (dict(scratch=P + 8), "aligned"), (dict(err=None), "null"), (dict(ntok=-1), "-1 given")])
def test_logprob_arguments(fnx, change, text):
    v = dict(logits=P, stride=100, n=100, T=2, v0=0, tok=P, ntok=1, k=4, top=P, scratch=P, err=P)
    v.update(change)
    with pytest.raises(fnx.FnxError, match=text):
        fnx.call("fnx_logprobs", v["logits"], v["stride"], v["n"], v["T"], v["v0"], v["tok"], v["ntok"], v["k"], P, P, P, v["top"], P, v["scratch"], v["err"], None)


def test_scratch_sizes_of_nonsense_are_zero(fnx):
    lib = fnx.load()
    assert lib.fnx_logprobs_scratch_bytes(0, 1, 1) == 0 and lib.fnx_logprobs_scratch_bytes(10, 1, 65) == 0
    assert lib.fnx_pages_scratch_bytes(fnx.byref(_pool(fnx, npages=0))) == 0
    assert lib.fnx_attn_seqs_scratch_bytes(fnx.byref(_seqs(fnx)), 0, 2, 128) == 0


def _i(x):
    return np.ascontiguousarray(x, np.int32)


def test_accept_tree(fnx):
    lib = fnx.load()
    rng = np.random.default_rng(0)
    for n in (1, 2, 16, 64):
        for _ in range(50):
            parent = [-1] + [int(rng.integers(0, i)) for i in range(1, n)]
            tok, out = rng.integers(0, 3, n), rng.integers(0, 3, n)
            want, at = [0], 0
            while True:
                child = [i for i in range(1, n) if parent[i] == at and tok[i] == out[at]]
                if not child:
                    break
                at = child[0]
                want.append(at)
            path, a = np.zeros(n, np.int32), [_i(tok), _i(parent), _i(out)]
            got = lib.fnx_accept_tree(*(x.ctypes.data for x in a), n, path.ctypes.data)
            assert path[:got].tolist() == want
    chain = [_i([7, 1, 2, 3]), _i([-1, 0, 1, 2]), _i([1, 2, 9, 4])]
    path = np.zeros(4, np.int32)
    assert lib.fnx_accept_tree(*(x.ctypes.data for x in chain), 4, path.ctypes.data) == lib.fnx_accept_greedy(chain[0].ctypes.data, chain[2].ctypes.data, 4) == 3
    for bad in ([-1, 1, 0, 0], [-1, -2, 0, 0], [-1, 0, 3, 0]):
        assert lib.fnx_accept_tree(chain[0].ctypes.data, _i(bad).ctypes.data, chain[2].ctypes.data, 4, path.ctypes.data) < 0
        assert b"parent" in lib.fnx_last_error()
    assert lib.fnx_accept_tree(None, chain[1].ctypes.data, chain[2].ctypes.data, 4, path.ctypes.data) < 0


def test_logprobs_merge_refuses(fnx):
    a = np.zeros(64, np.float32).ctypes.data
    for args, text in (((a, a, a, a, a, 0, 1, 1, 1), "0 slices"), ((a, a, a, a, a, 65, 1, 1, 1), "65 slices"), ((a, a, a, a, a, 1, 1, 1, 65), "65 alternatives"),
                       ((None, a, a, a, a, 1, 1, 1, 1), "null"), ((a, None, a, a, a, 1, 1, 1, 1), "null"), ((a, a, None, a, a, 1, 1, 1, 1), "null"),
                       ((a, a, a, None, a, 1, 1, 1, 1), "null")):
        with pytest.raises(fnx.FnxError, match=text):
            fnx.call("fnx_logprobs_merge", *args, a, a, a, a, a)


@pytest.mark.parametrize("cuts", [[0, 50], [0, 7, 20, 50], [0, 1, 2, 50]])
def test_logprobs_merge_equals_the_whole(fnx, cuts):
    rng = np.random.default_rng(len(cuts))
    T, n, k = 5, 50, 6
    x = rng.standard_normal((T, n)) * 5
    x[1, :20], x[2, 20:], x[3] = -np.inf, -np.inf, -np.inf
    x[4, ::3] = 2.5
    tok = rng.integers(0, n, (T, 2))

    def stats(y, v0, ids):
        with np.errstate(all="ignore"):
            m = y.max(1, keepdims=True)
            lse = np.where(np.isinf(m), -np.inf, m + np.log(np.exp(y - np.where(np.isinf(m), 0, m)).sum(1, keepdims=True)))
            lp = np.where(np.isinf(y), -np.inf, y - lse)
            p = np.where(np.isinf(lp), 0, np.exp(lp))
            ent = -np.where(p > 0, p * np.where(p > 0, lp, 0), 0).sum(1)
            inside = (ids >= v0) & (ids < v0 + y.shape[1])
            given = np.where(inside, np.take_along_axis(lp, np.clip(ids - v0, 0, y.shape[1] - 1), 1), -np.inf)
            order = np.argsort(-y, axis=1, kind="stable")
        return lse[:, 0], ent, given, np.take_along_axis(lp, order, 1), order + v0

    parts = []
    for a, b in zip(cuts, cuts[1:]):
        lse, ent, given, lp, order = stats(x[:, a:b], a, tok)
        wide = max(0, k - (b - a))   # a slice of fewer tokens than alternatives: filled up with what never wins
        parts.append([lse, ent, given, np.pad(lp, ((0, 0), (0, wide)), constant_values=-np.inf)[:, :k], np.pad(order, ((0, 0), (0, wide)), constant_values=1 << 20)[:, :k]])
    host = [np.ascontiguousarray(np.stack([p[i] for p in parts]), np.int32 if i == 4 else np.float32) for i in range(5)]
    out = [np.zeros(T, np.float32), np.zeros(T, np.float32), np.zeros((T, 2), np.float32), np.zeros((T, k), np.float32), np.zeros((T, k), np.int32)]
    fnx.call("fnx_logprobs_merge", *(h.ctypes.data for h in host), len(cuts) - 1, T, 2, k, *(o.ctypes.data for o in out))
    lse, ent, given, lp, order = stats(x, 0, tok)
    for got, want in zip(out, (lse, ent, given, lp[:, :k])):
        assert np.array_equal(np.isinf(got), np.isinf(want)) and np.allclose(got[np.isfinite(want)], want[np.isfinite(want)], rtol=1e-5, atol=1e-5)
    assert np.array_equal(out[4][:3], order[:3, :k]) and np.array_equal(out[4][4], order[4, :k])
