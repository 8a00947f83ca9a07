"""The rows of several sequences: append against the window's own append (bit for bit) and 64 bits, draft trees' masks, and the
attention of prompts, single tokens and trees against 64 bits, over pages in no order with NaN wherever nothing lives."""
import numpy as np
import pytest
import torch

from sfnx_b200 import lib as L
from tests import seqs_util as S
from tests.seqs_util import DEV

pytestmark = pytest.mark.gpu

EPS, BASE = 1e-6, 1e7
HEADS = [(24, 4, 256), (8, 2, 128), (16, 1, 256), (3, 3, 128), (10, 2, 256)]


def _check(s, out, bits=None, gate=True, pad=0):
    ref, tol = s.reference(bits, gate)
    w = s.nq * s.hd
    got = out[:s.rows, :w].double().view(s.rows, s.nq, s.hd)
    assert torch.isfinite(got).all()
    over = (got - ref).abs() - tol
    assert (over <= 0).all(), "off by %.3g where %.3g is allowed (row, head, dim %s)" % (
        float((got - ref).abs().view(-1)[over.argmax()]), float(tol.view(-1)[over.argmax()]), np.unravel_index(int(over.argmax()), over.shape))
    assert (out[s.rows:] == -7).all(), "rows behind the last sequence were written"
    assert (out[:, w:] == -7).all(), "columns between the rows were written"
    assert L.load().fnx_device_fault() == 0


# ---------------------------------------------------------------- append
def _append(s, k, v, qn, kn, depth=None, nrot=64, q16=None):
    q16 = torch.full((s.total, s.nq, s.hd), -7.0, dtype=torch.float16, device=DEV) if q16 is None else q16
    L.call("fnx_attn_seqs_append", s.qg.data_ptr(), k.data_ptr(), v.data_ptr(), qn.data_ptr(), kn.data_ptr(), s.kc.data_ptr(), s.vc.data_ptr(), s.geometry(),
           L.byref(s.seqs()), L.ptr(depth), q16.data_ptr(), EPS, L.Rope(BASE, nrot), s.nq, s.nkv, s.hd, s.err.data_ptr(), L.stream())
    return q16


@pytest.mark.parametrize("nq,nkv,hd", HEADS)
@pytest.mark.parametrize("page,nrot,tree", [(64, 64, False), (8, 128, True), (24, 2, False), (0, 32, True), (1, 64, False)])
def test_append_has_the_windows_bits(nq, nkv, hd, page, nrot, tree):
    s = S.Seqs([5, 0, 16, 1, 33], [0, 7, 129, 30011, 64], nq, nkv, hd, page=page, seed=nq + page, extra_rows=3, pitch=16)
    before = [s.rows_of(s.kc).clone(), s.rows_of(s.vc).clone()]
    k, v = torch.randn(s.total, nkv, hd, device=DEV) * 3, torch.randn(s.total, nkv, hd, device=DEV)
    qn, kn = 1 + 0.1 * torch.randn(hd, device=DEV), 1 + 0.1 * torch.randn(hd, device=DEV)
    _, _, dep = s.tree()
    depth = torch.from_numpy(dep).to(DEV) if tree else None
    qg0 = s.qg.clone()
    q16 = _append(s, k, v, qn, kn, depth, nrot)
    # every row through the window's append, one at a time: a cache of one row beginning at the row's own rotary position
    one = torch.zeros(1, dtype=torch.int32, device=DEV)
    kc, vc = s.rows_of(s.kc), s.rows_of(s.vc)
    live = torch.zeros(kc.shape[0], dtype=torch.bool, device=DEV)
    for i in range(s.n):
        for j in range(s.lens[i]):
            t, at = s.row0[i] + j, int(s.cells[i][s.ctx[i] + j])
            live[at] = True
            turn = s.ctx[i] + (int(dep[t]) if tree else j)
            one.fill_(turn)
            a, b = s.qg[t:t + 1].clone(), k[t:t + 1].clone()
            cache = torch.zeros(2, turn + 1, nkv, hd, dtype=torch.float16, device=DEV)
            L.call("fnx_attn_prep_append", a.data_ptr(), b.data_ptr(), v[t].data_ptr(), qn.data_ptr(), kn.data_ptr(), cache[0].data_ptr(), cache[1].data_ptr(),
                   L.KvPages(None, 0, 0, turn + 1, 0), 0, 1, 1, one.data_ptr(), EPS, L.Rope(BASE, nrot), nq, nkv, hd, L.stream())
            assert torch.equal(q16[t].view(torch.int16), a[0, :, :hd].half().view(torch.int16)), "queries of row %d" % t
            assert torch.equal(kc[at].view(torch.int16), cache[0, turn].view(torch.int16)) and torch.equal(vc[at].view(torch.int16), cache[1, turn].view(torch.int16))
    assert torch.equal(s.qg, qg0) and (q16[s.rows:] == -7).all() and int(s.err) == 0
    for now, was in ((kc, before[0]), (vc, before[1])):
        assert torch.equal(now[~live].view(torch.int16), was[~live].view(torch.int16)), "a row that is not the call's was written"


def test_append_against_64_bits():
    """One rounding to f16 after 32-bit arithmetic: 2^-11 of the value, and 32 roundings' 2^-24 of the row's largest."""
    s = S.Seqs([70, 3], [0, 2000], 24, 4, 256, seed=5)
    k, v = torch.randn(s.total, 4, 256, device=DEV), torch.randn(s.total, 4, 256, device=DEV)
    qn = 1 + 0.1 * torch.randn(256, device=DEV)
    q16 = _append(s, k, v, qn, qn)
    pos = torch.cat([torch.arange(m) + x for m, x in zip(s.lens, s.ctx)]).to(DEV)
    f = torch.tensor(np.float32(np.float64(BASE) ** (-2.0 * np.arange(32) / 64)), device=DEV)
    ang = (pos.float()[:, None] * f).double()[:, None]
    y = s.qg[..., :256].double()
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * qn.double()
    a, b = y[..., :32].clone(), y[..., 32:64].clone()
    y[..., :32], y[..., 32:64] = a * torch.cos(ang) - b * torch.sin(ang), b * torch.cos(ang) + a * torch.sin(ang)
    tol = 2.0 ** -11 * y.abs() + 32 * 2.0 ** -24 * y.abs().amax(-1, keepdim=True) + 2.0 ** -25
    assert ((q16.double() - y).abs() <= tol).all()


def test_append_leaves_rows_without_a_page():
    """A table that ends, an entry of -1, one past the pool and a negative position: nothing is written for such rows (their
    queries are), the word says so, and the other rows are there."""
    s = S.Seqs([4, 4, 4, 4], [62, 62, 62, 0], 8, 2, 128, page=64, seed=9)
    ok = s.cells[0].to(DEV)
    s.d_table[1, 1], s.d_table[2, 0] = -1, s.npages
    s.d_pos0[3] = -3
    before = s.rows_of(s.kc).clone()
    k, v = torch.randn(s.total, 2, 128, device=DEV), torch.randn(s.total, 2, 128, device=DEV)
    w = torch.ones(128, device=DEV)
    q16 = _append(s, k, v, w, w)
    assert int(s.err) == 32 and torch.isfinite(q16).all() and (q16 != -7).any(-1).all()
    now = s.rows_of(s.kc)
    changed = (now.view(torch.int16) != before.view(torch.int16)).flatten(1).any(1).nonzero()[:, 0]
    want = torch.cat([ok[62:], s.cells[1].to(DEV)[62:64], s.cells[2].to(DEV)[64:]])
    assert torch.equal(changed, want.sort().values)
    s.err.zero_()
    s.width = 1   # tables of one page: positions 64 and 65 have none
    _append(s, k, v, w, w)
    assert int(s.err) == 32


# ---------------------------------------------------------------- trees
@pytest.mark.parametrize("lens,words", [([16], 1), ([1, 0, 64, 33, 7], 2), ([40, 300, 3], 10), ([1024], 32)])
def test_tree_masks(lens, words):
    s = S.Seqs(lens, [0] * len(lens), 8, 2, 128, seed=sum(lens), extra_rows=2)
    par, bits, depth = s.tree(words)
    d_par = torch.tensor(par + [5, 5], dtype=torch.int32, device=DEV)
    anc, dep = (torch.full(shape, -7, dtype=torch.int32, device=DEV) for shape in ((s.total, words), (s.total,)))
    for with_depth in (True, False):
        L.call("fnx_tree_masks", d_par.data_ptr(), L.byref(s.seqs()), anc.data_ptr(), words, dep.data_ptr() if with_depth else None, s.err.data_ptr(), L.stream())
        assert int(s.err) == 0 and (anc[s.rows:] == -7).all() and (dep[s.rows:] == -7).all()
        assert np.array_equal(anc[:s.rows].cpu().numpy().view(np.uint32), bits) and np.array_equal(dep[:s.rows].cpu().numpy(), depth)


def test_tree_masks_of_bad_parents():
    """A row that is its own parent, one after itself, one below -1 start a path of their own; rows past the words see nothing."""
    s = S.Seqs([4, 35], [0, 0], 8, 2, 128)
    par = torch.tensor([-1, 1, 3, 2] + [-1] + list(range(34)), dtype=torch.int32, device=DEV)
    anc, dep = torch.zeros(39, 1, dtype=torch.int32, device=DEV), torch.zeros(39, dtype=torch.int32, device=DEV)
    L.call("fnx_tree_masks", par.data_ptr(), L.byref(s.seqs()), anc.data_ptr(), 1, dep.data_ptr(), s.err.data_ptr(), L.stream())
    assert int(s.err) == 64
    assert anc[:4, 0].tolist() == [1, 2, 4, 12] and dep[:4].tolist() == [0, 0, 0, 1]
    assert anc[4:36, 0].tolist() == [(1 << (i + 1)) - 1 - (2 ** 32 if i == 31 else 0) for i in range(32)] and anc[36:, 0].tolist() == [0, 0, 0]


# ---------------------------------------------------------------- attention
PROMPTS = [
    ([1], [0]), ([130], [0]), ([1, 0, 17, 300, 1, 64], [0, 5, 0, 0, 31, 200]), ([129, 2], [1000, 4097]), ([1] * 5, [0, 1, 63, 64, 2049]), ([700], [0]),
    ([0, 0, 3], [0, 9, 0]), ([1], [20000]), ([7, 260], [9000, 12]),
]


@pytest.mark.parametrize("lens,ctx", PROMPTS)
@pytest.mark.parametrize("nq,nkv,hd", HEADS)
def test_prompt_attention(nq, nkv, hd, lens, ctx):
    s = S.Seqs(lens, ctx, nq, nkv, hd, seed=len(lens) + nq, extra_rows=3)
    _check(s, s.attend())


@pytest.mark.parametrize("page,pitch", [(0, 0), (8, 0), (24, 8), (16, 64), (128, 0), (256, 8), (40, 0)])
@pytest.mark.parametrize("hd", [128, 256])
def test_prompt_attention_page_sizes(hd, page, pitch):
    """Pages that end inside a tile, pages larger than one, a pitch wider than the rows, no pages at all; strided queries and
    outputs, no gate."""
    s = S.Seqs([90, 1, 211], [37, 500, 0], 6, 2, hd, page=page, pitch=pitch, pad=24, seed=page)
    _check(s, s.attend(gate=False, out_pad=40), gate=False)


@pytest.mark.parametrize("lens,ctx,words", [([16], [3000], 1), ([1], [0], 1), ([40, 24, 64, 33, 9, 63], [700, 1, 0, 129, 64, 4000], 2), ([200, 0, 5], [10, 3, 70], 7),
                                            ([64], [0], 4), ([12], [20001], 1)])
@pytest.mark.parametrize("nq,nkv,hd", HEADS)
def test_tree_attention(nq, nkv, hd, lens, ctx, words):
    s = S.Seqs(lens, ctx, nq, nkv, hd, seed=sum(lens) + nq, extra_rows=1)
    _, bits, _ = s.tree(words)
    _check(s, s.attend(torch.from_numpy(bits.view(np.int32)).to(DEV)), bits)


def test_tree_masks_that_leave_rows_empty():
    """A row whose mask is empty over an empty context gives zeros (over a context: the context alone); a mask of all bits sees no
    row past the sequence's own."""
    s = S.Seqs([5, 5, 40], [0, 70, 3], 8, 2, 128, seed=3)
    _, bits, _ = s.tree(2)
    bits[[1, 6]] = 0
    bits[[2, 7]] = 0xFFFFFFFF
    out = s.attend(torch.from_numpy(bits.view(np.int32)).to(DEV))
    assert (out[1, :8 * 128] == 0).all()
    _check(s, out, bits)


@pytest.mark.parametrize("tree", [False, True])
def test_attention_of_a_thousand_sequences(tree):
    """More sequences than a warp has lanes, most of them empty, some long; runs of work begin and end anywhere among them."""
    rng = np.random.default_rng(21)
    lens = [int(rng.integers(1, 9)) if rng.random() < 0.15 else 0 for _ in range(1000)]
    lens[3], lens[40], lens[999] = 64, 50, 3
    ctx = [int(rng.integers(0, 40)) if n and rng.random() < 0.9 else 0 for n in lens]
    ctx[40], ctx[999] = 2500, 700
    s = S.Seqs(lens, ctx, 8, 2, 128, page=16, seed=21, extra_rows=5)
    bits = s.tree(2)[1] if tree else None
    _check(s, s.attend(None if bits is None else torch.from_numpy(bits.view(np.int32)).to(DEV)), bits)


@pytest.mark.parametrize("lens,ctx", [([1500], [0]), ([0, 1, 1029, 0, 257, 255, 256], [0, 5, 0, 77, 3, 1, 0]), ([640, 1], [333, 12000])])
def test_prompt_attention_long_and_ragged(lens, ctx):
    s = S.Seqs(lens, ctx, 8, 2, 128, seed=31, extra_rows=2)
    _check(s, s.attend())


@pytest.mark.parametrize("scale", [0.0, 40.0])
@pytest.mark.parametrize("lens,ctx", [([300], [0]), ([3, 1], [4000, 900])])
def test_prompt_attention_flat_and_sharp_scores(lens, ctx, scale):
    """All scores alike, and scores that rise by hundreds along the positions (the running maximum is raised many times)."""
    s = S.Seqs(lens, ctx, 12, 2, 256, seed=4)
    rise = torch.ones(s.k.shape[0], device=DEV)
    for c in s.cells:
        rise[c.to(DEV)] = torch.linspace(0.05, 1.0, len(c), device=DEV)
    live = s.live.to(DEV)
    s.k[live] = (torch.sign(s.k[live].float()) * rise[live][:, None, None] if scale else s.k[live].float() * 0).half()
    s.q[:] = (torch.sign(s.q.float()) * scale / 16).half() if scale else s.q
    if scale:
        s.q[:, :] = s.q.abs()
        s.k[live] = s.k[live].abs()
    s.kc, s.vc = s._pool(s.k), s._pool(s.v)
    _check(s, s.attend())


def test_prompt_attention_entries_outside_the_pool_are_rows_of_zeros():
    s = S.Seqs([2, 70], [300, 100], 8, 2, 128, page=64, seed=8)
    for i, j, bad in ((0, 1, -1), (0, 3, 10 ** 6), (1, 0, s.npages)):
        page = int(s.table[i, j])
        s.k[page * 64:(page + 1) * 64] = 0   # what the 64-bit form reads there
        s.v[page * 64:(page + 1) * 64] = 0
        s.d_table[i, j] = bad
    _check(s, s.attend())


@pytest.mark.parametrize("lens,ctx,at", [([70, 3], [200, 40], range(128, 192)), ([1, 3], [6000, 40], range(5000, 5064)), ([2], [1], range(0, 2)), ([1], [0], range(0, 1))])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_score_that_is_no_number_shows_in_the_rows_that_see_it(lens, ctx, at, value):
    """A NaN or infinity in a key, wherever in a tile it lies: rows that see it and get a NaN or +inf score give NaNs, all others what
    they gave before (a score of -inf weighs nothing)."""
    s = S.Seqs(lens, ctx, 8, 2, 128, seed=17)
    before = s.attend().view(-1, 8, 128)
    assert torch.isfinite(before).all()
    q0 = s.q[:s.rows].view(s.rows, 8, 128)[:, :4, 0]
    pos = torch.tensor([x + t for n, x in zip(lens, ctx) for t in range(n)], device=DEV)
    for p in at:
        row = s.rows_of(s.kc)[int(s.cells[0][p]), 0]
        keep = row.clone()
        s.rows_of(s.kc)[int(s.cells[0][p]), 0, 0] = value
        out = s.attend().view(-1, 8, 128)
        row.copy_(keep)
        hit = (torch.arange(s.rows, device=DEV) < lens[0])[:, None] & (pos >= p)[:, None] & ((q0 >= 0) if value == float("inf") else torch.ones_like(q0, dtype=torch.bool))
        assert torch.isnan(out[:, :4][hit]).all(), p
        if value != value:
            assert torch.equal(out[:, :4][~hit], before[:, :4][~hit]), p
        assert torch.isfinite(out[:, :4][~hit]).all() and torch.equal(out[:, 4:], before[:, 4:]), p


def test_a_gate_that_is_no_number_shows_in_its_own_element():
    for lens, ctx in (([5], [60]), ([1], [9000])):
        s = S.Seqs(lens, ctx, 8, 2, 128, seed=18)
        before = s.attend()
        s.qg[0, 3, 128 + 7], s.qg[0, 3, 128 + 20], s.qg[0, 3, 128 + 31] = float("nan"), float("inf"), -float("inf")
        out, want = s.attend(), before.clone()
        want[0, 3 * 128 + 7], want[0, 3 * 128 + 31] = float("nan"), 0.0
        plain = s.attend(gate=False)
        want[0, 3 * 128 + 20] = plain[0, 3 * 128 + 20]
        near = (out - want).abs() <= 2.0 ** -10 * want.abs()   # (a sigmoid of a pair's shared reciprocal: the last bit may differ)
        assert torch.isnan(out[0, 3 * 128 + 7]) and (near | torch.isnan(want)).all()


@pytest.mark.parametrize("hint", [0, 1, 50000])
def test_prompt_attention_whatever_the_hint(hint):
    """max_pos decides how the work is split, never what is computed: too small, unknown, far too large."""
    s = S.Seqs([1, 20, 1], [3000, 400, 0], 24, 4, 256, seed=6, max_pos=hint)
    _check(s, s.attend())


def test_prompt_attention_is_repeatable_and_takes_any_stream():
    s = S.Seqs([1, 140, 5], [5000, 60, 900], 24, 4, 256, seed=11)
    a = s.attend()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        b = s.attend(scratch=s.scratch(fill=0x7F))
    torch.cuda.synchronize()
    assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_prompt_attention_captured_then_replayed_on_other_lengths():
    """Two captured calls share one scratch; the sequences' rows and positions change between the replays, the tables grow."""
    s = S.Seqs([40, 3, 21], [100, 0, 333], 8, 2, 256, seed=12)
    first = (s.d_row0.clone(), s.d_pos0.clone())
    scratch = s.scratch()
    out = [torch.full((s.total, 8 * 256), -7.0, dtype=torch.float16, device=DEV) for _ in range(2)]
    s.attend(out=out[0], scratch=scratch)   # warm-up
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s.attend(out=out[0], scratch=scratch)
        s.attend(out=out[1], scratch=scratch, gate=False)
    s.lens, s.ctx = [10, 0, 8], [130, 3, 340]
    s.row0, s.rows = [0, 10, 10, 18], 18
    s.d_row0.copy_(torch.tensor(s.row0, dtype=torch.int32))
    s.d_pos0.copy_(torch.tensor(s.ctx, dtype=torch.int32))
    s.cells = [c[:a + b] for c, a, b in zip(s.cells, s.lens, s.ctx)]
    for o in out:
        o.fill_(-7.0)
    g.replay()
    torch.cuda.synchronize()
    _check(s, out[0])
    _check(s, out[1], gate=False)
    s.d_row0.copy_(first[0])
    g.replay()
    torch.cuda.synchronize()


@pytest.mark.parametrize("page,lens,ctx", [(0, [1], [0]), (0, [2, 1], [0, 3]), (8, [1], [0]), (8, [3], [5]), (256, [1], [2])])
@pytest.mark.parametrize("nq,nkv,hd", [(1, 1, 128), (16, 1, 256), (22, 2, 128)])
def test_caches_and_calls_smaller_than_a_tile(page, lens, ctx, nq, nkv, hd):
    """Pools of a page or two and contiguous caches of a few rows, shorter than any box that is copied out of them; no row behind
    the last sequence."""
    s = S.Seqs(lens, ctx, nq, nkv, hd, page=page, seed=page + nq)
    _check(s, s.attend())
    _, bits, _ = s.tree(1)
    _check(s, s.attend(torch.from_numpy(bits.view(np.int32)).to(DEV)), bits)


@pytest.mark.parametrize("page", [0, 64])
def test_sequences_without_any_rows(page):
    """Nothing is attended, appended or masked; rows that belong to nobody stay as they are."""
    s = S.Seqs([0, 0, 0], [0, 70, 3], 8, 2, 128, page=page, extra_rows=9)
    bits = np.zeros((0, 1), np.uint32)
    _, _, _ = s.tree(1)
    _check(s, s.attend())
    anc = torch.full((9, 1), -7, dtype=torch.int32, device=DEV)
    _check(s, s.attend(anc), bits)
    par, dep = torch.full((9,), -5, dtype=torch.int32, device=DEV), torch.full((9,), -7, dtype=torch.int32, device=DEV)
    L.call("fnx_tree_masks", par.data_ptr(), L.byref(s.seqs()), anc.data_ptr(), 1, dep.data_ptr(), s.err.data_ptr(), L.stream())
    k, w = torch.randn(9, 2, 128, device=DEV), torch.ones(128, device=DEV)
    before = s.kc.clone()
    q16 = _append(s, k, k, w, w)
    torch.cuda.synchronize()
    assert int(s.err) == 0 and (q16 == -7).all() and (anc == -7).all() and (dep == -7).all()
    assert torch.equal(s.kc.view(torch.int16), before.view(torch.int16))


def test_calls_on_two_streams_at_once():
    a, b = S.Seqs([300, 1, 17], [900, 4000, 3], 24, 4, 256, seed=41), S.Seqs([1] * 9, [500 * i for i in range(9)], 8, 2, 128, seed=42)
    want = [x.attend().clone() for x in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.empty_like(w) for _ in range(6)] for w in want]
    scratch = [x.scratch() for x in (a, b)]
    torch.cuda.synchronize()
    for i in range(6):
        for x, st, o, w in zip((a, b), streams, outs, scratch):
            with torch.cuda.stream(st):
                x.attend(out=o[i], scratch=w)
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert all(torch.equal(w[:-1].view(torch.int16), x[:-1].view(torch.int16)) for x in o)
    assert L.load().fnx_device_fault() == 0


def test_cache_past_2_to_31_elements():
    """A pool of more than 2^31 halves: the sequence's pages lie at its far end."""
    nq, nkv, hd, page = 2, 2, 256, 64
    npages = (1 << 31) // (page * nkv * hd) + 8
    s = S.Seqs([3], [130], nq, nkv, hd, page=page, seed=13)
    big = [torch.zeros(npages, page * nkv * hd, dtype=torch.float16, device=DEV) for _ in range(2)]
    shift = npages - s.npages
    for b, small in zip(big, (s.kc, s.vc)):
        b[shift:] = small
    s.kc, s.vc = big
    s.d_table[s.d_table >= 0] += shift
    s.npages = npages
    _check(s, s.attend())
    k, v = torch.randn(3, nkv, hd, device=DEV), torch.randn(3, nkv, hd, device=DEV)
    w = torch.ones(hd, device=DEV)
    _append(s, k, v, w, w)
    at = s.cells[0][130:] + shift * page
    assert torch.equal(s.rows_of(s.vc)[at.to(DEV)], v.half()) and int(s.err) == 0
