"""The attention over sequences at the ends of what it takes: units smaller than a box, runs of seconds."""
import numpy as np
import pytest
import torch

from sfnx_b200 import lib as L
from tests import seqs_util as S
from tests.seqs_util import DEV
from tests.test_gpu_seqs import _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [0, 8, 64])
@pytest.mark.parametrize("nq,nkv,hd", [(4, 2, 256), (6, 2, 128)])
def test_many_units_of_less_than_a_box(nq, nkv, hd, page):
    """Hundreds of units one after another on every pair of CTAs, of 1 to 64 positions (the second CTA copies no keys at all) and of a
    little more than a tile, ending anywhere in a step of 16, with NaN behind every sequence's newest row."""
    n = 640
    ctx = [(7 * i) % 64 if i % 5 else 128 + i % 19 for i in range(n)]
    s = S.Seqs([1] * n, ctx, nq, nkv, hd, page=page, seed=page + hd)
    out = s.attend()
    _check(s, out)
    for _ in range(20):
        assert torch.equal(s.attend().view(torch.int16), out.view(torch.int16))
    assert L.load().fnx_device_fault() == 0


def test_a_run_of_work_longer_than_any_wait():
    """A token after 2^29 positions, all in one page, its work on four pairs of CTAs (the hint): a pair is at it for more than a second,
    which no single wait may last.  All scores are zero and the values powers of two, so the sum of the weights is exact.  The tensor
    core cuts a product off 25 places below the sum it goes to (2^26 |v| and |v| give 2^26 |v|): a part of 2^27 positions comes to
    2^26 |v| at least, and the result lies between half of v, less the f16 rounding, and v."""
    nq, nkv, hd, page, total = 2, 1, 256, 256, 1 << 29
    v = torch.tensor([(-1.0) ** d * 2.0 ** -(d % 8) for d in range(hd)], device=DEV).half()
    kc, vc = torch.zeros(1, page, hd, dtype=torch.float16, device=DEV), v.repeat(1, page, 1).contiguous()
    table = torch.zeros(1, total // page, dtype=torch.int32, device=DEV)
    row0, pos0 = torch.tensor([0, 1], dtype=torch.int32, device=DEV), torch.tensor([total - 1], dtype=torch.int32, device=DEV)
    sq = L.Seqs(1, 1, row0.data_ptr(), pos0.data_ptr(), table.data_ptr(), table.shape[1], 1, None, 1)
    q, out = torch.randn(1, nq * hd, device=DEV).half(), torch.zeros(1, nq * hd, dtype=torch.float16, device=DEV)
    scratch = torch.empty(L.load().fnx_attn_seqs_scratch_bytes(L.byref(sq), nq, nkv, hd), dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    L.call("fnx_attn_prompt", q.data_ptr(), nq * hd, None, kc.data_ptr(), vc.data_ptr(), L.KvPages(None, page * hd, page, 0, 0), L.byref(sq), out.data_ptr(), nq * hd, nq,
           nkv, hd, scratch.data_ptr(), L.stream())
    b.record()
    torch.cuda.synchronize()
    assert L.load().fnx_device_fault() == 0, "a wait ran out"
    share = out.view(nq, hd).double() / v.double()
    assert (share >= 0.5 * (1 - 2.0 ** -10)).all() and (share <= 1).all()
    assert a.elapsed_time(b) > 1074, "%.0f ms: no longer than a wait may last (2^16 polls of 16.4 us)" % a.elapsed_time(b)


@pytest.mark.parametrize("tree", [False, True])
def test_positions_past_a_contiguous_cache_are_not_seen(tree):
    """A cache that ends inside a sequence which does not begin at its row 0, and before the last one: what append leaves out, attention
    does not see - not as rows of zeros either."""
    lens, ctx, short = [3, 40, 2], [50, 200, 10], 33
    s = S.Seqs(lens, ctx, 8, 2, 128, page=0, seed=23, extra_rows=2)
    s.cap = s.kv0_host[1] + ctx[1] + lens[1] - short
    s.kc[s.cap:], s.vc[s.cap:] = float("nan"), float("nan")
    bits = s.tree()[1] if tree else None
    out = s.attend(None if bits is None else torch.from_numpy(bits.view(np.int32)).to(DEV), gate=False)
    for i in range(3):
        r, m, x = slice(s.row0[i], s.row0[i] + lens[i]), lens[i], ctx[i]
        have = max(0, min(m + x, s.cap - s.kv0_host[i]))
        seen = torch.ones(m, m + x, dtype=torch.bool, device=DEV)
        if tree:
            seen[:, x:] = torch.tensor([[bool(bits[r][t, j // 32] >> np.uint32(j % 32) & 1) for j in range(m)] for t in range(m)], device=DEV)
        else:
            seen[:, x:] = torch.ones(m, m, dtype=torch.bool, device=DEV).tril()
        at = s.kv0_host[i] + torch.arange(have, device=DEV)
        ref, tol = S.formula(s.q[r, :1024].view(m, 8, 128).double(), s.k[at].double(), s.v[at].double(), seen[:, :have]) if have else (0.0, 0.0)
        assert ((out[r].view(m, 8, 128).double() - ref).abs() <= tol).all(), "sequence %d" % i
    assert (out[s.rows:] == -7).all()


def test_the_largest_hint_is_as_good_as_none():
    """max_pos at its largest splits the work as an unknown one does (how it is split shows in the last bits)."""
    a, b = (S.Seqs([1, 3], [9000, 2500], 8, 2, 128, seed=29, max_pos=hint) for hint in (0, 2 ** 31 - 1))
    assert torch.equal(a.attend().view(torch.int16), b.attend().view(torch.int16))


@pytest.mark.parametrize("spread", [0.0, 1.0])
@pytest.mark.parametrize("lens,ctx", [([1] * 80, 3000), ([1, 100], 1500)])
def test_a_tail_behind_a_position_that_takes_nearly_all_weight(lens, ctx, spread):
    """The first position has nearly all the weight and a value of zero, so the result is the others' sum: weights of 2^-25.5, or
    scattered about e^-17.  A weight is held as f16 of 2^7 times itself against the reference, which is the row's largest or less: off by
    2^-11 of itself or by 2^-32 of the largest weight; the sums, the scores' products (one product here, rounded once) and e^x add
    2^-18 of the magnitudes, as in the tests' formula; the result is rounded to f16."""
    s = S.Seqs(lens, [ctx] * len(lens), 8, 2, 128, seed=37, stale=0.0)
    g = torch.Generator(device=DEV).manual_seed(37)
    s.q.zero_()
    s.q[:, ::128] = 8.0   # the score is the key's first element / sqrt(2)
    s.k.zero_()
    s.k[:, :, 0] = (torch.randn(s.k.shape[:2], device=DEV, generator=g) * spread * 2 ** 0.5 + (25 - 17 * 2 ** 0.5) * (spread > 0)).half()
    s.v[:] = 1000.0 + 100 * torch.randn(s.v.shape, device=DEV, generator=g)
    for c in s.cells:
        s.k[c[0], :, 0], s.v[c[0]] = 25.0, 0.0
    s.kc, s.vc = s._pool(s.k), s._pool(s.v)
    out = s.attend(gate=False).view(-1, 8, 128)
    for i, n in enumerate(lens):
        r, c = slice(s.row0[i], s.row0[i] + n), s.cells[i].to(DEV)
        q, k, v = s.q[r].view(n, 8, 128).double(), s.k[c].double(), s.v[c].double()
        seen = torch.ones(n, ctx + n, dtype=torch.bool, device=DEV).tril(ctx)
        x = torch.einsum("thd,phd->htp", q, k.repeat_interleave(4, 1)) / 128 ** 0.5
        e = torch.exp(x - x.masked_fill(~seen, -torch.inf).amax(-1, keepdim=True)) * seen
        z, vv = e.sum(-1, keepdim=True), v.repeat_interleave(4, 1)
        ref, mag, all_v = (torch.einsum("htp,phd->thd", w, u) for w, u in ((e / z, vv), (e / z, vv.abs()), (seen / z, vv.abs())))
        tol = 2.0 ** -11 * ref.abs() + (2.0 ** -11 + 2.0 ** -18) * mag + 2.0 ** -32 * all_v + 2.0 ** -25
        assert ((out[r].double() - ref).abs() <= tol * (1 + 2.0 ** -10)).all(), "sequence %d: %.3g of the result" % (i, float(((out[r].double() - ref).abs() / ref).max()))


def test_outputs_as_far_apart_as_they_may_be():
    """Rows 2^24 halves apart, 128 of them a CTA: the last one's offset from the first is just below 2^31 halves."""
    s = S.Seqs([129], [3], 1, 1, 128, seed=41)
    base = torch.full((129 * (1 << 24),), -7.0, dtype=torch.float16, device=DEV)
    out = base.view(129, 1 << 24)
    s.attend(out=out)
    want = s.attend()
    assert torch.equal(out[:, :128].reshape(129, 128).view(torch.int16), want.view(torch.int16))
    assert (out[:, 128:1024] == -7).all() and (out[:, -64:] == -7).all()


@pytest.mark.parametrize("big", [300.0, 3000.0, 10000.0, 30000.0, 65504.0])
@pytest.mark.parametrize("lens,ctx", [([1, 40], [0, 300]), ([2], [9000])])
def test_scores_of_any_finite_size(lens, ctx, big):
    """Queries and keys whose elements are alike, so that a score is 128 times one product, exact in 32 bits, and up to 128^(1/2) 65504^2:
    some keys share the largest, the others are a sixteenth of it lower or negative, and weigh nothing.  The result is the mean of the
    values that share it, rounded as in the tests' formula (their weights are alike)."""
    s = S.Seqs(lens, ctx, 8, 2, 128, seed=43, stale=0.0)
    g = torch.Generator(device=DEV).manual_seed(43)
    s.q[:] = big
    pick = torch.rand(s.k.shape[:2], device=DEV, generator=g)
    s.k[:] = torch.where(pick < 0.3, big, torch.where(pick < 0.7, big * 15 / 16, -big)).half()[:, :, None]
    for sign in (1.0, -1.0):   # with the other sign the keys at -big are the largest
        s.q[:] = sign * big
        s.kc = s._pool(s.k)
        out = s.attend(gate=False).view(-1, 8, 128)
        for i, n in enumerate(lens):
            c = s.cells[i].to(DEV)
            x = (sign * s.k[c][:, :, 0].double()).repeat_interleave(4, 1)   # (the score over a positive factor) [positions][heads]
            v = s.v[c].double().repeat_interleave(4, 1)
            for t in range(n):
                seen = x[:ctx[i] + t + 1]
                w = (seen == seen.amax(0)).double()
                w = w / w.sum(0)
                ref, mag = torch.einsum("ph,phd->hd", w, v[:len(seen)]), torch.einsum("ph,phd->hd", w, v[:len(seen)].abs())
                got = out[s.row0[i] + t].double()
                assert ((got - ref).abs() <= (2.0 ** -11 * ref.abs() + (2.0 ** -11 + 2.0 ** -18) * mag + 2.0 ** -25) * (1 + 2.0 ** -10)).all(), (i, t, sign)
