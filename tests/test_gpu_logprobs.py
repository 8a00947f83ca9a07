"""Log probabilities, entropy and alternatives against 64 bits; ties, masked vocabularies, slices."""
import ctypes as C

import numpy as np
import pytest
import torch

from sfnx_b200 import lib as L

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _run(x, tok, k, v0=0, n=None, scratch=None):
    T, stride = x.shape
    n = n or stride
    ntok = tok.shape[1] if tok is not None else 0
    f = lambda *shape: torch.full(shape, -7.0, device=DEV)   # noqa: E731
    r = {"lse": f(T), "ent": f(T), "lp": f(T, ntok), "tv": f(T, k), "ti": torch.full((T, k), -7, dtype=torch.int32, device=DEV),
         "err": torch.zeros(1, dtype=torch.int32, device=DEV)}
    if scratch is None:
        scratch = torch.zeros(L.load().fnx_logprobs_scratch_bytes(n, T, k), dtype=torch.uint8, device=DEV)
    L.call("fnx_logprobs", x.data_ptr(), stride, n, T, v0, L.ptr(tok), ntok, k, r["lse"].data_ptr(), r["ent"].data_ptr(), r["lp"].data_ptr(), r["tv"].data_ptr(),
           r["ti"].data_ptr(), scratch.data_ptr(), r["err"].data_ptr(), L.stream())
    torch.cuda.synchronize()
    return r


def _reference(x):
    d = x.double()
    lse = torch.logsumexp(d, 1)
    p = torch.exp(d - lse[:, None])
    ent = -torch.where(p > 0, p * (d - lse[:, None]), 0.0).sum(1)
    return lse, ent


def _check(r, x, tok, k, v0=0):
    """A thread adds at most n / 512 / blocks terms in 32 bits (and rescales), then trees: under 2^-24 (n / 512 + 64) of z, and an
    exponential is off by 2^-22 + |x - m| 2^-24, at most 2^-18 for what weighs anything; the entropy's terms the same with weights
    |x - m| <= 100.  A difference of two 32-bit numbers is rounded once more."""
    n = x.shape[1]
    lse, ent = _reference(x)
    rel = 2.0 ** -24 * (n / 512 + 64) + 2.0 ** -18
    tol = rel + 2.0 ** -23 * lse.abs()
    assert ((r["lse"].double() - lse).abs() <= tol).all()
    assert ((r["ent"].double() - ent).abs() <= rel * (2 + ent)).all()
    if tok is not None:
        at = tok.long() - v0
        inside = (at >= 0) & (at < n)
        want = torch.where(inside, x.double().gather(1, at.clamp(0, n - 1)) - lse[:, None], -torch.inf)
        assert torch.equal(torch.isinf(r["lp"]), torch.isinf(want))
        fin = torch.isfinite(want)
        assert ((r["lp"].double() - want).abs()[fin] <= (tol[:, None] + 2.0 ** -23 * want.abs().nan_to_num(posinf=0.0))[fin]).all()
    if k:
        order = torch.sort(x + 0.0, dim=1, descending=True, stable=True)
        assert torch.equal(r["ti"].long(), order.indices[:, :k] + v0)
        want = order.values[:, :k].double() - lse[:, None]
        assert torch.equal(torch.isinf(r["tv"]), torch.isinf(want))
        fin = torch.isfinite(want)
        assert ((r["tv"].double() - want).abs()[fin] <= (tol[:, None] + 2.0 ** -23 * want.abs().nan_to_num(posinf=0.0))[fin]).all()


@pytest.mark.parametrize("T,n", [(1, 1), (1, 151936), (16, 151936), (3, 4097), (300, 33333), (295, 9000), (296, 9000), (5, 64), (2, 511), (700, 1000)])
@pytest.mark.parametrize("k", [0, 1, 5, 20, 64])
def test_logprobs(T, n, k):
    k = min(k, n)
    g = torch.Generator(device=DEV).manual_seed(T + n + k)
    x = torch.randn(T, n, device=DEV, generator=g) * 4
    tok = torch.randint(0, n, (T, 3), device=DEV, generator=g).to(torch.int32)
    tok[:, 1] = -1
    r = _run(x, tok, k)
    assert int(r["err"]) == 0
    _check(r, x, tok, k)


@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "masked", "few", "signed_zeros", "coarse", "large"])
@pytest.mark.parametrize("T,n,k", [(2, 151936, 64), (2, 20000, 1), (400, 9001, 20), (1, 8192, 7)])
def test_logprobs_orders_and_ties(kind, T, n, k):
    """Every value alike, in order (each batch exceeds all before it), most of the vocabulary masked, fewer finite values than
    alternatives, zeros of both signs, many ties, large logits."""
    g = torch.Generator(device=DEV).manual_seed(n + k)
    x = torch.randn(T, n, device=DEV, generator=g) * 3
    if kind == "equal":
        x[:] = 1.25
    elif kind == "rising":
        x = torch.linspace(-40, 40, n, device=DEV).repeat(T, 1)
    elif kind == "falling":
        x = torch.linspace(40, -40, n, device=DEV).repeat(T, 1)
    elif kind == "masked":
        x.masked_fill_(torch.rand(T, n, device=DEV, generator=g) < 0.97, -torch.inf)
    elif kind == "few":
        x[:, 3:] = -torch.inf
    elif kind == "signed_zeros":
        x = torch.where(torch.rand(T, n, device=DEV, generator=g) < 0.5, 0.0, -0.0)
    elif kind == "coarse":
        x = torch.round(x * 2) / 2
    elif kind == "large":
        x = x * 20 + 5000
    x = x.contiguous()
    tok = x.argmax(1, keepdim=True).to(torch.int32)
    r = _run(x, tok, k)
    assert int(r["err"]) == 0
    _check(r, x, tok, k)


def test_logprobs_slices_and_their_merge():
    """Two ragged slices of wider rows (a stride), tokens of the other slice -inf, merged on the host as the whole."""
    T, n, k, cut = 9, 5003, 20, 1777
    x = torch.randn(T, n, device=DEV) * 4
    x[4] = -torch.inf
    x[4, 10:15] = 1.0   # one slice of row 4 is nothing but -inf
    tok = torch.randint(0, n, (T, 2), device=DEV).to(torch.int32)
    parts = []
    for v0, m in ((0, cut), (cut, n - cut)):
        view = x[:, v0:]
        r = {"T": T}
        f = lambda *shape: torch.zeros(shape, device=DEV)   # noqa: E731
        r = [f(T), f(T), f(T, 2), f(T, k), torch.zeros(T, k, dtype=torch.int32, device=DEV)]
        err, scratch = torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(L.load().fnx_logprobs_scratch_bytes(m, T, k), dtype=torch.uint8, device=DEV)
        L.call("fnx_logprobs", view.data_ptr(), n, m, T, v0, tok.data_ptr(), 2, k, *(t.data_ptr() for t in r), scratch.data_ptr(), err.data_ptr(), L.stream())
        assert int(err) == (16 if v0 else 0)   # row 4 of the second slice has no distribution of its own
        parts.append([t.cpu() for t in r])
    host = [torch.stack([p[i] for p in parts]).contiguous() for i in range(5)]
    out = [torch.zeros_like(p) for p in parts[0]]
    L.call("fnx_logprobs_merge", *(t.data_ptr() for t in host), 2, T, 2, k, *(t.data_ptr() for t in out))
    lse, ent = _reference(x)
    assert torch.allclose(out[0].double(), lse.cpu(), rtol=0, atol=1e-5) and torch.allclose(out[1].double(), ent.cpu(), rtol=1e-5, atol=1e-5)
    want = (x.double().gather(1, tok.long()) - lse[:, None]).cpu()
    fin = torch.isfinite(want)
    assert torch.equal(fin, torch.isfinite(out[2])) and ((out[2].double() - want).abs()[fin] < 1e-5).all()
    order = torch.sort(x, dim=1, descending=True, stable=True)
    rows = [t for t in range(T) if t != 4]
    assert torch.equal(out[4].long()[rows], order.indices[:, :k].cpu()[rows])
    assert out[4][4, :5].tolist() == [10, 11, 12, 13, 14]


def test_logprobs_rows_without_a_distribution():
    x = torch.randn(6, 9000, device=DEV)
    x[1, 8999] = float("nan")
    x[2, 0] = float("inf")
    x[3] = -float("inf")
    tok = torch.zeros(6, 1, dtype=torch.int32, device=DEV)
    r = _run(x, tok, 4)
    assert int(r["err"]) == 16
    for t in (1, 2):
        assert all(torch.isnan(r[name][t]).all() for name in ("lse", "ent", "lp", "tv"))
    assert float(r["lse"][3]) == -np.inf and float(r["ent"][3]) == 0 and torch.isinf(r["lp"][3]).all() and torch.isinf(r["tv"][3]).all()
    assert r["ti"][3].tolist() == [0, 1, 2, 3]
    good = [0, 4, 5]
    _check({k: v[good] if k != "err" else v for k, v in r.items()}, x[good], tok[good], 4)


@pytest.mark.parametrize("T,n", [(1, 40000), (400, 9000)])
def test_logprobs_a_nan_among_masked_values(T, n):
    x = torch.full((T, n), -float("inf"), device=DEV)
    x[0, n - 7] = float("nan")
    r = _run(x, torch.zeros(T, 1, dtype=torch.int32, device=DEV), 3)
    assert int(r["err"]) == 16 and torch.isnan(r["lse"][0]) and r["ti"][0].tolist() == [-1] * 3
    assert (r["lse"][1:] == -float("inf")).all()


@pytest.mark.parametrize("shift", [1, 2, 3])
@pytest.mark.parametrize("T,n", [(3, 20001), (400, 4095), (1, 5)])
def test_logprobs_rows_that_begin_anywhere(T, n, shift):
    whole = torch.full((T * (n + 6) + 8,), 1e4, device=DEV)
    x = whole[shift:shift + T * (n + 6)].view(T, n + 6)
    x[:, :n] = torch.randn(T, n, device=DEV)
    k = min(n, 20)
    r = {"lse": torch.zeros(T, device=DEV), "ent": torch.zeros(T, device=DEV), "tv": torch.zeros(T, k, device=DEV), "ti": torch.zeros(T, k, dtype=torch.int32, device=DEV)}
    err, scratch = torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(L.load().fnx_logprobs_scratch_bytes(n, T, k), dtype=torch.uint8, device=DEV)
    L.call("fnx_logprobs", x.data_ptr(), n + 6, n, T, 0, None, 0, k, r["lse"].data_ptr(), r["ent"].data_ptr(), None, r["tv"].data_ptr(), r["ti"].data_ptr(),
           scratch.data_ptr(), err.data_ptr(), L.stream())
    assert int(err) == 0
    _check(r, x[:, :n].contiguous(), None, k)


def test_logprobs_one_scratch_for_calls_of_all_sizes_and_a_graph():
    scratch = torch.zeros(max(L.load().fnx_logprobs_scratch_bytes(n, T, 64) for T, n in ((16, 151936), (290, 40000), (1, 9000))), dtype=torch.uint8, device=DEV)
    for T, n, k in ((16, 151936, 64), (290, 40000, 3), (1, 9000, 20), (16, 151936, 0), (200, 40000, 64)):
        x = torch.randn(T, n, device=DEV)
        _check(_run(x, None, k, scratch=scratch), x, None, k)
    x, T, k = torch.randn(4, 50000, device=DEV), 4, 10
    lse, ti, tv, err = torch.zeros(4, device=DEV), torch.zeros(4, k, dtype=torch.int32, device=DEV), torch.zeros(4, k, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for _ in range(2):
            L.call("fnx_logprobs", x.data_ptr(), 50000, 50000, 4, 0, None, 0, k, lse.data_ptr(), None, None, tv.data_ptr(), ti.data_ptr(), scratch.data_ptr(),
                   err.data_ptr(), L.stream())
    for _ in range(3):
        x.normal_()
        g.replay()
        torch.cuda.synchronize()
        ref = _reference(x)[0]
        assert ((lse.double() - ref).abs() < 1e-4).all() and torch.equal(ti.long(), torch.topk(x, k, dim=1).indices)
