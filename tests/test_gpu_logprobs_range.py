"""Log probabilities of logits of any finite size, and of tokens that are all but certain."""
import pytest
import torch

from tests.test_gpu_logprobs import DEV, _run

pytestmark = pytest.mark.gpu
LOWEST, MOST = torch.finfo(torch.float32).min, torch.finfo(torch.float32).max


def _check(r, x, tok, k):
    """Against 64 bits, everything taken from the row's largest logit m.  The sum z of e^(x - m) is off by `rel` of itself (a thread adds at
    most n / 384 terms in 32 bits, in two sums, then trees: 2^-24 (n / 512 + 64) covers them; an exponential of what weighs anything
    2^-18), so its logarithm by as much.  A log probability (x - m) - log z is made in 64 bits and rounded once; lse too; the entropy's
    terms have weights |x - m| <= 100."""
    n, d = x.shape[1], x.double()
    m = d.amax(1, keepdim=True)
    lz = torch.log(torch.exp(d - m).sum(1, keepdim=True))
    p = torch.exp(d - m - lz)
    ent = -torch.where(p > 0, p * (d - m - lz), 0.0).sum(1)
    rel = 2.0 ** -24 * (n / 512 + 64) + 2.0 ** -18
    assert int(r["err"]) == 0
    lse = m + lz
    assert ((r["lse"].double() - lse[:, 0]).abs() <= rel + 2.0 ** -24 * lse[:, 0].abs()).all()
    assert ((r["ent"].double() - ent).abs() <= rel * (2 + ent)).all()

    def lp(got, at):
        want = d.gather(1, at.long()) - m - lz
        big = want < LOWEST   # (a difference of two logits may be past the type: -inf)
        assert torch.isinf(got[big]).all() and (got <= 0).all()
        assert ((got.double() - want).abs() <= rel + 2.0 ** -24 * want.abs())[~big].all()

    if tok is not None:
        lp(r["lp"], tok)
    order = torch.sort(x + 0.0, dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(r["ti"].long(), order)
    lp(r["tv"], order)


KINDS = ["one past 2^127", "all the lowest", "the lowest and normal", "all the largest", "scattered over the type", "near the lowest", "about 5000", "about -3e7"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,n,k", [(3, 40000, 20), (400, 3001, 5), (1, 70, 64)])
def test_logits_of_any_size(kind, T, n, k):
    g = torch.Generator(device=DEV).manual_seed(n)
    z = torch.randn(T, n, device=DEV, generator=g)
    if kind == "one past 2^127":
        x = z.clone()
        x[:, n // 2] = 2.4e38
    elif kind == "all the lowest":
        x = torch.full_like(z, LOWEST)
    elif kind == "the lowest and normal":
        x = torch.where(z > 1, z, LOWEST)
        x[:, 1] = 0.25
    elif kind == "all the largest":
        x = torch.full_like(z, MOST)
    elif kind == "scattered over the type":
        x = (torch.rand(T, n, device=DEV, generator=g) * 2 - 1) * MOST
    elif kind == "near the lowest":
        x = torch.where(z > 0, LOWEST, torch.nextafter(torch.tensor(LOWEST, device=DEV), torch.tensor(0.0, device=DEV)))
    elif kind == "about 5000":
        x = z * 3 + 5000
    else:
        x = (z * 4).round() * 2 - 3e7
    x = x.contiguous()
    tok = torch.randint(0, n, (T, 3), device=DEV, generator=g).to(torch.int32)
    tok[:, 0] = x.argmax(1)
    _check(_run(x, tok, k), x, tok, k)


@pytest.mark.parametrize("T,n", [(1500, 300), (4, 40000)])
def test_a_certain_token_has_no_positive_log_probability(T, n):
    g = torch.Generator(device=DEV).manual_seed(T)
    x = torch.randn(T, n, device=DEV, generator=g)
    at = torch.randint(0, n, (T, 1), device=DEV, generator=g)
    x.scatter_(1, at, x.gather(1, at) + torch.rand(T, 1, device=DEV, generator=g) * 30 + 8)
    tok = at.to(torch.int32)
    r = _run(x, tok, 5)
    _check(r, x, tok, 5)
    assert (r["lp"] <= 0).all() and (r["tv"] <= 0).all()
