"""The attention over sequences at the ends of what it takes."""
import pytest
import torch

from sfnx_b200 import lib as L
from tests import seqs_util as S
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
