"""The attention over sequences at the ends of what it takes: units smaller than a box, runs of seconds."""
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
