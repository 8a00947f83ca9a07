"""Rows too wide for the kernels' 32-bit offsets inside a unit of work: refused on the host (no launch is reached, so no GPU is needed)."""
import pytest

from tests.test_seqs_refusals import P, _geometry, _seqs


@pytest.mark.parametrize("nq,nkv,out_stride,text", [
    (8, 2, (1 << 24) + 8, "2\\^24"), (8, 2, 1 << 30, "2\\^24"), (8, 2, (1 << 31) - 8, "2\\^24"),
    (1 << 17, 1 << 13, 1 << 24, "2\\^23"), (1 << 24, 1 << 20, (1 << 31) - 8, "2\\^23")])
def test_attention_of_rows_too_wide(fnx, nq, nkv, out_stride, text):
    sq, g, wide = _seqs(fnx), _geometry(fnx, page=64 * nkv * 128), (1 << 31) - 8
    for name, more in (("fnx_attn_prompt", ()), ("fnx_attn_tree", (P, 1))):
        with pytest.raises(fnx.FnxError, match=text):
            fnx.call(name, P, wide, None, P, P, g, fnx.byref(sq), *more, P, out_stride, nq, nkv, 128, P, None)


@pytest.mark.parametrize("nq", [1 << 17, 1 << 24, (1 << 31) - 16])
def test_append_of_rows_too_wide(fnx, nq):
    with pytest.raises(fnx.FnxError, match="2\\^23"):
        fnx.call("fnx_attn_seqs_append", P, P, P, P, P, P, P, _geometry(fnx, page=64 * (nq // 16) * 128), fnx.byref(_seqs(fnx)), None, P, 1e-6, fnx.Rope(1e4, 64), nq,
                 nq // 16, 128, P, None)
