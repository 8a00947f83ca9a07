"""Calls over several sequences that share the GPU, a workspace or a pool with others: every row of every call is looked at."""
import pytest
import torch

from tests import seqs_util as S
from tests.seqs_util import DEV
from tests.test_gpu_pages import Pool
from tests.test_gpu_seqs import _check

pytestmark = pytest.mark.gpu


def test_every_row_of_calls_on_two_streams_at_once():
    a, b = S.Seqs([300, 1, 17], [900, 4000, 3], 24, 4, 256, seed=41), S.Seqs([1] * 9, [500 * i for i in range(9)], 8, 2, 128, seed=42)
    want = [x.attend() for x in (a, b)]
    for x, w in zip((a, b), want):
        _check(x, w)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.full_like(w, -7.0) for _ in range(6)] for w in want]
    scratch = [x.scratch() for x in (a, b)]
    torch.cuda.synchronize()
    for i in range(6):
        for x, st, o, w in zip((a, b), streams, outs, scratch):
            with torch.cuda.stream(st):
                x.attend(out=o[i], scratch=w)
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert all(torch.equal(w.view(torch.int16), x.view(torch.int16)) for x in o)


def test_two_captured_calls_share_a_workspace_whatever_the_lengths():
    """Graphs of two calls over one scratch, replayed in turn; lengths change, and change back, between the replays."""
    s = S.Seqs([40, 3, 21], [100, 0, 333], 8, 2, 256, seed=12)
    full = (s.lens, s.ctx, s.row0, s.rows, s.cells)
    scratch = s.scratch()
    out = [torch.full((s.total, 8 * 256), -7.0, dtype=torch.float16, device=DEV) for _ in range(2)]
    s.attend(out=out[0], scratch=scratch)   # warm-up
    torch.cuda.synchronize()
    graphs = []
    for o, gate in zip(out, (True, False)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.attend(out=o, scratch=scratch, gate=gate)
        graphs.append(g)
    less = ([10, 0, 8], [130, 3, 340])
    few = (less[0], less[1], [0, 10, 10, 18], 18, [c[:a + b] for c, a, b in zip(s.cells, *less)])
    for lens, ctx, row0, rows, cells in (few, full, few, full):
        s.lens, s.ctx, s.row0, s.rows, s.cells = lens, ctx, row0, rows, cells
        s.d_row0.copy_(torch.tensor(row0, dtype=torch.int32))
        s.d_pos0.copy_(torch.tensor(ctx, dtype=torch.int32))
        for o in out:
            o.fill_(-7.0)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        _check(s, out[0])
        _check(s, out[1], gate=False)


@pytest.mark.parametrize("rows", [1, 5, 64])
def test_reserve_takes_the_pages_that_it_needs_and_no_more(rows):
    p = Pool(400, rows, 4, 90, nplanes=2, seed=rows)
    page = lambda n: -(-n // rows)   # noqa: E731
    p.reserve([7, 0, 33, 1])
    assert int((p.ref > 0).sum()) == sum(page(n) for n in (7, 0, 33, 1))
    p.fork([0, 0, 2, 2])
    assert int((p.ref > 0).sum()) == page(7) + page(33)
    p.reserve([2, 2, 0, 5])   # of a page's two holders that both go on one copies it; where one stays, the other one copies
    copies = (7 % rows != 0) + (33 % rows != 0)
    fresh = 2 * (page(9) - page(7)) + page(38) - page(33)
    assert int((p.ref > 0).sum()) == page(7) + page(33) + copies + fresh
    assert int(p.err) == 0 and p.len.tolist() == [9, 9, 33, 38]
