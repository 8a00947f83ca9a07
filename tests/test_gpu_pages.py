"""Pages of a K/V pool: sharing, growth with copy on write, accepted paths moved together and pages given back, against a plain
simulation that keeps every position's contents; the invariants after every step."""
import numpy as np
import pytest
import torch

from sfnx_b200 import lib as L

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)   # noqa: E731


class Pool:
    def __init__(self, npages, rows, nseq, width, nplanes=4, nkv=2, hd=128, q8=False, pitch=0, seed=0):
        self.npages, self.rows, self.nseq, self.width, self.nkv, self.hd, self.q8 = npages, rows, nseq, width, nkv, hd, q8
        e = nkv * hd
        self.page = (rows * (e // 2 + e // 32) if q8 else rows * e) + pitch
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.planes = [torch.randint(-30000, 30000, (npages, self.page), dtype=torch.int16, device=DEV, generator=g) for _ in range(nplanes)]
        self.bases = torch.tensor([p.data_ptr() for p in self.planes], dtype=torch.int64, device=DEV)
        self.ref, self.len = torch.zeros(npages, dtype=torch.int32, device=DEV), torch.zeros(nseq, dtype=torch.int32, device=DEV)
        self.pt = torch.full((nseq, width), -1, dtype=torch.int32, device=DEV)
        self.pos0, self.row0 = torch.zeros(nseq, dtype=torch.int32, device=DEV), torch.zeros(nseq + 1, dtype=torch.int32, device=DEV)
        self.err = torch.zeros(1, dtype=torch.int32, device=DEV)
        self.pool = L.PagePool(npages, rows, self.ref.data_ptr(), nseq, self.pt.data_ptr(), width, self.len.data_ptr())
        self.scratch = torch.zeros(L.load().fnx_pages_scratch_bytes(L.byref(self.pool)), dtype=torch.uint8, device=DEV)
        self.g = L.KvPages(None, self.page, rows, 0, 1 if q8 else 0)

    def _tail(self):
        return self.scratch.data_ptr(), self.err.data_ptr(), L.stream()

    def fork(self, source, lim=None):
        self.a = (i32(source), None if lim is None else i32(lim))
        L.call("fnx_pages_fork", L.byref(self.pool), self.a[0].data_ptr(), L.ptr(self.a[1]), *self._tail())

    def reserve(self, add):
        self.b = i32(add)
        L.call("fnx_pages_reserve", L.byref(self.pool), self.b.data_ptr(), self.pos0.data_ptr(), self.row0.data_ptr(), self.bases.data_ptr(), len(self.planes),
               self.g, self.nkv, self.hd, *self._tail())

    def keep(self, lists, pos0=None):
        wide = max([len(x) for x in lists if x is not None] + [1])
        self.c = (i32([list(x or []) + [0] * (wide - len(x or [])) for x in lists]), i32([-1 if x is None else len(x) for x in lists]),
                  self.pos0 if pos0 is None else i32(pos0))
        L.call("fnx_pages_keep", L.byref(self.pool), self.c[2].data_ptr(), self.c[0].data_ptr(), wide, self.c[1].data_ptr(), self.bases.data_ptr(),
               len(self.planes), self.g, self.nkv, self.hd, *self._tail())

    def cells(self, plane):
        """[npages][rows][bytes of a row, its scales too]"""
        p = plane.view(torch.uint8).view(self.npages, -1).cpu().numpy()
        e = self.nkv * self.hd
        if not self.q8:
            return p[:, :self.rows * e * 2].reshape(self.npages, self.rows, e * 2)
        sc = self.rows * e
        return np.concatenate([p[:, :sc].reshape(self.npages, self.rows, e), p[:, sc:sc + self.rows * e // 16].reshape(self.npages, self.rows, e // 16)], axis=2)

    def write(self, s, lo, hi, rng):
        """New contents for positions lo .. hi - 1 of sequence s, in every plane; returns them."""
        pt = self.pt[s].cpu().numpy()
        out = []
        for plane in self.planes:
            p = plane.view(torch.uint8).view(self.npages, -1).cpu().numpy()
            e = self.nkv * self.hd
            rows = []
            for pos in range(lo, hi):
                page, r = pt[pos // self.rows], pos % self.rows
                assert 0 <= page < self.npages
                if self.q8:
                    row = rng.integers(0, 256, e + e // 16, dtype=np.uint8)
                    p[page, r * e:(r + 1) * e], p[page, self.rows * e + r * (e // 16):self.rows * e + (r + 1) * (e // 16)] = row[:e], row[e:]
                else:
                    row = rng.integers(0, 256, 2 * e, dtype=np.uint8)
                    p[page, r * 2 * e:(r + 1) * 2 * e] = row
                rows.append(row)
            plane.copy_(torch.from_numpy(p).view(torch.int16).view(plane.shape))
            out.append(rows)
        return out

    def check(self, want, err=0):
        """want[s][plane]: the rows sequence s holds."""
        assert int(self.err) == err
        pt, ref, ln = self.pt.cpu().numpy(), self.ref.cpu().numpy(), self.len.cpu().numpy()
        count = np.zeros(self.npages, int)
        planes = [self.cells(p) for p in self.planes]
        for s in range(self.nseq):
            held = -(-len(want[s][0]) // self.rows)
            assert ln[s] == len(want[s][0]) and (pt[s, held:] == -1).all()
            for page in pt[s, :held]:
                count[page] += 1
            for pl, cells in enumerate(planes):
                for pos, row in enumerate(want[s][pl]):
                    assert np.array_equal(cells[pt[s, pos // self.rows], pos % self.rows], row), "sequence %d, plane %d, position %d" % (s, pl, pos)
        assert np.array_equal(ref, count)


@pytest.mark.parametrize("rows,q8,pitch", [(8, False, 0), (5, True, 16), (64, False, 24), (1, False, 0), (24, True, 0)])
def test_a_long_run_of_forks_growth_and_kept_paths(rows, q8, pitch):
    rng = np.random.default_rng(rows)
    nseq, width = 7, max(4, 200 // rows)
    p = Pool(nseq * width, rows, nseq, width, nplanes=3, q8=q8, pitch=pitch, seed=rows)
    want = [[[] for _ in p.planes] for _ in range(nseq)]
    for step in range(12):
        # some sequences go on from others (cut short at times), some are emptied
        src = [int(rng.integers(-1, nseq)) if rng.random() < 0.35 else s for s in range(nseq)]
        lim = [int(rng.integers(0, 120)) if rng.random() < 0.3 else 10 ** 6 for _ in range(nseq)]
        p.fork(src, lim if step % 2 else None)
        want = [[list(want[a][pl][:lim[s] if step % 2 else None]) if a >= 0 else [] for pl in range(3)] for s, a in enumerate(src)]
        p.check(want)
        have = [len(w[0]) for w in want]
        add = [int(rng.integers(0, min(40, width * rows - h + 1))) if rng.random() < 0.8 else 0 for h in have]
        free = int((p.ref == 0).sum())
        p.reserve(add)
        assert p.pos0.tolist() == have and p.row0.tolist() == [0] + list(np.cumsum(add)) and free >= 0
        for s in range(nseq):
            for pl, new in enumerate(p.write(s, have[s], have[s] + add[s], rng)):
                want[s][pl] += new
        p.check(want)
        lists = [None if rng.random() < 0.3 else sorted(rng.choice(add[s], int(rng.integers(0, add[s] + 1)), replace=False).tolist()) for s in range(nseq)]
        p.keep(lists)
        want = [w if k is None else [pl[:have[s]] + [pl[have[s] + i] for i in k] for pl in w] for s, (w, k) in enumerate(zip(want, lists))]
        p.check(want)


def test_pages_are_handed_out_lowest_first_and_the_first_holder_keeps_a_shared_one():
    p = Pool(12, 4, 4, 5)
    p.reserve([6, 0, 0, 0])
    assert p.pt[0].tolist() == [0, 1, -1, -1, -1]
    p.fork([0, 0, 0, -1])
    p.reserve([1, 1, 5, 1])   # every holder of page 1 goes on: sequence 0 keeps it, 1 and 2 get copies before their new pages
    assert p.pt.tolist() == [[0, 1, -1, -1, -1], [0, 2, -1, -1, -1], [0, 3, 4, -1, -1], [5, -1, -1, -1, -1]]
    assert p.ref.tolist() == [3, 1, 1, 1, 1, 1, 0, 0, 0, 0, 0, 0]
    p.fork([0, 0, -1, 3])
    assert p.ref.tolist() == [2, 2, 0, 0, 0, 1, 0, 0, 0, 0, 0, 0]
    p.reserve([1, 0, 0, 0])   # sequence 1 holds the page without going on: sequence 0 has to leave it
    assert p.pt[:2].tolist() == [[0, 2, -1, -1, -1], [0, 1, -1, -1, -1]] and int(p.err) == 0
    assert p.row0.tolist() == [0, 1, 1, 1, 1]


def test_reserve_without_room_changes_nothing():
    for add, width, npages, word in (([9, 9, 9], 8, 6, 32), ([9, 17, 1], 4, 40, 32), ([3, -1, 3], 8, 40, 64)):
        p = Pool(npages, 4, 3, width)
        p.reserve([3, 5, 0])
        before = [t.clone() for t in (p.pt, p.ref, p.len)]
        p.reserve(add)
        assert int(p.err) == word and all(torch.equal(a, b) for a, b in zip(before, (p.pt, p.ref, p.len)))
        assert p.pos0.tolist() == [3, 5, 0] and p.row0.tolist() == [0, 0, 0, 0]
        p.err.zero_()
        p.reserve([1, 2, 1])   # the pool is as usable as before
        assert int(p.err) == 0 and p.len.tolist() == [4, 7, 1]


def test_keep_refuses_what_makes_no_sense_and_leaves_the_sequence():
    p = Pool(40, 4, 6, 8)
    p.reserve([10] * 6)
    p.fork([0, 1, 2, 3, 4, 4])   # sequences 4 and 5 share their pages
    before = [t.clone() for t in (p.pt, p.len)]
    p.keep([[0, 2, 2], [1, 10], [3, 1], [0, 1, 2, 3], [0, 1], None], pos0=[0, 0, 0, 8, 2, 0])
    assert int(p.err) == 64 and p.len.tolist() == [10, 10, 10, 10, 10, 10]
    assert torch.equal(p.pt, before[0])
    p.err.zero_()
    p.keep([None] * 4 + [[], None], pos0=[0, 0, 0, 0, 3, 0])   # nothing kept of what a shared page holds: a cut, which moves no row
    assert int(p.err) == 0 and p.len.tolist() == [10, 10, 10, 10, 3, 10]


def test_a_source_out_of_range_is_the_sequence_itself():
    p = Pool(10, 4, 2, 4)
    p.reserve([5, 6])
    before = p.pt.clone()
    p.fork([7, 0])
    assert int(p.err) == 64 and p.len.tolist() == [5, 5] and torch.equal(p.pt[0], before[0]) and torch.equal(p.pt[1], before[0])


@pytest.mark.parametrize("nseq,add,rows", [(4096, 3, 4), (1000, 70, 64), (1, 300000, 64), (3, 100000, 8)])
def test_reserve_of_many_sequences_and_long_ones(nseq, add, rows):
    width = -(-add // rows) + 2
    p = Pool(nseq * width, rows, nseq, width, nplanes=1, nkv=1)
    taken = torch.arange(0, p.npages, 3, device=DEV)[:nseq]   # pages that somebody else holds
    p.ref[taken] = 1
    p.reserve([add] * nseq)
    held = -(-add // rows)
    free = torch.ones(p.npages, dtype=torch.bool, device=DEV)
    free[taken] = False
    ids = free.nonzero()[:nseq * held, 0].to(torch.int32)
    assert int(p.err) == 0 and torch.equal(p.pt[:, :held].reshape(-1), ids) and (p.pt[:, held:] == -1).all()
    assert torch.equal(p.row0, torch.arange(nseq + 1, device=DEV, dtype=torch.int32) * add)
    p.fork([0] * nseq)
    assert (p.ref[ids[:held].long()] == nseq).all()
    p.fork([-1] * nseq)
    p.ref[taken] -= 1
    assert (p.ref == 0).all() and (p.pt == -1).all() and (p.len == 0).all()


@pytest.mark.parametrize("nseq,width", [(256, 37), (257, 13), (4096, 9)])
def test_forks_among_many_sequences(nseq, width):
    """Every sequence's source, and where it is cut, anywhere: tables, lengths and counts against the same done one by one."""
    rng = np.random.default_rng(nseq)
    rows = 4
    p = Pool(nseq * width, rows, nseq, width, nplanes=1, nkv=1)
    p.reserve(rng.integers(0, width * rows + 1, nseq))
    for step in range(3):
        pt, ln = p.pt.cpu().numpy(), p.len.cpu().numpy()
        src, lim = rng.integers(-1, nseq, nseq), rng.integers(0, width * rows + 5, nseq) if step else None
        p.fork(src, lim)
        want_len = np.where(src >= 0, ln[src], 0)
        if lim is not None:
            want_len = np.minimum(want_len, lim)
        want = np.where(np.arange(width)[None] < -(-want_len // rows)[:, None], pt[src], -1)
        assert int(p.err) == 0 and np.array_equal(p.len.cpu().numpy(), want_len) and np.array_equal(p.pt.cpu().numpy(), want)
        assert np.array_equal(p.ref.cpu().numpy(), np.bincount(want[want >= 0], minlength=p.npages))


@pytest.mark.parametrize("q8,nkv", [(False, 2), (True, 2), (False, 9)])
def test_long_paths_kept(q8, nkv):
    """Paths of hundreds of rows, rows wider than a block's threads take at once, all rows kept and none."""
    rng = np.random.default_rng(5)
    p = Pool(300, 8, 4, 70, nplanes=2, nkv=nkv, hd=256, q8=q8, seed=5)
    p.reserve([3, 0, 17, 1])
    want = [[rows for rows in p.write(s, 0, n, rng)] for s, n in enumerate([3, 0, 17, 1])]
    add = [500, 300, 129, 140]
    p.reserve(add)
    for s, n in enumerate(add):
        have = len(want[s][0])
        for pl, new in enumerate(p.write(s, have, have + n, rng)):
            want[s][pl] += new
    lists = [sorted(rng.choice(500, 333, replace=False).tolist()), list(range(300)), [], list(range(1, 140))]
    p.keep(lists)
    base = [3, 0, 17, 1]
    p.check([[pl[:base[s]] + [pl[base[s] + i] for i in k] for pl in want[s]] for s, k in enumerate(lists)])


def test_one_captured_step_replayed():
    """Growth, and the rows behind the first of them given back, captured once: the tables come back to where they were."""
    p = Pool(30, 8, 3, 8)
    p.reserve([5, 9, 17])
    torch.cuda.synchronize()
    keep, add = [[0], [0], [0]], [20, 3, 30]
    p.reserve(add)
    p.keep(keep)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        p.reserve(add) if False else L.call("fnx_pages_reserve", L.byref(p.pool), p.b.data_ptr(), p.pos0.data_ptr(), p.row0.data_ptr(), p.bases.data_ptr(),
                                            len(p.planes), p.g, p.nkv, p.hd, *p._tail())
        L.call("fnx_pages_keep", L.byref(p.pool), p.pos0.data_ptr(), p.c[0].data_ptr(), 1, p.c[1].data_ptr(), p.bases.data_ptr(), len(p.planes), p.g, p.nkv, p.hd,
               *p._tail())
    for i in range(4):
        g.replay()
        torch.cuda.synchronize()
        assert p.len.tolist() == [7 + i, 11 + i, 19 + i] and int(p.err) == 0
        assert int((p.ref > 0).sum()) == sum(-(-x // 8) for x in p.len.tolist())
