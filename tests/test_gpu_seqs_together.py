"""The calls over several sequences as a server strings them together: a prompt, samples that share its pages, and windows of draft
trees whose accepted paths stay - one window captured, its replays with other trees and lengths.  What every sequence has seen
is kept beside it row by row, so pages, copies and moves are checked by what the attention reads through them."""
import numpy as np
import pytest
import torch

from sfnx_b200 import lib as L
from tests import seqs_util as S
from tests.seqs_util import DEV
from tests.test_gpu_seqs import BASE, EPS

pytestmark = pytest.mark.gpu

i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)   # noqa: E731
NSEQ, ROWS, PAGES, WIDTH, LAYERS, WORDS, VOCAB, ALT = 5, 48, 96, 30, 2, 2, 1000, 5


class Server:
    def __init__(self, nq, nkv, hd, page, seed):
        self.g = torch.Generator(device=DEV).manual_seed(seed)
        self.rng = np.random.default_rng(seed)
        self.nq, self.nkv, self.hd, self.page = nq, nkv, hd, page
        self.planes = [torch.full((PAGES, page, nkv, hd), float("nan"), dtype=torch.float16, device=DEV) for _ in range(2 * LAYERS)]
        self.bases = torch.tensor([p.data_ptr() for p in self.planes], dtype=torch.int64, device=DEV)
        self.ref, self.len, self.pos0 = (torch.zeros(n, dtype=torch.int32, device=DEV) for n in (PAGES, NSEQ, NSEQ))
        self.row0, self.err = torch.zeros(NSEQ + 1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
        self.pt = torch.full((NSEQ, WIDTH), -1, dtype=torch.int32, device=DEV)
        self.pool = L.PagePool(PAGES, page, self.ref.data_ptr(), NSEQ, self.pt.data_ptr(), WIDTH, self.len.data_ptr())
        self.geometry = L.KvPages(None, page * nkv * hd, page, 0, 0)
        self.work = torch.zeros(L.load().fnx_pages_scratch_bytes(L.byref(self.pool)), dtype=torch.uint8, device=DEV)
        self.seqs = L.Seqs(NSEQ, ROWS, self.row0.data_ptr(), self.pos0.data_ptr(), self.pt.data_ptr(), WIDTH, PAGES, None, 0)
        self.room = torch.zeros(L.load().fnx_attn_seqs_scratch_bytes(L.byref(self.seqs), nq, nkv, hd), dtype=torch.uint8, device=DEV)
        self.lp_work = torch.zeros(L.load().fnx_logprobs_scratch_bytes(VOCAB, ROWS, ALT), dtype=torch.uint8, device=DEV)
        f = lambda *shape: torch.zeros(shape, device=DEV)   # noqa: E731
        self.qg, self.k, self.v = [f(ROWS, nq, 2 * hd) for _ in range(LAYERS)], [f(ROWS, nkv, hd) for _ in range(LAYERS)], [f(ROWS, nkv, hd) for _ in range(LAYERS)]
        self.norm = 1.0 + 0.1 * torch.randn(hd, device=DEV, generator=self.g)
        self.q16 = [torch.zeros(ROWS, nq, hd, dtype=torch.float16, device=DEV) for _ in range(LAYERS)]
        self.out = [torch.zeros(ROWS, nq * hd, dtype=torch.float16, device=DEV) for _ in range(LAYERS)]
        self.add, self.parent = i32([0] * NSEQ), i32([-1] * ROWS)
        self.anc, self.depth = torch.zeros(ROWS, WORDS, dtype=torch.int32, device=DEV), torch.zeros(ROWS, dtype=torch.int32, device=DEV)
        self.logits, self.tok = f(ROWS, VOCAB), i32(np.zeros((ROWS, 1)))
        self.lse, self.entropy, self.lp, self.top = f(ROWS), f(ROWS), f(ROWS, 1), f(ROWS, ALT)
        self.top_i = i32(np.zeros((ROWS, ALT)))
        # what each sequence holds: [layer] (k, v) rows in order
        self.held = [[(torch.zeros(0, nkv, hd, device=DEV).double(),) * 2 for _ in range(LAYERS)] for _ in range(NSEQ)]

    def fork(self, source):
        a = i32(source)
        L.call("fnx_pages_fork", L.byref(self.pool), a.data_ptr(), None, self.work.data_ptr(), self.err.data_ptr(), L.stream())
        torch.cuda.synchronize()
        empty = (torch.zeros(0, self.nkv, self.hd, device=DEV).double(),) * 2
        self.held = [[self.held[s][i] if s >= 0 else empty for i in range(LAYERS)] for s in source]

    def window(self, tree):
        """The launches of one window: everything they read and write stays where it is."""
        e, st = self.err.data_ptr(), L.stream()
        L.call("fnx_pages_reserve", L.byref(self.pool), self.add.data_ptr(), self.pos0.data_ptr(), self.row0.data_ptr(), self.bases.data_ptr(), 2 * LAYERS,
               self.geometry, self.nkv, self.hd, self.work.data_ptr(), e, st)
        if tree:
            L.call("fnx_tree_masks", self.parent.data_ptr(), L.byref(self.seqs), self.anc.data_ptr(), WORDS, self.depth.data_ptr(), e, st)
        for i in range(LAYERS):
            kc, vc = self.planes[2 * i].data_ptr(), self.planes[2 * i + 1].data_ptr()
            L.call("fnx_attn_seqs_append", self.qg[i].data_ptr(), self.k[i].data_ptr(), self.v[i].data_ptr(), self.norm.data_ptr(), self.norm.data_ptr(), kc, vc, self.geometry,
                   L.byref(self.seqs), self.depth.data_ptr() if tree else None, self.q16[i].data_ptr(), EPS, L.Rope(BASE, 64), self.nq, self.nkv, self.hd, e, st)
            head = [self.q16[i].data_ptr(), self.nq * self.hd, self.qg[i].data_ptr(), kc, vc, self.geometry, L.byref(self.seqs)]
            tail = [self.out[i].data_ptr(), self.nq * self.hd, self.nq, self.nkv, self.hd, self.room.data_ptr(), st]
            L.call("fnx_attn_tree", *head, self.anc.data_ptr(), WORDS, *tail) if tree else L.call("fnx_attn_prompt", *head, *tail)
        L.call("fnx_logprobs", self.logits.data_ptr(), VOCAB, VOCAB, ROWS, 0, self.tok.data_ptr(), 1, ALT, self.lse.data_ptr(), self.entropy.data_ptr(), self.lp.data_ptr(),
               self.top.data_ptr(), self.top_i.data_ptr(), self.lp_work.data_ptr(), e, st)

    def fill(self, add, parents=None, agree=0.0):
        """A window's inputs; with probability `agree` the token after a node is one of its children's."""
        for x in self.qg + self.k + self.v + [self.logits]:
            x.copy_(torch.randn(x.shape, device=DEV, generator=self.g))
        self.add.copy_(i32(add))
        tok = self.rng.integers(0, VOCAB, ROWS)
        if parents:
            flat = [x for p in parents for x in p]
            self.parent.copy_(i32(flat + [-1] * (ROWS - len(flat))))
            at = 0
            for p in parents:
                for node in range(len(p)):
                    children = [i for i in range(len(p)) if p[i] == node]
                    if children and self.rng.random() < agree:
                        self.logits[at + node, int(tok[at + int(self.rng.choice(children))])] += 40.0
                at += len(p)
        self.tok.copy_(i32(tok[:, None]))
        for o in self.out:
            o.fill_(-7.0)

    def check(self, add, bits=None, depth=None):
        """The window's results; what it appended joins what the sequences hold."""
        torch.cuda.synchronize()
        assert int(self.err) == 0 and L.load().fnx_device_fault() == 0
        ends = np.concatenate([[0], np.cumsum(add)])
        table = self.pt.cpu().long()
        for s in range(NSEQ):
            r, n0 = slice(int(ends[s]), int(ends[s + 1])), len(self.held[s][0][0])
            m = add[s]
            p = torch.arange(n0, n0 + m)
            cell = (table[s][p // self.page] * self.page + p % self.page).to(DEV)
            seen = torch.ones(m, n0 + m, dtype=torch.bool, device=DEV)
            seen[:, n0:] = torch.ones(m, m, dtype=torch.bool, device=DEV).tril()
            if bits is not None:
                seen[:, n0:] = torch.tensor([[bool(bits[r][t, i // 32] >> np.uint32(i % 32) & 1) for i in range(m)] for t in range(m)], device=DEV).view(m, m)
            for i in range(LAYERS):
                new = [self.planes[2 * i + j].view(-1, self.nkv, self.hd)[cell].double() for j in (0, 1)]
                assert torch.equal(new[1], self.v[i][r].half().double())   # (a key's bits are the append's own tests')
                k, v = (torch.cat([old, x]) for old, x in zip(self.held[s][i], new))
                self.held[s][i] = (k, v)
                if not m:
                    continue
                o, tol = S.formula(self.q16[i][r].double(), k, v, seen)
                sig = torch.sigmoid(self.qg[i][r, :, self.hd:].double())
                tol = (tol * sig + 2.0 ** -25) * (1 + 2.0 ** -10)
                assert ((self.out[i][r].view(m, self.nq, self.hd).double() - o * sig).abs() <= tol).all(), "sequence %d, layer %d" % (s, i)
        assert all((o[int(ends[-1]):] == -7).all() for o in self.out)
        d = self.logits.double()
        want = torch.log_softmax(d, 1)
        # sums of at most 1000 terms in 32 bits and a logarithm, rounded against values up to 60 (the logprobs' own tests derive it)
        tol = 2.0 ** -24 * (VOCAB / 512 + 64) + 2.0 ** -18 + 2.0 ** -22 * 60
        assert ((self.lp.double() - want.gather(1, self.tok.long())).abs() <= tol).all()
        assert torch.equal(self.top_i.long(), torch.sort(self.logits, dim=1, descending=True, stable=True).indices[:, :ALT])

    def keep(self, add, parents):
        """Each tree's accepted path stays."""
        best, tok = self.top_i[:, 0].cpu().numpy(), self.tok[:, 0].cpu().numpy()
        lists, at = [], 0
        for p in parents:
            path = np.zeros(max(len(p), 1), np.int32)
            a = [np.ascontiguousarray(x, np.int32) for x in (tok[at:at + len(p)], p, best[at:at + len(p)])]
            n = L.load().fnx_accept_tree(*(x.ctypes.data for x in a), len(p), path.ctypes.data) if p else 0
            assert n >= (1 if p else 0)
            lists.append(path[:n].tolist())
            at += len(p)
        wide = max([len(x) for x in lists] + [1])
        a, b = i32([x + [0] * (wide - len(x)) for x in lists]), i32([len(x) for x in lists])
        L.call("fnx_pages_keep", L.byref(self.pool), self.pos0.data_ptr(), a.data_ptr(), wide, b.data_ptr(), self.bases.data_ptr(), 2 * LAYERS, self.geometry, self.nkv, self.hd,
               self.work.data_ptr(), self.err.data_ptr(), L.stream())
        torch.cuda.synchronize()
        for s, x in enumerate(lists):
            n0 = len(self.held[s][0][0]) - add[s]
            self.held[s] = [tuple(torch.cat([y[:n0], y[n0:][x]]) for y in layer) for layer in self.held[s]]
        return lists

    def check_pool(self):
        torch.cuda.synchronize()
        assert int(self.err) == 0
        table, count = self.pt.cpu().long(), np.zeros(PAGES, int)
        assert self.len.tolist() == [len(h[0][0]) for h in self.held]
        for s in range(NSEQ):
            n = len(self.held[s][0][0])
            pages = table[s][:-(-n // self.page)].tolist()
            assert (table[s][len(pages):] == -1).all()
            for x in pages:
                count[x] += 1
            p = torch.arange(n)
            cell = (table[s][p // self.page] * self.page + p % self.page).to(DEV)
            for i in range(LAYERS):
                for j in (0, 1):
                    assert torch.equal(self.planes[2 * i + j].view(-1, self.nkv, self.hd)[cell].double(), self.held[s][i][j])
        assert self.ref.tolist() == count.tolist()


@pytest.mark.parametrize("nq,nkv,hd,page", [(8, 2, 128, 8), (12, 2, 256, 64), (3, 3, 128, 24)])
def test_prompts_samples_and_draft_windows(nq, nkv, hd, page):
    s = Server(nq, nkv, hd, page, seed=page)
    add = [45, 0, 3, 0, 0]
    s.fill(add)
    s.window(tree=False)
    s.check(add)
    add = [1, 0, 47, 0, 0]   # a token, a chunk of a prompt
    s.fill(add)
    s.window(tree=False)
    s.check(add)
    s.check_pool()
    s.fork([0, 0, 2, 0, 2])   # three samples of one prompt, two of another
    s.check_pool()
    g, accepted = None, 0
    for turn in range(6):
        sizes = [[9, 12, 1, 16, 10], [48, 0, 0, 0, 0], [1, 1, 1, 1, 1], [0, 33, 2, 0, 13], [3, 3, 3, 3, 3], [7, 20, 11, 1, 5]][turn]
        parents = [S.parents(n, s.rng) if n else [] for n in sizes]
        bits = np.concatenate([S.ancestors(p, WORDS)[0] for p in parents if p])
        s.fill(sizes, parents, agree=0.8)
        if turn == 1:   # (the first window ran as it comes)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                s.window(tree=True)
        if g is None:
            s.window(tree=True)
        else:
            g.replay()
        s.check(sizes, bits)
        accepted += sum(len(x) > 1 for x in s.keep(sizes, parents))
        s.check_pool()
        if turn == 3:
            s.fork([3, 1, -1, 3, 2])   # a beam goes on twice, one ends
            s.check_pool()
    assert accepted > 5
