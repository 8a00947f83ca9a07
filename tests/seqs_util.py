"""Sequences behind page tables for the tests of the entry points that take them: a cache whose pages lie in no order and hold
NaN wherever no live position is, the calls' structs, and the operators in 64 bits (test infrastructure)."""
import numpy as np
import torch

from sfnx_b200 import lib as L

DEV = "cuda:0"


def parents(n, rng):
    return [-1] + [int(rng.integers(max(0, i - 6), i)) for i in range(1, n)]


def ancestors(parent, words):
    """(mask words, depths) by walking to the root."""
    bits, depth = np.zeros((len(parent), words), np.uint32), np.zeros(len(parent), np.int32)
    for i in range(len(parent)):
        j, d = i, -1
        while j >= 0:
            bits[i, j // 32] |= np.uint32(1 << (j % 32))
            j, d = parent[j], d + 1
        depth[i] = d
    return bits, depth


def formula(q, k, v, seen):
    """(output, how far an f16 result may be off) in 64 bits, [rows][nq][hd], of q [rows][nq][hd] over k, v [positions][nkv][hd].

    A score is a sum of hd products in 32 bits: off by at most hd 2^-24 sum |q k| / sqrt(hd), call it d; e^x by twice that
    and 2^-20 for the exponential itself.  A weight is then rounded to f16: 2^-11 of itself, or 2^-25 where it is below
    2^-14, against a sum z of at least the exact one about the row's maximum.  The sum over the positions in 32 bits adds no
    more than 2^-20 of the sum of magnitudes (tiles of at most 256 terms, then one addition a tile: under 16 halvings
    of 2^-24 each for what the tests reach); the gated result is rounded to f16 once."""
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    hd, qpk = q.shape[2], q.shape[1] // k.shape[1]
    for h in range(q.shape[1]):
        kh, vh = k[:, h // qpk], v[:, h // qpk]
        w = q[:, h] @ kh.T / np.sqrt(hd)
        d = float((q[:, h].abs() @ kh.abs().T).max()) / np.sqrt(hd) * hd * 2.0 ** -24
        w = w.masked_fill(~seen, -torch.inf)
        top = w.amax(1, keepdim=True)
        e = torch.where(seen, torch.exp(w - torch.where(torch.isinf(top), 0.0, top)), 0.0)
        z = e.sum(1, keepdim=True)
        p = torch.where(z > 0, e / z, 0.0)
        o, mag = p @ vh, p @ vh.abs()
        small = torch.where(z > 0, 2.0 ** -25 * (seen.double() @ vh.abs()) / z, 0.0)
        out[:, h] = o
        tol[:, h] = 2.0 ** -11 * o.abs() + (2.0 ** -11 + 2 * d + 2.0 ** -19) * mag + small + 2.0 ** -25
    return out, tol


class Seqs:
    """lens new rows after ctx positions a sequence; page: rows a page (0: one contiguous cache)."""

    def __init__(self, lens, ctx, nq, nkv, hd, page=64, seed=0, pad=0, extra_rows=0, pitch=0, max_pos=None, stale=float("nan")):
        g = torch.Generator().manual_seed(seed)
        self.rng = np.random.default_rng(seed)
        self.lens, self.ctx, self.nq, self.nkv, self.hd, self.page = list(lens), list(ctx), nq, nkv, hd, page
        self.n, self.rows = len(lens), sum(lens)
        self.total = max(1, self.rows + extra_rows)
        self.row0 = [int(x) for x in np.concatenate([[0], np.cumsum(lens)])]
        ends = [a + b for a, b in zip(lens, ctx)]
        self.max_pos = max(ends + [1]) if max_pos is None else max_pos
        if page:
            held = [-(-e // page) for e in ends]
            self.npages, self.width = sum(held) + 3, max(held + [1]) + 1
            ids = torch.randperm(self.npages, generator=g)
            self.table = torch.full((self.n, self.width), -1, dtype=torch.int32)
            at = 0
            for i, h in enumerate(held):
                self.table[i, :h] = ids[at:at + h]
                at += h
            self.cap, self.pitch = 0, page * nkv * hd + pitch
            cells = self.npages * page
        else:
            self.npages, self.width, self.table = 0, 0, None
            gaps = [int(self.rng.integers(0, 5)) for _ in lens]
            self.kv0_host = [int(sum(ends[:i]) + sum(gaps[:i + 1])) for i in range(self.n)]
            cells = self.cap = max(1, sum(ends) + sum(gaps) + 2)
            self.pitch = 0
        live = torch.zeros(cells, dtype=torch.bool)
        self.cells = []
        for i, e in enumerate(ends):
            p = torch.arange(e)
            c = self.table[i].long()[p // page] * page + p % page if page else self.kv0_host[i] + p
            self.cells.append(c)
            live[c] = True
        self.live = live
        k, v = (torch.randn(cells, nkv, hd, generator=g).half() for _ in range(2))
        k[~live], v[~live] = stale, stale
        self.k, self.v = k.to(DEV), v.to(DEV)
        self.kc, self.vc = self._pool(self.k), self._pool(self.v)
        w = nq * hd + pad
        self.q = torch.randn(self.total, w, generator=g).half().to(DEV)
        self.qg = torch.randn(self.total, nq, 2 * hd, generator=g).to(DEV)
        self.stride = w
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)   # noqa: E731
        self.d_row0, self.d_pos0 = i32(self.row0), i32(self.ctx)
        self.d_table = self.table.to(DEV) if page else None
        self.d_kv0 = None if page else i32(self.kv0_host)
        self.err = torch.zeros(1, dtype=torch.int32, device=DEV)

    def _pool(self, x):
        """The rows as the pool holds them: pages self.pitch halves apart."""
        if not self.page:
            return x.clone()
        pool = torch.full((self.npages, self.pitch), float("nan"), dtype=torch.float16, device=DEV)
        pool[:, :self.page * self.nkv * self.hd] = x.view(self.npages, -1)
        return pool

    def rows_of(self, pool):
        """The pool's rows [cells][nkv][hd]."""
        x = pool[:, :self.page * self.nkv * self.hd] if self.page else pool
        return x.reshape(-1, self.nkv, self.hd)

    def seqs(self):
        return L.Seqs(self.n, self.total, self.d_row0.data_ptr(), self.d_pos0.data_ptr(), L.ptr(self.d_table), self.width, self.npages, L.ptr(self.d_kv0),
                      self.max_pos)

    def geometry(self):
        return L.KvPages(None, self.pitch, self.page, self.cap, 0)

    def scratch(self, fill=0xFF):
        n = L.load().fnx_attn_seqs_scratch_bytes(L.byref(self.seqs()), self.nq, self.nkv, self.hd)
        return torch.full((max(n, 16),), fill, dtype=torch.uint8, device=DEV)

    def tree(self, words=None):
        """Random parents of every sequence's rows; (parents, masks, depths) of all rows, and the masks on the device."""
        words = words or max(1, -(-max(self.lens + [1]) // 32))
        par = [parents(n, self.rng) if n else [] for n in self.lens]
        bits, depth = zip(*[ancestors(p, words) if p else (np.zeros((0, words), np.uint32), np.zeros(0, np.int32)) for p in par])
        self.words = words
        return [x for p in par for x in p], np.concatenate(bits), np.concatenate(depth)

    def attend(self, anc=None, gate=True, out=None, scratch=None, out_pad=0, call=None):
        """The entry point's output rows [total][nq hd + out_pad] (rows nobody writes keep -7)."""
        if out is None:
            out = torch.full((self.total, self.nq * self.hd + out_pad), -7.0, dtype=torch.float16, device=DEV)
        scratch = self.scratch() if scratch is None else scratch
        args = [self.q.data_ptr(), self.stride, self.qg.data_ptr() if gate else None, self.kc.data_ptr(), self.vc.data_ptr(), self.geometry(), L.byref(self.seqs())]
        tail = [out.data_ptr(), out.shape[1], self.nq, self.nkv, self.hd, scratch.data_ptr(), L.stream()]
        if anc is None:
            L.call("fnx_attn_prompt", *args, *tail)
        else:
            L.call("fnx_attn_tree", *args, anc.data_ptr(), self.words, *tail)
        return out

    def reference(self, bits=None, gate=True):
        """formula() of every sequence's rows, gated: (output, how far an f16 result may be off), [rows][nq][hd]."""
        out = torch.zeros(self.rows, self.nq, self.hd, dtype=torch.float64, device=DEV)
        tol = torch.zeros_like(out)
        for s in range(self.n):
            m, x = self.lens[s], self.ctx[s]
            if not m:
                continue
            c = self.cells[s].to(DEV)
            r = slice(self.row0[s], self.row0[s] + m)
            q = self.q[r, :self.nq * self.hd].view(m, self.nq, self.hd).double()
            seen = torch.ones(m, x + m, dtype=torch.bool, device=DEV)
            if bits is None:
                seen[:, x:] = torch.ones(m, m, dtype=torch.bool, device=DEV).tril()
            else:
                b = bits[r]
                seen[:, x:] = torch.tensor([[bool(i // 32 < b.shape[1] and b[t, i // 32] >> np.uint32(i % 32) & 1) for i in range(m)] for t in range(m)], device=DEV)
            out[r], tol[r] = formula(q, self.k[c].double(), self.v[c].double(), seen)
        if gate:
            sig = torch.sigmoid(self.qg[:self.rows, :, self.hd:].double())
            out, tol = out * sig, tol * sig + 2.0 ** -25
        return out, tol * (1 + 2.0 ** -10)
