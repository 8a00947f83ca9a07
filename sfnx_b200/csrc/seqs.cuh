// Several sequences' packed rows (FnxSeqs): where a row belongs and where its position lies in the cache; shared by the rows'
// append and their attention.
#pragma once

#include "common.cuh"

namespace fnxk {

constexpr unsigned SQ_ERR_ROOM = 32u, SQ_ERR_VALUE = 64u;

// The sequence of row t: the last one that begins at or before it (a warp looks at 32 starts a step); -1 when the row lies
// behind the last sequence or before the first.  Called by a converged warp.
__device__ __forceinline__ int sq_find(const int* __restrict__ row0, int nseq, int t) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = nseq;
    while (true) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        const unsigned in = __ballot_sync(0xffffffffu, at < hi && row0[at] <= t);
        const int c = __popc(in);   // the starts ascend
        if (c == 0) return -1;
        lo += (c - 1) * step;
        hi = min(hi, lo + step);
        if (step == 1) break;
    }
    return t < row0[lo + 1] ? lo : -1;
}

// The cache row of position pos of sequence s; -1 where it has none
__device__ __forceinline__ long long sq_cell(const FnxSeqs& sq, const FnxKvPages& g, int s, int pos) {
    if (pos < 0) return -1;
    if (!sq.pt) {
        const long long r = (long long) (sq.kv0 ? sq.kv0[s] : 0) + pos;
        return r >= 0 && r < g.cap ? r : -1;
    }
    const int j = pos / g.rows;
    if (j >= sq.pt_stride) return -1;
    const int page = sq.pt[(size_t) s * sq.pt_stride + j];
    return page >= 0 && page < sq.npages ? (long long) page * g.rows + pos % g.rows : -1;
}
// the first element of cache row `cell` (row_elems elements a row)
__device__ __forceinline__ size_t sq_at(const FnxSeqs& sq, const FnxKvPages& g, long long cell, size_t row_elems) {
    return sq.pt ? (size_t) (cell / g.rows) * g.page + (size_t) (cell % g.rows) * row_elems : (size_t) cell * row_elems;
}

__device__ __forceinline__ unsigned sq_pack(float lo, float hi) {   // both rounded to f16 by one instruction
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&h);
}

inline int sq_check(const FnxSeqs* sq, const FnxKvPages& g, int nq, int nkv, int hd, const char* what) {
    FNX_REQUIRE(sq && sq->row0 && sq->pos0, "%s: a null buffer", what);
    FNX_REQUIRE(sq->nseq >= 1 && sq->rows >= 1, "%s: %d rows of %d sequences", what, sq->rows, sq->nseq);
    FNX_REQUIRE(hd == 128 || hd == 256, "%s: head dim %d (128 or 256)", what, hd);
    FNX_REQUIRE(nkv >= 1 && nq >= 1 && nq % nkv == 0 && nq / nkv <= 16, "%s: %d query heads over %d KV heads", what, nq, nkv);
    FNX_REQUIRE((long long) nq * hd <= 1 << 23, "%s: rows of %d heads of %d (2^23 values at most)", what, nq, hd);
    FNX_REQUIRE(!g.q8, "%s: int8 rows are not taken (f16 only)", what);
    FNX_REQUIRE(sq->max_pos >= 0, "%s: max_pos %d", what, sq->max_pos);
    if (sq->pt) {
        FNX_REQUIRE(sq->pt_stride >= 1 && sq->npages >= 1 && g.rows >= 1, "%s: tables of %d, %d pages of %d rows", what, sq->pt_stride, sq->npages, g.rows);
        FNX_REQUIRE(g.page >= (size_t) g.rows * nkv * hd && g.page % 8 == 0, "%s: a page of %zu halves for %d rows of %d (a multiple of 8)", what, g.page, g.rows,
                    nkv * hd);
        FNX_REQUIRE((long long) g.rows * sq->pt_stride < (1ll << 31), "%s: a table of %d pages of %d rows holds 2^31 positions or more", what, sq->pt_stride,
                    g.rows);
    } else {
        FNX_REQUIRE(g.cap >= 1, "%s: a cache without page tables needs its row count (cap)", what);
    }
    return 0;
}

}  // namespace fnxk
