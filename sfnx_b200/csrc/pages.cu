// The pages of a K/V pool and the sequences' tables: sharing, growth with copy on write, an accepted path's rows moved
// together, and what nobody names any more free again (no counterpart in the reference, whose host keeps its tables).
//
// State is what the header says: a reference count a page, a table and a length a sequence.  Every result is a function of
// that state alone: reference counts are sums of integers, free pages are handed out lowest first in the sequences' order,
// and which holder of a shared page keeps it is the lowest, so no order of atomics shows.
// The tables are a few thousand words: what these calls cost is the latency of a handful of dependent loads and launches, so
// loads go out before their use is known and divisions are 32 bits wide; the row copies are DRAM's.  Seven forks and their
// copies of a partly filled page in 24 planes: 12.1 us (three launches; in reserve six dependent loads and four barriers of one
// block); growth of 32 sequences and their accepted paths in 4 planes: 14.7.
#include <algorithm>
#include <climits>

#include "common.cuh"
#include "moe_internal.cuh"

namespace fnxk {

constexpr int PG_SEQS = 4096, PG_THREADS = 1024, PG_WARPS = PG_THREADS / 32, PG_PER = PG_SEQS / PG_THREADS;
constexpr unsigned PG_ERR_ROOM = 32u, PG_ERR_VALUE = 64u;

// the scratch's words: a header (jobs of the copy; blocks of a fork that have the lengths, zero between calls), then per page:
// holders of a tail page in this call, the complement of the lowest of them (both zero between calls), the free list; per
// sequence: copy jobs (from, to, rows), the verdict
struct PgScratch {
    int *njobs, *holders, *lowest, *free_list, *jobs, *verdict;
    unsigned* seen;
};
__host__ __device__ inline PgScratch pg_scratch(const FnxPagePool& p, void* scratch) {
    int* w = (int*) scratch;
    PgScratch s;
    s.njobs = w, s.seen = (unsigned*) w + 1, w += 4;
    s.holders = w, w += p.npages;
    s.lowest = w, w += p.npages;
    s.free_list = w, w += p.npages;
    s.jobs = w, w += 3 * (size_t) p.nseq;
    s.verdict = w;
    return s;
}
__device__ __forceinline__ unsigned pg_pages(const FnxPagePool& p, unsigned len) {   // pages that len < 2^32 positions need
    const unsigned rows = (unsigned) p.rows, q = len / rows;
    return q + (q * rows != len);
}
__device__ __forceinline__ int pg_held(const FnxPagePool& p, int len) {   // at most the table's
    return min((int) pg_pages(p, (unsigned) max(len, 0)), p.pt_stride);
}
__device__ __forceinline__ bool pg_valid(const FnxPagePool& p, int page) { return page >= 0 && page < p.npages; }

// how a pool's rows lie: f16 rows are one run; int8 rows are their values' run and, after the page's values, their scales'
struct PgRows {
    size_t page_bytes, row_bytes, scale_at, scale_bytes;   // a page's pitch, a row's, the scales' start in a page (0: none), a row's scales
};
__host__ inline PgRows pg_rows(const FnxPagePool& p, const FnxKvPages& g, int nkv, int hd) {
    const size_t e = (size_t) nkv * hd;
    if (g.q8) return PgRows{g.page * 2, e, (size_t) p.rows * e, e / 32 * 2};
    return PgRows{g.page * 2, e * 2, 0, 0};
}

// ---------------------------------------------------------------- fork
// A sequence's new table is another's old one, column by column: block i has 2^shift columns of all sequences in shared memory
// before it writes one.  The lengths are one column for all blocks, so the last block to have read them writes them.
__global__ void __launch_bounds__(256) k_pages_fork(const FnxPagePool p, const int* __restrict__ from, const int* __restrict__ lim, int shift, void* scratch,
                                                    unsigned* err) {
    extern __shared__ int pf_sm[];
    __shared__ bool last;
    const PgScratch w = pg_scratch(p, scratch);
    int *src = pf_sm, *held = src + p.nseq, *now_held = held + p.nseq, *now_len = now_held + p.nseq, *was = now_len + p.nseq;
    const int j0 = (int) blockIdx.x << shift, n = p.nseq << shift, mask = (1 << shift) - 1;
    pdl_wait();
    pdl_go();
    for (int i = threadIdx.x; i < n; i += 256) {
        const int j = j0 + (i & mask);
        was[i] = j < p.pt_stride ? p.pt[(size_t) (i >> shift) * p.pt_stride + j] : -1;
    }
    for (int s = threadIdx.x; s < p.nseq; s += 256) {
        int f = from[s];
        if (f >= p.nseq) {
            if (blockIdx.x == 0) atomicOr(err, PG_ERR_VALUE);
            f = s;
        }
        int len = f < 0 ? 0 : max(p.len[f], 0);
        if (lim) len = min(len, max(lim[s], 0));
        src[s] = f, held[s] = pg_held(p, p.len[s]), now_held[s] = pg_held(p, len), now_len[s] = len;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicAdd(w.seen, 1u) == gridDim.x - 1;
    }
    for (int i = threadIdx.x; i < n; i += 256) {
        const int s = i >> shift, c = i & mask, j = j0 + c;
        if (j >= p.pt_stride) continue;
        const int before = j < held[s] ? was[i] : -1, now = j < now_held[s] ? was[(src[s] << shift) + c] : -1;
        if (before != now) {
            if (pg_valid(p, now)) atomicAdd(&p.ref[now], 1);
            if (pg_valid(p, before)) atomicSub(&p.ref[before], 1);
        }
        if (was[i] != now) p.pt[(size_t) s * p.pt_stride + j] = now;
    }
    __syncthreads();
    if (!last) return;
    for (int s = threadIdx.x; s < p.nseq; s += 256) p.len[s] = now_len[s];
    if (threadIdx.x == 0) *w.seen = 0u;
}

// ---------------------------------------------------------------- reserve
// Sums that stop at a cap of at most 2^31 (associative over values up to it, so their order is free)
__device__ __forceinline__ unsigned pg_add(unsigned a, unsigned b, unsigned cap) { return min(a + b, cap); }
// exclusive sums over the block of two values a thread, in ascending thread order; totals in t0, t1; flags: every thread's or'ed
__device__ __forceinline__ void pg_scan2(unsigned& a, unsigned& b, unsigned cap_a, unsigned cap_b, unsigned& flags, unsigned& t0, unsigned& t1, unsigned (*sh)[4]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto scan = [&](unsigned& x, unsigned cap) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x = pg_add(x, y, cap);
        }
    };
    auto before = [&](unsigned x, int at) {   // what lies before lane `at`
        const unsigned y = __shfl_sync(0xffffffffu, x, (at - 1) & 31);
        return at ? y : 0u;
    };
    unsigned sa = min(a, cap_a), sb = min(b, cap_b);
    scan(sa, cap_a), scan(sb, cap_b);
    flags = __reduce_or_sync(0xffffffffu, flags);
    if (lane == 31) *reinterpret_cast<uint4*>(sh[warp]) = make_uint4(sa, sb, flags, 0u);
    const unsigned own_a = __shfl_up_sync(0xffffffffu, sa, 1), own_b = __shfl_up_sync(0xffffffffu, sb, 1);
    __syncthreads();
    const uint4 all = *reinterpret_cast<const uint4*>(sh[lane]);   // (PG_WARPS = 32)
    unsigned wa = all.x, wb = all.y;
    scan(wa, cap_a), scan(wb, cap_b);
    flags = __reduce_or_sync(0xffffffffu, all.z);
    t0 = __shfl_sync(0xffffffffu, wa, 31), t1 = __shfl_sync(0xffffffffu, wb, 31);
    a = pg_add(before(wa, warp), lane ? own_a : 0u, cap_a), b = pg_add(before(wb, warp), lane ? own_b : 0u, cap_b);
}

constexpr int PG_NEAR = 2048;   // places of the list of pages handed out that lie in shared memory
__global__ void __launch_bounds__(PG_THREADS) k_pages_reserve(const FnxPagePool p, const int* __restrict__ add, int* pos0, int* row0, void* scratch, unsigned* err) {
    const PgScratch w = pg_scratch(p, scratch);
    __shared__ __align__(16) unsigned sh[PG_WARPS][4];
    __shared__ int first[PG_SEQS], near[PG_NEAR], wcount[PG_WARPS];   // first: a sequence's first place in the list of pages handed out
    __shared__ unsigned fresh[PG_SEQS];                                // where its new pages begin in its table, times two, + 1: after a copy
    __shared__ unsigned njobs_s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, per = (p.nseq + PG_THREADS - 1) / PG_THREADS;
    if (tid == 0) njobs_s = 0u;
    pdl_wait();
    pdl_go();
    auto ask_refs = [&](int q0, int* ref) {   // a warp has 128 neighbouring pages of 4 * PG_THREADS
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int q = q0 + warp * 128 + k * 32 + lane;
            ref[k] = q < p.npages ? p.ref[q] : 1;
        }
    };
    int ref[4];
    ask_refs(0, ref);
    // ---- what each sequence holds and wants; thread i has `per` neighbouring sequences
    int len[PG_PER], more[PG_PER], tail[PG_PER], want[PG_PER], refs[PG_PER];
    bool bad = false, room = true;
#pragma unroll
    for (int k = 0; k < PG_PER; ++k) {
        const int s = tid * per + k;
        len[k] = more[k] = want[k] = refs[k] = 0, tail[k] = -1;
        if (k >= per || s >= p.nseq) continue;
        len[k] = max(p.len[s], 0), more[k] = add[s];
    }
#pragma unroll
    for (int k = 0; k < PG_PER; ++k) {
        const int s = tid * per + k;
        if (k >= per || s >= p.nseq) continue;
        if (more[k] < 0) bad = true;
        else if (pg_pages(p, (unsigned) len[k] + (unsigned) more[k]) > (unsigned) p.pt_stride) room = false;
        else if (more[k] > 0 && (unsigned) len[k] % (unsigned) p.rows) {
            tail[k] = p.pt[(size_t) s * p.pt_stride + len[k] / p.rows];
            if (!pg_valid(p, tail[k])) room = false, tail[k] = -1;
            else {
                atomicAdd(&w.holders[tail[k]], 1), atomicMax(&w.lowest[tail[k]], INT_MAX - s);
                refs[k] = p.ref[tail[k]];
            }
        }
    }
    __threadfence_block();
    __syncthreads();
    bool copy[PG_PER];
    unsigned a = 0u, b = 0u, pages, rows, flags = (bad ? 1u : 0u) | (room ? 0u : 2u);
    const unsigned cap_pages = (unsigned) p.npages + 1u, cap_rows = 1u << 31;
#pragma unroll
    for (int k = 0; k < PG_PER; ++k) {
        const int s = tid * per + k;
        copy[k] = false;
        if (k >= per || s >= p.nseq) continue;
        if (tail[k] >= 0) {
            const int holders = __ldcg(&w.holders[tail[k]]), lowest = __ldcg(&w.lowest[tail[k]]);
            copy[k] = refs[k] > holders || lowest != INT_MAX - s;
        }
        if (more[k] >= 0 && room)
            want[k] = (int) (pg_pages(p, (unsigned) len[k] + (unsigned) more[k]) - pg_pages(p, (unsigned) len[k])) + (copy[k] ? 1 : 0);
        a = pg_add(a, min((unsigned) want[k], cap_pages), cap_pages), b = pg_add(b, more[k] > 0 ? (unsigned) more[k] : 0u, cap_rows);
    }
    pg_scan2(a, b, cap_pages, cap_rows, flags, pages, rows, sh);   // (everyone has looked at the holders when it returns)
#pragma unroll
    for (int k = 0; k < PG_PER; ++k)
        if (tail[k] >= 0) w.holders[tail[k]] = 0, w.lowest[tail[k]] = 0;
    bad = flags & 1u, room = !(flags & 2u) && rows < cap_rows;
    // ---- the lowest free pages, as many as are wanted
    unsigned got = 0u;
    if (room && !bad)
        for (int q0 = 0; q0 < p.npages && got < pages; q0 += 4 * PG_THREADS) {
            if (q0) ask_refs(q0, ref);
            unsigned is[4];
            int mine = 0, before[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) is[k] = __ballot_sync(0xffffffffu, ref[k] == 0), before[k] = mine, mine += __popc(is[k]);
            if (lane == 0) wcount[warp] = mine;
            __syncthreads();
            const int others = wcount[lane];   // (PG_WARPS = 32)
            unsigned below = got + __reduce_add_sync(0xffffffffu, lane < warp ? others : 0);
            got += __reduce_add_sync(0xffffffffu, others);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const unsigned at = below + before[k] + __popc(is[k] & ((1u << lane) - 1u));
                if ((is[k] >> lane & 1u) && at < pages) (at < PG_NEAR ? near[at] : w.free_list[at]) = q0 + warp * 128 + k * 32 + lane;
            }
            __syncthreads();
        }
    const bool ok = room && !bad && got >= pages;
    if (!ok) {   // nothing changes
#pragma unroll
        for (int k = 0; k < PG_PER; ++k) {
            const int s = tid * per + k;
            if (k < per && s < p.nseq) pos0[s] = len[k], row0[s] = 0;
        }
        if (tid == 0) {
            row0[p.nseq] = 0, *w.njobs = 0;
            atomicOr(err, (bad ? PG_ERR_VALUE : 0u) | (!bad || !room ? PG_ERR_ROOM : 0u));
        }
        return;
    }
    auto handed = [&](int i) { return i < PG_NEAR ? near[i] : w.free_list[i]; };
    // ---- the lengths and the copies, then the new entries: place i of the list belongs to the last sequence that begins at or before it
#pragma unroll
    for (int k = 0; k < PG_PER; ++k) {
        const int s = tid * per + k;
        if (k >= per || s >= p.nseq) continue;
        first[s] = (int) a, fresh[s] = 2u * pg_pages(p, (unsigned) len[k]) + (copy[k] ? 1u : 0u);
        pos0[s] = len[k], row0[s] = (int) b;
        p.len[s] = len[k] + more[k];
        if (copy[k]) {
            const int page = handed((int) a);
            p.pt[(size_t) s * p.pt_stride + len[k] / p.rows] = page;
            p.ref[page] = 1;
            atomicSub(&p.ref[tail[k]], 1);
            const unsigned at = atomicAdd(&njobs_s, 1u);
            w.jobs[3 * at] = tail[k], w.jobs[3 * at + 1] = page, w.jobs[3 * at + 2] = len[k] % p.rows;
        }
        a += want[k], b += more[k];
    }
    __syncthreads();
    if (tid == 0) row0[p.nseq] = (int) rows, *w.njobs = (int) njobs_s;
    for (int i = tid; i < (int) pages; i += PG_THREADS) {
        int lo = 0, hi = p.nseq;   // first[lo] <= i
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (first[mid] <= i) lo = mid;
            else hi = mid;
        }
        const int j = i - first[lo] - (int) (fresh[lo] & 1u);
        if (j < 0) continue;
        const int page = handed(i);
        p.pt[(size_t) lo * p.pt_stride + (fresh[lo] >> 1) + j] = page;
        p.ref[page] = 1;
    }
}

// the rows so far of the pages that reserve copies: block (job, plane, piece of PG_PIECE bytes of a page)
constexpr int PG_PIECE = 32768;
__global__ void __launch_bounds__(256) k_pages_copy(const FnxPagePool p, void* const* __restrict__ planes, const PgRows r, void* scratch) {
    const PgScratch w = pg_scratch(p, scratch);
    pdl_wait();
    pdl_go();
    // a first job's words (there are as many places as sequences) together with the number of jobs
    const int n = *w.njobs;
    int from = w.jobs[3 * blockIdx.x], to = w.jobs[3 * blockIdx.x + 1], rows = w.jobs[3 * blockIdx.x + 2];
    char* base = (char*) planes[blockIdx.y];
    for (int job = blockIdx.x; job < n; job += gridDim.x) {
        if (job != (int) blockIdx.x) from = w.jobs[3 * job], to = w.jobs[3 * job + 1], rows = w.jobs[3 * job + 2];
        const char* src = base + (size_t) from * r.page_bytes;
        char* dst = base + (size_t) to * r.page_bytes;
        const size_t bytes = rows * r.row_bytes, lo = (size_t) blockIdx.z * PG_PIECE, hi = min(bytes, lo + PG_PIECE);
        uint4 v[PG_PIECE / (256 * 16)];
#pragma unroll
        for (int k = 0; k < PG_PIECE / (256 * 16); ++k) {
            const size_t at = lo + (size_t) (k * 256 + threadIdx.x) * 16;
            if (at < hi) v[k] = *reinterpret_cast<const uint4*>(src + at);
        }
#pragma unroll
        for (int k = 0; k < PG_PIECE / (256 * 16); ++k) {
            const size_t at = lo + (size_t) (k * 256 + threadIdx.x) * 16;
            if (at < hi) *reinterpret_cast<uint4*>(dst + at) = v[k];
        }
        if (r.scale_at && blockIdx.z == 0)
            for (size_t at = (size_t) threadIdx.x * 8; at < rows * r.scale_bytes; at += 256 * 8)
                *reinterpret_cast<uint2*>(dst + r.scale_at + at) = *reinterpret_cast<const uint2*>(src + r.scale_at + at);
    }
}

// ---------------------------------------------------------------- keep
// Block (sequence, plane).  Where each kept row lies goes to shared memory, PK_ROWS at a time; a thread has 16 bytes of a row and
// walks the path in ascending order, PK_BATCH rows' loads before their stores: a kept row's old place is never before its new
// one, and the list ascends, so a store meets only rows whose loads are done.  (Scales of int8 rows the same way, 8 bytes a
// thread.)  The first batch's loads are under way before the block has agreed that the list and its pages are sound; nothing
// is stored before that.
constexpr int PK_THREADS = 128, PK_ROWS = PK_THREADS, PK_BATCH = 16;   // (batches of 8: a step of 32 sequences takes 1 us longer)
struct PkMove {
    int from, from_row, to, to_row;   // page and row in it; from negative: the row stays, or the list is senseless
};
__global__ void __launch_bounds__(PK_THREADS, 3) k_pages_keep(const FnxPagePool p, const int* __restrict__ pos0, const int* __restrict__ keep, int keep_stride,
                                                    const int* __restrict__ nkeep, void* const* __restrict__ planes, const PgRows r, void* scratch, unsigned* err) {
    __shared__ PkMove moves[PK_ROWS];
    const PgScratch w = pg_scratch(p, scratch);
    pdl_wait();
    pdl_go();
    const int s = blockIdx.x, n = nkeep[s], tid = threadIdx.x, len = p.len[s], at0 = pos0[s];
    char* base = (char*) planes[blockIdx.y];
    const bool head = blockIdx.y == 0;
    if (n < 0) {
        if (head && tid == 0) w.verdict[s] = -1;
        return;
    }
    const int have = len - at0;
    const int* list = keep + (size_t) s * keep_stride;
    const int* pt = p.pt + (size_t) s * p.pt_stride;
    bool bad = at0 < 0 || at0 > len || n > keep_stride || n > have || pg_pages(p, (unsigned) max(len, 0)) > (unsigned) p.pt_stride;
    const bool sound = !bad;   // (the whole block agrees)
    auto find = [&](int i) {   // kept row i's way; i < n
        PkMove m{-1, 0, 0, 0};
        const int e = list[i];
        if (e < i || e >= have) return m;
        const unsigned rows = (unsigned) p.rows, f = (unsigned) (at0 + e) / rows, t = (unsigned) (at0 + i) / rows;
        m.from = pt[f], m.to = pt[t], m.from_row = (int) (at0 + e - f * rows), m.to_row = (int) (at0 + i - t * rows);
        if (e == i || !pg_valid(p, m.from) || !pg_valid(p, m.to)) m.from = -1;
        return m;
    };
    if (sound) {   // the list, and the pages that rows are read from and written to; all first loads together
        const unsigned rows = (unsigned) p.rows;
        const int end = (int) pg_pages(p, (unsigned) len), first = (int) ((unsigned) at0 / rows);
        auto page_bad = [&](int j, int page) { return !pg_valid(p, page) || (n > 0 && j * p.rows < at0 + n && p.ref[page] != 1); };
        const int page0 = first + tid < end ? pt[first + tid] : 0, l0 = tid < n ? list[tid] : 0, l1 = tid && tid < n ? list[tid - 1] + 1 : 0;
        const bool page0_bad = first + tid < end && page_bad(first + tid, page0);
        if (tid < n) moves[tid] = find(tid);
        bad = page0_bad || (tid < n && (l0 < l1 || l0 >= have));
        for (int i = tid + PK_THREADS; i < n; i += PK_THREADS) bad = bad || list[i] < list[i - 1] + 1 || list[i] >= have;
        for (int j = first + tid + PK_THREADS; j < end; j += PK_THREADS) bad = bad || page_bad(j, pt[j]);
    }
    __syncthreads();
    auto ask = [&](auto* v, int k0, int count, size_t start, size_t row_bytes, size_t c) {
#pragma unroll
        for (int k = 0; k < PK_BATCH; ++k)
            if (k0 + k < count && moves[k0 + k].from >= 0)
                v[k] = *reinterpret_cast<decltype(v)>(base + (size_t) moves[k0 + k].from * r.page_bytes + start + (size_t) moves[k0 + k].from_row * row_bytes + c);
    };
    auto put = [&](auto* v, int k0, int count, size_t start, size_t row_bytes, size_t c) {
#pragma unroll
        for (int k = 0; k < PK_BATCH; ++k)
            if (k0 + k < count && moves[k0 + k].from >= 0)
                *reinterpret_cast<decltype(v)>(base + (size_t) moves[k0 + k].to * r.page_bytes + start + (size_t) moves[k0 + k].to_row * row_bytes + c) = v[k];
    };
    uint4 v[PK_BATCH];
    const bool mine = sound && (size_t) tid * 16 < r.row_bytes;
    if (mine) ask(v, 0, min(n, PK_ROWS), 0, r.row_bytes, (size_t) tid * 16);
    bad = __syncthreads_or(bad);
    if (head && tid == 0) {
        w.verdict[s] = bad ? -1 : at0 + n;
        if (bad) atomicOr(err, PG_ERR_VALUE);
    }
    if (bad) return;
    if (mine) put(v, 0, min(n, PK_ROWS), 0, r.row_bytes, (size_t) tid * 16);
    for (int i0 = 0; i0 < n; i0 += PK_ROWS) {
        const int count = min(n - i0, PK_ROWS);
        if (i0) {
            __syncthreads();   // everyone is done with the moves before these
            if (tid < count) moves[tid] = find(i0 + tid);
            __syncthreads();
        }
        for (size_t c = (size_t) tid * 16; c < r.row_bytes; c += PK_THREADS * 16)
            for (int k0 = i0 == 0 && c == (size_t) tid * 16 ? PK_BATCH : 0; k0 < count; k0 += PK_BATCH) {
                ask(v, k0, count, 0, r.row_bytes, c);
                put(v, k0, count, 0, r.row_bytes, c);
            }
        if (r.scale_at)
            for (size_t c = (size_t) tid * 8; c < r.scale_bytes; c += PK_THREADS * 8)
                for (int k0 = 0; k0 < count; k0 += PK_BATCH) {
                    uint2 u[PK_BATCH];
                    ask(u, k0, count, r.scale_at, r.scale_bytes, c);
                    put(u, k0, count, r.scale_at, r.scale_bytes, c);
                }
    }
}
// the lengths and what lies behind them, once every plane's rows are in place
__global__ void __launch_bounds__(128) k_pages_trim(const FnxPagePool p, void* scratch) {
    const PgScratch w = pg_scratch(p, scratch);
    pdl_wait();
    pdl_go();
    const int s = blockIdx.x, len = w.verdict[s], was = p.len[s];
    if (len < 0) return;
    const int held = pg_held(p, was);
    __syncthreads();
    for (int j = pg_held(p, len) + threadIdx.x; j < held; j += 128) {
        int* e = p.pt + (size_t) s * p.pt_stride + j;
        if (pg_valid(p, *e)) atomicSub(&p.ref[*e], 1);
        *e = -1;
    }
    if (threadIdx.x == 0) p.len[s] = len;
}

static int pg_check(const FnxPagePool* p, const void* scratch, const unsigned* err, const char* what) {
    FNX_REQUIRE(p && p->ref && p->pt && p->len && scratch && err, "%s: a null buffer", what);
    FNX_REQUIRE(p->npages >= 1 && p->rows >= 1 && p->pt_stride >= 1, "%s: %d pages of %d rows, tables of %d", what, p->npages, p->rows, p->pt_stride);
    FNX_REQUIRE(p->npages <= 1 << 30 && p->pt_stride <= 1 << 30, "%s: %d pages, tables of %d (2^30 at most)", what, p->npages, p->pt_stride);
    FNX_REQUIRE(p->nseq >= 1 && p->nseq <= PG_SEQS, "%s: %d sequences outside 1..%d", what, p->nseq, PG_SEQS);
    FNX_REQUIRE((long long) p->rows * p->pt_stride < (1ll << 31), "%s: a table of %d pages of %d rows holds 2^31 positions or more", what, p->pt_stride, p->rows);
    return 0;
}
static int pg_check_planes(const FnxPagePool* p, void* const* planes, int nplanes, const FnxKvPages& g, int nkv, int hd, const char* what) {
    FNX_REQUIRE(planes && nplanes >= 1 && nplanes <= 65535, "%s: %d planes", what, nplanes);
    FNX_REQUIRE(nkv >= 1 && (hd == 128 || hd == 256), "%s: %d KV heads of %d (128 or 256)", what, nkv, hd);
    FNX_REQUIRE(g.rows == p->rows, "%s: pages of %d rows in a pool of pages of %d", what, g.rows, p->rows);
    const size_t row = (size_t) nkv * hd, need = g.q8 ? (size_t) p->rows * (row / 2 + row / 32) : (size_t) p->rows * row;
    FNX_REQUIRE(g.page >= need && g.page % 8 == 0, "%s: a page of %zu halves for %d rows that take %zu (a multiple of 8)", what, g.page, p->rows, need);
    return 0;
}

}  // namespace fnxk

using namespace fnxk;

extern "C" {

size_t fnx_pages_scratch_bytes(const FnxPagePool* p) {
    if (!p || p->npages < 1 || p->nseq < 1 || p->pt_stride < 1) return 0;
    return 4 * (4 + 3 * (size_t) p->npages + 4 * (size_t) p->nseq);
}

int fnx_pages_fork(const FnxPagePool* p, const int* from, const int* lim, void* scratch, unsigned* err, void* st) {
    if (pg_check(p, scratch, err, "pages_fork")) return 1;
    FNX_REQUIRE(from, "pages_fork: a null buffer");
    const int shift = p->nseq > 256 ? 3 : 5;   // a sector or four of each table a block; 196 KB of shared memory at most
    const size_t smem = (size_t) p->nseq * ((1 << shift) + 4) * 4;
    if (smem > 32 * 1024 && smem_optin(k_pages_fork, (size_t) PG_SEQS * 12 * 4, "pages_fork")) return 1;   // (one size for all calls: they may come from several threads)
    launch(0, k_pages_fork, dim3((p->pt_stride + (1 << shift) - 1) >> shift), 256, smem, strm(st), *p, from, lim, shift, scratch, err);
    return launch_ok("pages_fork");
}

int fnx_pages_reserve(const FnxPagePool* p, const int* add, int* pos0, int* row0, void* const* planes, int nplanes, FnxKvPages g, int nkv, int hd,
                      void* scratch, unsigned* err, void* st) {
    if (pg_check(p, scratch, err, "pages_reserve") || pg_check_planes(p, planes, nplanes, g, nkv, hd, "pages_reserve")) return 1;
    FNX_REQUIRE(add && pos0 && row0, "pages_reserve: a null buffer");
    const PgRows r = pg_rows(*p, g, nkv, hd);
    const unsigned pieces = (unsigned) ((p->rows * r.row_bytes + PG_PIECE - 1) / PG_PIECE);
    FNX_REQUIRE(pieces <= 65535, "pages_reserve: a page of %zu bytes", p->rows * r.row_bytes);
    launch(0, k_pages_reserve, dim3(1), PG_THREADS, 0, strm(st), *p, add, pos0, row0, scratch, err);
    if (launch_ok("pages_reserve")) return 1;
    launch(0, k_pages_copy, dim3(std::min(p->nseq, 64), nplanes, pieces), 256, 0, strm(st), *p, planes, r, scratch);
    return launch_ok("pages_reserve (copies)");
}

int fnx_pages_keep(const FnxPagePool* p, const int* pos0, const int* keep, int keep_stride, const int* nkeep, void* const* planes, int nplanes,
                   FnxKvPages g, int nkv, int hd, void* scratch, unsigned* err, void* st) {
    if (pg_check(p, scratch, err, "pages_keep") || pg_check_planes(p, planes, nplanes, g, nkv, hd, "pages_keep")) return 1;
    FNX_REQUIRE(pos0 && keep && nkeep && keep_stride >= 1, "pages_keep: a null buffer, or lists of %d", keep_stride);
    const PgRows r = pg_rows(*p, g, nkv, hd);
    launch(0, k_pages_keep, dim3(p->nseq, nplanes), PK_THREADS, 0, strm(st), *p, pos0, keep, keep_stride, nkeep, planes, r, scratch, err);
    if (launch_ok("pages_keep")) return 1;
    launch(0, k_pages_trim, dim3(p->nseq), 128, 0, strm(st), *p, scratch);
    return launch_ok("pages_keep (lengths)");
}
}
