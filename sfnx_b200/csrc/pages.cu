// The pages of a K/V pool and the sequences' tables: sharing, growth with copy on write, an accepted path's rows moved
// together, and what nobody names any more free again (no counterpart in the reference, whose host keeps its tables).
//
// State is what the header says: a reference count a page, a table and a length a sequence.  Every result is a function of
// that state alone: reference counts are sums of integers, free pages are handed out lowest first in the sequences' order,
// and which holder of a shared page keeps it is the lowest, so no order of atomics shows.
// The tables are a few thousand words: fork and reserve are bound by the latency of a handful of dependent steps and launches,
// the row copies by DRAM.
#include <algorithm>
#include <climits>

#include "common.cuh"
#include "exact_math.cuh"

namespace fnxk {

constexpr int PG_SEQS = 4096, PG_THREADS = 1024, PG_WARPS = PG_THREADS / 32, PG_PER = PG_SEQS / PG_THREADS;
constexpr unsigned PG_ERR_ROOM = 32u, PG_ERR_VALUE = 64u;

// the scratch's words: a header (jobs of the copy), then per page: holders of a tail page in this call, the complement of the
// lowest of them (both zero between calls), the free list; per sequence: copy jobs (from, to, rows), the verdict, the old length;
// the old tables
struct PgScratch {
    int *njobs, *holders, *lowest, *free_list, *jobs, *verdict, *old_len, *old_pt;
};
__host__ __device__ inline PgScratch pg_scratch(const FnxPagePool& p, void* scratch) {
    int* w = (int*) scratch;
    PgScratch s;
    s.njobs = w, w += 4;
    s.holders = w, w += p.npages;
    s.lowest = w, w += p.npages;
    s.free_list = w, w += p.npages;
    s.jobs = w, w += 3 * (size_t) p.nseq;
    s.verdict = w, w += p.nseq;
    s.old_len = w, w += p.nseq;
    s.old_pt = w;
    return s;
}
__device__ __forceinline__ int pg_held(const FnxPagePool& p, int len) {   // pages that len positions need, at most the table's
    return min((int) (((long long) max(len, 0) + p.rows - 1) / p.rows), p.pt_stride);
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
__global__ void __launch_bounds__(256) k_pages_save(const FnxPagePool p, void* scratch) {
    const PgScratch w = pg_scratch(p, scratch);
    pdl_wait();
    pdl_go();
    const long long n = (long long) p.nseq * p.pt_stride;
    for (long long i = (long long) blockIdx.x * 256 + threadIdx.x; i < n; i += (long long) gridDim.x * 256) w.old_pt[i] = p.pt[i];
    for (int s = blockIdx.x * 256 + threadIdx.x; s < p.nseq; s += gridDim.x * 256) w.old_len[s] = p.len[s];
}
__global__ void __launch_bounds__(256) k_pages_fork(const FnxPagePool p, const int* __restrict__ from, const int* __restrict__ lim, void* scratch, unsigned* err) {
    const PgScratch w = pg_scratch(p, scratch);
    pdl_wait();
    pdl_go();
    const long long n = (long long) p.nseq * p.pt_stride;
    for (long long i = (long long) blockIdx.x * 256 + threadIdx.x; i < n; i += (long long) gridDim.x * 256) {
        const int s = (int) (i / p.pt_stride), j = (int) (i % p.pt_stride);
        int src = from[s];
        if (src >= p.nseq) {
            if (j == 0) atomicOr(err, PG_ERR_VALUE);
            src = s;
        }
        int len = src < 0 ? 0 : max(w.old_len[src], 0);
        if (lim) len = min(len, max(lim[s], 0));
        const int was = j < pg_held(p, w.old_len[s]) ? w.old_pt[i] : -1;
        const int now = j < pg_held(p, len) ? w.old_pt[(long long) src * p.pt_stride + j] : -1;
        if (was != now) {
            if (pg_valid(p, now)) atomicAdd(&p.ref[now], 1);
            if (pg_valid(p, was)) atomicSub(&p.ref[was], 1);
        }
        p.pt[i] = now;
        if (j == 0) p.len[s] = len;
    }
}

// ---------------------------------------------------------------- reserve
// exclusive sums of two values a thread over the block (in ascending thread order); totals in t0, t1
__device__ __forceinline__ void pg_scan2(long long& a, long long& b, long long& t0, long long& t1, long long (*sh)[2]) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long a0 = a, b0 = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
        if (lane >= o) a += x, b += y;
    }
    if (lane == 31) sh[warp][0] = a, sh[warp][1] = b;
    __syncthreads();
    long long pa = 0, pb = 0;
    t0 = t1 = 0;
    for (int i = 0; i < PG_WARPS; ++i) {
        if (i == warp) pa = t0, pb = t1;
        t0 += sh[i][0], t1 += sh[i][1];
    }
    __syncthreads();
    a += pa - a0, b += pb - b0;
}

__global__ void __launch_bounds__(PG_THREADS) k_pages_reserve(const FnxPagePool p, const int* __restrict__ add, int* pos0, int* row0, void* scratch, unsigned* err) {
    const PgScratch w = pg_scratch(p, scratch);
    __shared__ long long sh[PG_WARPS][2];
    __shared__ int first[PG_SEQS], wcount[PG_WARPS];   // a sequence's first place in the list of pages handed out
    __shared__ unsigned njobs_s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) njobs_s = 0u;
    pdl_wait();
    pdl_go();
    // ---- what each sequence holds and wants; thread i has PG_PER neighbouring sequences
    int len[PG_PER], more[PG_PER], tail[PG_PER], want[PG_PER];
    bool bad = false, room = true;
#pragma unroll
    for (int k = 0; k < PG_PER; ++k) {
        const int s = tid * PG_PER + k;
        len[k] = more[k] = want[k] = 0, tail[k] = -1;
        if (s >= p.nseq) continue;
        len[k] = max(p.len[s], 0), more[k] = add[s];
        if (more[k] < 0) bad = true;
        else if (((long long) len[k] + more[k] + p.rows - 1) / p.rows > p.pt_stride) room = false;
        else if (more[k] > 0 && len[k] % p.rows) {
            tail[k] = p.pt[(size_t) s * p.pt_stride + len[k] / p.rows];
            if (!pg_valid(p, tail[k])) room = false, tail[k] = -1;
            else atomicAdd(&w.holders[tail[k]], 1), atomicMax(&w.lowest[tail[k]], INT_MAX - s);
        }
    }
    __threadfence_block();
    __syncthreads();
    bool copy[PG_PER];
    long long a = 0, b = 0, pages, rows;
#pragma unroll
    for (int k = 0; k < PG_PER; ++k) {
        const int s = tid * PG_PER + k;
        copy[k] = tail[k] >= 0 && (p.ref[tail[k]] > __ldcg(&w.holders[tail[k]]) || __ldcg(&w.lowest[tail[k]]) != INT_MAX - s);
        if (s < p.nseq && more[k] >= 0 && room)
            want[k] = (int) (((long long) len[k] + more[k] + p.rows - 1) / p.rows - ((long long) len[k] + p.rows - 1) / p.rows) + (copy[k] ? 1 : 0);
        a += want[k], b += more[k] > 0 ? more[k] : 0;
    }
    __syncthreads();   // everyone has looked at the holders
#pragma unroll
    for (int k = 0; k < PG_PER; ++k)
        if (tail[k] >= 0) w.holders[tail[k]] = 0, w.lowest[tail[k]] = 0;
    pg_scan2(a, b, pages, rows, sh);
    bad = __syncthreads_or(bad);
    room = !__syncthreads_or(!room) && rows <= INT_MAX;
    // ---- the lowest free pages, as many as are wanted
    int got = 0;
    if (room && !bad)
        for (int q0 = 0; q0 < p.npages && got < pages; q0 += 4 * PG_THREADS) {   // a warp has 128 neighbouring pages
            unsigned is[4];
            int mine = 0, before[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int q = q0 + warp * 128 + k * 32 + lane;
                is[k] = __ballot_sync(0xffffffffu, q < p.npages && p.ref[q] == 0);
                before[k] = mine;
                mine += __popc(is[k]);
            }
            if (lane == 0) wcount[warp] = mine;
            __syncthreads();
            int below = got;
            for (int i = 0; i < PG_WARPS; ++i) {
                if (i < warp) below += wcount[i];
                got += wcount[i];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int at = below + before[k] + __popc(is[k] & ((1u << lane) - 1u));
                if ((is[k] >> lane & 1u) && at < pages) w.free_list[at] = q0 + warp * 128 + k * 32 + lane;
            }
            __syncthreads();
        }
    const bool ok = room && !bad && got >= pages;
    if (!ok) {   // nothing changes
#pragma unroll
        for (int k = 0; k < PG_PER; ++k) {
            const int s = tid * PG_PER + k;
            if (s < p.nseq) pos0[s] = len[k], row0[s] = 0;
        }
        if (tid == 0) {
            row0[p.nseq] = 0, *w.njobs = 0;
            atomicOr(err, (bad ? PG_ERR_VALUE : 0u) | (!bad || !room ? PG_ERR_ROOM : 0u));
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < PG_PER; ++k) {
        const int s = tid * PG_PER + k;
        first[s] = s < p.nseq ? (int) a : (int) pages;
        if (s < p.nseq) {
            pos0[s] = len[k], row0[s] = (int) b;
            p.len[s] = len[k] + more[k];
        }
        a += want[k], b += more[k];
    }
    if (tid == 0) row0[p.nseq] = (int) rows;
    __threadfence_block();
    __syncthreads();
    // ---- the copies, then the new entries: place i of the list belongs to the last sequence that begins at or before it
#pragma unroll
    for (int k = 0; k < PG_PER; ++k) {
        const int s = tid * PG_PER + k;
        if (!copy[k]) continue;
        const int page = w.free_list[first[s]];
        p.pt[(size_t) s * p.pt_stride + len[k] / p.rows] = page;
        p.ref[page] = 1;
        atomicSub(&p.ref[tail[k]], 1);
        const unsigned at = atomicAdd(&njobs_s, 1u);
        w.jobs[3 * at] = tail[k], w.jobs[3 * at + 1] = page, w.jobs[3 * at + 2] = len[k] % p.rows;
    }
    for (int i = tid; i < (int) pages; i += PG_THREADS) {
        int lo = 0, hi = p.nseq;   // first[lo] <= i
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (first[mid] <= i) lo = mid;
            else hi = mid;
        }
        const int held = (pos0[lo] + p.rows - 1) / p.rows, total = (lo + 1 < p.nseq ? first[lo + 1] : (int) pages) - first[lo];
        const int fresh = (int) (((long long) p.len[lo] + p.rows - 1) / p.rows) - held, j = i - first[lo] - (total - fresh);   // total - fresh: 1 with a copy
        if (j < 0) continue;
        const int page = w.free_list[i];
        p.pt[(size_t) lo * p.pt_stride + held + j] = page;
        p.ref[page] = 1;
    }
    __syncthreads();
    if (tid == 0) *w.njobs = (int) njobs_s;
}

// the rows so far of the pages that reserve copies: block (job, plane, piece of PG_PIECE bytes of a page)
constexpr int PG_PIECE = 32768;
__global__ void __launch_bounds__(256) k_pages_copy(const FnxPagePool p, void* const* __restrict__ planes, const PgRows r, void* scratch) {
    const PgScratch w = pg_scratch(p, scratch);
    pdl_wait();
    pdl_go();
    const int n = *w.njobs;
    for (int job = blockIdx.x; job < n; job += gridDim.x) {
        const int rows = w.jobs[3 * job + 2];
        char* base = (char*) planes[blockIdx.y];
        const char* src = base + (size_t) w.jobs[3 * job] * r.page_bytes;
        char* dst = base + (size_t) w.jobs[3 * job + 1] * r.page_bytes;
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
// Block (sequence, plane).  A thread has 16 bytes of a row and walks the path in ascending order, eight rows' loads before
// their stores: a kept row's old place is never before its new one, and the list ascends, so a store meets only rows whose
// loads are done.  (Scales of int8 rows the same way, 8 bytes a thread.)
__global__ void __launch_bounds__(128) k_pages_keep(const FnxPagePool p, const int* __restrict__ pos0, const int* __restrict__ keep, int keep_stride,
                                                    const int* __restrict__ nkeep, void* const* __restrict__ planes, const PgRows r, void* scratch, unsigned* err) {
    const PgScratch w = pg_scratch(p, scratch);
    pdl_wait();
    pdl_go();
    const int s = blockIdx.x, n = nkeep[s], tid = threadIdx.x;
    const bool head = blockIdx.y == 0;
    if (n < 0) {
        if (head && tid == 0) w.verdict[s] = -1;
        return;
    }
    const int len = p.len[s], at0 = pos0[s], have = len - at0;
    const int* list = keep + (size_t) s * keep_stride;
    const int* pt = p.pt + (size_t) s * p.pt_stride;
    bool bad = at0 < 0 || at0 > len || n > keep_stride || n > have || ((long long) len + p.rows - 1) / p.rows > p.pt_stride;
    if (!bad) {
        for (int i = tid; i < n; i += 128) bad = bad || list[i] < (i ? list[i - 1] + 1 : 0) || list[i] >= have;
        for (int j = at0 / p.rows + tid; j < (len + p.rows - 1) / p.rows; j += 128) {   // the pages that rows are read from and written to
            const bool ours = pg_valid(p, pt[j]);
            bad = bad || !ours || (n > 0 && j * p.rows < at0 + n && p.ref[pt[j]] != 1);
        }
    }
    bad = __syncthreads_or(bad);
    if (head && tid == 0) {
        w.verdict[s] = bad ? -1 : at0 + n;
        if (bad) atomicOr(err, PG_ERR_VALUE);
    }
    if (bad) return;
    char* base = (char*) planes[blockIdx.y];
    auto move = [&](size_t start, size_t row_bytes, auto unit) {
        using U = decltype(unit);
        for (size_t c = (size_t) tid * sizeof(U); c < row_bytes; c += 128 * sizeof(U)) {
            auto at = [&](int pos) { return base + (size_t) pt[pos / p.rows] * r.page_bytes + start + (size_t) (pos % p.rows) * row_bytes + c; };
            for (int i0 = 0; i0 < n; i0 += 8) {
                U v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (i0 + k < n && list[i0 + k] != i0 + k) v[k] = *reinterpret_cast<const U*>(at(at0 + list[i0 + k]));
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (i0 + k < n && list[i0 + k] != i0 + k) *reinterpret_cast<U*>(at(at0 + i0 + k)) = v[k];
            }
        }
    };
    move(0, r.row_bytes, uint4{});
    if (r.scale_at) move(r.scale_at, r.scale_bytes, uint2{});
}
// the lengths and what lies behind them, once every plane's rows are in place
__global__ void __launch_bounds__(128) k_pages_trim(const FnxPagePool p, void* scratch) {
    const PgScratch w = pg_scratch(p, scratch);
    pdl_wait();
    pdl_go();
    const int s = blockIdx.x, len = w.verdict[s];
    if (len < 0) return;
    const int held = pg_held(p, p.len[s]);
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
    return 4 * (4 + 3 * (size_t) p->npages + 5 * (size_t) p->nseq + (size_t) p->nseq * p->pt_stride);
}

int fnx_pages_fork(const FnxPagePool* p, const int* from, const int* lim, void* scratch, unsigned* err, void* st) {
    if (pg_check(p, scratch, err, "pages_fork")) return 1;
    FNX_REQUIRE(from, "pages_fork: a null buffer");
    const long long n = (long long) p->nseq * p->pt_stride;
    const unsigned blocks = (unsigned) std::min<long long>(148 * 8, (n + 255) / 256);
    launch(0, k_pages_save, dim3(blocks), 256, 0, strm(st), *p, scratch);
    if (launch_ok("pages_fork (tables as they were)")) return 1;
    launch(0, k_pages_fork, dim3(blocks), 256, 0, strm(st), *p, from, lim, scratch, err);
    return launch_ok("pages_fork");
}

int fnx_pages_reserve(const FnxPagePool* p, const int* add, int* pos0, int* row0, void* const* planes, int nplanes, FnxKvPages g, int nkv, int hd,
                      void* scratch, unsigned* err, void* st) {
    if (pg_check(p, scratch, err, "pages_reserve") || pg_check_planes(p, planes, nplanes, g, nkv, hd, "pages_reserve")) return 1;
    FNX_REQUIRE(add && pos0 && row0, "pages_reserve: a null buffer");
    launch(0, k_pages_reserve, dim3(1), PG_THREADS, 0, strm(st), *p, add, pos0, row0, scratch, err);
    if (launch_ok("pages_reserve")) return 1;
    const PgRows r = pg_rows(*p, g, nkv, hd);
    const unsigned pieces = (unsigned) ((p->rows * r.row_bytes + PG_PIECE - 1) / PG_PIECE);
    FNX_REQUIRE(pieces <= 65535, "pages_reserve: a page of %zu bytes", p->rows * r.row_bytes);
    launch(0, k_pages_copy, dim3(std::min(p->nseq, 64), nplanes, pieces), 256, 0, strm(st), *p, planes, r, scratch);
    return launch_ok("pages_reserve (copies)");
}

int fnx_pages_keep(const FnxPagePool* p, const int* pos0, const int* keep, int keep_stride, const int* nkeep, void* const* planes, int nplanes,
                   FnxKvPages g, int nkv, int hd, void* scratch, unsigned* err, void* st) {
    if (pg_check(p, scratch, err, "pages_keep") || pg_check_planes(p, planes, nplanes, g, nkv, hd, "pages_keep")) return 1;
    FNX_REQUIRE(pos0 && keep && nkeep && keep_stride >= 1, "pages_keep: a null buffer, or lists of %d", keep_stride);
    const PgRows r = pg_rows(*p, g, nkv, hd);
    launch(0, k_pages_keep, dim3(p->nseq, nplanes), 128, 0, strm(st), *p, pos0, keep, keep_stride, nkeep, planes, r, scratch, err);
    if (launch_ok("pages_keep")) return 1;
    launch(0, k_pages_trim, dim3(p->nseq), 128, 0, strm(st), *p, scratch);
    return launch_ok("pages_keep (lengths)");
}
}
