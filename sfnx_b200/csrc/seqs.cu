// The rows of several sequences on their way into the cache: per-head RMS norm, rotary and K/V append for any number of rows
// (prompts, windows, draft trees), and a draft tree's ancestor masks and depths.  The norm and the rotation are
// fnx_attn_prep_append's (reference src/kernels.cu:1539-1569), with its order of every sum, so a cache may be filled by either.
#include <climits>
#include <cmath>

#include "exact_math.cuh"
#include "seqs.cuh"

namespace fnxk {

// ---------------------------------------------------------------- draft trees
// A block per sequence, a thread per row: the walk to the root over parents in shared memory, a step per ancestor.  Parents have
// lower indices, so the walk meets the mask's words from the highest down and ends after at most as many steps as rows.
constexpr int TM_NODES = 1024, TM_THREADS = 128;
__global__ void __launch_bounds__(TM_THREADS) k_tree_masks(const int* __restrict__ parent, const FnxSeqs sq, unsigned* __restrict__ anc, int words,
                                                           int* __restrict__ depth, unsigned* err) {
    __shared__ short par[TM_NODES];
    pdl_wait();
    pdl_go();
    const int s = blockIdx.x, r0 = max(sq.row0[s], 0), n = min(sq.row0[s + 1], sq.rows) - r0, most = 32 * words;
    bool bad = n > most;
    for (int i = threadIdx.x; i < min(n, most); i += TM_THREADS) {
        const int p = parent[r0 + i];
        const bool ok = p >= -1 && p < i;
        par[i] = (short) (ok ? p : -1);
        bad = bad || !ok;
    }
    if (bad) atomicOr(err, SQ_ERR_VALUE);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += TM_THREADS) {
        int j = i < most ? i : -1, d = -1;
        for (int w = words - 1; w >= 0; --w) {
            unsigned bits = 0u;
            for (; j >= 32 * w; j = par[j], ++d) bits |= 1u << (j & 31);
            anc[(size_t) (r0 + i) * words + w] = bits;
        }
        if (depth) depth[r0 + i] = max(d, 0);
    }
}

// ---------------------------------------------------------------- append
// A block per row, a warp per head at a time (four heads' loads in flight): a lane holds E neighbouring elements of its head.  The
// angles' sines and cosines (double precision) are made once a row for all heads.  A row's queries and K/V are read in f32 and
// written in f16 (40 us of copying at 5301 rows of 24 + 2 * 4 heads of 256); a block's own chain of dependent loads and the angles
// bound it before DRAM does, so the loads come first and four blocks lie on a processor: 64.5 us (4.1 TB/s), with three 71.7.
struct SaArgs {
    const float *qg, *k, *v, *qn, *kn;
    uint16_t *kc, *vc, *q16;
    FnxKvPages g;
    FnxSeqs sq;
    const int* depth;
    unsigned* err;
    float eps;
    int nq, nkv, nrot;
    float freq[64];   // of pair i, base^(-2 i / nrot), computed by the host's powf
};
constexpr int SA_THREADS = 256, SA_WARPS = SA_THREADS / 32, SA_HEADS = 4;

template <int E> struct SaVec {
    float x[E];
};
template <int E> __device__ __forceinline__ SaVec<E> sa_load(const float* p) {
    SaVec<E> r;
#pragma unroll
    for (int i = 0; i < E; i += 4) {
        const float4 f = *reinterpret_cast<const float4*>(p + i);
        r.x[i] = f.x, r.x[i + 1] = f.y, r.x[i + 2] = f.z, r.x[i + 3] = f.w;
    }
    return r;
}
template <int E> __device__ __forceinline__ void sa_store(uint16_t* p, const SaVec<E>& r) {
    unsigned u[E / 2];
#pragma unroll
    for (int i = 0; i < E; i += 2) u[i / 2] = (unsigned) f2h(r.x[i]) | ((unsigned) f2h(r.x[i + 1]) << 16);
    if (E == 8) *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[E / 2 - 2], u[E / 2 - 1]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[1]);
}

// The sum of 32 neighbouring values (E a lane) as the xor-tree over a warp forms it, offsets 16 .. 1: at each of the first steps a
// lane keeps the half of its values that its partner does not, so nobody adds what another adds.  Every lane gets the sum.
template <int E> __device__ __forceinline__ float sa_tree(const float* q, int lane) {
    if constexpr (E == 8) {   // offset 16: lane ^ 2, 8: lane ^ 1, 4 .. 1: within a lane at first
        const bool hi = lane & 2, odd = lane & 1;
        float a[4], b[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = fadd(hi ? q[4 + i] : q[i], __shfl_xor_sync(0xffffffffu, hi ? q[i] : q[4 + i], 2));
#pragma unroll
        for (int i = 0; i < 2; ++i) b[i] = fadd(odd ? a[2 + i] : a[i], __shfl_xor_sync(0xffffffffu, odd ? a[i] : a[2 + i], 1));
        // b[i]: elements 4 hi + 2 odd + i of offsets 4 and less
        float c = fadd(hi ? b[1] : b[0], __shfl_xor_sync(0xffffffffu, hi ? b[0] : b[1], 2));   // offset 4; element 2 odd + hi
        c = fadd(c, __shfl_xor_sync(0xffffffffu, c, 1));                                         // offset 2
        return fadd(c, __shfl_xor_sync(0xffffffffu, c, 2));                                      // offset 1
    } else {   // offset 16: lane ^ 4, 8: lane ^ 2, 4: lane ^ 1
        const bool hi = lane & 4, mid = lane & 2;
        float a[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) a[i] = fadd(hi ? q[2 + i] : q[i], __shfl_xor_sync(0xffffffffu, hi ? q[i] : q[2 + i], 4));
        float c = fadd(mid ? a[1] : a[0], __shfl_xor_sync(0xffffffffu, mid ? a[0] : a[1], 2));   // offset 8; element 2 hi + mid
        c = fadd(c, __shfl_xor_sync(0xffffffffu, c, 1));                                         // offset 4
        c = fadd(c, __shfl_xor_sync(0xffffffffu, c, 4));                                         // offset 2
        return fadd(c, __shfl_xor_sync(0xffffffffu, c, 2));                                      // offset 1
    }
}

template <int HD>
__global__ void __launch_bounds__(SA_THREADS, 4) k_seqs_append(const __grid_constant__ SaArgs a) {
    constexpr int E = HD / 32;
    __shared__ __align__(16) float sn[64], cs[64], wt[2][HD];
    __shared__ float rot[SA_WARPS][128];
    const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nh = a.nq + 2 * a.nkv;
    pdl_wait();
    pdl_go();
    const size_t row_elems = (size_t) a.nkv * HD;
    const float *rq = a.qg + (size_t) t * a.nq * 2 * HD + lane * E, *rk = a.k + (size_t) t * row_elems + lane * E, *rv = a.v + (size_t) t * row_elems + lane * E;
    auto source = [&](int h) { return h < a.nq ? rq + h * 2 * HD : h < a.nq + a.nkv ? rk + (h - a.nq) * HD : rv + (h - a.nq - a.nkv) * HD; };
    SaVec<E> x[SA_HEADS];
    auto ask = [&](int h0) {
#pragma unroll
        for (int b = 0; b < SA_HEADS; ++b)
            if (h0 + b * SA_WARPS < nh) x[b] = sa_load<E>(source(h0 + b * SA_WARPS));
    };
    ask(warp);   // on their way while the row's place and angles are worked out
    const int s = sq_find(a.sq.row0, a.sq.nseq, t);
    if (s < 0) return;   // behind the last sequence (the whole block agrees)
    const int i0 = t - a.sq.row0[s], p0 = a.sq.pos0[s];
    const int turn = max(0, p0) + (a.depth ? max(0, a.depth[t]) : i0);
    if (threadIdx.x < a.nrot / 2) {
        const float theta = fmul((float) turn, a.freq[threadIdx.x]);
        ex_sincos((double) theta, &sn[threadIdx.x], &cs[threadIdx.x]);
    }
    for (int i = threadIdx.x; i < HD; i += SA_THREADS) wt[0][i] = a.qn[i], wt[1][i] = a.kn[i];
    const long long cell = sq_cell(a.sq, a.g, s, p0 < 0 || i0 > INT_MAX - p0 ? -1 : p0 + i0);
    if (threadIdx.x == 0 && cell < 0) atomicOr(a.err, SQ_ERR_ROOM);
    const size_t at = cell < 0 ? 0 : sq_at(a.sq, a.g, cell, row_elems);
    __syncthreads();
    // element i < nrot pairs with i -+ half: the lower one becomes x c - x' s, the upper one x c + x' s, the first product rounded before the
    // fused second.  Whole lanes apart (half a multiple of E) the partner comes by a shuffle, else through shared memory
    const int half = a.nrot / 2, apart = half % E ? 0 : half / E;
    const bool turned = lane * E < a.nrot, lower = lane * E < half;
    for (int h0 = warp; h0 < nh; h0 += SA_HEADS * SA_WARPS) {
        if (h0 != warp) ask(h0);
        // ---- the heads' square sums, one root for all: lane b takes head b's
        float mine = 1.f;
#pragma unroll
        for (int b = 0; b < SA_HEADS; ++b) {
            if (h0 + b * SA_WARPS >= a.nq + a.nkv) continue;
            float q[E];
#pragma unroll
            for (int e = 0; e < E; ++e) q[e] = fmul(x[b].x[e], x[b].x[e]);
            const float group = sa_tree<E>(q, lane);
            float tot = 0.f;
#pragma unroll
            for (int g = 0; g < E; ++g) tot = fadd(tot, __shfl_sync(0xffffffffu, group, g * (32 / E)));
            mine = lane == b ? tot : mine;
        }
        mine = ex_rsqrt(fadd(fmul(mine, 1.0f / (float) HD), a.eps));   // (HD is a power of two: the quotient's bits)
#pragma unroll
        for (int b = 0; b < SA_HEADS; ++b) {
            const int h = h0 + b * SA_WARPS;
            if (h >= nh) break;
            if (h < a.nq + a.nkv) {
                const float r = __shfl_sync(0xffffffffu, mine, b);
                const SaVec<E> w = sa_load<E>(&wt[h < a.nq ? 0 : 1][lane * E]);
#pragma unroll
                for (int e = 0; e < E; ++e) x[b].x[e] = fmul(fmul(x[b].x[e], r), w.x[e]);
                if (apart) {
                    float other[E];
#pragma unroll
                    for (int e = 0; e < E; ++e) other[e] = __shfl_sync(0xffffffffu, x[b].x[e], lower ? lane + apart : lane - apart);
                    if (turned) {
                        const int i = lane * E - (lower ? 0 : half);
                        const SaVec<E> c = sa_load<E>(lower ? &cs[i] : &sn[i]), d = sa_load<E>(lower ? &sn[i] : &cs[i]);
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            const float y = x[b].x[e];
                            x[b].x[e] = ffma(lower ? -other[e] : y, d.x[e], fmul(lower ? y : other[e], c.x[e]));
                        }
                    }
                } else {
                    if (turned)
#pragma unroll
                        for (int e = 0; e < E; ++e) rot[warp][lane * E + e] = x[b].x[e];
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const int i = lane * E + e;
                        if (i < half) x[b].x[e] = ffma(-rot[warp][i + half], sn[i], fmul(x[b].x[e], cs[i]));
                        else if (i < a.nrot) x[b].x[e] = ffma(x[b].x[e], cs[i - half], fmul(rot[warp][i - half], sn[i - half]));
                    }
                    __syncwarp();
                }
            }
            if (h < a.nq) sa_store<E>(a.q16 + ((size_t) t * a.nq + h) * HD + lane * E, x[b]);
            else if (h < a.nq + a.nkv) {
                if (cell >= 0) sa_store<E>(a.kc + at + (h - a.nq) * HD + lane * E, x[b]);
            } else if (cell >= 0) sa_store<E>(a.vc + at + (h - a.nq - a.nkv) * HD + lane * E, x[b]);
        }
    }
}

}  // namespace fnxk

using namespace fnxk;

extern "C" {

int fnx_tree_masks(const int* parent, const FnxSeqs* sq, unsigned* anc, int anc_words, int* depth, unsigned* err, void* st) {
    FNX_REQUIRE(parent && sq && sq->row0 && anc && err, "tree_masks: a null buffer");
    FNX_REQUIRE(sq->nseq >= 1 && sq->rows >= 1, "tree_masks: %d rows of %d sequences", sq->rows, sq->nseq);
    FNX_REQUIRE(anc_words >= 1 && 32 * anc_words <= TM_NODES, "tree_masks: masks of %d words (1..%d)", anc_words, TM_NODES / 32);
    launch(0, k_tree_masks, dim3(sq->nseq), TM_THREADS, 0, strm(st), parent, *sq, anc, anc_words, depth, err);
    return launch_ok("tree_masks");
}

int fnx_attn_seqs_append(const float* qg, const float* k, const float* v, const float* q_norm, const float* k_norm, uint16_t* kc, uint16_t* vc,
                         FnxKvPages g, const FnxSeqs* sq, const int* depth, uint16_t* q16, float eps, FnxRope rope, int nq, int nkv, int hd,
                         unsigned* err, void* st) {
    if (sq_check(sq, g, nq, nkv, hd, "attn_seqs_append")) return 1;
    FNX_REQUIRE(qg && k && v && q_norm && k_norm && kc && vc && q16 && err, "attn_seqs_append: a null buffer");
    FNX_REQUIRE(((uintptr_t) qg | (uintptr_t) k | (uintptr_t) v | (uintptr_t) q_norm | (uintptr_t) k_norm | (uintptr_t) kc | (uintptr_t) vc | (uintptr_t) q16) % 16 == 0,
                "attn_seqs_append: a buffer that is not 16-byte aligned");
    FNX_REQUIRE(rope.nrot % 2 == 0 && rope.nrot >= 2 && rope.nrot <= 128 && rope.nrot <= hd, "attn_seqs_append: rotary width %d", rope.nrot);
    SaArgs a{qg, k, v, q_norm, k_norm, kc, vc, q16, g, *sq, depth, err, eps, nq, nkv, rope.nrot, {}};
    for (int i = 0; i < rope.nrot / 2; ++i) a.freq[i] = powf(rope.base, -2.0f * (float) i / (float) rope.nrot);
    if (hd == 256) launch(0, k_seqs_append<256>, dim3(sq->rows), SA_THREADS, 0, strm(st), a);
    else launch(0, k_seqs_append<128>, dim3(sq->rows), SA_THREADS, 0, strm(st), a);
    return launch_ok("attn_seqs_append");
}
}
