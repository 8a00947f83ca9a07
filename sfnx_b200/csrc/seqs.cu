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
// angles' sines and cosines (double precision) are made once a row for all heads.  Bound by DRAM: a row's queries and K/V are
// read in f32 and written in f16.
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

template <int HD>
__global__ void __launch_bounds__(SA_THREADS, 3) k_seqs_append(const __grid_constant__ SaArgs a) {
    constexpr int E = HD / 32;
    __shared__ __align__(16) float sn[64], cs[64];
    __shared__ float rot[SA_WARPS][128];
    const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nh = a.nq + 2 * a.nkv;
    pdl_wait();
    pdl_go();
    const int s = sq_find(a.sq.row0, a.sq.nseq, t);
    if (s < 0) return;   // behind the last sequence (the whole block agrees)
    const size_t row_elems = (size_t) a.nkv * HD;
    auto source = [&](int h) {
        return (h < a.nq ? a.qg + ((size_t) t * a.nq + h) * 2 * HD : h < a.nq + a.nkv ? a.k + (size_t) t * row_elems + (size_t) (h - a.nq) * HD
                                                                                        : a.v + (size_t) t * row_elems + (size_t) (h - a.nq - a.nkv) * HD) + lane * E;
    };
    SaVec<E> x[SA_HEADS];
    auto ask = [&](int h0) {
#pragma unroll
        for (int b = 0; b < SA_HEADS; ++b)
            if (h0 + b * SA_WARPS < nh) x[b] = sa_load<E>(source(h0 + b * SA_WARPS));
    };
    ask(warp);   // on their way while the row's place and angles are worked out
    const int i0 = t - a.sq.row0[s], p0 = a.sq.pos0[s];
    const int turn = max(0, p0) + (a.depth ? max(0, a.depth[t]) : i0);
    if (threadIdx.x < a.nrot / 2) {
        const float theta = fmul((float) turn, a.freq[threadIdx.x]);
        ex_sincos((double) theta, &sn[threadIdx.x], &cs[threadIdx.x]);
    }
    const long long cell = sq_cell(a.sq, a.g, s, p0 < 0 || i0 > INT_MAX - p0 ? -1 : p0 + i0);
    if (threadIdx.x == 0 && cell < 0) atomicOr(a.err, SQ_ERR_ROOM);
    const size_t at = cell < 0 ? 0 : sq_at(a.sq, a.g, cell, row_elems);
    __syncthreads();
    // element i < nrot pairs with i -+ half: y = c x + d x', d negative for the lower one.  Whole lanes apart (half a multiple of
    // E) the partner comes by a shuffle, else through shared memory
    const int half = a.nrot / 2, apart = half % E ? 0 : half / E;
    const bool turned = lane * E < a.nrot, lower = lane * E < half;
    for (int h0 = warp; h0 < nh; h0 += SA_HEADS * SA_WARPS) {
        if (h0 != warp) ask(h0);
#pragma unroll
        for (int b = 0; b < SA_HEADS; ++b) {
            const int h = h0 + b * SA_WARPS;
            if (h >= nh) break;
            if (h < a.nq + a.nkv) {
                // squares of 32 neighbouring elements summed as the xor-tree over a warp does (offsets 16 .. 1), the groups ascending
                float q[E];
#pragma unroll
                for (int e = 0; e < E; ++e) q[e] = fmul(x[b].x[e], x[b].x[e]);
#pragma unroll
                for (int o = 16; o >= E; o >>= 1)
#pragma unroll
                    for (int e = 0; e < E; ++e) q[e] = fadd(q[e], __shfl_xor_sync(0xffffffffu, q[e], o / E));
#pragma unroll
                for (int o = E / 2; o; o >>= 1)
#pragma unroll
                    for (int e = 0; e < o; ++e) q[e] = fadd(q[e], q[e + o]);
                float tot = 0.f;
#pragma unroll
                for (int g = 0; g < E; ++g) tot = fadd(tot, __shfl_sync(0xffffffffu, q[0], g * (32 / E)));
                const float r = ex_rsqrt(fadd(fmul(tot, 1.0f / (float) HD), a.eps));   // (HD is a power of two: the quotient's bits)
                const SaVec<E> wt = sa_load<E>((h < a.nq ? a.qn : a.kn) + lane * E);
#pragma unroll
                for (int e = 0; e < E; ++e) x[b].x[e] = fmul(fmul(x[b].x[e], r), wt.x[e]);
                if (apart) {
                    float other[E];
#pragma unroll
                    for (int e = 0; e < E; ++e) other[e] = __shfl_sync(0xffffffffu, x[b].x[e], lower ? lane + apart : lane - apart);
                    if (turned) {
                        const SaVec<E> c = sa_load<E>(&cs[lane * E - (lower ? 0 : half)]), d = sa_load<E>(&sn[lane * E - (lower ? 0 : half)]);
#pragma unroll
                        for (int e = 0; e < E; ++e)
                            x[b].x[e] = lower ? ffma(-other[e], d.x[e], fmul(x[b].x[e], c.x[e])) : ffma(x[b].x[e], c.x[e], fmul(other[e], d.x[e]));
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
                if (cell >= 0) sa_store<E>(a.kc + at + (size_t) (h - a.nq) * HD + lane * E, x[b]);
            } else if (cell >= 0) sa_store<E>(a.vc + at + (size_t) (h - a.nq - a.nkv) * HD + lane * E, x[b]);
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
