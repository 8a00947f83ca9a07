// The rows of several sequences on their way into the cache: per-head RMS norm, rotary and K/V append for any number of rows
// (prompts, windows, draft trees), and a draft tree's ancestor masks and depths.  The norm and the rotation are
// fnx_attn_prep_append's (reference src/kernels.cu:1539-1569), with its order of every sum, so a cache may be filled by either.
#include <algorithm>
#include <climits>
#include <cmath>

#include "exact_math.cuh"
#include "moe_internal.cuh"
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
// A block has a run of neighbouring rows, a warp four heads of a row at a time.  A row's queries and K/V are read in f32 and written in
// f16, 40 us of copying at 5301 rows of 24 + 2 * 4 heads of 256; what stands in the way is the chain before a row can be written (its
// sequence, its page, its angles in double precision) and what a head costs in shuffles.  So the next row's heads are on their way
// into shared memory while one is worked on, the next eight rows' places and angles are made before these eight, a warp a row, and a
// lane's elements lie as they are read without conflicts: 51.0 us (5.1 TB/s; 52.3 with the eight made when they are wanted).  With a block a row, the loads in registers, 62.2; with three blocks a
// multiprocessor, or three rows' copies under way, it is slower (by 0.9 and 5).
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
constexpr int SA_THREADS = 256, SA_WARPS = SA_THREADS / 32, SA_HEADS = 4, SA_BLOCKS = 2;   // (the last: a multiprocessor's)

// A lane has elements 4 lane .. + 3 of a head's first 128, and of its second.  The sums of 32 neighbouring values as the xor-tree over
// a warp forms them, offsets 16 .. 1: at each step lanes share the work out, so nobody adds what another adds.  Lanes 8 g .. + 7
// get the sum of the first 128's 32 from 32 g on; with E = 8 only the first four of them, and the last four the second 128's.
template <int E> __device__ __forceinline__ float sa_tree(const float* q, int lane) {
    const bool b2 = lane & 4, b1 = lane & 2, b0 = lane & 1;
    auto add = [](float own, float give, int mask) { return fadd(own, __shfl_xor_sync(0xffffffffu, give, mask)); };
    if constexpr (E == 8) {
        float a[4], b[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = add(b2 ? q[4 + i] : q[i], b2 ? q[i] : q[4 + i], 4);           // offset 16
#pragma unroll
        for (int i = 0; i < 2; ++i) b[i] = add(b1 ? a[2 + i] : a[i], b1 ? a[i] : a[2 + i], 2);           // offset 8
        float c = add(b0 ? b[1] : b[0], b0 ? b[0] : b[1], 1);                                            // offset 4; element 2 b1 + b0
        c = add(c, c, 2);                                                                                // offset 2
        return add(c, c, 1);                                                                             // offset 1
    } else {
        float a[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) a[i] = add(b2 ? q[2 + i] : q[i], b2 ? q[i] : q[2 + i], 4);           // offset 16
        float c = add(b1 ? a[1] : a[0], b1 ? a[0] : a[1], 2);                                            // offset 8; element 2 b2 + b1
        c = add(c, c, 1);                                                                                // offset 4
        c = add(c, c, 4);                                                                                // offset 2
        return add(c, c, 2);                                                                             // offset 1
    }
}
__device__ __forceinline__ void sa_get(float* x, const float* p) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
}

template <int HD>
__global__ void __launch_bounds__(SA_THREADS, SA_BLOCKS) k_seqs_append(const __grid_constant__ SaArgs a) {
    constexpr int E = HD / 32, CHUNK = SA_HEADS * SA_WARPS;
    extern __shared__ __align__(16) unsigned char sa_ring[];   // [2][SA_HEADS][SA_WARPS][HD] floats: a warp's own heads
    __shared__ __align__(16) float sn[2][SA_WARPS][64], cs[2][SA_WARPS][64], wt[2][HD];
    __shared__ __align__(16) float sums[SA_WARPS][SA_HEADS][E];
    __shared__ long long place[2][SA_WARPS];   // of the rows prepared together: where K and V go (-1: nowhere, -2: not even a query)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nh = a.nq + 2 * a.nkv, chunks = (nh + CHUNK - 1) / CHUNK;
    const int begin = (int) ((long long) a.sq.rows * blockIdx.x / gridDim.x), end = (int) ((long long) a.sq.rows * (blockIdx.x + 1) / gridDim.x);
    const unsigned ring = (unsigned) __cvta_generic_to_shared(sa_ring) + warp * HD * 4;
    const size_t row_elems = (size_t) a.nkv * HD;
    auto load = [&](int t, int chunk, int stage) {   // a row's heads chunk * CHUNK .., whole lines
        if (t < end) {
            const float *rq = a.qg + (size_t) t * a.nq * 2 * HD + lane * 4, *rk = a.k + (size_t) t * row_elems + lane * 4, *rv = a.v + (size_t) t * row_elems + lane * 4;
#pragma unroll
            for (int b = 0; b < SA_HEADS; ++b) {
                const int h = chunk * CHUNK + b * SA_WARPS + warp;
                if (h >= nh) break;
                const float* src = h < a.nq ? rq + h * 2 * HD : h < a.nq + a.nkv ? rk + (h - a.nq) * HD : rv + (h - a.nq - a.nkv) * HD;
#pragma unroll
                for (int e = 0; e < E / 4; ++e)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ring + ((stage * SA_HEADS + b) * SA_WARPS * HD + e * 128 + lane * 4) * 4), "l"(src + 128 * e)
                                 : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    pdl_wait();
    pdl_go();
    load(begin, 0, 0);   // on its way while the rows' places and angles are worked out
    for (int i = threadIdx.x; i < HD; i += SA_THREADS) wt[0][i] = a.qn[i], wt[1][i] = a.kn[i];
    // element i < nrot pairs with i -+ half: the lower one becomes x c - x' s, the upper one x c + x' s, the first product rounded before the
    // fused second.  Whole lanes apart (half a multiple of 4) the partner comes by a shuffle, else through shared memory
    const int half = a.nrot / 2, apart = half % 4 ? 0 : half / 4;
    const bool turned = lane * 4 < a.nrot, lower = lane * 4 < half;
    int stage = 0;
    auto prepare = [&](int t, int set) {   // a warp's row of the eight
        if (t >= end) return;
        const int s = sq_find(a.sq.row0, a.sq.nseq, t);
        long long at = -2;
        if (s >= 0) {
            const int i0 = t - a.sq.row0[s], p0 = a.sq.pos0[s];
            const int turn = max(0, p0) + (a.depth ? max(0, a.depth[t]) : i0);
            for (int i = lane; i < half; i += 32) ex_sincos((double) fmul((float) turn, a.freq[i]), &sn[set][warp][i], &cs[set][warp][i]);
            const long long cell = sq_cell(a.sq, a.g, s, p0 < 0 || i0 > INT_MAX - p0 ? -1 : p0 + i0);
            if (lane == 0 && cell < 0) atomicOr(a.err, SQ_ERR_ROOM);
            at = cell < 0 ? -1 : (long long) sq_at(a.sq, a.g, cell, row_elems);
        }
        if (lane == 0) place[set][warp] = at;
    };
    int set = 1;
    for (int t0 = begin - SA_WARPS; t0 < end; t0 += SA_WARPS, set ^= 1) {
        prepare(t0 + SA_WARPS + warp, set ^ 1);   // the next eight before these
        if (t0 >= begin)
            for (int t = t0; t < min(t0 + SA_WARPS, end); ++t)
            for (int chunk = 0; chunk < chunks; ++chunk, stage ^= 1) {
                __syncwarp();
                load(chunk + 1 < chunks ? t : t + 1, chunk + 1 < chunks ? chunk + 1 : 0, stage ^ 1);   // (what lay there is in registers and used)
                asm volatile("cp.async.wait_group 1;" ::: "memory");
                __syncwarp();
                const long long at = place[set][t - t0];
                if (at == -2) continue;   // behind the last sequence
                const int h0 = chunk * CHUNK + warp;
                float x[SA_HEADS][E], c[4], d[4];
                if (turned && apart) {   // the rotation's factors of this lane's elements and of their partners
                    const int i = lane * 4 - (lower ? 0 : half);
                    sa_get(c, lower ? &cs[set][t - t0][i] : &sn[set][t - t0][i]), sa_get(d, lower ? &sn[set][t - t0][i] : &cs[set][t - t0][i]);
                }
#pragma unroll
                for (int b = 0; b < SA_HEADS; ++b)
#pragma unroll
                    for (int e = 0; e < E; e += 4)
                        if (h0 + b * SA_WARPS < nh)
                            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                                         : "=f"(x[b][e]), "=f"(x[b][e + 1]), "=f"(x[b][e + 2]), "=f"(x[b][e + 3])
                                         : "r"(ring + ((stage * SA_HEADS + b) * SA_WARPS * HD + e * 32 + lane * 4) * 4)
                                         : "memory");
                float* rot = reinterpret_cast<float*>(sa_ring) + (stage * SA_HEADS * SA_WARPS + warp) * HD;   // (these values are in registers)
                // ---- the heads' square sums, one root for all: lane b takes head b's
#pragma unroll
                for (int b = 0; b < SA_HEADS; ++b) {
                    if (h0 + b * SA_WARPS >= a.nq + a.nkv) continue;
                    float q[E];
#pragma unroll
                    for (int e = 0; e < E; ++e) q[e] = fmul(x[b][e], x[b][e]);
                    const float group = sa_tree<E>(q, lane);
                    if (lane % (E == 8 ? 4 : 8) == 0) sums[warp][b][E == 8 ? (lane >> 3) + (lane & 4) : lane >> 3] = group;
                }
                __syncwarp();
                float g[E], tot = 0.f;
#pragma unroll
                for (int e = 0; e < E; e += 4) sa_get(g + e, &sums[warp][lane % SA_HEADS][e]);
#pragma unroll
                for (int e = 0; e < E; ++e) tot = fadd(tot, g[e]);
                const float mine = ex_rsqrt(fadd(fmul(tot, 1.0f / (float) HD), a.eps));   // (HD is a power of two: the quotient's bits)
#pragma unroll
                for (int b = 0; b < SA_HEADS; ++b) {
                    const int h = h0 + b * SA_WARPS;
                    if (h >= nh) break;
                    if (h < a.nq + a.nkv) {
                        const float r = __shfl_sync(0xffffffffu, mine, b);
#pragma unroll
                        for (int e = 0; e < E; e += 4) {
                            float w[4];
                            sa_get(w, &wt[h < a.nq ? 0 : 1][e * 32 + lane * 4]);
#pragma unroll
                            for (int i = 0; i < 4; ++i) x[b][e + i] = fmul(fmul(x[b][e + i], r), w[i]);
                        }
                        if (apart) {
                            float other[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) other[e] = __shfl_sync(0xffffffffu, x[b][e], lower ? lane + apart : lane - apart);
                            if (turned)
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const float y = x[b][e];
                                    x[b][e] = ffma(lower ? -other[e] : y, d[e], fmul(lower ? y : other[e], c[e]));
                                }
                        } else {
                            __syncwarp();
                            if (turned)
#pragma unroll
                                for (int e = 0; e < 4; ++e) rot[lane * 4 + e] = x[b][e];
                            __syncwarp();
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int i = lane * 4 + e;
                                const float *sr = sn[set][t - t0], *cr = cs[set][t - t0];
                                if (i < half) x[b][e] = ffma(-rot[i + half], sr[i], fmul(x[b][e], cr[i]));
                                else if (i < a.nrot) x[b][e] = ffma(x[b][e], cr[i - half], fmul(rot[i - half], sr[i - half]));
                            }
                            __syncwarp();
                        }
                    }
                    if (h >= a.nq && at < 0) continue;
                    uint16_t* to = h < a.nq            ? a.q16 + ((size_t) t * a.nq + h) * HD
                                   : h < a.nq + a.nkv ? a.kc + at + (h - a.nq) * HD
                                                      : a.vc + at + (h - a.nq - a.nkv) * HD;
#pragma unroll
                    for (int e = 0; e < E; e += 4)
                        *reinterpret_cast<uint2*>(to + e * 32 + lane * 4) = make_uint2(sq_pack(x[b][e], x[b][e + 1]), sq_pack(x[b][e + 2], x[b][e + 3]));
                }
            }
        __syncthreads();
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

template <int HD> static int sa_launch(const SaArgs& a, void* st) {
    constexpr size_t ring = (size_t) 2 * SA_HEADS * SA_THREADS * HD / 8;
    if (smem_optin(k_seqs_append<HD>, ring, "attn_seqs_append")) return 1;
    launch(0, k_seqs_append<HD>, dim3(std::min(a.sq.rows, SA_BLOCKS * 148)), SA_THREADS, ring, strm(st), a);
    return launch_ok("attn_seqs_append");
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
    return hd == 256 ? sa_launch<256>(a, st) : sa_launch<128>(a, st);
}
}
