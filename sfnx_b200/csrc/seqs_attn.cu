// Attention of several sequences' rows over the f16 cache: prompts, chunks of prompts, single tokens and draft trees (no
// counterpart in the reference's windows), on the fifth-generation tensor cores.
//
// A CTA takes one KV head, up to 128 query rows of one sequence - 128 / qpk tokens (qpk query heads a KV head, rounded down), row
// m = token m / qpk, head m % qpk, so that one pass over K and V serves all heads that share them and single tokens fill more
// than one row - and a range of that sequence's positions in tiles of 128.  S = Q K^T (128 x 128 fp32, operands in shared memory)
// and O += P V (P in tensor memory as the A operand, V as it lies: dims contiguous, "MN-major") both accumulate in tensor
// memory.  Roles: warp 0 copies (TMA, K and V boxes found through the page table), warp 1 issues the MMAs, warps 4 - 11 take the
// softmax step: a thread has one row and half of a tile's columns, the halves of a row agree on the maximum through shared
// memory.
//   tensor memory: O (HD columns), one S tile (128), two P tiles (64 columns each, f16 pairs).  S(i + 1) is issued when the softmax
//   warps have S(i) in registers, so the tensor core computes it - and, when P(i) is written, O += P(i) V(i) - while they take
//   exponentials: a tile costs the longer of the two, not the sum.
//   shared memory: Q, and a ring of 32 KB slots (for HD 256 half a K tile: 128 rows x 128 dims, or half a V tile: 64 rows x 256
//   dims) that are asked for in the order of their use: K(0), K(1), V(0), K(2), V(1), ...
// Softmax: x = s log2 e / sqrt(hd); weights 2^(x - ref) against a reference that is raised - and O and the sums rescaled - only when
// a row's maximum has grown by more than 8 over it, so weights stay below 2^8 and (O, ref, z) is an exact partial for any
// reference.  z sums the weights in 32 bits before they are rounded to f16 for the product (2^-11 of a weight: the
// result's own rounding is as large; f16 queries, keys and values enter exactly).
// Positions past a CTA's last visible one are not loaded beyond their box; V rows there are cleared in shared memory, since a
// weight of zero times a stray NaN is a NaN.
// Few rows over many positions: nsplit CTAs share a sequence's positions, their (O, ref, z) are joined by a second kernel.
// Every wait on an mbarrier is bounded; on a timeout the fault word is set and the CTA ends with nothing in flight.
#include <cstring>

#include "exact_math.cuh"
#include "moe_internal.cuh"
#include "seqs.cuh"
#include "umma.cuh"

namespace fnxk {

constexpr int SA_ROWS = 128, SA_KT = 128, SA_SLOT = 32768, SA_THREADS = 384, SA_SOFT = 256;
template <int HD> struct SaShape {
    static constexpr int HALVES = HD / 128;                 // slots a K or V tile takes
    static constexpr int VROWS = SA_KT / HALVES;            // V rows a slot holds
    static constexpr int QBYTES = SA_ROWS * HD * 2;
    static constexpr int SLOTS = HD == 256 ? 5 : 6;
    static constexpr int COL_S = HD, COL_P = HD + SA_KT;    // tensor memory columns; O from 0
    static constexpr size_t SMEM = (size_t) QBYTES + (size_t) SLOTS * SA_SLOT + 1024 /* alignment */ + 2 * SA_ROWS * 4 + 256;
};

struct SqMaps {
    CUtensorMap q, k, v;
};
struct SqAttn {
    const float* qg;
    FnxKvPages g;
    FnxSeqs sq;
    const unsigned* anc;
    uint16_t* out;
    int out_stride, nq, nkv, words;
    int tok;      // tokens a CTA takes: 128 / qpk
    int box;      // cache rows a copy brings: a power of two that divides a page's rows
    int nsplit;
    float* part;  // [nsplit][rows][nq][HD], then (ref, z) [nsplit][rows][nq][2]
    unsigned* fault;
};

__device__ __forceinline__ void sa_init(unsigned long long* bar, unsigned n) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(um_s32(bar)), "r"(n));
}
__device__ __forceinline__ void sa_arrive(unsigned long long* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(um_s32(bar)) : "memory");
}
__device__ __forceinline__ void sa_tma3d(unsigned dst, const CUtensorMap* map, int x, int y, int z, unsigned long long* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map),
                 "r"(x), "r"(y), "r"(z), "r"(um_s32(bar))
                 : "memory");
}
// D[tmem] (+)= A B with A in tensor memory (a lane a row, two f16 a column)
__device__ __forceinline__ void sa_mma_ts(unsigned tmem, unsigned a, unsigned long long db, unsigned idesc, unsigned accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem), "r"(a), "l"(db),
                 "r"(idesc), "r"(accumulate)
                 : "memory");
}
// 32 columns of the calling thread's lane of tensor memory
__device__ __forceinline__ void sa_ld32(unsigned* r, unsigned addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, "
        "[%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
          "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
          "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void sa_st32(unsigned addr, const unsigned* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
        "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]),
        "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(addr)
        : "memory");
}
__device__ __forceinline__ void sa_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void sa_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void sa_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void sa_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Unit u of the call, a KV head of a sequence's token block: the sequences' blocks one after another, a sequence's last (its
// longest) first.  false: there are not that many.  Called by a converged warp.
struct SqUnit {
    int s, tok0, ntok, head, kv_len, pos0, row;   // sequence, first token, tokens, KV head, positions the CTA's rows see, packed row
};
__device__ __forceinline__ bool sq_unit(const SqAttn& a, int u, SqUnit& w) {
    const int lane = threadIdx.x & 31;
    int t = u / a.nkv;
    w.head = u % a.nkv;
    for (int s0 = 0; s0 < a.sq.nseq; s0 += 32) {
        const int s = s0 + lane;
        int r0 = 0, len = 0;
        if (s < a.sq.nseq) r0 = max(a.sq.row0[s], 0), len = max(min(a.sq.row0[s + 1], a.sq.rows) - r0, 0);
        const int mine = (len + a.tok - 1) / a.tok;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        const unsigned past = __ballot_sync(0xffffffffu, upto > t);
        if (past) {
            const int l = __ffs(past) - 1;
            const int b = __shfl_sync(0xffffffffu, upto, l) - 1 - t;   // blocks from the sequence's last back
            len = __shfl_sync(0xffffffffu, len, l), r0 = __shfl_sync(0xffffffffu, r0, l);
            w.s = s0 + l, w.tok0 = b * a.tok, w.ntok = min(a.tok, len - w.tok0), w.row = r0 + w.tok0;
            w.pos0 = max(a.sq.pos0[w.s], 0);
            const long long cap = a.sq.pt ? (long long) a.sq.pt_stride * a.g.rows : (long long) a.g.cap;
            w.kv_len = (int) min((long long) w.pos0 + (a.anc ? len : w.tok0 + w.ntok), cap);
            return true;
        }
        t -= __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
}
// the range of tiles that split `split` of a unit takes
__device__ __forceinline__ void sq_range(int kv_len, int split, int nsplit, int& first, int& n) {
    const int tiles = (kv_len + SA_KT - 1) / SA_KT, per = (tiles + nsplit - 1) / nsplit;
    first = min(split * per, tiles);
    n = min(per, tiles - first);
}

// 32 positions' visibility of a tree's row, from position rel past the sequence's pos0 on
__device__ __forceinline__ unsigned sq_tree_bits(const unsigned* anc, int words, int rel) {
    if (rel <= -32) return 0xffffffffu;
    if (rel < 0) return ((1u << -rel) - 1u) | ((words > 0 ? anc[0] : 0u) << -rel);
    const int w = rel >> 5, sh = rel & 31;
    const unsigned lo = w < words ? anc[w] : 0u, hi = w + 1 < words ? anc[w + 1] : 0u;
    return __funnelshift_r(lo, hi, sh);
}
__device__ __forceinline__ unsigned sq_first(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

template <int HD>
__global__ void __launch_bounds__(SA_THREADS, 1) k_attn_seqs(const __grid_constant__ SqMaps maps, const __grid_constant__ SqAttn a) {
    using S = SaShape<HD>;
    extern __shared__ unsigned char sa_smem[];
    unsigned char* Q = sa_smem + ((1024u - (um_s32(sa_smem) & 1023u)) & 1023u);
    unsigned char* ring = Q + S::QBYTES;
    float* xmax = reinterpret_cast<float*>(ring + S::SLOTS * SA_SLOT);   // [2][128] the halves' maxima (at the end: their sums)
    unsigned long long* bars = reinterpret_cast<unsigned long long*>(xmax + 2 * SA_ROWS);
    unsigned long long *full = bars, *empty = bars + S::SLOTS, *q_full = empty + S::SLOTS, *s_full = q_full + 1, *s_free = q_full + 2, *p_full = q_full + 3,
                       *o_full = q_full + 5, *idle = q_full + 7;
    volatile unsigned* tmem_at = reinterpret_cast<unsigned*>(q_full + 8);
    const int tid = threadIdx.x, warp = (int) um_uniform(tid >> 5), lane = tid & 31;
    pdl_wait();
    pdl_go();
    SqUnit w;
    if (!sq_unit(a, blockIdx.x, w)) return;
    int first, n;
    sq_range(w.kv_len, blockIdx.y, a.nsplit, first, n);
    if (n <= 0 && a.nsplit > 1) return;   // (the join knows)
    const int qpk = a.nq / a.nkv;
    if (tid == 0) {
        for (int i = 0; i < S::SLOTS; ++i) sa_init(&full[i], 1), sa_init(&empty[i], 1);
        sa_init(q_full, 1), sa_init(s_full, 1), sa_init(s_free, SA_SOFT / 32), sa_init(idle, 1);
        for (int i = 0; i < 2; ++i) sa_init(&p_full[i], SA_SOFT / 32), sa_init(&o_full[i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(um_s32((const void*) tmem_at)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    sa_before();
    __syncthreads();
    sa_after();
    const unsigned tm = um_uniform(*tmem_at);
    bool alive = true;

    if (warp == 0) {
        // ---- copies.  Load number c of the ring takes slot c % SLOTS; tile i's K loads come before tile i - 1's V loads
        int c = 0;
        const int boxes = SA_KT / a.box;
        auto acquire = [&]() {
            const int slot = c % S::SLOTS;
            if (c >= S::SLOTS) alive = alive && __all_sync(0xffffffffu, um_wait(&empty[slot], (unsigned) (c / S::SLOTS - 1) & 1u, a.fault));
            return slot;
        };
        // lane j < boxes: where box j of a tile lies (row in the page, page)
        auto place = [&](int tile, int& y, int& z) {
            const int p = tile * SA_KT + lane * a.box;
            y = z = 0;
            if (lane >= boxes || p >= w.kv_len) return;
            if (!a.sq.pt) {
                y = (a.sq.kv0 ? a.sq.kv0[w.s] : 0) + p;
                return;
            }
            const int page = a.sq.pt[(size_t) w.s * a.sq.pt_stride + p / a.g.rows];
            y = p % a.g.rows, z = page >= 0 && page < a.sq.npages ? page : a.sq.npages;   // past the pool: zeros
        };
        // rows lo .. hi - 1 of a tile, column blocks of 64 dims cb .. cb + nb - 1, into a slot; a block's rows are `stride` bytes apart from the next's
        auto load = [&](const CUtensorMap* map, int tile, int y, int z, int lo, int hi, int cb, int nb, int stride) {
            if (!alive) return;
            const int slot = acquire();
            if (!alive) return;
            const int have = min(hi, w.kv_len - tile * SA_KT) - lo, nbox = max(0, (have + a.box - 1) / a.box);
            const unsigned dst = um_s32(ring) + slot * SA_SLOT;
            const bool elected = um_elect();
            if (elected) um_expect_tx(&full[slot], (unsigned) (nbox * nb * a.box * 128));
            for (int j = 0; j < nbox; ++j) {
                const int at = lo / a.box + j, yj = __shfl_sync(0xffffffffu, y, at), zj = __shfl_sync(0xffffffffu, z, at);
                if (elected)
                    for (int b = 0; b < nb; ++b) sa_tma3d(dst + b * stride + j * a.box * 128, map, w.head * HD + (cb + b) * 64, yj, zj, &full[slot]);
            }
            __syncwarp();
            ++c;
        };
        if (n > 0 && um_elect()) {
            um_expect_tx(q_full, (unsigned) (a.tok * qpk * HD * 2));
            for (int b = 0; b < HD / 64; ++b) sa_tma3d(um_s32(Q) + b * (SA_ROWS * 128), &maps.q, b * 64, w.head * qpk, w.row, q_full);
        }
        __syncwarp();
        int y0, z0, y1, z1;
        if (n > 0) place(first, y0, z0);
        for (int i = 0; i < n && alive; ++i) {
            if (i == 0)
                for (int h = 0; h < S::HALVES; ++h) load(&maps.k, first, y0, z0, 0, SA_KT, 2 * h, 2, SA_KT * 128);
            if (i + 1 < n) {
                place(first + i + 1, y1, z1);
                for (int h = 0; h < S::HALVES; ++h) load(&maps.k, first + i + 1, y1, z1, 0, SA_KT, 2 * h, 2, SA_KT * 128);
            }
            for (int h = 0; h < S::HALVES; ++h) load(&maps.v, first + i, y0, z0, h * S::VROWS, (h + 1) * S::VROWS, 0, HD / 64, S::VROWS * 128);
            y0 = y1, z0 = z1;
        }
        // nothing is in flight when the block ends: the last load into every slot has landed (loads over another waited for its use)
        if (n > 0 && lane == 0) um_wait(q_full, 0u, a.fault);
        for (int k = max(0, c - S::SLOTS); k < c; ++k)
            if (lane == 0) um_wait(&full[k % S::SLOTS], (unsigned) (k / S::SLOTS) & 1u, a.fault);
        __syncwarp();
    } else if (warp == 1) {
        // ---- the MMAs
        int c = 0;   // slots used, in the order of their loads
        const unsigned idesc_s = (1u << 4) | ((SA_KT >> 3) << 17) | ((128u >> 4) << 24);                // S: both operands K-major
        const unsigned idesc_o = (1u << 4) | (1u << 16) | ((HD >> 3) << 17) | ((128u >> 4) << 24);   // O: B MN-major
        auto wait = [&](unsigned long long* bar, unsigned parity) {
            alive = alive && __all_sync(0xffffffffu, um_wait(bar, parity, a.fault));
            sa_after();
        };
        auto scores = [&]() {
            const unsigned long long dq = um_desc(um_s32(Q));
#pragma unroll 1
            for (int h = 0; h < S::HALVES; ++h, ++c) {
                const int slot = c % S::SLOTS;
                wait(&full[slot], (unsigned) (c / S::SLOTS) & 1u);
                if (!alive) return;
                const unsigned long long dk = um_desc(um_s32(ring) + slot * SA_SLOT);
                if (um_elect()) {
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks)
                            um_mma(tm + S::COL_S, dq + (unsigned long long) (((2 * h + b) * (SA_ROWS * 128) + ks * 32) >> 4),
                                   dk + (unsigned long long) ((b * (SA_KT * 128) + ks * 32) >> 4), idesc_s, (unsigned) (h | b | ks));
                    um_commit(&empty[slot]);
                    if (h == S::HALVES - 1) um_commit(s_full);
                }
                __syncwarp();
            }
        };
        auto output = [&](int i) {
            const int left = w.kv_len - (first + i) * SA_KT;   // positions of the tile that exist
#pragma unroll 1
            for (int h = 0; h < S::HALVES; ++h, ++c) {
                const int slot = c % S::SLOTS, have = min(left - h * S::VROWS, S::VROWS), steps = (have + 15) / 16;
                wait(&full[slot], (unsigned) (c / S::SLOTS) & 1u);
                if (!alive) return;
                unsigned char* v = ring + slot * SA_SLOT;
                if (have > 0 && have % 16) {   // rows of the last step past the newest position
                    for (int r = have; r < 16 * steps; ++r)
                        for (int x = lane; x < HD / 8; x += 32) *reinterpret_cast<uint4*>(v + (x >> 3) * (S::VROWS * 128) + r * 128 + (x & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                const unsigned long long dv = um_desc_x(um_s32(v), S::VROWS * 128, 1024, 2);
                if (um_elect()) {
                    for (int ks = 0; ks < steps; ++ks)
                        sa_mma_ts(tm, tm + S::COL_P + (i & 1) * (SA_KT / 2) + (h * S::VROWS + ks * 16) / 2, dv + (unsigned long long) (ks * 2048 >> 4), idesc_o,
                                  (unsigned) (i | h | ks));
                    um_commit(&empty[slot]);
                    if (h == S::HALVES - 1) um_commit(&o_full[i & 1]);
                }
                __syncwarp();
            }
        };
        if (n > 0) {
            wait(q_full, 0u);
            if (alive) scores();
        }
        for (int i = 0; i < n && alive; ++i) {
            if (i + 1 < n) {
                wait(s_free, (unsigned) i & 1u);   // S(i) is in registers
                if (alive) scores();
            }
            if (alive) wait(&p_full[i & 1], (unsigned) (i >> 1) & 1u);
            if (alive) output(i);
        }
        // nothing is under way when the block ends, also after a wait that ran out
        if (um_elect()) um_commit(idle);
        __syncwarp();
        um_wait(idle, 0u, a.fault);
    } else if (warp >= 4) {
        // ---- softmax: row m, columns 64 half .. + 63 of every tile
        const int half = (warp - 4) >> 2, m = (warp & 3) * 32 + lane, token = m / qpk, hh = m % qpk;
        const bool real = token < w.ntok;
        const unsigned tl = tm + ((unsigned) ((warp & 3) * 32) << 16);
        const float scale = 1.44269504f / sqrtf((float) HD);
        const int row = w.row + token;   // packed row
        // positions this row sees: the causal count, or all, with a mask from pos0 on
        const int lim = !real ? 0 : a.anc ? w.kv_len : min(w.kv_len, w.pos0 + w.tok0 + token + 1);
        const int clear = a.anc ? w.pos0 : w.pos0 + w.tok0 + 1;   // positions below are seen by every row
        const unsigned* anc = a.anc ? a.anc + (size_t) (real ? row : w.row) * a.words : nullptr;
        float ref = -INFINITY, z = 0.f;   // this row's reference (in units of log2) and this half's sum
        auto wait = [&](unsigned long long* bar, unsigned parity) {
            alive = alive && __all_sync(0xffffffffu, um_wait(bar, parity, a.fault));
            sa_after();
        };
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
            if (alive) wait(s_full, (unsigned) i & 1u);
            float x[64];
            if (alive) {
                sa_ld32(reinterpret_cast<unsigned*>(x), tl + S::COL_S + half * 64);
                sa_ld32(reinterpret_cast<unsigned*>(x) + 32, tl + S::COL_S + half * 64 + 32);
                sa_wait_ld();
            }
            sa_before();
            __syncwarp();
            if (lane == 0) sa_arrive(s_free);
            const int p0 = (first + i) * SA_KT + half * 64;
            if (p0 + 64 > min(clear, w.kv_len)) {
                unsigned see0 = sq_first(lim - p0), see1 = sq_first(lim - p0 - 32);
                if (a.anc) see0 &= sq_tree_bits(anc, a.words, p0 - w.pos0), see1 &= sq_tree_bits(anc, a.words, p0 + 32 - w.pos0);
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    if (!(see0 >> j & 1u)) x[j] = -INFINITY;
                    if (!(see1 >> j & 1u)) x[32 + j] = -INFINITY;
                }
            }
            float mx = x[0];
#pragma unroll
            for (int j = 1; j < 64; ++j) mx = fmaxf(mx, x[j]);
            xmax[half * SA_ROWS + m] = mx;
            asm volatile("bar.sync 1, %0;" ::"n"(SA_SOFT) : "memory");
            mx = fmaxf(mx, xmax[(half ^ 1) * SA_ROWS + m]) * scale;
            asm volatile("bar.sync 2, %0;" ::"n"(SA_SOFT) : "memory");   // read before the next tile's are written
            const bool up = mx > ref + 8.0f || (ref == -INFINITY && mx != -INFINITY);
            const float f = !up ? 1.0f : ref == -INFINITY ? 0.f : ex2_ftz(ref - mx);
            if (up) ref = mx;
            z *= f;
            if (i > 0 && __any_sync(0xffffffffu, up)) {   // O row *= f, this half's columns
                if (alive) wait(&o_full[(i - 1) & 1], (unsigned) ((i - 1) >> 1) & 1u);
                if (alive)
#pragma unroll 1
                    for (int cb = 0; cb < HD / 2; cb += 32) {
                        unsigned r[32];
                        sa_ld32(r, tl + half * (HD / 2) + cb);
                        sa_wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * f);
                        sa_st32(tl + half * (HD / 2) + cb, r);
                    }
            }
            const float base = ref == -INFINITY ? 0.f : ref;
            unsigned pk[32];
            float s0 = 0.f, s1 = 0.f;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
                const float p = ex2_ftz(fmaf(x[2 * j], scale, -base)), q = ex2_ftz(fmaf(x[2 * j + 1], scale, -base));
                s0 += p, s1 += q;
                const __half2 h = __floats2half2_rn(p, q);
                pk[j] = *reinterpret_cast<const unsigned*>(&h);
            }
            z += s0 + s1;
            if (i > 1 && alive) wait(&o_full[i & 1], (unsigned) ((i >> 1) - 1) & 1u);   // the P tile's last reader is done
            if (alive) sa_st32(tl + S::COL_P + (i & 1) * (SA_KT / 2) + half * 32, pk);
            sa_wait_st();
            sa_before();
            __syncwarp();
            if (lane == 0) sa_arrive(&p_full[i & 1]);
        }
        // ---- the rows' results
        xmax[half * SA_ROWS + m] = z;
        asm volatile("bar.sync 1, %0;" ::"n"(SA_SOFT) : "memory");
        z += xmax[(half ^ 1) * SA_ROWS + m];
        if (n > 0 && alive) wait(&o_full[(n - 1) & 1], (unsigned) ((n - 1) >> 1) & 1u);
        const float inv = z > 0.f ? 1.0f / z : 0.f;
        const int head = w.head * qpk + hh;
        const size_t cell = (size_t) row * a.nq + head, all = (size_t) a.sq.rows * a.nq;
#pragma unroll 1
        for (int cb = half * (HD / 2); cb < (half + 1) * (HD / 2); cb += 32) {
            unsigned r[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] = 0u;
            if (n > 0 && alive) {
                sa_ld32(r, tl + cb);
                sa_wait_ld();
            }
            if (!real) continue;
            if (a.nsplit > 1) {
                float* o = a.part + ((size_t) blockIdx.y * all + cell) * HD + cb;
#pragma unroll
                for (int j = 0; j < 32; j += 4) *reinterpret_cast<uint4*>(o + j) = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
                continue;
            }
            uint16_t* o = a.out + (size_t) row * a.out_stride + (size_t) head * HD + cb;
            const float* gate = a.qg ? a.qg + cell * 2 * HD + HD + cb : nullptr;
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
                float y[8];
                unsigned u[4];
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = z > 0.f ? __uint_as_float(r[j + e]) * inv : 0.f;
                if (gate)
#pragma unroll
                    for (int e = 0; e < 8; e += 4) {
                        const float4 t = *reinterpret_cast<const float4*>(gate + j + e);
                        y[e] = __fdividef(y[e], 1.0f + __expf(-t.x)), y[e + 1] = __fdividef(y[e + 1], 1.0f + __expf(-t.y));
                        y[e + 2] = __fdividef(y[e + 2], 1.0f + __expf(-t.z)), y[e + 3] = __fdividef(y[e + 3], 1.0f + __expf(-t.w));
                    }
#pragma unroll
                for (int e = 0; e < 4; ++e) u[e] = (unsigned) f2h(y[2 * e]) | ((unsigned) f2h(y[2 * e + 1]) << 16);
                *reinterpret_cast<uint4*>(o + j) = make_uint4(u[0], u[1], u[2], u[3]);
            }
        }
        if (a.nsplit > 1 && real && half == 0)
            *reinterpret_cast<float2*>(a.part + (size_t) a.nsplit * all * HD + ((size_t) blockIdx.y * all + cell) * 2) = make_float2(ref, z);
    }
    sa_before();
    __syncthreads();
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(512));
}

// the splits' partials of row t, head h joined (a warp a head), gated and rounded
template <int HD> __global__ void __launch_bounds__(128) k_attn_seqs_join(const __grid_constant__ SqAttn a) {
    constexpr int E = HD / 32;
    const int t = blockIdx.x, h = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    pdl_wait();
    pdl_go();
    const int s = sq_find(a.sq.row0, a.sq.nseq, t);
    if (s < 0 || h >= a.nq) return;
    const int r0 = max(a.sq.row0[s], 0), len = min(a.sq.row0[s + 1], a.sq.rows) - r0, i0 = t - r0, pos0 = max(a.sq.pos0[s], 0);
    const long long cap = a.sq.pt ? (long long) a.sq.pt_stride * a.g.rows : (long long) a.g.cap;
    const int kv_len = (int) min((long long) pos0 + (a.anc ? len : min(len, (i0 / a.tok + 1) * a.tok)), cap);   // as the row's CTAs had it
    const size_t all = (size_t) a.sq.rows * a.nq, cell = (size_t) t * a.nq + h;
    const float* mz = a.part + (size_t) a.nsplit * all * HD;
    float ref = -INFINITY, z = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    for (int p = 0; p < a.nsplit; ++p) {
        int first, n;
        sq_range(kv_len, p, a.nsplit, first, n);
        if (n <= 0) break;
        const float2 x = *reinterpret_cast<const float2*>(mz + ((size_t) p * all + cell) * 2);
        if (x.x == -INFINITY) continue;   // the row sees nothing there
        const float rn = fmaxf(ref, x.x), f0 = ex2_ftz(ref - rn), f1 = ex2_ftz(x.x - rn);
        z = z * f0 + x.y * f1;
        ref = rn;
        const float* src = a.part + ((size_t) p * all + cell) * HD + lane * E;
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const float4 v = *reinterpret_cast<const float4*>(src + e);
            o[e] = o[e] * f0 + v.x * f1, o[e + 1] = o[e + 1] * f0 + v.y * f1, o[e + 2] = o[e + 2] * f0 + v.z * f1, o[e + 3] = o[e + 3] * f0 + v.w * f1;
        }
    }
    const float inv = z > 0.f ? 1.0f / z : 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        float y = o[e] * inv;
        if (a.qg) y = __fdividef(y, 1.0f + __expf(-a.qg[cell * 2 * HD + HD + lane * E + e]));
        a.out[(size_t) t * a.out_stride + (size_t) h * HD + lane * E + e] = f2h(y);
    }
}

// CTAs that share a unit's positions: as many as make the fewest rounds of the GPU's 148, a round's length taken as the longest
// split's tiles and three more for a CTA's beginning and end
static int sq_splits(long long units, long long positions) {
    const long long tiles = (positions + SA_KT - 1) / SA_KT;
    long long best = 0;
    int ns = 1;
    for (int s = 1; s <= 64 && s <= tiles; ++s) {
        const long long per = (tiles + s - 1) / s;
        if ((tiles + per - 1) / per != s) continue;   // the same longest split with fewer
        const long long cost = (units * s + 147) / 148 * (per + 3) + (s > 1 ? 3 : 0);
        if (s == 1 || cost < best) best = cost, ns = s;
    }
    return ns;
}
static long long sq_units(const FnxSeqs* sq, int tok, int nkv) {   // at most
    const long long blocks = (long long) sq->rows / tok + sq->nseq;
    return (blocks < sq->rows ? blocks : (long long) sq->rows) * nkv;
}
// what a split is decided by: the units at most, and the positions a sequence has at most - where the caller does not say, 64 a
// page (the scratch is sized from the same struct, which does not know a page's rows), and one split without pages
static int sq_plan(const FnxSeqs* sq, int nq, int nkv) {
    const int tok = SA_ROWS / (nq / nkv);
    return sq_splits(sq_units(sq, tok, nkv), sq->max_pos ? sq->max_pos : sq->pt ? (long long) sq->pt_stride * 64 : 0);
}

template <int HD> static int sq_launch(const SqMaps& maps, const SqAttn& a, long long units, const char* what, cudaStream_t st) {
    if (cudaFuncSetAttribute(k_attn_seqs<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) SaShape<HD>::SMEM) != cudaSuccess)
        return fail("%s: shared memory opt-in: %s", what, cudaGetErrorString(cudaGetLastError()));
    launch(0, k_attn_seqs<HD>, dim3((unsigned) units, a.nsplit), SA_THREADS, SaShape<HD>::SMEM, st, maps, a);
    if (launch_ok(what)) return 1;
    if (a.nsplit == 1) return 0;
    launch(0, k_attn_seqs_join<HD>, dim3(a.sq.rows, (a.nq + 3) / 4), 128, 0, st, a);
    return launch_ok(what);
}

static int attn_seqs(const uint16_t* q16, int q_stride, const float* qg, const uint16_t* kc, const uint16_t* vc, FnxKvPages g, const FnxSeqs* sq,
                     const unsigned* anc, int words, uint16_t* out, int out_stride, int nq, int nkv, int hd, void* scratch, void* st, const char* what) {
    if (sq_check(sq, g, nq, nkv, hd, what)) return 1;
    FNX_REQUIRE(q16 && kc && vc && out && scratch, "%s: a null buffer", what);
    FNX_REQUIRE(((uintptr_t) q16 | (uintptr_t) qg | (uintptr_t) kc | (uintptr_t) vc | (uintptr_t) out | (uintptr_t) scratch) % 16 == 0,
                "%s: a buffer that is not 16-byte aligned", what);
    FNX_REQUIRE(q_stride >= nq * hd && q_stride % 8 == 0 && out_stride >= nq * hd && out_stride % 8 == 0,
                "%s: rows of %d halves %d and %d apart (multiples of 8)", what, nq * hd, q_stride, out_stride);
    FNX_REQUIRE(!sq->pt || g.rows % 8 == 0, "%s: pages of %d rows (a multiple of 8)", what, g.rows);
    const int qpk = nq / nkv, tok = SA_ROWS / qpk;
    int box = 64;
    while (sq->pt && g.rows % box) box /= 2;
    unsigned* fault = device_fault_word();
    UmEncode enc = um_encoder();
    FNX_REQUIRE(fault && enc, "%s: no fault word or no tensor-map encoder", what);
    SqMaps maps;
    memset(&maps, 0, sizeof(maps));
    const cuuint32_t es[3] = {1, 1, 1};
    const cuuint64_t qd[3] = {(cuuint64_t) hd, (cuuint64_t) nq, (cuuint64_t) sq->rows}, qs[2] = {(cuuint64_t) hd * 2, (cuuint64_t) q_stride * 2};
    const cuuint32_t qb[3] = {64, (cuuint32_t) qpk, (cuuint32_t) tok};
    const cuuint64_t row = (cuuint64_t) nkv * hd, rows = sq->pt ? g.rows : g.cap;
    const cuuint64_t kd[3] = {row, rows, (cuuint64_t) (sq->pt ? sq->npages : 1)}, ks[2] = {row * 2, sq->pt ? (cuuint64_t) g.page * 2 : rows * row * 2};
    const cuuint32_t kb[3] = {64, (cuuint32_t) box, 1};
    auto encode = [&](CUtensorMap* m, const void* p, const cuuint64_t* d, const cuuint64_t* s, const cuuint32_t* b) {
        return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(p), d, s, b, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    };
    FNX_REQUIRE(encode(&maps.q, q16, qd, qs, qb) && encode(&maps.k, kc, kd, ks, kb) && encode(&maps.v, vc, kd, ks, kb),
                "%s: no tensor map for %d rows %d apart or %d pages of %zu halves", what, sq->rows, q_stride, sq->npages, g.page);
    const long long units = sq_units(sq, tok, nkv);
    FNX_REQUIRE(units < (1ll << 31), "%s: %d rows of %d KV heads", what, sq->rows, nkv);
    const int ns = sq_plan(sq, nq, nkv);
    const SqAttn a{qg, g, *sq, anc, out, out_stride, nq, nkv, words, tok, box, ns, (float*) scratch, fault};
    return hd == 256 ? sq_launch<256>(maps, a, units, what, strm(st)) : sq_launch<128>(maps, a, units, what, strm(st));
}

}  // namespace fnxk

using namespace fnxk;

extern "C" {

size_t fnx_attn_seqs_scratch_bytes(const FnxSeqs* sq, int nq, int nkv, int hd) {
    if (!sq || nq < 1 || nkv < 1 || hd < 1 || nq % nkv || nq / nkv > 16 || sq->nseq < 1 || sq->rows < 1) return 0;
    const int ns = sq_plan(sq, nq, nkv);
    return ns == 1 ? 16 : (size_t) ns * sq->rows * nq * (hd + 2) * 4;
}

int fnx_attn_prompt(const uint16_t* q16, int q_stride, const float* qg, const uint16_t* kc, const uint16_t* vc, FnxKvPages g, const FnxSeqs* sq,
                    uint16_t* out, int out_stride, int nq, int nkv, int hd, void* scratch, void* st) {
    return attn_seqs(q16, q_stride, qg, kc, vc, g, sq, nullptr, 0, out, out_stride, nq, nkv, hd, scratch, st, "attn_prompt");
}

int fnx_attn_tree(const uint16_t* q16, int q_stride, const float* qg, const uint16_t* kc, const uint16_t* vc, FnxKvPages g, const FnxSeqs* sq,
                  const unsigned* anc, int anc_words, uint16_t* out, int out_stride, int nq, int nkv, int hd, void* scratch, void* st) {
    FNX_REQUIRE(anc && anc_words >= 1, "attn_tree: no ancestor masks");
    return attn_seqs(q16, q_stride, qg, kc, vc, g, sq, anc, anc_words, out, out_stride, nq, nkv, hd, scratch, st, "attn_tree");
}
}
