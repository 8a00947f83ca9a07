// Attention of several sequences' rows over the f16 cache: prompts, chunks of prompts, single tokens and draft trees (no
// counterpart in the reference's windows), on the fifth-generation tensor cores.
//
// A unit of work is one KV head, up to 256 query rows of one sequence - 2 x 128 / qpk tokens (qpk query heads a KV head, rounded
// down); row m of each 128 is token m / qpk, head m % qpk, so that one pass over K and V serves all heads that share them and
// single tokens fill more than one row - and the positions they see, in tiles of 128.  A pair of CTAs on neighbouring
// multiprocessors takes it (cta_group::2): each holds 128 of the rows, and half of every K tile (64 positions) and V tile (half of
// the dims), which the pair's MMAs read from both, so a tile crosses from L2 once for 256 rows.  (One CTA a unit moved 128 KB
// of K and V a tile and 128 rows, 11 TB/s out of L2 at 880 TFLOP/s, and was bound by it.)
// The work of all units, one after another, is dealt to the pairs (one on every two multiprocessors, persistent) in equal runs,
// whatever the sequences' lengths; where a run begins or ends inside a unit the pair leaves its part of the result, (O,
// reference, z), and a second kernel joins the parts.
// S = Q K^T (256 x 128 fp32, operands in shared memory) and O += P V (P in tensor memory as the A operand, V as it lies: dims
// contiguous, "MN-major") both accumulate in tensor memory, each CTA's rows in its own.  Roles: warp 0 copies (TMA, K and V
// boxes found through the page table; both CTAs' copies count on the first one's barriers), warp 1 of the first CTA issues the MMAs,
// warp 2 clears V rows behind a sequence's newest, warps 4 - 11 take the softmax step: a thread has one row and half of a tile's columns,
// the halves of a row agree on the maximum through shared memory.
//   tensor memory: O (HD columns), one S tile (128), two P tiles (64 columns each, f16 pairs).  S(i + 1) is issued when the softmax
//   warps have S(i) in registers, and O += P(i - 1) V(i - 1) behind it, so the tensor core has both to do while they take
//   exponentials: a tile costs the longer of the two, not the sum.  (With O += P(i) V(i) issued as soon as P(i) is written, S(i + 1)
//   came behind it and the softmax warps waited for it every other tile: 2500 and 3600 cycles a tile.)  The next unit's copies
//   and first scores run while the softmax warps write this one's rows.
//   shared memory: Q, a ring of slots of half a tile each, asked for in the order of their use: K(0), K(1), K(2), V(0), K(3),
//   V(1), ..., and a strip a softmax warp to turn rows into whole lines on their way out.
// Softmax: x = s log2 e / sqrt(hd); weights 2^(x - ref + 7) against a reference that is raised - and O and the sums rescaled - only when
// a row's maximum has grown by more than 8 over it, so weights stay below 2^15, what f16 holds, and (O, ref, z) is an exact partial
// for any reference (the 7 is a factor of O and z alike).  z sums the weights in 32 bits before they are rounded to f16 for the
// product: by 2^-11 of a weight (f16 queries, keys and values enter exactly) or, of a weight below 2^-21 of the reference's, by 2^-32
// of that one's.  Many such weights can be the whole result, where the position that has the rest holds zeros: without the 7, 3000 of
// 2^-25.5 of the largest were lost, now they are off by 1 %.  A tile's 128 x 128 exponentials are 1024 cycles of the special-function
// units; part of them is taken by a polynomial on the FMA units instead.
// O is summed by the tensor core: in 32 bits, a product cut off 25 places below the sum that it goes to, which for values of one
// sign costs a part of n positions about 2^-27 n of their weighted magnitude (measured: 4.2e-4 at 65 536 positions of one pair, 8.4e-4
// at 131 072; values of either sign 3.5e-6).
// Positions past a unit's last visible one are not loaded beyond their box; V rows there are cleared in shared memory, since a
// weight of zero times a stray NaN is a NaN.
// Every wait on an mbarrier is bounded; on a timeout the fault word is set and the CTA ends with nothing in flight.
#include <algorithm>
#include <cstring>

#include "exact_math.cuh"
#include "moe_internal.cuh"
#include "seqs.cuh"
#include "umma.cuh"

namespace fnxk {

constexpr int SA_ROWS = 128, SA_KT = 128, SA_THREADS = 384, SA_SOFT = 256, SA_STRIP = 4096;
// Of a thread's 32 pairs of exponentials a tile, those by polynomial: 1000 rows after 31 000 positions 600 us with 0, 593 with 8, 606
// with 12
constexpr int SA_POLY = 8;
constexpr int SA_LIFT = 7;   // weights are held 2^7 times as large, so that their smallest are not lost in f16
// What a unit's beginning and end cost, in positions (the dealing of the work): a prompt of 8192 tokens, whose first units are short,
// 692 us with 640, 647 with 768, 647 with 896; eight packed short prompts 33.0, 32.8, 33.4
constexpr int SA_COST = 768;
constexpr int SA_LEAST = 256;   // work a pair gets at least, in positions
template <int HD> struct SaShape {
    static constexpr int QBYTES = SA_ROWS * HD * 2;
    static constexpr int SLOT = SA_KT / 2 * HD * 2;         // half a K or V tile
    static constexpr int SLOTS = HD == 256 ? 4 : 8;
    static constexpr int COL_S = HD, COL_P = HD + SA_KT;    // tensor memory columns; O from 0
    static constexpr size_t SMEM = (size_t) QBYTES + (size_t) SLOTS * SLOT + SA_SOFT / 32 * SA_STRIP + 4 * SA_ROWS * 4 + 512;
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
    int tok;      // tokens of a CTA's rows: 128 / qpk
    int box, lg;  // cache rows a copy brings: a power of two that divides a page's rows; its logarithm
    int pairs;    // the scan's pairs of CTAs
    float4* part; // parts of units, as the threads hold them: [2 pairs][2][4 quarters of the rows][HD / 4][32 rows]
    float2* mz;   // their (ref, z): [2 pairs][2][128]
    int4* cuts;   // [pairs][2] what there is to join at the end of a pair's run
    unsigned* fault;
};

__device__ __forceinline__ void sa_init(unsigned long long* bar, unsigned n) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(um_s32(bar)), "r"(n));
}
// arrives at the barrier of the pair's first CTA that lies there where `bar` does in this one (`first`: from this one's addresses to that
// one's): sa_tell for tensor memory, whose accesses are ordered by the tcgen05 fences; sa_tell_shared for what this CTA's threads have
// written to shared memory, which is released to the cluster and acquired there at that scope (a release takes 1000 cycles: with one a
// tile, twelve single tokens took 139 us instead of 104)
__device__ __forceinline__ void sa_tell(unsigned long long* bar, unsigned first) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(um_s32(bar) + first) : "memory");
}
__device__ __forceinline__ void sa_tell_shared(unsigned long long* bar, unsigned first) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(um_s32(bar) + first) : "memory");
}
// both CTAs of the pair, every thread.  Without a release (1000 cycles): before it come the barriers' own fence and a barrier of the
// CTA for what that shares, or nothing that the other one reads
__device__ __forceinline__ void sa_cluster() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// boxes into this CTA's shared memory (plain loads: no multicast), their bytes counted on `bar`, an address in either CTA of the pair
__device__ __forceinline__ void sa_tma4d(unsigned dst, const CUtensorMap* map, int x, int y, int z, int w, unsigned bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void sa_tma3d(unsigned dst, const CUtensorMap* map, int x, int y, int z, unsigned bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}
// the pair's MMAs, 256 rows: D[tmem] (+)= A B, each CTA's half of A's rows and of B's columns in its own memories
__device__ __forceinline__ void sa_mma(unsigned tmem, unsigned long long da, unsigned long long db, unsigned idesc, unsigned accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem), "l"(da), "l"(db),
                 "r"(idesc), "r"(accumulate)
                 : "memory");
}
// the same with A in tensor memory (a lane a row, two f16 a column)
__device__ __forceinline__ void sa_mma_ts(unsigned tmem, unsigned a, unsigned long long db, unsigned idesc, unsigned accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem), "r"(a), "l"(db),
                 "r"(idesc), "r"(accumulate)
                 : "memory");
}
// `bar` of both CTAs gets one arrival when every MMA that this thread has issued is done
__device__ __forceinline__ void sa_commit(unsigned long long* bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(um_s32(bar)), "h"((unsigned short) 3)
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

// A unit: a KV head of a sequence's block of 2 tok tokens.  Units follow one another head by head, block by block, sequence by
// sequence; a unit's work is counted as SA_COST and the positions it sees.
struct SqUnit {
    int s, r0, len, pos0;   // sequence, its first packed row, its rows, the positions before them
    int tok0, head;         // first token, KV head
    int end, kv_len;        // positions the unit's rows see; those of them that the cache has room for
};
__device__ __forceinline__ void sq_seq(const SqAttn& a, int s, int& r0, int& len, int& pos0) {
    r0 = max(a.sq.row0[s], 0), len = max(min(a.sq.row0[s + 1], a.sq.rows) - r0, 0), pos0 = min(max(a.sq.pos0[s], 0), 1 << 30);
}
// work of a KV head's first b blocks (all but a sequence's last are whole)
__device__ __forceinline__ long long sq_blocks(const SqAttn& a, int len, int pos0, int b) {
    const long long n = b, each = (long long) pos0 + SA_COST + (a.anc ? len : 0);
    return n * each + (a.anc ? 0 : n * (n + 1) * a.tok);
}
__device__ __forceinline__ long long sq_work(const SqAttn& a, int len, int pos0) {   // of a sequence
    return len ? (sq_blocks(a, len, pos0, (len - 1) / (2 * a.tok)) + pos0 + len + SA_COST) * a.nkv : 0;
}
__device__ __forceinline__ void sq_fill(const SqAttn& a, SqUnit& u) {
    u.end = u.pos0 + (a.anc ? u.len : min(u.tok0 + 2 * a.tok, u.len));
    const long long room = a.sq.pt ? (long long) a.sq.pt_stride * a.g.rows : (long long) a.g.cap - (a.sq.kv0 ? a.sq.kv0[u.s] : 0);
    u.kv_len = (int) max(0ll, min((long long) u.end, room));
}
__device__ __forceinline__ long long sq_shfl(long long v, int lane) { return __shfl_sync(0xffffffffu, v, lane); }
// how the work is dealt: all of it, and the pairs that get any
__device__ __forceinline__ long long sq_div(long long x, unsigned d) { return x >> 32 ? x / d : (long long) ((unsigned) x / d); }   // x >= 0
struct SqPlan {
    long long total, each;   // each = total / pairs
    int pairs;
    __device__ __forceinline__ long long begin(int g) const { return each * g + (unsigned) (total - each * pairs) * (unsigned) g / (unsigned) pairs; }
};
// a lane's sequence of 32 neighbouring ones: its rows and the work up to and with it
struct SqLane {
    int r0, len, pos0;
    long long mine, upto;
    __device__ __forceinline__ void get(const SqAttn& a, int s) {   // called by a converged warp
        r0 = len = pos0 = 0;
        if (s < a.sq.nseq) sq_seq(a, s, r0, len, pos0);
        mine = upto = sq_work(a, len, pos0);
        if (a.sq.nseq == 1) {   // (lane 0's, all the same)
            upto = sq_shfl(upto, 0);
            return;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, upto, o);
            if ((int) (threadIdx.x & 31) >= o) upto += y;
        }
    }
};
// called by a converged warp; `lanes`: the first 32 sequences
__device__ __forceinline__ SqPlan sq_plan(const SqAttn& a, SqLane& lanes) {
    const int lane = threadIdx.x & 31;
    lanes.get(a, lane);
    long long w = sq_shfl(lanes.upto, 31);
    for (int s0 = 32; s0 < a.sq.nseq; s0 += 32) {
        SqLane more;
        more.get(a, s0 + lane);
        w += sq_shfl(more.upto, 31);
    }
    SqPlan p;
    p.total = w;
    p.pairs = (int) min((long long) a.pairs, w ? max(1ll, w / SA_LEAST) : 0ll);   // a run is never shorter than a tile
    p.each = p.pairs ? sq_div(w, p.pairs) : 0;
    return p;
}
// the unit that work item `at` (below the plan's total) belongs to; `at` is left relative to the unit.  Called by a converged warp
__device__ __forceinline__ SqUnit sq_locate(const SqAttn& a, const SqLane& lanes, long long& at) {
    const int lane = threadIdx.x & 31;
    SqUnit u;
    SqLane x = lanes;
    for (int s0 = 0;;) {   // the sequence
        const unsigned past = __ballot_sync(0xffffffffu, x.upto > at);
        if (past || s0 + 32 >= a.sq.nseq) {
            const int l = past ? __ffs(past) - 1 : 0;
            at -= sq_shfl(x.upto - x.mine, l);
            u.s = s0 + l, u.r0 = __shfl_sync(0xffffffffu, x.r0, l), u.len = __shfl_sync(0xffffffffu, x.len, l), u.pos0 = __shfl_sync(0xffffffffu, x.pos0, l);
            break;
        }
        at -= sq_shfl(x.upto, 31);
        s0 += 32;
        x.get(a, s0 + lane);
    }
    int lo = 0, hi = (u.len + 2 * a.tok - 1) / (2 * a.tok);   // the block: the last that does not begin past `at`
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, b = lo + lane * step;
        const unsigned in = __ballot_sync(0xffffffffu, b < hi && sq_blocks(a, u.len, u.pos0, b) * a.nkv <= at);
        lo += (__popc(in) - 1) * step;
        hi = min(hi, lo + step);
    }
    at -= sq_blocks(a, u.len, u.pos0, lo) * a.nkv;
    u.tok0 = lo * 2 * a.tok;
    sq_fill(a, u);
    u.head = (int) sq_div(at, u.end + SA_COST);
    at -= (long long) u.head * (u.end + SA_COST);
    return u;
}
__device__ __forceinline__ void sq_next(const SqAttn& a, SqUnit& u) {   // there is one
    if (++u.head < a.nkv) return;
    u.head = 0;
    u.tok0 += 2 * a.tok;
    while (u.tok0 >= u.len && u.s + 1 < a.sq.nseq) {
        ++u.s;
        u.tok0 = 0;
        sq_seq(a, u.s, u.r0, u.len, u.pos0);
    }
    sq_fill(a, u);
}
// the tile of a unit that work item x of it stands for: a run that ends at x ends before that tile
__device__ __forceinline__ int sq_tile(long long x) { return x <= SA_COST ? 0 : (int) ((x - SA_COST) / SA_KT); }

// A pair's run of work as segments, one a unit: tiles [t0, t0 + n) of it, n 0 where the cache ends before them
struct SqRun {
    SqUnit u;
    long long left;   // from the unit's beginning to the run's end
    int t0, n;
    int cut, first;   // the segment is part of its unit only; it is the run's first
    // field by field: a struct copied whole would live on the stack, 300 cycles from the MMAs' issue
    __device__ __forceinline__ void put(volatile int* w) const {
        w[0] = u.s, w[1] = u.r0, w[2] = u.len, w[3] = u.pos0, w[4] = u.tok0, w[5] = u.head, w[6] = u.end, w[7] = u.kv_len;
        w[8] = (int) left, w[9] = (int) (left >> 32), w[10] = t0, w[11] = n, w[12] = cut, w[13] = first;
    }
    __device__ __forceinline__ void get(const volatile int* w) {
        u.s = w[0], u.r0 = w[1], u.len = w[2], u.pos0 = w[3], u.tok0 = w[4], u.head = w[5], u.end = w[6], u.kv_len = w[7];
        left = (long long) ((unsigned long long) (unsigned) w[8] | ((unsigned long long) (unsigned) w[9] << 32)), t0 = w[10], n = w[11], cut = w[12], first = w[13];
    }
    __device__ __forceinline__ bool measure(int from) {
        const int tiles = (u.end + SA_KT - 1) / SA_KT, to = left >= u.end + SA_COST ? tiles : sq_tile(left);
        t0 = from;
        n = max(0, min(to, (u.kv_len + SA_KT - 1) / SA_KT) - t0);
        cut = from > 0 || to < tiles;
        return to > from;
    }
    __device__ __forceinline__ bool next(const SqAttn& a) {
        left -= u.end + SA_COST;
        if (left <= 0) return false;
        sq_next(a, u);
        first = 0;
        return measure(0);
    }
};

// 32 positions' visibility of a tree's row, from position rel past the sequence's pos0 on
__device__ __forceinline__ unsigned sq_tree_bits(const unsigned* anc, int words, int rel) {
    if (rel <= -32) return 0xffffffffu;
    if (rel < 0) return ((1u << -rel) - 1u) | ((words > 0 ? anc[0] : 0u) << -rel);
    const int w = rel >> 5, sh = rel & 31;
    const unsigned lo = w < words ? anc[w] : 0u, hi = w + 1 < words ? anc[w + 1] : 0u;
    return __funnelshift_r(lo, hi, sh);
}
__device__ __forceinline__ unsigned sq_first(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

// What there is to join where the run of pair g ends: the unit that is cut there, unless an earlier run's end has cut it before;
// (parts, the first part's place, first packed row, tokens), (head, 0, 0, 0).  Called by a converged warp
__device__ __forceinline__ void sq_cut(const SqAttn& a, const SqPlan& plan, const SqLane& lanes, int g, int4& x, int& head) {
    x = make_int4(0, 0, 0, 0), head = 0;
    if (g + 1 >= plan.pairs) return;
    const long long cut = plan.begin(g + 1);
    long long at = cut;
    const SqUnit u = sq_locate(a, lanes, at);
    const long long begin = cut - at;
    // the tile of the unit that the run of pair p begins with
    auto tile = [&](int p) { return plan.begin(p) <= begin ? 0 : sq_tile(plan.begin(p) - begin); };
    if (!sq_tile(at) || tile(g)) return;
    int parts = 2;
    while (g + parts < plan.pairs && plan.begin(g + parts) < begin + u.end + SA_COST) ++parts;
    // pair g's part is its run's first where the run does not begin in a unit before; the later pairs' runs begin inside the unit
    x = make_int4(parts, 2 * g + (plan.begin(g) >= begin ? 0 : 1), u.r0 + u.tok0, min(u.len - u.tok0, 2 * a.tok));
    head = u.head;
}

// whether V rows behind the newest position lie in the last 16 that tile t's product takes
__device__ __forceinline__ bool sq_unclean(int kv_len, int t) { return kv_len - t * SA_KT < SA_KT && kv_len % 16; }

// Waits for a phase of `bar`, at most `spins` polls of up to 16 us (asleep: warps that poll without a break keep the barriers'
// unit from the one that issues the MMAs); a wait that ran out is reported, and later ones of the thread do not linger
constexpr int SA_SPINS = 1 << 16;
__device__ __forceinline__ bool sa_wait(unsigned long long* bar, unsigned parity, int& spins, unsigned* fault) {
    unsigned ok = 0;
    for (int spin = 0; spin < spins && !ok; ++spin)
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok)
                     : "r"(um_s32(bar)), "r"(parity), "r"(16384u)
                     : "memory");
    if (!ok) spins = 1, atomicOr(fault, 8u);
    return ok != 0;
}
// the same for what both CTAs' threads have released with sa_tell_shared
__device__ __forceinline__ bool sa_wait_shared(unsigned long long* bar, unsigned parity, int& spins, unsigned* fault) {
    unsigned ok = 0;
    for (int spin = 0; spin < spins && !ok; ++spin)
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok)
                     : "r"(um_s32(bar)), "r"(parity), "r"(16384u)
                     : "memory");
    if (!ok) spins = 1, atomicOr(fault, 8u);
    return ok != 0;
}
// whether the phase is over
__device__ __forceinline__ bool sa_test(unsigned long long* bar, unsigned parity) {
    unsigned ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok)
                 : "r"(um_s32(bar)), "r"(parity)
                 : "memory");
    return ok != 0;
}
// the larger one, a NaN if either is
__device__ __forceinline__ float sa_max(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// 2^x of two values on the FMA units: x = n + f, n the nearest integer (by adding and taking away 1.5 2^23, whose low bits then hold
// n), a polynomial of degree 5 for 2^f on [-1/2, 1/2] (fitted to the relative error: 2.4e-7 with its roundings in 32 bits),
// n added to the exponent.  Below -126 (and of a NaN, which the row's maximum shows): 2^-126 or so instead of zero, which f16 rounds to
// zero and no sum notices (the lifted weights are 2^7 where the reference is)
__device__ __forceinline__ float2 sa_ex2_poly(float2 x) {
    const float magic = 12582912.f;
    x.x = fmaxf(x.x, -126.f), x.y = fmaxf(x.y, -126.f);
    const float2 t = add2(x, make_float2(magic, magic)), n = add2(t, make_float2(-magic, -magic));
    const float2 f = fma2(n, make_float2(-1.f, -1.f), x);
    float2 p = fma2(f, make_float2(1.3276456157e-3f, 1.3276456157e-3f), make_float2(9.6755409613e-3f, 9.6755409613e-3f));
    p = fma2(p, f, make_float2(5.5507134646e-2f, 5.5507134646e-2f));
    p = fma2(p, f, make_float2(2.4022120237e-1f, 2.4022120237e-1f));
    p = fma2(p, f, make_float2(6.9314694405e-1f, 6.9314694405e-1f));
    p = fma2(p, f, make_float2(1.0000001192f, 1.0000001192f));
    return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(t.x) << 23)), __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(t.y) << 23)));
}
// a pair of gated values: y / (1 + e^-g), one reciprocal for both (the gates cut at -40, where no f16 value has anything left)
__device__ __forceinline__ void sa_gate(float& y0, float& y1, float g0, float g1) {
    const float a = 1.0f + ex2_ftz(-1.44269504f * (g0 < -40.f ? -40.f : g0)), b = 1.0f + ex2_ftz(-1.44269504f * (g1 < -40.f ? -40.f : g1));
    const float am = fmaxf(a, 1.f), bm = fmaxf(b, 1.f);   // (only a NaN differs, and only its own value shall)
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(am * bm));
    y0 = fmaf(a, 0.f, y0 * (r * bm)), y1 = fmaf(b, 0.f, y1 * (r * am));
}
// the same by one lane for its warp (all lanes get the answer)
__device__ __forceinline__ bool sa_wait_warp(unsigned long long* bar, unsigned parity, int& spins, unsigned* fault) {
    bool ok = true;
    if (um_elect()) ok = sa_wait(bar, parity, spins, fault);
    __syncwarp();   // what that lane has seen, all have
    return __all_sync(0xffffffffu, ok);
}

template <int HD>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(SA_THREADS, 1) k_attn_seqs(const __grid_constant__ SqMaps maps, const __grid_constant__ SqAttn a) {
    using S = SaShape<HD>;
    extern __shared__ __align__(1024) unsigned char sa_smem[];
    unsigned char *Q = sa_smem, *ring = Q + S::QBYTES, *strips = ring + S::SLOTS * S::SLOT;
    float* xmax = reinterpret_cast<float*>(strips + SA_SOFT / 32 * SA_STRIP);   // [2][2][128] the halves' maxima, of odd and even tiles
    unsigned long long* bars = reinterpret_cast<unsigned long long*>(xmax + 4 * SA_ROWS);
    // ready, q_ready: both CTAs' copies have landed (their bytes, which the first CTA expects; or both have cleared their V rows).  full: this
    // CTA's copy of V rows of which some are to be cleared.  ready, q_ready, s_free, p_full, o_free count both CTAs', in the first
    // one's memory.  empty, q_empty, s_full, o_full: MMAs are done, told to both
    unsigned long long *full = bars, *empty = full + S::SLOTS, *ready = empty + S::SLOTS, *q_ready = ready + S::SLOTS, *q_empty = q_ready + 1, *s_full = q_ready + 2,
                       *s_free = q_ready + 3, *o_free = q_ready + 4, *idle = q_ready + 5, *p_full = q_ready + 6, *o_full = q_ready + 8;
    volatile unsigned *tmem_at = reinterpret_cast<unsigned*>(q_ready + 10), *work_at = tmem_at + 1;
    volatile int* run_at = reinterpret_cast<int*>(q_ready + 11);
    const int tid = threadIdx.x, warp = (int) um_uniform(tid >> 5), lane = tid & 31, rank = blockIdx.x & 1, g = blockIdx.x >> 1;
    unsigned first;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(first) : "r"(um_s32(bars)));
    first -= um_s32(bars);
    if (tid == 0) {
        for (int i = 0; i < S::SLOTS; ++i) sa_init(&full[i], 1), sa_init(&empty[i], 1), sa_init(&ready[i], 2);
        sa_init(q_ready, 1), sa_init(q_empty, 1), sa_init(s_full, 1), sa_init(s_free, 2 * (SA_SOFT / 32 + 1)), sa_init(o_free, 2 * SA_SOFT / 32);
        sa_init(idle, 1);
        for (int i = 0; i < 2; ++i) sa_init(&p_full[i], 2 * SA_SOFT / 32), sa_init(&o_full[i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0 && um_elect()) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.q) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.k) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.v) : "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(um_s32((const void*) tmem_at)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    if (rank && tid >= SA_THREADS - SA_SOFT) {   // Q, for a first unit without rows here
        for (int i = tid - (SA_THREADS - SA_SOFT); i < S::QBYTES / 16; i += SA_SOFT) reinterpret_cast<uint4*>(Q)[i] = make_uint4(0u, 0u, 0u, 0u);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    sa_before();
    __syncthreads();
    sa_cluster();   // barriers and tensor memory of both CTAs are there
    sa_after();
    const unsigned tm = um_uniform(*tmem_at);
    const int qpk = a.nq / a.nkv;
    int spins = SA_SPINS;
    pdl_wait();   // all of the above while the kernel before still runs
    pdl_go();
    if (warp == 3) {   // the pair's run of work, and what there is to join at its end
        SqLane lanes;
        const SqPlan plan = sq_plan(a, lanes);
        SqRun r = {};
        bool some = g < plan.pairs;
        if (some) {
            const long long lo = plan.begin(g);
            long long at = lo;
            r.u = sq_locate(a, lanes, at);
            r.left = plan.begin(g + 1) - lo + at;
            r.first = 1;
            some = r.measure(sq_tile(at));
        }
        if (lane == 0) {
            r.put(run_at);
            *work_at = some;
        }
        __syncwarp();
        asm volatile("bar.arrive 2, %0;" ::"n"(SA_THREADS) : "memory");   // the others go on while the record is made
        if (rank == 0) {
            int4 x;
            int head;
            sq_cut(a, plan, lanes, g, x, head);
            if (lane == 0) a.cuts[2 * g] = x, a.cuts[2 * g + 1] = make_int4(head, 0, 0, 0);
        }
    } else {
        asm volatile("bar.sync 2, %0;" ::"n"(SA_THREADS) : "memory");
    }
    const bool work = warp != 3 && um_uniform(*work_at) != 0;
    auto leave = [&]() {
        sa_before();
        asm volatile("bar.sync 0, %0;" ::"n"(SA_THREADS) : "memory");
        // the last MMAs' arrival in the second CTA.  Here, where the softmax warps have met the last o_full: from the role's beginning on the
        // bounded wait would have had to last as long as the whole run of work, which may be seconds
        if (rank && warp == 1) sa_wait_warp(idle, 0u, spins, a.fault);
        sa_cluster();   // the pair's MMAs read both CTAs' memories
        if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(512));
    };
    // the softmax warps hold 64 scores and 32 packed weights a thread: they take registers from the first four warps (128 x 72 +
    // 256 x 216 of the launch's 384 x 168)
    if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 0) {
        // ---- copies.  Load number c of the ring takes slot c % SLOTS; tile i's K load comes before tile i - 2's V load.  A slot
        // holds groups of 64 rows, each as column blocks of 64 dims (8 KB, swizzled)
        int c = 0, nseg = 0, kv0 = 0;
        unsigned odd = 0u;    // of a slot's bit: how often `full` was used
        bool zeroed = true;   // Q
        SqRun r;
        r.get(run_at);
        bool alive = true;
        // lane j looks after box j of a tile: the table's entry, asked for a tile ahead, and with it where the box lies
        auto entry = [&](int tile) {
            const int p = tile * SA_KT + lane * a.box;
            return a.sq.pt && lane * a.box < SA_KT && p < r.u.kv_len ? a.sq.pt[(size_t) r.u.s * a.sq.pt_stride + p / a.g.rows] : 0;
        };
        auto place = [&](int tile, int e, int& y, int& z) {   // row in the page, page (past the pool: zeros)
            const int p = tile * SA_KT + lane * a.box;
            y = a.sq.pt ? p % a.g.rows : kv0 + p, z = !a.sq.pt ? 0 : e >= 0 && e < a.sq.npages ? e : a.sq.npages;
        };
        // boxes of a tile's rows lo .. lo + rows - 1 that have positions
        auto boxes = [&](int tile, int lo, int rows) { return max(0, (min(rows, r.u.kv_len - tile * SA_KT - lo) + a.box - 1) >> a.lg); };
        // half a K tile (64 rows) or V tile (half of the dims) into the next slot.  One body for both: what this warp runs again every tile
        // takes the softmax warps' place in the instruction cache (with a body for each, eight packed prompts took 33.5 us instead of 32.9)
        auto load = [&](bool v, int tile, int y, int z) {
            const CUtensorMap* map = v ? &maps.v : &maps.k;
            const int lo = v ? 0 : rank * (SA_KT / 2), nb = v ? HD / 128 : HD / 64, x = r.u.head * (HD / 64) + (v ? rank * (HD / 128) : 0);
            const int slot = c % S::SLOTS, nbox = boxes(tile, lo, v ? SA_KT : SA_KT / 2), bytes = boxes(tile, 0, SA_KT) * (HD / 64) * 128 << a.lg;   // of both CTAs
            const bool dirty = v && sq_unclean(r.u.kv_len, tile);   // some rows will be cleared
            const unsigned dst = um_s32(ring) + slot * S::SLOT, bar = dirty ? um_s32(&full[slot]) : um_s32(&ready[slot]) + first;
            const int y0 = __shfl_sync(0xffffffffu, y, lo / 64), z0 = __shfl_sync(0xffffffffu, z, lo / 64), y1 = __shfl_sync(0xffffffffu, y, 1),
                      z1 = __shfl_sync(0xffffffffu, z, 1);   // of whole groups
            // the slot may be written; what will land there is expected (the other CTA's bytes may be counted before: the phase lasts until
            // both CTAs are here)
            auto claim = [&]() {
                if (c >= S::SLOTS && !sa_wait(&empty[slot], (unsigned) (c / S::SLOTS - 1) & 1u, spins, a.fault)) return false;
                if (dirty) um_expect_tx(&full[slot], (unsigned) (nbox * nb * 128 << a.lg));   // (`ready` is told when they are clean)
                else if (rank == 0) um_expect_tx(&ready[slot], (unsigned) bytes);
                else sa_tell(&ready[slot], first);   // (so that no slot goes round without this CTA, which may have no box to load)
                return true;
            };
            if (!alive) return;
            const bool elected = um_elect();
            bool ok = true;
            if (a.box == 64) {   // a box is a group, with its column blocks
                if (elected) {
                    ok = claim();
                    if (ok && nbox > 0) sa_tma4d(dst, map, 0, y0, x, z0, bar);
                    if (ok && nbox > 1) sa_tma4d(dst + nb * 8192, map, 0, y1, x, z1, bar);
                }
            } else {
                if (elected) ok = claim();
                for (int j = 0; j < nbox; ++j) {
                    const int at = lo / a.box + j, yj = __shfl_sync(0xffffffffu, y, at), zj = __shfl_sync(0xffffffffu, z, at), row = j * a.box;
                    if (elected && ok)
                        for (int b = 0; b < nb; ++b) sa_tma4d(dst + (row / 64 * nb + b) * 8192 + row % 64 * 128, map, 0, yj, x + b, zj, bar);
                }
            }
            __syncwarp();
            alive = __all_sync(0xffffffffu, ok);
            if (!alive) return;
            if (dirty) odd ^= 1u << slot;
            ++c;
        };
        for (bool more = work; more && alive; more = r.next(a)) {
            if (!r.n) continue;
            kv0 = !a.sq.pt && a.sq.kv0 ? a.sq.kv0[r.u.s] : 0;
            const int end = r.t0 + r.n;
            int e = entry(r.t0), y0 = 0, z0 = 0, y1 = 0, z1 = 0, y2 = 0, z2 = 0;
            if (nseg) alive = sa_wait_warp(q_empty, (unsigned) (nseg - 1) & 1u, spins, a.fault);   // the scores before are done
            if (!alive) break;
            const int tok0 = r.u.tok0 + rank * a.tok;
            if (rank == 0 && um_elect()) um_expect_tx(q_ready, (unsigned) ((tok0 + a.tok < r.u.len ? 2 : 1) * a.tok * qpk * HD * 2));
            if (tok0 < r.u.len) {
                if (um_elect())
                    for (int b = 0; b < HD / 64; ++b) sa_tma3d(um_s32(Q) + b * (SA_ROWS * 128), &maps.q, b * 64, r.u.head * qpk, r.u.r0 + tok0, um_s32(q_ready) + first);
                zeroed = false;
            } else if (!zeroed) {   // no rows of this CTA's: products with zeros take less power than with what lies there (no result depends on it)
                for (int i = lane; i < S::QBYTES / 16; i += 32) reinterpret_cast<uint4*>(Q)[i] = make_uint4(0u, 0u, 0u, 0u);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                zeroed = true;
            }
            __syncwarp();
            ++nseg;
            // K(t), then V(t - 2)
#pragma unroll 1
            for (int t = r.t0; t < end + 2; ++t) {
                if (t < end) {
                    place(t, e, y2, z2);
                    e = entry(t + 1);
                }
#pragma unroll 1
                for (int v = t < end ? 0 : 1; v <= (t >= r.t0 + 2) && alive; ++v) load(v != 0, v ? t - 2 : t, v ? y0 : y2, v ? z0 : z2);
                y0 = y1, z0 = z1, y1 = y2, z1 = z2;
            }
        }
        // nothing is in flight when the blocks end: the last loads have landed (a load over another waited for that one's use).  The second
        // CTA's count on the first one's barriers, and it waits for that one in leave()
        if (lane == 0) {
            spins = SA_SPINS;
            if (rank == 0) {
                if (nseg) sa_wait(q_ready, (unsigned) (nseg - 1) & 1u, spins, a.fault);
                for (int k = max(0, c - S::SLOTS); k < c; ++k) sa_wait(&ready[k % S::SLOTS], (unsigned) (k / S::SLOTS) & 1u, spins, a.fault);
            }
            for (int k = 0; k < S::SLOTS; ++k) sa_wait(&full[k], (odd >> k & 1u) ^ 1u, spins, a.fault);   // (true at once where it was not used)
        }
        __syncwarp();
    } else if (warp == 2) {
        // ---- V rows past the newest position, of the last step of 16 that is multiplied, cleared where they have landed.  This warp follows
        // the tiles by their scores, and S(i + 1) waits for it too: a phase met once, and no wait longer than a tile's
        int c = 0, j = 0;
        unsigned odd = 0u;
        SqRun r;
        r.get(run_at);
        for (bool more = work; more; more = r.next(a)) {
            if (!r.n) continue;
            c += 2 * r.n;
            const int t = r.t0 + r.n - 1, slot = (c - 1) % S::SLOTS, have = r.u.kv_len - t * SA_KT, dirty = sq_unclean(r.u.kv_len, t);   // the segment's last load
            // one wait for both (with a second place of it, whether reached or not, a prompt of 8192 took 674 us instead of 645)
#pragma unroll 1
            for (int i = 0; i < r.n + dirty; ++i) {
                const bool tile = i < r.n;
                sa_wait_warp(tile ? s_full : &full[slot], (tile ? (unsigned) j : odd >> slot) & 1u, spins, a.fault);
                if (tile) {
                    if (lane == 0) sa_tell(s_free, first);
                    ++j;
                    continue;
                }
                odd ^= 1u << slot;
                const unsigned row = um_s32(ring) + slot * S::SLOT + (have >> 6) * (HD / 128) * 8192 + (have & 63) * 128;   // the first to clear (all lie in one group)
#pragma unroll 1
                for (int k = lane; k < (16 - have % 16) * (HD / 16); k += 32)   // a row is HD / 128 blocks of 8 runs
                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(row + k / (HD / 16) * 128 + k / 8 % (HD / 128) * 8192 + k % 8 * 16), "r"(0u) : "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) sa_tell_shared(&ready[slot], first);
            }
        }
    } else if (warp == 1 && rank == 0) {
        // ---- the pair's MMAs, one lane's work from wait to commit
        int c = 0, j = 0, nseg = 0;   // slots used in the order of their loads (the elected lane's); tiles; segments
        bool alive = true;            // the elected lane's
        SqRun r;
        r.get(run_at);
        const unsigned idesc_s = (1u << 4) | ((SA_KT >> 3) << 17) | ((256u >> 4) << 24);             // S: both operands K-major
        const unsigned idesc_o = (1u << 4) | (1u << 16) | ((HD >> 3) << 17) | ((256u >> 4) << 24);   // O: B MN-major
        auto wait = [&](unsigned long long* bar, unsigned parity) {
            alive = alive && sa_wait(bar, parity, spins, a.fault);
            sa_after();
        };
        // short loops: an MMA takes the tensor core 64 or 128 cycles, and a long body would have to be fetched again every time, the
        // softmax warps' code having gone over it
        auto scores = [&](bool last) {   // (the elected lane)
            const int slot = c % S::SLOTS;
            wait(&ready[slot], (unsigned) (c / S::SLOTS) & 1u);
            ++c;
            if (!alive) return;
            unsigned long long dq = um_desc(um_s32(Q)), dk = um_desc(um_s32(ring) + slot * S::SLOT);
#pragma unroll 1
            for (int b = 0; b < HD / 64; ++b, dq += SA_ROWS * 128 >> 4, dk += 8192 >> 4)
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) sa_mma(tm + S::COL_S, dq + (ks * 32 >> 4), dk + (ks * 32 >> 4), idesc_s, (unsigned) (b | ks));
            sa_commit(&empty[slot]);
            sa_commit(s_full);
            if (last) sa_commit(q_empty);
        };
        auto output = [&](int t) {
            const int slot = c % S::SLOTS, steps = (min(r.u.kv_len - t * SA_KT, SA_KT) + 15) / 16;   // of 16 positions that exist
            alive = alive && sa_wait_shared(&ready[slot], (unsigned) (c / S::SLOTS) & 1u, spins, a.fault);
            ++c;
            if (!alive) return;
            unsigned long long dv = um_desc_x(um_s32(ring) + slot * S::SLOT, 8192, 1024, 2);
            unsigned dp = tm + S::COL_P + (j & 1) * (SA_KT / 2), more = (unsigned) (t - r.t0);
            int ks = 0;
#pragma unroll 1
            for (; ks + 4 <= steps; ks += 4, dv += HD / 128 * 8192 >> 4, dp += 32, more = 1u)   // a group of 64 positions
#pragma unroll
                for (int i = 0; i < 4; ++i) sa_mma_ts(tm, dp + i * 8, dv + (i * 2048 >> 4), idesc_o, more | (unsigned) i);
#pragma unroll 1
            for (; ks < steps; ++ks, dv += 2048 >> 4, dp += 8, more = 1u) sa_mma_ts(tm, dp, dv, idesc_o, more);
            sa_commit(&empty[slot]);
            sa_commit(&o_full[j & 1]);
        };
        for (bool more = work; more; more = r.next(a)) {
            if (!r.n) continue;
            const int end = r.t0 + r.n;
            if (um_elect()) {
                wait(q_ready, (unsigned) nseg & 1u);
                if (j) wait(s_free, (unsigned) (j - 1) & 1u);
                scores(r.n == 1);
                if (r.n > 1) {
                    wait(s_free, (unsigned) j & 1u);   // the first tile's scores are in registers
                    scores(r.n == 2);
                }
            }
            __syncwarp();
            for (int t = r.t0; t < end; ++t, ++j) {
                if (um_elect()) {
                    if (t + 2 < end) wait(s_free, (unsigned) (j + 1) & 1u);   // S(t + 1) is in registers, and so P(t) is written
                    wait(&p_full[j & 1], (unsigned) (j >> 1) & 1u);
                    if (t + 2 < end) scores(t + 3 == end);
                    if (t == r.t0 && nseg) wait(o_free, (unsigned) (nseg - 1) & 1u);   // the rows before are out of O
                    output(t);
                }
                __syncwarp();
            }
            ++nseg;
        }
        // nothing is under way when the blocks end, also after a wait that ran out: neither MMAs nor arrivals from the other CTA
        if (um_elect()) {
            sa_commit(idle);
            if (j && alive) sa_wait(s_free, (unsigned) (j - 1) & 1u, spins, a.fault), sa_wait(o_free, (unsigned) (nseg - 1) & 1u, spins, a.fault);
            spins = SA_SPINS;
            sa_wait(idle, 0u, spins, a.fault);
        }
        __syncwarp();
    }
    leave();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        // ---- softmax: row m, columns 64 half .. + 63 of every tile
        const int half = (warp - 4) >> 2, m = (warp & 3) * 32 + lane, token = m / qpk, hh = m % qpk;
        const unsigned tl = tm + ((unsigned) ((warp & 3) * 32) << 16);
        const float scale = 1.44269504f / sqrtf((float) HD);
        const int inv_qpk = (65536 + qpk - 1) / qpk;   // x / qpk = x inv_qpk >> 16 for x < 128
        unsigned char* strip = strips + (warp - 4) * SA_STRIP;
        int j = 0;   // tiles
        bool zeroed = false;
        SqRun r;
        r.get(run_at);
        auto agree = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(SA_SOFT) : "memory"); };   // the rows' halves
        auto wait = [&](unsigned long long* bar, unsigned parity) {
            if (um_elect()) sa_wait(bar, parity, spins, a.fault);
            __syncwarp();
            sa_after();
        };
        for (bool more = work; more; more = r.next(a)) {
            const SqUnit& u = r.u;
            const int tok0 = u.tok0 + rank * a.tok, first_row = u.r0 + tok0;   // this CTA's
            const bool real = token < a.tok && tok0 + token < u.len;
            // a warp without rows only keeps step, P zero and O what comes of it: they reach no other rows, and the tensor core takes less
            // power over zeros.  (Twelve single tokens: 115 us with all warps at work, 109 keeping step, 104 with P and Q zero; a prompt of
            // 8192 tokens 647 and 635, short ones 32.1 and 32.8)
            if (tok0 + ((warp & 3) * 32) / qpk >= u.len) {
                if (!zeroed) {   // (nothing reads P between two segments)
                    unsigned zero[32];
#pragma unroll
                    for (int k = 0; k < 32; ++k) zero[k] = 0u;
                    sa_st32(tl + S::COL_P + half * 32, zero), sa_st32(tl + S::COL_P + SA_KT / 2 + half * 32, zero);
                    sa_wait_st();
                    sa_before();
                    zeroed = true;
                }
                for (int i = 0; i < r.n; ++i, ++j) {
                    wait(s_full, (unsigned) j & 1u);   // (the scores were issued behind p_full of two tiles before: no phase is met twice)
                    if (lane == 0) sa_tell(s_free, first), sa_tell(&p_full[j & 1], first);
                    agree();
                }
                agree(); agree();
                if (r.n) wait(&o_full[(j - 1) & 1], (unsigned) ((j - 1) >> 1) & 1u);
                if (r.n && lane == 0) sa_tell(o_free, first);
                continue;
            }
            zeroed = false;
            if (a.qg && !r.cut && real)   // the gate will be wanted
                for (int i = half * (HD / 2); i < (half + 1) * (HD / 2); i += 32)
                    l2_ask(a.qg + ((size_t) (first_row + token) * a.nq + u.head * qpk + hh) * 2 * HD + HD + i);
            // positions this row sees: the causal count, or all, with a mask from pos0 on
            const int lim = !real ? 0 : a.anc ? u.kv_len : min(u.kv_len, u.pos0 + tok0 + token + 1);
            const int clear = min(u.kv_len, a.anc ? u.pos0 : u.pos0 + tok0 + 1);   // positions below are seen by every row
            const unsigned* anc = a.anc ? a.anc + (size_t) (real ? first_row + token : u.r0) * a.words : nullptr;
            float ref = -INFINITY, z = 0.f;   // this row's reference (in units of log2) and this half's sum
#pragma unroll 1
            for (int i = 0; i < r.n; ++i, ++j) {
                wait(s_full, (unsigned) j & 1u);
                float x[64];
                sa_ld32(reinterpret_cast<unsigned*>(x), tl + S::COL_S + half * 64);
                sa_ld32(reinterpret_cast<unsigned*>(x) + 32, tl + S::COL_S + half * 64 + 32);
                sa_wait_ld();
                sa_before();
                __syncwarp();
                if (lane == 0) sa_tell(s_free, first);
                const int p0 = (r.t0 + i) * SA_KT + half * 64;
                if (p0 + 64 > clear) {
                    unsigned see0 = sq_first(lim - p0), see1 = sq_first(lim - p0 - 32);
                    if (a.anc) see0 &= sq_tree_bits(anc, a.words, p0 - u.pos0), see1 &= sq_tree_bits(anc, a.words, p0 + 32 - u.pos0);
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        if (!(see0 >> k & 1u)) x[k] = -INFINITY;
                        if (!(see1 >> k & 1u)) x[32 + k] = -INFINITY;
                    }
                }
                float mq[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                for (int k = 4; k < 64; ++k) mq[k & 3] = sa_max(mq[k & 3], x[k]);
                float mx = sa_max(sa_max(mq[0], mq[1]), sa_max(mq[2], mq[3]));
                float* xm = xmax + (j & 1) * 2 * SA_ROWS;
                xm[half * SA_ROWS + m] = mx;
                agree();
                const float top = sa_max(mx, xm[(half ^ 1) * SA_ROWS + m]);
                mx = top * scale;
                if (!(mx < INFINITY)) z = NAN;   // a score that is no number, or infinite: so is the row
                const bool up = real && mx - ref > 8.0f;   // (other rows hold what was there before; nothing is -inf - -inf)
                if (__any_sync(0xffffffffu, up)) {
                    const float f = !up ? 1.0f : ref == -INFINITY ? 0.f : ex2_ftz(ref - mx);
                    if (up) ref = mx;
                    z *= f;
                    if (i > 0) {   // O row *= f, this half's columns
                        wait(&o_full[(j - 1) & 1], (unsigned) ((j - 1) >> 1) & 1u);
#pragma unroll 1
                        for (int cb = 0; cb < HD / 2; cb += 32) {
                            unsigned o[32];
                            sa_ld32(o, tl + half * (HD / 2) + cb);
                            sa_wait_ld();
#pragma unroll
                            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                            sa_st32(tl + half * (HD / 2) + cb, o);
                        }
                    }
                }
                float less = ref == -INFINITY ? 0.f : (float) SA_LIFT - ref;
                const bool far = fabsf(mx) > 4194304.f && fabsf(mx) < INFINITY;
                if (__any_sync(0xffffffffu, far)) {   // mx is off by more than a weight can be: the scores against their own maximum first
                    const float own = far ? top : 0.f;
#pragma unroll
                    for (int k = 0; k < 64; ++k) x[k] -= own;
                    if (far) less = mx - ref + (float) SA_LIFT;
                }
                const bool p_free = j < 2 || sa_test(&o_full[j & 1], (unsigned) ((j >> 1) - 1) & 1u);   // the P tile's last reader is done
                unsigned pk[32];
                float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                    float2 e = fma2(make_float2(x[2 * k], x[2 * k + 1]), make_float2(scale, scale), make_float2(less, less));
                    if (k * SA_POLY / 32 != (k + 1) * SA_POLY / 32) e = sa_ex2_poly(e);
                    else e.x = ex2_ftz(e.x), e.y = ex2_ftz(e.y);
                    sum = add2(sum, e);
                    const __half2 h = __floats2half2_rn(e.x, e.y);
                    pk[k] = *reinterpret_cast<const unsigned*>(&h);
                }
                z += sum.x + sum.y;
                if (!__all_sync(0xffffffffu, p_free)) wait(&o_full[j & 1], (unsigned) ((j >> 1) - 1) & 1u);
                else sa_after();
                sa_st32(tl + S::COL_P + (j & 1) * (SA_KT / 2) + half * 32, pk);
                sa_wait_st();
                sa_before();
                __syncwarp();
                if (lane == 0) sa_tell(&p_full[j & 1], first);
            }
            // ---- the rows' results: through the warp's strip, so that a line of 32 columns leaves (and its gates come) whole
            float* xm = xmax + (j & 1) * 2 * SA_ROWS;   // the last tile's are in the other half
            xm[half * SA_ROWS + m] = z;
            agree();
            z += xm[(half ^ 1) * SA_ROWS + m];
            agree();   // (a segment without tiles would write there again)
            if (z != z) ref = 0.f;
            const bool none = ref == -INFINITY;   // the row saw nothing
            const float inv = none ? 0.f : 1.0f / z;
            const size_t slot = (size_t) (2 * g + (r.first ? 0 : 1)) * 2 + rank;   // of the parts
            float4* part = a.part + ((slot * 4 + (warp & 3)) * (HD / 4) + half * (HD / 8)) * 32 + lane;
            if (r.cut && real && half == 0) a.mz[slot * SA_ROWS + m] = make_float2(ref, z);
            // lane l's part of row 4 k + l / 8 of this warp's: columns 4 (l % 8) .. + 3 of every 32; where those rows lie
            const int sub = lane >> 3, col = half * (HD / 2) + 4 * (lane & 7), rows = min(a.tok, u.len - tok0) * qpk - (warp & 3) * 32;   // rows of the warp that are real
            uint16_t* out = a.out + (size_t) first_row * a.out_stride + (size_t) u.head * qpk * HD + col;
            const float* gates = a.qg + ((size_t) first_row * a.nq + u.head * qpk) * 2 * HD + HD + col;
            int out_at[8], gate_at[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int mm = (warp & 3) * 32 + 4 * k + sub, t = mm * inv_qpk >> 16, h = mm - t * qpk;
                out_at[k] = 4 * k + sub < rows ? t * a.out_stride + h * HD : -1, gate_at[k] = (t * a.nq + h) * 2 * HD;
            }
            constexpr int STRIPS = HD / 64;   // of 32 columns, this half's
            float4 gate[8];
            const bool gated = !r.cut && a.qg;
            auto ask = [&](int k, int st) {   // a strip ahead
                if (gated && st < STRIPS && out_at[k] >= 0) gate[k] = *reinterpret_cast<const float4*>(gates + gate_at[k] + st * 32);
            };
#pragma unroll
            for (int k = 0; k < 8; ++k) ask(k, 0);
            if (r.n) wait(&o_full[(j - 1) & 1], (unsigned) ((j - 1) >> 1) & 1u);
#pragma unroll 1
            for (int st = 0; st < STRIPS; ++st) {
                unsigned o[32];
                if (r.n) {
                    sa_ld32(o, tl + half * (HD / 2) + st * 32);
                    sa_wait_ld();
                    if (st == STRIPS - 1) {   // O is in registers
                        sa_before();
                        __syncwarp();
                        if (lane == 0) sa_tell(o_free, first);
                    }
                }
                if (__any_sync(0xffffffffu, none || !r.n))   // rows that saw nothing
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] = none || !r.n ? 0u : o[k];
                if (r.cut) {
                    if (real)
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            part[(st * 8 + k) * 32] =
                                make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]), __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3]));
                    continue;
                }
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    *reinterpret_cast<float4*>(strip + lane * 128 + ((k ^ (lane & 7)) << 4)) =
                        make_float4(__uint_as_float(o[4 * k]) * inv, __uint_as_float(o[4 * k + 1]) * inv, __uint_as_float(o[4 * k + 2]) * inv,
                                    __uint_as_float(o[4 * k + 3]) * inv);
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int l = 4 * k + sub;
                    float4 y = *reinterpret_cast<const float4*>(strip + l * 128 + (((lane & 7) ^ (l & 7)) << 4));
                    if (gated) sa_gate(y.x, y.y, gate[k].x, gate[k].y), sa_gate(y.z, y.w, gate[k].z, gate[k].w);
                    ask(k, st + 1);
                    if (out_at[k] >= 0)
                        *reinterpret_cast<uint2*>(out + out_at[k] + st * 32) =
                            make_uint2(sq_pack(y.x, y.y), sq_pack(y.z, y.w));
                }
                __syncwarp();
            }
        }
        leave();
    }
}

// The parts of units that were cut, joined: where a pair's run ends, a block takes 32 rows of the unit that it cut, a warp eight of
// their columns, a lane a row, as the parts lie; PARTS parts' loads are in flight together.  FEW: fewer units than runs, and blocks
// for the units only, which look their run up (a tree of 16 after 3000 positions: 17.3 us with blocks for all runs and four parts in
// flight, 16.6 so, with eight; eight short prompts with more units than runs: 32.7 us, with this form's early gates 33.3).
constexpr int SJ_PAIRS = 128;
template <int HD, int PARTS, bool FEW> __global__ void __launch_bounds__(256, PARTS == 4 ? 3 : 2) k_attn_seqs_join(const __grid_constant__ SqAttn a) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = blockIdx.y >> 2, quarter = blockIdx.y & 3;   // CTA of the pair, quarter of its rows
    const int qpk = a.nq / a.nkv, m = quarter * 32 + lane, token = m / qpk, hh = m - token * qpk, c = warp + 8 * blockIdx.z;   // c: which eight columns
    pdl_wait();
    pdl_go();
    int g = blockIdx.x;
    int4 x = make_int4(0, 0, 0, 0);
    if constexpr (FEW) {   // the x-th that is cut
        int4 cut[SJ_PAIRS / 32];
        int which = g;
#pragma unroll
        for (int k = 0; k < SJ_PAIRS / 32; ++k) cut[k] = k * 32 + lane < a.pairs ? a.cuts[2 * (k * 32 + lane)] : make_int4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < SJ_PAIRS / 32; ++k) {
            const unsigned some = __ballot_sync(0xffffffffu, cut[k].x != 0);
            const unsigned it = __ballot_sync(0xffffffffu, cut[k].x != 0 && __popc(some & ((1u << lane) - 1u)) == which);
            if (it) {
                const int l = __ffs(it) - 1;
                g = k * 32 + l;
                x = make_int4(__shfl_sync(0xffffffffu, cut[k].x, l), __shfl_sync(0xffffffffu, cut[k].y, l), __shfl_sync(0xffffffffu, cut[k].z, l),
                              __shfl_sync(0xffffffffu, cut[k].w, l));
            }
            which -= __popc(some);
        }
    } else {
        x = a.cuts[2 * g];
    }
    const int n = x.x;
    if (!n || m >= min(a.tok, x.w - rank * a.tok) * qpk) return;
    const int head = a.cuts[2 * g + 1].x * qpk + hh;
    const size_t row = (size_t) x.z + rank * a.tok + token;
    const float4* gates = reinterpret_cast<const float4*>(a.qg + (row * a.nq + head) * 2 * HD + HD + c * 8);
    float4 gate[2];
    if (!FEW && a.qg) l2_ask(reinterpret_cast<const float*>(gates));
    auto slot = [&](int p) { return (p ? 2 * (g + p) : x.y) * 2 + rank; };
    const float4* part = a.part + (quarter * (HD / 4) + c * 2) * 32 + lane;
    float top = -INFINITY, z = 0.f, acc[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k] = 0.f;
#pragma unroll 1
    for (int p0 = 0; p0 < n; p0 += PARTS) {
        float2 q[PARTS];
        float4 v[PARTS][2];
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            q[i] = make_float2(-INFINITY, 0.f), v[i][0] = v[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (p0 + i >= n) continue;
            const int at = slot(p0 + i);
            q[i] = a.mz[at * SA_ROWS + m];
            v[i][0] = part[at * (SA_ROWS * HD / 4)], v[i][1] = part[at * (SA_ROWS * HD / 4) + 32];
        }
        if (FEW && !p0 && a.qg) gate[0] = gates[0], gate[1] = gates[1];   // behind the first parts' loads
        float most = top;
#pragma unroll
        for (int i = 0; i < PARTS; ++i) most = fmaxf(most, q[i].x);
        if (most == -INFINITY) continue;   // the row sees nothing there
        const float f0 = top == -INFINITY ? 0.f : ex2_ftz(top - most);
        top = most, z *= f0;
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] *= f0;
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            const float f = q[i].x == -INFINITY ? 0.f : ex2_ftz(q[i].x - top);
            z = fmaf(f, q[i].y, z);
            acc[0] = fmaf(f, v[i][0].x, acc[0]), acc[1] = fmaf(f, v[i][0].y, acc[1]), acc[2] = fmaf(f, v[i][0].z, acc[2]), acc[3] = fmaf(f, v[i][0].w, acc[3]);
            acc[4] = fmaf(f, v[i][1].x, acc[4]), acc[5] = fmaf(f, v[i][1].y, acc[5]), acc[6] = fmaf(f, v[i][1].z, acc[6]), acc[7] = fmaf(f, v[i][1].w, acc[7]);
        }
    }
    const float inv = z == 0.f ? 0.f : 1.0f / z;
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k] *= inv;
    if (!FEW && a.qg) gate[0] = gates[0], gate[1] = gates[1];
    if (a.qg)
        sa_gate(acc[0], acc[1], gate[0].x, gate[0].y), sa_gate(acc[2], acc[3], gate[0].z, gate[0].w), sa_gate(acc[4], acc[5], gate[1].x, gate[1].y),
            sa_gate(acc[6], acc[7], gate[1].z, gate[1].w);
    *reinterpret_cast<uint4*>(a.out + row * a.out_stride + (size_t) head * HD + c * 8) =
        make_uint4(sq_pack(acc[0], acc[1]), sq_pack(acc[2], acc[3]), sq_pack(acc[4], acc[5]), sq_pack(acc[6], acc[7]));
}

static long long sq_units(const FnxSeqs* sq, int tok, int nkv) {   // at most
    const long long blocks = (long long) sq->rows / (2 * tok) + sq->nseq;
    return (blocks < sq->rows ? blocks : (long long) sq->rows) * nkv;
}
static int sq_processors() {   // multiprocessors of the current device
    static int n[64] = {};   // written without a lock: every writer stores the same value
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if (!n[dev] && cudaDeviceGetAttribute(&n[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) n[dev] = 148;
    return n[dev];
}

template <int HD> static int sq_launch(const SqMaps& maps, const SqAttn& a, long long units, const char* what, cudaStream_t st) {
    if (cudaFuncSetAttribute(k_attn_seqs<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) SaShape<HD>::SMEM) != cudaSuccess)
        return fail("%s: shared memory opt-in: %s", what, cudaGetErrorString(cudaGetLastError()));
    launch(0, k_attn_seqs<HD>, dim3(2 * a.pairs), SA_THREADS, SaShape<HD>::SMEM, st, maps, a);
    if (launch_ok(what)) return 1;
    if (a.pairs == 1) return 0;
    const int qpk = a.nq / a.nkv, most = std::min(a.sq.rows, 2 * a.tok);   // tokens of a unit
    const int quarters = most > a.tok ? 4 + ((most - a.tok) * qpk + 31) / 32 : (most * qpk + 31) / 32;
    const dim3 grid((unsigned) std::min<long long>(a.pairs - 1, units), quarters, HD / 64);
    if ((int) grid.x == a.pairs - 1) launch(0, k_attn_seqs_join<HD, 4, false>, grid, 256, 0, st, a);
    else if (grid.x * grid.y * grid.z > (unsigned) sq_processors()) launch(0, k_attn_seqs_join<HD, 4, true>, grid, 256, 0, st, a);
    else launch(0, k_attn_seqs_join<HD, 8, true>, grid, 256, 0, st, a);   // few blocks, with many parts each
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
    // (a CTA's up to 128 rows have 32-bit offsets from its first)
    FNX_REQUIRE(out_stride <= 1 << 24, "%s: output rows %d halves apart (2^24 at most)", what, out_stride);
    FNX_REQUIRE(!sq->pt || g.rows % 8 == 0, "%s: pages of %d rows (a multiple of 8)", what, g.rows);
    const int qpk = nq / nkv, tok = SA_ROWS / qpk;
    int box = 64, lg = 6;
    while (sq->pt && g.rows % box) box /= 2, --lg;
    unsigned* fault = device_fault_word();
    UmEncode enc = um_encoder();
    FNX_REQUIRE(fault && enc, "%s: no fault word or no tensor-map encoder", what);
    SqMaps maps;
    memset(&maps, 0, sizeof(maps));
    const cuuint32_t es[4] = {1, 1, 1, 1};
    // queries: dims, heads, rows.  The cache: 64 dims, rows of a page, column blocks, pages
    const cuuint64_t qd[3] = {(cuuint64_t) hd, (cuuint64_t) nq, (cuuint64_t) sq->rows}, qs[2] = {(cuuint64_t) hd * 2, (cuuint64_t) q_stride * 2};
    const cuuint32_t qb[3] = {64, (cuuint32_t) qpk, (cuuint32_t) tok};
    const cuuint64_t row = (cuuint64_t) nkv * hd, rows = sq->pt ? g.rows : g.cap;
    const cuuint64_t kd[4] = {64, rows, row / 64, (cuuint64_t) (sq->pt ? sq->npages : 1)}, ks[3] = {row * 2, 128, sq->pt ? (cuuint64_t) g.page * 2 : rows * row * 2};
    const cuuint32_t kb[4] = {64, (cuuint32_t) box, (cuuint32_t) (box == 64 ? hd / 64 : 1), 1}, vb[4] = {64, (cuuint32_t) box, (cuuint32_t) (box == 64 ? hd / 128 : 1), 1};
    auto encode = [&](CUtensorMap* m, int n, const void* p, const cuuint64_t* d, const cuuint64_t* s, const cuuint32_t* b) {
        return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, n, const_cast<void*>(p), d, s, b, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    };
    FNX_REQUIRE(encode(&maps.q, 3, q16, qd, qs, qb) && encode(&maps.k, 4, kc, kd, ks, kb) && encode(&maps.v, 4, vc, kd, ks, vb),
                "%s: no tensor map for %d rows %d apart or %d pages of %zu halves", what, sq->rows, q_stride, sq->npages, g.page);
    // no more pairs than there can be work for
    const long long units = sq_units(sq, tok, nkv);   // (2^20 of them are more than enough)
    const long long most = sq->max_pos ? std::min(units, 1ll << 20) * ((long long) sq->max_pos + SA_COST) : 1ll << 60;
    const int pairs = (int) std::max(1ll, std::min((long long) std::min(sq_processors() / 2, SJ_PAIRS), (most + SA_LEAST - 1) / SA_LEAST));
    float4* part = (float4*) scratch;
    float2* mz = reinterpret_cast<float2*>(part + (size_t) 4 * pairs * SA_ROWS * (hd / 4));
    const SqAttn a{qg, g, *sq, anc, out, out_stride, nq, nkv, words, tok, box, lg, pairs, part, mz, reinterpret_cast<int4*>(mz + (size_t) 4 * pairs * SA_ROWS), fault};
    return hd == 256 ? sq_launch<256>(maps, a, units, what, strm(st)) : sq_launch<128>(maps, a, units, what, strm(st));
}

}  // namespace fnxk

using namespace fnxk;

extern "C" {

size_t fnx_attn_seqs_scratch_bytes(const FnxSeqs* sq, int nq, int nkv, int hd) {
    if (!sq || nq < 1 || nkv < 1 || hd < 1) return 0;
    const size_t pairs = (size_t) std::max(1, std::min(sq_processors() / 2, SJ_PAIRS));
    return pairs * (4 * SA_ROWS * (hd + 2) * 4 + 2 * sizeof(int4));
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
