// Log probabilities of given tokens, the entropy of their distribution and the likeliest alternatives, in one pass over the
// logits (no counterpart in the reference, which returns tokens only).
//
// With t = (x - R) log2 e for a reference R, z = sum 2^t and s = sum t 2^t:  lse = R + ln z,  H = (log2 z - s / z) ln 2, and a
// token's log probability is x - lse.  R is one of the logits, so it is exact and finite where they are, and x - R is rounded once
// (R log2 e would leave the type from 2.4e38 on).  The reference is raised - z' = f z, s' = f (s + d z), d = (R - R') log2 e, f = 2^d -
// only when a value exceeds it by more than 5.5, so a thread rescales once or twice a row and 2^t stays below 2^8.  The centred s keeps H free of the cancellation
// that sum p x - lse has for large logits.  A NaN or +inf makes z a NaN, which is how the row is found out.
// The k best: a bound that k values of the row's first batch reach or exceed (the k-th largest of the maxima of groups of
// threads), made anew from the lists some batches on, and of the rest of the row every warp lists what exceeds it, a few hundredths of a
// percent of the values, without a word to the other warps.  A list that is full (rising logits) is cut to its own k best, which
// raises that warp's bound.  In the end a bound over the lists' entries leaves little more than k, and an entry's place is the number
// of larger ones.  Entries are 64-bit composites (the value's order-preserving key, the index's complement), no two equal, so ties go
// to the lower index whatever order they come in.
// A row goes to one block when there are many, else to as many as the GPU holds at once; the row's last block joins the parts.
// A pass is bound by DRAM when there are many rows: a thread copies its own values into shared memory three batches ahead
// (cp.async; nobody else reads them, so no barrier belongs to it), 72 KB in flight a multiprocessor.  2000 rows of 151 936 logits with
// five alternatives: 216 us (5.6 TB/s); with one batch ahead in registers 342.  16 rows with twenty: 12.2 us, latency - a bound, the
// lists through memory to the row's last block, a bound and the choice there.
#include <algorithm>

#include "common.cuh"
#include "exact_math.cuh"
#include "moe_internal.cuh"

namespace fnxk {

constexpr int LP_THREADS = 384, LP_WARPS = LP_THREADS / 32, LP_PER = 8, LP_BATCH = LP_THREADS * LP_PER, LP_LIST = 256;
constexpr int LP_CAP = LP_WARPS * LP_LIST;   // entries of all lists
constexpr int LP_STAGES = 4;            // batches in the ring
constexpr int LP_TIGHTEN = 6;           // batches after which the bound is made anew
constexpr int LP_BLOCKS = 2 * 148;   // blocks the GPU holds at once; rows that go to several blocks are fewer

struct LpPart {   // the sums over a block's part of a row
    float r, z, s, pad;
};
struct LpArgs {
    const float* logits;
    size_t stride;
    int rows, n, v0, k, ntok, nsplit;
    int per;    // positions a part of a row, whole batches
    int ship;   // entries that a block leaves for the row's last block, k at least
    const int* tok;
    float *lse, *ent, *lp, *top_lp;
    int* top_i;
    unsigned* count;             // [T] blocks of the row that are done (left at zero)
    LpPart* part;                // [T][nsplit]
    unsigned long long* cand;    // [T][nsplit][ship], zero where there are fewer
    unsigned* err;
};

__device__ __forceinline__ unsigned long long lp_composite(float v, unsigned idx) {
    return ((unsigned long long) fkey(fadd(v, 0.f)) << 32) | (0xffffffffu - idx);
}

constexpr float LP_L2E = 1.44269504f;
// (r, z, s) of two parts of a row together
__device__ __forceinline__ void lp_join(float& r, float& z, float& s, float r2, float z2, float s2) {
    const float rn = fmaxf(r, r2);
    if (rn == -INFINITY) {   // nothing on either side, but for a NaN
        z += z2, s += s2;
        return;
    }
    const float d1 = fmaxf((r - rn) * LP_L2E, -200.f), d2 = fmaxf((r2 - rn) * LP_L2E, -200.f);   // 2^-200 is zero: a part of nothing (-inf) drops out
    const float f1 = ex2_ftz(d1), f2 = ex2_ftz(d2);
    s = f1 * (s + d1 * z) + f2 * (s2 + d2 * z2);
    z = f1 * z + f2 * z2;
    r = rn;
}

// the same of a warp's 32 parts: one reference for all, then plain sums
__device__ __forceinline__ void lp_join_warp(float& r, float& z, float& s) {
    const float top = fkey_inv(__reduce_max_sync(0xffffffffu, fkey(r)));
    const float d = r == top ? 0.f : fmaxf((r - top) * LP_L2E, -200.f), f = ex2_ftz(d);
    s = f * (s + d * z), z *= f, r = top;
#pragma unroll
    for (int o = 16; o; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o), s += __shfl_xor_sync(0xffffffffu, s, o);
}

// Bisection by a warp: a bound b that between k and k + slack of the entries reach or exceed (a lane has N; 0: no entry), or 0
// when there are fewer than k.  Entries are distinct, so it ends after at most 64 steps.
template <int N> __device__ __forceinline__ unsigned long long lp_bound(const unsigned long long (&e)[N], int k, int slack) {
    unsigned long long most = 0ull;
    int have = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        most = e[i] > most ? e[i] : most;
        have += e[i] != 0ull;
    }
    if ((int) __reduce_add_sync(0xffffffffu, (unsigned) have) < k) return 0ull;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const unsigned long long x = __shfl_xor_sync(0xffffffffu, most, o);
        most = x > most ? x : most;
    }
    unsigned long long lo = 1ull, hi = most;   // at least k reach lo; the answer is not above hi
    // the k-th best is seldom far below the best: the first guess is half of it
    unsigned long long mid = hi > (24ull << 55) ? hi - (1ull << 55) : lo + (hi - lo) / 2;
    while (lo < hi) {
        unsigned c = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) c += e[i] >= mid;
        c = __reduce_add_sync(0xffffffffu, c);
        if ((int) c >= k) {
            lo = mid;
            if ((int) c <= k + slack) break;
        } else {
            hi = mid - 1ull;
        }
        mid = lo + (hi - lo + 1ull) / 2;
    }
    return lo;
}

struct LpShared {
    unsigned long long list[LP_WARPS][LP_LIST];
    alignas(16) unsigned long long best[LP_THREADS >> 2];   // groups' maxima
    float r[LP_WARPS], z[LP_WARPS], s[LP_WARPS];
    int cnt[LP_WARPS];
    unsigned long long bound;
    unsigned n, last;
    float ref;
    double lz;   // lse = ref + lz; a NaN, or ref -inf: the row has no distribution
};

// A bound that at least k of the threads' entries reach (0 where there are too few): the k-th largest of the maxima of groups of
// threads, 12 groups, 48 or 96.  Their ranks are counted, which has no steps that wait for one another: a bisection over all
// threads' maxima took 1 us longer.
__device__ __forceinline__ unsigned long long lp_block_bound(LpShared& sh, unsigned long long mine, int k) {
    const int tid = threadIdx.x, shift = k <= LP_WARPS ? 5 : k <= 40 ? 3 : 2, groups = LP_THREADS >> shift;
    for (int o = 1; o < 1 << shift; o <<= 1) {
        const unsigned long long x = __shfl_xor_sync(0xffffffffu, mine, o);
        mine = x > mine ? x : mine;
    }
    if (!(tid & ((1 << shift) - 1))) sh.best[tid >> shift] = mine;
    __syncthreads();
    if (tid < groups) {
        const unsigned long long own = sh.best[tid];
        int above = 0;
#pragma unroll 4
        for (int i = 0; i < groups; i += 2) {
            const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(&sh.best[i]);
            above += x.x > own, above += x.y > own;
        }
        if (above == k - 1 || (!own && above < k)) sh.bound = own;   // (entries are distinct, but for the zeros)
    }
    __syncthreads();
    return sh.bound;
}

// The k best of the threads' entries (N each, 0: none), in order, at place 0 .. k - 1 of `place`; at least k entries exist.
template <int N, typename F> __device__ __forceinline__ void lp_best(LpShared& sh, const unsigned long long (&e)[N], int k, F place) {
    const int tid = threadIdx.x;
    unsigned long long most = 0ull;
#pragma unroll
    for (int i = 0; i < N; ++i) most = e[i] > most ? e[i] : most;
    if (tid == 0) sh.n = 0u;
    const unsigned long long b = lp_block_bound(sh, most, k);
    unsigned long long* all = &sh.list[0][0];   // (the lists are in registers)
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (e[i] && e[i] >= b) all[atomicAdd(&sh.n, 1u)] = e[i];
    __syncthreads();
    const unsigned n = min(sh.n, (unsigned) LP_CAP);
    for (unsigned i = tid; i < n; i += LP_THREADS) {
        const unsigned long long c = all[i];
        int at = 0;
        for (unsigned j = 0; j < n; ++j) at += all[j] > c;
        if (at < k) place(at, c);
    }
}

struct LpItem {   // a block's part of a row
    const float* base;   // positions are counted from the 16-byte boundary at or before the row's first logit
    int row, split, shift, lo, hi;
};
__device__ __forceinline__ LpItem lp_item(const LpArgs& a, int row, int split) {
    LpItem t;
    t.row = row, t.split = split;
    const float* x = a.logits + (size_t) row * a.stride;
    t.shift = (int) (((uintptr_t) x >> 2) & 3u), t.base = x - t.shift;
    const long long end = a.n + t.shift, lo = (long long) split * a.per;
    t.lo = (int) min(lo, end), t.hi = (int) min(lo + a.per, end);
    return t;
}

__global__ void __launch_bounds__(LP_THREADS, 2) k_logprobs(const LpArgs a) {
    __shared__ LpShared sh;
    extern __shared__ __align__(16) unsigned char lp_ring[];   // [LP_STAGES][2][LP_THREADS] runs of four
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned long long* list = sh.list[warp];
    const unsigned ring = (unsigned) __cvta_generic_to_shared(lp_ring) + tid * 16;   // this thread's slots, a stage's two LP_THREADS * 16 bytes apart
    constexpr unsigned RUN = LP_THREADS * 16;
    auto load = [&](const LpItem& t, int i0, unsigned slot) {   // a thread has two runs of four a batch
        if (i0 >= t.lo + 4 && i0 + LP_BATCH <= t.hi) {   // whole runs all
            const float* src = t.base + i0 + tid * 4;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot), "l"(src) : "memory");
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot + RUN), "l"(src + LP_BATCH / 2) : "memory");
        } else if (i0 < t.hi) {
#pragma unroll 1
            for (int g = 0; g < 2; ++g) {
                const int p = i0 + g * (LP_BATCH / 2) + tid * 4;
                if (p >= t.shift && p + 4 <= t.hi) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot + g * RUN), "l"(t.base + p) : "memory");
                } else {
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = p + e >= t.shift && p + e < t.hi ? t.base[p + e] : -INFINITY;
                    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(slot + g * RUN), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]) : "memory");
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto slot = [&](int stage) { return ring + (unsigned) stage * (2 * RUN); };
    auto index = [&](int i0, int j) { return i0 + (j >> 2) * (LP_BATCH / 2) + tid * 4 + (j & 3); };
    pdl_wait();
    pdl_go();
    const bool parts_of_rows = a.nsplit > 1;   // a block a part; else a block every gridDim.x-th row
    const unsigned step = parts_of_rows ? (unsigned) a.rows : gridDim.x;
    LpItem next = lp_item(a, parts_of_rows ? blockIdx.y : blockIdx.x, parts_of_rows ? blockIdx.x : 0);
    int stage = 0;
#pragma unroll
    for (int i = 0; i < LP_STAGES - 1; ++i) load(next, next.lo + i * LP_BATCH, slot(i));
    for (unsigned row = (unsigned) next.row; row < (unsigned) a.rows; row += step) {
        const LpItem t = next;
        float r = -INFINITY, bound_v = -INFINITY;                        // r: the reference
        float2 z2 = make_float2(0.f, 0.f), s2 = make_float2(0.f, 0.f);   // the sums of the even and the odd values
        unsigned long long bound = 0ull;                                 // an entry has to be above it
        int cnt = 0;                                                     // this warp's list
        for (int i0 = t.lo; i0 < t.hi; i0 += LP_BATCH) {
            asm volatile("cp.async.wait_group %0;" ::"n"(LP_STAGES - 2) : "memory");
            float v[LP_PER];
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(slot(stage)) : "memory");
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]) : "r"(slot(stage) + RUN) : "memory");
            load(t, i0 + (LP_STAGES - 1) * LP_BATCH, slot((stage + LP_STAGES - 1) % LP_STAGES));
            stage = (stage + 1) % LP_STAGES;
            float mx = v[0];
#pragma unroll
            for (int j = 1; j < LP_PER; ++j) mx = fmaxf(mx, v[j]);
            if (mx > r + 5.5f || (r == -INFINITY && mx > -INFINITY)) {
                const float d = fmaxf((r - mx) * LP_L2E, -200.f), f = ex2_ftz(d);
                s2.x = f * (s2.x + d * z2.x), s2.y = f * (s2.y + d * z2.y);
                z2.x *= f, z2.y *= f;
                r = mx;
            }
            const float less = r == -INFINITY ? 0.f : -r;
#pragma unroll
            for (int j = 0; j < LP_PER; j += 2) {
                float2 q = mul2(add2(make_float2(v[j], v[j + 1]), make_float2(less, less)), make_float2(LP_L2E, LP_L2E));
                const float2 e = make_float2(ex2_ftz(q.x), ex2_ftz(q.y));
                q.x = fmaxf(q.x, -200.f), q.y = fmaxf(q.y, -200.f);
                z2 = add2(z2, e);
                s2 = fma2(e, q, s2);
            }
            if (!a.k) continue;
            if (i0 == t.lo) {
                unsigned long long most = 0ull;
#pragma unroll
                for (int j = 0; j < LP_PER; ++j) {
                    const int p = index(i0, j);
                    const unsigned long long c = p >= t.shift && p < t.hi && v[j] == v[j] ? lp_composite(v[j], (unsigned) (p - t.shift)) : 0ull;
                    most = c > most ? c : most;
                }
                bound = lp_block_bound(sh, most, a.k);
                bound_v = bound ? fkey_inv((unsigned) (bound >> 32)) : -INFINITY;
                bound -= bound != 0ull;   // the bound itself may enter
            }
            // some way on, the bound of everything so far: fewer values pass it from there on
            if (i0 == t.lo + LP_TIGHTEN * LP_BATCH) {
                unsigned long long most = 0ull;
                __syncwarp();
                for (int i = lane; i < cnt; i += 32) most = list[i] > most ? list[i] : most;
                const unsigned long long b = lp_block_bound(sh, most, a.k);
                if (b > bound + 1ull) bound = b - 1ull, bound_v = fkey_inv((unsigned) (b >> 32));
            }
            if (!__any_sync(0xffffffffu, mx >= bound_v)) continue;
            unsigned any = 0u;
#pragma unroll
            for (int j = 0; j < LP_PER; ++j) any |= v[j] >= bound_v ? 1u << j : 0u;
            any = __reduce_or_sync(0xffffffffu, any);
#pragma unroll
            for (int j = 0; j < LP_PER; ++j) {
                if (!(any >> j & 1u)) continue;
                const int p = index(i0, j);
                bool in = v[j] >= bound_v && p >= t.shift && p < t.hi;
                if (cnt + 32 > LP_LIST) {   // full: its best k stay
                    unsigned long long e[LP_LIST / 32];
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < LP_LIST / 32; ++i) e[i] = i * 32 + lane < cnt ? list[i * 32 + lane] : 0ull;
                    const unsigned long long b = lp_bound(e, a.k, 0);
                    __syncwarp();
                    cnt = 0;
#pragma unroll
                    for (int i = 0; i < LP_LIST / 32; ++i) {
                        const bool keep = e[i] >= b;
                        const unsigned kept = __ballot_sync(0xffffffffu, keep);
                        if (keep) list[cnt + __popc(kept & ((1u << lane) - 1u))] = e[i];
                        cnt += __popc(kept);
                    }
                    bound = b, bound_v = fkey_inv((unsigned) (b >> 32));
                }
                const unsigned long long c = lp_composite(v[j], (unsigned) (p - t.shift));
                in = in && c > bound;
                const unsigned who = __ballot_sync(0xffffffffu, in);
                if (in) list[cnt + __popc(who & ((1u << lane) - 1u))] = c;
                cnt += __popc(who);
            }
        }
        if (row + step < (unsigned) a.rows) {   // the next row's first batches are on their way while this one is finished
            next = lp_item(a, (int) (row + step), 0);
#pragma unroll
            for (int i = 0; i < LP_STAGES - 1; ++i) load(next, next.lo + i * LP_BATCH, slot((stage + i) % LP_STAGES));
        }
        // ---- the block's statistics
        float z = z2.x + z2.y, s = s2.x + s2.y;
        lp_join_warp(r, z, s);
        if (lane == 0) sh.r[warp] = r, sh.z[warp] = z, sh.s[warp] = s, sh.cnt[warp] = cnt;
        unsigned long long e[LP_LIST / 32];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < LP_LIST / 32; ++i) e[i] = i * 32 + lane < cnt ? list[i * 32 + lane] : 0ull;
        __syncthreads();
        LpPart* parts = a.part + (size_t) t.row * a.nsplit;
        unsigned long long* cands = a.cand + (size_t) t.row * a.nsplit * a.ship;
        if (warp == 0) {
            r = lane < LP_WARPS ? sh.r[lane] : -INFINITY, z = lane < LP_WARPS ? sh.z[lane] : 0.f, s = lane < LP_WARPS ? sh.s[lane] : 0.f;
            lp_join_warp(r, z, s);
        }
        bool mine = true;   // whether the row's results are this block's to write
        if (a.nsplit > 1) {   // the row's last block joins the parts
            if (tid == 0) parts[t.split] = LpPart{r, z, s, 0.f};
            if (a.k) {
                unsigned long long* mine_at = cands + (size_t) t.split * a.ship;
                const int held = lane < LP_WARPS ? sh.cnt[lane] : 0;
                const int before = (int) __reduce_add_sync(0xffffffffu, (unsigned) (lane < warp ? held : 0)), total = (int) __reduce_add_sync(0xffffffffu, (unsigned) held);
                const bool all = total <= a.ship;   // the lists as they are; else the k best
                for (int i = tid + (all ? total : 0); i < a.ship; i += LP_THREADS) mine_at[i] = 0ull;
                if (all) {
                    for (int i = lane; i < cnt; i += 32) mine_at[before + i] = list[i];
                } else {
                    __syncthreads();
                    lp_best(sh, e, a.k, [&](int place, unsigned long long c) { mine_at[place] = c; });
                }
            }
            __threadfence();
            __syncthreads();
            if (tid == 0) sh.last = atomicAdd(&a.count[t.row], 1u) == (unsigned) a.nsplit - 1u;
            __syncthreads();
            mine = sh.last != 0u;
            if (mine) {
                __threadfence();
                if (warp == 0) {
                    r = -INFINITY, z = 0.f, s = 0.f;
                    for (int i = lane; i < a.nsplit; i += 32) {
                        const LpPart p = parts[i];
                        lp_join(r, z, s, p.r, p.z, p.s);
                    }
                    lp_join_warp(r, z, s);
                }
#pragma unroll
                for (int i = 0; i < LP_LIST / 32; ++i) e[i] = i * LP_THREADS + tid < a.nsplit * a.ship ? cands[i * LP_THREADS + tid] : 0ull;
                if (tid == 0) a.count[t.row] = 0u;
            }
        }
        if (mine) {
            if (tid == 0) {
                const bool bad = z != z, none = r == -INFINITY && !bad;
                if (bad || none) atomicOr(a.err, 16u);
                const double ln2 = 0.6931471805599453, lz = log2((double) z);
                sh.ref = r, sh.lz = bad ? NAN : lz * ln2;
                a.lse[t.row] = bad ? NAN : none ? -INFINITY : (float) ((double) r + lz * ln2);
                if (a.ent) a.ent[t.row] = bad ? NAN : none ? 0.f : fmaxf((float) ((lz - (double) s / z) * ln2), 0.f);
            }
            __syncthreads();
            const double ref = sh.ref, lz = sh.lz;
            const bool bad = lz != lz, none = ref == -INFINITY;
            auto log_p = [&](float x) { return none ? -INFINITY : (float) fmin((double) x - ref - lz, 0.0); };   // rounded once
            for (int j = tid; j < a.ntok; j += LP_THREADS) {
                const long long i = (long long) a.tok[(size_t) t.row * a.ntok + j] - a.v0;
                const bool in = i >= 0 && i < a.n;
                a.lp[(size_t) t.row * a.ntok + j] = !in ? -INFINITY : bad ? NAN : log_p(t.base[t.shift + i]);
            }
            if (a.k && bad) {   // no order to speak of
                for (int j = tid; j < a.k; j += LP_THREADS) a.top_i[(size_t) t.row * a.k + j] = -1, a.top_lp[(size_t) t.row * a.k + j] = NAN;
            } else if (a.k) {
                lp_best(sh, e, a.k, [&](int place, unsigned long long c) {
                    a.top_i[(size_t) t.row * a.k + place] = a.v0 + (int) (0xffffffffu - (unsigned) (c & 0xffffffffu));
                    a.top_lp[(size_t) t.row * a.k + place] = log_p(fkey_inv((unsigned) (c >> 32)));
                });
            }
        }
        __syncthreads();   // the lists are the next row's
    }
}

// blocks a row: as many as the GPU holds at once, each with a batch of the row at least; their k best have room in one block
static int lp_splits(int n, int T, int k, int* each = nullptr) {
    const int batches = (n + 3 + LP_BATCH - 1) / LP_BATCH, want = std::max(1, LP_BLOCKS / T);   // n + 3: a row may begin inside a 16-byte run
    const int s = std::max(1, std::min(want, std::min(batches, std::min(64, LP_CAP / std::max(k, 1)))));
    const int per = (batches + s - 1) / s;
    if (each) *each = per * LP_BATCH;
    return (batches + per - 1) / per;   // no empty block
}
// entries that a block of a row in several parts leaves for the last one: its lists as they are where they have room, which spares
// choosing the best twice (16 rows, 20 alternatives: 13.8 us with k each, 12.2 so)
static int lp_ship(int ns, int k) { return k ? std::max(k, std::min(128, LP_CAP / ns)) : 0; }

}  // namespace fnxk

using namespace fnxk;

extern "C" {

size_t fnx_logprobs_scratch_bytes(int n, int T, int k) {
    if (n < 1 || T < 1 || k < 0 || k > FNX_TOPK_N) return 0;
    const size_t s = (size_t) lp_splits(n, T, k);
    return s == 1 ? 16 : (size_t) LP_BLOCKS * 4 + (size_t) T * s * (sizeof(LpPart) + 8 * (size_t) lp_ship((int) s, k));
}

int fnx_logprobs(const float* logits, size_t stride, int n, int T, int v0, const int* tok, int ntok, int k, float* lse, float* entropy, float* lp,
                 float* top_lp, int* top_i, void* scratch, unsigned* err, void* st) {
    FNX_REQUIRE(n >= 1 && T >= 1 && stride >= (size_t) n && v0 >= 0, "logprobs: %d rows of %d logits, %zu apart, from token %d", T, n, stride, v0);
    FNX_REQUIRE(k >= 0 && k <= FNX_TOPK_N && k <= n, "logprobs: %d alternatives of %d (at most %d)", k, n, FNX_TOPK_N);
    FNX_REQUIRE(n <= (1 << 30) && v0 <= (1 << 30), "logprobs: tokens %d .. %d + %d", v0, v0, n);
    FNX_REQUIRE(ntok >= 0 && (!ntok || (tok && lp)), "logprobs: %d given tokens without their buffers", ntok);
    FNX_REQUIRE(logits && lse && scratch && err && (!k || (top_lp && top_i)), "logprobs: a null buffer");
    FNX_REQUIRE((uintptr_t) scratch % 16 == 0, "logprobs: scratch not 16-byte aligned");
    int per;
    const int ns = lp_splits(n, T, k, &per);
    LpArgs a{logits, stride, T, n, v0, k, ntok, ns, per, lp_ship(ns, k), tok, lse, entropy, lp, top_lp, top_i, (unsigned*) scratch, nullptr, nullptr, err};
    // the counters have their place whatever the call's sizes, so that one scratch serves calls of different ones
    a.part = reinterpret_cast<LpPart*>((char*) scratch + LP_BLOCKS * 4);
    a.cand = reinterpret_cast<unsigned long long*>(a.part + (size_t) T * ns);
    constexpr size_t ring = (size_t) LP_STAGES * LP_BATCH * 4;
    if (smem_optin(k_logprobs, ring, "logprobs")) return 1;
    launch(0, k_logprobs, ns > 1 ? dim3(ns, T) : dim3(std::min(T, LP_BLOCKS)), LP_THREADS, ring, strm(st), a);
    return launch_ok("logprobs");
}
}
