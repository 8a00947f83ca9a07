// Log probabilities of given tokens, the entropy of their distribution and the likeliest alternatives, in one pass over the
// logits (no counterpart in the reference, which returns tokens only).
//
// With m the row's maximum, z = sum e^(x - m) and s = sum (x - m) e^(x - m):  lse = m + log z,  H = log z - s / z, and a
// token's log probability is x - lse.  (m, z, s) are kept while the row streams by: a batch whose maximum exceeds m rescales
// z' = f z, s' = f (s + (m - m') z), f = e^(m - m').  The centred s keeps H free of the cancellation that sum p x - lse has
// for large logits.
// The k best are kept beside it: a block holds a list of candidates and a bound, the k-th best so far; of a batch only what
// exceeds the bound enters, and when the list is full it is sorted and cut to k, which raises the bound.  The first bound
// costs one batch: it is cut into groups, every group's maximum is an element, so the smallest maximum of at least k groups
// has k elements at or above it.  Entries are 64-bit composites (the value's order-preserving key, the index's complement), no two
// equal, so ties go to the lower index whatever order the entries come in.
// A row goes to one block when there are many, else to as many as fill the GPU (at most 32 or so: their lists meet in the
// row's last block), each block's part a multiple of a batch.
#include <algorithm>

#include "common.cuh"
#include "exact_math.cuh"

namespace fnxk {

constexpr int LP_THREADS = 512, LP_WARPS = LP_THREADS / 32, LP_PER = 8, LP_BATCH = LP_THREADS * LP_PER, LP_CAP = 2048;
constexpr int LP_BLOCKS = 2 * 148;   // a call's blocks when it has few rows, so the rows that go to several blocks are fewer

struct LpPart {   // a block's part of a row
    float m, z, s;
    unsigned bad;
};
struct LpArgs {
    const float* logits;
    size_t stride;
    int n, v0, k, ntok, nsplit;
    const int* tok;
    float *lse, *ent, *lp, *top_lp;
    int* top_i;
    unsigned* count;             // [T] blocks of the row that are done (left at zero)
    LpPart* part;                // [T][nsplit]
    unsigned long long* cand;    // [T][nsplit][k]
    unsigned* err;
};

__device__ __forceinline__ unsigned long long lp_composite(float v, unsigned idx) {
    return ((unsigned long long) fkey(fadd(v, 0.f)) << 32) | (0xffffffffu - idx);
}

// (m, z, s) of two parts of a row together
__device__ __forceinline__ void lp_join(float& m, float& z, float& s, float m2, float z2, float s2) {
    const float mn = fmaxf(m, m2);
    if (mn == -INFINITY) return;
    const float d1 = fmaxf(m - mn, -200.f), d2 = fmaxf(m2 - mn, -200.f);   // e^-200 is zero: a part of nothing (-inf) drops out
    const float f1 = __expf(d1), f2 = __expf(d2);
    s = f1 * (s + d1 * z) + f2 * (s2 + d2 * z2);
    z = f1 * z + f2 * z2;
    m = mn;
}

// descending bitonic sort of list[0 .. n) (n <= LP_CAP), filled up to a power of two with zeros, which are below every entry
__device__ void lp_sort(unsigned long long* list, unsigned n, int tid) {
    unsigned p = 1;
    while (p < n) p <<= 1;
    for (unsigned i = n + tid; i < p; i += LP_THREADS) list[i] = 0ull;
    __syncthreads();
    for (unsigned size = 2; size <= p; size <<= 1)
        for (unsigned step = size >> 1; step; step >>= 1) {
            for (unsigned i = tid; i < p / 2; i += LP_THREADS) {
                const unsigned a = 2 * i - (i & (step - 1)), b = a + step;
                const unsigned long long x = list[a], y = list[b];
                if ((x < y) == ((a & size) == 0)) list[a] = y, list[b] = x;
            }
            __syncthreads();
        }
}

__global__ void __launch_bounds__(LP_THREADS) k_logprobs(const LpArgs a) {
    __shared__ unsigned long long list[LP_CAP];
    __shared__ float wm[LP_WARPS], wz[LP_WARPS], ws[LP_WARPS];
    __shared__ unsigned long long gmin[LP_WARPS];
    __shared__ unsigned n_list, fail_at, bad_s, last_s;
    __shared__ float lse_s;
    const int row = blockIdx.x / a.nsplit, split = blockIdx.x % a.nsplit, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float* x = a.logits + (size_t) row * a.stride;
    const int nbatch = (a.n + LP_BATCH - 1) / LP_BATCH, per = (nbatch + a.nsplit - 1) / a.nsplit;
    const int lo = min((long long) split * per * LP_BATCH, (long long) a.n), hi = (int) min((long long) lo + (long long) per * LP_BATCH, (long long) a.n);
    if (tid == 0) n_list = 0u, fail_at = 0xffffffffu, bad_s = 0u;
    pdl_wait();
    pdl_go();
    __syncthreads();
    float m = -INFINITY, z = 0.f, s = 0.f, floor_v = -INFINITY;
    unsigned long long floor_c = 0ull;   // the bound: an entry has to be above it
    bool bad = false;
    int group = 1;   // threads of a group: at least k groups in the block
    while (LP_THREADS / (2 * group) >= a.k && group < 32) group *= 2;
    for (int i0 = lo; i0 < hi; i0 += LP_BATCH) {
        float v[LP_PER];
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < LP_PER; ++j) {
            const int i = i0 + j * LP_THREADS + tid;
            v[j] = i < hi ? __ldcs(x + i) : -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < LP_PER; ++j) {
            bad = bad || !(v[j] < INFINITY);   // +inf or NaN
            mx = fmaxf(mx, v[j]);
        }
        if (mx > m) {
            const float d = fmaxf(m - mx, -200.f), f = __expf(d);
            s = f * (s + d * z);
            z *= f;
            m = mx;
        }
        if (mx != -INFINITY) {
#pragma unroll
            for (int j = 0; j < LP_PER; ++j) {
                const float d = fmaxf(v[j] - m, -200.f), e = __expf(d);
                z += e;
                s += e * d;
            }
        }
        if (!a.k) continue;
        if (i0 == lo) {   // the first bound
            unsigned long long best = 0ull;
#pragma unroll
            for (int j = 0; j < LP_PER; ++j) {
                const int i = i0 + j * LP_THREADS + tid;
                const unsigned long long c = i < hi ? lp_composite(v[j], (unsigned) i) : 0ull;
                best = c > best ? c : best;
            }
            for (int o = 1; o < group; o <<= 1) {
                const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
                best = other > best ? other : best;
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
                best = other < best ? other : best;
            }
            if (lane == 0) gmin[warp] = best;
            __syncthreads();
            best = gmin[0];
            for (int w = 1; w < LP_WARPS; ++w) best = gmin[w] < best ? gmin[w] : best;
            floor_c = best ? best - 1ull : 0ull;   // the bound itself may enter
            floor_v = best ? fkey_inv((unsigned) (floor_c >> 32)) : -INFINITY;
            if (floor_v != floor_v) floor_v = -INFINITY;   // (a NaN's key)
        }
        bool todo = true;   // this warp's entries of the batch are still to be written
        while (true) {
            if (todo) {
                unsigned mine = 0;
                if (!(mx < floor_v) || bad) {
#pragma unroll
                    for (int j = 0; j < LP_PER; ++j) {
                        const int i = i0 + j * LP_THREADS + tid;
                        if (i < hi && lp_composite(v[j], (unsigned) i) > floor_c) mine |= 1u << j;
                    }
                }
                if (__any_sync(0xffffffffu, mine)) {
                    unsigned before = (unsigned) __popc(mine), total;   // inclusive, then exclusive count over the lanes
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const unsigned y = __shfl_up_sync(0xffffffffu, before, o);
                        if (lane >= o) before += y;
                    }
                    total = __shfl_sync(0xffffffffu, before, 31);
                    before -= (unsigned) __popc(mine);
                    unsigned base = 0;
                    if (lane == 0) base = atomicAdd(&n_list, total);
                    base = __shfl_sync(0xffffffffu, base, 0);
                    if (base + total <= LP_CAP) {
#pragma unroll
                        for (int j = 0; j < LP_PER; ++j)
                            if (mine >> j & 1u) list[base + before++] = lp_composite(v[j], (unsigned) (i0 + j * LP_THREADS + tid));
                        todo = false;
                    } else if (lane == 0) {
                        atomicMin(&fail_at, base);   // places are handed out in order: below the first failure all is written
                    }
                } else {
                    todo = false;
                }
            }
            if (!__syncthreads_or(todo)) break;
            // the list is full: its best k stay, the last of them is the bound.  A list cut to k (at most 64) takes at least one
            // warp's entries (at most 256), so the batch is through after LP_WARPS rounds
            const unsigned have = fail_at;
            lp_sort(list, have, tid);
            floor_c = list[a.k - 1];
            floor_v = fkey_inv((unsigned) (floor_c >> 32));
            if (floor_v != floor_v) floor_v = -INFINITY;
            __syncthreads();
            if (tid == 0) n_list = (unsigned) a.k, fail_at = 0xffffffffu;
            __syncthreads();
        }
    }
    // ---- the block's statistics
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o), z2 = __shfl_xor_sync(0xffffffffu, z, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
        lp_join(m, z, s, m2, z2, s2);
    }
    if (lane == 0) wm[warp] = m, wz[warp] = z, ws[warp] = s;
    if (bad) bad_s = 1u;
    __syncthreads();
    m = wm[0], z = wz[0], s = ws[0];
    for (int w = 1; w < LP_WARPS; ++w) lp_join(m, z, s, wm[w], wz[w], ws[w]);
    bool any_bad = bad_s != 0u;
    unsigned have = min(n_list, (unsigned) LP_CAP);
    if (a.k) lp_sort(list, have, tid);
    if (a.nsplit > 1) {   // the row's last block joins the parts
        LpPart* parts = a.part + (size_t) row * a.nsplit;
        unsigned long long* cands = a.cand + (size_t) row * a.nsplit * a.k;
        for (int i = tid; i < a.k; i += LP_THREADS) cands[(size_t) split * a.k + i] = (unsigned) i < have ? list[i] : 0ull;
        if (tid == 0) parts[split] = LpPart{m, z, s, any_bad ? 1u : 0u};
        __threadfence();
        __syncthreads();
        if (tid == 0) last_s = atomicAdd(&a.count[row], 1u) == (unsigned) a.nsplit - 1u;
        __syncthreads();
        if (!last_s) return;
        __threadfence();
        m = -INFINITY, z = 0.f, s = 0.f, any_bad = false;
        for (int i = 0; i < a.nsplit; ++i) {
            const LpPart p = parts[i];
            lp_join(m, z, s, p.m, p.z, p.s);
            any_bad = any_bad || p.bad;
        }
        have = (unsigned) (a.nsplit * a.k);
        for (unsigned i = tid; i < have; i += LP_THREADS) list[i] = cands[i];
        __syncthreads();
        if (a.k) lp_sort(list, have, tid);
        if (tid == 0) a.count[row] = 0u;
    }
    const bool none = m == -INFINITY && !any_bad;
    if (tid == 0) {
        if (any_bad || none) atomicOr(a.err, 16u);
        const float lz = logf(z);
        lse_s = any_bad ? NAN : none ? -INFINITY : m + lz;
        a.lse[row] = lse_s;
        if (a.ent) a.ent[row] = any_bad ? NAN : none ? 0.f : fmaxf(lz - s / z, 0.f);
    }
    __syncthreads();
    const float lse = lse_s;
    for (int j = tid; j < a.ntok; j += LP_THREADS) {
        const long long t = (long long) a.tok[(size_t) row * a.ntok + j] - a.v0;
        const bool in = t >= 0 && t < a.n;
        a.lp[(size_t) row * a.ntok + j] = !in ? -INFINITY : any_bad ? NAN : none ? -INFINITY : x[t] - lse;
    }
    for (int j = tid; j < a.k; j += LP_THREADS) {
        const unsigned long long c = list[j];
        a.top_i[(size_t) row * a.k + j] = a.v0 + (int) (0xffffffffu - (unsigned) (c & 0xffffffffu));
        a.top_lp[(size_t) row * a.k + j] = any_bad ? NAN : none ? -INFINITY : fkey_inv((unsigned) (c >> 32)) - lse;
    }
}

// blocks a row: enough that the GPU has about two a multiprocessor, each with a batch at least; the lists of a row's blocks
// together fit the last block's
static int lp_splits(int n, int T, int k) {
    const int batches = (n + LP_BATCH - 1) / LP_BATCH, want = (LP_BLOCKS + T - 1) / T;
    int s = std::max(1, std::min(want, std::min(batches, LP_CAP / std::max(k, LP_CAP / 64))));
    const int per = (batches + s - 1) / s;
    return (batches + per - 1) / per;   // no empty block
}

}  // namespace fnxk

using namespace fnxk;

extern "C" {

size_t fnx_logprobs_scratch_bytes(int n, int T, int k) {
    if (n < 1 || T < 1 || k < 0 || k > FNX_TOPK_N) return 0;
    const size_t s = (size_t) lp_splits(n, T, k);
    return s == 1 ? 16 : (size_t) LP_BLOCKS * 4 + (size_t) T * s * (sizeof(LpPart) + 8 * (size_t) k);
}

int fnx_logprobs(const float* logits, size_t stride, int n, int T, int v0, const int* tok, int ntok, int k, float* lse, float* entropy, float* lp,
                 float* top_lp, int* top_i, void* scratch, unsigned* err, void* st) {
    FNX_REQUIRE(n >= 1 && T >= 1 && stride >= (size_t) n && v0 >= 0, "logprobs: %d rows of %d logits, %zu apart, from token %d", T, n, stride, v0);
    FNX_REQUIRE(k >= 0 && k <= FNX_TOPK_N && k <= n, "logprobs: %d alternatives of %d (at most %d)", k, n, FNX_TOPK_N);
    FNX_REQUIRE(n <= (1 << 30) && v0 <= (1 << 30), "logprobs: tokens %d .. %d + %d", v0, v0, n);
    FNX_REQUIRE(ntok >= 0 && (!ntok || (tok && lp)), "logprobs: %d given tokens without their buffers", ntok);
    FNX_REQUIRE(logits && lse && scratch && err && (!k || (top_lp && top_i)), "logprobs: a null buffer");
    FNX_REQUIRE((uintptr_t) scratch % 16 == 0, "logprobs: scratch not 16-byte aligned");
    const int ns = lp_splits(n, T, k);
    FNX_REQUIRE((long long) T * ns < (1ll << 31), "logprobs: %d rows", T);
    LpArgs a{logits, stride, n, v0, k, ntok, ns, tok, lse, entropy, lp, top_lp, top_i, (unsigned*) scratch, nullptr, nullptr, err};
    // the counters have their place whatever the call's sizes, so that one scratch serves calls of different ones
    a.part = reinterpret_cast<LpPart*>((char*) scratch + LP_BLOCKS * 4);
    a.cand = reinterpret_cast<unsigned long long*>(a.part + (size_t) T * ns);
    launch(0, k_logprobs, dim3((unsigned) T * ns), LP_THREADS, 0, strm(st), a);
    return launch_ok("logprobs");
}
}
