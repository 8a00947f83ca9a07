// Attention of several sequences' rows over the f16 cache: prompts, chunks of prompts, single tokens and draft trees (no
// counterpart in the reference's windows).  Plain form: a warp a (row, query head), one pass over the positions with the running
// maximum and sum of the softmax.
#include "exact_math.cuh"
#include "seqs.cuh"

namespace fnxk {

struct SqAttn {
    const uint16_t* q;
    const float* qg;
    const uint16_t *kc, *vc;
    FnxKvPages g;
    FnxSeqs sq;
    const unsigned* anc;
    uint16_t* out;
    int q_stride, out_stride, nq, nkv, words;
};

template <int HD>
__global__ void __launch_bounds__(128) k_attn_seqs_plain(const SqAttn a) {
    constexpr int E = HD / 32;
    const int t = blockIdx.x, h = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    pdl_wait();
    pdl_go();
    const int s = sq_find(a.sq.row0, a.sq.nseq, t);
    if (s < 0 || h >= a.nq) return;
    const int i0 = t - a.sq.row0[s], n = min(a.sq.row0[s + 1], a.sq.rows) - a.sq.row0[s], p0 = max(a.sq.pos0[s], 0);
    const size_t row_elems = (size_t) a.nkv * HD, head = (size_t) (h / (a.nq / a.nkv)) * HD + lane * E;
    float q[E], o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) q[e] = h2f(a.q[(size_t) t * a.q_stride + (size_t) h * HD + lane * E + e]), o[e] = 0.f;
    const float rs = 1.0f / sqrtf((float) HD);
    float m = -INFINITY, z = 0.f;
    const long long cap = a.sq.pt ? (long long) a.sq.pt_stride * a.g.rows : (long long) a.g.cap, end = min((long long) p0 + (a.anc ? n : i0 + 1), cap);
    for (int p = 0; p < end; ++p) {
        const int i = p - p0;
        if (a.anc && i >= 0 && !(i / 32 < a.words && (a.anc[(size_t) t * a.words + i / 32] >> (i % 32) & 1u))) continue;
        const long long cell = sq_cell(a.sq, a.g, s, p);
        float x = 0.f, v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = 0.f;
        if (cell >= 0) {
            const size_t at = sq_at(a.sq, a.g, cell, row_elems) + head;
#pragma unroll
            for (int e = 0; e < E; ++e) x += q[e] * h2f(a.kc[at + e]), v[e] = h2f(a.vc[at + e]);
        }
        x = wsum(x) * rs;
        const float mn = fmaxf(m, x), f = __expf(m - mn), w = __expf(x - mn);
        z = z * f + w;
        m = mn;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = o[e] * f + w * v[e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
        float y = z > 0.f ? o[e] / z : 0.f;
        if (a.qg) y *= ex_sigmoid(a.qg[((size_t) t * a.nq + h) * 2 * HD + HD + lane * E + e]);
        a.out[(size_t) t * a.out_stride + (size_t) h * HD + lane * E + e] = f2h(y);
    }
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
    const SqAttn a{q16, qg, kc, vc, g, *sq, anc, out, q_stride, out_stride, nq, nkv, words};
    const dim3 grid(sq->rows, (nq + 3) / 4);
    if (hd == 256) launch(0, k_attn_seqs_plain<256>, grid, 128, 0, strm(st), a);
    else launch(0, k_attn_seqs_plain<128>, grid, 128, 0, strm(st), a);
    return launch_ok(what);
}

}  // namespace fnxk

using namespace fnxk;

extern "C" {

size_t fnx_attn_seqs_scratch_bytes(const FnxSeqs* sq, int nq, int nkv, int hd) {
    if (!sq || nq < 1 || nkv < 1 || hd < 1) return 0;
    return 16;
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
