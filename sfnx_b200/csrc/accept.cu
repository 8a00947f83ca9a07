// Acceptance of a verify window on the host: greedy prefix match and rejection sampling against fixed drafts over the
// rows' 64 candidates, and the merge of the GPUs' candidate lists.  Restated from the reference's Session, statement for
// statement where the arithmetic demands it (src/session.cpp:39-82 make_dist / draw, 469-510 the acceptance loop;
// src/engine_common.cu:640-653 the merge), as free functions over plain arrays: this is host policy the drop-in keeps,
// and the reference's own object code is its checker (oracle/ref_accept.cpp).  Without a counterpart there: the walk down a draft
// tree and the merge of the slices' log probabilities.
#include <algorithm>
#include <cmath>
#include <limits>
#include <random>
#include <vector>

#include "common.cuh"

namespace {

struct Dist {
    int n = 0;
    int ids[FNX_TOPK_N];
    double p[FNX_TOPK_N];
    double prob(int id) const {
        for (int i = 0; i < n; ++i)
            if (ids[i] == id) return p[i];
        return 0.0;
    }
};

// top_k, then top_p over the untempered softmax (double), then min_p as a logit threshold, then the temperature's
// softmax over the survivors; cand sorted by (logit desc, id asc)
Dist make_dist(const float* cv, const int* ci, int ncand, const FnxSampling& s) {
    const int k = (s.top_k <= 0 || s.top_k > ncand) ? ncand : s.top_k;
    int keep = k;
    const double mx = cv[0];
    if (s.top_p < 1.f) {
        double sum = 0.0;
        for (int i = 0; i < k; ++i) sum += std::exp((double) cv[i] - mx);
        double cum = 0.0;
        for (int i = 0; i < k; ++i) {
            cum += std::exp((double) cv[i] - mx) / sum;
            if (cum >= (double) s.top_p) {
                keep = i + 1;
                break;
            }
        }
    }
    if (s.min_p > 0.f) {
        const float thresh = cv[0] + std::log(s.min_p);
        for (int i = 1; i < keep; ++i)
            if (cv[i] < thresh) {
                keep = i;
                break;
            }
    }
    Dist d;
    const double inv_t = 1.0 / s.temperature, smx = cv[0] * inv_t;
    double sum = 0.0;
    d.n = keep;
    for (int i = 0; i < keep; ++i) {
        d.ids[i] = ci[i];
        d.p[i] = std::exp(cv[i] * inv_t - smx);
        sum += d.p[i];
    }
    for (int i = 0; i < keep; ++i) d.p[i] /= sum;
    return d;
}

int draw(const Dist& d, double u) {
    double cum = 0.0;
    for (int i = 0; i < d.n; ++i) {
        cum += d.p[i];
        if (u < cum) return d.ids[i];
    }
    return d.ids[d.n - 1];
}

struct Rng {
    std::mt19937_64 gen;
    std::uniform_real_distribution<double> unif{0.0, 1.0};
};

}  // namespace

extern "C" {

int fnx_accept_greedy(const int* rows, const int* out, int T) {
    int n = 1;
    while (n < T && rows[n] == out[n - 1]) ++n;
    return n;
}

void* fnx_rng_new(unsigned long long seed) {
    Rng* r = new Rng;
    r->gen.seed(seed);
    return r;
}
void fnx_rng_free(void* rng) { delete (Rng*) rng; }

// draft rows[n + 1] stands with probability min(1, p_n(draft)) (a fixed draft's q is all on it); else row n's token is
// drawn from max(0, p_n - q_n) normalised and the window ends; all standing: one more from the last row.  One uniform
// per test and per draw.
int fnx_accept_sampled(const int* rows, int T, const float* cand_v, const int* cand_i, const FnxSampling* s, void* rng, int* o) {
    Rng& r = *(Rng*) rng;
    int n;
    for (n = 0; n < T; ++n) {
        Dist d = make_dist(cand_v + (size_t) n * FNX_TOPK_N, cand_i + (size_t) n * FNX_TOPK_N, FNX_TOPK_N, *s);
        if (n + 1 < T) {
            const int dr = rows[n + 1];
            if (r.unif(r.gen) * 1.0 < d.prob(dr)) {
                o[n] = dr;
                continue;
            }
            const Dist p0 = d;
            double rest = 0.0;
            for (int i = 0; i < d.n; ++i) {
                const double qi = d.ids[i] == dr ? 1.0 : 0.0;
                d.p[i] = std::max(0.0, d.p[i] - qi);
                rest += d.p[i];
            }
            if (rest > 1e-12)
                for (int i = 0; i < d.n; ++i) d.p[i] /= rest;
            else d = p0;
        }
        o[n] = draw(d, r.unif(r.gen));
        ++n;
        break;
    }
    return n;
}

// n-gram lookup drafts (reference src/session.cpp:377-394, lookup_drafts; LOOKUP_N = LOOKUP_MIN = 3): the tokens that followed
// the latest earlier occurrence of the context's last three tokens.  Only that latest occurrence is looked at; it offers
// drafts if a token follows it and (d1 >= 0) that token is d1.  How many: the match is grown backwards from the trigram, up
// to lk tokens, and k = min(lk, max(3, match length)) tokens are taken (fewer at the context's end); tokens from the first
// image cell (>= image_tok) on are dropped.  Returns the number of drafts written to out (room for lk).
int fnx_lookup_drafts(const int* ctx, int n, int lk, int d1, int image_tok, int* out) {
    constexpr int NG = 3, KMIN = 3;
    if (!ctx || !out || n < 0 || lk < 0) return -fnxk::fail("lookup_drafts: bad arguments (%d tokens, %d drafts)", n, lk);
    if (lk == 0 || n <= NG) return 0;
    const int tail = n - NG;   // where the context's last trigram starts
    int found = -1;
    for (int s = tail - 1; s >= 0 && found < 0; --s)
        if (ctx[s] == ctx[tail] && ctx[s + 1] == ctx[tail + 1] && ctx[s + 2] == ctx[tail + 2]) found = s;
    if (found < 0 || found + NG >= n || (d1 >= 0 && ctx[found + NG] != d1)) return 0;
    int m = NG;   // tokens before the two trigrams that agree as well
    while (m < lk && m - NG < found && ctx[found - 1 - (m - NG)] == ctx[tail - 1 - (m - NG)]) ++m;
    const int k = std::min(lk, std::max(KMIN, m)), end = std::min(n, found + NG + k);
    int cnt = 0;
    for (int i = found + NG; i < end && ctx[i] < image_tok; ++i) out[cnt++] = ctx[i];
    return cnt;
}

int fnx_top_merge(const float* vs, const int* is, int nslice, int T, float* out_v, int* out_i) {
    if (nslice < 1 || T < 1) return fnxk::fail("top_merge: %d slices, %d rows", nslice, T);
    std::vector<std::pair<float, int>> c((size_t) nslice * FNX_TOPK_N);
    for (int t = 0; t < T; ++t) {
        for (int s = 0; s < nslice; ++s)
            for (int k = 0; k < FNX_TOPK_N; ++k)
                c[(size_t) s * FNX_TOPK_N + k] = {vs[((size_t) s * T + t) * FNX_TOPK_N + k], is[((size_t) s * T + t) * FNX_TOPK_N + k]};
        std::sort(c.begin(), c.end(), [](const std::pair<float, int>& a, const std::pair<float, int>& b) {
            return a.first > b.first || (a.first == b.first && a.second < b.second);
        });
        for (int k = 0; k < FNX_TOPK_N; ++k) out_v[t * FNX_TOPK_N + k] = c[k].first, out_i[t * FNX_TOPK_N + k] = c[k].second;
    }
    return 0;
}

// the slices' softmax statistics joined: with lse = log sum e^lse_i and w_i = e^(lse_i - lse), a log probability of slice i changes by
// log w_i, and H = sum w_i (H_i - log w_i).  Only differences of the lse_i are formed, in double, so their size costs nothing.
int fnx_logprobs_merge(const float* lse_s, const float* entropy_s, const float* lp_s, const float* top_lp_s, const int* top_i_s, int nslice, int T,
                       int ntok, int k, float* lse, float* entropy, float* lp, float* top_lp, int* top_i) {
    constexpr int MOST = 64;
    const float ninf = -std::numeric_limits<float>::infinity();
    if (nslice < 1 || nslice > MOST || T < 1 || ntok < 0 || k < 0 || k > FNX_TOPK_N)
        return fnxk::fail("logprobs_merge: %d slices (1..%d), %d rows, %d tokens, %d alternatives", nslice, MOST, T, ntok, k);
    if (!lse_s || !lse || (entropy && !entropy_s) || (ntok && (!lp_s || !lp)) || (k && (!top_lp_s || !top_i_s || !top_lp || !top_i)))
        return fnxk::fail("logprobs_merge: a null buffer");
    auto raw = [ninf](float l, float z) { return l == ninf ? ninf : l + z; };   // the logit that a log probability was made of
    for (int t = 0; t < T; ++t) {
        double m = ninf, z = 0.0, h = 0.0, shift[MOST];   // shift: log w_i
        bool nan = false;
        for (int i = 0; i < nslice; ++i) {
            const double x = lse_s[(size_t) i * T + t];
            nan = nan || x != x;
            if (x > m) m = x;
        }
        const bool none = !(m > ninf);
        if (!none && !nan) {
            for (int i = 0; i < nslice; ++i) z += std::exp(lse_s[(size_t) i * T + t] - m);
            for (int i = 0; i < nslice; ++i) {
                shift[i] = lse_s[(size_t) i * T + t] - m - std::log(z);
                const double w = std::exp(shift[i]);
                if (w > 0.0 && entropy) h += w * ((double) entropy_s[(size_t) i * T + t] - shift[i]);
            }
        }
        lse[t] = nan ? std::numeric_limits<float>::quiet_NaN() : none ? ninf : (float) (m + std::log(z));
        if (entropy) entropy[t] = nan ? lse[t] : none ? 0.f : (float) std::max(h, 0.0);
        auto whole = [&](float l, int i) { return none || l == ninf ? ninf : (float) std::min(l + shift[i], 0.0); };   // of a slice's log probability
        for (int j = 0; j < ntok; ++j) {
            float x = ninf;
            for (int i = 0; i < nslice && !nan; ++i) x = std::max(x, whole(lp_s[((size_t) i * T + t) * ntok + j], i));
            lp[(size_t) t * ntok + j] = nan ? lse[t] : x;
        }
        int head[MOST] = {};
        for (int j = 0; j < k; ++j) {   // every slice's list is in order: the best of the heads
            if (nan) {   // no order to speak of, in the whole row
                top_i[(size_t) t * k + j] = -1, top_lp[(size_t) t * k + j] = lse[t];
                continue;
            }
            int best = -1, bi = 0;
            float bx = 0.f, bl = 0.f;
            for (int i = 0; i < nslice; ++i) {
                if (head[i] >= k) continue;
                const size_t at = (size_t) i * T + t;
                const float x = raw(top_lp_s[at * k + head[i]], lse_s[at]);
                const int id = top_i_s[at * k + head[i]];
                if (best < 0 || x > bx || (x == bx && id < bi)) best = i, bx = x, bi = id, bl = top_lp_s[at * k + head[i]];
            }
            ++head[best];
            top_i[(size_t) t * k + j] = bi;
            top_lp[(size_t) t * k + j] = j ? std::min(whole(bl, best), top_lp[(size_t) t * k + j - 1]) : whole(bl, best);   // (in order, whatever was rounded)
        }
    }
    return 0;
}

int fnx_accept_tree(const int* tok, const int* parent, const int* out, int n, int* path) {
    if (!tok || !parent || !out || !path || n < 1) return -fnxk::fail("accept_tree: a null buffer or %d nodes", n);
    for (int i = 1; i < n; ++i)
        if (parent[i] < -1 || parent[i] >= i) return -fnxk::fail("accept_tree: node %d's parent %d", i, parent[i]);
    int len = 0, at = 0;
    path[len++] = 0;
    for (int i = 1; i < n; ++i)   // a child comes after its parent, so one pass in order finds the path
        if (parent[i] == at && tok[i] == out[at]) path[len++] = at = i;
    return len;
}
}
