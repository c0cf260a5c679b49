// The language-model operators through the C++ host layer (deepnet_amd/cpp/hip_tensor.hpp), against plain loops in double precision.
// Sizes of a few hundred terms: single precision stays within 1e-5 of each result's scale, far above its 2^-24 per term.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <random>
#include <vector>

#include "hip_tensor.hpp"

namespace tn = Tensor;
using TF = tn::Tensor<float>;
using TI = tn::Tensor<int64_t>;
using TB = tn::Tensor<bool>;

static int g_failed = 0, g_passed = 0;
static void report(const char* name, bool ok) {
    std::printf("%s %s\n", ok ? "PASS" : "FAIL", name);
    (ok ? g_passed : g_failed)++;
}
static std::vector<float> download(const TF& t) {
    std::vector<float> v(t.NElems());
    t.toHost(v.data());
    return v;
}
static void close(const char* name, const TF& got, const std::vector<double>& want, double tol) {
    auto g = download(got);
    bool ok = g.size() == want.size();
    for (size_t i = 0; ok && i < g.size(); i++) ok = std::fabs(g[i] - want[i]) <= tol;
    report(name, ok);
}
template <class E, class F> static void throws(const char* name, F f) {
    try {
        f();
        report(name, false);
    } catch (const E&) {
        report(name, true);
    }
}

int main() {
    try {
        tn::check(dnh_init(0));
        std::mt19937 rng(5);
        std::normal_distribution<float> normal;
        auto rnd = [&](size_t n) { std::vector<float> v(n); for (auto& x : v) x = normal(rng); return v; };
        // embedding and its gradient
        const int V = 13, D = 6, N = 40;
        auto table = rnd(V * D), g = rnd(N * D);
        std::vector<int64_t> tok(N);
        for (auto& t : tok) t = rng() % V;
        TF T = TF::ofHost(table, {V, D});
        TI K = TI::ofHost(tok, {N / 4, 4});
        std::vector<double> rows, dt(V * D, 0.0);
        for (int i = 0; i < N; i++)
            for (int d = 0; d < D; d++) {
                rows.push_back(2.0 * table[tok[i] * D + d]);
                dt[tok[i] * D + d] += 2.0 * g[i * D + d];
            }
        TF emb = TF::embedding(T, K, 2.0f);
        report("embedding.shape", emb.Shape_() == tn::Shape({N / 4, 4, D}));
        close("embedding", emb, rows, 0);
        close("embeddingGrad", TF::embeddingGrad(K, TF::ofHost(g, {N / 4, 4, D}), V, 2.0f), dt, 1e-5);
        tok[3] = V;
        throws<std::out_of_range>("embedding.outOfRange", [&] { TF::embedding(T, TI::ofHost(tok, {N})); });
        throws<std::invalid_argument>("embedding.rank", [&] { TF::embedding(TF::ofHost(table, {V * D}), K); });
        // log probabilities and their gradient
        const int R = 5, W = 300;
        auto x = rnd(R * W), up = rnd(R);
        std::vector<int64_t> y(R);
        for (auto& t : y) t = rng() % W;
        std::vector<double> lp, lse, ent, best, dx;
        std::vector<int64_t> idx;
        for (int r = 0; r < R; r++) {
            double s = 0, e = 0;
            for (int j = 0; j < W; j++) s += std::exp((double)x[r * W + j]);
            const double l = std::log(s);
            for (int j = 0; j < W; j++) {
                const double q = x[r * W + j] - l;
                e -= std::exp(q) * q;
                dx.push_back(up[r] * ((j == y[r]) - std::exp(q)));
            }
            lp.push_back(x[r * W + y[r]] - l);
            lse.push_back(l);
            ent.push_back(e);
            std::vector<int64_t> o(W);
            for (int j = 0; j < W; j++) o[j] = j;
            std::stable_sort(o.begin(), o.end(), [&](int64_t a, int64_t b) { return x[r * W + a] > x[r * W + b]; });
            for (int k = 0; k < 3; k++) {
                idx.push_back(o[k]);
                best.push_back(x[r * W + o[k]] - l);
            }
        }
        TF X = TF::ofHost(x, {R, W});
        TI Y = TI::ofHost(y, {R});
        auto p = TF::tokenLogProbs(X, Y, 3);
        close("tokenLogProbs", p.logProbs, lp, 1e-5);
        close("tokenLogProbs.lse", p.lse, lse, 1e-5);
        close("tokenLogProbs.entropy", p.entropy, ent, 1e-4);
        close("tokenLogProbs.top", p.topLogProbs, best, 1e-5);
        std::vector<int64_t> gi(R * 3);
        p.topTokens.toHost(gi.data());
        report("tokenLogProbs.topTokens", gi == idx);
        close("tokenLogProbs.withoutTop", TF::tokenLogProbs(X, Y).logProbs, lp, 1e-5);
        close("tokenLogProbsGrad", TF::tokenLogProbsGrad(X, Y, p.lse, TF::ofHost(up, {R})), dx, 1e-5);
        throws<tn::NotSupportedException>("tokenLogProbs.tooMany", [&] { TF::tokenLogProbs(X, Y, 65); });
        // cross attention and its gradient: two query heads on one key head, a masked key
        const int H = 2, L = 3, S = 7, C = 8;
        auto q = rnd(H * L * C), k = rnd(S * C), v = rnd(S * C), go = rnd(H * L * C);
        std::vector<char> keep(S, 1);
        keep[4] = 0;
        std::vector<double> out(H * L * C, 0), dq(H * L * C, 0), dk(S * C, 0), dv(S * C, 0);
        const double sc = 1 / std::sqrt((double)C);
        for (int r = 0; r < H * L; r++) {
            std::vector<double> w(S, 0);
            double s = 0, delta = 0;
            for (int j = 0; j < S; j++) {
                if (!keep[j]) continue;
                double a = 0;
                for (int d = 0; d < C; d++) a += (double)q[r * C + d] * k[j * C + d];
                s += w[j] = std::exp(a * sc);
            }
            std::vector<double> dp(S, 0);
            for (int j = 0; j < S; j++) {
                w[j] /= s;
                for (int d = 0; d < C; d++) {
                    out[r * C + d] += w[j] * v[j * C + d];
                    dp[j] += (double)go[r * C + d] * v[j * C + d];
                    dv[j * C + d] += w[j] * go[r * C + d];
                }
                delta += w[j] * dp[j];
            }
            for (int j = 0; j < S; j++)
                for (int d = 0; d < C; d++) {
                    const double ds = w[j] * (dp[j] - delta) * sc;
                    dq[r * C + d] += ds * k[j * C + d];
                    dk[j * C + d] += ds * q[r * C + d];
                }
        }
        TF Q = TF::ofHost(q, {1, H, L, C}), Kk = TF::ofHost(k, {1, 1, S, C}), Vv = TF::ofHost(v, {1, 1, S, C});
        TB M = TB::ofHost(reinterpret_cast<const bool*>(keep.data()), {1, S});
        auto a = TF::crossAttention(Q, Kk, Vv, &M);
        close("crossAttention", a.out, out, 1e-5);
        auto gr = TF::crossAttentionGrad(TF::ofHost(go, {1, H, L, C}), Q, Kk, Vv, a, &M);
        close("crossAttentionGrad.dQ", gr.dQ, dq, 1e-5);
        close("crossAttentionGrad.dK", gr.dK, dk, 1e-5);
        close("crossAttentionGrad.dV", gr.dV, dv, 1e-5);
        throws<std::invalid_argument>("crossAttention.rank", [&] { TF::crossAttention(TF::ofHost(q, {H, L, C}), Kk, Vv); });
        tn::check(dnh_device_sync());
    } catch (const std::exception& e) {
        std::printf("FAIL uncaught exception: %s\n", e.what());
        g_failed++;
    }
    std::printf("%d passed, %d failed\n", g_passed, g_failed);
    return g_failed ? 1 : 0;
}
