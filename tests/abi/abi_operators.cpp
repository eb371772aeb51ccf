// The checkpoint, group norm and class score entry points of include/magnet_hip.h called from plain C++ (no torch, no Python), each
// result checked on the host against its formula in double precision, and the memory behind every output for stray writes.  Built by
// the Makefile and run by tests/test_operators_repairs_gpu.py; built a second time with the host side under AddressSanitizer by
// tools/host_asan.sh.
//
//   abi_operators        -> all cases, prints "operators ok"
//
// u = 2^-24, the rounding of a float32 operation; bounds count those along the formula.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <vector>

#include <unistd.h>

#include <hip/hip_runtime.h>

#include "../../include/magnet_hip.h"

static int g_fail = 0;
#define HIP_OK(x) do { hipError_t e_ = (x); if (e_ != hipSuccess) { fprintf(stderr, "%s:%d %s: %s\n", __FILE__, __LINE__, #x, hipGetErrorString(e_)); exit(2); } } while (0)
#define MH_CALL(x) do { int rc_ = (x); if (rc_ != MH_OK) { fprintf(stderr, "%s:%d %s -> %d: %s\n", __FILE__, __LINE__, #x, rc_, mh_last_error()); exit(3); } } while (0)
#define EXPECT(c, ...) do { if (!(c)) { fprintf(stderr, "%s:%d FAILED %s: ", __FILE__, __LINE__, #c); fprintf(stderr, __VA_ARGS__); fprintf(stderr, "\n"); if (++g_fail > 20) exit(4); } } while (0)

static const double U = std::ldexp(1.0, -24);
constexpr size_t kGuard = 512;                    // bytes behind an output that have to stay as they are

template <class T>
struct Dev {
    T* p = nullptr;
    size_t n = 0;
    explicit Dev(size_t count) : n(count) {
        HIP_OK(hipMalloc(reinterpret_cast<void**>(&p), n * sizeof(T) + kGuard));
        HIP_OK(hipMemset(p, 0xA5, n * sizeof(T) + kGuard));
    }
    explicit Dev(const std::vector<T>& h) : Dev(h.size()) { if (n) HIP_OK(hipMemcpy(p, h.data(), n * sizeof(T), hipMemcpyHostToDevice)); }
    Dev(const Dev&) = delete;
    Dev& operator=(const Dev&) = delete;
    ~Dev() { if (p) (void)hipFree(p); }
    std::vector<T> get(const char* what) const {
        std::vector<uint8_t> h(n * sizeof(T) + kGuard);
        HIP_OK(hipMemcpy(h.data(), p, h.size(), hipMemcpyDeviceToHost));
        for (size_t i = 0; i < kGuard; ++i) EXPECT(h[n * sizeof(T) + i] == 0xA5, "%s: byte %zu behind its end", what, i);
        std::vector<T> r(n);
        if (n) std::memcpy(r.data(), h.data(), n * sizeof(T));
        return r;
    }
};

struct Rng {                                      // splitmix64
    uint64_t s;
    explicit Rng(uint64_t seed) : s(seed) {}
    uint64_t next() { uint64_t z = (s += 0x9e3779b97f4a7c15ull); z = (z ^ (z >> 30)) * 0xbf58476d1ce4e5b9ull; z = (z ^ (z >> 27)) * 0x94d049bb133111ebull; return z ^ (z >> 31); }
    double uni() { return double(next() >> 11) * (1.0 / 9007199254740992.0); }
    float value() { return float((2.0 * uni() - 1.0) * std::exp2(4.0 * uni() - 2.0)); }
    std::vector<float> values(size_t n) { std::vector<float> v(n); for (float& x : v) x = value(); return v; }
};

static size_t up(size_t n, size_t to) { return (n + to - 1) / to * to; }

static void near_to(const std::vector<float>& got, const std::vector<double>& want, const std::vector<double>& bound, const char* what) {
    EXPECT(got.size() == want.size(), "%s: %zu values, %zu expected", what, got.size(), want.size());
    for (size_t i = 0; i < got.size() && g_fail < 20; ++i)
        EXPECT(std::fabs(double(got[i]) - want[i]) <= bound[i], "%s[%zu] = %.9g, %.9g expected, bound %.3g", what, i, got[i], want[i], bound[i]);
}

// ---- checkpoints: the bytes by their definition ------------------------------------------------------------------------
struct Bytes { std::vector<uint8_t> codes, scales; std::vector<double> values; };

static Bytes encoded(const std::vector<float>& x, size_t rows, size_t m) {
    const size_t mp = up(m, 32), rp = up(rows, 8);
    Bytes b{std::vector<uint8_t>(rows * mp, 128), std::vector<uint8_t>(mp / 32 * rp, 0), std::vector<double>(rows * m)};
    for (size_t r = 0; r < rows; ++r)
        for (size_t c0 = 0; c0 < m; c0 += 32) {
            const size_t c1 = std::min(m, c0 + 32);
            double top = 0.0;
            bool finite = true;
            for (size_t c = c0; c < c1; ++c) { finite = finite && std::isfinite(x[r * m + c]); top = std::max(top, std::fabs(double(x[r * m + c]))); }
            if (!finite) { for (size_t c = c0; c < c1; ++c) b.values[r * m + c] = NAN; continue; }
            int p = 0;
            const double f = std::frexp(top, &p);
            const int s = std::min(121, std::max(-110, std::nearbyint(f * 128.0) > 127.0 ? p - 6 : p - 7));
            b.scales[c0 / 32 * rp + r] = uint8_t(s + 128);
            for (size_t c = c0; c < c1; ++c) {
                const double q = std::min(127.0, std::max(-127.0, std::nearbyint(std::ldexp(double(x[r * m + c]), -s))));
                b.codes[r * mp + c] = uint8_t(int(q) + 128);
                b.values[r * m + c] = std::ldexp(q, s);
            }
        }
    return b;
}

static void checkpoints(hipStream_t stream, size_t n, size_t m, size_t k, uint64_t seed) {
    Rng rng(seed);
    std::vector<float> x = rng.values(2 * n * m);
    const std::vector<float> g = rng.values(2 * n * k);
    const Bytes want = encoded(x, 2 * n, m);
    Dev<float> dx(x), dg(g), back(2 * n * m), out(m * k);
    Dev<uint8_t> codes(want.codes.size()), scales(want.scales.size());
    MH_CALL(mh_ckpt_store(dx.p, int64_t(2 * m), int64_t(m), int64_t(n), int32_t(m), codes.p, scales.p, stream));
    MH_CALL(mh_ckpt_restore(codes.p, scales.p, int64_t(n), int32_t(m), back.p, int64_t(2 * m), int64_t(m), stream));
    const size_t bytes = mh_ckpt_gram_workspace_bytes(int64_t(n), int32_t(m), int32_t(k));
    EXPECT((n == 0) == (bytes == 0), "workspace of %zu bytes", bytes);
    Dev<uint8_t> ws(bytes);
    MH_CALL(mh_ckpt_gram(codes.p, scales.p, int64_t(n), int32_t(m), dg.p, int64_t(2 * k), int64_t(k), int32_t(k), out.p, ws.p, bytes, stream));
    HIP_OK(hipStreamSynchronize(stream));
    EXPECT(codes.get("codes") == want.codes && scales.get("scales") == want.scales, "checkpoint of %zu x %zu", n, m);
    const std::vector<float> values = back.get("restored");
    for (size_t i = 0; i < values.size(); ++i) EXPECT(double(values[i]) == want.values[i], "restored[%zu]", i);
    (void)ws.get("workspace");
    std::vector<double> dw(m * k, 0.0), mag(m * k, 0.0);
    for (size_t r = 0; r < 2 * n; ++r)
        for (size_t i = 0; i < m; ++i)
            for (size_t j = 0; j < k; ++j) {
                const double t = want.values[r * m + i] * double(g[r * k + j]);
                dw[i * k + j] += t;
                mag[i * k + j] += std::fabs(t);
            }
    // a float32 sum of up to min(rows, 1024) terms in some order, 64 bits behind that, three products for each term
    for (double& b : mag) b = b * U * double(std::min<size_t>(2 * n, 1024) + 8);
    near_to(out.get("gradient"), dw, mag, "gradient");
}

// ---- group norm --------------------------------------------------------------------------------------------------------
static void norms(hipStream_t stream, size_t n, size_t f, size_t groups, const std::vector<int32_t>& ptr, bool relu, bool held, uint64_t seed) {
    Rng rng(seed);
    std::vector<float> x = rng.values(2 * n * f), g = rng.values(2 * n * f), w = rng.values(f), b = rng.values(f);
    const size_t graphs = ptr.empty() ? (n ? 1 : 0) : ptr.size() - 1, d = f / groups;
    const std::vector<int32_t> at = ptr.empty() ? std::vector<int32_t>{0, int32_t(n)} : ptr;
    const double eps = double(1e-5f);
    auto centre = [&](size_t gr, size_t q, double& mr, double& mi, double& sd) {
        double s0 = 0, s1 = 0, s2 = 0;
        const double count = double(at[gr + 1] - at[gr]) * double(d);
        for (size_t r = size_t(at[gr]); r < size_t(at[gr + 1]); ++r)
            for (size_t c = q * d; c < (q + 1) * d; ++c) { s0 += x[(2 * r) * f + c]; s1 += x[(2 * r + 1) * f + c]; }
        mr = count > 0 ? s0 / count : 0.0; mi = count > 0 ? s1 / count : 0.0;
        for (size_t r = size_t(at[gr]); r < size_t(at[gr + 1]); ++r)
            for (size_t c = q * d; c < (q + 1) * d; ++c) {
                const double a = x[(2 * r) * f + c] - mr, e = x[(2 * r + 1) * f + c] - mi;
                s2 += a * a + e * e;
            }
        sd = std::sqrt((count > 0 ? s2 / count : 0.0) + eps);
    };
    // values whose gate hangs on a rounding are moved off it, twice, since moving them moves the statistics
    for (int turn = 0; relu && turn < 3; ++turn)
        for (size_t gr = 0; gr < graphs; ++gr)
            for (size_t q = 0; q < groups; ++q) {
                double mr, mi, sd;
                centre(gr, q, mr, mi, sd);
                for (size_t r = size_t(at[gr]); r < size_t(at[gr + 1]); ++r)
                    for (size_t c = q * d; c < (q + 1) * d; ++c)
                        if (std::fabs((x[(2 * r) * f + c] - mr) / sd * w[c] + b[c]) < 1e-4) x[(2 * r) * f + c] += float(0.05 * sd);
            }
    const Bytes kept = encoded(x, 2 * n, f);
    std::vector<double> y(2 * n * f, 0.0), ty(2 * n * f, 0.0), dx(2 * n * f, 0.0), tdx(2 * n * f, 0.0), dw(f, 0.0), tw(f, 0.0), db(f, 0.0), tb(f, 0.0);
    for (size_t gr = 0; gr < graphs; ++gr)
        for (size_t q = 0; q < groups; ++q) {
            double mr, mi, sd;
            centre(gr, q, mr, mi, sd);
            const double count = double(at[gr + 1] - at[gr]) * double(d), mean[2] = {mr, mi};
            double flat[2] = {0, 0}, aflat[2] = {0, 0}, along = 0, aalong = 0;
            auto each = [&](const std::function<void(size_t, size_t, double, const double*, const double*)>& fn) {
                for (size_t r = size_t(at[gr]); r < size_t(at[gr + 1]); ++r)
                    for (size_t c = q * d; c < (q + 1) * d; ++c) {
                        double xh[2], dy[2], yy[2];
                        for (int p = 0; p < 2; ++p) yy[p] = (x[(2 * r + p) * f + c] - mean[p]) / sd * w[c] + b[c];
                        const double open = !relu || yy[0] >= 0.0 ? 1.0 : 0.0;
                        for (int p = 0; p < 2; ++p) {
                            y[(2 * r + p) * f + c] = yy[p] * open;
                            ty[(2 * r + p) * f + c] = 8 * U * (std::fabs(yy[p] - b[c]) + std::fabs(b[c]));
                            xh[p] = ((held ? kept.values[(2 * r + p) * f + c] : double(x[(2 * r + p) * f + c])) - mean[p]) / sd;
                            dy[p] = g[(2 * r + p) * f + c] * open;
                        }
                        fn(r, c, open, xh, dy);
                    }
            };
            each([&](size_t, size_t c, double, const double* xh, const double* dy) {
                for (int p = 0; p < 2; ++p) {
                    flat[p] += w[c] * dy[p] / count; aflat[p] += std::fabs(w[c] * dy[p]) / count;
                    along += w[c] * dy[p] * xh[p] / count; aalong += std::fabs(w[c] * dy[p] * xh[p]) / count;
                    dw[c] += dy[p] * xh[p]; tw[c] += 8 * U * std::fabs(dy[p] * xh[p]);
                    db[c] += dy[p]; tb[c] += 4 * U * std::fabs(dy[p]);
                }
            });
            each([&](size_t r, size_t c, double, const double* xh, const double* dy) {
                for (int p = 0; p < 2; ++p) {
                    dx[(2 * r + p) * f + c] = (w[c] * dy[p] - flat[p] - xh[p] * along) / sd;
                    tdx[(2 * r + p) * f + c] = 20 * U * (std::fabs(w[c] * dy[p]) + aflat[p] + std::fabs(xh[p]) * aalong) / sd;
                }
            });
        }
    for (double* t : {ty.data(), tdx.data()}) for (size_t i = 0; i < ty.size(); ++i) t[i] += 1e-37;
    for (double& t : tw) t += 1e-37;
    for (double& t : tb) t += 1e-37;
    Dev<float> vx(x), vg(g), vw(w), vb(b), vy(2 * n * f), vdx(2 * n * f), vdw(f), vdb(f), stats(graphs * groups * MH_NORM_STATS);
    Dev<int32_t> vp(at);
    Dev<uint8_t> mask(n * f), codes(kept.codes.size()), scales(kept.scales.size());
    const size_t bytes = mh_group_norm_workspace_bytes(int64_t(n), int32_t(graphs), int32_t(f), int32_t(groups));
    Dev<uint8_t> ws(bytes);
    const int32_t* p = ptr.empty() ? nullptr : vp.p;
    const int64_t ld = int64_t(2 * f), im = int64_t(f);
    MH_CALL(mh_group_norm(vx.p, ld, im, int64_t(n), int32_t(f), int32_t(groups), p, int32_t(graphs), 1e-5f, vw.p, vb.p, relu, vy.p, ld, im,
                          relu ? mask.p : nullptr, held ? codes.p : nullptr, held ? scales.p : nullptr, stats.p, ws.p, bytes, stream));
    MH_CALL(mh_group_norm_bwd(held ? nullptr : vx.p, ld, im, held ? codes.p : nullptr, held ? scales.p : nullptr, held && relu ? mask.p : nullptr,
                              int64_t(n), int32_t(f), int32_t(groups), p, int32_t(graphs), stats.p, vw.p, vb.p, relu, vg.p, ld, im, vdx.p, ld, im,
                              vdw.p, vdb.p, ws.p, bytes, stream));
    HIP_OK(hipStreamSynchronize(stream));
    near_to(vy.get("result"), y, ty, "result");
    near_to(vdx.get("dx"), dx, tdx, "dx");
    near_to(vdw.get("dgamma"), dw, tw, "dgamma");
    near_to(vdb.get("dbeta"), db, tb, "dbeta");
    if (held) EXPECT(codes.get("codes") == kept.codes && scales.get("scales") == kept.scales, "checkpoint of the norm's input");
    if (relu && n) {
        const std::vector<uint8_t> m = mask.get("mask");
        for (size_t gr = 0; gr < graphs; ++gr)
            for (size_t r = size_t(at[gr]); r < size_t(at[gr + 1]); ++r)
                for (size_t c = 0; c < f; ++c) EXPECT((m[r * f + c] != 0) == (y[2 * r * f + c] != 0.0), "mask of row %zu", r);
    }
    (void)ws.get("workspace");
    (void)stats.get("stats");
}

// ---- class scores: [batch][classes][inner] or [inner][classes], float32 --------------------------------------------------
static void scores(hipStream_t stream, size_t batch, size_t inner, size_t c, bool by_class, size_t top, uint64_t seed) {
    Rng rng(seed);
    const size_t rows = batch * inner;
    const std::vector<float> x = rng.values(rows * c), gl = rng.values(rows), gh = rng.values(rows), gt = rng.values(rows * top);
    std::vector<int64_t> lab(rows);
    for (int64_t& l : lab) l = rng.uni() < 0.3 ? -100 : int64_t(rng.next() % c);
    if (rows) lab[0] = int64_t(c) - 1;
    const int64_t sb = by_class ? int64_t(c * inner) : 0, sc = by_class ? int64_t(inner) : 1, sn = by_class ? 1 : int64_t(c);
    auto place = [&](size_t r, size_t k) { return by_class ? r / inner * c * inner + k * inner + r % inner : r * c + k; };
    auto top_place = [&](size_t r, size_t k) { return by_class ? r / inner * top * inner + k * inner + r % inner : r * top + k; };
    std::vector<double> lp(rows), tlp(rows), ent(rows), tent(rows), tl(rows * top), ttl(rows * top), d(rows * c), td(rows * c), nd(rows * c), tnd(rows * c);
    std::vector<int64_t> ti(rows * top);
    double loss = 0.0, hits = 0.0, count = 0.0, tloss = 0.0;
    for (size_t r = 0; r < rows; ++r) count += lab[r] != -100;
    for (size_t r = 0; r < rows; ++r) {
        std::vector<double> p(c), l(c);
        std::vector<size_t> order(c);
        double m = -INFINITY, low = INFINITY, s = 0.0, h = 0.0, wide = 0.0;
        for (size_t k = 0; k < c; ++k) { m = std::max(m, double(x[place(r, k)])); low = std::min(low, double(x[place(r, k)])); }
        for (size_t k = 0; k < c; ++k) s += std::exp(double(x[place(r, k)]) - m);
        for (size_t k = 0; k < c; ++k) {
            order[k] = k;
            l[k] = double(x[place(r, k)]) - m - std::log(s);
            p[k] = std::exp(l[k]);
            h -= p[k] * l[k];
            wide += p[k] * (m - double(x[place(r, k)]));
        }
        std::stable_sort(order.begin(), order.end(), [&](size_t a, size_t b) { return x[place(r, a)] > x[place(r, b)]; });
        // e^x to 2 u, a sum of up to c terms, log to 2 u, the differences u each of what they subtract
        const double depth = double(c + 16) * U, spread = m - low + 1.0;
        const bool use = lab[r] != -100;
        lp[r] = use ? l[size_t(lab[r])] : 0.0;
        tlp[r] = depth + 4 * U * (std::fabs(lp[r]) + spread);
        ent[r] = h;
        tent[r] = (2 * depth + 8 * U) * (1.0 + h + wide);
        double a = use ? double(gl[r]) : 0.0, size = std::fabs(a);
        for (size_t k = 0; k < top; ++k) {
            const size_t at = top_place(r, k);
            ti[at] = int64_t(order[k]); tl[at] = l[order[k]];
            ttl[at] = depth + 4 * U * (std::fabs(tl[at]) + spread);
            a += gt[at]; size += std::fabs(double(gt[at]));
        }
        if (use) { loss -= lp[r] / count; tloss = std::max(tloss, tlp[r]); hits += order[0] == size_t(lab[r]); }
        for (size_t k = 0; k < c; ++k) {
            const size_t at = place(r, k);
            double own = use && size_t(lab[r]) == k ? double(gl[r]) : 0.0;
            for (size_t j = 0; j < top; ++j) own += order[j] == k ? double(gt[top_place(r, j)]) : 0.0;
            d[at] = own - p[k] * a - p[k] * (l[k] + h) * double(gh[r]);
            td[at] = 1e-37 + 2 * (depth + 4 * U * (spread + std::fabs(l[k])) + 24 * U) * (std::fabs(own) + size + p[k] * (std::fabs(l[k]) + h + 1) * std::fabs(double(gh[r])));
            nd[at] = use ? (p[k] - (size_t(lab[r]) == k ? 1.0 : 0.0)) / count : 0.0;
            tnd[at] = use ? 1e-37 + 2 * (depth + 8 * U + 4 * U * (spread + std::fabs(l[k]))) / count : 0.0;
        }
    }
    Dev<float> vx(x), vgl(gl), vgh(gh), vgt(gt), vlp(rows), vent(rows), stat(2 * rows), vtl(rows * top), vd(rows * c), vnd(rows * c), out(3), one(std::vector<float>{1.0f});
    Dev<int64_t> vlab(lab), vti(rows * top);
    const int64_t tb = by_class ? int64_t(top * inner) : 0, tk = by_class ? int64_t(inner) : 1, tn = by_class ? 1 : int64_t(top);
    const int64_t nb = int64_t(batch), ni = int64_t(inner);
    MH_CALL(mh_class_logprobs(vx.p, 0, nb, ni, int32_t(c), sb, sc, sn, vlab.p, -100, vlp.p, vent.p, stat.p, int32_t(top), vtl.p, vti.p, tb, tk, tn, stream));
    MH_CALL(mh_class_logprobs_bwd(vx.p, 0, nb, ni, int32_t(c), sb, sc, sn, vlab.p, -100, stat.p, vent.p, vgl.p, 1, vgh.p, 1, int32_t(top), vgt.p, vti.p,
                                  tb, tk, tn, vd.p, sb, sc, sn, stream));
    HIP_OK(hipStreamSynchronize(stream));
    near_to(vlp.get("logprob"), lp, tlp, "logprob");
    near_to(vent.get("entropy"), ent, tent, "entropy");
    near_to(vtl.get("top_logprob"), tl, ttl, "top_logprob");
    EXPECT(vti.get("top_index") == ti, "alternatives of %zu x %zu", rows, c);
    near_to(vd.get("d_scores"), d, td, "d_scores");
    (void)stat.get("stat");
    const size_t bytes = mh_class_nll_workspace_bytes(), kept = mh_class_nll_stat_bytes(nb, ni, int32_t(c), sc, sn);
    EXPECT(kept == 0 || kept == 8 * rows, "stat of %zu bytes", kept);
    Dev<uint8_t> ws(bytes), keep(kept);
    float* st = kept ? reinterpret_cast<float*>(keep.p) : nullptr;
    MH_CALL(mh_class_nll(vx.p, 0, nb, ni, int32_t(c), sb, sc, sn, vlab.p, -100, st, out.p, out.p + 1, out.p + 2, ws.p, bytes, stream));
    MH_CALL(mh_class_nll_bwd(vx.p, 0, nb, ni, int32_t(c), sb, sc, sn, vlab.p, -100, st, out.p + 2, one.p, vnd.p, sb, sc, sn, stream));
    HIP_OK(hipStreamSynchronize(stream));
    const std::vector<float> o = out.get("loss");
    if (rows) {
        EXPECT(std::fabs(double(o[0]) - loss) <= tloss + U * std::fabs(loss), "loss %.9g, %.9g expected", o[0], loss);
        EXPECT(o[1] == float(hits / count) && o[2] == float(1.0 / count), "accuracy %.9g of %.9g", o[1], hits / count);
    } else {
        EXPECT(std::isnan(o[0]) && std::isnan(o[1]), "loss of no rows");
    }
    near_to(vnd.get("d_scores of the loss"), nd, tnd, "d_scores of the loss");
    (void)keep.get("stat of the loss");
    (void)ws.get("workspace");
}

int main() {
    hipStream_t stream;
    HIP_OK(hipStreamCreate(&stream));
    struct { size_t n, m, k; } grams[] = {{0, 5, 3}, {1, 1, 1}, {3, 33, 2}, {67, 48, 16}, {501, 120, 30}, {1203, 40, 70}, {90, 300, 65}};
    for (const auto& s : grams) {
        printf("checkpoint %zu x %zu, %zu columns\n", s.n, s.m, s.k); fflush(stdout);
        checkpoints(stream, s.n, s.m, s.k, s.n + s.m);
    }
    struct { size_t n, f, groups; std::vector<int32_t> ptr; } batches[] = {
        {0, 8, 2, {}}, {1, 3, 3, {}}, {301, 20, 4, {}}, {130, 32, 4, {}}, {77, 65, 5, {}}, {200, 30, 5, {0, 0, 70, 71, 180}}, {40, 128, 8, {0, 40}}};
    for (const auto& s : batches)
        for (int kind = 0; kind < 4; ++kind) {
            printf("norm %zu x %zu, %zu groups, %zu borders, relu %d, 8 bits %d\n", s.n, s.f, s.groups, s.ptr.size(), kind & 1, kind >> 1); fflush(stdout);
            norms(stream, s.n, s.f, s.groups, s.ptr, kind & 1, kind >> 1, s.n + s.f);
        }
    struct { size_t batch, inner, c; bool by_class; size_t top; } reports[] = {
        {1, 0, 4, false, 2}, {1, 1, 1, false, 1}, {1, 300, 5, true, 2}, {1, 300, 5, false, 3}, {2, 131, 9, true, 4}, {1, 77, 65, false, 5}, {1, 40, 349, false, 16},
        {1, 9, 1100, false, 2}, {1, 7, 700, true, 1}, {1, 65537, 3, true, 1}, {3, 22001, 8, true, 0}};
    for (const auto& s : reports) {
        printf("scores %zu x %zu rows, %zu classes, class-major %d, top %zu\n", s.batch, s.inner, s.c, int(s.by_class), s.top); fflush(stdout);
        scores(stream, s.batch, s.inner, s.c, s.by_class, s.top, s.inner + s.c);
    }
    HIP_OK(hipStreamDestroy(stream));
    if (g_fail) { fprintf(stderr, "%d failures\n", g_fail); return 1; }
    printf("operators ok\n");
    fflush(stdout);
#ifdef ABI_SWEEP_SKIP_TEARDOWN
    _exit(0);                                     // host-sanitizer build: as in abi_sweep.cpp
#endif
    return 0;
}
