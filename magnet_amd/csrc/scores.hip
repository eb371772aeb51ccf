// Class scores -> log probabilities of given classes, entropy, top alternatives; mean negative log-likelihood and accuracy.
// One read of the scores per direction.
//
// For a row x[0..C):  m = max x,  s = sum e^(x-m),  w = sum e^(x-m) (x-m)
//     log p_c = (x_c - m) - log s          entropy H = log s - w / s
//     d log p_y / d x_c = [c = y] - p_c    d H / d x_c = -p_c (log p_c + H)
// (m, s, w) of two parts of a row join as  m' = max(m1, m2), s' = sum e^(mi-m') si, w' = sum e^(mi-m') (wi + si (mi-m')).
// All of it in 32 bits whatever the type of the scores, the sum over rows of the loss in 64.
//
// A row belongs to a group of `1 << ll` lanes, 64 >> ll rows to a wavefront.  Row-major scores: the lanes of a group are
// neighbours (consecutive classes are consecutive in memory); class-major scores: neighbouring lanes hold neighbouring rows
// and a group's lanes lie 64 >> ll apart.  A lane takes kPer classes at a time into registers (two passes over registers,
// none over memory), the joins are xor shuffles.  With few rows and many classes the waves of a workgroup share the rows'
// classes and join through LDS (JOIN).  Bound by the read of the scores; a short case by its two launches.
#include <cstdint>

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "common.h"

namespace {

constexpr int kBlock = 256;
constexpr int kPer = 8;                    // classes a lane holds at a time
constexpr int kMostTop = 16;
constexpr unsigned kMostBlocks = 2048;     // 8 workgroups of 4 waves per CU

__device__ inline float to_f(float v) { return v; }
__device__ inline float to_f(__hip_bfloat16 v) { return __bfloat162float(v); }
__device__ inline float to_f(__half v) { return __half2float(v); }
template <class T> __device__ inline T from_f(float v);
template <> __device__ inline float from_f<float>(float v) { return v; }
template <> __device__ inline __hip_bfloat16 from_f<__hip_bfloat16>(float v) { return __float2bfloat16(v); }
template <> __device__ inline __half from_f<__half>(float v) { return __float2half(v); }

// order-preserving integer of a float: NaN above everything (as torch's max and topk have it), -0 = +0, never 0
__device__ inline uint32_t order_key(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ inline float key_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? ((k == 0xffffffffu) ? 0x7fc00000u : (k ^ 0x80000000u)) : ~k);
}
// (value, class) as one integer: the larger value first, then the lower class
__device__ inline uint64_t candidate(float x, uint32_t c) { return (uint64_t(order_key(x)) << 32) | uint32_t(~c); }

struct Soft {
    float m = -INFINITY, s = 0.0f, w = 0.0f;
};

__device__ inline void join(Soft& a, const Soft& b) {
    const float m = fmaxf(a.m, b.m);
    const float da = a.m - m, db = b.m - m;
    const float ea = a.s == 0.0f ? 0.0f : expf(da), eb = b.s == 0.0f ? 0.0f : expf(db);
    // a part that has no weight left next to the other takes its (possibly infinite) exponent with it
    const float wa = ea == 0.0f ? 0.0f : ea * (a.w + a.s * da), wb = eb == 0.0f ? 0.0f : eb * (b.w + b.s * db);
    a.s = ea * a.s + eb * b.s;                                      // a NaN in s stays, whatever its part's maximum
    a.w = wa + wb;
    a.m = m;
}

__device__ inline Soft of_values(const float (&x)[kPer]) {
    Soft r;
#pragma unroll
    for (int j = 0; j < kPer; ++j) r.m = fmaxf(r.m, x[j]);
    const float m = r.m == -INFINITY ? 0.0f : r.m;     // nothing but -inf: the sums stay 0 (and NaN stays NaN)
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const float t = x[j] - m, e = expf(t);
        r.s += e;
        r.w += e == 0.0f ? 0.0f : e * t;
    }
    return r;
}

template <int N>
struct TopList {                            // the N best candidates, best first
    uint64_t v[N > 0 ? N : 1];
    __device__ TopList() {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = 0;
    }
    __device__ void add(uint64_t c) {
        if (N > 0 && c > v[N > 0 ? N - 1 : 0]) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const uint64_t hi = c > v[i] ? c : v[i];
                c = c > v[i] ? v[i] : c;
                v[i] = hi;
            }
        }
    }
    __device__ void pop() {
#pragma unroll
        for (int i = 0; i + 1 < N; ++i) v[i] = v[i + 1];
        if (N > 0) v[N > 0 ? N - 1 : 0] = 0;
    }
};

struct ScoreArgs {
    const void* x;
    int64_t rows, inner, sb, sc, sn;        // rows = batches * inner; strides in elements
    int32_t classes;
    int32_t ll;                             // log2 of the lanes of a row
    int32_t by_class;                       // neighbouring lanes hold neighbouring rows
    const int64_t* labels;
    int64_t ignore;
    float2* stat;                           // (m, log s) of every row, for the backward pass
    // report
    float *logprob, *entropy, *top_lp;
    int64_t* top_idx;
    int32_t top;
    int64_t tb, tk, tn;
    // loss
    double* partial;                        // [workgroups][3]: sum of log p, rows counted, rows hit
};

__device__ inline void place(const ScoreArgs& a, int64_t row, int64_t& b, int64_t& i) {
    b = a.rows == a.inner ? 0 : row / a.inner;
    i = row - b * a.inner;
}

template <class T, int TOPN, bool NLL, bool JOIN>
__global__ void __launch_bounds__(kBlock) score_rows(const ScoreArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int rows_of_wave = 64 >> a.ll, lanes = 1 << a.ll;
    const int r = a.by_class ? lane & (rows_of_wave - 1) : lane >> a.ll;
    const int l = a.by_class ? lane >> (6 - a.ll) : lane & (lanes - 1);
    const int near = a.by_class ? rows_of_wave : 1;                 // distance of two neighbours of a group
    const int waves = kBlock / 64;
    const int64_t step = int64_t(rows_of_wave) * (JOIN ? 1 : waves) * gridDim.x;
    const int64_t first = (int64_t(blockIdx.x) * (JOIN ? 1 : waves) + (JOIN ? 0 : wave)) * rows_of_wave;
    double sum = 0.0;
    int32_t used = 0, hits = 0;
    // every lane of a wave makes the same number of turns: a row past the end only takes part in the shuffles
    for (int64_t row0 = first; row0 < a.rows; row0 += step) {
        const int64_t row = row0 + r;
        const bool live = row < a.rows;
        int64_t b = 0, i = 0;
        if (live) place(a, row, b, i);
        const T* x = static_cast<const T*>(a.x) + b * a.sb + i * a.sn;
        Soft acc;
        TopList<TOPN> best;
        for (int32_t c0 = JOIN ? wave * kPer * lanes : 0; c0 < a.classes; c0 += kPer * lanes * (JOIN ? waves : 1)) {
            float v[kPer];
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const int32_t c = c0 + j * lanes + l;
                v[j] = live && c < a.classes ? to_f(x[c * a.sc]) : -INFINITY;
            }
            join(acc, of_values(v));
            if (TOPN > 0) {
#pragma unroll
                for (int j = 0; j < kPer; ++j) {
                    const int32_t c = c0 + j * lanes + l;
                    if (c < a.classes) best.add(candidate(v[j], uint32_t(c)));
                }
            }
        }
        for (int o = near; o < near * lanes; o <<= 1) {
            Soft other;
            other.m = __shfl_xor(acc.m, o); other.s = __shfl_xor(acc.s, o); other.w = __shfl_xor(acc.w, o);
            join(acc, other);
        }
        if (JOIN) {
            __shared__ float soft[kBlock / 64][64][3];
            __shared__ uint64_t lists[TOPN > 0 ? kBlock / 64 : 1][64][TOPN > 0 ? TOPN : 1];
            __syncthreads();                                       // the turn before has been read
            soft[wave][lane][0] = acc.m; soft[wave][lane][1] = acc.s; soft[wave][lane][2] = acc.w;
#pragma unroll
            for (int t = 0; t < TOPN; ++t) lists[wave][lane][t] = best.v[t];
            __syncthreads();
            if (wave == 0) {
                for (int v = 1; v < waves; ++v) {
                    Soft other;
                    other.m = soft[v][lane][0]; other.s = soft[v][lane][1]; other.w = soft[v][lane][2];
                    join(acc, other);
#pragma unroll
                    for (int t = 0; t < TOPN; ++t) best.add(lists[v][lane][t]);
                }
            }
        }
        if (JOIN && wave != 0) continue;                           // waves leave the turn together: row0 is the workgroup's
        const float log_s = logf(acc.s);
        const bool writes = live && l == 0;
        float lp = 0.0f;
        int64_t label = 0;
        bool counted = false;
        if (writes && a.labels) {
            label = a.labels[row];
            counted = label != a.ignore;
            if (counted) lp = label >= 0 && label < a.classes ? (to_f(x[label * a.sc]) - acc.m) - log_s : NAN;
        }
        if (writes && a.stat) a.stat[row] = make_float2(acc.m, log_s);
        if (NLL) {
            uint64_t top1 = best.v[0];
            for (int o = near; o < near * lanes; o <<= 1) {
                const uint64_t other = __shfl_xor(static_cast<unsigned long long>(top1), o);
                top1 = other > top1 ? other : top1;
            }
            if (counted) {
                sum += double(lp);
                ++used;
                hits += int64_t(uint32_t(~uint32_t(top1))) == label;
            }
        } else {
            if (writes) {
                if (a.logprob) a.logprob[row] = lp;
                a.entropy[row] = log_s - acc.w / acc.s;
            }
            if (TOPN > 0) {
                for (int t = 0; t < a.top; ++t) {
                    uint64_t top1 = best.v[0];
                    for (int o = near; o < near * lanes; o <<= 1) {
                        const uint64_t other = __shfl_xor(static_cast<unsigned long long>(top1), o);
                        top1 = other > top1 ? other : top1;
                    }
                    if (best.v[0] == top1) best.pop();             // one lane holds it: a candidate carries its class
                    if (writes) {
                        const int64_t at = b * a.tb + t * a.tk + i * a.tn;
                        a.top_idx[at] = int64_t(uint32_t(~uint32_t(top1)));
                        a.top_lp[at] = (key_value(uint32_t(top1 >> 32)) - acc.m) - log_s;
                    }
                }
            }
        }
    }
    if (NLL) {
        __shared__ double part[kBlock / 64][3];
        double n = double(used), h = double(hits);
        for (int o = 32; o > 0; o >>= 1) { sum += __shfl_xor(sum, o); n += __shfl_xor(n, o); h += __shfl_xor(h, o); }
        if (lane == 0) { part[wave][0] = sum; part[wave][1] = n; part[wave][2] = h; }
        __syncthreads();
        if (threadIdx.x < 3) {
            double t = 0.0;
            for (int v = 0; v < waves; ++v) t += part[v][threadIdx.x];
            a.partial[int64_t(blockIdx.x) * 3 + threadIdx.x] = t;
        }
    }
}

// loss, accuracy and 1 / rows counted from the workgroups' sums, in a fixed order
__global__ void __launch_bounds__(kBlock) nll_finish(const double* __restrict__ partial, int n, float* loss, float* accuracy, float* inv_count) {
    __shared__ double part[kBlock / 64][3];
    double t[3] = {0.0, 0.0, 0.0};
    for (int i = threadIdx.x; i < n; i += kBlock)
        for (int k = 0; k < 3; ++k) t[k] += partial[int64_t(i) * 3 + k];
    for (int k = 0; k < 3; ++k) {
        for (int o = 32; o > 0; o >>= 1) t[k] += __shfl_xor(t[k], o);
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6][k] = t[k];
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int v = 1; v < kBlock / 64; ++v)
            for (int k = 0; k < 3; ++k) part[0][k] += part[v][k];
        *loss = float(-part[0][0] / part[0][1]);
        *accuracy = float(part[0][2] / part[0][1]);
        *inv_count = float(1.0 / part[0][1]);
    }
}

struct GradArgs {
    const void* x;
    void* d;
    int64_t rows, inner, sb, sc, sn, db, dc, dn;
    int32_t classes, ll, by_class;
    const int64_t* labels;
    int64_t ignore;
    const float2* stat;
    const float *entropy, *g_lp, *g_h, *g_top, *g_loss, *inv_count;
    int64_t g_lp_s, g_h_s;                  // 0: one value for every row
    const int64_t* top_idx;
    int32_t top;
    int64_t tb, tk, tn;
};

// d x_c = [c = y] g_y + sum_t [c = i_t] g_t - p_c (g_y + sum_t g_t) - p_c (log p_c + H) g_H
template <class T, bool NLL>
__global__ void __launch_bounds__(kBlock) score_grads(const GradArgs a) {
    const int lane = threadIdx.x & 63;
    const int rows_of_wave = 64 >> a.ll, lanes = 1 << a.ll;
    const int r = a.by_class ? lane & (rows_of_wave - 1) : lane >> a.ll;
    const int l = a.by_class ? lane >> (6 - a.ll) : lane & (lanes - 1);
    const int waves = kBlock / 64;
    const int64_t step = int64_t(rows_of_wave) * waves * gridDim.x;
    const float scale = NLL ? -a.g_loss[0] * a.inv_count[0] : 0.0f;
    for (int64_t row = (int64_t(blockIdx.x) * waves + (threadIdx.x >> 6)) * rows_of_wave + r; row < a.rows; row += step) {
        const int64_t b = a.rows == a.inner ? 0 : row / a.inner, i = row - b * a.inner;
        const T* x = static_cast<const T*>(a.x) + b * a.sb + i * a.sn;
        T* d = static_cast<T*>(a.d) + b * a.db + i * a.dn;
        const int64_t label = a.labels ? a.labels[row] : a.ignore;
        const bool counted = a.labels && label != a.ignore;
        float gy = !counted ? 0.0f : NLL ? scale : a.g_lp ? a.g_lp[row * a.g_lp_s] : 0.0f;
        if (counted && (label < 0 || label >= a.classes)) gy = NAN;      // as its log probability
        const float gh = !NLL && a.g_h ? a.g_h[row * a.g_h_s] : 0.0f;
        const float h = !NLL && a.g_h ? a.entropy[row] : 0.0f;
        float all = gy;
        bool any = gy != 0.0f || gh != 0.0f;
        const int64_t at = b * a.tb + i * a.tn;
        if (!NLL && a.g_top)
            for (int t = 0; t < a.top; ++t) {
                const float g = a.g_top[at + t * a.tk];
                all += g;
                any |= g != 0.0f;
            }
        const float2 st = a.stat[row];
        for (int32_t c0 = l; c0 < a.classes; c0 += kPer * lanes) {
            float v[kPer];
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const int32_t c = c0 + j * lanes;
                if (c < a.classes) v[j] = to_f(x[c * a.sc]);
            }
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const int32_t c = c0 + j * lanes;
                if (c < a.classes) {
                    float g = 0.0f;                                  // a row no gradient reaches stays clean whatever it holds
                    if (any) {
                        const float lp = (v[j] - st.x) - st.y, p = expf(lp);
                        g = (c == label && counted ? gy : 0.0f) - p * all;
                        if (!NLL && a.g_h) g -= p == 0.0f ? 0.0f : p * (lp + h) * gh;
                        if (!NLL && a.g_top)
                            for (int t = 0; t < a.top; ++t)
                                if (a.top_idx[at + t * a.tk] == c) g += a.g_top[at + t * a.tk];
                    }
                    d[c * a.dc] = from_f<T>(g);
                }
            }
        }
    }
}

struct Shape {
    int ll, by_class;
    bool join;
    unsigned blocks;
};

// Lanes of a row.  Row-major: as many as hold the row at kPer classes each (fewer joins, whole lines read once), at most a
// wavefront.  Class-major: one, unless there are too few rows to fill the GPU.  A workgroup joins on its rows when even
// whole wavefronts per row are too few for the GPU and every wave gets classes.
Shape shape_of(int64_t rows, int32_t classes, int64_t sc, int64_t sn, bool can_join) {
    Shape s;
    s.by_class = sc > sn && sn != 0;
    const int64_t fill = int64_t(256) * 8 * 64;            // two waves per SIMD
    s.ll = 0;
    while (s.ll < 6 && (int64_t(kPer) << s.ll) < classes && (!s.by_class || (rows << s.ll) < fill)) ++s.ll;
    const int64_t tiles = (rows + (64 >> s.ll) - 1) / (64 >> s.ll);
    s.join = can_join && s.ll == 6 && tiles < 1024 && classes > 2 * kPer * 64;
    const int64_t b = s.join ? tiles : (tiles + kBlock / 64 - 1) / (kBlock / 64);
    s.blocks = unsigned(b < 1 ? 1 : b > kMostBlocks ? kMostBlocks : b);
    return s;
}

template <class T, int TOPN, bool NLL>
void launch_rows(const ScoreArgs& a, const Shape& s, hipStream_t stream) {
    if (s.join) score_rows<T, TOPN, NLL, true><<<s.blocks, kBlock, 0, stream>>>(a);
    else score_rows<T, TOPN, NLL, false><<<s.blocks, kBlock, 0, stream>>>(a);
}

template <class T>
void launch_report(const ScoreArgs& a, const Shape& s, hipStream_t stream) {
    if (a.top == 0) launch_rows<T, 0, false>(a, s, stream);
    else if (a.top <= 2) launch_rows<T, 2, false>(a, s, stream);
    else if (a.top <= 8) launch_rows<T, 8, false>(a, s, stream);
    else launch_rows<T, kMostTop, false>(a, s, stream);
}

int check_scores(const void* x, int dtype, int64_t n_batch, int64_t n_inner, int32_t classes, int64_t sb, int64_t sc, int64_t sn) {
    MH_REQUIRE(dtype >= 0 && dtype <= 2, "dtype=%d: 0 (float32), 1 (bfloat16) and 2 (float16) are known", dtype);
    MH_REQUIRE(n_batch >= 0 && n_inner >= 0 && classes >= 1, "n_batch=%lld n_inner=%lld classes=%d", (long long)n_batch, (long long)n_inner, classes);
    MH_REQUIRE(sb >= 0 && sc >= 0 && sn >= 0, "negative stride");
    MH_REQUIRE(n_batch == 0 || n_inner == 0 || x, "scores is null");
    return MH_OK;
}

}  // namespace

extern "C" int mh_class_logprobs(const void* scores, int dtype, int64_t n_batch, int64_t n_inner, int32_t classes, int64_t sb,
                                 int64_t sc, int64_t sn, const int64_t* labels, int64_t ignore, float* logprob, float* entropy,
                                 float* stat, int32_t top, float* top_logprob, int64_t* top_index, int64_t tb, int64_t tk,
                                 int64_t tn, void* stream_) {
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    if (int rc = check_scores(scores, dtype, n_batch, n_inner, classes, sb, sc, sn)) return rc;
    MH_REQUIRE(top >= 0 && top <= kMostTop && top <= classes, "top=%d: at most %d and the number of classes (%d)", top, kMostTop, classes);
    const int64_t rows = n_batch * n_inner;
    if (rows == 0) return MH_OK;
    MH_REQUIRE(entropy && (!labels || logprob) && (top == 0 || (top_logprob && top_index)), "null output");
    MH_REQUIRE(tb >= 0 && tk >= 0 && tn >= 0, "negative stride");
    ScoreArgs a{};
    a.x = scores; a.rows = rows; a.inner = n_inner; a.sb = sb; a.sc = sc; a.sn = sn; a.classes = classes;
    a.labels = labels; a.ignore = ignore; a.stat = reinterpret_cast<float2*>(stat);
    a.logprob = labels ? logprob : nullptr; a.entropy = entropy; a.top_lp = top_logprob; a.top_idx = top_index; a.top = top;
    a.tb = tb; a.tk = tk; a.tn = tn;
    const Shape s = shape_of(rows, classes, sc, sn, true);
    a.ll = s.ll; a.by_class = s.by_class;
    if (dtype == 0) launch_report<float>(a, s, stream);
    else if (dtype == 1) launch_report<__hip_bfloat16>(a, s, stream);
    else launch_report<__half>(a, s, stream);
    MH_LAUNCH_CHECK("class_logprobs");
    return MH_OK;
}

extern "C" int mh_class_logprobs_bwd(const void* scores, int dtype, int64_t n_batch, int64_t n_inner, int32_t classes, int64_t sb,
                                     int64_t sc, int64_t sn, const int64_t* labels, int64_t ignore, const float* stat,
                                     const float* entropy, const float* g_logprob, int64_t g_logprob_stride,
                                     const float* g_entropy, int64_t g_entropy_stride, int32_t top, const float* g_top,
                                     const int64_t* top_index, int64_t tb, int64_t tk, int64_t tn, void* d_scores, int64_t db,
                                     int64_t dc, int64_t dn, void* stream_) {
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    if (int rc = check_scores(scores, dtype, n_batch, n_inner, classes, sb, sc, sn)) return rc;
    MH_REQUIRE(top >= 0 && top <= kMostTop && top <= classes, "top=%d: at most %d and the number of classes (%d)", top, kMostTop, classes);
    const int64_t rows = n_batch * n_inner;
    if (rows == 0) return MH_OK;
    MH_REQUIRE(stat && d_scores && (!g_logprob || labels) && (!g_entropy || entropy) && (!g_top || top == 0 || top_index), "null pointer");
    MH_REQUIRE(db >= 0 && dc >= 0 && dn >= 0 && tb >= 0 && tk >= 0 && tn >= 0 && g_logprob_stride >= 0 && g_entropy_stride >= 0, "negative stride");
    GradArgs a{};
    a.x = scores; a.d = d_scores; a.rows = rows; a.inner = n_inner; a.sb = sb; a.sc = sc; a.sn = sn; a.db = db; a.dc = dc; a.dn = dn;
    a.classes = classes; a.labels = g_logprob ? labels : nullptr; a.ignore = ignore; a.stat = reinterpret_cast<const float2*>(stat);
    a.entropy = entropy; a.g_lp = g_logprob; a.g_lp_s = g_logprob_stride; a.g_h = g_entropy; a.g_h_s = g_entropy_stride;
    a.g_top = top ? g_top : nullptr; a.top_idx = top_index; a.top = top; a.tb = tb; a.tk = tk; a.tn = tn;
    const Shape s = shape_of(rows, classes, sc, sn, false);
    a.ll = s.ll; a.by_class = s.by_class;
    if (dtype == 0) score_grads<float, false><<<s.blocks, kBlock, 0, stream>>>(a);
    else if (dtype == 1) score_grads<__hip_bfloat16, false><<<s.blocks, kBlock, 0, stream>>>(a);
    else score_grads<__half, false><<<s.blocks, kBlock, 0, stream>>>(a);
    MH_LAUNCH_CHECK("class_logprobs_bwd");
    return MH_OK;
}

extern "C" size_t mh_class_nll_workspace_bytes(void) { return size_t(kMostBlocks) * 3 * sizeof(double); }

extern "C" int mh_class_nll(const void* scores, int dtype, int64_t n_batch, int64_t n_inner, int32_t classes, int64_t sb, int64_t sc,
                            int64_t sn, const int64_t* labels, int64_t ignore, float* stat, float* loss, float* accuracy,
                            float* inv_count, void* workspace, size_t workspace_bytes, void* stream_) {
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    if (int rc = check_scores(scores, dtype, n_batch, n_inner, classes, sb, sc, sn)) return rc;
    const int64_t rows = n_batch * n_inner;
    MH_REQUIRE(loss && accuracy && inv_count && (rows == 0 || (labels && workspace)), "null pointer");
    if (rows > 0 && workspace_bytes < mh_class_nll_workspace_bytes())
        return mh::fail(MH_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, mh_class_nll_workspace_bytes());
    unsigned blocks = 0;
    ScoreArgs a{};
    a.partial = static_cast<double*>(workspace);
    if (rows > 0) {
        a.x = scores; a.rows = rows; a.inner = n_inner; a.sb = sb; a.sc = sc; a.sn = sn; a.classes = classes;
        a.labels = labels; a.ignore = ignore; a.stat = reinterpret_cast<float2*>(stat);
        const Shape s = shape_of(rows, classes, sc, sn, true);
        a.ll = s.ll; a.by_class = s.by_class;
        blocks = s.blocks;
        if (dtype == 0) launch_rows<float, 1, true>(a, s, stream);
        else if (dtype == 1) launch_rows<__hip_bfloat16, 1, true>(a, s, stream);
        else launch_rows<__half, 1, true>(a, s, stream);
        MH_LAUNCH_CHECK("class_nll");
    }
    nll_finish<<<1, kBlock, 0, stream>>>(a.partial, int(blocks), loss, accuracy, inv_count);
    MH_LAUNCH_CHECK("nll_finish");
    return MH_OK;
}

extern "C" int mh_class_nll_bwd(const void* scores, int dtype, int64_t n_batch, int64_t n_inner, int32_t classes, int64_t sb,
                                int64_t sc, int64_t sn, const int64_t* labels, int64_t ignore, const float* stat,
                                const float* inv_count, const float* g_loss, void* d_scores, int64_t db, int64_t dc, int64_t dn,
                                void* stream_) {
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    if (int rc = check_scores(scores, dtype, n_batch, n_inner, classes, sb, sc, sn)) return rc;
    const int64_t rows = n_batch * n_inner;
    if (rows == 0) return MH_OK;
    MH_REQUIRE(labels && stat && inv_count && g_loss && d_scores, "null pointer");
    MH_REQUIRE(db >= 0 && dc >= 0 && dn >= 0, "negative stride");
    GradArgs a{};
    a.x = scores; a.d = d_scores; a.rows = rows; a.inner = n_inner; a.sb = sb; a.sc = sc; a.sn = sn; a.db = db; a.dc = dc; a.dn = dn;
    a.classes = classes; a.labels = labels; a.ignore = ignore; a.stat = reinterpret_cast<const float2*>(stat);
    a.g_loss = g_loss; a.inv_count = inv_count;
    const Shape s = shape_of(rows, classes, sc, sn, false);
    a.ll = s.ll; a.by_class = s.by_class;
    if (dtype == 0) score_grads<float, true><<<s.blocks, kBlock, 0, stream>>>(a);
    else if (dtype == 1) score_grads<__hip_bfloat16, true><<<s.blocks, kBlock, 0, stream>>>(a);
    else score_grads<__half, true><<<s.blocks, kBlock, 0, stream>>>(a);
    MH_LAUNCH_CHECK("class_nll_bwd");
    return MH_OK;
}
