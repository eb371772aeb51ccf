// Class scores -> log probabilities of given classes, entropy, top alternatives; mean negative log-likelihood and accuracy.
// One read of the scores per direction.
//
// For a row x[0..C):  m = max x,  s = sum e^(x-m),  w = sum e^(x-m) (x-m)
//     log p_c = (x_c - m) - log s          entropy H = log s - w / s
//     d log p_y / d x_c = [c = y] - p_c    d H / d x_c = -p_c (log p_c + H)
// (m, s, w) of a part of a row go to a larger maximum m' as  s' = e^(m-m') s, w' = e^(m-m') (w + s (m - m')), and then add.
// All of it in 32 bits whatever the type of the scores, the sum over rows of the loss in 64.
//
// A row belongs to a group of `1 << ll` lanes, 64 >> ll rows to a wavefront.  Row-major scores: the lanes of a group are
// neighbours (consecutive classes are consecutive in memory); class-major scores: neighbouring lanes hold neighbouring rows
// and a group's lanes lie 64 >> ll apart.  A lane takes kPer classes at a time into registers (two passes over registers,
// none over memory), the joins are xor shuffles.  With few rows and many classes the waves of a workgroup share the rows'
// classes and join through LDS (JOIN).  Bound by the read of the scores; a short case by its two launches.
#include <cstdint>
#include <type_traits>

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "common.h"

namespace {

constexpr int kBlock = 256;
constexpr int kPer = 8;                    // classes a lane holds at a time
constexpr int kMore = 24;                  // the same where a row of more than 64 classes fits a few lanes that way
constexpr int kMostTop = 16;
constexpr int32_t kMostClasses = 1 << 24;
constexpr int64_t kMostRows = int64_t(1) << 40;               // of all batches
constexpr unsigned kMostSums = 2048;       // workgroups that leave a partial sum of the loss: 8 of 4 waves for each CU
constexpr unsigned kMostBlocks = 1u << 20;

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

// e^x for a sum over a row's classes: x <= 0, and what |x| costs its accuracy (|x| 2^-23 of itself) its share of the sum forgives
__device__ inline float weight(float x) { return __expf(x); }
// e^x to 2 units in the last place however far x lies below 0, for a probability that is an answer by itself (a gradient's element):
// h = fl(x log2 e) is short of x log2 e by r, at most 2^-17, which two fused products give back: e^x = 2^h 2^r = 2^h (1 + r ln 2).
// Three instructions more (gradient of 60k x 349 bf16: 26.4 -> 30.7 us, of the loss of 2M x 5: 16.1 -> 16.4).
__device__ inline float accurate_weight(float x) {
    constexpr float kLog2e = 1.44269504f, kLog2eRest = 1.92596303e-8f, kLn2 = 0.693147181f;
    const float h = x * kLog2e, r = fmaf(x, kLog2eRest, fmaf(x, kLog2e, -h)), e = __builtin_amdgcn_exp2f(h);
    return fmaf(e, r * kLn2, e);
}

constexpr float kLowest = -200.0f;         // below the logarithm of the smallest weight

// (m, s, w) of a part of a row
struct Soft {
    float m = -INFINITY, s = 0.0f, w = 0.0f;
    // to a maximum that is no less; a part without weight takes its infinite exponent with it, a NaN in s stays
    __device__ void raise(float to) {
        const float d = m - to, e = s == 0.0f ? 0.0f : weight(d);
        w = e == 0.0f ? 0.0f : e * (w + s * d);
        s = e * s;
        m = to;
    }
    __device__ void join(Soft o) {
        const float to = fmaxf(m, o.m);
        raise(to);
        o.raise(to);
        s += o.s;
        w += o.w;
    }
    // values below or at the maximum
    template <int P>
    __device__ void add(const float (&x)[P]) {
        const float from = m == -INFINITY ? 0.0f : m;          // nothing but -inf: the sums stay 0 (and NaN stays NaN)
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const float t = x[j] - from, e = weight(t);
            s += e;
            w = fmaf(e, fmaxf(t, kLowest), w);                  // no weight, no infinity to multiply (NaN stays by e)
        }
    }
};

template <int P>
__device__ inline float largest(const float (&x)[P]) {
    float m = x[0];
#pragma unroll
    for (int j = 1; j < P; ++j) m = fmaxf(m, x[j]);
    return m == m ? m : -INFINITY;                              // nothing but NaN
}

// Sum, maximum and minimum over the lanes of a group: over a whole wavefront or 16 neighbours by data-parallel moves (six or four
// instructions, no LDS), else by xor shuffles.
template <int CTRL, int ROWS>
__device__ inline uint32_t moved(uint32_t v, uint32_t idle) { return uint32_t(__builtin_amdgcn_update_dpp(int(idle), int(v), CTRL, ROWS, 0xf, false)); }
struct Add { static __device__ uint32_t of(uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); } };
struct MaxF { static __device__ uint32_t of(uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); } };
struct MaxU { static __device__ uint32_t of(uint32_t a, uint32_t b) { return a > b ? a : b; } };
struct MinU { static __device__ uint32_t of(uint32_t a, uint32_t b) { return a < b ? a : b; } };

struct Group {
    int lanes, near;                        // lanes of a row, distance of two neighbours
    template <class Op>
    __device__ uint32_t fold(uint32_t v, uint32_t idle) const {
        if (lanes == 64) {                  // shift by 1, 2, 4, 8 inside rows of 16, then across them; lane 63 has it all
            v = Op::of(v, moved<0x111, 0xf>(v, idle)); v = Op::of(v, moved<0x112, 0xf>(v, idle)); v = Op::of(v, moved<0x114, 0xf>(v, idle));
            v = Op::of(v, moved<0x118, 0xf>(v, idle)); v = Op::of(v, moved<0x142, 0xa>(v, idle)); v = Op::of(v, moved<0x143, 0xc>(v, idle));
            return uint32_t(__builtin_amdgcn_readlane(int(v), 63));
        }
        if (lanes == 16 && near == 1) {     // rotate by 8, 4, 2, 1
            v = Op::of(v, moved<0x128, 0xf>(v, idle)); v = Op::of(v, moved<0x124, 0xf>(v, idle));
            v = Op::of(v, moved<0x122, 0xf>(v, idle)); return Op::of(v, moved<0x121, 0xf>(v, idle));
        }
        for (int o = near; o < near * lanes; o <<= 1) v = Op::of(v, uint32_t(__shfl_xor(int(v), o)));
        return v;
    }
    __device__ float sum(float x) const { return __uint_as_float(fold<Add>(__float_as_uint(x), 0u)); }
    __device__ float max(float x) const { return __uint_as_float(fold<MaxF>(__float_as_uint(x), 0xff800000u)); }
    __device__ uint64_t max(uint64_t x) const {
        for (int o = near; o < near * lanes; o <<= 1) {
            const uint64_t other = __shfl_xor(static_cast<unsigned long long>(x), o);
            x = other > x ? other : x;
        }
        return x;
    }
};

// The best candidate of a row whose keys all lie in registers (class j * lanes + l, key 0: none), taken out of them: the largest key,
// then the first class that has it
template <int P>
__device__ inline uint64_t take_best(uint32_t (&key)[P], const Group& g, int l) {
    uint32_t best = key[0];
    int at = 0;
#pragma unroll
    for (int j = 1; j < P; ++j) {
        at = key[j] > best ? j : at;
        best = MaxU::of(best, key[j]);
    }
    const uint32_t top = g.fold<MaxU>(best, 0u), mine = best == top ? uint32_t(at * g.lanes + l) : ~0u;
    const uint32_t c = g.fold<MinU>(mine, ~0u);
    at = mine == c ? at : -1;
#pragma unroll
    for (int j = 0; j < P; ++j) key[j] = j == at ? 0u : key[j];
    return (uint64_t(top) << 32) | uint32_t(~c);
}

// Scores of 16 bits whose classes all lie in registers: order and class fit 32 bits, distinct in a row, and nothing needs to be taken
// out.  Of the keys below the last best, the nearest has the largest difference to it modulo 2^32 (those above it have the
// smallest): a subtraction and half a maximum of three for each class, where taking the best out costs five instructions.
__device__ inline uint32_t short_bits(float x, __hip_bfloat16) { return __float_as_uint(x) >> 16; }
__device__ inline uint32_t short_bits(float x, __half) { return __half_as_ushort(__float2half(x)); }
__device__ inline uint32_t short_bits(float, float) { return 0u; }
template <class T>
__device__ inline uint32_t short_key(float x, uint32_t c, bool clean) {              // clean: no NaN in the row
    const float y = x + 0.0f;
    const uint32_t u = sizeof(T) == 2 && std::is_same_v<T, __hip_bfloat16> ? __float_as_uint(y) : short_bits(y, T()) << 16;
    uint32_t k = u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u);
    if (!clean && x != x) k = 0xffffffffu;
    return (k & 0xffff0000u) | (0xffffu - c);
}
template <class T> __device__ inline float short_value(uint32_t key) {
    const uint32_t k = key >> 16, b = (k & 0x8000u) ? k ^ 0x8000u : k ^ 0xffffu;
    return to_f(__builtin_bit_cast(T, uint16_t(b)));
}
template <> __device__ inline float short_value<float>(uint32_t) { return 0.0f; }
template <int P>
__device__ inline uint32_t next_below(const uint32_t (&key)[P], uint32_t last, const Group& g) {
    uint32_t t = key[0] - last;
#pragma unroll
    for (int j = 1; j < P; ++j) t = MaxU::of(t, key[j] - last);
    return last + g.fold<MaxU>(t, 0u);
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

// a workgroup's share of the loss
__device__ inline void leave_sums(double* partial, double sum, double n, double h) {
    __shared__ double part[kBlock / 64][3];
    for (int o = 32; o > 0; o >>= 1) { sum += __shfl_xor(sum, o); n += __shfl_xor(n, o); h += __shfl_xor(h, o); }
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) { part[wave][0] = sum; part[wave][1] = n; part[wave][2] = h; }
    __syncthreads();
    if (threadIdx.x < 3) {
        double t = 0.0;
        for (int v = 0; v < kBlock / 64; ++v) t += part[v][threadIdx.x];
        partial[int64_t(blockIdx.x) * 3 + threadIdx.x] = t;
    }
}

// ONE: a row's classes fit its lanes' registers, and the best are taken from there.  Else a lane keeps a list of its TOPN best.
// UNIT: 16 lanes to a row and classes one behind the other, known when compiled: offsets become part of the load instructions.
template <class T, int P, int TOPN, bool NLL, bool ONE, bool JOIN, bool UNIT>
__global__ void __launch_bounds__(kBlock) score_rows(const ScoreArgs a) {
    constexpr bool kShort = sizeof(T) == 2 && kMore * 64 <= 0x10000;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int ll = UNIT ? 4 : a.ll, rows_of_wave = 64 >> ll, lanes = 1 << ll;
    const bool by_class = !UNIT && a.by_class;
    const int64_t sc = UNIT ? 1 : a.sc;
    const int r = by_class ? lane & (rows_of_wave - 1) : lane >> ll;
    const int l = by_class ? lane >> (6 - ll) : lane & (lanes - 1);
    const Group group{lanes, by_class ? rows_of_wave : 1};
    const int waves = kBlock / 64;
    const int64_t step = int64_t(rows_of_wave) * (JOIN ? 1 : waves) * gridDim.x;
    const int64_t first = (int64_t(blockIdx.x) * (JOIN ? 1 : waves) + (JOIN ? 0 : wave)) * rows_of_wave;
    const bool wanted = NLL || a.top > 0;                          // of the best classes
    double sum = 0.0;
    int32_t used = 0, hits = 0;
    // every lane of a wave makes the same number of turns: a row past the end only takes part in the exchanges
    for (int64_t row0 = first; row0 < a.rows; row0 += step) {
        const int64_t row = row0 + r;
        const bool live = row < a.rows;
        int64_t b = 0, i = 0;
        if (live) place(a, row, b, i);
        const T* x = static_cast<const T*>(a.x) + b * a.sb + i * a.sn;      // past the end: the first row
        const bool writes = live && l == 0;
        const int64_t label = writes && a.labels ? a.labels[row] : 0;
        Soft acc;
        TopList<TOPN> best;
        uint32_t key[P], last = 0;
        float of_label = 0.0f;
        for (int32_t c0 = JOIN ? wave * P * lanes : 0; c0 < a.classes; c0 += P * lanes * (JOIN ? waves : 1)) {
            float v[P];
            const T* at = x + (c0 + l) * sc;
            if (ONE) {
                // behind the last class the last is read again: without branches all loads are on their way before the first is
                // waited for
                T raw[P];
#pragma unroll
                for (int j = 0; j < P; ++j) {
                    const int32_t c = j * lanes + l;
                    raw[j] = x[(c < a.classes ? c : a.classes - 1) * sc];
                }
#pragma unroll
                for (int j = 0; j < P; ++j) v[j] = j * lanes + l < a.classes ? to_f(raw[j]) : -INFINITY;
            } else
#pragma unroll
            for (int j = 0; j < P; ++j) v[j] = live && c0 + j * lanes + l < a.classes ? to_f(at[j * lanes * sc]) : -INFINITY;
            if (ONE) acc.m = group.max(largest(v));
            else acc.raise(fmaxf(acc.m, largest(v)));
            acc.add(v);
#pragma unroll
            for (int j = 0; j < P; ++j) {
                const int32_t c = c0 + j * lanes + l;
                if (ONE) key[j] = __float_as_uint(v[j]);
                else if (TOPN > 0 && c < a.classes) best.add(candidate(v[j], uint32_t(c)));
                if (ONE && P == kPer) of_label = c == label ? v[j] : of_label;
            }
            if (ONE) break;
        }
        if (!ONE) acc.raise(group.max(acc.m));
        acc.s = group.sum(acc.s);
        acc.w = group.sum(acc.w);
        if (ONE && wanted) {
            const bool clean = __ballot(acc.s != acc.s) == 0;
#pragma unroll
            for (int j = 0; j < P; ++j) {
                const float x = __uint_as_float(key[j]);
                // behind the last class lie values of -inf, and as classes of their own they come after all others of -inf
                key[j] = !kShort ? order_key(x) : short_key<T>(x, uint32_t(j * lanes + l), clean);
            }
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
                    acc.join(other);
#pragma unroll
                    for (int t = 0; t < TOPN; ++t) best.add(lists[v][lane][t]);
                }
            }
        }
        if (JOIN && wave != 0) continue;                           // waves leave the turn together: row0 is the workgroup's
        auto next_best = [&]() {
            if (ONE && kShort) {
                last = next_below(key, last, group);
                return (uint64_t(order_key(short_value<T>(last))) << 32) | uint32_t(~(0xffffu - (last & 0xffffu)));
            }
            if (ONE) return take_best(key, group, l);
            const uint64_t top = group.max(best.v[0]);
            if (best.v[0] == top) best.pop();                      // one lane holds it: a candidate carries its class
            return top;
        };
        const float log_s = logf(acc.s);
        float lp = 0.0f;
        const bool counted = writes && a.labels && label != a.ignore;
        if (counted) {
            const bool inside = label >= 0 && label < a.classes;
            if (inside && !(ONE && P == kPer && lanes == 1)) of_label = to_f(x[label * sc]);
            lp = inside ? (of_label - acc.m) - log_s : NAN;
        }
        if (writes && a.stat) a.stat[row] = make_float2(acc.m, log_s);
        if (NLL) {
            const uint64_t top = next_best();
            if (counted) {
                sum += double(lp);
                ++used;
                hits += int64_t(uint32_t(~uint32_t(top))) == label;
            }
        } else {
            if (writes) {
                if (a.logprob) a.logprob[row] = lp;
                a.entropy[row] = log_s - acc.w / acc.s;
            }
            if (ONE || TOPN > 0) {
                int64_t at = b * a.tb + i * a.tn;
                for (int t = 0; t < a.top; ++t, at += a.tk) {
                    const uint64_t top = next_best();
                    if (writes) {
                        a.top_idx[at] = int64_t(uint32_t(~uint32_t(top)));
                        a.top_lp[at] = (key_value(uint32_t(top >> 32)) - acc.m) - log_s;
                    }
                }
            }
        }
    }
    if (NLL) leave_sums(a.partial, sum, double(used), double(hits));
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

// d x_c = [c = y] g_y + sum_t [c = i_t] g_t - p_c (a + g_H log p_c) with a = g_y + sum_t g_t + g_H H: what it takes of a row.
// p = e^(x-m) / s and not e^(log p): rounding log p to 32 bits would cost p |log p| 2^-24 of itself.  x - m is kept above
// kLowest, where p is 0 already, so that a class without probability multiplies no infinity; a row without a distribution has
// a = NaN, one that no gradient reaches has p = 0 whatever it holds.
struct RowGrad {
    int64_t at;                             // of the alternatives
    int32_t label;                          // -1: none
    float gy, gh, a, m, log_s, inverse;     // 1 / s
};

template <bool NLL>
__device__ inline RowGrad row_grad(const GradArgs& a, int64_t row, int64_t b, int64_t i, float scale) {
    RowGrad r;
    // all of a row's values are asked for before the first is looked at: one wait instead of one for each
    const int64_t label = a.labels ? a.labels[row] : a.ignore;
    const float gl = NLL ? scale : a.g_lp ? a.g_lp[row * a.g_lp_s] : 0.0f;
    const float entropy = !NLL && a.g_h ? a.entropy[row] : 0.0f;
    const float2 st = a.stat[row];
    r.gh = !NLL && a.g_h ? a.g_h[row * a.g_h_s] : 0.0f;
    const bool counted = label != a.ignore, inside = label >= 0 && label < a.classes;
    r.label = counted && inside ? int32_t(label) : -1;
    r.gy = !counted ? 0.0f : !inside ? NAN : gl;                     // NaN as its log probability
    r.a = r.gy;
    bool any = r.gy != 0.0f || r.gh != 0.0f;
    r.at = b * a.tb + i * a.tn;
    if (!NLL && a.g_top)
        for (int t = 0; t < a.top; ++t) {
            const float g = a.g_top[r.at + t * a.tk];
            r.a += g;
            any |= g != 0.0f;
        }
    r.a = fmaf(r.gh, r.gh != 0.0f ? entropy : 0.0f, r.a);
    r.m = st.x;
    r.log_s = st.y;
    r.inverse = accurate_weight(-st.y);
    if (!any) r.a = r.inverse = r.log_s = 0.0f;
    else if (!(st.y >= 0.0f)) r.a = NAN;                            // log s of a row with a largest value is at least 0
    return r;
}

template <bool NLL>
__device__ inline float score_grad(const RowGrad& r, float x, int32_t c) {
    const float t = fmaxf(x - r.m, kLowest), p = accurate_weight(t) * r.inverse;
    return (c == r.label ? r.gy : 0.0f) - p * (NLL ? r.a : fmaf(r.gh, t - r.log_s, r.a));
}

// the alternatives' own gradients, to d[j] of class from + j * step
template <int P>
__device__ inline void add_top(const GradArgs& a, int64_t at, int32_t from, int32_t step, float (&d)[P]) {
    for (int t = 0; t < a.top; ++t, at += a.tk) {
        const int32_t c = int32_t(a.top_idx[at]) - from;
        const float g = a.g_top[at];
#pragma unroll
        for (int j = 0; j < P; ++j) d[j] += c == j * step ? g : 0.0f;
    }
}

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
        const RowGrad g = row_grad<NLL>(a, row, b, i, scale);
        for (int32_t c0 = l; c0 < a.classes; c0 += kPer * lanes) {
            float v[kPer];
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const int32_t c = c0 + j * lanes;
                if (c < a.classes) v[j] = to_f(x[c * a.sc]);
            }
            float out[kPer];
#pragma unroll
            for (int j = 0; j < kPer; ++j) out[j] = c0 + j * lanes < a.classes ? score_grad<NLL>(g, v[j], c0 + j * lanes) : 0.0f;
            if (!NLL && a.g_top) add_top(a, g.at, c0, lanes, out);
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const int32_t c = c0 + j * lanes;
                if (c < a.classes) d[c * a.dc] = from_f<T>(out[j]);
            }
        }
    }
}

// Dense rows one behind the other, at least as many classes as 16 bytes hold: the gradient is elementwise once (m, log s, H) are
// known, so a thread takes 16 bytes wherever they fall in at most two rows, and a row's length and alignment do not matter.
template <class T, bool NLL>
__global__ void __launch_bounds__(kBlock) score_grads_flat(const GradArgs a) {
    constexpr int E = 16 / sizeof(T);
    struct alignas(16) Pack { T v[E]; };
    const int64_t total = a.rows * a.classes, first = (int64_t(blockIdx.x) * kBlock + threadIdx.x) * E;
    if (first >= total) return;
    const float scale = NLL ? -a.g_loss[0] * a.inv_count[0] : 0.0f;
    const int64_t row = total <= UINT32_MAX ? int64_t(uint32_t(first) / uint32_t(a.classes)) : first / a.classes;
    const int32_t c0 = int32_t(first - row * a.classes);
    const T* x = static_cast<const T*>(a.x) + first;
    T* d = static_cast<T*>(a.d) + first;
    const bool whole = first + E <= total;
    Pack in;
    if (whole) in = *reinterpret_cast<const Pack*>(x);
    else
        for (int e = 0; e < E; ++e)
            if (first + e < total) in.v[e] = x[e];
    const int64_t after = row + 1 < a.rows ? row + 1 : row;
    RowGrad g = row_grad<NLL>(a, row, 0, row, scale), g1 = row_grad<NLL>(a, after, 0, after, scale);
    g.label -= c0;                                                  // as an element of this piece
    g1.label = g1.label < 0 ? -1 : g1.label + a.classes - c0;
    const int32_t border = a.classes - c0;
    const int64_t at = g.at;
    float grad[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (e == border) g = g1;
        grad[e] = score_grad<NLL>(g, to_f(in.v[e]), e);
    }
    if (!NLL && a.g_top) {
        add_top(a, at, c0, 1, grad);
        if (border < E && row + 1 < a.rows) add_top(a, g1.at, -border, 1, grad);
    }
    Pack out;
#pragma unroll
    for (int e = 0; e < E; ++e) out.v[e] = from_f<T>(grad[e]);
    if (whole) *reinterpret_cast<Pack*>(d) = out;
    else
        for (int e = 0; e < E; ++e)
            if (first + e < total) d[e] = out.v[e];
}

// Loss of many rows of up to kPer classes, class-major with unit stride along the rows: a thread takes 4 neighbouring rows, one load
// of 4 values for each class (the hardware takes them at any alignment), and the backward pass makes the maxima and sums again
// from the scores it reads anyway, instead of 8 bytes a row kept by one pass and read by the other.  2M x 5: 14.1 us forward and
// 16.3 back, 4.0 and 5.9 TB/s (a lane for each row: 20.8 and 19.4); 4M x 5 in bf16: 17.6 and 20.4 (48 and 41).
constexpr int kQuad = 4;
template <class T> struct Raw;
template <> struct Raw<float> { using v4 = __attribute__((ext_vector_type(4), aligned(4))) uint32_t; using v1 = uint32_t; };
template <> struct Raw<__hip_bfloat16> { using v4 = __attribute__((ext_vector_type(4), aligned(2))) uint16_t; using v1 = uint16_t; };
template <> struct Raw<__half> { using v4 = __attribute__((ext_vector_type(4), aligned(2))) uint16_t; using v1 = uint16_t; };
using label2 = __attribute__((ext_vector_type(2), aligned(8))) int64_t;

template <class T, int C>
__device__ inline void load_quad(const T* x, int64_t sc, const int64_t* labels, int64_t ignore, int64_t left, float (&v)[C][kQuad], int64_t (&label)[kQuad]) {
    if (left >= kQuad) {
        typename Raw<T>::v4 raw[C];
#pragma unroll
        for (int c = 0; c < C; ++c) raw[c] = *reinterpret_cast<const typename Raw<T>::v4*>(x + c * sc);
        const label2 l0 = *reinterpret_cast<const label2*>(labels), l1 = *reinterpret_cast<const label2*>(labels + 2);
        label[0] = l0[0]; label[1] = l0[1]; label[2] = l1[0]; label[3] = l1[1];
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int r = 0; r < kQuad; ++r) v[c][r] = to_f(__builtin_bit_cast(T, typename Raw<T>::v1(raw[c][r])));
        return;
    }
#pragma unroll
    for (int r = 0; r < kQuad; ++r) {
        label[r] = r < left ? labels[r] : ignore;
#pragma unroll
        for (int c = 0; c < C; ++c) v[c][r] = r < left ? to_f(x[c * sc + r]) : 0.0f;
    }
}

// maximum and sum of a row's weights, which it leaves in e
template <int C, bool ACCURATE>
__device__ inline float quad_sum(const float (&v)[C][kQuad], int r, float& m, float (&e)[C]) {
    float x[C];
#pragma unroll
    for (int c = 0; c < C; ++c) x[c] = v[c][r];
    m = largest(x);
    const float from = m == -INFINITY ? 0.0f : m;
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const float t = x[c] - from;
        e[c] = ACCURATE ? accurate_weight(t < kLowest ? kLowest : t) : weight(t);           // NaN stays
        s += e[c];
    }
    return s;
}

template <class T, int C>
__global__ void __launch_bounds__(kBlock) nll_quads(const ScoreArgs a) {
    const int64_t quads = (a.inner + kQuad - 1) / kQuad, total = a.rows / a.inner * quads;
    double sum = 0.0;
    int32_t used = 0, hits = 0;
    for (int64_t q = int64_t(blockIdx.x) * kBlock + threadIdx.x; q < total; q += int64_t(gridDim.x) * kBlock) {
        const int64_t b = total == quads ? 0 : q / quads, i = (q - b * quads) * kQuad;
        float v[C][kQuad];
        int64_t label[kQuad];
        load_quad<T, C>(static_cast<const T*>(a.x) + b * a.sb + i, a.sc, a.labels + b * a.inner + i, a.ignore, a.inner - i, v, label);
#pragma unroll
        for (int r = 0; r < kQuad; ++r) {
            float m, e[C], of_label = 0.0f, best = v[0][r];
            int at = 0;
            const float log_s = logf(quad_sum<C, false>(v, r, m, e));
#pragma unroll
            for (int c = 0; c < C; ++c) {
                of_label = c == label[r] ? v[c][r] : of_label;
                const bool more = v[c][r] > best || (v[c][r] != v[c][r] && best == best);      // NaN above everything
                best = more ? v[c][r] : best;
                at = more ? c : at;
            }
            if (label[r] != a.ignore) {
                sum += label[r] >= 0 && label[r] < C ? double((of_label - m) - log_s) : double(NAN);
                ++used;
                hits += at == label[r];
            }
        }
    }
    leave_sums(a.partial, sum, double(used), double(hits));
}

template <class T, int C>
__global__ void __launch_bounds__(kBlock) nll_quad_grads(const GradArgs a) {
    const int64_t quads = (a.inner + kQuad - 1) / kQuad, total = a.rows / a.inner * quads;
    const float scale = -a.g_loss[0] * a.inv_count[0];
    for (int64_t q = int64_t(blockIdx.x) * kBlock + threadIdx.x; q < total; q += int64_t(gridDim.x) * kBlock) {
        const int64_t b = total == quads ? 0 : q / quads, i = (q - b * quads) * kQuad, left = a.inner - i;
        float v[C][kQuad];
        int64_t label[kQuad];
        load_quad<T, C>(static_cast<const T*>(a.x) + b * a.sb + i, a.sc, a.labels + b * a.inner + i, a.ignore, left, v, label);
#pragma unroll
        for (int r = 0; r < kQuad; ++r) {
            float m, e[C];
            const float inverse = 1.0f / quad_sum<C, true>(v, r, m, e);
            // without a gradient 0 whatever the row holds, as where RowGrad says it
            const bool counted = label[r] != a.ignore && (scale != 0.0f || label[r] < 0 || label[r] >= C);
            const float gy = label[r] >= 0 && label[r] < C ? scale : NAN;
#pragma unroll
            for (int c = 0; c < C; ++c) v[c][r] = counted ? (c == label[r] ? gy : 0.0f) - e[c] * inverse * gy : 0.0f;
        }
        T* d = static_cast<T*>(a.d) + b * a.db + i * a.dn;
        if (left >= kQuad && a.dn == 1) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                typename Raw<T>::v4 raw;
#pragma unroll
                for (int r = 0; r < kQuad; ++r) raw[r] = __builtin_bit_cast(typename Raw<T>::v1, from_f<T>(v[c][r]));
                *reinterpret_cast<typename Raw<T>::v4*>(d + c * a.dc) = raw;
            }
        } else {
#pragma unroll
            for (int r = 0; r < kQuad; ++r)
#pragma unroll
                for (int c = 0; c < C; ++c)
                    if (r < left) d[c * a.dc + r * a.dn] = from_f<T>(v[c][r]);
        }
    }
}

// The same answer for the pass forward and the one back, which look at the scores' layout alone.  65536 x 5: 4.8 and 4.0 us either way.
constexpr int64_t kQuadRows = 1 << 16;
bool in_quads(int64_t rows, int64_t inner, int32_t classes, int64_t sc, int64_t sn) {
    return sn == 1 && sc > 1 && classes >= 2 && classes <= kPer && rows >= kQuadRows && inner >= 256;
}

unsigned quad_blocks(int64_t rows, int64_t inner, unsigned most) {
    const int64_t b = (rows / inner * ((inner + kQuad - 1) / kQuad) + kBlock - 1) / kBlock;
    return unsigned(b > most ? most : b);
}

template <class T, class Args>
void launch_quads(const Args& a, unsigned blocks, hipStream_t stream) {
    auto go = [&](auto classes) {
        constexpr int C = decltype(classes)::value;
        if constexpr (std::is_same_v<Args, ScoreArgs>) nll_quads<T, C><<<blocks, kBlock, 0, stream>>>(a);
        else nll_quad_grads<T, C><<<blocks, kBlock, 0, stream>>>(a);
    };
    switch (a.classes) {
        case 2: go(std::integral_constant<int, 2>()); break;
        case 3: go(std::integral_constant<int, 3>()); break;
        case 4: go(std::integral_constant<int, 4>()); break;
        case 5: go(std::integral_constant<int, 5>()); break;
        case 6: go(std::integral_constant<int, 6>()); break;
        case 7: go(std::integral_constant<int, 7>()); break;
        default: go(std::integral_constant<int, 8>()); break;
    }
}

struct Shape {
    int ll, by_class, per;
    bool join, one;
    unsigned blocks;
};

// Lanes of a row.  Row-major: as many as hold the row at kPer classes each, past 64 classes at kMore each but 16 at least (60k x 349
// with 5 alternatives: 80 us on 64 lanes of 8, 47 us on 16 of 24 while each load was waited for, 30 us now).  Class-major: one, unless
// there are too few rows to fill the GPU.  Measured at 349 classes and kept for its neighbours: a row of 65 classes takes the same 384
// places.  60k rows in bf16, report with 5 alternatives (loss forward): 65 classes 30 us (25), 128 30 (24), 172 31 (24), 349 32 (25), 500 108
// (52) and 1000 150 (71), which take strides that are not known when compiled and two waves a SIMD.  Class-major past kPer classes a lane
// keeps a list of its best classes: 2M x 40 float32 169 us (86), where the read alone takes 68.
// A workgroup joins on its rows when even whole wavefronts per row are too few for the GPU and every wave gets classes.
Shape shape_of(int64_t rows, int32_t classes, int64_t sc, int64_t sn, bool can_join, unsigned most) {
    Shape s;
    s.by_class = sc > sn && sn != 0;
    const int64_t fill = int64_t(256) * 8 * 64;            // two waves per SIMD
    s.per = !s.by_class && classes > 64 && classes <= kMore * 64 ? kMore : kPer;
    s.ll = s.per == kMore ? 4 : 0;
    while (s.ll < 6 && (int64_t(s.per) << s.ll) < classes && (!s.by_class || (rows << s.ll) < fill)) ++s.ll;
    const int64_t tiles = (rows + (64 >> s.ll) - 1) / (64 >> s.ll);
    s.one = (int64_t(s.per) << s.ll) >= classes;
    s.join = can_join && s.ll == 6 && tiles < 1024 && !s.one && classes > 2 * kPer * 64;
    const int64_t b = s.join ? tiles : (tiles + kBlock / 64 - 1) / (kBlock / 64);
    s.blocks = unsigned(b < 1 ? 1 : b > most ? most : b);
    return s;
}

template <class T, int TOPN, bool NLL>
void launch_rows(const ScoreArgs& a, const Shape& s, hipStream_t stream) {
    if (s.join) score_rows<T, kPer, TOPN, NLL, false, true, false><<<s.blocks, kBlock, 0, stream>>>(a);
    else score_rows<T, kPer, TOPN, NLL, false, false, false><<<s.blocks, kBlock, 0, stream>>>(a);
}

template <class T, bool NLL>
void launch_one(const ScoreArgs& a, const Shape& s, hipStream_t stream) {
    if (s.per == kPer) score_rows<T, kPer, 0, NLL, true, false, false><<<s.blocks, kBlock, 0, stream>>>(a);
    else if (s.ll == 4 && a.sc == 1) score_rows<T, kMore, 0, NLL, true, false, true><<<s.blocks, kBlock, 0, stream>>>(a);
    else score_rows<T, kMore, 0, NLL, true, false, false><<<s.blocks, kBlock, 0, stream>>>(a);
}

template <class T>
void launch_report(const ScoreArgs& a, const Shape& s, hipStream_t stream) {
    if (s.one) launch_one<T, false>(a, s, stream);
    else if (a.top == 0) launch_rows<T, 0, false>(a, s, stream);
    else if (a.top <= 2) launch_rows<T, 2, false>(a, s, stream);
    else if (a.top <= 8) launch_rows<T, 8, false>(a, s, stream);
    else launch_rows<T, kMostTop, false>(a, s, stream);
}

template <class T, bool NLL>
void launch_grads(GradArgs a, hipStream_t stream) {
    if (NLL && in_quads(a.rows, a.inner, a.classes, a.sc, a.sn)) {
        launch_quads<T>(a, quad_blocks(a.rows, a.inner, kMostBlocks), stream);
        return;
    }
    constexpr int E = 16 / sizeof(T);
    const int64_t total = a.rows * a.classes, blocks = (total + int64_t(kBlock) * E - 1) / (int64_t(kBlock) * E);
    const bool dense = a.rows == a.inner && a.sc == 1 && a.dc == 1 && a.sn == a.classes && a.dn == a.classes && a.classes >= E;
    if (dense && blocks <= (1 << 23) && mh_aligned16(a.x) && mh_aligned16(a.d)) {
        score_grads_flat<T, NLL><<<unsigned(blocks), kBlock, 0, stream>>>(a);
        return;
    }
    const Shape s = shape_of(a.rows, a.classes, a.sc, a.sn, false, kMostBlocks);
    a.ll = s.ll; a.by_class = s.by_class;
    score_grads<T, NLL><<<s.blocks, kBlock, 0, stream>>>(a);
}

template <class T>
void launch_nll(const ScoreArgs& a, const Shape& s, hipStream_t stream) {
    if (in_quads(a.rows, a.inner, a.classes, a.sc, a.sn)) launch_quads<T>(a, quad_blocks(a.rows, a.inner, kMostSums), stream);
    else if (s.one) launch_one<T, true>(a, s, stream);
    else launch_rows<T, 1, true>(a, s, stream);
}

bool countable(int64_t n_batch, int64_t n_inner) {
    return n_batch >= 0 && n_inner >= 0 && n_batch <= kMostRows && (n_batch == 0 || n_inner <= kMostRows / n_batch);
}

int check_scores(const void* x, int dtype, int64_t n_batch, int64_t n_inner, int32_t classes, int64_t sb, int64_t sc, int64_t sn) {
    MH_REQUIRE(dtype >= 0 && dtype <= 2, "dtype=%d: 0 (float32), 1 (bfloat16) and 2 (float16) are known", dtype);
    MH_REQUIRE(countable(n_batch, n_inner) && classes >= 1 && classes <= kMostClasses, "n_batch=%lld n_inner=%lld classes=%d", (long long)n_batch, (long long)n_inner, classes);
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
    const Shape s = shape_of(rows, classes, sc, sn, true, kMostBlocks);
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
    if (dtype == 0) launch_grads<float, false>(a, stream);
    else if (dtype == 1) launch_grads<__hip_bfloat16, false>(a, stream);
    else launch_grads<__half, false>(a, stream);
    MH_LAUNCH_CHECK("class_logprobs_bwd");
    return MH_OK;
}

extern "C" size_t mh_class_nll_workspace_bytes(void) { return size_t(kMostSums) * 3 * sizeof(double); }

extern "C" size_t mh_class_nll_stat_bytes(int64_t n_batch, int64_t n_inner, int32_t classes, int64_t sc, int64_t sn) {
    if (n_batch <= 0 || n_inner <= 0 || !countable(n_batch, n_inner) || in_quads(n_batch * n_inner, n_inner, classes, sc, sn)) return 0;
    return size_t(n_batch) * size_t(n_inner) * sizeof(float2);
}

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
        const Shape s = shape_of(rows, classes, sc, sn, true, kMostSums);
        a.ll = s.ll; a.by_class = s.by_class;
        blocks = in_quads(rows, n_inner, classes, sc, sn) ? quad_blocks(rows, n_inner, kMostSums) : s.blocks;
        if (dtype == 0) launch_nll<float>(a, s, stream);
        else if (dtype == 1) launch_nll<__hip_bfloat16>(a, s, stream);
        else launch_nll<__half>(a, s, stream);
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
    MH_REQUIRE(labels && (stat || in_quads(rows, n_inner, classes, sc, sn)) && inv_count && g_loss && d_scores, "null pointer");
    MH_REQUIRE(db >= 0 && dc >= 0 && dn >= 0, "negative stride");
    GradArgs a{};
    a.x = scores; a.d = d_scores; a.rows = rows; a.inner = n_inner; a.sb = sb; a.sc = sc; a.sn = sn; a.db = db; a.dc = dc; a.dn = dn;
    a.classes = classes; a.labels = labels; a.ignore = ignore; a.stat = reinterpret_cast<const float2*>(stat);
    a.g_loss = g_loss; a.inv_count = inv_count;
    if (dtype == 0) launch_grads<float, true>(a, stream);
    else if (dtype == 1) launch_grads<__hip_bfloat16, true>(a, stream);
    else launch_grads<__half, true>(a, stream);
    MH_LAUNCH_CHECK("class_nll_bwd");
    return MH_OK;
}
