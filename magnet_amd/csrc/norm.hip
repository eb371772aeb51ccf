// Group norm of row-planar complex features over the graphs of a batch, channels last, with the complex ReLU behind it.
//
// Graph b owns rows ptr[b] .. ptr[b+1], group g the channels g D .. (g+1) D, D = F / groups, M = n_b D complex values:
//     m = mean z (complex)   v = mean |z - m|^2   xh = (z - m) / sqrt(v + eps)   y = gamma xh + beta (1 + i)
//     complex ReLU: both parts of y are kept where Re y >= 0
// Backward, dy the gated gradient:
//     dgamma = sum (dy_r xh_r + dy_i xh_i)    dbeta = sum (dy_r + dy_i)    dxh = gamma dy
//     dx = (dxh - mean dxh - xh mean(dxh_r xh_r + dxh_i xh_i)) / sqrt(v + eps)
//
// Two passes over the rows per direction: sums, then the elementwise result.  Rows are cut into tiles of T rows and at the
// graphs' borders; piece d = tile + graph in the merged order of both kinds of border, so a workgroup finds its piece by one
// binary search in ptr and nothing is planned on the host.  A thread keeps its channels (4, or 1 where a width does not divide)
// while it walks down its rows; sums are held in 64 bits (a group may hold 10^8 values, and mean |z|^2 - |m|^2 loses what the
// mean exceeds the deviation by), joined through LDS and then over the pieces in a fixed order: no atomics, the same result
// every time.  The mean is kept as the sum of two floats, so z - m is exact to 32 bits however far the mean lies from 0.
// Bound by HBM: the passes read 8 NF and 8 NF bytes and write 8 NF forward, 16 NF + 16 NF and 8 NF backward.
// Rows behind the last graph (a padded batch) get zeros, forward and backward.
#include <cstdint>

#include <hip/hip_runtime.h>

#include "ckpt.h"
#include "common.h"

namespace {

constexpr int kBlock = 256;
constexpr int64_t kMostTiles = 2048;       // 8 workgroups of 4 waves per CU
constexpr int kStats = 5;                  // re mean (high, low), im mean (high, low), 1 / deviation

struct NormArgs {
    const float* x;
    int64_t ld, im;
    const uint8_t *codes, *scales;         // instead of x in the backward pass of a checkpointed norm
    int64_t rp;
    int32_t mp;
    int64_t rows, tile_rows;
    int32_t F, groups, D, graphs;
    const int32_t* ptr;                    // [graphs + 1], or NULL: one graph of all rows
    float eps;
    const float *gamma, *beta;
    int32_t relu;
    float* stats;                          // [graphs][groups][kStats]
    double* partial;                       // [pieces][3][F]
    double* sums;                          // [graphs][3][F]
    float* means;                          // [graphs][groups][3]
    const float* g;
    int64_t ldg, img;
    float* out;
    int64_t ldo, imo;
    uint8_t* mask;                         // [rows][F]
    float *dgamma, *dbeta;
    int32_t lanes, chunks;                 // threads side by side on a row; channel chunks (grid y)
};

struct Piece {
    int64_t lo, hi;
    int32_t graph;                         // == graphs: rows behind the last graph
};

__device__ inline int64_t row_start(const NormArgs& a, int32_t b) {
    if (b == 0) return 0;
    const int64_t p = a.ptr ? a.ptr[b] : a.rows;
    return p < 0 ? 0 : p > a.rows ? a.rows : p;
}

__device__ inline int64_t first_piece(const NormArgs& a, int32_t b) { return row_start(a, b) / a.tile_rows + b; }

__device__ inline Piece piece_of(const NormArgs& a, int64_t d) {
    int32_t lo = 0, hi = a.graphs;         // the last b with first_piece(b) <= d
    while (lo < hi) {
        const int32_t mid = (lo + hi + 1) >> 1;
        if (first_piece(a, mid) <= d) lo = mid; else hi = mid - 1;
    }
    Piece p;
    p.graph = lo;
    const int64_t t = (d - lo) * a.tile_rows, s = row_start(a, lo), e = lo < a.graphs ? row_start(a, lo + 1) : a.rows;
    p.lo = s > t ? s : t;
    p.hi = e < t + a.tile_rows ? e : t + a.tile_rows;
    return p;
}

template <int V> struct Vec { float v[V]; };

template <int V>
__device__ inline Vec<V> load(const float* p) {
    Vec<V> r;
    if (V == 4) { const float4 t = *reinterpret_cast<const float4*>(p); r.v[0] = t.x; r.v[V > 1 ? 1 : 0] = t.y; r.v[V > 2 ? 2 : 0] = t.z; r.v[V > 3 ? 3 : 0] = t.w; }
    else r.v[0] = *p;
    return r;
}
template <int V>
__device__ inline void store(float* p, const Vec<V>& r) {
    if (V == 4) *reinterpret_cast<float4*>(p) = make_float4(r.v[0], r.v[V > 1 ? 1 : 0], r.v[V > 2 ? 2 : 0], r.v[V > 3 ? 3 : 0]);
    else *p = r.v[0];
}

// the normalisation of a thread's channels
template <int V>
struct Channels {
    float mh[2][V], ml[2][V], rstd[V], scale[V], shift[V], gamma[V];
};

template <int V>
__device__ inline Channels<V> channels(const NormArgs& a, int32_t graph, int32_t c) {
    Channels<V> k;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float* s = a.stats + (int64_t(graph) * a.groups + (c + j) / a.D) * kStats;
        k.mh[0][j] = s[0]; k.ml[0][j] = s[1]; k.mh[1][j] = s[2]; k.ml[1][j] = s[3]; k.rstd[j] = s[4];
        k.gamma[j] = a.gamma ? a.gamma[c + j] : 1.0f;
        k.scale[j] = k.rstd[j] * k.gamma[j];
        k.shift[j] = a.beta ? a.beta[c + j] : 0.0f;
    }
    return k;
}

template <int V>
__device__ inline float centred(const Channels<V>& k, int part, int j, float x) { return (x - k.mh[part][j]) - k.ml[part][j]; }
// y; written once, so that the gate of the backward pass is the forward's to the last bit
template <int V>
__device__ inline float result(const Channels<V>& k, int part, int j, float x) { return fmaf(centred(k, part, j, x), k.scale[j], k.shift[j]); }

template <int V, bool HELD>
__device__ inline Vec<V> input(const NormArgs& a, int64_t row, int part, int32_t c) {
    if (!HELD) return load<V>(a.x + row * a.ld + part * a.im + c);
    const int64_t r = 2 * row + part;
    const uint32_t e = a.scales[int64_t(c / mhckpt::kBlockCols) * a.rp + r];
    Vec<V> v;
    if (V == 4) {
        const float4 t = mhckpt::decode(*reinterpret_cast<const uint32_t*>(a.codes + r * a.mp + c), e);
        v.v[0] = t.x; v.v[V > 1 ? 1 : 0] = t.y; v.v[V > 2 ? 2 : 0] = t.z; v.v[V > 3 ? 3 : 0] = t.w;
    } else {
        v.v[0] = mhckpt::decode1(a.codes[r * a.mp + c], mhckpt::scale_of(e));
    }
    return v;
}

// gated gradient and normalised input of a thread's channels in a row
template <int V, bool HELD>
__device__ inline void gated(const NormArgs& a, const Channels<V>& k, int64_t row, int32_t c, Vec<V> (&dy)[2], Vec<V> (&xh)[2]) {
    Vec<V> x[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        x[p] = input<V, HELD>(a, row, p, c);
        dy[p] = load<V>(a.g + row * a.ldg + p * a.img + c);
    }
    uint32_t keep = 0;
    if (HELD && a.relu) keep = V == 4 ? *reinterpret_cast<const uint32_t*>(a.mask + row * a.F + c) : a.mask[row * a.F + c];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const bool open = !a.relu || (HELD ? ((keep >> (8 * j)) & 255u) != 0u : result(k, 0, j, x[0].v[j]) >= 0.0f);
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            xh[p].v[j] = centred(k, p, j, x[p].v[j]) * k.rstd[j];
            dy[p].v[j] = open ? dy[p].v[j] : 0.0f;
        }
    }
}

// sums of a workgroup's rows, joined over the threads of a channel and left as a piece's partial sums
template <int V>
__device__ inline void leave_partial(const NormArgs& a, int64_t d, double (&acc)[3][V]) {
    __shared__ double part[3 * V][kBlock];
    const int lanes = a.lanes, tid = threadIdx.x;
#pragma unroll
    for (int s = 0; s < 3; ++s)
#pragma unroll
        for (int j = 0; j < V; ++j) part[s * V + j][tid] = acc[s][j];
    for (int n = kBlock / lanes; n > 1; n >>= 1) {
        __syncthreads();
        for (int i = tid; i < 3 * V * (n >> 1) * lanes; i += kBlock) {
            const int s = i / ((n >> 1) * lanes), at = i - s * ((n >> 1) * lanes);
            part[s][at] += part[s][at + (n >> 1) * lanes];
        }
    }
    __syncthreads();
    for (int i = tid; i < 3 * V * lanes; i += kBlock) {
        const int s = i / (V * lanes), at = i - s * (V * lanes), c = int(blockIdx.y) * lanes * V + at;
        if (c < a.F) a.partial[(d * 3 + s) * a.F + c] = part[s * V + at % V][at / V];
    }
}

template <int V>
__global__ void __launch_bounds__(kBlock) norm_sums_kernel(const NormArgs a) {
    const Piece p = piece_of(a, blockIdx.x);
    if (p.graph == a.graphs || p.lo >= p.hi) return;                // read by nobody
    const int32_t c = (int32_t(blockIdx.y) * a.lanes + int32_t(threadIdx.x) % a.lanes) * V;
    double acc[3][V] = {};
    if (c < a.F) {
        const int step = kBlock / a.lanes;
#pragma unroll 4
        for (int64_t row = p.lo + threadIdx.x / a.lanes; row < p.hi; row += step) {
            const Vec<V> re = load<V>(a.x + row * a.ld + c), im = load<V>(a.x + row * a.ld + a.im + c);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const double r = re.v[j], i = im.v[j];
                acc[0][j] += r;
                acc[1][j] += i;
                acc[2][j] = fma(r, r, fma(i, i, acc[2][j]));
            }
        }
    }
    leave_partial<V>(a, blockIdx.x, acc);
}

// a workgroup's sum of three values per thread
__device__ inline void join3(double (&v)[3]) {
    __shared__ double part[16][3];
    const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
    for (int s = 0; s < 3; ++s) {
        for (int o = 32; o > 0; o >>= 1) v[s] += __shfl_xor(v[s], o);
        if ((threadIdx.x & 63) == 0) part[wave][s] = v[s];
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 3; ++s) {
        v[s] = 0.0;
        for (int w = 0; w < waves; ++w) v[s] += part[w][s];
    }
}

__device__ inline void leave_stats(const NormArgs& a, int32_t b, int32_t g, int64_t n, const double (&v)[3]) {
    const double count = double(n) * a.D;
    const double mr = n ? v[0] / count : 0.0, mi = n ? v[1] / count : 0.0;
    double var = n ? v[2] / count - mr * mr - mi * mi : 0.0;
    if (var < 0.0) var = 0.0;                                       // NaN stays
    float* s = a.stats + (int64_t(b) * a.groups + g) * kStats;
    s[0] = float(mr); s[1] = float(mr - double(float(mr)));
    s[2] = float(mi); s[3] = float(mi - double(float(mi)));
    s[4] = float(1.0 / sqrt(var + double(a.eps)));
}

// one workgroup per (graph, group)
__global__ void __launch_bounds__(1024) norm_stats_kernel(const NormArgs a) {
    const int32_t b = blockIdx.x / a.groups, g = blockIdx.x - b * a.groups;
    const int64_t lo = row_start(a, b), hi = row_start(a, b + 1);
    double v[3] = {0.0, 0.0, 0.0};
    if (lo < hi) {
        const int64_t d0 = lo / a.tile_rows + b, d1 = (hi - 1) / a.tile_rows + b + 1;
        const int64_t items = (d1 - d0) * a.D;
#pragma unroll 2
        for (int64_t i = threadIdx.x; i < items; i += blockDim.x) {
            const int64_t d = i / a.D;
            const double* p = a.partial + (d0 + d) * 3 * a.F + g * a.D + (i - d * a.D);
            v[0] += p[0]; v[1] += p[a.F]; v[2] += p[2 * a.F];
        }
    }
    join3(v);
    if (threadIdx.x == 0) leave_stats(a, b, g, hi - lo, v);
}

template <int V>
__global__ void __launch_bounds__(kBlock) norm_apply_kernel(const NormArgs a) {
    const Piece p = piece_of(a, blockIdx.x);
    const int32_t c = (int32_t(blockIdx.y) * a.lanes + int32_t(threadIdx.x) % a.lanes) * V;
    if (c >= a.F || p.lo >= p.hi) return;
    const int step = kBlock / a.lanes;
    if (p.graph == a.graphs) {
        Vec<V> zero;
#pragma unroll
        for (int j = 0; j < V; ++j) zero.v[j] = 0.0f;
        for (int64_t row = p.lo + threadIdx.x / a.lanes; row < p.hi; row += step) {
            store<V>(a.out + row * a.ldo + c, zero);
            store<V>(a.out + row * a.ldo + a.imo + c, zero);
        }
        return;
    }
    const Channels<V> k = channels<V>(a, p.graph, c);
#pragma unroll 4
    for (int64_t row = p.lo + threadIdx.x / a.lanes; row < p.hi; row += step) {
        Vec<V> re = load<V>(a.x + row * a.ld + c), im = load<V>(a.x + row * a.ld + a.im + c);
        uint32_t keep = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float yr = result(k, 0, j, re.v[j]), yi = result(k, 1, j, im.v[j]);
            // the gate multiplies, as the framework's complex ReLU does: what is not finite stays visible
            const float open = !a.relu || yr >= 0.0f ? 1.0f : 0.0f;
            re.v[j] = yr * open;
            im.v[j] = yi * open;
            keep |= uint32_t(open != 0.0f) << (8 * j);
        }
        store<V>(a.out + row * a.ldo + c, re);
        store<V>(a.out + row * a.ldo + a.imo + c, im);
        if (a.mask) {
            if (V == 4) *reinterpret_cast<uint32_t*>(a.mask + row * a.F + c) = keep;
            else a.mask[row * a.F + c] = uint8_t(keep);
        }
    }
}

template <int V, bool HELD>
__global__ void __launch_bounds__(kBlock) norm_bwd_sums_kernel(const NormArgs a) {
    const Piece p = piece_of(a, blockIdx.x);
    if (p.graph == a.graphs || p.lo >= p.hi) return;
    const int32_t c = (int32_t(blockIdx.y) * a.lanes + int32_t(threadIdx.x) % a.lanes) * V;
    double acc[3][V] = {};
    if (c < a.F) {
        const Channels<V> k = channels<V>(a, p.graph, c);
        const int step = kBlock / a.lanes;
#pragma unroll 2
        for (int64_t row = p.lo + threadIdx.x / a.lanes; row < p.hi; row += step) {
            Vec<V> dy[2], xh[2];
            gated<V, HELD>(a, k, row, c, dy, xh);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                acc[0][j] += double(dy[0].v[j]);
                acc[1][j] += double(dy[1].v[j]);
                acc[2][j] += double(fmaf(dy[0].v[j], xh[0].v[j], dy[1].v[j] * xh[1].v[j]));
            }
        }
    }
    leave_partial<V>(a, blockIdx.x, acc);
}

// per graph and channel: the pieces' partial sums; 32 channels to a workgroup
__global__ void __launch_bounds__(1024) norm_bwd_channels_kernel(const NormArgs a) {
    __shared__ double part[32][33];
    const int32_t b = blockIdx.x, cl = threadIdx.x & 31, q = threadIdx.x >> 5, c = int32_t(blockIdx.y) * 32 + cl;
    const int64_t lo = row_start(a, b), hi = row_start(a, b + 1);
    for (int s = 0; s < 3; ++s) {
        double v = 0.0;
        if (lo < hi && c < a.F) {
            const int64_t d0 = lo / a.tile_rows + b, d1 = (hi - 1) / a.tile_rows + b + 1;
#pragma unroll 4
            for (int64_t d = d0 + q; d < d1; d += 32) v += a.partial[(d * 3 + s) * a.F + c];
        }
        __syncthreads();
        part[q][cl] = v;
        __syncthreads();
        if (q == 0 && c < a.F) {
            double t = 0.0;
            for (int i = 0; i < 32; ++i) t += part[i][cl];
            a.sums[(int64_t(b) * 3 + s) * a.F + c] = t;
        }
    }
}

// the first graphs * groups workgroups: a group's means of dxh and of dxh xh; the others: dgamma and dbeta of 64 channels
__global__ void __launch_bounds__(kBlock) norm_bwd_means_kernel(const NormArgs a) {
    const int32_t first = a.graphs * a.groups;
    if (int32_t(blockIdx.x) < first) {
        const int32_t b = blockIdx.x / a.groups, g = blockIdx.x - b * a.groups;
        const int64_t n = row_start(a, b + 1) - row_start(a, b);
        double v[3] = {0.0, 0.0, 0.0};
        for (int32_t j = threadIdx.x; j < a.D; j += kBlock) {
            const int32_t c = g * a.D + j;
            const double w = a.gamma ? double(a.gamma[c]) : 1.0;
            const double* s = a.sums + int64_t(b) * 3 * a.F + c;
            v[0] += w * s[0]; v[1] += w * s[a.F]; v[2] += w * s[2 * a.F];
        }
        join3(v);
        if (threadIdx.x < 3) {
            const double count = double(n > 0 ? n : 1) * a.D;
            a.means[(int64_t(b) * a.groups + g) * 3 + threadIdx.x] = float((threadIdx.x == 0 ? v[0] : threadIdx.x == 1 ? v[1] : v[2]) / count);
        }
        return;
    }
    __shared__ double part[2][4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int32_t c = (int32_t(blockIdx.x) - first) * 64 + lane;
    double w = 0.0, s = 0.0;
    if (c < a.F)
#pragma unroll 4
        for (int32_t b = wave; b < a.graphs; b += 4) {
            const double* p = a.sums + int64_t(b) * 3 * a.F + c;
            s += p[0] + p[a.F];
            w += p[2 * a.F];
        }
    part[0][wave][lane] = w;
    part[1][wave][lane] = s;
    __syncthreads();
    if (wave == 0 && c < a.F) {
        if (a.dgamma) a.dgamma[c] = float((part[0][0][lane] + part[0][1][lane]) + (part[0][2][lane] + part[0][3][lane]));
        if (a.dbeta) a.dbeta[c] = float((part[1][0][lane] + part[1][1][lane]) + (part[1][2][lane] + part[1][3][lane]));
    }
}

// (dxh - flat) - xh along with separate roundings: where a group's gradient is its mean, the difference is 0 and not the last
// bits of a product
__device__ inline float less_means(float gamma, float dy, float flat, float xh, float along) {
#pragma clang fp contract(off)
    const float dxh = gamma * dy, pull = xh * along;
    return (dxh - flat) - pull;
}

template <int V, bool HELD>
__global__ void __launch_bounds__(kBlock) norm_bwd_apply_kernel(const NormArgs a) {
    const Piece p = piece_of(a, blockIdx.x);
    const int32_t c = (int32_t(blockIdx.y) * a.lanes + int32_t(threadIdx.x) % a.lanes) * V;
    if (c >= a.F || p.lo >= p.hi) return;
    const int step = kBlock / a.lanes;
    const bool behind = p.graph == a.graphs;
    const Channels<V> k = channels<V>(a, behind ? 0 : p.graph, c);
    float flat[2][V], along[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float* m = a.means + (int64_t(behind ? 0 : p.graph) * a.groups + (c + j) / a.D) * 3;
        flat[0][j] = m[0]; flat[1][j] = m[1]; along[j] = m[2];
    }
#pragma unroll 2
    for (int64_t row = p.lo + threadIdx.x / a.lanes; row < p.hi; row += step) {
        Vec<V> dy[2], xh[2];
        if (!behind) gated<V, HELD>(a, k, row, c, dy, xh);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            Vec<V> d;
#pragma unroll
            for (int j = 0; j < V; ++j)
                d.v[j] = behind ? 0.0f : k.rstd[j] * less_means(k.gamma[j], dy[q].v[j], flat[q][j], xh[q].v[j], along[j]);
            store<V>(a.out + row * a.ldo + q * a.imo + c, d);
        }
    }
}

struct Layout {
    int32_t v, lanes, chunks;
    int64_t tile_rows, pieces;
};

Layout layout_of(int64_t rows, int32_t graphs, int32_t F, bool vec) {
    Layout l;
    l.v = vec ? 4 : 1;
    const int32_t units = (F + l.v - 1) / l.v;
    l.lanes = 1;
    while (l.lanes < 64 && l.lanes < units) l.lanes <<= 1;
    l.chunks = (units + l.lanes - 1) / l.lanes;
    const int64_t at_once = kBlock / l.lanes;
    const int64_t least = (rows + kMostTiles - 1) / kMostTiles;
    l.tile_rows = (least + at_once - 1) / at_once * at_once;
    if (l.tile_rows < at_once) l.tile_rows = at_once;
    l.pieces = (rows + l.tile_rows - 1) / l.tile_rows + graphs;
    return l;
}

struct Workspace {
    size_t partial, sums, means, bytes;
};

// sized for the narrower layout of the two, so that it does not depend on a call's alignment
Workspace workspace_of(int64_t rows, int32_t graphs, int32_t F, int32_t groups) {
    const int64_t a = layout_of(rows, graphs, F, true).pieces, b = layout_of(rows, graphs, F, false).pieces;
    Workspace w;
    w.partial = 0;
    w.sums = w.partial + size_t(a > b ? a : b) * 3 * F * sizeof(double);
    w.means = w.sums + size_t(graphs) * 3 * F * sizeof(double);
    w.bytes = w.means + (size_t(graphs) * groups * 3 * sizeof(float) + 15) / 16 * 16;
    return w;
}

int check_norm(int64_t rows, int32_t F, int32_t groups, const void* ptr, int32_t graphs) {
    MH_REQUIRE(rows >= 0 && rows <= INT32_MAX && F >= 1 && F <= (1 << 20), "n_rows=%lld F=%d", (long long)rows, F);
    MH_REQUIRE(groups >= 1 && F % groups == 0, "%d channels do not divide into %d groups", F, groups);
    MH_REQUIRE(graphs >= (rows > 0 ? 1 : 0) && graphs <= (1 << 24) && int64_t(graphs) * groups <= (int64_t(1) << 30), "n_graphs=%d", graphs);
    MH_REQUIRE(ptr || graphs <= 1, "n_graphs=%d without graph_ptr", graphs);
    return MH_OK;
}

bool vec_planar(const void* p, int64_t ld, int64_t im) { return (ld & 3) == 0 && (im & 3) == 0 && mh_aligned16(p); }

template <class Kernel1, class Kernel4>
void pick(const Layout& l, Kernel1 k1, Kernel4 k4, const NormArgs& a, hipStream_t stream) {
    const dim3 grid(unsigned(l.pieces), unsigned(l.chunks));
    if (l.v == 4) k4<<<grid, kBlock, 0, stream>>>(a);
    else k1<<<grid, kBlock, 0, stream>>>(a);
}

}  // namespace

extern "C" size_t mh_group_norm_workspace_bytes(int64_t n_rows, int32_t n_graphs, int32_t F, int32_t groups) {
    if (n_rows < 0 || n_graphs < 0 || F < 1 || groups < 1) return 0;
    return workspace_of(n_rows, n_graphs, F, groups).bytes;
}

extern "C" int mh_group_norm(const float* X, int64_t ld, int64_t im, int64_t n_rows, int32_t F, int32_t groups,
                             const int32_t* graph_ptr, int32_t n_graphs, float eps, const float* gamma, const float* beta, int relu,
                             float* Y, int64_t ldy, int64_t imy, uint8_t* mask_out, float* stats, void* workspace,
                             size_t workspace_bytes, void* stream_) {
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    if (int rc = check_norm(n_rows, F, groups, graph_ptr, n_graphs)) return rc;
    if (n_rows == 0) return MH_OK;
    MH_REQUIRE(X && Y && stats && workspace, "null pointer");
    MH_REQUIRE(ld >= 0 && im >= 0 && ldy >= F && imy >= F, "stride smaller than F");
    const Workspace w = workspace_of(n_rows, n_graphs, F, groups);
    if (workspace_bytes < w.bytes) return mh::fail(MH_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, w.bytes);
    MH_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 7) == 0, "workspace must be 8-byte aligned");
    const bool vec = (F & 3) == 0 && vec_planar(X, ld, im) && vec_planar(Y, ldy, imy) && (reinterpret_cast<uintptr_t>(mask_out) & 3) == 0;
    const Layout l = layout_of(n_rows, n_graphs, F, vec);
    NormArgs a{};
    a.x = X; a.ld = ld; a.im = im; a.rows = n_rows; a.tile_rows = l.tile_rows; a.F = F; a.groups = groups; a.D = F / groups;
    a.graphs = n_graphs; a.ptr = graph_ptr; a.eps = eps; a.gamma = gamma; a.beta = beta; a.relu = relu ? 1 : 0; a.stats = stats;
    a.partial = reinterpret_cast<double*>(static_cast<char*>(workspace) + w.partial);
    a.out = Y; a.ldo = ldy; a.imo = imy; a.mask = relu ? mask_out : nullptr; a.lanes = l.lanes; a.chunks = l.chunks;
    pick(l, norm_sums_kernel<1>, norm_sums_kernel<4>, a, stream);
    norm_stats_kernel<<<unsigned(n_graphs) * unsigned(groups), 1024, 0, stream>>>(a);
    pick(l, norm_apply_kernel<1>, norm_apply_kernel<4>, a, stream);
    MH_LAUNCH_CHECK("group_norm");
    return MH_OK;
}

extern "C" int mh_group_norm_bwd(const float* X, int64_t ld, int64_t im, const uint8_t* codes, const uint8_t* scales,
                                 const uint8_t* mask, int64_t n_rows, int32_t F, int32_t groups, const int32_t* graph_ptr,
                                 int32_t n_graphs, const float* stats, const float* gamma, const float* beta, int relu, const float* G,
                                 int64_t ldg, int64_t img, float* dX, int64_t lddx, int64_t imdx, float* dgamma, float* dbeta,
                                 void* workspace, size_t workspace_bytes, void* stream_) {
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    if (int rc = check_norm(n_rows, F, groups, graph_ptr, n_graphs)) return rc;
    const bool held = codes != nullptr;
    const bool any = n_rows > 0;
    MH_REQUIRE(!any || ((X || (codes && scales && (!relu || mask))) && G && stats), "null pointer");
    MH_REQUIRE(workspace, "null pointer");
    MH_REQUIRE(ld >= 0 && im >= 0 && ldg >= 0 && img >= 0 && (!any || !dX || (lddx >= F && imdx >= F)), "stride smaller than F");
    const Workspace w = workspace_of(n_rows, n_graphs, F, groups);
    if (workspace_bytes < w.bytes) return mh::fail(MH_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, w.bytes);
    MH_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 7) == 0, "workspace must be 8-byte aligned");
    MH_REQUIRE((reinterpret_cast<uintptr_t>(codes) & 3) == 0, "codes must be 4-byte aligned");
    const bool vec = (F & 3) == 0 && (held ? (reinterpret_cast<uintptr_t>(mask) & 3) == 0 : vec_planar(X, ld, im)) &&
                     vec_planar(G, ldg, img) && (!dX || vec_planar(dX, lddx, imdx));
    const Layout l = layout_of(n_rows, n_graphs, F, vec);
    NormArgs a{};
    a.x = X; a.ld = ld; a.im = im; a.codes = codes; a.scales = scales; a.rp = (2 * n_rows + 7) & ~int64_t(7); a.mp = (F + 31) & ~31;
    a.rows = n_rows; a.tile_rows = l.tile_rows; a.F = F; a.groups = groups; a.D = F / groups; a.graphs = n_graphs; a.ptr = graph_ptr;
    a.gamma = gamma; a.beta = beta; a.relu = relu ? 1 : 0; a.stats = const_cast<float*>(stats);
    a.partial = reinterpret_cast<double*>(static_cast<char*>(workspace) + w.partial);
    a.sums = reinterpret_cast<double*>(static_cast<char*>(workspace) + w.sums);
    a.means = reinterpret_cast<float*>(static_cast<char*>(workspace) + w.means);
    a.g = G; a.ldg = ldg; a.img = img; a.out = dX; a.ldo = lddx; a.imo = imdx; a.mask = const_cast<uint8_t*>(mask);
    a.dgamma = dgamma; a.dbeta = dbeta; a.lanes = l.lanes; a.chunks = l.chunks;
    if (any) {
        if (held) pick(l, norm_bwd_sums_kernel<1, true>, norm_bwd_sums_kernel<4, true>, a, stream);
        else pick(l, norm_bwd_sums_kernel<1, false>, norm_bwd_sums_kernel<4, false>, a, stream);
    }
    if (n_graphs > 0) norm_bwd_channels_kernel<<<dim3(unsigned(n_graphs), unsigned((F + 31) / 32)), 1024, 0, stream>>>(a);
    norm_bwd_means_kernel<<<unsigned(n_graphs) * unsigned(groups) + unsigned((F + 63) / 64), kBlock, 0, stream>>>(a);
    if (any && dX) {
        if (held) pick(l, norm_bwd_apply_kernel<1, true>, norm_bwd_apply_kernel<4, true>, a, stream);
        else pick(l, norm_bwd_apply_kernel<1, false>, norm_bwd_apply_kernel<4, false>, a, stream);
    }
    MH_LAUNCH_CHECK("group_norm_bwd");
    return MH_OK;
}
