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
// binary search in ptr and nothing is planned on the host.  A thread keeps its channels (4, 2 or 1, as the width divides)
// while it walks down its rows; sums are held in 64 bits (a group may hold 10^8 values) and taken of z - z0, z0 the group's
// first value: mean |z|^2 - |m|^2 loses twice the digits that the mean exceeds the deviation by; they are joined through LDS and then over the pieces in a fixed order: no atomics, the same result
// every time.  The mean is kept as the sum of two floats, so z - m is exact to 32 bits however far the mean lies from 0.
// Rows behind the last graph (a padded batch) get zeros, forward and backward.
//
// Bound by HBM: the passes read 8 NF and 8 NF bytes and write 8 NF forward, 16 NF + 16 NF and 8 NF backward.  The pass for
// sums has as many tiles as the GPU holds workgroups at once, the elementwise pass small ones.  The elementwise pass walks the
// pieces backwards: the rows read last are still in the 256 MB cache in front of the memory.
//
// Made for batches of up to a few thousand graphs.  1M x 64 in 8 groups, forward and backward: one graph 264 and 438 us, 512 graphs 284 and
// 455, 2000 301 and 479, 10000 353 and 612, 50000 766 and 1431, 200000 (5 rows each) 2386 and 5487 us: each graph has pieces of its own to
// join, and 16 threads to a channel add the graphs' sums for dgamma and dbeta.  The workspace, one size for both
// directions, is 8 MB at 2000 graphs, 160 MB at 50000 and 635 MB at 200000 beside an input of 512 MB.
#include <cstdint>

#include <hip/hip_runtime.h>

#include "ckpt.h"
#include "common.h"

namespace {

constexpr int kBlock = 256;
constexpr int64_t kSumTiles = 1024;        // 4 workgroups of 4 waves for each CU
constexpr int64_t kMostTiles = 65536;      // of the elementwise pass
constexpr int kStats = 5;                  // re mean (high, low), im mean (high, low), 1 / deviation
// Results from this size on are written past the caches: nothing here reads them again, and lines waiting to be written back slow
// the reads of the next pass (1M x 128: sums 199 -> 170 us forward and 379 -> 340 us backward, 6.0 TB/s; the four passes over
// 200k x 64 together 183 -> 167 us).  Smaller ones stay, for the convolution that comes next.
constexpr int64_t kPast = int64_t(64) << 20;
constexpr int64_t kFewPieces = 64;
constexpr int32_t kMostGraphs = 1 << 22, kMostChannels = 1 << 20;
constexpr int kMostParts = 16;             // shares of a graph's pieces

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
    double* partial;                       // forward [pieces][3][chunks * slots], backward [pieces][3][F]
    double* sums;                          // [graphs][parts][3][F]
    float* means;                          // [graphs][groups][3]
    const float* g;
    int64_t ldg, img;
    float* out;
    int64_t ldo, imo;
    uint8_t* mask;                         // [rows][F]
    float *dgamma, *dbeta;
    int32_t lanes, width, chunks, slots;   // threads side by side on a row, their channels; chunks of these (grid y); groups in one
    int32_t parts;
    uint8_t *codes_out, *scales_out;       // checkpoint of x that the elementwise pass leaves, or NULL
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

__device__ inline int64_t first_piece(const NormArgs& a, int32_t b) { return uint32_t(row_start(a, b)) / uint32_t(a.tile_rows) + b; }
// the pieces of a graph that has rows
__device__ inline void pieces_of(const NormArgs& a, int32_t b, int64_t lo, int64_t hi, int64_t& d0, int64_t& d1) {
    d0 = uint32_t(lo) / uint32_t(a.tile_rows) + b;
    d1 = uint32_t(hi - 1) / uint32_t(a.tile_rows) + b + 1;
}

// all lanes of a wave ask for the same piece
__device__ inline Piece piece_of(const NormArgs& a, int64_t d) {
    int32_t lo = 0;                        // the last b with first_piece(b) <= d: 64 candidates at a time
    if (a.ptr) {
        for (int32_t n = a.graphs + 1; n > 1;) {
            const int32_t step = (n + 63) >> 6, at = int32_t(threadIdx.x & 63) * step;
            // the candidates up to the first that begins behind d; the first of all does not, whatever ptr holds
            const uint64_t behind = ~__ballot(at < n && first_piece(a, lo + at) <= d);
            const int32_t first = behind ? __ffsll(static_cast<unsigned long long>(behind)) - 1 : 64, below = first > 0 ? first - 1 : 0;
            const int32_t left = n - below * step;
            lo += below * step;
            n = left < step ? left : step;
        }
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
    else if (V == 2) { const float2 t = *reinterpret_cast<const float2*>(p); r.v[0] = t.x; r.v[V > 1 ? 1 : 0] = t.y; }
    else r.v[0] = *p;
    return r;
}
// PAST: past the caches, see kPast
template <int V, bool PAST>
__device__ inline void store(float* p, const Vec<V>& r) {
    using vec = __attribute__((ext_vector_type(V))) float;
    vec t;
#pragma unroll
    for (int j = 0; j < V; ++j) t[j] = r.v[j];
    if (PAST) __builtin_nontemporal_store(t, reinterpret_cast<vec*>(p));
    else *reinterpret_cast<vec*>(p) = t;
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
    } else if (V == 2) {
        const uint32_t u = *reinterpret_cast<const uint16_t*>(a.codes + r * a.mp + c);
        const float f = mhckpt::scale_of(e);
        v.v[0] = mhckpt::decode1(u & 255u, f); v.v[V > 1 ? 1 : 0] = mhckpt::decode1(u >> 8, f);
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
    if (HELD && a.relu) {
        const uint8_t* m = a.mask + row * a.F + c;
        keep = V == 4 ? *reinterpret_cast<const uint32_t*>(m) : V == 2 ? *reinterpret_cast<const uint16_t*>(m) : *m;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const bool open = !a.relu || (HELD ? ((keep >> (8 * j)) & 255u) != 0u : result(k, 0, j, x[0].v[j]) >= 0.0f);
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            xh[p].v[j] = centred(k, p, j, x[p].v[j]) * k.rstd[j];
            dy[p].v[j] *= open ? 1.0f : 0.0f;                       // as the gate of mh_relu_bwd: what is not finite stays visible
        }
    }
}

// sums of a workgroup's rows, joined over the threads of a channel: part[s * V + j][unit], s of the three sums
template <int V>
__device__ inline void join_rows(const NormArgs& a, double (&part)[3 * V][kBlock], const double (&acc)[3][V]) {
    const int lanes = a.lanes, tid = threadIdx.x;
#pragma unroll
    for (int s = 0; s < 3; ++s)
#pragma unroll
        for (int j = 0; j < V; ++j) part[s * V + j][tid] = acc[s][j];
    for (int half = kBlock / 2; half >= lanes; half >>= 1) {
        __syncthreads();
        for (int i = tid; i < 3 * V * half; i += kBlock) {
            const int s = i / half, at = i - s * half;
            part[s][at] += part[s][at + half];
        }
    }
    __syncthreads();
}

template <int V>
__global__ void __launch_bounds__(kBlock) norm_sums_kernel(const NormArgs a) {
    const Piece p = piece_of(a, blockIdx.x);
    if (p.graph == a.graphs || p.lo >= p.hi) return;                // read by nobody
    const int32_t c = int32_t(blockIdx.y) * a.width + int32_t(threadIdx.x) % a.lanes * V;
    double acc[3][V] = {};
    if (c < a.F) {
        const int step = kBlock / a.lanes;
        double origin[2][V];
        const float* first = a.x + row_start(a, p.graph) * a.ld;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int32_t at = (c + j) / a.D * a.D;
            origin[0][j] = first[at]; origin[1][j] = first[a.im + at];
        }
#pragma unroll 4
        for (int64_t row = p.lo + threadIdx.x / a.lanes; row < p.hi; row += step) {
            const Vec<V> re = load<V>(a.x + row * a.ld + c), im = load<V>(a.x + row * a.ld + a.im + c);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const double r = re.v[j] - origin[0][j], i = im.v[j] - origin[1][j];
                acc[0][j] += r;
                acc[1][j] += i;
                acc[2][j] = fma(r, r, fma(i, i, acc[2][j]));
            }
        }
    }
    __shared__ double part[3 * V][kBlock];
    join_rows<V>(a, part, acc);
    // over the channels of a group: `each` threads for each sum of each group of this chunk
    const int32_t c0 = int32_t(blockIdx.y) * a.width, c1 = c0 + a.width < a.F ? c0 + a.width : a.F;
    const int32_t g0 = c0 / a.D, n = 3 * ((c1 - 1) / a.D - g0 + 1);
    int32_t each = 64;
    while (each > 1 && n * each > kBlock) each >>= 1;
    const int32_t turns = (n * each + kBlock - 1) / kBlock;
    for (int32_t t = 0; t < turns; ++t) {
        const int32_t i = (t * kBlock + int32_t(threadIdx.x)) / each, k = int32_t(threadIdx.x) % each, g = i / 3, s = i - 3 * g;
        double sum = 0.0;
        if (i < n) {
            const int32_t lo = (g0 + g) * a.D > c0 ? (g0 + g) * a.D - c0 : 0, hi = (g0 + g + 1) * a.D < c1 ? (g0 + g + 1) * a.D - c0 : c1 - c0;
            for (int32_t at = lo + k; at < hi; at += each) sum += part[s * V + at % V][at / V];
        }
        for (int o = each >> 1; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        if (i < n && k == 0) a.partial[(int64_t(blockIdx.x) * 3 + s) * a.chunks * a.slots + int32_t(blockIdx.y) * a.slots + g] = sum;
    }
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
    if (waves == 1) return;
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 3; ++s) {
        v[s] = 0.0;
        for (int w = 0; w < waves; ++w) v[s] += part[w][s];
    }
}

__device__ inline void leave_stats(const NormArgs& a, int32_t b, int32_t g, int64_t lo, int64_t n, const double (&v)[3]) {
    const double count = double(n) * a.D;
    double mr = n ? v[0] / count : 0.0, mi = n ? v[1] / count : 0.0;
    double var = n ? v[2] / count - mr * mr - mi * mi : 0.0;
    if (var < 0.0) var = 0.0;                                       // NaN stays
    if (n) {
        const float* first = a.x + lo * a.ld + g * a.D;
        mr += double(first[0]); mi += double(first[a.im]);
    }
    float* s = a.stats + (int64_t(b) * a.groups + g) * kStats;
    s[0] = float(mr); s[1] = float(mr - double(float(mr)));
    s[2] = float(mi); s[3] = float(mi - double(float(mi)));
    s[4] = float(1.0 / sqrt(var + double(a.eps)));
}

// one workgroup per (graph, group): a wave where a graph has few pieces, 16 where it has many
__global__ void __launch_bounds__(1024) norm_stats_kernel(const NormArgs a) {
    const int32_t b = blockIdx.x / a.groups, g = blockIdx.x - b * a.groups;
    const int64_t lo = row_start(a, b), hi = row_start(a, b + 1);
    double v[3] = {0.0, 0.0, 0.0};
    if (lo < hi) {
        int64_t d0, d1;
        pieces_of(a, b, lo, hi, d0, d1);
        const int32_t y0 = g * a.D / a.width, y1 = ((g + 1) * a.D - 1) / a.width, pitch = a.chunks * a.slots;
        for (int32_t y = y0; y <= y1; ++y) {
            const double* p = a.partial + d0 * 3 * pitch + y * a.slots + (g - y * a.width / a.D);
#pragma unroll 4
            for (int32_t d = threadIdx.x; d < int32_t(d1 - d0); d += blockDim.x) {
                const double* q = p + int64_t(d) * 3 * pitch;
                v[0] += q[0]; v[1] += q[pitch]; v[2] += q[2 * pitch];
            }
        }
    }
    join3(v);
    if (threadIdx.x == 0) leave_stats(a, b, g, lo, hi - lo, v);
}

// KEEP (V = 4, F a multiple of 32): also leaves a checkpoint of x, whose values are here anyway.  The 8 threads of a block of 32
// channels are neighbours; a node's two rows are two bytes of scales side by side.
template <int V, bool KEEP, bool PAST>
__global__ void __launch_bounds__(kBlock) norm_apply_kernel(const NormArgs a) {
    const Piece p = piece_of(a, gridDim.x - 1 - blockIdx.x);
    const int32_t c = int32_t(blockIdx.y) * a.width + int32_t(threadIdx.x) % a.lanes * V;
    if (c >= a.F || p.lo >= p.hi) return;
    const int step = kBlock / a.lanes;
    const bool behind = p.graph == a.graphs;
    const Channels<V> k = channels<V>(a, behind ? 0 : p.graph, c);
#pragma unroll 4
    for (int64_t row = p.lo + threadIdx.x / a.lanes; row < p.hi; row += step) {
        Vec<V> re = load<V>(a.x + row * a.ld + c), im = load<V>(a.x + row * a.ld + a.im + c);
        if (KEEP) {
            uint32_t top[2], e[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const Vec<V>& v = q ? im : re;
                const float4 f = make_float4(v.v[0], v.v[V > 1 ? 1 : 0], v.v[V > 2 ? 2 : 0], v.v[V > 3 ? 3 : 0]);
                top[q] = mhckpt::magnitude(f);
#pragma unroll
                for (int o = 1; o < 8; o <<= 1) { const uint32_t other = __shfl_xor(top[q], o); top[q] = other > top[q] ? other : top[q]; }
                e[q] = mhckpt::scale_byte(top[q]);
                *reinterpret_cast<uint32_t*>(a.codes_out + (2 * row + q) * a.mp + c) = mhckpt::encode(f, e[q]);
            }
            if ((c & (mhckpt::kBlockCols - 1)) == 0) {
                uint8_t* s = a.scales_out + int64_t(c / mhckpt::kBlockCols) * a.rp + 2 * row;
                *reinterpret_cast<uint16_t*>(s) = uint16_t(e[0] | (e[1] << 8));
                if (row == a.rows - 1)
                    for (int64_t r = 2 * a.rows; r < a.rp; ++r) s[r - 2 * row] = 0;
            }
        }
        uint32_t keep = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float yr = result(k, 0, j, re.v[j]), yi = result(k, 1, j, im.v[j]);
            // the gate multiplies, as the framework's complex ReLU does: what is not finite stays visible
            const float open = !a.relu || yr >= 0.0f ? 1.0f : 0.0f;
            re.v[j] = behind ? 0.0f : yr * open;
            im.v[j] = behind ? 0.0f : yi * open;
            keep |= uint32_t(open != 0.0f) << (8 * j);
        }
        store<V, PAST>(a.out + row * a.ldo + c, re);
        store<V, PAST>(a.out + row * a.ldo + a.imo + c, im);
        if (a.mask) {
            uint8_t* m = a.mask + row * a.F + c;
            if (V == 4) *reinterpret_cast<uint32_t*>(m) = keep;
            else if (V == 2) *reinterpret_cast<uint16_t*>(m) = uint16_t(keep);
            else *m = uint8_t(keep);
        }
    }
}

template <int V, bool HELD>
__global__ void __launch_bounds__(kBlock) norm_bwd_sums_kernel(const NormArgs a) {
    const Piece p = piece_of(a, blockIdx.x);
    if (p.graph == a.graphs || p.lo >= p.hi) return;
    const int32_t c = int32_t(blockIdx.y) * a.width + int32_t(threadIdx.x) % a.lanes * V;
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
    __shared__ double part[3 * V][kBlock];
    join_rows<V>(a, part, acc);
    for (int i = threadIdx.x; i < 3 * a.width; i += kBlock) {
        const int s = i / a.width, at = i - s * a.width, ch = int(blockIdx.y) * a.width + at;
        if (ch < a.F) a.partial[(int64_t(blockIdx.x) * 3 + s) * a.F + ch] = part[s * V + at % V][at / V];
    }
}

// per graph, share of its pieces and channel: the partial sums; 32 channels to a workgroup
__global__ void __launch_bounds__(1024) norm_bwd_channels_kernel(const NormArgs a) {
    __shared__ double part[3][32][33];
    const int32_t b = blockIdx.x, cl = threadIdx.x & 31, q = threadIdx.x >> 5, rows = blockDim.x >> 5, c = int32_t(blockIdx.y) * 32 + cl;
    const int64_t lo = row_start(a, b), hi = row_start(a, b + 1);
    double v[3] = {0.0, 0.0, 0.0};
    if (lo < hi && c < a.F) {
        int64_t d0, d1;
        pieces_of(a, b, lo, hi, d0, d1);
        const int64_t n = d1 - d0, first = d0 + n * blockIdx.z / gridDim.z, last = d0 + n * (blockIdx.z + 1) / gridDim.z;
#pragma unroll 4
        for (int64_t d = first + q; d < last; d += rows) {
            const double* p = a.partial + d * 3 * a.F + c;
            v[0] += p[0]; v[1] += p[a.F]; v[2] += p[2 * a.F];
        }
    }
#pragma unroll
    for (int s = 0; s < 3; ++s) part[s][q][cl] = v[s];
    __syncthreads();
    if (q < 3 && c < a.F) {
        double t = 0.0;
        for (int i = 0; i < rows; ++i) t += part[q][i][cl];
        a.sums[((int64_t(b) * a.parts + blockIdx.z) * 3 + q) * a.F + c] = t;
    }
}

// the first workgroups: a wave for each group of each graph, its means of dxh and of dxh xh; the others: dgamma and dbeta of 16
// channels
__global__ void __launch_bounds__(kBlock) norm_bwd_means_kernel(const NormArgs a) {
    const int32_t items = a.graphs * a.groups, first = (items + 3) / 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (int32_t(blockIdx.x) < first) {
        const int32_t item = int32_t(blockIdx.x) * 4 + wave;
        if (item >= items) return;
        const int32_t b = item / a.groups, g = item - b * a.groups;
        const int64_t n = row_start(a, b + 1) - row_start(a, b);
        double v[3] = {0.0, 0.0, 0.0};
        for (int32_t i = lane; i < a.D * a.parts; i += 64) {
            const int32_t part = i / a.D, c = g * a.D + (i - part * a.D);
            const double w = a.gamma ? double(a.gamma[c]) : 1.0;
            const double* s = a.sums + (int64_t(b) * a.parts + part) * 3 * a.F + c;
            v[0] += w * s[0]; v[1] += w * s[a.F]; v[2] += w * s[2 * a.F];
        }
        const double count = double(n > 0 ? n : 1) * a.D;
#pragma unroll
        for (int s = 0; s < 3; ++s) {
            for (int o = 32; o > 0; o >>= 1) v[s] += __shfl_xor(v[s], o);
            if (lane == 0) a.means[int64_t(item) * 3 + s] = float(v[s] / count);
        }
        return;
    }
    __shared__ double part[2][16][17];
    const int cl = threadIdx.x & 15, q = threadIdx.x >> 4;
    const int32_t c = (int32_t(blockIdx.x) - first) * 16 + cl;
    double w = 0.0, s = 0.0;
    if (c < a.F)
#pragma unroll 4
        for (int32_t i = q; i < a.graphs * a.parts; i += 16) {
            const double* p = a.sums + int64_t(i) * 3 * a.F + c;
            s += p[0] + p[a.F];
            w += p[2 * a.F];
        }
    part[0][q][cl] = w;
    part[1][q][cl] = s;
    __syncthreads();
    if (q == 0 && c < a.F) {
        for (int i = 1; i < 16; ++i) { w += part[0][i][cl]; s += part[1][i][cl]; }
        if (a.dgamma) a.dgamma[c] = float(w);
        if (a.dbeta) a.dbeta[c] = float(s);
    }
}

// (dxh - flat) - xh along with separate roundings: where a group's gradient is its mean, the difference is 0 and not the last
// bits of a product
__device__ inline float less_means(float gamma, float dy, float flat, float xh, float along) {
#pragma clang fp contract(off)
    const float dxh = gamma * dy, pull = xh * along;
    return (dxh - flat) - pull;
}

template <int V, bool HELD, bool PAST>
__global__ void __launch_bounds__(kBlock) norm_bwd_apply_kernel(const NormArgs a) {
    const Piece p = piece_of(a, gridDim.x - 1 - blockIdx.x);
    const int32_t c = int32_t(blockIdx.y) * a.width + int32_t(threadIdx.x) % a.lanes * V;
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
            store<V, PAST>(a.out + row * a.ldo + q * a.imo + c, d);
        }
    }
}

struct Layout {
    int32_t v, lanes, width, chunks, slots, parts, stats_threads, channel_threads;
    int64_t sum_rows, sum_pieces, rows, pieces;    // tiles of the pass for sums, of the elementwise one
};

Layout layout_of(int64_t rows, int32_t graphs, int32_t F, int32_t groups, int v) {
    Layout l;
    l.v = v;
    const int32_t units = (F + v - 1) / v;
    l.lanes = 1;
    while (l.lanes < 64 && l.lanes < units) l.lanes <<= 1;
    l.width = l.lanes * v;
    l.chunks = (F + l.width - 1) / l.width;
    const int32_t D = F / groups;
    l.slots = (l.width + D - 1) / D + 1 < groups ? (l.width + D - 1) / D + 1 : groups;
    const int64_t at_once = kBlock / l.lanes;
    auto tile = [&](int64_t tiles) { return ((rows + tiles - 1) / tiles + at_once - 1) / at_once * at_once; };
    l.sum_rows = rows > 0 ? tile(kSumTiles / l.chunks > 1 ? kSumTiles / l.chunks : 1) : at_once;
    // few rows: one turn of a workgroup's threads for each tile; more: 4 turns, the loads of which are in flight together; past
    // 65536 turns 2 (1M x 128: backward 516 us, with 4 turns 538, with 16 590; 200k x 64: 47 us against 43)
    l.rows = rows > 0 ? tile(kMostTiles) : at_once;
    const int64_t turns = rows / at_once;
    if (turns >= 4 * kSumTiles && l.rows < (turns > 65536 ? 2 : 4) * at_once) l.rows = (turns > 65536 ? 2 : 4) * at_once;
    l.sum_pieces = (rows + l.sum_rows - 1) / l.sum_rows + graphs;
    l.pieces = (rows + l.rows - 1) / l.rows + graphs;
    const int64_t each = l.sum_pieces / (graphs > 0 ? graphs : 1);
    l.stats_threads = each > 256 ? 1024 : 64;
    l.channel_threads = each > 64 ? 1024 : 256;
    // shares of a graph's pieces: enough workgroups for the GPU, 64 pieces at least to each
    const int64_t blocks = int64_t(graphs > 0 ? graphs : 1) * ((F + 31) / 32);
    l.parts = 1;
    while (l.parts < kMostParts && blocks * l.parts < 128 && each / (2 * l.parts) >= 64) l.parts <<= 1;
    return l;
}

struct Workspace {
    size_t partial, sums, means, bytes;
};

// sized for the largest of the layouts, so that it does not depend on a call's alignment
Workspace workspace_of(int64_t rows, int32_t graphs, int32_t F, int32_t groups) {
    size_t partial = 0, sums = 0;
    for (int v = 1; v <= 4; v <<= 1) {
        const Layout l = layout_of(rows, graphs, F, groups, v);
        const int64_t across = int64_t(l.chunks) * l.slots > F ? int64_t(l.chunks) * l.slots : F;
        const size_t p = size_t(l.sum_pieces) * 3 * across * sizeof(double), q = size_t(graphs) * l.parts * 3 * F * sizeof(double);
        partial = p > partial ? p : partial;
        sums = q > sums ? q : sums;
    }
    Workspace w;
    w.partial = 0;
    w.sums = w.partial + partial;
    w.means = w.sums + sums;
    w.bytes = w.means + (size_t(graphs) * groups * 3 * sizeof(float) + 15) / 16 * 16;
    return w;
}

int check_norm(int64_t rows, int32_t F, int32_t groups, const void* ptr, int32_t graphs) {
    MH_REQUIRE(rows >= 0 && rows <= INT32_MAX && F >= 1 && F <= kMostChannels, "n_rows=%lld F=%d", (long long)rows, F);
    MH_REQUIRE(groups >= 1 && F % groups == 0, "%d channels do not divide into %d groups", F, groups);
    MH_REQUIRE(graphs >= (rows > 0 ? 1 : 0) && graphs <= kMostGraphs && int64_t(graphs) * groups <= (int64_t(1) << 25), "n_graphs=%d", graphs);
    MH_REQUIRE(ptr || graphs <= 1, "n_graphs=%d without graph_ptr", graphs);
    return MH_OK;
}

// channels to a thread that a planar operand allows
int width_of(const void* p, int64_t ld, int64_t im) {
    const int64_t all = ld | im | int64_t(reinterpret_cast<uintptr_t>(p) >> 2);
    return (all & 3) == 0 ? 4 : (all & 1) == 0 ? 2 : 1;
}
int width_of(int32_t F) { return (F & 3) == 0 ? 4 : (F & 1) == 0 ? 2 : 1; }
int width_of(const uint8_t* mask) { return (reinterpret_cast<uintptr_t>(mask) & 3) == 0 ? 4 : (reinterpret_cast<uintptr_t>(mask) & 1) == 0 ? 2 : 1; }
int least(int a, int b) { return a < b ? a : b; }

void take_layout(NormArgs& a, const Layout& l) {
    a.lanes = l.lanes; a.width = l.width; a.chunks = l.chunks; a.slots = l.slots; a.parts = l.parts;
}

enum Pass { kSums, kApply, kApplyKeep, kBwdSums, kBwdSumsHeld, kBwdApply, kBwdApplyHeld };

template <int V, bool PAST>
void launch_pass(Pass pass, const dim3& grid, const NormArgs& a, hipStream_t stream) {
    switch (pass) {
        case kSums: norm_sums_kernel<V><<<grid, kBlock, 0, stream>>>(a); break;
        case kApply: norm_apply_kernel<V, false, PAST><<<grid, kBlock, 0, stream>>>(a); break;
        case kApplyKeep: norm_apply_kernel<4, true, PAST><<<grid, kBlock, 0, stream>>>(a); break;
        case kBwdSums: norm_bwd_sums_kernel<V, false><<<grid, kBlock, 0, stream>>>(a); break;
        case kBwdSumsHeld: norm_bwd_sums_kernel<V, true><<<grid, kBlock, 0, stream>>>(a); break;
        case kBwdApply: norm_bwd_apply_kernel<V, false, PAST><<<grid, kBlock, 0, stream>>>(a); break;
        case kBwdApplyHeld: norm_bwd_apply_kernel<V, true, PAST><<<grid, kBlock, 0, stream>>>(a); break;
    }
}

void run_pass(Pass pass, const Layout& l, NormArgs a, hipStream_t stream) {
    const bool sums = pass == kSums || pass == kBwdSums || pass == kBwdSumsHeld;
    a.tile_rows = sums ? l.sum_rows : l.rows;
    const dim3 grid(unsigned(sums ? l.sum_pieces : l.pieces), unsigned(l.chunks));
    if (l.v == 4 && 8 * a.rows * a.F >= kPast) launch_pass<4, true>(pass, grid, a, stream);
    else if (l.v == 4) launch_pass<4, false>(pass, grid, a, stream);
    else if (l.v == 2) launch_pass<2, false>(pass, grid, a, stream);
    else launch_pass<1, false>(pass, grid, a, stream);
}

}  // namespace

extern "C" size_t mh_group_norm_workspace_bytes(int64_t n_rows, int32_t n_graphs, int32_t F, int32_t groups) {
    if (n_rows < 0 || n_rows > INT32_MAX || n_graphs < 0 || n_graphs > kMostGraphs || F < 1 || F > kMostChannels || groups < 1 || F % groups) return 0;
    return workspace_of(n_rows, n_graphs, F, groups).bytes;
}

extern "C" int mh_group_norm(const float* X, int64_t ld, int64_t im, int64_t n_rows, int32_t F, int32_t groups,
                             const int32_t* graph_ptr, int32_t n_graphs, float eps, const float* gamma, const float* beta, int relu,
                             float* Y, int64_t ldy, int64_t imy, uint8_t* mask_out, uint8_t* codes_out, uint8_t* scales_out,
                             float* stats, void* workspace, size_t workspace_bytes, void* stream_) {
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    if (int rc = check_norm(n_rows, F, groups, graph_ptr, n_graphs)) return rc;
    if (n_rows == 0) return MH_OK;
    MH_REQUIRE(X && Y && stats && workspace && !codes_out == !scales_out, "null pointer");
    MH_REQUIRE(ld >= 0 && im >= 0 && ldy >= F && imy >= F, "stride smaller than F");
    const Workspace w = workspace_of(n_rows, n_graphs, F, groups);
    if (workspace_bytes < w.bytes) return mh::fail(MH_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, w.bytes);
    MH_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 7) == 0, "workspace must be 8-byte aligned");
    const int v = least(least(width_of(F), width_of(mask_out)), least(width_of(X, ld, im), width_of(Y, ldy, imy)));
    const Layout l = layout_of(n_rows, n_graphs, F, groups, v);
    NormArgs a{};
    a.x = X; a.ld = ld; a.im = im; a.rows = n_rows; a.F = F; a.groups = groups; a.D = F / groups;
    a.graphs = n_graphs; a.ptr = graph_ptr; a.eps = eps; a.gamma = gamma; a.beta = beta; a.relu = relu ? 1 : 0; a.stats = stats;
    a.partial = reinterpret_cast<double*>(static_cast<char*>(workspace) + w.partial);
    a.out = Y; a.ldo = ldy; a.imo = imy; a.mask = relu ? mask_out : nullptr;
    a.rp = (2 * n_rows + 7) & ~int64_t(7); a.mp = (F + 31) & ~31; a.codes_out = codes_out; a.scales_out = scales_out;
    take_layout(a, l);
    const bool joined = codes_out && l.v == 4 && F % mhckpt::kBlockCols == 0;
    if (codes_out && !joined)
        if (int rc = mh_ckpt_store(X, ld, im, n_rows, F, codes_out, scales_out, stream_)) return rc;
    if (joined) MH_REQUIRE((reinterpret_cast<uintptr_t>(codes_out) & 3) == 0 && (reinterpret_cast<uintptr_t>(scales_out) & 7) == 0,
                           "codes must be 4-byte and scales 8-byte aligned");
    run_pass(kSums, l, a, stream);
    a.tile_rows = l.sum_rows;
    norm_stats_kernel<<<unsigned(n_graphs) * unsigned(groups), l.stats_threads, 0, stream>>>(a);
    run_pass(joined ? kApplyKeep : kApply, l, a, stream);
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
    MH_REQUIRE(!any || ((held ? scales && (!relu || mask) : X != nullptr) && G && stats), "null pointer");
    MH_REQUIRE(workspace, "null pointer");
    MH_REQUIRE(ld >= 0 && im >= 0 && ldg >= 0 && img >= 0 && (!any || !dX || (lddx >= F && imdx >= F)), "stride smaller than F");
    const Workspace w = workspace_of(n_rows, n_graphs, F, groups);
    if (workspace_bytes < w.bytes) return mh::fail(MH_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, w.bytes);
    MH_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 7) == 0, "workspace must be 8-byte aligned");
    MH_REQUIRE((reinterpret_cast<uintptr_t>(codes) & 3) == 0, "codes must be 4-byte aligned");
    int v = least(width_of(F), width_of(G, ldg, img));
    v = least(v, held ? width_of(mask) : width_of(X, ld, im));
    if (dX) v = least(v, width_of(dX, lddx, imdx));
    const Layout l = layout_of(n_rows, n_graphs, F, groups, v);
    NormArgs a{};
    a.x = X; a.ld = ld; a.im = im; a.codes = codes; a.scales = scales; a.rp = (2 * n_rows + 7) & ~int64_t(7); a.mp = (F + 31) & ~31;
    a.rows = n_rows; a.F = F; a.groups = groups; a.D = F / groups; a.graphs = n_graphs; a.ptr = graph_ptr;
    a.gamma = gamma; a.beta = beta; a.relu = relu ? 1 : 0; a.stats = const_cast<float*>(stats);
    a.partial = reinterpret_cast<double*>(static_cast<char*>(workspace) + w.partial);
    a.sums = reinterpret_cast<double*>(static_cast<char*>(workspace) + w.sums);
    a.means = reinterpret_cast<float*>(static_cast<char*>(workspace) + w.means);
    a.g = G; a.ldg = ldg; a.img = img; a.out = dX; a.ldo = lddx; a.imo = imdx; a.mask = const_cast<uint8_t*>(mask);
    a.dgamma = dgamma; a.dbeta = dbeta;
    take_layout(a, l);
    a.tile_rows = l.sum_rows;
    if (any) run_pass(held ? kBwdSumsHeld : kBwdSums, l, a, stream);
    // one graph of few pieces: the pieces are the shares, and need no joining first (2500 x 16: one launch of four)
    const int64_t tiles = l.sum_pieces - n_graphs;
    if (any && n_graphs == 1 && !graph_ptr && tiles <= kFewPieces) {
        a.sums = a.partial;
        a.parts = int32_t(tiles);
    } else if (n_graphs > 0)
        norm_bwd_channels_kernel<<<dim3(unsigned(n_graphs), unsigned((F + 31) / 32), unsigned(l.parts)), l.channel_threads, 0, stream>>>(a);
    norm_bwd_means_kernel<<<unsigned((n_graphs * groups + 3) / 4) + unsigned((F + 15) / 16), kBlock, 0, stream>>>(a);
    if (any && dX) run_pass(held ? kBwdApplyHeld : kBwdApply, l, a, stream);
    MH_LAUNCH_CHECK("group_norm_bwd");
    return MH_OK;
}
