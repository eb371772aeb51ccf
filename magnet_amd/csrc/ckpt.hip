// Activation checkpoints in 8 bits, and the weight gradient taken from them.
//
// Format.  A row-planar matrix [N][2][m] is seen as R = 2N rows of m columns; 32 neighbouring columns of a row share a
// power-of-two scale 2^s.  With the block's largest magnitude f 2^p, f in [1/2, 1), s = p - 7, or p - 6 where rounding would
// reach 128; -110 <= s <= 121.  code = rint(x / 2^s) (ties to even) lies in -127 .. 127 and is kept as code + 128.
//     codes  uint8 [R][mp], mp = m rounded up to 32 (the columns behind m hold 128)
//     scales uint8 [mp / 32][Rp], s + 128, Rp = R rounded up to 8 (the rows behind R hold 0); 0: a value of the block was not
//            finite, and the whole block (of codes 128) is restored as NaN
// The error of a value is at most 2^s / 2: between 1 / 255 and 1 / 127.5 of its block's largest magnitude.  At the ends of s: a block
// below 2^-103 keeps multiples of 2^-110, and a magnitude from 127.5 2^121 on is held at 127 2^121, up to a whole 2^s away (64 2^122
// would leave float32).  A power of two costs up to one bit against a free scale and buys that code * 2^s is exact in bf16 (7 bits): the weight gradient runs on
// the bf16 matrix cores without a further rounding of the activations.  The scales of 8 consecutive rows are 8 consecutive
// bytes: one load for a thread that holds 8 rows of a block.
#include <cstdint>

#include <hip/hip_runtime.h>

#include "ckpt.h"
#include "common.h"

namespace {

using mhckpt::kBlockCols;
constexpr int kBlock = 256;
constexpr unsigned kMostBlocks = 1u << 16;

// ---- store / restore -------------------------------------------------------------------------------------------------
// A thread holds 4 columns of 8 consecutive rows (4 nodes): 8 independent 16-byte accesses, the 8 scales of its block as one
// 8-byte word, written by the first of the 8 threads that share a block.  Bound by HBM.  Float32 matrices from kPast bytes on are
// read and written past the caches (PAST), which leaves these to the bytes of the checkpoint: 500k x 2 x 384 is stored in 314 us
// (395 without) and restored in 357 us (320), 5.4 and 5.7 TB/s together.
constexpr int64_t kPast = int64_t(64) << 20;
using f4 = __attribute__((ext_vector_type(4))) float;
struct PlanarArgs {
    float* x;
    int64_t ld, im;
    int64_t rows, rp;                       // rows = 2 N
    int32_t m, mp;
    uint8_t *codes, *scales;
};

template <bool VEC, bool PAST>
__device__ inline float4 load4(const float* p, int32_t c, int32_t m) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (VEC) {
        if (c < m) {
            const f4* q = reinterpret_cast<const f4*>(p + c);
            const f4 t = PAST ? __builtin_nontemporal_load(q) : *q;
            v = make_float4(t[0], t[1], t[2], t[3]);
        }
    } else {
        if (c < m) v.x = p[c];
        if (c + 1 < m) v.y = p[c + 1];
        if (c + 2 < m) v.z = p[c + 2];
        if (c + 3 < m) v.w = p[c + 3];
    }
    return v;
}

template <bool VEC, bool PAST>
__global__ void __launch_bounds__(kBlock) ckpt_store_kernel(const PlanarArgs a) {
    const int32_t quads = a.mp >> 2;
    const int64_t total = (a.rp >> 3) * quads;                     // a multiple of 8: the 8 threads of a block stay together
    for (int64_t t = int64_t(blockIdx.x) * kBlock + threadIdx.x; t < total; t += int64_t(gridDim.x) * kBlock) {
        const int64_t oct = t / quads;
        const int32_t c = int32_t(t - oct * quads) << 2;
        const int64_t r0 = oct << 3;
        float4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int64_t r = r0 + k;
            v[k] = r < a.rows ? load4<VEC, PAST>(a.x + (r >> 1) * a.ld + (k & 1) * a.im, c, a.m) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        uint64_t word = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            uint32_t top = mhckpt::magnitude(v[k]);
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) { const uint32_t other = __shfl_xor(top, o); top = other > top ? other : top; }
            const uint32_t e = mhckpt::scale_byte(top);
            if (r0 + k < a.rows) {
                *reinterpret_cast<uint32_t*>(a.codes + (r0 + k) * a.mp + c) = mhckpt::encode(v[k], e);
                word |= uint64_t(e) << (8 * k);
            }
        }
        if ((c & (kBlockCols - 1)) == 0) *reinterpret_cast<uint64_t*>(a.scales + int64_t(c / kBlockCols) * a.rp + r0) = word;
    }
}

template <bool VEC, bool PAST>
__global__ void __launch_bounds__(kBlock) ckpt_restore_kernel(const PlanarArgs a) {
    const int32_t quads = (a.m + 3) >> 2;
    const int64_t total = (a.rp >> 3) * quads;
    for (int64_t t = int64_t(blockIdx.x) * kBlock + threadIdx.x; t < total; t += int64_t(gridDim.x) * kBlock) {
        const int64_t oct = t / quads;
        const int32_t c = int32_t(t - oct * quads) << 2;
        const int64_t r0 = oct << 3;
        const uint64_t word = *reinterpret_cast<const uint64_t*>(a.scales + int64_t(c / kBlockCols) * a.rp + r0);
        uint32_t code[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) code[k] = r0 + k < a.rows ? *reinterpret_cast<const uint32_t*>(a.codes + (r0 + k) * a.mp + c) : 0u;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (r0 + k >= a.rows) break;
            const float4 v = mhckpt::decode(code[k], uint32_t(word >> (8 * k)) & 255u);
            float* p = a.x + ((r0 + k) >> 1) * a.ld + (k & 1) * a.im;
            if (VEC) {
                const f4 t = {v.x, v.y, v.z, v.w};
                if (PAST) __builtin_nontemporal_store(t, reinterpret_cast<f4*>(p + c));
                else *reinterpret_cast<f4*>(p + c) = t;
            } else {
                p[c] = v.x;
                if (c + 1 < a.m) p[c + 1] = v.y;
                if (c + 2 < a.m) p[c + 2] = v.z;
                if (c + 3 < a.m) p[c + 3] = v.w;
            }
        }
    }
}

// ---- weight gradient -------------------------------------------------------------------------------------------------
// out[i][j] = sum_r A[r][i] G[r][j]: A the decoded checkpoint [R][m], G float32 [R][n].
//
// A is exact in bf16; G is cut into three bf16 numbers g1 + g2 + g3 = g, each the next 8 bits of its significand (exact): three
// bf16 matrix products with 32-bit sums give the float32 product at 3 / 16 of the cost of the float32 matrix instruction.
//
// The sum runs over millions of rows and the result is small, so the rows are cut into slabs; a workgroup takes one slab and
// one BM x BN tile of the result and leaves a partial sum, a second kernel adds the slabs in order (64 bits; no atomics, the
// same result every time).  Both operands are row-major and the sum runs down the rows, so a thread gathers 8 consecutive rows
// of its columns (coalesced across the threads), converts them in registers and writes them to LDS as the 16 bytes that one
// lane of the matrix instruction takes: layout [rows / 8][column][8], written and read as contiguous 16-byte accesses without
// bank conflicts.  A thread decodes 4 neighbouring columns of A; column 4 u + q goes to place q BM / 4 + u (contiguous writes),
// which permutes the rows of the tile and is undone when the slabs are added.
//
// A step takes 32 rows.  Its loads were issued three steps before, its conversion (2.5 instructions per value of A, 5.5 per
// value of G) ran between the matrix instructions of the step before.  Conversion of G is repeated for every tile across A's
// columns, hence the wide tiles: 2M x 384 with 128 columns of G takes 0.58 ms in one 384-wide tile, 1.27 ms in three of 128 with
// one step in flight.  That is 1.0 PFLOP/s of bf16 products, what the library's largest bf16 product reaches on this card (1.1):
// the matrix unit bounds it, at the clock it runs at under that load (1.9 GHz).  Narrow results (30 columns) run at 4.3 TB/s.
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f32x16 = __attribute__((ext_vector_type(16))) float;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;

struct GramArgs {
    const uint8_t *codes, *scales;
    const float* g;
    int64_t ldg, img, rows, rp, slab_rows;
    int32_t m, mp, n, slabs, tiles_m, tiles_n;
    float* partial;
};

// the high halves (bf16 by truncation) of two floats in one word
__device__ inline uint32_t high_halves(float lo, float hi) { return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u); }
__device__ inline float cut(float v) { return __uint_as_float(__float_as_uint(v) & 0xffff0000u); }
// address = uniform base + 32-bit offset of the thread: one load instruction, its base kept by the scalar unit
template <class T>
__device__ inline T at(const void* base, uint32_t offset) { return *reinterpret_cast<const T*>(static_cast<const char*>(base) + offset); }

constexpr int kRows = 32;                  // rows of a step
constexpr int64_t kLeast = 128;            // rows of a slab: below, the sums to join cost more than the rows

template <int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN, 2) ckpt_gram_kernel(const GramArgs a) {
    constexpr int threads = 64 * WM * WN, kg = kRows / 8;
    constexpr int ta = BM / 4 * kg, tb = BN * kg;                   // conversion tasks of a step: 8 rows x 4 columns, 8 rows x 1
    constexpr int na = (ta + threads - 1) / threads, nb = (tb + threads - 1) / threads;
    constexpr int kFill = (na * 110 + nb * 60) / ((BM / 32 / WM) * (BN / 32 / WN) * 3 * kg / 2) + 1;
    constexpr int mi = BM / 32 / WM, ni = BN / 32 / WN;             // 32 x 32 products of a wave
    __shared__ __align__(16) uint16_t as[2][kg][BM][8];
    __shared__ __align__(16) uint16_t bs[2][3][kg][BN][8];

    // workgroups go to the XCDs in turn: the tiles of a slab are given to one XCD, whose L2 then serves the slab's rows to all
    const int32_t tiles = a.tiles_m * a.tiles_n;
    const int32_t slab = int32_t(blockIdx.x / (8 * tiles)) * 8 + int32_t(blockIdx.x & 7);
    const int32_t tile = int32_t(blockIdx.x >> 3) % tiles;
    if (slab >= a.slabs) return;
    const int32_t i0 = (tile % a.tiles_m) * BM, j0 = (tile / a.tiles_m) * BN;
    const int64_t r_begin = slab * a.slab_rows;
    const int64_t r_end = r_begin + a.slab_rows < a.rows ? r_begin + a.slab_rows : a.rows;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = (wave / WN) * (BM / WM), wc = (wave % WN) * (BN / WN);

    uint32_t code[2][na][8];
    uint64_t word[2][na];
    float gv[2][nb][8];
    // what lies behind the last column of A or G is read from the last one: its products end in places of the tile nobody reads
    uint32_t offset_a[na], offset_b[nb];
    const uint8_t* scale_at[na];
    int k_a[na], k_b[nb];
#pragma unroll
    for (int u = 0; u < na; ++u) {
        const int t = u * threads + tid;
        int32_t c = i0 + (t % (BM / 4)) * 4;
        c = c < a.mp ? c : a.mp - 4;
        k_a[u] = t / (BM / 4) % kg;
        offset_a[u] = uint32_t(k_a[u] * 8) * uint32_t(a.mp) + uint32_t(c);
        scale_at[u] = a.scales + int64_t(c / kBlockCols) * a.rp + k_a[u] * 8;
    }
#pragma unroll
    for (int u = 0; u < nb; ++u) {
        const int t = u * threads + tid;
        int32_t j = j0 + t % BN;
        j = j < a.n ? j : a.n - 1;
        k_b[u] = t / BN % kg;
        offset_b[u] = (uint32_t(k_b[u] * 4) * uint32_t(a.ldg) + uint32_t(j)) * 4u;
    }
    // where there are fewer tasks than threads, the threads that are left do the first ones again and write the same: without
    // branches a step is one block, in which conversions and products are scheduled into each other
    auto load = [&](int set, int64_t r0) {
        const uint8_t* codes = a.codes + r0 * a.mp;
        const float* g = a.g + (r0 >> 1) * a.ldg;
#pragma unroll
        for (int u = 0; u < na; ++u) {
            word[set][u] = *reinterpret_cast<const uint64_t*>(scale_at[u] + r0);
#pragma unroll
            for (int q = 0; q < 8; ++q) code[set][u][q] = at<uint32_t>(codes + int64_t(q) * a.mp, offset_a[u]);
        }
#pragma unroll
        for (int u = 0; u < nb; ++u)
#pragma unroll
            for (int q = 0; q < 8; ++q) gv[set][u][q] = at<float>(g + (q >> 1) * a.ldg + (q & 1) * a.img, offset_b[u]);
    };
    // the rows behind the last whole step
    auto load_rest = [&](int64_t r0) {
#pragma unroll
        for (int u = 0; u < na; ++u) {
            const int64_t left = r_end - (r0 + k_a[u] * 8);
            word[0][u] = left > 0 ? *reinterpret_cast<const uint64_t*>(scale_at[u] + r0) : 0;
            for (int q = 0; q < 8; ++q) {
                code[0][u][q] = q < left ? at<uint32_t>(a.codes + (r0 + q) * a.mp, offset_a[u]) : 0x80808080u;
                if (q >= left) word[0][u] = (word[0][u] & ~(uint64_t(255) << (8 * q))) | (uint64_t(1) << (8 * q));       // scale 0
            }
        }
#pragma unroll
        for (int u = 0; u < nb; ++u) {
            const int64_t left = r_end - (r0 + k_b[u] * 8);
            const float* g = a.g + (r0 >> 1) * a.ldg;
            for (int q = 0; q < 8; ++q) gv[0][u][q] = q < left ? at<float>(g + (q >> 1) * a.ldg + (q & 1) * a.img, offset_b[u]) : 0.0f;
        }
    };
    auto stage = [&](int set, int buf) {
#pragma unroll
        for (int u = 0; u < na; ++u) {
            const int t = u * threads + tid;
            float s[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) s[q] = mhckpt::scale_of(uint32_t(word[set][u] >> (8 * q)) & 255u);
#pragma unroll
            for (int q = 0; q < 8; ++q) code[set][u][q] ^= 0x80808080u;                             // two's complement
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                u32x4 w;
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    w[q] = high_halves(float(int8_t(code[set][u][2 * q] >> (8 * c))) * s[2 * q], float(int8_t(code[set][u][2 * q + 1] >> (8 * c))) * s[2 * q + 1]);
                *reinterpret_cast<u32x4*>(&as[buf][t / (BM / 4) % kg][c * (BM / 4) + t % (BM / 4)][0]) = w;
            }
        }
#pragma unroll
        for (int u = 0; u < nb; ++u) {
            const int t = u * threads + tid;
            u32x4 w[3];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float x1 = gv[set][u][2 * q], y1 = gv[set][u][2 * q + 1];
                const float x2 = x1 - cut(x1), y2 = y1 - cut(y1);
                const float x3 = x2 - cut(x2), y3 = y2 - cut(y2);
                w[0][q] = high_halves(x1, y1);
                w[1][q] = high_halves(x2, y2);
                w[2][q] = high_halves(x3, y3);
            }
#pragma unroll
            for (int s = 0; s < 3; ++s) *reinterpret_cast<u32x4*>(&bs[buf][s][t / BN % kg][t % BN][0]) = w[s];
        }
    };

    f32x16 acc[mi][ni];
#pragma unroll
    for (int i = 0; i < mi; ++i)
#pragma unroll
        for (int j = 0; j < ni; ++j)
#pragma unroll
            for (int k = 0; k < 16; ++k) acc[i][j][k] = 0.0f;
    auto product = [&](int buf, int k) {                            // 16 rows: lanes 0-31 take the first 8, lanes 32-63 the others
        bf16x8 af[mi];
#pragma unroll
        for (int i = 0; i < mi; ++i) af[i] = *reinterpret_cast<const bf16x8*>(&as[buf][k + (lane >> 5)][wr + i * 32 + (lane & 31)][0]);
#pragma unroll
        for (int j = 0; j < ni; ++j)
#pragma unroll
            for (int s = 2; s >= 0; --s) {                          // the smallest part first
                const bf16x8 bf = *reinterpret_cast<const bf16x8*>(&bs[buf][s][k + (lane >> 5)][wc + j * 32 + (lane & 31)][0]);
#pragma unroll
                for (int i = 0; i < mi; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(af[i], bf, acc[i][j], 0, 0, 0);
            }
    };

    // LDS holds two steps: while the products of one are made, the next is converted into the other half, and the two after
    // that are on their way into registers.  Past the last whole step the loads repeat it and what they bring is not used.
    const int64_t whole = (r_end - r_begin) / kRows;
    if (whole > 0) {
        const int64_t last = r_begin + (whole - 1) * kRows;
        auto row = [&](int64_t k) { const int64_t r = r_begin + k * kRows; return r < last ? r : last; };
        auto step = [&](int buf, int64_t k) {
            product(buf, 0);
            stage(buf ^ 1, buf ^ 1);
            load(buf ^ 1, row(k + 3));
            product(buf, 2);
            // a matrix instruction, then what the vector unit can do while it runs
#pragma unroll
            for (int i = 0; i < mi * ni * 3 * kg / 2; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, kFill, 0);
            }
            __syncthreads();
        };
        load(0, row(0));
        load(1, row(1));
        stage(0, 0);
        load(0, row(2));
        __syncthreads();
        int64_t k = 0;
        for (; k + 1 < whole; k += 2) {
            step(0, k);
            step(1, k + 1);
        }
        if (k < whole) step(0, k);
    }
    if (r_begin + whole * kRows < r_end) {
        __syncthreads();
        load_rest(r_begin + whole * kRows);
        stage(0, 0);
        __syncthreads();
        product(0, 0);
        product(0, 2);
    }
    float* out = a.partial + (int64_t(slab) * tiles + tile) * (BM * BN);
#pragma unroll
    for (int i = 0; i < mi; ++i)
#pragma unroll
        for (int j = 0; j < ni; ++j)
#pragma unroll
            for (int k = 0; k < 16; ++k)
                out[(wr + i * 32 + 8 * (k >> 2) + 4 * (lane >> 5) + (k & 3)) * BN + wc + j * 32 + (lane & 31)] = acc[i][j][k];
}

// The slabs' partial sums: O results to a workgroup, 1024 / O threads to a result, each with every so many-th slab, joined in a
// fixed order.  16 where the result is small, for more workgroups (940 slabs of 120 x 30: 8.7 us, with 64 results 10.4), else 64,
// for whole lines (256 slabs of 384 x 128: 11 us, with 16 results 21).
constexpr int kJoin = 1024;
template <int O>
__global__ void __launch_bounds__(kJoin) ckpt_gram_join(const float* __restrict__ partial, int32_t slabs, int32_t tiles_m, int32_t tiles_n,
                                                        int32_t bm, int32_t bn, int32_t m, int32_t n, float* __restrict__ out) {
    __shared__ double part[kJoin / 64][O];
    const int o = threadIdx.x % O, q = threadIdx.x / O, wave = threadIdx.x >> 6;
    const int32_t e = int32_t(blockIdx.x) * O + o;
    const bool in = e < m * n;
    double sum = 0.0;
    if (in) {
        const int32_t i = e / n, j = e - i * n;
        const int32_t tile = i / bm + (j / bn) * tiles_m, ii = i % bm;
        const float* p = partial + int64_t(tile) * bm * bn + ((ii & 3) * (bm / 4) + (ii >> 2)) * bn + j % bn;
        const int64_t step = int64_t(tiles_m) * tiles_n * bm * bn;
#pragma unroll 8
        for (int32_t s = q; s < slabs; s += kJoin / O) sum += double(p[s * step]);
    }
#pragma unroll
    for (int k = O; k < 64; k <<= 1) sum += __shfl_xor(sum, k);
    if ((threadIdx.x & 63) < O) part[wave][o] = sum;
    __syncthreads();
    if (threadIdx.x < O && in) {
        for (int w = 1; w < kJoin / 64; ++w) sum += part[w][o];
        out[e] = float(sum);
    }
}

struct GramPlan {
    int32_t bm, bn, tiles_m, tiles_n, slabs;
    int64_t slab_rows;
};

constexpr int64_t kMostResults = int64_t(1) << 24;        // m n: what follows counts tiles and their workgroups in 32 bits
constexpr int64_t kMostNodes = int64_t(1) << 40;          // more than any memory; products with sizes and strides stay in 64 bits

// Tile: 64 or 128 rows of a small result, 256 up to 256 columns, beyond 768 and for narrow results, else 384; 32, 64 or 128 columns.
// 384 rows take 257 to 384 columns with one conversion of G (1M x 384 x 128: 597 us).  Past 384 columns they need two, as 256 rows do up
// to 512 and with a third of the tiles or more empty: 1M x 512 x 128 takes 1380 us, in tiles of 256 766 us; 768 columns 1410 to 1470 and 1395 us.
GramPlan gram_plan(int64_t rows, int32_t m, int32_t n) {
    GramPlan p;
    const int32_t mp = (m + 31) & ~31;
    p.bm = mp <= 64 && n <= 64 ? 64 : mp <= 128 ? 128 : mp <= 256 || n <= 64 || mp > 768 ? 256 : 384;
    p.bn = n <= 32 ? 32 : n <= 64 ? 64 : 128;
    p.tiles_m = (mp + p.bm - 1) / p.bm;
    p.tiles_n = (n + p.bn - 1) / p.bn;
    // workgroups that a CU holds at once (registers and LDS of the tile); no more, or the last ones run alone
    const int32_t held = p.bm == 384 ? 1 : p.bn == 128 ? 2 : p.bm == 256 ? (p.bn == 32 ? 3 : 2) : 4;
    const int64_t want = (256 * held) / (p.tiles_m * p.tiles_n);
    int64_t each = want > 1 ? (rows + want - 1) / want : rows;
    // A sum in the matrix unit's 32 bits runs over 1024 rows of a small tile and bm bn / 4 of a larger one (16 bytes of partial sums
    // to a row), as long as all of them take 64 MB at most: 1.4M nodes x 3 x 46 are off by
    // 9e-7 of the result in 201 us, in slabs of 2816 rows by 1.5e-6 in 182 us.  384 x 128 tiles sum 12288 rows: 1M nodes are off by
    // 1.6e-6, a float32 product over slabs of 16384 rows by 1.5e-6.
    const int64_t results = int64_t(p.tiles_m) * p.tiles_n * p.bm * p.bn, most = (int64_t(1) << 24) / results;
    const int64_t fits = most > 1 ? (rows + most - 1) / most : rows, tile = p.bm * p.bn / 4 > 1024 ? p.bm * p.bn / 4 : 1024;
    const int64_t longest = fits > tile ? fits : tile;
    each = each < longest ? each : longest;
    each = (each + kRows - 1) / kRows * kRows;
    // half of that where there would be few slabs (5000 x 48 x 16: 9.3 us, with 128 rows 10.4, with 256 12.4)
    const int64_t least = rows < 64 * kLeast ? kLeast / 2 : kLeast;
    p.slab_rows = each < least ? least : each;
    p.slabs = int32_t((rows + p.slab_rows - 1) / p.slab_rows);
    return p;
}

template <int BM, int BN, int WM, int WN>
void launch_gram(const GramArgs& a, hipStream_t stream) {
    const unsigned blocks = unsigned((a.slabs + 7) / 8 * 8) * unsigned(a.tiles_m * a.tiles_n);
    ckpt_gram_kernel<BM, BN, WM, WN><<<blocks, 64 * WM * WN, 0, stream>>>(a);
}

unsigned grid_of(int64_t items) {
    const int64_t b = (items + kBlock - 1) / kBlock;
    return unsigned(b < 1 ? 1 : b > kMostBlocks ? kMostBlocks : b);
}

bool vec_ok(const float* x, int64_t ld, int64_t im, int32_t m) { return (m & 3) == 0 && (ld & 3) == 0 && (im & 3) == 0 && mh_aligned16(x); }

int check_checkpoint(const void* codes, const void* scales, int64_t n_rows, int32_t m) {
    MH_REQUIRE(n_rows >= 0 && n_rows <= kMostNodes && m >= 1 && m <= (1 << 24), "n_rows=%lld m=%d", (long long)n_rows, m);
    if (n_rows == 0) return MH_OK;
    MH_REQUIRE(codes && scales, "null pointer");
    MH_REQUIRE((reinterpret_cast<uintptr_t>(codes) & 3) == 0 && (reinterpret_cast<uintptr_t>(scales) & 7) == 0,
               "codes must be 4-byte and scales 8-byte aligned");
    return MH_OK;
}

PlanarArgs planar_args(float* x, int64_t ld, int64_t im, int64_t n_rows, int32_t m, uint8_t* codes, uint8_t* scales) {
    PlanarArgs a{};
    a.x = x; a.ld = ld; a.im = im; a.rows = 2 * n_rows; a.rp = (a.rows + 7) & ~int64_t(7); a.m = m; a.mp = (m + 31) & ~31;
    a.codes = codes; a.scales = scales;
    return a;
}

}  // namespace

extern "C" int mh_ckpt_store(const float* X, int64_t ld, int64_t im, int64_t n_rows, int32_t m, uint8_t* codes, uint8_t* scales,
                             void* stream_) {
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    if (int rc = check_checkpoint(codes, scales, n_rows, m)) return rc;
    if (n_rows == 0) return MH_OK;
    MH_REQUIRE(X, "null pointer");
    MH_REQUIRE(ld >= 0 && im >= 0, "negative stride");
    const PlanarArgs a = planar_args(const_cast<float*>(X), ld, im, n_rows, m, codes, scales);
    const unsigned grid = grid_of((a.rp >> 3) * (a.mp >> 2));
    const bool vec = vec_ok(X, ld, im, m);
    if (vec && 8 * n_rows * m >= kPast) ckpt_store_kernel<true, true><<<grid, kBlock, 0, stream>>>(a);
    else if (vec) ckpt_store_kernel<true, false><<<grid, kBlock, 0, stream>>>(a);
    else ckpt_store_kernel<false, false><<<grid, kBlock, 0, stream>>>(a);
    MH_LAUNCH_CHECK("ckpt_store");
    return MH_OK;
}

extern "C" int mh_ckpt_restore(const uint8_t* codes, const uint8_t* scales, int64_t n_rows, int32_t m, float* X, int64_t ld, int64_t im,
                               void* stream_) {
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    if (int rc = check_checkpoint(codes, scales, n_rows, m)) return rc;
    if (n_rows == 0) return MH_OK;
    MH_REQUIRE(X, "null pointer");
    MH_REQUIRE(ld >= m && im >= m, "stride smaller than m");
    const PlanarArgs a = planar_args(X, ld, im, n_rows, m, const_cast<uint8_t*>(codes), const_cast<uint8_t*>(scales));
    const unsigned grid = grid_of((a.rp >> 3) * ((m + 3) >> 2));
    const bool vec = vec_ok(X, ld, im, m);
    if (vec && 8 * n_rows * m >= kPast) ckpt_restore_kernel<true, true><<<grid, kBlock, 0, stream>>>(a);
    else if (vec) ckpt_restore_kernel<true, false><<<grid, kBlock, 0, stream>>>(a);
    else ckpt_restore_kernel<false, false><<<grid, kBlock, 0, stream>>>(a);
    MH_LAUNCH_CHECK("ckpt_restore");
    return MH_OK;
}

extern "C" size_t mh_ckpt_gram_workspace_bytes(int64_t n_rows, int32_t m, int32_t n) {
    if (n_rows <= 0 || n_rows > kMostNodes || m < 1 || n < 1 || int64_t(m) * n > kMostResults) return 0;
    const GramPlan p = gram_plan(2 * n_rows, m, n);
    return size_t(p.slabs) * p.tiles_m * p.tiles_n * p.bm * p.bn * sizeof(float);
}

extern "C" int mh_ckpt_gram(const uint8_t* codes, const uint8_t* scales, int64_t n_rows, int32_t m, const float* G, int64_t ldg,
                            int64_t img, int32_t n, float* out, void* workspace, size_t workspace_bytes, void* stream_) {
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    if (int rc = check_checkpoint(codes, scales, n_rows, m)) return rc;
    MH_REQUIRE(n >= 1 && int64_t(m) * n <= kMostResults, "m=%d n=%d", m, n);
    MH_REQUIRE(out, "null pointer");
    MH_REQUIRE(ldg >= 0 && img >= 0 && ldg <= (1 << 24) && img <= (int64_t(1) << 40), "row stride of G: %lld", (long long)ldg);
    GramArgs a{};
    if (n_rows > 0) {
        MH_REQUIRE(G && workspace, "null pointer");
        const size_t need = mh_ckpt_gram_workspace_bytes(n_rows, m, n);
        if (workspace_bytes < need) return mh::fail(MH_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
    }
    const GramPlan p = gram_plan(2 * n_rows, m, n);
    a.codes = codes; a.scales = scales; a.g = G; a.ldg = ldg; a.img = img; a.rows = 2 * n_rows; a.rp = (a.rows + 7) & ~int64_t(7);
    a.slab_rows = p.slab_rows; a.m = m; a.mp = (m + 31) & ~31; a.n = n; a.slabs = p.slabs; a.tiles_m = p.tiles_m; a.tiles_n = p.tiles_n;
    a.partial = static_cast<float*>(workspace);
    if (n_rows > 0) {
        switch (p.bm * 1000 + p.bn) {
            case 64032: launch_gram<64, 32, 2, 1>(a, stream); break;
            case 64064: launch_gram<64, 64, 2, 1>(a, stream); break;
            case 128032: launch_gram<128, 32, 2, 1>(a, stream); break;
            case 128064: launch_gram<128, 64, 2, 1>(a, stream); break;
            case 128128: launch_gram<128, 128, 2, 2>(a, stream); break;
            case 256032: launch_gram<256, 32, 4, 1>(a, stream); break;
            case 256064: launch_gram<256, 64, 4, 1>(a, stream); break;
            case 256128: launch_gram<256, 128, 2, 2>(a, stream); break;
            default: launch_gram<384, 128, 4, 2>(a, stream); break;
        }
        MH_LAUNCH_CHECK("ckpt_gram");
    }
    const int32_t results = m * n;
    if (results < 64 * 256) ckpt_gram_join<16><<<unsigned(results + 15) / 16, kJoin, 0, stream>>>(a.partial, a.slabs, a.tiles_m, a.tiles_n, p.bm, p.bn, m, n, out);
    else ckpt_gram_join<64><<<unsigned(results + 63) / 64, kJoin, 0, stream>>>(a.partial, a.slabs, a.tiles_m, a.tiles_n, p.bm, p.bn, m, n, out);
    MH_LAUNCH_CHECK("ckpt_gram_join");
    return MH_OK;
}
