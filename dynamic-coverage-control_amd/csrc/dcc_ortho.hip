// dcc_ortho.hip -- orthogonalised updates by Newton-Schulz products (include/dcc_ortho.h).
//
// Two orders of the same polynomial, chosen by shape (m <= n):
//  * m x m side (m <= 704, or n long enough): A = X X^T once, then with p(A) = a I + b A + c A^2 the steps A <- p(A) A p(A), Q <- p(A) Q on
//    m x m matrices, and X <- Q X at the end: two passes over X instead of two per step.  An error of A along a direction of small
//    singular value grows by a^2 = 12 per step, so this side runs in float64 (fp64 MFMA): measured against float64 throughout, five steps
//    of 256 x 2704 are 5e-8 off, where float32 steps are 5e-6 off (and float32 on this side 1e-4).  A group holds at most five steps.
//    All its matrices are polynomials of one symmetric matrix: only lower tiles are computed, and mirrored.  |X|_F^2 is the trace of
//    the unscaled A, so nothing else reads X before the end.
//  * step by step (large and nearly square, where the float64 products would take longer): A = X X^T, B = a I + b A + c A^2, X <- B X.
// Large products over X are C = A B^T of bf16 planes: fp32 MFMA has 1/16 of the bf16 rate, so a value is kept as the sum of bf16 parts
// and the products of the parts are accumulated in float32.  float32 and float16 matrices take three parts (x = hi + mid + lo to
// 24 bits) and the six products hh, hm, mh, hl, lh, mm; what is dropped is below 2^-26 of a product.  bfloat16 matrices take two parts and
// hh, hm, mh (2^-17 of a product), with X itself kept in float32: X <- a X + (b A + c A^2) X, the first term without a product.  The errors of
// the products are of either sign and average out over their depth: 1e-5 to 3e-5 of the result after five steps, where float32 products
// leave 3e-6 to 3e-5.  (X in two parts, with a X among the products, left 8e-5 to 6e-4: its own rounding does not average out.)
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>
#include <utility>
#include <vector>

#include "dcc_internal.h"
#include "dcc_ortho.h"

#pragma clang fp contract(fast)

namespace {

constexpr int kEINVAL = -1, kEHIP = -2;
constexpr int kMaxProds = 20;           // products per launch (their descriptions travel as kernel arguments)
constexpr int kNormBlocks = 256;        // partial sums of a matrix's norm, at most
constexpr int kBK = 32;                 // depth of one staged slice of a plane product
constexpr int kTile = 128;              // its tile; planes are padded to it with zeros

typedef float f4 __attribute__((ext_vector_type(4)));
typedef double d4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef unsigned int u4 __attribute__((ext_vector_type(4)));
typedef unsigned short ushort_t;

__device__ __forceinline__ float get(float x) { return x; }
__device__ __forceinline__ float get(__hip_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float get(__half x) { return __half2float(x); }
__device__ __forceinline__ void store1(void* p, long long i, int dt, float v) {
    if (dt == 0) reinterpret_cast<float*>(p)[i] = v;
    else if (dt == 1) reinterpret_cast<__hip_bfloat16*>(p)[i] = __float2bfloat16(v);
    else reinterpret_cast<__half*>(p)[i] = __float2half(v);
}

template <typename E> struct alignas(4 * sizeof(E)) Four { E e[4]; };
__device__ __forceinline__ void store4(void* p, long long i, int dt, f4 v) {
    if (dt == 0) {
        *reinterpret_cast<f4*>(reinterpret_cast<float*>(p) + i) = v;
    } else if (dt == 1) {
        Four<__hip_bfloat16> o;
#pragma unroll
        for (int c = 0; c < 4; ++c) o.e[c] = __float2bfloat16(v[c]);
        *reinterpret_cast<Four<__hip_bfloat16>*>(reinterpret_cast<__hip_bfloat16*>(p) + i) = o;
    } else {
        Four<__half> o;
#pragma unroll
        for (int c = 0; c < 4; ++c) o.e[c] = __float2half(v[c]);
        *reinterpret_cast<Four<__half>*>(reinterpret_cast<__half*>(p) + i) = o;
    }
}

// Up to kMaxProds descriptions of one kind; workgroups first[i] .. first[i + 1] - 1 work on p[i].  The bounds lie together: one cache
// line says which description to read.
template <typename P> struct Batch { int first[kMaxProds + 4]; P p[kMaxProds]; };
template <typename P>
__device__ __forceinline__ int which(const Batch<P>& bt, int blk) {
    int pi = 0;
#pragma unroll
    for (int i = 1; i < kMaxProds; ++i) pi += blk >= bt.first[i];       // (unused bounds are the largest int)
    return pi;
}

// Consecutive workgroups go to the eight dies in turn: numbered so, each die gets a run of neighbouring tiles of every product, which share
// operands in its L2.  A product has a multiple of eight workgroups; those numbered from `tiles` on have no work.  (Runs over a whole launch
// would give the long products to some dies: 2048 x 2048, 1000 x 2500 and 4096 x 1024 together, X <- B X in 134 us, 112 so.)
__device__ __forceinline__ int die_order(int blk, int tiles) { return (blk & 7) * ((tiles + 7) >> 3) + (blk >> 3); }

// tile (ti, tj), tj <= ti, of the lower triangle counted row by row
__device__ __forceinline__ void lower_tile(int blk, int& ti, int& tj) {
    ti = (int)((sqrtf(8.f * blk + 1.f) - 1.f) * 0.5f);
    while (ti * (ti + 1) / 2 > blk) --ti;
    while ((ti + 1) * (ti + 2) / 2 <= blk) ++ti;
    tj = blk - ti * (ti + 1) / 2;
}

// Where |X|_F^2 comes from: `n` numbers at stride `step` (the diagonal of X X^T, or partial sums).  Every workgroup that needs it sums
// them for itself, in one order.  A null pointer: X is scaled already.
struct Scale { const double* at; long long step; int n; float eps; };
__device__ __forceinline__ double inverse_norm(const Scale& s, double* red, double* note = nullptr) {    // red: 8 doubles of LDS; all threads
    if (!s.at) return 1.;
    double v = 0.;
    for (int i = threadIdx.x; i < s.n; i += blockDim.x) v += s.at[i * s.step];
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.;
    for (int w = 0; w < (int)blockDim.x / 64; ++w) v += red[w];
    if (note && threadIdx.x == 0) *note = v;
    v = sqrt(v) + (double)s.eps;
    return v == 0. ? 0. : 1. / v;       // (X == 0 without an eps stays 0)
}

struct NormMat { const void* x; double* out; long long n; int blocks; };
using NormBatch = Batch<NormMat>;

// sum of squares in float64, by fixed ranges
template <typename E>
__global__ __launch_bounds__(256) void ortho_norm_k(const NormBatch nb) {
    __shared__ double red[4];
    const int i = which(nb, blockIdx.x);
    const NormMat& m = nb.p[i];
    const E* x = reinterpret_cast<const E*>(m.x);
    const int blk = blockIdx.x - nb.first[i];
    const long long per = (m.n + m.blocks - 1) / m.blocks, lo = blk * per, hi = lo + per < m.n ? lo + per : m.n;
    double s[4] = {0., 0., 0., 0.};
    long long j = lo + threadIdx.x;
    for (; j + 768 < hi; j += 1024)
#pragma unroll
        for (int e = 0; e < 4; ++e) { const double v = get(x[j + 256 * e]); s[e] += v * v; }
    for (; j < hi; j += 256) { const double v = get(x[j]); s[0] += v * v; }
    double t = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) t += __shfl_xor(t, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = t;
    __syncthreads();
    if (threadIdx.x == 0) m.out[blk] = (red[0] + red[1]) + (red[2] + red[3]);
}

// ---- the m x m side in float64 -------------------------------------------------------------------------------------------------
// v_mfma_f64_16x16x4_f64: A[i = lane%16][k = lane/16], B[k = lane/16][j = lane%16], D[i = 4 r + lane/16][j = lane%16]; a lane's four
// consecutive k make four steps.  Its accumulators must be ordinary registers: 16 of them in a row run at 77 TFLOP/s, at 34 where the compiler
// puts them into accumulation registers, which it does for kernels that may use more than 256 (hence the launch bounds).  Square matrices are stored [mq][mq], mq = m rounded up to 16, zero outside m: no bounds to check.
struct Gram {                           // out = X X^T, X [m, K] in memory as [m][K] or, tall, [K][m]
    const void* x;
    double *out, *part;                 // part: [slices][mq * mq] where slices > 1
    long long ld;
    int m, mq, K, slices, kper, tiles;  // kper: a multiple of 32
};
using GramBatch = Batch<Gram>;

// four values of row i at depth k: as they lie in memory (a valid place where i or k is outside) ...
template <typename E, bool TALL, bool VEC>
__device__ __forceinline__ Four<E> load_x(const E* x, long long ld, int i, int m, int k, int kend) {
    Four<E> f;
    const int ic = i < m ? i : m - 1;
    if constexpr (VEC) {
        f = *reinterpret_cast<const Four<E>*>(x + (long long)ic * ld + (k < kend ? k : 0));
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int kc = k + j < kend ? k + j : kend - 1;
            f.e[j] = TALL ? x[(long long)kc * ld + ic] : x[(long long)ic * ld + kc];
        }
    }
    return f;
}
// ... and as operands, zero outside
template <typename E>
__device__ __forceinline__ d4 clear_x(const Four<E>& f, int i, int m, int k, int kend) {
    d4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = i < m && k + j < kend ? (double)get(f.e[j]) : 0.;
    return v;
}
template <typename E, bool TALL, bool VEC>
__device__ __forceinline__ d4 fetch_x(const E* x, long long ld, int i, int m, int k, int kend) {
    return clear_x<E>(load_x<E, TALL, VEC>(x, ld, i, m, k, kend), i, m, k, kend);
}

__device__ __forceinline__ void mirror(double* out, int mq, int i, int j, double v) {
    out[(long long)i * mq + j] = v;
    out[(long long)j * mq + i] = v;
}

// Short depths: a 32 x 32 tile per workgroup of eight waves, each of which takes every eighth run of 16 of the depth for the whole tile
// (latency counts: a wave's loads are all under way together, and its chain of products is short); the partial tiles are added in LDS.
// A product of 256 x 256 takes 6.4 us and more in a launch of its own (median 7.6) (launch, two loads one after the other, 16 MFMA, LDS, store), 1 us of it MFMA.
constexpr int kWaves = 8;
struct Tile32 { d4 t[2][2]; };
template <typename FA, typename FB>
__device__ __forceinline__ Tile32 tile32(int K, FA fa, FB fb) {         // fa(s, k): four values of row s * 16 + lane % 16 at depth k + 4 * (lane / 16)
    const int wave = threadIdx.x >> 6;
    Tile32 r;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) r.t[x][y] = d4{0., 0., 0., 0.};
    for (int k0 = wave * 16; k0 < K; k0 += kWaves * 32) {
        const int k1 = k0 + kWaves * 16, kc = k1 < K ? k1 : k0;
        const d4 a00 = fa(0, k0), a01 = fa(1, k0), b00 = fb(0, k0), b01 = fb(1, k0);
        const d4 a10 = fa(0, kc), a11 = fa(1, kc), b10 = fb(0, kc), b11 = fb(1, kc);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            r.t[0][0] = __builtin_amdgcn_mfma_f64_16x16x4f64(a00[i], b00[i], r.t[0][0], 0, 0, 0);
            r.t[0][1] = __builtin_amdgcn_mfma_f64_16x16x4f64(a00[i], b01[i], r.t[0][1], 0, 0, 0);
            r.t[1][0] = __builtin_amdgcn_mfma_f64_16x16x4f64(a01[i], b00[i], r.t[1][0], 0, 0, 0);
            r.t[1][1] = __builtin_amdgcn_mfma_f64_16x16x4f64(a01[i], b01[i], r.t[1][1], 0, 0, 0);
        }
        if (k1 >= K) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            r.t[0][0] = __builtin_amdgcn_mfma_f64_16x16x4f64(a10[i], b10[i], r.t[0][0], 0, 0, 0);
            r.t[0][1] = __builtin_amdgcn_mfma_f64_16x16x4f64(a10[i], b11[i], r.t[0][1], 0, 0, 0);
            r.t[1][0] = __builtin_amdgcn_mfma_f64_16x16x4f64(a11[i], b10[i], r.t[1][0], 0, 0, 0);
            r.t[1][1] = __builtin_amdgcn_mfma_f64_16x16x4f64(a11[i], b11[i], r.t[1][1], 0, 0, 0);
        }
    }
    return r;
}
// the whole tile's entries e = threadIdx.x and + 512: row e / 32, column e % 32
__device__ __forceinline__ void sum32(const Tile32& r, double (*sh)[1024], double (&v)[2]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, g = lane >> 4;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int i = 0; i < 4; ++i) sh[wave][(16 * x + 4 * i + g) * 32 + 16 * y + li] = r.t[x][y][i];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int e = threadIdx.x + 512 * q;
        v[q] = ((sh[0][e] + sh[1][e]) + (sh[2][e] + sh[3][e])) + ((sh[4][e] + sh[5][e]) + (sh[6][e] + sh[7][e]));
    }
}

// VEC: rows of X may be read four elements at a time (K a multiple of 4)
template <typename E, bool TALL, bool VEC>
__global__ __launch_bounds__(64 * kWaves) void ortho_gram_k(const GramBatch bt) {
    __shared__ double sh[kWaves][1024];
    const int pi = which(bt, blockIdx.x);
    const Gram& p = bt.p[pi];
    const E* x = reinterpret_cast<const E*>(p.x);
    const int m = p.m, K = p.K, li = threadIdx.x & 15, g4 = (threadIdx.x >> 4 & 3) * 4;
    const long long ld = p.ld;
    int ti, tj;
    lower_tile(blockIdx.x - bt.first[pi], ti, tj);
    const int i0 = ti * 32, j0 = tj * 32;
    const Tile32 r = tile32(K, [&](int s, int k) { return fetch_x<E, TALL, VEC>(x, ld, i0 + 16 * s + li, m, k + g4, K); },
                            [&](int s, int k) { return fetch_x<E, TALL, VEC>(x, ld, j0 + 16 * s + li, m, k + g4, K); });
    double v[2];
    sum32(r, sh, v);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int e = threadIdx.x + 512 * q, i = i0 + (e >> 5), j = j0 + (e & 31);
        if (i < p.mq && j <= i) mirror(p.out, p.mq, i, j, v[q]);
    }
}

// Long depths, where reading the operands counts: a 64 x 64 tile by 2 x 2 waves of 32 x 32 over one slice of the depth.  Bound by the fp64
// MFMA, which is busy in two cycles of three: 256 x 165952 float32 in 259 us, 47 TFLOP/s of the 77 that the instruction alone reaches.
template <typename E, bool TALL, bool VEC>
__global__ __launch_bounds__(256, 2) void ortho_gram_wide_k(const GramBatch bt) {
    const int pi = which(bt, blockIdx.x);
    const Gram& p = bt.p[pi];
    const E* x = reinterpret_cast<const E*>(p.x);
    const int blk = die_order(blockIdx.x - bt.first[pi], p.tiles), m = p.m, mq = p.mq, nt = (mq + 63) / 64, tiles = nt * (nt + 1) / 2, slice = blk / tiles;
    const long long ld = p.ld;
    if (blk >= p.tiles) return;
    int ti, tj;
    lower_tile(blk - slice * tiles, ti, tj);
    // (turned by the slice, so that what is above the diagonal is not always the same SIMD's)
    const int lane = threadIdx.x & 63, wave = (threadIdx.x >> 6) + slice & 3, li = lane & 15, g = lane >> 4;
    const int i0 = ti * 64 + (wave >> 1) * 32, j0 = tj * 64 + (wave & 1) * 32;
    if (j0 > i0) return;                // above the diagonal
    const int kbeg = slice * p.kper, kend = kbeg + p.kper < p.K ? kbeg + p.kper : p.K;
    d4 acc[2][2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int c = 0; c < 2; ++c) acc[u][c] = d4{0., 0., 0., 0.};
    // Two steps of 16 are on their way while one is multiplied (as they lie: half the registers of operands).  A lane's two steps are 8
    // consecutive of a run of 32: the lanes of a row read whole cache lines.  Rows behind m repeat the last, and nobody reads what they
    // give; a depth behind kend is cleared, in a slice's last run only.
    Four<E> na[2][2], nb[2][2];
    auto depth = [&](int k, int h) { return k + 8 * g + 4 * h; };
    auto fetch = [&](int k, int h) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            na[h][t] = load_x<E, TALL, VEC>(x, ld, i0 + 16 * t + li, m, depth(k, h), kend);
            nb[h][t] = load_x<E, TALL, VEC>(x, ld, j0 + 16 * t + li, m, depth(k, h), kend);
        }
    };
    auto multiply = [&](const d4 (&a)[2], const d4 (&b)[2]) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int c = 0; c < 2; ++c) acc[u][c] = __builtin_amdgcn_mfma_f64_16x16x4f64(a[u][r], b[c][r], acc[u][c], 0, 0, 0);
    };
    fetch(kbeg, 0);
    fetch(kbeg, 1);
    int k = kbeg;
    for (; k + 32 < kend; k += 32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            d4 a[2], b[2];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) { a[t][j] = get(na[h][t].e[j]); b[t][j] = get(nb[h][t].e[j]); }
            fetch(k + 32, h);
            multiply(a, b);
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        d4 a[2], b[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            a[t] = clear_x<E>(na[h][t], 0, 1, depth(k, h), kend);
            b[t] = clear_x<E>(nb[h][t], 0, 1, depth(k, h), kend);
        }
        multiply(a, b);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = i0 + 16 * u + 4 * r + g, j = j0 + 16 * c + li;
                if (i >= mq || j > i) continue;
                const double v = i < m && j < m ? acc[u][c][r] : 0.;
                if (p.slices > 1) p.part[((long long)slice * mq + i) * mq + j] = v;
                else mirror(p.out, mq, i, j, v);
            }
}

__global__ __launch_bounds__(256) void ortho_join_k(const GramBatch bt) {
    const Gram& p = bt.p[blockIdx.y];
    if (p.slices <= 1) return;
    const long long n = (long long)p.mq * p.mq;
    for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < n; at += (long long)gridDim.x * 256) {
        const int i = (int)(at / p.mq), j = (int)(at - (long long)i * p.mq);
        if (j > i) continue;
        double s = 0.;
#pragma unroll 8
        for (int q = 0; q < p.slices; ++q) s += p.part[q * n + at];
        mirror(p.out, p.mq, i, j, s);
    }
}

// Few products: 16 x 16 tiles, so that more of the chip takes part.  (An entry's sum has the order that it has in a 32 x 32 tile: what else
// is in a list does not change a matrix's result.)
template <typename FA, typename FB>
__device__ __forceinline__ d4 tile16(int K, FA fa, FB fb) {
    d4 t = {0., 0., 0., 0.};
    for (int k0 = (threadIdx.x >> 6) * 16; k0 < K; k0 += kWaves * 32) {
        const int k1 = k0 + kWaves * 16, kc = k1 < K ? k1 : k0;
        const d4 a0 = fa(0, k0), b0 = fb(0, k0), a1 = fa(0, kc), b1 = fb(0, kc);
#pragma unroll
        for (int i = 0; i < 4; ++i) t = __builtin_amdgcn_mfma_f64_16x16x4f64(a0[i], b0[i], t, 0, 0, 0);
        if (k1 >= K) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) t = __builtin_amdgcn_mfma_f64_16x16x4f64(a1[i], b1[i], t, 0, 0, 0);
    }
    return t;
}

struct Square {                         // out = alpha A B + beta E + diag I, all symmetric [mq][mq]; A is E of the unscaled matrix: see sa
    const double *a, *b, *e;
    double* out;
    int m, mq;
    double alpha, beta, diag;
    Scale s;                            // beta (E) is scaled by 1 / norm^2, alpha by its power sa (twice for A A of the unscaled A)
    int sa;
    double* note;                       // the first workgroup leaves norm^2 here, or null
};
using SquareBatch = Batch<Square>;

// T: 2 for tiles of 32 x 32, 1 for 16 x 16
template <int T>
__global__ __launch_bounds__(64 * kWaves) void ortho_square_k(const SquareBatch bt) {
    constexpr int D = 16 * T, NV = T == 2 ? 2 : 1;
    __shared__ double sh[kWaves][D * D], red[kWaves];
    const int pi = which(bt, blockIdx.x);
    const Square& p = bt.p[pi];
    int ti, tj;
    lower_tile(blockIdx.x - bt.first[pi], ti, tj);
    const int mq = p.mq, i0 = ti * D, j0 = tj * D, li = threadIdx.x & 15, g = threadIdx.x >> 4 & 3, g4 = g * 4;
    // (rows behind mq repeat the last: mq is a multiple of 16 only; what they give is not written)
    const double* pa[T];
    const double* pb[T];
#pragma unroll
    for (int s = 0; s < T; ++s) {
        const int i = i0 + 16 * s + li, j = j0 + 16 * s + li;
        pa[s] = p.a + (long long)(i < mq ? i : mq - 1) * mq + g4;
        pb[s] = p.b + (long long)(j < mq ? j : mq - 1) * mq + g4;
    }
    int ei[NV], ej[NV];                 // this thread's entries (16 x 16: of the first four waves)
    double ev[NV];                      // E there, on its way with the operands
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        const int e = (T == 2 ? threadIdx.x : threadIdx.x & 255) + 512 * q;
        ei[q] = i0 + e / D;
        ej[q] = j0 + e % D;
        ev[q] = 0.;
        if (p.e) ev[q] = p.e[(long long)(ei[q] < mq ? ei[q] : mq - 1) * mq + (ej[q] < mq ? ej[q] : mq - 1)];
    }
    auto fa = [&](int s, int k) { return *reinterpret_cast<const d4*>(pa[s] + k); };
    auto fb = [&](int s, int k) { return *reinterpret_cast<const d4*>(pb[s] + k); };
    double v[NV];
    double inv;
    auto norm = [&]() { inv = inverse_norm(p.s, red, (int)blockIdx.x == bt.first[pi] ? p.note : nullptr); };
    if constexpr (T == 2) {
        const Tile32 r = tile32(mq, fa, fb);
        norm();
        sum32(r, sh, v);
    } else {
        const d4 r = tile16(mq, fa, fb);
        norm();
#pragma unroll
        for (int i = 0; i < 4; ++i) sh[threadIdx.x >> 6][(4 * i + g) * 16 + li] = r[i];
        __syncthreads();
        if (threadIdx.x >= 256) return;
        const int e = threadIdx.x;
        v[0] = ((sh[0][e] + sh[1][e]) + (sh[2][e] + sh[3][e])) + ((sh[4][e] + sh[5][e]) + (sh[6][e] + sh[7][e]));
    }
    const double inv2 = inv * inv, alpha = p.alpha * (p.sa > 1 ? inv2 * inv2 : p.sa > 0 ? inv2 : 1.);
#pragma unroll
    for (int q = 0; q < NV; ++q) {
        if (ej[q] > ei[q] || ei[q] >= mq) continue;
        double w = alpha * v[q];
        if (p.e) w += p.beta * inv2 * ev[q];
        if (ei[q] == ej[q] && ei[q] < p.m) w += p.diag;
        mirror(p.out, mq, ei[q], ej[q], w);
    }
}

// X <- Q X in float64
struct Apply {                          // out [rows][cols] = Q X (wide: X [m][n]) or X Q (tall: X [n][m])
    const void* x;
    const double* q;
    void* out;
    long long ld;                       // of X and out
    int m, mq, rows, cols, tcols, dto, tiles;
    Scale s;
};
using ApplyBatch = Batch<Apply>;

// few tiles: as the short depths above
template <typename E, bool TALL>
__global__ __launch_bounds__(64 * kWaves) void ortho_apply_k(const ApplyBatch bt) {
    __shared__ double sh[kWaves][1024], red[kWaves];
    const int pi = which(bt, blockIdx.x);
    const Apply& p = bt.p[pi];
    const E* x = reinterpret_cast<const E*>(p.x);
    const int m = p.m, mq = p.mq, li = threadIdx.x & 15, g4 = (threadIdx.x >> 4 & 3) * 4, blk = blockIdx.x - bt.first[pi];
    const int ti = blk / p.tcols, tj = blk - ti * p.tcols, i0 = ti * 32, j0 = tj * 32;
    const long long ld = p.ld;
    const double inv = inverse_norm(p.s, red);
    const int q0 = TALL ? j0 : i0, x0 = TALL ? i0 : j0, xn = TALL ? p.rows : p.cols;
    auto fq = [&](int s, int k) {
        const int i = q0 + 16 * s + li;
        return *reinterpret_cast<const d4*>(p.q + (long long)(i < mq ? i : mq - 1) * mq + k + g4);
    };
    auto fx = [&](int s, int k) {       // (Q is zero behind m: what X gives there only has to be finite when X is)
        const int i = x0 + 16 * s + li, ic = i < xn ? i : xn - 1;
        d4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int kk = k + g4 + r, kc = kk < m ? kk : m - 1;
            v[r] = get(TALL ? x[ic * ld + kc] : x[kc * ld + ic]);
        }
        return v;
    };
    Tile32 r;
    if constexpr (TALL) r = tile32(mq, fx, fq);
    else r = tile32(mq, fq, fx);
    double v[2];
    sum32(r, sh, v);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int e = threadIdx.x + 512 * q, i = i0 + (e >> 5), j = j0 + (e & 31);
        if (i < p.rows && j < p.cols) store1(p.out, i * ld + j, p.dto, (float)(v[q] * inv));
    }
}

// Many tiles: 64 x 128 by 2 x 2 waves of 32 x 64, each over the whole depth.  A lane's four columns lie side by side (tile c holds columns
// 4 (lane % 16) + c), so that X and the result move four elements at a time; VEC: they may (rows and addresses are multiples of four).
// Bound by the fp64 MFMA, busy in three cycles of four: 256 x 165952 float32 in 419 us, 52 TFLOP/s.  (Products of three bf16 planes, with
// the splitting before them, took 330 us, but left the result at 2e-6 or, with fewer rows, at 1e-5 where this is at 5e-8.)
template <typename E, bool TALL, bool VEC>
__global__ __launch_bounds__(256, 2) void ortho_apply_wide_k(const ApplyBatch bt) {
    __shared__ double red[8];
    const int pi = which(bt, blockIdx.x);
    const Apply& p = bt.p[pi];
    const E* x = reinterpret_cast<const E*>(p.x);
    const int m = p.m, mq = p.mq, rows = p.rows, cols = p.cols, blk = die_order(blockIdx.x - bt.first[pi], p.tiles), trows = (rows + 63) / 64;
    if (blk >= p.tiles) return;         // (tiles along the shorter side first, like the plane products: neighbours share X or Q)
    const int ti = TALL ? blk / p.tcols : blk % trows, tj = TALL ? blk - ti * p.tcols : blk / trows;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, g = lane >> 4;
    const int i0 = ti * 64 + (wave >> 1) * 32, j0 = tj * 128 + (wave & 1) * 64, jl = j0 + 4 * li;
    const long long ld = p.ld;
    const double inv = inverse_norm(p.s, red);
    if (i0 >= rows || j0 >= cols) return;
    constexpr int NQ = TALL ? 4 : 2, NX = TALL ? 2 : 4;
    const double* qrow[NQ];
    const E* xrow[NX];                  // tall: rows of X at the lane's depth; else its columns (moved on with the depth)
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
        const int i = TALL ? jl + t : i0 + 16 * t + li;
        qrow[t] = p.q + (long long)(i < mq ? i : mq - 1) * mq + 4 * g;
    }
#pragma unroll
    for (int t = 0; t < NX; ++t) {
        const int i = i0 + 16 * t + li;
        xrow[t] = TALL ? x + (i < rows ? i : rows - 1) * ld : x + (VEC ? (jl < cols ? jl : 0) : jl + t < cols ? jl + t : cols - 1);
    }
    struct Step { d4 q[NQ]; Four<E> x[NX]; };           // (Q is zero behind m: what X gives there only has to be finite when X is)
    auto fetch = [&](Step& n, int k) {
#pragma unroll
        for (int t = 0; t < NQ; ++t) n.q[t] = *reinterpret_cast<const d4*>(qrow[t] + k);
        const int kl = k + 4 * g;
#pragma unroll
        for (int t = 0; t < NX; ++t)
            if constexpr (TALL && VEC) {
                n.x[t] = *reinterpret_cast<const Four<E>*>(xrow[t] + (kl < m ? kl : 0));
            } else if constexpr (TALL) {
#pragma unroll
                for (int j = 0; j < 4; ++j) n.x[t].e[j] = xrow[t][kl + j < m ? kl + j : m - 1];
            } else {                    // t: the depth
                const long long at = (kl + t < m ? kl + t : m - 1) * ld;
                if constexpr (VEC) {
                    n.x[t] = *reinterpret_cast<const Four<E>*>(xrow[0] + at);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) n.x[t].e[j] = xrow[j][at];
                }
            }
    };
    d4 acc[2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[u][c] = d4{0., 0., 0., 0.};
    auto multiply = [&](const Step& n) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const double b = TALL ? n.q[TALL ? c : 0][r] : (double)get(n.x[TALL ? 0 : r].e[c]);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const double a = TALL ? (double)get(n.x[u].e[r]) : n.q[u][r];
                    acc[u][c] = __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, acc[u][c], 0, 0, 0);
                }
            }
    };
    Step s0, s1;                        // one on its way while the other is multiplied
    fetch(s0, 0);
    int k = 0;
    for (; k + 32 < mq; k += 32) {
        fetch(s1, k + 16);
        multiply(s0);
        fetch(s0, k + 32);
        multiply(s1);
    }
    if (k + 16 < mq) fetch(s1, k + 16);
    multiply(s0);
    if (k + 16 < mq) multiply(s1);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = i0 + 16 * u + 4 * r + g;
            if (i >= rows) continue;
            f4 o;
#pragma unroll
            for (int c = 0; c < 4; ++c) o[c] = (float)(acc[u][c][r] * inv);
            if constexpr (VEC) {
                if (jl < cols) store4(p.out, i * ld + jl, p.dto, o);
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (jl + c < cols) store1(p.out, i * ld + jl + c, p.dto, o[c]);
            }
        }
}

// ---- plane products ------------------------------------------------------------------------------------------------------------
// The planes of a value: each part is the rest rounded to nearest, so that three parts hold 24 bits and the dropped products (mid lo, lo mid,
// lo lo) are below 2^-26 of a product and of either sign.
template <int NP>
__device__ __forceinline__ void split(float v, ushort_t (&h)[NP]) {
#pragma unroll
    for (int s = 0; s < NP; ++s) {
        const __hip_bfloat16 r = __float2bfloat16(v);
        h[s] = __builtin_bit_cast(ushort_t, r);
        v -= __bfloat162float(r);
    }
}

// Planes of a matrix [rows][K], K a multiple of 32: every row holds, for each 32 of its depth, the NP parts of
// those 32 side by side, so that a slice of 32 is 64 NP consecutive bytes of a row.
template <int NP>
__device__ __forceinline__ long long plane_at(long long row, int k, int s, long long K) {
    return row * (K * NP) + (k >> 5) * (32 * NP) + s * 32 + (k & 31);
}

struct Split {                          // planes of the scaled X [R][C]: as it lies (`same` [rp][cp]) and / or transposed (`turned` [cp][rp])
    const void* x;
    ushort_t *same, *turned;
    float* whole;                       // and the scaled X in float32, [rp][cp] (or null)
    int R, C, rp, cp, tcols;     // padded to kTile with zeros
    Scale s;
};
using SplitBatch = Batch<Split>;

template <typename E, int NP>
__global__ __launch_bounds__(256) void ortho_split_k(const SplitBatch bt) {
    __shared__ double red[8];
    __shared__ alignas(16) ushort_t sh[NP][64][72];         // transposed tile: rows of 144 bytes
    const int pi = which(bt, blockIdx.x);
    const Split& p = bt.p[pi];
    const E* x = reinterpret_cast<const E*>(p.x);
    const int blk = blockIdx.x - bt.first[pi], i0 = blk / p.tcols * 64, j0 = blk % p.tcols * 64;
    const double inv = inverse_norm(p.s, red);          // (in float32 it may be subnormal or infinite where the products are neither)
    const int c = threadIdx.x & 63, r0 = threadIdx.x >> 6;
    const int jc = j0 + c < p.C ? j0 + c : p.C - 1;
    float v[16];
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        const int i = i0 + r0 * 16 + q, ic = i < p.R ? i : p.R - 1;
        v[q] = get(x[(long long)ic * p.C + jc]);
        v[q] = i < p.R && j0 + c < p.C ? (float)(v[q] * inv) : 0.f;
    }
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        ushort_t h[NP];
        split<NP>(v[q], h);
#pragma unroll
        for (int s = 0; s < NP; ++s) {
            if (s == 0 && p.whole) p.whole[(long long)(i0 + r0 * 16 + q) * p.cp + j0 + c] = v[q];
            if (p.same) p.same[plane_at<NP>(i0 + r0 * 16 + q, j0 + c, s, p.cp)] = h[s];
            if (p.turned) sh[s][c][r0 * 16 + q] = h[s];
        }
    }
    if (!p.turned) return;
    __syncthreads();
#pragma unroll
    for (int s = 0; s < NP; ++s)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int e = threadIdx.x + q * 256, j = e >> 3, i = (e & 7) * 8;
            *reinterpret_cast<u4*>(p.turned + plane_at<NP>(j0 + j, i0 + i, s, p.rp)) = *reinterpret_cast<const u4*>(&sh[s][j][i]);
        }
}

struct Gemm {                           // v = alpha A B^T + beta E + diag I
    const ushort_t *a, *b, *e;          // planes; rows of A and B are contiguous over the depth
    ushort_t *d1, *d2;                  // planes of v as [i][j] and as [j][i] (either may be null)
    void* out;                          // or, bounded by rows and cols, v itself
    float* x;                           // two parts: v += xa x, and x = v unless out is given; [i][j] or, xt, [j][i]
    long long ldo;                      // row length of out
    int lda, ldb, lde, ld1, ld2, K,     // depths of the planes' rows; of this product
         rows, cols, dto, sym, tcols, tiles, ldx, xt;
    float alpha, beta, diag, xa;
};
using GemmBatch = Batch<Gemm>;

// A staged slice in LDS: 4 NP pieces of 16 bytes a row, as in memory but turned by the row, so that the 16 rows that one MFMA operand
// reads at one piece lie in 16 different groups of banks.  turned() gives the place of piece q and, being its own inverse, what lies at q.
template <int NP>
__device__ __forceinline__ int turned(int row, int q) {
    return NP == 2 ? q ^ ((row >> 1) & 7) : q ^ ((row >> 2) & 3);
}

// One 128 x 128 tile of one product: 8 waves as 2 x 4 of 64 x 32 (two on a SIMD: one multiplies while the other waits).  Slices of 32 go to
// LDS directly, kAhead of them under way while one is multiplied: a slice takes 0.3 - 0.6 us of MFMA and 1.5 us to arrive.
// 2048 x 2048 (one tile per compute unit) takes 50 us with two parts, 88 with three: 1.03 and 1.17 PFLOP/s of bf16; 4096 x 4096 with two
// 405 us, 1.02 PFLOP/s, where a large library product of the same type reaches 1.09.  Two or three slices ahead, the waits are below a
// tenth: what is left is the reading of fragments from LDS beside the products.
template <int NP> constexpr int kAhead = NP == 2 ? 3 : 2;       // (as many as LDS holds)

// 16 bytes a lane from base + off to LDS bytes to + 16 * lane.  Written out, and with it the waits: the compiler's own barrier waits for
// every load that is under way (2048 x 2048, two parts: 76 us instead of 50), there being no way to tell it which slice a
// barrier is about.  Nothing but LDS and m0 is written.  m0 is reserved (it can't be declared): the compiler keeps nothing in it between
// instructions, and sets it right before each that reads it, of which this kernel has no other.
__device__ __forceinline__ void load_lds(const char* base, unsigned off, unsigned to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off), "s"(base) : "memory");
}
// this wave's LDS reads and all but its last N loads are done; then all waves meet
template <int N>
__device__ __forceinline__ void meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | 7 << 4 | (N >> 4) << 14);     // vmcnt N, lgkmcnt 0 (the compiler counts along)
    asm volatile("s_barrier" ::: "memory");
}

template <int NP>
__global__ __launch_bounds__(512) void ortho_gemm_k(const GemmBatch bt) {
    constexpr int kSlice = kTile * 4 * NP;              // 16-byte pieces of one operand's slice
    constexpr int kStage = 2 * kSlice, NS = kAhead<NP> + 1;
    extern __shared__ u4 lds[];                         // [NS][2][kSlice]
    const int pi = which(bt, blockIdx.x);
    const Gemm& p = bt.p[pi];
    const int blk = die_order(blockIdx.x - bt.first[pi], p.tiles);
    if (blk >= p.tiles) return;
    int ti, tj;
    if (p.sym) {
        lower_tile(blk, ti, tj);
    } else if (p.rows <= p.cols) {                      // along the shorter side first
        const int trows = (p.rows + kTile - 1) / kTile;
        tj = blk / trows;
        ti = blk - tj * trows;
    } else {
        ti = blk / p.tcols;
        tj = blk - ti * p.tcols;
    }
    const int i0 = ti * kTile, j0 = tj * kTile;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, kg = lane >> 4, g4 = kg << 2;
    const int wi = (wave >> 2) * 64, wj = (wave & 3) * 32;
    // wave w brings rows 16 w .. 16 w + 15 of both operands, 64 pieces at a time
    constexpr int NL = NP;
    const char* ga = reinterpret_cast<const char*>(p.a + (long long)i0 * p.lda * NP);
    const char* gb = reinterpret_cast<const char*>(p.b + (long long)j0 * p.ldb * NP);
    unsigned oa[NL], ob[NL];
#pragma unroll
    for (int n = 0; n < NL; ++n) {
        const int t = n * 64 + lane, row = 16 * wave + t / (4 * NP), q = turned<NP>(row, t % (4 * NP));
        oa[n] = (unsigned)row * (unsigned)(p.lda * NP * 2) + q * 16;
        ob[n] = (unsigned)row * (unsigned)(p.ldb * NP * 2) + q * 16;
    }
    const unsigned lds0 = (unsigned)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) u4*)lds) + wave * (16 * 64 * NP);
    auto stage = [&](int buffer) {
        const unsigned to = lds0 + buffer * (kStage * 16);
#pragma unroll
        for (int n = 0; n < NL; ++n) {
            load_lds(ga, oa[n], to + n * 1024);
            load_lds(gb, ob[n], to + kSlice * 16 + n * 1024);
        }
        ga += kBK * NP * 2;
        gb += kBK * NP * 2;
    };
    // With three parts the products of the leading parts have sums of their own, which are rounded once a step and not six times: the
    // matrix unit's sums lose what they drop to one side (five steps of 2048 x 4096: 7.6e-6 off, 1.4e-5 with one sum; float32 8.0e-6).
    f4 acc[4][2], low[NP == 3 ? 4 : 1][2];
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            acc[x][y] = f4{0.f, 0.f, 0.f, 0.f};
            if constexpr (NP == 3) low[x][y] = f4{0.f, 0.f, 0.f, 0.f};
        }
    // A step's operands are read from LDS while the step before it is multiplied: one barrier a step, which says that the slice of the
    // next step has arrived and that nobody reads the buffer any more that the following load goes to.
    struct Frag { bf8 a[4][NP], b[2][NP]; };
    auto read = [&](Frag& f, int k) {
        const u4* sa = lds + (k % NS) * kStage;
        const u4* sb = sa + kSlice;
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int s = 0; s < NP; ++s) f.b[y][s] = __builtin_bit_cast(bf8, sb[(wj + 16 * y + li) * (4 * NP) + turned<NP>(wj + 16 * y + li, s * 4 + kg)]);
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int s = 0; s < NP; ++s) f.a[x][s] = __builtin_bit_cast(bf8, sa[(wi + 16 * x + li) * (4 * NP) + turned<NP>(wi + 16 * x + li, s * 4 + kg)]);
    };
    auto multiply = [&](const Frag& f) {        // small products first
#pragma unroll
        for (int o = NP - 1; o >= 0; --o)
#pragma unroll
            for (int s = 0; s <= o; ++s)
#pragma unroll
                for (int x = 0; x < 4; ++x)
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        f4& to = NP == 3 && o > 0 ? low[NP == 3 ? x : 0][y] : acc[x][y];
                        to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.a[x][s], f.b[y][o - s], to, 0, 0, 0);
                    }
    };
    const int steps = p.K / kBK;        // an even number, at least 4: planes are padded to 128
#pragma unroll
    for (int k = 0; k < kAhead<NP>; ++k) stage(k);
    meet<2 * NP * (kAhead<NP> - 1)>();
    Frag f0, f1;
    read(f0, 0);
    // (the last step reads on into a buffer that nobody needs: a branch there would make the compiler wait for the reads before it)
    int k = 0;
    for (; k + 1 + kAhead<NP> < steps; k += 2) {
        stage((k + kAhead<NP>) % NS);
        meet<2 * NP * (kAhead<NP> - 1)>();              // all but the slices after the next
        read(f1, k + 1);
        multiply(f0);
        stage((k + 1 + kAhead<NP>) % NS);
        meet<2 * NP * (kAhead<NP> - 1)>();
        read(f0, k + 2);
        multiply(f1);
    }
    if (k + kAhead<NP> < steps) stage((k + kAhead<NP>) % NS);
    for (; k < steps; k += 2) {
        meet<0>();
        read(f1, k + 1);
        multiply(f0);
        read(f0, k + 2);
        multiply(f1);
    }
    __syncthreads();
    f4 whole[NP == 2 ? 4 : 1][2];
    if constexpr (NP == 2) {            // (padded like the planes: no bounds)
        if (p.x) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const long long i = i0 + wi + 16 * x + g4, j = j0 + wj + 16 * y + li;
                    if (p.xt) {
                        whole[x][y] = *reinterpret_cast<const f4*>(p.x + j * p.ldx + i);
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r) whole[x][y][r] = p.x[(i + r) * p.ldx + j];
                    }
                }
        }
    }
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            const int i = i0 + wi + 16 * x + g4, j = j0 + wj + 16 * y + li;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float v = acc[x][y][r];
                if constexpr (NP == 3) v += low[x][y][r];
                v *= p.alpha;
                if constexpr (NP == 2) v += p.x ? p.xa * whole[x][y][r] : 0.f;
                if (p.e) {
                    float e = 0.f;
#pragma unroll
                    for (int s = NP - 1; s >= 0; --s) e += __uint_as_float((unsigned)p.e[plane_at<NP>(i + r, j, s, p.lde)] << 16);
                    v += p.beta * e;
                    if (i + r == j && j < p.rows) v += p.diag;
                }
                acc[x][y][r] = v;
                if (p.out && i + r < p.rows && j < p.cols) store1(p.out, (long long)(i + r) * p.ldo + j, p.dto, v);
            }
        }
    if (p.out) return;
    if constexpr (NP == 2) {
        if (p.x) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const long long i = i0 + wi + 16 * x + g4, j = j0 + wj + 16 * y + li;
                    if (p.xt) {
                        *reinterpret_cast<f4*>(p.x + j * p.ldx + i) = acc[x][y];
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r) p.x[(i + r) * p.ldx + j] = acc[x][y][r];
                    }
                }
        }
    }
    // planes leave through LDS, whole rows at a time
    constexpr int kRow = kTile + 8;
    ushort_t* sh = reinterpret_cast<ushort_t*>(lds);
#pragma unroll
    for (int s = 0; s < NP; ++s) {
#pragma unroll
        for (int turn = 0; turn < 2; ++turn) {
            ushort_t* dst = turn ? p.d2 : p.d1;
            if (!dst) continue;
            __syncthreads();
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const int i = wi + 16 * x + g4, j = wj + 16 * y + li;
                    ushort_t h[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        ushort_t all[NP];
                        split<NP>(acc[x][y][r], all);
                        h[r] = all[s];
                    }
                    if (turn) {
                        *reinterpret_cast<uint2*>(sh + j * kRow + i) = make_uint2(h[0] | (unsigned)h[1] << 16, h[2] | (unsigned)h[3] << 16);
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r) sh[(i + r) * kRow + j] = h[r];
                    }
                }
            __syncthreads();
            const int ld = turn ? p.ld2 : p.ld1, ro = turn ? j0 : i0, co = turn ? i0 : j0;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int e = threadIdx.x + q * 512, r = e >> 4, c = (e & 15) * 8;
                *reinterpret_cast<u4*>(dst + plane_at<NP>(ro + r, co + c, s, ld)) = *reinterpret_cast<const u4*>(sh + r * kRow + c);
            }
        }
    }
}

// ---- the element-wise ends of a step: bound by their bytes ---------------------------------------------------------------------
constexpr int kMaxSegs = 64;
struct Segs { long long off[kMaxSegs], n[kMaxSegs]; float scale[kMaxSegs]; int first[kMaxSegs + 1]; int count; float keep; };

__global__ __launch_bounds__(256) void muon_momentum_k(const float* __restrict__ g, float* __restrict__ buf, float* __restrict__ dir, long long n,
                                                       float mu, int nesterov, const float* __restrict__ clip_p) {
    const float clip = clip_p ? *clip_p : 1.f;
    const long long n4 = n >> 2;
    const long long i0 = (long long)blockIdx.x * 256 + threadIdx.x;
    for (long long i = i0; i < n4 + (n & 3); i += (long long)gridDim.x * 256) {
        if (i < n4) {
            f4 x = reinterpret_cast<const f4*>(g)[i], m = reinterpret_cast<f4*>(buf)[i];
            x *= clip;
            m = mu * m + x;
            reinterpret_cast<f4*>(buf)[i] = m;
            reinterpret_cast<f4*>(dir)[i] = nesterov ? x + mu * m : m;
        } else {
            const long long e = (n4 << 2) + (i - n4);
            const float x = g[e] * clip, m = mu * buf[e] + x;
            buf[e] = m;
            dir[e] = nesterov ? x + mu * m : m;
        }
    }
}

__global__ __launch_bounds__(256) void muon_apply_k(float* __restrict__ p, const float* __restrict__ dir, const Segs s) {
    int q = 0;
    while (q + 1 < s.count && (int)blockIdx.x >= s.first[q + 1]) ++q;
    const long long lo = s.off[q] + (long long)(blockIdx.x - s.first[q]) * 4096, end = s.off[q] + s.n[q];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const long long i = lo + j * 1024 + 4 * threadIdx.x;
        if (i + 3 < end) {
            const f4 v = s.keep * *reinterpret_cast<const f4*>(p + i) - s.scale[q] * *reinterpret_cast<const f4*>(dir + i);
            *reinterpret_cast<f4*>(p + i) = v;
        } else {
            for (long long e = i; e < end && e < i + 4; ++e) p[e] = s.keep * p[e] - s.scale[q] * dir[e];
        }
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------
constexpr int64_t kAlign = 256;
int64_t up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }
constexpr int kChip = 256;              // compute units

struct Shape { int64_t m, n; bool tall; };
Shape shape_of(const dcc_ortho_mat& t) { return Shape{std::min(t.M, t.N), std::max(t.M, t.N), t.M > t.N}; }

// The m x m side in float64: always up to 704, where a product's 32 x 32 tiles (253) have a compute unit each (600 x 700, five steps: 258 us
// here, step by step 508 in float32 and 317 in bfloat16; 704 x 704 and 705 x 705: 282 and 344 in bfloat16), above it where X is long enough.
// 1000 x 2500 float32: 907 and 902 us,
// 1000 x 5000: 1042 and 1457, 2048 x 8192: 6225 and 3419; bfloat16: 1000 x 5000 1062 and 812, 1000 x 10000 1289 and 1330.
bool on_square_side(const Shape& s, int dtype) { return s.m <= 704 || s.n >= s.m * s.m / (dtype == DCC_ORTHO_BF16 ? 100 : 256); }
constexpr int kGroup = 5;               // steps on that side before X X^T is formed anew
// X <- Q X in tiles of 64 x 128 where they fill the chip twice (256 x 32768: 226 us in all, in tiles of 32 x 32 284; 256 x 4096: 134 and 128)
bool wide_apply(const Shape& s) { return (s.m + 63) / 64 * ((s.n + 127) / 128) >= 2 * kChip; }

// tiles of 64 for long depths of X X^T, and then as many depth slices as fill the chip three times (what is resident), none shorter than 256
bool wide_gram(const Shape& s) { return s.n >= 1536; }
int gram_slices(const Shape& s) {
    const int64_t nt = (s.m + 63) / 64, tiles = nt * (nt + 1) / 2;
    if (!wide_gram(s)) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(3 * kChip / tiles, s.n / 256), 128));
}
int planes_of(int dtype) { return dtype == DCC_ORTHO_BF16 ? 2 : 3; }
int norm_blocks(const dcc_ortho_mat& t) { return (int)std::max<int64_t>(1, std::min<int64_t>(kNormBlocks, t.M * t.N / 4096)); }

// where a matrix's intermediate results lie in the workspace
struct Place { int64_t norm, A, B, W, Q0, Q1, Xp, Xt0, Xt1, X0, X1, whole, part, end; };
Place place_of(const Shape& s, int dtype, int steps, int64_t at) {
    Place p = {};
    auto take = [&](int64_t bytes) { const int64_t o = at; at += up(bytes, kAlign); return o; };
    const int64_t mq = up(s.m, 16), mp = up(s.m, kTile), np = up(s.n, kTile), mn = 4 * s.m * s.n, np2 = 2 * planes_of(dtype);
    if (on_square_side(s, dtype)) {
        p.norm = take(8);
        for (int64_t* o : {&p.A, &p.B, &p.W, &p.Q0, &p.Q1}) *o = take(8 * mq * mq);
        if (gram_slices(s) > 1) p.part = take(8 * mq * mq * gram_slices(s));
        if (steps > kGroup) p.X0 = take(mn);
        if (steps > 2 * kGroup) p.X1 = take(mn);
    } else {
        p.norm = take(8 * kNormBlocks);
        p.A = take(np2 * mp * mp); p.B = take(np2 * mp * mp);
        p.Xp = take(np2 * mp * np); p.Xt0 = take(np2 * np * mp);
        if (steps > 1) p.Xt1 = take(np2 * np * mp);
        if (planes_of(dtype) == 2) p.whole = take(4 * mp * np);
    }
    p.end = at;
    return p;
}

const char* list_error(const dcc_ortho_mat* mats, int32_t count, int32_t dtype, int32_t steps) {
    if (count < 0 || (count > 0 && !mats)) return "null list";
    if (dtype < DCC_ORTHO_F32 || dtype > DCC_ORTHO_F16) return "dtype must be float32, bfloat16 or float16";
    if (steps < 1 || steps > DCC_ORTHO_MAX_STEPS) return "steps must lie in 1..32";
    for (int i = 0; i < count; ++i) {
        if (mats[i].M < 0 || mats[i].N < 0) return "negative size";
        if (mats[i].M > (1 << 28) || mats[i].N > (1 << 28)) return "more than 2^28 rows or columns";
        if (shape_of(mats[i]).m > 16384) return "both sides over 16384";
    }
    return nullptr;
}

// do two arrays of n floats share bytes?
bool meet(const float* a, const float* b, int64_t n) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b), len = (uintptr_t)n * 4;
    return x < y + len && y < x + len;
}

// numbers the workgroups of a batch's n descriptions: returns how many there are
template <typename P, typename Blocks>
unsigned number(Batch<P>& bt, int n, Blocks blocks) {
    int64_t first = 0;
    for (int i = 0; i < kMaxProds; ++i) {
        bt.first[i] = i < n ? (int)first : 2147483647;
        if (i < n) first += blocks(bt.p[i]);
    }
    bt.first[kMaxProds] = (int)first;
    return (unsigned)first;
}
// does an output share bytes with an input or with another output?  (a list may hold thousands of matrices: sorted, not pair by pair)
bool outputs_meet(const dcc_ortho_mat* mats, const std::vector<int>& live, int64_t esize) {
    typedef std::pair<uintptr_t, uintptr_t> Range;
    auto range = [&](const void* p, int i) {
        const uintptr_t a = reinterpret_cast<uintptr_t>(p);
        return Range(a, a + mats[i].M * mats[i].N * esize);
    };
    std::vector<Range> outs;
    for (int i : live) outs.push_back(range(mats[i].out, i));
    std::sort(outs.begin(), outs.end());
    for (size_t i = 1; i < outs.size(); ++i)
        if (outs[i].first < outs[i - 1].second) return true;
    for (int i : live) {
        const Range r = range(mats[i].in, i);
        const auto next = std::lower_bound(outs.begin(), outs.end(), Range(r.second, 0));        // the first output from r's end on
        if (next != outs.begin() && (next - 1)->second > r.first) return true;
    }
    return false;
}
// calls f with batches of at most kMaxProds of `all` and their numbers of blocks and descriptions; what makes a launch larger than kMaxBlocks
// (of up to 512 threads: a launch holds less than 2^32) begins the next
constexpr int64_t kMaxBlocks = 1 << 22;
template <typename P, typename Blocks, typename F>
void batches(const std::vector<P>& all, Blocks blocks, F f) {
    for (size_t from = 0, to; from < all.size(); from = to) {
        Batch<P> bt;
        int64_t held = 0;
        for (to = from; to < all.size() && to < from + kMaxProds; ++to) {
            held += blocks(all[to]);
            if (to > from && held > kMaxBlocks) break;
            bt.p[to - from] = all[to];
        }
        const int n = (int)(to - from);
        const unsigned sum = number(bt, n, blocks);
        f(bt, sum, n);
    }
}
int64_t in_eights(int64_t n) { return (n + 7) / 8 * 8; }
int64_t lower(int64_t t) { return t * (t + 1) / 2; }
int64_t square_tiles(const Square& p, int d) { return lower((p.mq + d - 1) / d); }
constexpr unsigned kFewTiles = 80;      // fewer tiles of 32 x 32 than that in a launch: tiles of 16 x 16 (one 256 x 256, 36 or 72 of them: 103 us in all
                                        // for 133 with 32; one 512 x 512, 136 or 272: 258 for 224)

// a round: products (of all matrices) that do not depend on each other
struct Round {
    std::vector<Gram> gram[2][2][2];    // [tall][vec][wide]
    std::vector<Square> square;
    std::vector<Split> split[2];        // [planes - 2]
    std::vector<Gemm> gemm[2];
    std::vector<Apply> apply[2], wide_apply[2][2];      // [tall][vec]
};

template <typename E, bool TALL, bool VEC>
void launch_gram(const std::vector<Gram>& all, hipStream_t st) {
    batches(all, [](const Gram& p) { return lower((p.mq + 31) / 32); }, [&](const GramBatch& bt, unsigned blocks, int) {
        hipLaunchKernelGGL((ortho_gram_k<E, TALL, VEC>), dim3(blocks), dim3(64 * kWaves), 0, st, bt);
    });
}
template <typename E, bool TALL, bool VEC>
void launch_gram_wide(const std::vector<Gram>& all, hipStream_t st) {
    batches(all, [](const Gram& p) { return in_eights(p.tiles); }, [&](const GramBatch& bt, unsigned blocks, int n) {
        hipLaunchKernelGGL((ortho_gram_wide_k<E, TALL, VEC>), dim3(blocks), dim3(256), 0, st, bt);
        int64_t longest = 0;
        for (int i = 0; i < n; ++i)
            if (bt.p[i].slices > 1) longest = std::max<int64_t>(longest, (int64_t)bt.p[i].mq * bt.p[i].mq);
        if (longest) hipLaunchKernelGGL(ortho_join_k, dim3((unsigned)std::min<int64_t>((longest + 255) / 256, 1024), n), dim3(256), 0, st, bt);
    });
}
template <typename E, bool TALL, bool VEC>
void launch_apply_wide(const std::vector<Apply>& all, hipStream_t st) {
    batches(all, [](const Apply& p) { return in_eights(p.tiles); }, [&](const ApplyBatch& bt, unsigned blocks, int) {
        hipLaunchKernelGGL((ortho_apply_wide_k<E, TALL, VEC>), dim3(blocks), dim3(256), 0, st, bt);
    });
}
template <typename E>
void launch_x(const Round& q, hipStream_t st) {         // what reads X: E is its type
    launch_gram<E, false, false>(q.gram[0][0][0], st);
    launch_gram_wide<E, false, false>(q.gram[0][0][1], st);
    launch_gram<E, false, true>(q.gram[0][1][0], st);
    launch_gram_wide<E, false, true>(q.gram[0][1][1], st);
    launch_gram<E, true, false>(q.gram[1][0][0], st);
    launch_gram_wide<E, true, false>(q.gram[1][0][1], st);
    const auto tiles = [](const Split& p) { return (int64_t)(p.rp / 64) * (p.cp / 64); };
    batches(q.split[0], tiles, [&](const SplitBatch& bt, unsigned n, int) { hipLaunchKernelGGL((ortho_split_k<E, 2>), dim3(n), dim3(256), 0, st, bt); });
    batches(q.split[1], tiles, [&](const SplitBatch& bt, unsigned n, int) { hipLaunchKernelGGL((ortho_split_k<E, 3>), dim3(n), dim3(256), 0, st, bt); });
    launch_apply_wide<E, false, false>(q.wide_apply[0][0], st);
    launch_apply_wide<E, false, true>(q.wide_apply[0][1], st);
    launch_apply_wide<E, true, false>(q.wide_apply[1][0], st);
    launch_apply_wide<E, true, true>(q.wide_apply[1][1], st);
    const auto squares = [](const Apply& p) { return (int64_t)((p.rows + 31) / 32) * p.tcols; };
    batches(q.apply[0], squares, [&](const ApplyBatch& bt, unsigned n, int) { hipLaunchKernelGGL((ortho_apply_k<E, false>), dim3(n), dim3(64 * kWaves), 0, st, bt); });
    batches(q.apply[1], squares, [&](const ApplyBatch& bt, unsigned n, int) { hipLaunchKernelGGL((ortho_apply_k<E, true>), dim3(n), dim3(64 * kWaves), 0, st, bt); });
}
template <int NP>
bool launch_gemm(const std::vector<Gemm>& all, hipStream_t st) {
    constexpr int bytes = (kAhead<NP> + 1) * 2 * NP * kTile * 4 * 16;
    if (all.empty()) return true;
    if (bytes > 65536 && hipFuncSetAttribute(reinterpret_cast<const void*>(ortho_gemm_k<NP>), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return false;
    std::vector<Gemm> longest = all;     // first: what starts last is short
    std::stable_sort(longest.begin(), longest.end(), [](const Gemm& x, const Gemm& y) { return x.K > y.K; });
    for (Gemm& p : longest) {
        const int64_t t = (p.rows + kTile - 1) / kTile;
        p.tiles = (int)(p.sym ? lower(t) : t * p.tcols);
    }
    batches(longest, [](const Gemm& p) { return in_eights(p.tiles); }, [&](const GemmBatch& bt, unsigned n, int) {
        hipLaunchKernelGGL(ortho_gemm_k<NP>, dim3(n), dim3(512), bytes, st, bt);
    });
    return true;
}

}  // namespace

extern "C" {

DCC_API int64_t dcc_ortho_workspace_bytes(const dcc_ortho_mat* mats, int32_t count, int32_t dtype, int32_t steps) {
    if (list_error(mats, count, dtype, steps)) return 0;
    int64_t at = 0;
    for (int i = 0; i < count; ++i)
        if (mats[i].M > 0 && mats[i].N > 0) at = place_of(shape_of(mats[i]), dtype, steps, at).end;
    return at;
}

DCC_API int dcc_orthogonalize(const dcc_ortho_mat* mats, int32_t count, int32_t dtype, int32_t steps, float a, float b, float c,
                              float eps, void* workspace, void* stream) try {
    if (const char* e = list_error(mats, count, dtype, steps)) return dcc_fail_nothrow(kEINVAL, "dcc_orthogonalize: ", e);
    if (!(eps >= 0.f)) return dcc_fail_nothrow(kEINVAL, "dcc_orthogonalize: eps must not be negative");
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const int64_t esize = dtype == DCC_ORTHO_F32 ? 4 : 2;
    std::vector<int> live;
    for (int i = 0; i < count; ++i) {
        if (mats[i].M == 0 || mats[i].N == 0) continue;
        if (!mats[i].in || !mats[i].out) return dcc_fail_nothrow(kEINVAL, "dcc_orthogonalize: null matrix");
        if ((reinterpret_cast<uintptr_t>(mats[i].in) | reinterpret_cast<uintptr_t>(mats[i].out)) & (esize - 1))
            return dcc_fail_nothrow(kEINVAL, "dcc_orthogonalize: a matrix is not aligned to its elements");
        live.push_back(i);
    }
    if (live.empty()) return 0;
    if (outputs_meet(mats, live, esize)) return dcc_fail_nothrow(kEINVAL, "dcc_orthogonalize: an output overlaps an input or another output");
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & (kAlign - 1))) return dcc_fail_nothrow(kEINVAL, "dcc_orthogonalize: workspace must be 256-byte aligned");
    char* ws = reinterpret_cast<char*>(workspace);

    // every matrix's products, round by round; a round's products (of all matrices) run together
    std::vector<Round> rounds, later;   // later: what reads intermediate X in float32
    std::vector<NormMat> norms;
    auto round = [&](size_t r) -> Round& {
        if (rounds.size() <= r) { rounds.resize(r + 1); later.resize(r + 1); }
        return rounds[r];
    };
    int64_t at = 0;
    for (int idx : live) {
        const dcc_ortho_mat& t = mats[idx];
        const Shape s = shape_of(t);
        const Place pl = place_of(s, dtype, steps, at);
        at = pl.end;
        const int m = (int)s.m, n = (int)s.n, mq = (int)up(m, 16), mp = (int)up(m, kTile), np = (int)up(n, kTile);
        size_t r = 0;
        int left = steps;
        if (on_square_side(s, dtype)) {
            const void* X = t.in;
            bool raw = true, flip = false;
            double *A = reinterpret_cast<double*>(ws + pl.A), *B = reinterpret_cast<double*>(ws + pl.B), *W = reinterpret_cast<double*>(ws + pl.W);
            double* Qs[2] = {reinterpret_cast<double*>(ws + pl.Q0), reinterpret_cast<double*>(ws + pl.Q1)};
            auto square = [&](const double* x, const double* y, double* out) {
                Square p = {};
                p.a = x; p.b = y; p.out = out; p.m = m; p.mq = mq; p.alpha = 1.;
                return p;
            };
            while (left > 0) {
                const int groups = (left + kGroup - 1) / kGroup, len = (left + groups - 1) / groups;
                left -= len;
                const bool last = left == 0;
                double* note = reinterpret_cast<double*>(ws + pl.norm);
                Scale scale = {};       // after the first p(A), which takes |X|_F^2 from the unscaled A's diagonal and notes it
                if (raw) scale = Scale{note, 1, 1, eps};
                Gram g = {};            // A = X X^T
                g.x = X; g.out = A; g.ld = t.N; g.m = m; g.mq = mq; g.K = n;
                g.part = reinterpret_cast<double*>(ws + pl.part);
                g.kper = (int)up((n + gram_slices(s) - 1) / gram_slices(s), 32);
                g.slices = (n + g.kper - 1) / g.kper;
                g.tiles = (int)(lower((mq + 63) / 64) * g.slices);
                const int64_t es = raw ? esize : 4;
                const bool vec = !s.tall && n % 4 == 0 && (reinterpret_cast<uintptr_t>(X) & (4 * es - 1)) == 0;
                round(r);
                (raw ? rounds : later)[r].gram[s.tall][vec][wide_gram(s)].push_back(g);
                ++r;
                int cur = -1;           // Qs[cur] holds Q
                for (int k = 0; k < len; ++k) {
                    const bool end = k + 1 == len;
                    Square p = square(A, A, k > 0 ? B : Qs[0]);         // p(A); the first one works on the unscaled A
                    p.alpha = c; p.e = A; p.beta = b; p.diag = a;
                    if (k == 0 && raw) { p.s = Scale{A, mq + 1, m, eps}; p.sa = 2; p.note = note; }
                    round(r++).square.push_back(p);
                    double* Pk = k > 0 ? B : Qs[0];
                    if (k > 0) {                                        // Q <- p(A) Q
                        round(r).square.push_back(square(Pk, Qs[cur], Qs[cur ^ 1]));
                        cur ^= 1;
                        if (end) ++r;
                    } else {
                        cur = 0;
                    }
                    if (!end) {                                         // A <- p(A) A p(A)
                        Square w = square(Pk, A, W);
                        if (k == 0 && raw) { w.s = scale; w.sa = 1; }
                        round(r++).square.push_back(w);
                        round(r++).square.push_back(square(W, Pk, A));
                    }
                }
                void* out = last ? t.out : static_cast<void*>(ws + (flip ? pl.X1 : pl.X0));
                flip = !flip;
                Apply q = {};
                q.x = X; q.q = Qs[cur]; q.out = out; q.ld = t.N; q.m = m; q.mq = mq; q.rows = (int)t.M; q.cols = (int)t.N;
                q.dto = last ? dtype : 0; q.s = scale;
                const bool wide = wide_apply(s);
                const int64_t ds = last ? esize : 4;
                const bool vec4 = t.N % 4 == 0 && (reinterpret_cast<uintptr_t>(X) & (4 * es - 1)) == 0 && (reinterpret_cast<uintptr_t>(out) & (4 * ds - 1)) == 0;
                q.tcols = (int)((t.N + (wide ? 127 : 31)) / (wide ? 128 : 32));
                q.tiles = (int)((t.M + 63) / 64) * q.tcols;             // (of the wide form)
                round(r);
                Round& to = (raw ? rounds : later)[r++];
                (wide ? to.wide_apply[s.tall][vec4] : to.apply[s.tall]).push_back(q);
                X = out;
                raw = false;
            }
        } else {
            const int np2 = planes_of(dtype), nb = norm_blocks(t);
            ushort_t *A = reinterpret_cast<ushort_t*>(ws + pl.A), *B = reinterpret_cast<ushort_t*>(ws + pl.B), *Xp = reinterpret_cast<ushort_t*>(ws + pl.Xp);
            ushort_t* Xt[2] = {reinterpret_cast<ushort_t*>(ws + pl.Xt0), reinterpret_cast<ushort_t*>(ws + pl.Xt1)};
            double* norm = reinterpret_cast<double*>(ws + pl.norm);
            norms.push_back(NormMat{t.in, norm, t.M * t.N, nb});
            Split sp = {};
            sp.x = t.in; sp.R = (int)t.M; sp.C = (int)t.N; sp.rp = s.tall ? np : mp; sp.cp = s.tall ? mp : np;
            sp.same = s.tall ? Xt[0] : Xp; sp.turned = s.tall ? Xp : Xt[0];
            float* whole = np2 == 2 ? reinterpret_cast<float*>(ws + pl.whole) : nullptr;
            sp.whole = whole;
            sp.tcols = sp.cp / 64; sp.s = Scale{norm, 1, nb, eps};
            round(r++).split[np2 - 2].push_back(sp);
            int cur = 0;
            while (left > 0) {
                --left;
                Gemm g = {};            // A = X X^T
                g.a = g.b = Xp; g.lda = g.ldb = np; g.K = np; g.rows = g.cols = m; g.sym = 1; g.alpha = 1.f;
                g.d1 = g.d2 = A; g.ld1 = g.ld2 = mp; g.tcols = mp / kTile;
                round(r++).gemm[np2 - 2].push_back(g);
                Gemm p = g;             // B = a I + b A + c A^2, with two parts without a I
                p.a = p.b = p.e = A; p.lda = p.ldb = p.lde = mp; p.K = mp; p.d1 = p.d2 = B; p.alpha = c; p.beta = b; p.diag = whole ? 0.f : a;
                round(r++).gemm[np2 - 2].push_back(p);
                Gemm q = {};            // X <- B X (+ a X)
                q.K = q.lda = q.ldb = mp; q.alpha = 1.f;
                q.x = whole; q.xa = a; q.ldx = sp.cp; q.xt = s.tall && left > 0;
                if (left == 0) {
                    q.a = s.tall ? Xt[cur] : B; q.b = s.tall ? B : Xt[cur];
                    q.rows = (int)t.M; q.cols = (int)t.N; q.out = t.out; q.ldo = t.N; q.dto = dtype;
                } else {                // as [m][n] for the next X X^T, as [n][m] for the next step
                    q.a = B; q.b = Xt[cur]; q.rows = m; q.cols = n;
                    q.d1 = Xp; q.ld1 = np; q.d2 = Xt[cur ^ 1]; q.ld2 = mp;
                }
                q.tcols = (q.cols + kTile - 1) / kTile;
                round(r++).gemm[np2 - 2].push_back(q);
                cur ^= 1;
            }
        }
    }
    batches(norms, [](const NormMat& p) { return (int64_t)p.blocks; }, [&](const NormBatch& nb, unsigned n, int) {
        if (dtype == DCC_ORTHO_F32) hipLaunchKernelGGL(ortho_norm_k<float>, dim3(n), dim3(256), 0, st, nb);
        else if (dtype == DCC_ORTHO_BF16) hipLaunchKernelGGL(ortho_norm_k<__hip_bfloat16>, dim3(n), dim3(256), 0, st, nb);
        else hipLaunchKernelGGL(ortho_norm_k<__half>, dim3(n), dim3(256), 0, st, nb);
    });
    for (size_t r = 0; r < rounds.size(); ++r) {
        const Round& q = rounds[r];
        if (dtype == DCC_ORTHO_F32) launch_x<float>(q, st);
        else if (dtype == DCC_ORTHO_BF16) launch_x<__hip_bfloat16>(q, st);
        else launch_x<__half>(q, st);
        launch_x<float>(later[r], st);
        batches(q.square, [](const Square& p) { return square_tiles(p, 32); }, [&](const SquareBatch& bt, unsigned blocks, int n) {
            if (blocks >= kFewTiles) {
                hipLaunchKernelGGL(ortho_square_k<2>, dim3(blocks), dim3(64 * kWaves), 0, st, bt);
            } else {
                SquareBatch fine = bt;
                const unsigned all = number(fine, n, [](const Square& p) { return square_tiles(p, 16); });
                hipLaunchKernelGGL(ortho_square_k<1>, dim3(all), dim3(64 * kWaves), 0, st, fine);
            }
        });
        if (!launch_gemm<2>(q.gemm[0], st) || !launch_gemm<3>(q.gemm[1], st)) return dcc_fail_nothrow(kEHIP, "dcc_orthogonalize: shared memory refused");
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : dcc_fail_nothrow(kEHIP, "dcc_orthogonalize: ", hipGetErrorString(e));
} catch (...) {
    return dcc_fail_nothrow(kEINVAL, "dcc_orthogonalize: out of host memory");
}

DCC_API int dcc_muon_momentum(const float* grad, float* buf, float* dir, int64_t n, float momentum, int32_t nesterov, const float* clip,
                              void* stream) {
    if (!grad || !buf || !dir || n < 1) return dcc_fail_nothrow(kEINVAL, "dcc_muon_momentum: null pointer or n < 1");
    if ((reinterpret_cast<uintptr_t>(grad) | reinterpret_cast<uintptr_t>(buf) | reinterpret_cast<uintptr_t>(dir)) & 15)
        return dcc_fail_nothrow(kEINVAL, "dcc_muon_momentum: arrays must be 16-byte aligned");
    if (meet(grad, buf, n) || meet(grad, dir, n) || meet(buf, dir, n)) return dcc_fail_nothrow(kEINVAL, "dcc_muon_momentum: arrays must lie apart");
    const int64_t nb = std::min<int64_t>(((n >> 2) + 3 + 255) / 256, 2048);
    hipLaunchKernelGGL(muon_momentum_k, dim3((unsigned)nb), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), grad, buf, dir, (long long)n, momentum,
                       nesterov, clip);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : dcc_fail_nothrow(kEHIP, "dcc_muon_momentum: ", hipGetErrorString(e));
}

DCC_API int dcc_muon_apply(float* param, const float* dir, const dcc_muon_seg* segs, int32_t count, float keep, void* stream) {
    if (count < 0 || !param || !dir || (count > 0 && !segs)) return dcc_fail_nothrow(kEINVAL, "dcc_muon_apply: null pointer or negative count");
    if ((reinterpret_cast<uintptr_t>(param) | reinterpret_cast<uintptr_t>(dir)) & 15) return dcc_fail_nothrow(kEINVAL, "dcc_muon_apply: arrays must be 16-byte aligned");
    for (int i = 0; i < count; ++i)
        if (segs[i].offset < 0 || segs[i].offset % 4 || segs[i].numel < 0 || segs[i].numel > (1ll << 40))
            return dcc_fail_nothrow(kEINVAL, "dcc_muon_apply: a range must start at a multiple of 4 and hold 0..2^40 elements");
    int64_t end = 0;
    for (int i = 0; i < count; ++i) end = std::max(end, segs[i].offset + segs[i].numel);
    if (meet(param, dir, end)) return dcc_fail_nothrow(kEINVAL, "dcc_muon_apply: param and dir must lie apart");
    for (int from = 0; from < count; from += kMaxSegs) {
        Segs s;
        s.count = 0;
        s.keep = keep;
        int64_t first = 0;
        for (int i = from; i < count && i < from + kMaxSegs; ++i) {
            if (segs[i].numel == 0) continue;
            s.off[s.count] = segs[i].offset; s.n[s.count] = segs[i].numel; s.scale[s.count] = segs[i].scale; s.first[s.count] = (int)first;
            first += (segs[i].numel + 4095) / 4096;
            ++s.count;
        }
        if (first > 2147483647) return dcc_fail_nothrow(kEINVAL, "dcc_muon_apply: more than 2^43 elements in one list");
        if (s.count) hipLaunchKernelGGL(muon_apply_k, dim3((unsigned)first), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), param, dir, s);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : dcc_fail_nothrow(kEHIP, "dcc_muon_apply: ", hipGetErrorString(e));
}

}  // extern "C"
