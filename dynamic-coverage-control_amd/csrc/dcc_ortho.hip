// dcc_ortho.hip -- orthogonalised updates by Newton-Schulz products (include/dcc_ortho.h).
//
// Two orders of the same polynomial, chosen by shape (m <= n):
//  * m x m side (m <= 512, or n >= 5 m): A = X X^T once, then with p(A) = a I + b A + c A^2 the steps A <- p(A) A p(A), Q <- p(A) Q on
//    m x m matrices, and X <- Q X at the end: two passes over X instead of two per step.  An error of A along a direction of small
//    singular value grows by a^2 = 12 per step, so this side runs in float64 (fp64 MFMA): measured against float64 throughout, five steps
//    of 256 x 2704 are 4e-7 off, where float32 steps are 5e-6 off (and float32 on this side 1e-4).  A group holds at most five steps.
//    All its matrices are polynomials of one symmetric matrix: only lower tiles are computed, and mirrored.  |X|_F^2 is the trace of
//    the unscaled A, so nothing else reads X before the end.
//  * step by step (large and nearly square, where the float64 products would take longer): A = X X^T, B = a I + b A + c A^2, X <- B X.
// Large products over X are C = A B^T of bf16 planes: fp32 MFMA has 1/16 of the bf16 rate, so a value is kept as the sum of bf16 parts
// and the products of the parts are accumulated in float32.  float32 and float16 matrices take three parts (x = hi + mid + lo exactly:
// 8 + 8 + 8 significant bits) and the six products hh, hm, mh, hl, lh, mm; what is dropped is below 2^-23 of a product.  bfloat16 matrices
// take two parts and hh, hm, mh (2^-16 of a product: 1/64 of the half step that the result is rounded by).
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>
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
__device__ __forceinline__ double inverse_norm(const Scale& s, double* red, double* note = nullptr) {    // red: 4 doubles of LDS; all 256 threads
    if (!s.at) return 1.;
    double v = 0.;
    for (int i = threadIdx.x; i < s.n; i += 256) v += s.at[i * s.step];
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (red[0] + red[1]) + (red[2] + red[3]);
    if (note && threadIdx.x == 0) *note = v;
    return 1. / (sqrt(v) + (double)s.eps);
}

struct NormMat { const void* x; double* out; long long n; int blocks, first; };
struct NormBatch { NormMat m[2 * kMaxProds]; int n; };

// sum of squares in float64, by fixed ranges
template <typename E>
__global__ __launch_bounds__(256) void ortho_norm_k(const NormBatch nb) {
    __shared__ double red[4];
    int i = 0;
    while (i + 1 < nb.n && (int)blockIdx.x >= nb.m[i + 1].first) ++i;
    const NormMat& m = nb.m[i];
    const E* x = reinterpret_cast<const E*>(m.x);
    const int blk = blockIdx.x - m.first;
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
// consecutive k make four steps.  Square matrices are stored [mq][mq], mq = m rounded up to 16, zero outside m: no bounds to check.
struct Gram {                           // out = X X^T, X [m, K] in memory as [m][K] or, tall, [K][m]
    const void* x;
    double *out, *part;                 // part: [slices][mq * mq] where slices > 1
    long long ld;
    int m, mq, K, slices, kper, first;  // kper: a multiple of 16
};
struct GramBatch { Gram p[kMaxProds]; int n; };

// four values of row i (< m, or cleared) at depth k
template <typename E, bool TALL, bool VEC>
__device__ __forceinline__ d4 fetch_x(const E* x, long long ld, int i, int m, int k, int kend) {
    d4 v;
    const int ic = i < m ? i : m - 1;
    if constexpr (VEC) {
        struct alignas(4 * sizeof(E)) Four { E e[4]; };
        const Four f = *reinterpret_cast<const Four*>(x + (long long)ic * ld + (k < kend ? k : 0));
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = i < m && k < kend ? (double)get(f.e[j]) : 0.;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int kc = k + j < kend ? k + j : kend - 1;
            const float f = get(TALL ? x[(long long)kc * ld + ic] : x[(long long)ic * ld + kc]);
            v[j] = i < m && k + j < kend ? (double)f : 0.;
        }
    }
    return v;
}

__device__ __forceinline__ void mirror(double* out, int mq, int i, int j, double v) {
    out[(long long)i * mq + j] = v;
    out[(long long)j * mq + i] = v;
}

// WIDE: a 64 x 64 tile by 2 x 2 waves of 32 x 32 (long depths, where reading the operands counts); else a 16 x 16 tile whose depth the
// four waves share (short ones, where latency does).  VEC: rows of X may be read four elements at a time (K a multiple of 4).
template <typename E, bool TALL, bool VEC, bool WIDE>
__global__ __launch_bounds__(256) void ortho_gram_k(const GramBatch bt) {
    constexpr int T = WIDE ? 2 : 1, TM = WIDE ? 64 : 16;
    __shared__ double sh[WIDE ? 1 : 4 * 256];
    int pi = 0;
    while (pi + 1 < bt.n && (int)blockIdx.x >= bt.p[pi + 1].first) ++pi;
    const Gram& p = bt.p[pi];
    const E* x = reinterpret_cast<const E*>(p.x);
    const int blk = blockIdx.x - p.first, slice = blk % p.slices, m = p.m, mq = p.mq;
    const long long ld = p.ld;
    int ti, tj;
    lower_tile(blk / p.slices, ti, tj);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, g = lane >> 4;
    const int i0 = ti * TM + (WIDE ? (wave >> 1) * 32 : 0), j0 = tj * TM + (WIDE ? (wave & 1) * 32 : 0);
    int kbeg = slice * p.kper, kend = kbeg + p.kper < p.K ? kbeg + p.kper : p.K;
    if (!WIDE) {
        const int quarter = ((kend - kbeg + 3) / 4 + 15) & ~15;
        kbeg += wave * quarter;
        kend = kbeg + quarter < kend ? kbeg + quarter : kend;
    }
    d4 acc[T][T];
#pragma unroll
    for (int a = 0; a < T; ++a)
#pragma unroll
        for (int c = 0; c < T; ++c) acc[a][c] = d4{0., 0., 0., 0.};
    if (kbeg < kend) {
        d4 na[T], nb[T];
#pragma unroll
        for (int t = 0; t < T; ++t) {
            na[t] = fetch_x<E, TALL, VEC>(x, ld, i0 + 16 * t + li, m, kbeg + 4 * g, kend);
            nb[t] = fetch_x<E, TALL, VEC>(x, ld, j0 + 16 * t + li, m, kbeg + 4 * g, kend);
        }
        for (int k = kbeg; k < kend; k += 16) {
            d4 a[T], b[T];
#pragma unroll
            for (int t = 0; t < T; ++t) { a[t] = na[t]; b[t] = nb[t]; }
            const int kn = k + 16 < kend ? k + 16 : k;
#pragma unroll
            for (int t = 0; t < T; ++t) {
                na[t] = fetch_x<E, TALL, VEC>(x, ld, i0 + 16 * t + li, m, kn + 4 * g, kend);
                nb[t] = fetch_x<E, TALL, VEC>(x, ld, j0 + 16 * t + li, m, kn + 4 * g, kend);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int s = 0; s < T; ++s)
#pragma unroll
                    for (int c = 0; c < T; ++c) acc[s][c] = __builtin_amdgcn_mfma_f64_16x16x4f64(a[s][r], b[c][r], acc[s][c], 0, 0, 0);
        }
    }
    if (!WIDE) {
#pragma unroll
        for (int r = 0; r < 4; ++r) sh[wave * 256 + (4 * r + g) * 16 + li] = acc[0][0][r];
        __syncthreads();
        const int i = i0 + (threadIdx.x >> 4), j = j0 + (threadIdx.x & 15);
        const double v = (sh[threadIdx.x] + sh[256 + threadIdx.x]) + (sh[512 + threadIdx.x] + sh[768 + threadIdx.x]);
        if (j <= i) {
            if (p.slices > 1) p.part[((long long)slice * mq + i) * mq + j] = v;
            else mirror(p.out, mq, i, j, v);
        }
        return;
    }
#pragma unroll
    for (int s = 0; s < T; ++s)
#pragma unroll
        for (int c = 0; c < T; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = i0 + 16 * s + 4 * r + g, j = j0 + 16 * c + li;
                if (i >= mq || j > i) continue;
                if (p.slices > 1) p.part[((long long)slice * mq + i) * mq + j] = acc[s][c][r];
                else mirror(p.out, mq, i, j, acc[s][c][r]);
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
        for (int q = 0; q < p.slices; ++q) s += p.part[q * n + at];
        mirror(p.out, p.mq, i, j, s);
    }
}

// Three planes of a value (NP 2: two).  All but the last part are truncated, so that the parts add up to the value exactly while it has
// bits left; the last is rounded to nearest.
template <int NP>
__device__ __forceinline__ void split(float v, ushort_t (&h)[NP]) {
#pragma unroll
    for (int s = 0; s + 1 < NP; ++s) {
        const unsigned u = __float_as_uint(v) & 0xffff0000u;
        h[s] = (ushort_t)(u >> 16);
        v -= __uint_as_float(u);
    }
    const __hip_bfloat16 r = __float2bfloat16(v);
    h[NP - 1] = __builtin_bit_cast(ushort_t, r);
}

struct Square {                         // out = alpha A B + beta E + diag I, all symmetric [mq][mq]; A is E of the unscaled matrix: see sa
    const double *a, *b, *e;
    double* out;                        // null: three planes instead, [mp][mp] of stride plane
    ushort_t* planes;
    long long plane;
    int m, mq, mp, first;
    double alpha, beta, diag;
    Scale s;                            // beta (E) is scaled by 1 / norm^2, alpha by its power sa (twice for A A of the unscaled A)
    int sa;
    double* note;                       // the first workgroup leaves norm^2 here, or null
};
struct SquareBatch { Square p[kMaxProds]; int n; };

__global__ __launch_bounds__(256) void ortho_square_k(const SquareBatch bt) {
    __shared__ double sh[4 * 256], red[4];
    int pi = 0;
    while (pi + 1 < bt.n && (int)blockIdx.x >= bt.p[pi + 1].first) ++pi;
    const Square& p = bt.p[pi];
    int ti, tj;
    lower_tile(blockIdx.x - p.first, ti, tj);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, g = lane >> 4, mq = p.mq;
    const int i0 = ti * 16, j0 = tj * 16;
    d4 acc0 = {0., 0., 0., 0.}, acc1 = acc0;
    if (i0 < mq) {                      // (padded planes reach behind mq: zeros)
        const int quarter = ((mq + 3) / 4 + 15) & ~15, kbeg = wave * quarter, kend = kbeg + quarter < mq ? kbeg + quarter : mq;
        const double* pa = p.a + (long long)(i0 + li) * mq + 4 * g;
        const double* pb = p.b + (long long)(j0 + li) * mq + 4 * g;
        for (int k = kbeg; k < kend; k += 16) {
            const d4 a = *reinterpret_cast<const d4*>(pa + k), b = *reinterpret_cast<const d4*>(pb + k);
            acc0 = __builtin_amdgcn_mfma_f64_16x16x4f64(a[0], b[0], acc0, 0, 0, 0);
            acc1 = __builtin_amdgcn_mfma_f64_16x16x4f64(a[1], b[1], acc1, 0, 0, 0);
            acc0 = __builtin_amdgcn_mfma_f64_16x16x4f64(a[2], b[2], acc0, 0, 0, 0);
            acc1 = __builtin_amdgcn_mfma_f64_16x16x4f64(a[3], b[3], acc1, 0, 0, 0);
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) sh[wave * 256 + (4 * r + g) * 16 + li] = acc0[r] + acc1[r];
    const double inv = inverse_norm(p.s, red, (int)blockIdx.x == p.first ? p.note : nullptr), inv2 = inv * inv;
    __syncthreads();
    const int i = i0 + (threadIdx.x >> 4), j = j0 + (threadIdx.x & 15);
    double v = (sh[threadIdx.x] + sh[256 + threadIdx.x]) + (sh[512 + threadIdx.x] + sh[768 + threadIdx.x]);
    v *= p.alpha * (p.sa > 1 ? inv2 * inv2 : p.sa > 0 ? inv2 : 1.);
    if (j > i) return;
    if (p.e && i < mq) v += p.beta * inv2 * p.e[(long long)i * mq + j];
    if (i == j && i < p.m) v += p.diag;
    if (p.out) {
        mirror(p.out, mq, i, j, v);
    } else {
        // (rounded once, from 64 bits to the planes' 24)
        const float hi = (float)v;
        ushort_t h[3];
        split<3>(hi, h);
#pragma unroll
        for (int s = 0; s < 3; ++s) {
            p.planes[s * p.plane + (long long)i * p.mp + j] = h[s];
            p.planes[s * p.plane + (long long)j * p.mp + i] = h[s];
        }
    }
}

// X <- Q X in float64, for products that are too small to split: a 16 x 16 tile per wave, operands straight from memory.
struct Apply {                          // out [rows][cols] = Q X (wide: X [m][n]) or X Q (tall: X [n][m])
    const void* x;
    const double* q;
    void* out;
    long long ld;                       // of X and out
    int m, mq, rows, cols, tcols, dto, first;
    Scale s;
};
struct ApplyBatch { Apply p[kMaxProds]; int n; };

template <typename E, bool TALL>
__global__ __launch_bounds__(256) void ortho_apply_k(const ApplyBatch bt) {
    __shared__ double red[4];
    int pi = 0;
    while (pi + 1 < bt.n && (int)blockIdx.x >= bt.p[pi + 1].first) ++pi;
    const Apply& p = bt.p[pi];
    const E* x = reinterpret_cast<const E*>(p.x);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, g = lane >> 4, m = p.m, mq = p.mq;
    const long long ld = p.ld;
    const double inv = inverse_norm(p.s, red);
    const int tile = (blockIdx.x - p.first) * 4 + wave, ti = tile / p.tcols, tj = tile - ti * p.tcols, i0 = ti * 16, j0 = tj * 16;
    if (i0 >= p.rows) return;
    d4 acc0 = {0., 0., 0., 0.}, acc1 = acc0;
    const double* pq = p.q + (long long)((TALL ? j0 : i0) + li) * mq + 4 * g;
    const int row = TALL ? (i0 + li < p.rows ? i0 + li : p.rows - 1) : 0, c = TALL ? 0 : (j0 + li < p.cols ? j0 + li : p.cols - 1);
    for (int k = 0; k < mq; k += 16) {
        const d4 q = *reinterpret_cast<const d4*>(pq + k);
        double v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int kk = k + 4 * g + r, kc = kk < m ? kk : m - 1;         // (Q is zero behind m)
            v[r] = get(TALL ? x[(long long)row * ld + kc] : x[(long long)kc * ld + c]);
        }
        if (TALL) {
            acc0 = __builtin_amdgcn_mfma_f64_16x16x4f64(v[0], q[0], acc0, 0, 0, 0);
            acc1 = __builtin_amdgcn_mfma_f64_16x16x4f64(v[1], q[1], acc1, 0, 0, 0);
            acc0 = __builtin_amdgcn_mfma_f64_16x16x4f64(v[2], q[2], acc0, 0, 0, 0);
            acc1 = __builtin_amdgcn_mfma_f64_16x16x4f64(v[3], q[3], acc1, 0, 0, 0);
        } else {
            acc0 = __builtin_amdgcn_mfma_f64_16x16x4f64(q[0], v[0], acc0, 0, 0, 0);
            acc1 = __builtin_amdgcn_mfma_f64_16x16x4f64(q[1], v[1], acc1, 0, 0, 0);
            acc0 = __builtin_amdgcn_mfma_f64_16x16x4f64(q[2], v[2], acc0, 0, 0, 0);
            acc1 = __builtin_amdgcn_mfma_f64_16x16x4f64(q[3], v[3], acc1, 0, 0, 0);
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int i = i0 + 4 * r + g, j = j0 + li;
        if (i < p.rows && j < p.cols) store1(p.out, (long long)i * ld + j, p.dto, (float)((acc0[r] + acc1[r]) * inv));
    }
}

// ---- plane products ------------------------------------------------------------------------------------------------------------
struct Split {                          // planes of the scaled X [R][C]: as it lies (`same` [rp][cp]) and / or transposed (`turned` [cp][rp])
    const void* x;
    ushort_t *same, *turned;
    long long plane;                    // elements between planes
    int R, C, rp, cp, tcols, first;     // padded to kTile with zeros
    Scale s;
};
struct SplitBatch { Split p[kMaxProds]; int n; };

template <typename E, int NP>
__global__ __launch_bounds__(256) void ortho_split_k(const SplitBatch bt) {
    __shared__ double red[4];
    __shared__ alignas(16) ushort_t sh[NP][64][72];         // transposed tile: rows of 144 bytes
    int pi = 0;
    while (pi + 1 < bt.n && (int)blockIdx.x >= bt.p[pi + 1].first) ++pi;
    const Split& p = bt.p[pi];
    const E* x = reinterpret_cast<const E*>(p.x);
    const int blk = blockIdx.x - p.first, i0 = blk / p.tcols * 64, j0 = blk % p.tcols * 64;
    const float inv = (float)inverse_norm(p.s, red);
    const int c = threadIdx.x & 63, r0 = threadIdx.x >> 6;
    const int jc = j0 + c < p.C ? j0 + c : p.C - 1;
    float v[16];
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        const int i = i0 + r0 * 16 + q, ic = i < p.R ? i : p.R - 1;
        v[q] = get(x[(long long)ic * p.C + jc]);
        v[q] = i < p.R && j0 + c < p.C ? v[q] * inv : 0.f;
    }
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        ushort_t h[NP];
        split<NP>(v[q], h);
#pragma unroll
        for (int s = 0; s < NP; ++s) {
            if (p.same) p.same[s * p.plane + (long long)(i0 + r0 * 16 + q) * p.cp + j0 + c] = h[s];
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
            *reinterpret_cast<u4*>(p.turned + s * p.plane + (long long)(j0 + j) * p.rp + i0 + i) = *reinterpret_cast<const u4*>(&sh[s][j][i]);
        }
}

struct Gemm {                           // v = alpha A B^T + beta E + diag I
    const ushort_t *a, *b, *e;          // planes; rows of A and B are contiguous over the depth
    ushort_t *d1, *d2;                  // planes of v as [i][j] and as [j][i] (either may be null)
    void* out;                          // or, bounded by rows and cols, v itself
    long long pa, pb, pe, p1, p2, ldo;  // elements between planes; row length of out
    int lda, ldb, lde, ld1, ld2, K, rows, cols, dto, sym, tcols, first;     // K: a multiple of kBK
    float alpha, beta, diag;
};
struct GemmBatch { Gemm p[kMaxProds]; int n; };

// 16-byte piece kg of row i in a staged slice: the pieces of a row are turned by i / 4, so that the 16 rows that one MFMA operand
// reads at one kg lie in 16 different groups of banks
__device__ __forceinline__ int piece(int i, int kg) { return i * 4 + (kg ^ ((i >> 2) & 3)); }

// One 128 x 128 tile of one product: 4 waves as 2 x 2 of 64 x 64, slices of 32 in two stages that go to LDS directly.
template <int NP>
__global__ __launch_bounds__(256) void ortho_gemm_k(const GemmBatch bt) {
    constexpr int kSlice = kTile * 4;                   // 16-byte pieces of one plane's slice
    constexpr int kStage = 2 * NP * kSlice;
    extern __shared__ u4 lds[];                         // [2][2 * NP][kSlice]
    int pi = 0;
    while (pi + 1 < bt.n && (int)blockIdx.x >= bt.p[pi + 1].first) ++pi;
    const Gemm& p = bt.p[pi];
    const int blk = blockIdx.x - p.first;
    int ti, tj;
    if (p.sym) {
        lower_tile(blk, ti, tj);
    } else {
        ti = blk / p.tcols;
        tj = blk - ti * p.tcols;
    }
    const int i0 = ti * kTile, j0 = tj * kTile;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, kg = lane >> 4, g4 = kg << 2;
    const int wi = (wave >> 1) * 64, wj = (wave & 1) * 64;
    // wave w brings rows 32 w .. 32 w + 31 of every plane, 16 at a time: lane l puts piece l % 4 of row l / 4
    const int lrow = 32 * wave + (lane >> 2), lk = ((lane & 3) ^ ((lane >> 4) & 3)) * 8;
    const ushort_t* ga = p.a + (long long)(i0 + lrow) * p.lda + lk;
    const ushort_t* gb = p.b + (long long)(j0 + lrow) * p.ldb + lk;
    const long long ra = 16ll * p.lda, rb = 16ll * p.ldb, pa = p.pa, pb = p.pb;
    auto stage = [&](int which) {
        u4* base = lds + which * kStage + wave * 128;
#pragma unroll
        for (int s = 0; s < NP; ++s)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(ga + s * pa + q * ra),
                                                 (__attribute__((address_space(3))) void*)(base + s * kSlice + q * 64), 16, 0, 0);
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(gb + s * pb + q * rb),
                                                 (__attribute__((address_space(3))) void*)(base + (NP + s) * kSlice + q * 64), 16, 0, 0);
            }
        ga += kBK;
        gb += kBK;
    };
    f4 acc[4][4];
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[x][y] = f4{0.f, 0.f, 0.f, 0.f};
    const int steps = p.K / kBK;
    stage(0);
    for (int k = 0; k < steps; ++k) {
        if (k + 1 < steps) {
            stage((k + 1) & 1);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(4 * NP) : "memory");       // all but the 4 NP loads just issued
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        __syncthreads();
        const u4* sa = lds + (k & 1) * kStage;
        const u4* sb = sa + NP * kSlice;
        bf8 fb[4][NP];
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
            for (int s = 0; s < NP; ++s) fb[y][s] = __builtin_bit_cast(bf8, sb[s * kSlice + piece(wj + 16 * y + li, kg)]);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            bf8 fa[NP];
#pragma unroll
            for (int s = 0; s < NP; ++s) fa[s] = __builtin_bit_cast(bf8, sa[s * kSlice + piece(wi + 16 * x + li, kg)]);
            // small products first
#pragma unroll
            for (int o = NP - 1; o >= 0; --o)
#pragma unroll
                for (int s = 0; s <= o; ++s)
#pragma unroll
                    for (int y = 0; y < 4; ++y) acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[s], fb[y][o - s], acc[x][y], 0, 0, 0);
        }
        __syncthreads();
    }
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            const int i = i0 + wi + 16 * x + g4, j = j0 + wj + 16 * y + li;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float v = p.alpha * acc[x][y][r];
                if (p.e) {
                    float e = 0.f;
#pragma unroll
                    for (int s = NP - 1; s >= 0; --s) e += __uint_as_float((unsigned)p.e[s * p.pe + (long long)(i + r) * p.lde + j] << 16);
                    v += p.beta * e;
                    if (i + r == j && j < p.rows) v += p.diag;
                }
                acc[x][y][r] = v;
                if (p.out && i + r < p.rows && j < p.cols) store1(p.out, (long long)(i + r) * p.ldo + j, p.dto, v);
            }
        }
    if (p.out) return;
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
                for (int y = 0; y < 4; ++y) {
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
            const long long pl = s * (turn ? p.p2 : p.p1);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const int e = threadIdx.x + q * 256, r = e >> 4, c = (e & 15) * 8;
                *reinterpret_cast<u4*>(dst + pl + (long long)(ro + r) * ld + co + c) = *reinterpret_cast<const u4*>(sh + r * kRow + c);
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

// the m x m side in float64: always for small m (its products are latency there), else where n is long enough to pay for their rate
bool on_square_side(const Shape& s) { return s.m <= 512 || s.n >= 5 * s.m; }
constexpr int kGroup = 5;               // steps on that side before X X^T is formed anew
// X <- Q X there in float64 where that takes no longer than splitting X first (at about 50 TFLOP/s, 15 us)
bool small_apply(const Shape& s) { return 2 * s.m * s.m * s.n < 750000000; }

// tiles of 64 for long depths of X X^T, and then as many depth slices as fill the chip twice, none shorter than 256
bool wide_gram(const Shape& s) { return s.n >= 4096; }
int gram_slices(const Shape& s) {
    const int64_t nt = (s.m + 63) / 64, tiles = nt * (nt + 1) / 2;
    if (!wide_gram(s)) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(4 * kChip / tiles, s.n / 256), 128));
}
int planes_of(int dtype) { return dtype == DCC_ORTHO_BF16 ? 2 : 3; }
int norm_blocks(const dcc_ortho_mat& t) { return (int)std::max<int64_t>(1, std::min<int64_t>(kNormBlocks, t.M * t.N / 4096)); }

// where a matrix's intermediate results lie in the workspace
struct Place { int64_t norm, A, B, W, Q0, Q1, Qp, Xp, Xt0, Xt1, X0, X1, part, end; };
Place place_of(const Shape& s, int dtype, int steps, int64_t at) {
    Place p = {};
    auto take = [&](int64_t bytes) { const int64_t o = at; at += up(bytes, kAlign); return o; };
    const int64_t mq = up(s.m, 16), mp = up(s.m, kTile), np = up(s.n, kTile), mn = 4 * s.m * s.n, np2 = 2 * planes_of(dtype);
    if (on_square_side(s)) {
        p.norm = take(8);
        p.A = take(8 * mq * mq); p.B = take(8 * mq * mq); p.W = take(8 * mq * mq); p.Q0 = take(8 * mq * mq); p.Q1 = take(8 * mq * mq);
        if (!small_apply(s)) { p.Qp = take(6 * mp * mp); p.Xt0 = take(6 * mp * np); }
        if (gram_slices(s) > 1) p.part = take(8 * mq * mq * gram_slices(s));
        if (steps > kGroup) p.X0 = take(mn);
        if (steps > 2 * kGroup) p.X1 = take(mn);
    } else {
        p.norm = take(8 * kNormBlocks);
        p.A = take(np2 * mp * mp); p.B = take(np2 * mp * mp);
        p.Xp = take(np2 * mp * np); p.Xt0 = take(np2 * mp * np);
        if (steps > 1) p.Xt1 = take(np2 * mp * np);
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

// calls f with batches of at most kMaxProds of `all`, their first blocks set from blocks(p)
template <typename Batch, typename P, typename Blocks, typename F>
void batches(const std::vector<P>& all, Blocks blocks, F f) {
    for (size_t from = 0; from < all.size(); from += kMaxProds) {
        Batch bt;
        bt.n = (int)std::min<size_t>(kMaxProds, all.size() - from);
        int64_t first = 0;
        for (int i = 0; i < bt.n; ++i) {
            bt.p[i] = all[from + i];
            bt.p[i].first = (int)first;
            first += blocks(bt.p[i]);
        }
        f(bt, (unsigned)first);
    }
}
int64_t lower(int64_t t) { return t * (t + 1) / 2; }

// a round: products (of all matrices) that do not depend on each other
struct Round {
    std::vector<Gram> gram[2][2][2];    // [tall][vec][wide]
    std::vector<Square> square;
    std::vector<Split> split[2];        // [planes - 2]
    std::vector<Gemm> gemm[2];
    std::vector<Apply> apply[2];        // [tall]
};

template <typename E, bool TALL, bool VEC, bool WIDE>
void launch_gram(const std::vector<Gram>& all, hipStream_t st) {
    constexpr int tm = WIDE ? 64 : 16;
    batches<GramBatch>(all, [](const Gram& p) { return lower((p.mq + tm - 1) / tm) * p.slices; }, [&](const GramBatch& bt, unsigned blocks) {
        hipLaunchKernelGGL((ortho_gram_k<E, TALL, VEC, WIDE>), dim3(blocks), dim3(256), 0, st, bt);
        int64_t longest = 0;
        for (int i = 0; i < bt.n; ++i)
            if (bt.p[i].slices > 1) longest = std::max<int64_t>(longest, (int64_t)bt.p[i].mq * bt.p[i].mq);
        if (longest) hipLaunchKernelGGL(ortho_join_k, dim3((unsigned)std::min<int64_t>((longest + 255) / 256, 1024), bt.n), dim3(256), 0, st, bt);
    });
}
template <typename E>
void launch_x(const Round& q, hipStream_t st) {         // what reads X: E is its type
    launch_gram<E, false, false, false>(q.gram[0][0][0], st);
    launch_gram<E, false, false, true>(q.gram[0][0][1], st);
    launch_gram<E, false, true, false>(q.gram[0][1][0], st);
    launch_gram<E, false, true, true>(q.gram[0][1][1], st);
    launch_gram<E, true, false, false>(q.gram[1][0][0], st);
    launch_gram<E, true, false, true>(q.gram[1][0][1], st);
    const auto tiles = [](const Split& p) { return (int64_t)(p.rp / 64) * (p.cp / 64); };
    batches<SplitBatch>(q.split[0], tiles, [&](const SplitBatch& bt, unsigned n) { hipLaunchKernelGGL((ortho_split_k<E, 2>), dim3(n), dim3(256), 0, st, bt); });
    batches<SplitBatch>(q.split[1], tiles, [&](const SplitBatch& bt, unsigned n) { hipLaunchKernelGGL((ortho_split_k<E, 3>), dim3(n), dim3(256), 0, st, bt); });
    const auto quads = [](const Apply& p) { return ((int64_t)((p.rows + 15) / 16) * p.tcols + 3) / 4; };
    batches<ApplyBatch>(q.apply[0], quads, [&](const ApplyBatch& bt, unsigned n) { hipLaunchKernelGGL((ortho_apply_k<E, false>), dim3(n), dim3(256), 0, st, bt); });
    batches<ApplyBatch>(q.apply[1], quads, [&](const ApplyBatch& bt, unsigned n) { hipLaunchKernelGGL((ortho_apply_k<E, true>), dim3(n), dim3(256), 0, st, bt); });
}
template <int NP>
bool launch_gemm(const std::vector<Gemm>& all, hipStream_t st) {
    constexpr int bytes = 2 * 2 * NP * kTile * 4 * 16;
    if (all.empty()) return true;
    if (bytes > 65536 && hipFuncSetAttribute(reinterpret_cast<const void*>(ortho_gemm_k<NP>), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return false;
    const auto tiles = [](const Gemm& p) { const int64_t t = (p.rows + kTile - 1) / kTile; return p.sym ? lower(t) : t * p.tcols; };
    batches<GemmBatch>(all, tiles, [&](const GemmBatch& bt, unsigned n) { hipLaunchKernelGGL(ortho_gemm_k<NP>, dim3(n), dim3(256), bytes, st, bt); });
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
    if (const char* e = list_error(mats, count, dtype, steps)) return dcc_fail(kEINVAL, std::string("dcc_orthogonalize: ") + e);
    if (!(eps >= 0.f)) return dcc_fail(kEINVAL, "dcc_orthogonalize: eps must not be negative");
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const int64_t esize = dtype == DCC_ORTHO_F32 ? 4 : 2;
    std::vector<int> live;
    for (int i = 0; i < count; ++i) {
        if (mats[i].M == 0 || mats[i].N == 0) continue;
        if (!mats[i].in || !mats[i].out) return dcc_fail(kEINVAL, "dcc_orthogonalize: null matrix");
        if ((reinterpret_cast<uintptr_t>(mats[i].in) | reinterpret_cast<uintptr_t>(mats[i].out)) & (esize - 1))
            return dcc_fail(kEINVAL, "dcc_orthogonalize: a matrix is not aligned to its elements");
        live.push_back(i);
    }
    if (live.empty()) return 0;
    auto meet = [&](const void* x, const void* y, int64_t nx, int64_t ny) {
        const uintptr_t p = reinterpret_cast<uintptr_t>(x), q = reinterpret_cast<uintptr_t>(y);
        return p < q + ny * esize && q < p + nx * esize;
    };
    for (int i : live)
        for (int j : live) {
            const int64_t ni = mats[i].M * mats[i].N, nj = mats[j].M * mats[j].N;
            if (meet(mats[i].out, mats[j].in, ni, nj) || (i != j && meet(mats[i].out, mats[j].out, ni, nj)))
                return dcc_fail(kEINVAL, "dcc_orthogonalize: an output overlaps an input or another output");
        }
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & (kAlign - 1))) return dcc_fail(kEINVAL, "dcc_orthogonalize: workspace must be 256-byte aligned");
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
        const int64_t pmm = (int64_t)mp * mp, pmn = (int64_t)mp * np;
        size_t r = 0;
        int left = steps;
        if (on_square_side(s)) {
            const void* X = t.in;
            bool raw = true, flip = false;
            double *A = reinterpret_cast<double*>(ws + pl.A), *B = reinterpret_cast<double*>(ws + pl.B), *W = reinterpret_cast<double*>(ws + pl.W);
            double* Qs[2] = {reinterpret_cast<double*>(ws + pl.Q0), reinterpret_cast<double*>(ws + pl.Q1)};
            ushort_t* Qp = small_apply(s) ? nullptr : reinterpret_cast<ushort_t*>(ws + pl.Qp);
            auto square = [&](const double* x, const double* y, double* out) {
                Square p = {};
                p.a = x; p.b = y; p.out = out; p.m = m; p.mq = p.mp = mq; p.alpha = 1.;
                return p;
            };
            auto to_planes = [&](Square& p) { p.out = nullptr; p.planes = Qp; p.plane = pmm; p.mp = mp; };
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
                g.kper = (int)up((n + gram_slices(s) - 1) / gram_slices(s), 16);
                g.slices = (n + g.kper - 1) / g.kper;
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
                    if (k == 0 && end && Qp) to_planes(p);
                    round(r++).square.push_back(p);
                    double* Pk = k > 0 ? B : Qs[0];
                    if (k > 0) {                                        // Q <- p(A) Q
                        Square q = square(Pk, Qs[cur], Qs[cur ^ 1]);
                        if (end && Qp) to_planes(q);
                        round(r).square.push_back(q);
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
                if (Qp) {
                    ushort_t* Xt = reinterpret_cast<ushort_t*>(ws + pl.Xt0);        // [np][mp]: X^T
                    Split sp = {};
                    sp.x = X; sp.plane = pmn; sp.R = (int)t.M; sp.C = (int)t.N; sp.rp = s.tall ? np : mp; sp.cp = s.tall ? mp : np;
                    (s.tall ? sp.same : sp.turned) = Xt;
                    sp.tcols = sp.cp / 64; sp.s = scale;
                    if (len == 1) ++r;                                  // (not beside the p(A) that notes the norm)
                    round(r - 1);
                    (raw ? rounds : later)[r - 1].split[1].push_back(sp);
                    Gemm q = {};
                    q.a = s.tall ? Xt : Qp; q.b = s.tall ? Qp : Xt; q.pa = s.tall ? pmn : pmm; q.pb = s.tall ? pmm : pmn;
                    q.lda = q.ldb = mp; q.K = mp; q.rows = (int)t.M; q.cols = (int)t.N; q.ldo = t.N; q.out = out; q.dto = last ? dtype : 0;
                    q.tcols = (int)(up(t.N, kTile) / kTile); q.alpha = 1.f;
                    round(r++).gemm[1].push_back(q);
                } else {
                    Apply q = {};
                    q.x = X; q.q = Qs[cur]; q.out = out; q.ld = t.N; q.m = m; q.mq = mq; q.rows = (int)t.M; q.cols = (int)t.N;
                    q.tcols = (int)((t.N + 15) / 16); q.dto = last ? dtype : 0; q.s = scale;
                    round(r);
                    (raw ? rounds : later)[r++].apply[s.tall].push_back(q);
                }
                X = out;
                raw = false;
            }
        } else {
            const int np2 = planes_of(dtype), nb = norm_blocks(t);
            ushort_t *A = reinterpret_cast<ushort_t*>(ws + pl.A), *B = reinterpret_cast<ushort_t*>(ws + pl.B), *Xp = reinterpret_cast<ushort_t*>(ws + pl.Xp);
            ushort_t* Xt[2] = {reinterpret_cast<ushort_t*>(ws + pl.Xt0), reinterpret_cast<ushort_t*>(ws + pl.Xt1)};
            double* norm = reinterpret_cast<double*>(ws + pl.norm);
            norms.push_back(NormMat{t.in, norm, t.M * t.N, nb, 0});
            Split sp = {};
            sp.x = t.in; sp.plane = pmn; sp.R = (int)t.M; sp.C = (int)t.N; sp.rp = s.tall ? np : mp; sp.cp = s.tall ? mp : np;
            sp.same = s.tall ? Xt[0] : Xp; sp.turned = s.tall ? Xp : Xt[0];
            sp.tcols = sp.cp / 64; sp.s = Scale{norm, 1, nb, eps};
            round(r++).split[np2 - 2].push_back(sp);
            int cur = 0;
            while (left > 0) {
                --left;
                Gemm g = {};            // A = X X^T
                g.a = g.b = Xp; g.pa = g.pb = pmn; g.lda = g.ldb = np; g.K = np; g.rows = g.cols = m; g.sym = 1; g.alpha = 1.f;
                g.d1 = g.d2 = A; g.p1 = g.p2 = pmm; g.ld1 = g.ld2 = mp; g.tcols = mp / kTile;
                round(r++).gemm[np2 - 2].push_back(g);
                Gemm p = g;             // B = a I + b A + c A^2
                p.a = p.b = p.e = A; p.pa = p.pb = p.pe = pmm; p.lda = p.ldb = p.lde = mp; p.K = mp; p.d1 = p.d2 = B; p.alpha = c; p.beta = b; p.diag = a;
                round(r++).gemm[np2 - 2].push_back(p);
                Gemm q = {};            // X <- B X
                q.K = q.lda = q.ldb = mp; q.alpha = 1.f;
                if (left == 0) {
                    q.a = s.tall ? Xt[cur] : B; q.b = s.tall ? B : Xt[cur]; q.pa = s.tall ? pmn : pmm; q.pb = s.tall ? pmm : pmn;
                    q.rows = (int)t.M; q.cols = (int)t.N; q.out = t.out; q.ldo = t.N; q.dto = dtype;
                } else {                // as [m][n] for the next X X^T, as [n][m] for the next step
                    q.a = B; q.pa = pmm; q.b = Xt[cur]; q.pb = pmn; q.rows = m; q.cols = n;
                    q.d1 = Xp; q.p1 = pmn; q.ld1 = np; q.d2 = Xt[cur ^ 1]; q.p2 = pmn; q.ld2 = mp;
                }
                q.tcols = (q.cols + kTile - 1) / kTile;
                round(r++).gemm[np2 - 2].push_back(q);
                cur ^= 1;
            }
        }
    }
    for (size_t from = 0; from < norms.size(); from += 2 * kMaxProds) {
        NormBatch nb;
        nb.n = (int)std::min<size_t>(2 * kMaxProds, norms.size() - from);
        int first = 0;
        for (int i = 0; i < nb.n; ++i) {
            nb.m[i] = norms[from + i];
            nb.m[i].first = first;
            first += nb.m[i].blocks;
        }
        if (dtype == DCC_ORTHO_F32) hipLaunchKernelGGL(ortho_norm_k<float>, dim3(first), dim3(256), 0, st, nb);
        else if (dtype == DCC_ORTHO_BF16) hipLaunchKernelGGL(ortho_norm_k<__hip_bfloat16>, dim3(first), dim3(256), 0, st, nb);
        else hipLaunchKernelGGL(ortho_norm_k<__half>, dim3(first), dim3(256), 0, st, nb);
    }
    for (size_t r = 0; r < rounds.size(); ++r) {
        const Round& q = rounds[r];
        if (dtype == DCC_ORTHO_F32) launch_x<float>(q, st);
        else if (dtype == DCC_ORTHO_BF16) launch_x<__hip_bfloat16>(q, st);
        else launch_x<__half>(q, st);
        launch_x<float>(later[r], st);
        batches<SquareBatch>(q.square, [](const Square& p) { return lower(p.mp / 16); },
                             [&](const SquareBatch& bt, unsigned blocks) { hipLaunchKernelGGL(ortho_square_k, dim3(blocks), dim3(256), 0, st, bt); });
        if (!launch_gemm<2>(q.gemm[0], st) || !launch_gemm<3>(q.gemm[1], st)) return dcc_fail(kEHIP, "dcc_orthogonalize: shared memory refused");
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : dcc_fail(kEHIP, std::string("dcc_orthogonalize: ") + hipGetErrorString(e));
} catch (...) {
    return dcc_fail(kEINVAL, "dcc_orthogonalize: out of host memory");
}

DCC_API int dcc_muon_momentum(const float* grad, float* buf, float* dir, int64_t n, float momentum, int32_t nesterov, const float* clip,
                              void* stream) {
    if (!grad || !buf || !dir || n < 1) return dcc_fail(kEINVAL, "dcc_muon_momentum: null pointer or n < 1");
    if ((reinterpret_cast<uintptr_t>(grad) | reinterpret_cast<uintptr_t>(buf) | reinterpret_cast<uintptr_t>(dir)) & 15)
        return dcc_fail(kEINVAL, "dcc_muon_momentum: arrays must be 16-byte aligned");
    const int64_t nb = std::min<int64_t>(((n >> 2) + 3 + 255) / 256, 2048);
    hipLaunchKernelGGL(muon_momentum_k, dim3((unsigned)nb), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), grad, buf, dir, (long long)n, momentum,
                       nesterov, clip);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : dcc_fail(kEHIP, std::string("dcc_muon_momentum: ") + hipGetErrorString(e));
}

DCC_API int dcc_muon_apply(float* param, const float* dir, const dcc_muon_seg* segs, int32_t count, float keep, void* stream) {
    if (count < 0 || !param || !dir || (count > 0 && !segs)) return dcc_fail(kEINVAL, "dcc_muon_apply: null pointer or negative count");
    if ((reinterpret_cast<uintptr_t>(param) | reinterpret_cast<uintptr_t>(dir)) & 15) return dcc_fail(kEINVAL, "dcc_muon_apply: arrays must be 16-byte aligned");
    for (int i = 0; i < count; ++i)
        if (segs[i].offset < 0 || segs[i].offset % 4 || segs[i].numel < 0 || segs[i].numel > (1ll << 40))
            return dcc_fail(kEINVAL, "dcc_muon_apply: a range must start at a multiple of 4 and hold 0..2^40 elements");
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
        if (first > 2147483647) return dcc_fail(kEINVAL, "dcc_muon_apply: more than 2^43 elements in one list");
        if (s.count) hipLaunchKernelGGL(muon_apply_k, dim3((unsigned)first), dim3(256), 0, reinterpret_cast<hipStream_t>(stream), param, dir, s);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : dcc_fail(kEHIP, std::string("dcc_muon_apply: ") + hipGetErrorString(e));
}

}  // extern "C"
