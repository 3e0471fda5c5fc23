// dcc_ortho.hip -- orthogonalised updates by Newton-Schulz products (include/dcc_ortho.h).
//
// Two orders of the same polynomial, chosen by shape (m <= n):
//  * m x m side (m <= 512, or n >= 5 m): A = X X^T once, then with p(A) = a I + b A + c A^2 the steps A <- p(A) A p(A), Q <- p(A) Q on
//    m x m matrices, and X <- Q X at the end: two passes over X instead of two per step.  An error of A along a direction of small
//    singular value grows by a^2 = 12 per step, so this side runs in float64 (fp64 MFMA): measured against float64 throughout, five steps
//    of 256 x 2704 are 4e-7 off, where float32 steps are 5e-6 off (and float32 on this side 1e-4).  A group holds at most five steps.
//    All its matrices are polynomials of one symmetric matrix: only lower tiles are computed, and mirrored.
//  * step by step (large and nearly square, where the float64 products would take longer): A = X X^T, B = a I + b A + c A^2, X <- B X.
// Products over X are C = A B^T to 32 bits.  fp32 MFMA has 1/16 of the bf16 rate, so the operands are split into three bf16 parts
// (x = hi + mid + lo exactly: 8 + 8 + 8 significant bits) while they are staged, and six bf16 products (hh, hm, mh, hl, lh, mm) are
// accumulated in float32; what is dropped is below 2^-23 of a product.
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
constexpr int kNormBlocks = 64;         // partial sums of a matrix's norm, at most
constexpr int kBK = 32;                 // depth of one staged slice

typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef unsigned int u4 __attribute__((ext_vector_type(4)));

struct Prod {                           // out = alpha * A B^T + beta * E + diag * I
    const void *a, *b;
    const float* e;
    void* out;
    const double* norm;                 // operands marked raw are divided by sqrt(sum of these) + eps
    long long lda, ldb, ldo;
    int rows, cols, K;
    int dta, dtb, dto;                  // 0 f32, 1 bf16, 2 f16
    int amode, bmode;                   // 0: (i, k) at i * ld + k;  1: at k * ld + i
    int rawa, rawb, nnorm;
    int sym, tcols;
    float alpha, beta, diag;
    int first;                          // first block of this product
};
struct Batch { Prod p[kMaxProds]; int n; float eps; };

struct NormMat { const void* x; double* out; long long n; int blocks, first; };
struct NormBatch { NormMat m[kMaxProds * 2]; int n, dtype; };

__device__ __forceinline__ float load1(const void* p, long long i, int dt) {
    if (dt == 0) return reinterpret_cast<const float*>(p)[i];
    if (dt == 1) return __uint_as_float((unsigned)reinterpret_cast<const unsigned short*>(p)[i] << 16);
    return __half2float(reinterpret_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store1(void* p, long long i, int dt, float v) {
    if (dt == 0) reinterpret_cast<float*>(p)[i] = v;
    else if (dt == 1) reinterpret_cast<__hip_bfloat16*>(p)[i] = __float2bfloat16(v);
    else reinterpret_cast<__half*>(p)[i] = __float2half(v);
}

// sum of squares in float64, kNormBlocks fixed ranges per matrix
__global__ __launch_bounds__(256) void ortho_norm_k(const NormBatch nb) {
    __shared__ double red[4];
    int i = 0;
    while (i + 1 < nb.n && (int)blockIdx.x >= nb.m[i + 1].first) ++i;
    const NormMat& m = nb.m[i];
    const int blk = blockIdx.x - m.first;
    const long long per = ((m.n + m.blocks - 1) / m.blocks + 3) & ~3ll;
    const long long lo = blk * per, hi = lo + per < m.n ? lo + per : m.n;
    double s0 = 0., s1 = 0., s2 = 0., s3 = 0.;
    const long long hi4 = lo + ((hi > lo ? hi - lo : 0) & ~3ll);
    const bool v4 = nb.dtype == 0 && (reinterpret_cast<uintptr_t>(m.x) & 15) == 0;
    for (long long j = lo + 4 * threadIdx.x; j < hi4; j += 1024) {
        float4 x;
        if (v4) x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(m.x) + j);
        else x = make_float4(load1(m.x, j, nb.dtype), load1(m.x, j + 1, nb.dtype), load1(m.x, j + 2, nb.dtype), load1(m.x, j + 3, nb.dtype));
        s0 += (double)x.x * x.x; s1 += (double)x.y * x.y; s2 += (double)x.z * x.z; s3 += (double)x.w * x.w;
    }
    if (hi4 + threadIdx.x < hi) { const double x = load1(m.x, hi4 + threadIdx.x, nb.dtype); s0 += x * x; }
    double s = (s0 + s1) + (s2 + s3);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) m.out[blk] = (red[0] + red[1]) + (red[2] + red[3]);
}

__device__ __forceinline__ float inverse_norm(const Prod& p, float eps) {
    double s = 0.;
    for (int i = 0; i < p.nnorm; ++i) s += p.norm[i];
    return (float)(1.0 / (sqrt(s) + (double)eps));
}

// eight values of row i at depth k (zero outside); consecutive in memory for mode 0
__device__ __forceinline__ void fetch8(float (&x)[8], const void* base, int dt, long long ld, int mode, int i, int rows, int k, int kend, bool vec) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = 0.f;
    if (i >= rows) return;
    if (mode == 0) {
        const long long at = (long long)i * ld + k;
        if (vec && k + 7 < kend) {
            if (dt == 0) {
                const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + at);
                const float4 a = p[0], b = p[1];
                x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
            } else {
                const u4 a = *reinterpret_cast<const u4*>(reinterpret_cast<const unsigned short*>(base) + at);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (dt == 1) {
                        x[2 * j] = __uint_as_float(a[j] << 16);
                        x[2 * j + 1] = __uint_as_float(a[j] & 0xffff0000u);
                    } else {
                        const unsigned w = a[j];
                        const __half2 h = *reinterpret_cast<const __half2*>(&w);
                        x[2 * j] = __low2float(h);
                        x[2 * j + 1] = __high2float(h);
                    }
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (k + j < kend) x[j] = load1(base, at + j, dt);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (k + j < kend) x[j] = load1(base, (long long)(k + j) * ld + i, dt);
    }
}

// x * s split into three bf16 parts by truncation: exact, every part has at most 8 significant bits
__device__ __forceinline__ void split8(const float (&x)[8], float s, u4& hi, u4& mid, u4& lo) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        unsigned h[2], m[2], l[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float v = x[2 * j + e] * s;
            h[e] = __float_as_uint(v) & 0xffff0000u;
            const float r = v - __uint_as_float(h[e]);
            m[e] = __float_as_uint(r) & 0xffff0000u;
            l[e] = __float_as_uint(r - __uint_as_float(m[e]));
        }
        hi[j] = (h[0] >> 16) | h[1];
        mid[j] = (m[0] >> 16) | m[1];
        lo[j] = (l[0] >> 16) | (l[1] & 0xffff0000u);
    }
}

// 16-byte piece kg of row i in a staged plane: the pieces of a row are turned by i / 4, so that the 16 rows that one MFMA operand
// reads at one kg lie in 16 different groups of banks
__device__ __forceinline__ int piece(int i, int kg) { return i * 4 + (kg ^ ((i >> 2) & 3)); }

// tile (ti, tj), tj <= ti, of the lower triangle counted row by row
__device__ __forceinline__ void lower_tile(int blk, int& ti, int& tj) {
    ti = (int)((sqrtf(8.f * blk + 1.f) - 1.f) * 0.5f);
    while (ti * (ti + 1) / 2 > blk) --ti;
    while ((ti + 1) * (ti + 2) / 2 <= blk) ++ti;
    tj = blk - ti * (ti + 1) / 2;
}

// One workgroup: one TM x TM tile of one product (4 waves as 2 x 2).
template <int TM>
__global__ __launch_bounds__(256) void ortho_prod_k(const Batch bt) {
    constexpr int TW = TM / 2, NT = TW / 16, PASS = TM / 64;
    __shared__ u4 sh[2 * 3 * TM * 4];
    int pi = 0;
    while (pi + 1 < bt.n && (int)blockIdx.x >= bt.p[pi + 1].first) ++pi;
    const Prod& p = bt.p[pi];
    int blk = blockIdx.x - p.first;
    int ti, tj;
    if (p.sym) {
        lower_tile(blk, ti, tj);
    } else {
        ti = blk / p.tcols;
        tj = blk - ti * p.tcols;
    }
    const int i0 = ti * TM, j0 = tj * TM;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 15, kg = lane >> 4, g4 = kg << 2;
    const int wi = (wave >> 1) * TW, wj = (wave & 1) * TW;
    const float inv = (p.rawa | p.rawb) ? inverse_norm(p, bt.eps) : 1.f;
    const float sa = p.rawa ? inv : 1.f, sb = p.rawb ? inv : 1.f;
    const bool va = p.amode == 0 && (reinterpret_cast<uintptr_t>(p.a) & 15) == 0 && p.lda % 8 == 0;
    const bool vb = p.bmode == 0 && (reinterpret_cast<uintptr_t>(p.b) & 15) == 0 && p.ldb % 8 == 0;
    const int ra = p.amode == 0 ? tid >> 2 : tid & 63, ka = p.amode == 0 ? tid & 3 : tid >> 6;
    const int rb = p.bmode == 0 ? tid >> 2 : tid & 63, kb = p.bmode == 0 ? tid & 3 : tid >> 6;
    const int kend = p.K;

    f4 acc[NT][NT];
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int y = 0; y < NT; ++y) acc[x][y] = f4{0.f, 0.f, 0.f, 0.f};
    float xa[PASS][8], xb[PASS][8];
#pragma unroll
    for (int q = 0; q < PASS; ++q) {
        fetch8(xa[q], p.a, p.dta, p.lda, p.amode, i0 + q * 64 + ra, p.rows, ka * 8, kend, va);
        fetch8(xb[q], p.b, p.dtb, p.ldb, p.bmode, j0 + q * 64 + rb, p.cols, kb * 8, kend, vb);
    }
    for (int k = 0; k < kend; k += kBK) {
        __syncthreads();
#pragma unroll
        for (int q = 0; q < PASS; ++q) {
            u4 h, m, l;
            split8(xa[q], sa, h, m, l);
            const int pa = piece(q * 64 + ra, ka), pb = piece(q * 64 + rb, kb);
            sh[pa] = h; sh[TM * 4 + pa] = m; sh[2 * TM * 4 + pa] = l;
            split8(xb[q], sb, h, m, l);
            sh[3 * TM * 4 + pb] = h; sh[4 * TM * 4 + pb] = m; sh[5 * TM * 4 + pb] = l;
        }
        __syncthreads();
        if (k + kBK < kend) {
#pragma unroll
            for (int q = 0; q < PASS; ++q) {
                fetch8(xa[q], p.a, p.dta, p.lda, p.amode, i0 + q * 64 + ra, p.rows, k + kBK + ka * 8, kend, va);
                fetch8(xb[q], p.b, p.dtb, p.ldb, p.bmode, j0 + q * 64 + rb, p.cols, k + kBK + kb * 8, kend, vb);
            }
        }
        bf8 fb[NT][3];
#pragma unroll
        for (int y = 0; y < NT; ++y) {
            const int pb = piece(wj + 16 * y + li, kg);
#pragma unroll
            for (int s = 0; s < 3; ++s) fb[y][s] = __builtin_bit_cast(bf8, sh[(3 + s) * TM * 4 + pb]);
        }
#pragma unroll
        for (int x = 0; x < NT; ++x) {
            const int pa = piece(wi + 16 * x + li, kg);
            bf8 fa[3];
#pragma unroll
            for (int s = 0; s < 3; ++s) fa[s] = __builtin_bit_cast(bf8, sh[s * TM * 4 + pa]);
#pragma unroll
            for (int y = 0; y < NT; ++y) {
                acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[0], fb[y][2], acc[x][y], 0, 0, 0);
                acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[2], fb[y][0], acc[x][y], 0, 0, 0);
                acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[1], fb[y][1], acc[x][y], 0, 0, 0);
                acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[0], fb[y][1], acc[x][y], 0, 0, 0);
                acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[1], fb[y][0], acc[x][y], 0, 0, 0);
                acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[0], fb[y][0], acc[x][y], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int y = 0; y < NT; ++y)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = i0 + wi + 16 * x + g4 + r, j = j0 + wj + 16 * y + li;
                if (i >= p.rows || j >= p.cols) continue;
                if (p.sym && j > i) continue;               // its mirror is written below
                float v = p.alpha * acc[x][y][r];
                if (p.e) v += p.beta * p.e[(long long)i * p.cols + j];
                if (i == j) v += p.diag;
                store1(p.out, (long long)i * p.ldo + j, p.dto, v);
                if (p.sym && i != j) store1(p.out, (long long)j * p.ldo + i, p.dto, v);
            }
}

// ---- the m x m side in float64 -------------------------------------------------------------------------------------------------
struct DProd {                          // out = alpha * A B^T + beta * E + diag * I, symmetric, m x m
    const void *a, *b;
    const double* e;
    void* out;
    double* part;                       // slices > 1: partial sums [slices][m * m]
    const double* norm;                 // raw operands: the result is divided by (sqrt(sum of these) + eps)^2
    long long lda, ldb;
    int m, K, dt, mode, nnorm, slices, kper, out32, first;      // dt: 0 f32, 1 bf16, 2 f16, 3 f64; mode as above (f64: 0)
    double alpha, beta, diag;
};
struct DBatch { DProd p[kMaxProds]; int n; float eps; };
typedef double d4 __attribute__((ext_vector_type(4)));

// four values of row i at depth k, zero outside
__device__ __forceinline__ d4 fetch4(const void* base, int dt, long long ld, int mode, int i, int rows, int k, int kend, bool vec) {
    d4 x = {0., 0., 0., 0.};
    if (i >= rows) return x;
    const long long at = mode == 0 ? (long long)i * ld + k : (long long)k * ld + i, step = mode == 0 ? 1 : ld;
    if (dt == 3) {
        const double* p = reinterpret_cast<const double*>(base) + at;
        if (vec && k + 3 < kend) {
            const double2 u = reinterpret_cast<const double2*>(p)[0], w = reinterpret_cast<const double2*>(p)[1];
            x[0] = u.x; x[1] = u.y; x[2] = w.x; x[3] = w.y;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (k + j < kend) x[j] = p[j];
        }
    } else if (vec && dt == 0 && k + 3 < kend) {
        const float4 u = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + at);
        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (k + j < kend) x[j] = load1(base, at + j * step, dt);
    }
    return x;
}

__device__ __forceinline__ void dstore(const DProd& p, const DBatch& bt, double v, int i, int j) {
    if (p.nnorm > 0) {
        double s = 0.;
        for (int q = 0; q < p.nnorm; ++q) s += p.norm[q];
        s = sqrt(s) + (double)bt.eps;
        v /= s * s;
    }
    v *= p.alpha;
    const long long ij = (long long)i * p.m + j, ji = (long long)j * p.m + i;
    if (p.e) v += p.beta * p.e[ij];
    if (i == j) v += p.diag;
    if (p.out32) {
        reinterpret_cast<float*>(p.out)[ij] = (float)v;
        reinterpret_cast<float*>(p.out)[ji] = (float)v;
    } else {
        reinterpret_cast<double*>(p.out)[ij] = v;
        reinterpret_cast<double*>(p.out)[ji] = v;
    }
}

// v_mfma_f64_16x16x4_f64: A[i = lane%16][k = lane/16], B[k = lane/16][j = lane%16], D[i = 4 r + lane/16][j = lane%16].  Operands come from
// memory as they are (a lane's four consecutive k make four steps).  WIDE: a 64 x 64 tile by 2 x 2 waves of 32 x 32 (long depths, where
// reading the operands counts); else a 16 x 16 tile whose depth the four waves share (short ones, where latency does).
template <bool WIDE>
__global__ __launch_bounds__(256) void ortho_dprod_k(const DBatch bt) {
    constexpr int T = WIDE ? 2 : 1, TM = WIDE ? 64 : 16;
    __shared__ double sh[WIDE ? 1 : 4 * 256];
    int pi = 0;
    while (pi + 1 < bt.n && (int)blockIdx.x >= bt.p[pi + 1].first) ++pi;
    const DProd& p = bt.p[pi];
    int blk = blockIdx.x - p.first, ti, tj;
    const int slice = blk % p.slices;
    lower_tile(blk / p.slices, ti, tj);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, g = lane >> 4;
    const int i0 = ti * TM + (WIDE ? (wave >> 1) * 32 : 0), j0 = tj * TM + (WIDE ? (wave & 1) * 32 : 0);
    int kbeg = slice * p.kper, kend = kbeg + p.kper < p.K ? kbeg + p.kper : p.K;
    if (!WIDE) {
        const int quarter = ((kend - kbeg + 3) / 4 + 15) & ~15;
        kbeg += wave * quarter;
        kend = kbeg + quarter < kend ? kbeg + quarter : kend;
    }
    const bool va = p.mode == 0 && (reinterpret_cast<uintptr_t>(p.a) & 15) == 0 && p.lda % 4 == 0;
    const bool vb = p.mode == 0 && (reinterpret_cast<uintptr_t>(p.b) & 15) == 0 && p.ldb % 4 == 0;
    d4 acc[T][T];
#pragma unroll
    for (int x = 0; x < T; ++x)
#pragma unroll
        for (int y = 0; y < T; ++y) acc[x][y] = d4{0., 0., 0., 0.};
    for (int k = kbeg; k < kend; k += 16) {
        d4 a[T], b[T];
#pragma unroll
        for (int x = 0; x < T; ++x) {
            a[x] = fetch4(p.a, p.dt, p.lda, p.mode, i0 + 16 * x + li, p.m, k + 4 * g, kend, va);
            b[x] = fetch4(p.b, p.dt, p.ldb, p.mode, j0 + 16 * x + li, p.m, k + 4 * g, kend, vb);
        }
#pragma unroll
        for (int x = 0; x < T; ++x)
#pragma unroll
            for (int y = 0; y < T; ++y)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[x][y] = __builtin_amdgcn_mfma_f64_16x16x4f64(a[x][r], b[y][r], acc[x][y], 0, 0, 0);
    }
    if (!WIDE) {
#pragma unroll
        for (int r = 0; r < 4; ++r) sh[wave * 256 + (4 * r + g) * 16 + li] = acc[0][0][r];
        __syncthreads();
        const int i = i0 + (threadIdx.x >> 4), j = j0 + (threadIdx.x & 15);
        const double v = (sh[threadIdx.x] + sh[256 + threadIdx.x]) + (sh[512 + threadIdx.x] + sh[768 + threadIdx.x]);
        if (i < p.m && j <= i) {
            if (p.slices > 1) p.part[((long long)slice * p.m + i) * p.m + j] = v;
            else dstore(p, bt, v, i, j);
        }
        return;
    }
#pragma unroll
    for (int x = 0; x < T; ++x)
#pragma unroll
        for (int y = 0; y < T; ++y)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = i0 + 16 * x + 4 * r + g, j = j0 + 16 * y + li;
                if (i >= p.m || j > i) continue;
                if (p.slices > 1) p.part[((long long)slice * p.m + i) * p.m + j] = acc[x][y][r];
                else dstore(p, bt, acc[x][y][r], i, j);
            }
}

__global__ __launch_bounds__(256) void ortho_djoin_k(const DBatch bt) {
    const DProd& p = bt.p[blockIdx.y];
    if (p.slices <= 1) return;
    const long long n = (long long)p.m * p.m;
    for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < n; at += (long long)gridDim.x * 256) {
        const int i = (int)(at / p.m), j = (int)(at - (long long)i * p.m);
        if (j > i) continue;
        double s = 0.;
        for (int q = 0; q < p.slices; ++q) s += p.part[q * n + at];
        dstore(p, bt, s, i, j);
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
int64_t up(int64_t x) { return (x + kAlign - 1) / kAlign * kAlign; }
constexpr int kChip = 256;              // compute units

struct Shape { int64_t m, n; bool tall; };
Shape shape_of(const dcc_ortho_mat& t) { return Shape{std::min(t.M, t.N), std::max(t.M, t.N), t.M > t.N}; }

// the m x m side in float64: always for small m (its products are latency there), else where n is long enough to pay for their rate
bool on_square_side(const Shape& s) { return s.m <= 512 || s.n >= 5 * s.m; }
constexpr int kGroup = 5;               // steps on that side before X X^T is formed anew

// tiles of 64 for long depths of X X^T, and then as many depth slices as fill the chip twice, none shorter than 256
bool wide_gram(const Shape& s) { return s.n >= 4096; }
int gram_slices(const Shape& s) {
    const int64_t nt = (s.m + 63) / 64, tiles = nt * (nt + 1) / 2;
    if (!wide_gram(s)) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(2 * kChip / tiles, s.n / 256), 128));
}

// where a matrix's intermediate results lie in the workspace
struct Place { int64_t norm, A, B, W, Q0, Q1, Q, X0, X1, part, end; };
Place place_of(const Shape& s, int steps, int64_t at) {
    Place p = {};
    auto take = [&](int64_t bytes) { const int64_t o = at; at += up(bytes); return o; };
    const int64_t mm = s.m * s.m, mn = 4 * s.m * s.n;
    p.norm = take(8 * kNormBlocks);
    if (on_square_side(s)) {
        p.A = take(8 * mm); p.B = take(8 * mm); p.W = take(8 * mm); p.Q0 = take(8 * mm); p.Q1 = take(8 * mm); p.Q = take(4 * mm);
        if (gram_slices(s) > 1) p.part = take(8 * mm * gram_slices(s));
        if (steps > kGroup) p.X0 = take(mn);
        if (steps > 2 * kGroup) p.X1 = take(mn);
    } else {
        p.A = take(4 * mm); p.B = take(4 * mm);
        if (steps > 1) p.X0 = take(mn);
        if (steps > 2) p.X1 = take(mn);
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
        if (mats[i].M > (1 << 30) || mats[i].N > (1 << 30)) return "more than 2^30 rows or columns";
        if (shape_of(mats[i]).m > 32768) return "both sides over 32768";
    }
    return nullptr;
}

// a round: products (of all matrices) that do not depend on each other
struct Round { std::vector<Prod> x; std::vector<DProd> d, dwide; };

void launch_prods(const std::vector<Prod>& all, float eps, hipStream_t st) {
    for (size_t from = 0; from < all.size(); from += kMaxProds) {
        Batch bt;
        bt.n = (int)std::min<size_t>(kMaxProds, all.size() - from);
        bt.eps = eps;
        int64_t big = 0;
        for (int i = 0; i < bt.n; ++i) {
            const Prod& p = all[from + i];
            const int64_t tr = (p.rows + 127) / 128, tc = (p.cols + 127) / 128;
            big += p.sym ? tr * (tr + 1) / 2 : tr * tc;
        }
        // tiles of 128 where they fill the chip, of 64 (more compute units share the depth's latency) where they do not
        const int tm = big >= kChip ? 128 : 64;
        int64_t first = 0;
        for (int i = 0; i < bt.n; ++i) {
            Prod& p = bt.p[i] = all[from + i];
            const int64_t tr = (p.rows + tm - 1) / tm, tc = (p.cols + tm - 1) / tm;
            p.tcols = (int)tc;
            p.first = (int)first;
            first += p.sym ? tr * (tr + 1) / 2 : tr * tc;
        }
        if (tm == 128) hipLaunchKernelGGL(ortho_prod_k<128>, dim3((unsigned)first), dim3(256), 0, st, bt);
        else hipLaunchKernelGGL(ortho_prod_k<64>, dim3((unsigned)first), dim3(256), 0, st, bt);
    }
}

template <bool WIDE>
void launch_dprods(const std::vector<DProd>& all, float eps, hipStream_t st) {
    constexpr int tm = WIDE ? 64 : 16;
    for (size_t from = 0; from < all.size(); from += kMaxProds) {
        DBatch bt;
        bt.n = (int)std::min<size_t>(kMaxProds, all.size() - from);
        bt.eps = eps;
        int64_t first = 0, longest = 0;
        for (int i = 0; i < bt.n; ++i) {
            DProd& p = bt.p[i] = all[from + i];
            const int64_t t = (p.m + tm - 1) / tm;
            p.first = (int)first;
            first += t * (t + 1) / 2 * p.slices;
            if (p.slices > 1) longest = std::max<int64_t>(longest, (int64_t)p.m * p.m);
        }
        hipLaunchKernelGGL(ortho_dprod_k<WIDE>, dim3((unsigned)first), dim3(256), 0, st, bt);
        if (longest) hipLaunchKernelGGL(ortho_djoin_k, dim3((unsigned)std::min<int64_t>((longest + 255) / 256, 1024), bt.n), dim3(256), 0, st, bt);
    }
}

}  // namespace

extern "C" {

DCC_API int64_t dcc_ortho_workspace_bytes(const dcc_ortho_mat* mats, int32_t count, int32_t dtype, int32_t steps) {
    if (list_error(mats, count, dtype, steps)) return 0;
    int64_t at = 0;
    for (int i = 0; i < count; ++i)
        if (mats[i].M > 0 && mats[i].N > 0) at = place_of(shape_of(mats[i]), steps, at).end;
    return at;
}

DCC_API int dcc_orthogonalize(const dcc_ortho_mat* mats, int32_t count, int32_t dtype, int32_t steps, float a, float b, float c,
                              float eps, void* workspace, void* stream) try {
    if (const char* e = list_error(mats, count, dtype, steps)) return dcc_fail(kEINVAL, std::string("dcc_orthogonalize: ") + e);
    if (!(eps >= 0.f)) return dcc_fail(kEINVAL, "dcc_orthogonalize: eps must not be negative");
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    std::vector<int> live;
    for (int i = 0; i < count; ++i) {
        if (mats[i].M == 0 || mats[i].N == 0) continue;
        if (!mats[i].in || !mats[i].out) return dcc_fail(kEINVAL, "dcc_orthogonalize: null matrix");
        live.push_back(i);
    }
    if (live.empty()) return 0;
    const int64_t esize = dtype == DCC_ORTHO_F32 ? 4 : 2;
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
    std::vector<Place> place(live.size());
    std::vector<int> nnorm(live.size());
    int64_t at = 0;
    NormBatch nb;
    nb.n = 0;
    nb.dtype = dtype;
    int first = 0;
    for (size_t i = 0; i < live.size(); ++i) {
        const dcc_ortho_mat& t = mats[live[i]];
        place[i] = place_of(shape_of(t), steps, at);
        at = place[i].end;
        nnorm[i] = (int)std::min<int64_t>(kNormBlocks, (t.M * t.N + 4095) / 4096);
        NormMat& m = nb.m[nb.n++];
        m.x = t.in; m.out = reinterpret_cast<double*>(ws + place[i].norm); m.n = t.M * t.N; m.blocks = nnorm[i]; m.first = first;
        first += nnorm[i];
        if (nb.n == kMaxProds * 2 || i + 1 == live.size()) {
            hipLaunchKernelGGL(ortho_norm_k, dim3(first), dim3(256), 0, st, nb);
            nb.n = 0;
            first = 0;
        }
    }
    std::vector<Round> rounds;
    auto round = [&](size_t r) -> Round& {
        if (rounds.size() <= r) rounds.resize(r + 1);
        return rounds[r];
    };
    for (size_t i = 0; i < live.size(); ++i) {
        const dcc_ortho_mat& t = mats[live[i]];
        const Shape s = shape_of(t);
        const Place& pl = place[i];
        const int m = (int)s.m, n = (int)s.n;
        const double* norm = reinterpret_cast<const double*>(ws + pl.norm);
        const void* X = t.in;
        bool raw = true, flip = false;
        size_t r = 0;
        int left = steps;
        auto apply = [&](const float* Q) {      // X <- Q X
            Prod p = {};
            const bool last = left == 0;
            void* out = last ? t.out : static_cast<void*>(ws + (flip ? pl.X1 : pl.X0));
            flip = !flip;
            p.alpha = 1.f; p.norm = norm; p.nnorm = nnorm[i];
            if (s.tall) {       // stored as X^T [n, m]: its rows times the symmetric Q
                p.a = X; p.dta = raw ? dtype : 0; p.rawa = raw; p.lda = m; p.b = Q; p.ldb = m;
                p.rows = n; p.cols = m; p.ldo = m;
            } else {
                p.a = Q; p.lda = m; p.b = X; p.dtb = raw ? dtype : 0; p.rawb = raw; p.ldb = n; p.bmode = 1;
                p.rows = m; p.cols = n; p.ldo = n;
            }
            p.K = m; p.out = out; p.dto = last ? dtype : 0;
            round(r++).x.push_back(p);
            X = out;
            raw = false;
        };
        if (on_square_side(s)) {
            double *A = reinterpret_cast<double*>(ws + pl.A), *B = reinterpret_cast<double*>(ws + pl.B), *W = reinterpret_cast<double*>(ws + pl.W);
            double* Qs[2] = {reinterpret_cast<double*>(ws + pl.Q0), reinterpret_cast<double*>(ws + pl.Q1)};
            float* Qf = reinterpret_cast<float*>(ws + pl.Q);
            auto square = [&](const double* x, const double* y, void* out) {
                DProd p = {};
                p.a = x; p.b = y; p.out = out; p.lda = p.ldb = m; p.m = p.K = m; p.dt = 3; p.slices = 1; p.kper = m; p.alpha = 1.;
                return p;
            };
            while (left > 0) {
                const int groups = (left + kGroup - 1) / kGroup, len = (left + groups - 1) / groups;
                left -= len;
                DProd g = {};           // A = X X^T
                g.a = g.b = X; g.dt = raw ? dtype : 0; g.lda = g.ldb = t.N; g.mode = s.tall; g.m = m; g.K = n; g.out = A; g.alpha = 1.;
                if (raw) { g.norm = norm; g.nnorm = nnorm[i]; }
                g.part = reinterpret_cast<double*>(ws + pl.part);
                g.kper = (n + gram_slices(s) - 1) / gram_slices(s);
                g.kper = (g.kper + 15) / 16 * 16;
                g.slices = (n + g.kper - 1) / g.kper;
                (wide_gram(s) ? round(r).dwide : round(r).d).push_back(g);
                ++r;
                int cur = -1;           // Qs[cur] holds Q
                for (int k = 0; k < len; ++k) {
                    const bool end = k + 1 == len;
                    DProd p = square(A, A, k > 0 ? B : end ? static_cast<void*>(Qf) : Qs[0]);       // p(A)
                    p.alpha = c; p.e = A; p.beta = b; p.diag = a; p.out32 = k == 0 && end;
                    round(r++).d.push_back(p);
                    const double* Pk = k > 0 ? B : Qs[0];
                    if (k > 0) {                            // Q <- p(A) Q
                        DProd q = square(Pk, Qs[cur], end ? static_cast<void*>(Qf) : Qs[cur ^ 1]);
                        q.out32 = end;
                        round(r).d.push_back(q);
                        cur ^= 1;
                        if (end) ++r;
                    } else {
                        cur = 0;
                    }
                    if (!end) {                             // A <- p(A) A p(A)
                        round(r++).d.push_back(square(Pk, A, W));
                        round(r++).d.push_back(square(W, Pk, A));
                    }
                }
                apply(Qf);
            }
        } else {
            float *A = reinterpret_cast<float*>(ws + pl.A), *B = reinterpret_cast<float*>(ws + pl.B);
            while (left > 0) {
                --left;
                Prod g = {};            // A = X X^T
                g.a = g.b = X; g.dta = g.dtb = raw ? dtype : 0; g.rawa = g.rawb = raw; g.lda = g.ldb = t.N; g.amode = g.bmode = s.tall;
                g.out = A; g.ldo = m; g.rows = g.cols = m; g.K = n; g.sym = 1; g.alpha = 1.f; g.norm = norm; g.nnorm = nnorm[i];
                round(r++).x.push_back(g);
                Prod p = {};            // B = a I + b A + c A^2
                p.a = p.b = A; p.lda = p.ldb = p.ldo = m; p.out = B; p.rows = p.cols = p.K = m; p.sym = 1; p.alpha = c; p.e = A; p.beta = b; p.diag = a;
                round(r++).x.push_back(p);
                apply(B);
            }
        }
    }
    for (const Round& q : rounds) {
        launch_dprods<true>(q.dwide, eps, st);
        launch_dprods<false>(q.d, eps, st);
        launch_prods(q.x, eps, st);
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
