// dcc_delta.hip -- the gated delta rule: sequence form, its gradient, one token (include/dcc_delta.h).
//
// Sequence form over chunks of C = 16 tokens.  With gam_i the decay from the chunk's start to token i, D_ij the decay from token j to
// token i (0 across a restart) and N_ij = D_ij k_i.k_j for j < i, the chunk's updates solve a unit lower triangular system:
//     U = (I + diag(beta) N)^-1 diag(beta) (V - diag(gam) K S0)
//     O = scale (diag(gam) Q S0 + (Q K^T . D) U),        S_C = gam_C S0 + K^T diag(D_C.) U
// C = 16 is one 16x16 fp32 MFMA tile: the state products (3 * 2 * DK * DV flop per token) are then 80 % of the work, where C = 64 would
// double the total.  The inverse comes from forward substitution (a product form of it loses all digits when neighbouring keys are
// nearly equal, which is what slowly moving scenes give).
//
// Matrix operands: v_mfma_f32_16x16x4_f32 wants A[i = lane%16][k = lane/16], B[k = lane/16][j = lane%16] and returns
// D[i = 4*(lane/16) + r][j = lane%16].  The sum over k may run in any order, so its step (t, r) takes k = 16 t + 4*(lane/16) + r: a
// result is then the B operand of the next product as it stands (states, right-hand sides and updates never leave their registers),
// and A operands are one float4 per lane and 16 columns.
// All arithmetic is fp32 whatever the type of q, k, v: states, gates and solves stay exact to 32 bits.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "dcc_delta.h"
#include "dcc_internal.h"

#pragma clang fp contract(fast)

namespace {

constexpr int kEINVAL = -1, kEHIP = -2;
constexpr int kC = 16;                  // tokens per chunk
constexpr int kMaxWaves = 4;
constexpr float kDead = -103.98f;       // exp() below this is 0 in float32: a restart

typedef float f4 __attribute__((ext_vector_type(4)));

template <typename E> struct Elem;
template <> struct Elem<float> {
    typedef float4 vec;
    static __device__ __forceinline__ float get(float x) { return x; }
    static __device__ __forceinline__ float put(float x) { return x; }
    static __device__ __forceinline__ float4 get4(const float4& x) { return x; }
};
template <> struct Elem<__hip_bfloat16> {
    typedef uint2 vec;
    static __device__ __forceinline__ float get(__hip_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ __hip_bfloat16 put(float x) { return __float2bfloat16(x); }
    static __device__ __forceinline__ float4 get4(const uint2& x) {
        return make_float4(__uint_as_float(x.x << 16), __uint_as_float(x.x & 0xffff0000u), __uint_as_float(x.y << 16), __uint_as_float(x.y & 0xffff0000u));
    }
};
template <> struct Elem<__half> {
    typedef uint2 vec;
    static __device__ __forceinline__ float get(__half x) { return __half2float(x); }
    static __device__ __forceinline__ __half put(float x) { return __float2half(x); }
    static __device__ __forceinline__ float4 get4(const uint2& x) {
        const __half2 a = *reinterpret_cast<const __half2*>(&x.x), b = *reinterpret_cast<const __half2*>(&x.y);
        return make_float4(__low2float(a), __high2float(a), __low2float(b), __high2float(b));
    }
};

struct Seq {        // dcc_delta_seq / dcc_delta_grad as the kernels read them
    long long T, B;
    int HK, H, DK, DV, rep, nchunk;
    float scale;
    const void *q, *k, *v, *dout;
    const float *g, *beta, *masks, *state0, *dstate1, *state1;
    long long sq[3], sk[3], sv[3], sg[3], sb[3], sm[2], sdo[3];
    void* o;
    float *state_out, *ckpt, *dq32, *dk32;
    void *dq, *dk, *dv;
    float *dg, *dbeta, *dstate0;
    int vec;        // rows of q, k (and dout, v) may be read four elements at a time
};

// lanes of one wave exchange values through LDS between the two sides of this (a wave's LDS operations complete in order)
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ f4 mfma(float a, float b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4 zero4() { f4 z = {0.f, 0.f, 0.f, 0.f}; return z; }
__device__ __forceinline__ f4 lds4(const float* p) { return *reinterpret_cast<const f4*>(p); }

// sum over the 16 lanes that share lane/16
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// `rows` rows of `dim` elements (row i: base + i * stride; rows >= valid and columns >= dim are zero) into LDS rows of `pitch` floats
template <typename E>
__device__ __forceinline__ void load_rows(float* dst, int pitch, const void* base, long long stride, int rows, int valid, int dim, int dimp,
                                          int vec, float mul) {
    const E* src = reinterpret_cast<const E*>(base);
    const int c4 = dimp >> 2;
    for (int e = threadIdx.x; e < rows * c4; e += blockDim.x) {
        const int i = e / c4, c = (e - i * c4) << 2;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < valid) {
            const E* p = src + (long long)i * stride + c;
            if (vec && c + 3 < dim) {
                x = Elem<E>::get4(*reinterpret_cast<const typename Elem<E>::vec*>(p));
            } else {
                if (c < dim) x.x = Elem<E>::get(p[0]);
                if (c + 1 < dim) x.y = Elem<E>::get(p[1]);
                if (c + 2 < dim) x.z = Elem<E>::get(p[2]);
                if (c + 3 < dim) x.w = Elem<E>::get(p[3]);
            }
        }
        f4 y = {x.x * mul, x.y * mul, x.z * mul, x.w * mul};
        *reinterpret_cast<f4*>(dst + i * pitch + c) = y;
    }
}

constexpr int kSP = 20;                         // pitch of the 16x16 tiles in LDS (rows 16-byte aligned)
struct ChunkVec { float beta[kC], gam[kC], toend[kC], seg[kC], gend; float pad[3]; };     // per chunk: gates as the products use them

// Decays of one chunk, by one wave: lane l works on token l % 16 (the four groups repeat each other).  Running sums in double: the
// difference of two float sums would carry the error of the larger one into every D_ij.  Returns this lane's running sum and segment.
__device__ __forceinline__ void chunk_gates(const Seq& p, long long b, int h, long long t0, int lane, double& run, int& seg, ChunkVec* cv) {
    const int i = lane & 15;
    const long long t = t0 + i;
    float g = 0.f, be = 0.f;
    int cut = 0;
    if (t < p.T) {
        g = p.g[t * p.sg[0] + b * p.sg[1] + h * p.sg[2]];
        be = p.beta[t * p.sb[0] + b * p.sb[1] + h * p.sb[2]];
        if (p.masks) cut = p.masks[t * p.sm[0] + b * p.sm[1]] == 0.f;
        if (g < kDead) cut = 1;
        if (cut) g = 0.f;
    }
    double s = (double)g;
    int c = cut;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
        const double su = __shfl_up(s, o, 16);
        const int cu = __shfl_up(c, o, 16);
        if (i >= o) { s += su; c += cu; }
    }
    run = s;
    seg = c;
    const double send = __shfl(s, 15, 16);
    const int cend = __shfl(c, 15, 16);
    if (lane < 16) {
        cv->beta[i] = be;
        cv->gam[i] = c == 0 ? expf((float)s) : 0.f;
        cv->toend[i] = c == cend ? expf((float)(send - s)) : 0.f;
        cv->seg[i] = cut ? -1.f - c : (float)c;         // sign: a restart at this token
        if (i == 15) cv->gend = c == 0 ? expf((float)s) : 0.f;
    }
}

// D_ij of this lane's four entries (row i = 4*(lane/16) + r, column j = lane % 16), 0 above the diagonal
__device__ __forceinline__ f4 chunk_decay(double run, int seg, int lane) {
    const int j = lane & 15, g4 = (lane >> 4) << 2;
    f4 d;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int i = g4 + r;
        const double si = __shfl(run, i, 16);
        const int ci = __shfl(seg, i, 16);
        d[r] = (i >= j && ci == seg) ? expf((float)(si - run)) : 0.f;
    }
    return d;
}

// (I + L)^-1 in place, L strictly lower triangular in `t` [16][kSP]; one wave, lane l solves column l % 16 by forward substitution
__device__ __forceinline__ void unit_lower_inverse(float* t, int lane) {
    const int c = lane & 15;
    float x[kC];
#pragma unroll
    for (int i = 0; i < kC; ++i) {
        float a = i == c ? 1.f : 0.f;
#pragma unroll
        for (int j = 0; j < kC; ++j)
            if (j < i) a -= t[i * kSP + j] * x[j];
        x[i] = a;
    }
    wave_sync();        // every lane has read t
    if (lane < 16) {
#pragma unroll
        for (int i = 0; i < kC; ++i) t[i * kSP + c] = x[i];
    }
}

// ---- forward -------------------------------------------------------------------------------------------------------------------
// One workgroup per (row, head) and up to kMaxWaves tiles of 16 value columns; each wave keeps its [DK, 16] slice of the state in
// registers and walks the chunks.  Blocks of BT chunks are staged in LDS: the waves first split the state-free part (K K^T, Q K^T, gates,
// inverse) of the BT chunks among them, then every wave runs the BT chunks on its own columns without a barrier.
template <typename E, int DKT, int BT>
__global__ __launch_bounds__(256) void delta_fwd_k(const Seq p) {
    constexpr int DKP = DKT * 16, KP = DKP + 4;
    extern __shared__ float sh[];
    float* Ks = sh;
    float* Qs = Ks + BT * kC * KP;
    float* Ti = Qs + BT * kC * KP;              // [BT][16][kSP] inverse
    float* Am = Ti + BT * kC * kSP;             // [BT][16][kSP] (Q K^T) . D
    ChunkVec* cvs = reinterpret_cast<ChunkVec*>(Am + BT * kC * kSP);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nw = blockDim.x >> 6;
    const int li = lane & 15, g4 = (lane >> 4) << 2;
    const long long bh = blockIdx.x, b = bh / p.H;
    const int h = (int)(bh - b * p.H), hk = h / p.rep;
    const int tile = blockIdx.y * nw + wave, col = tile * 16 + li;
    const bool live = tile * 16 < p.DV, mine = col < p.DV;
    const E* q = reinterpret_cast<const E*>(p.q) + b * p.sq[1] + hk * p.sq[2];
    const E* k = reinterpret_cast<const E*>(p.k) + b * p.sk[1] + hk * p.sk[2];
    const E* v = reinterpret_cast<const E*>(p.v) + b * p.sv[1] + h * p.sv[2];
    E* o = reinterpret_cast<E*>(p.o) + (b * p.H + h) * (long long)p.DV;
    const long long so = p.B * p.H * (long long)p.DV, sst = (long long)p.DK * p.DV;

    f4 S[DKT];
#pragma unroll
    for (int t = 0; t < DKT; ++t) S[t] = zero4();
    if (p.state0 && mine) {
#pragma unroll
        for (int t = 0; t < DKT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = 16 * t + g4 + r;
                if (d < p.DK) S[t][r] = p.state0[bh * sst + (long long)d * p.DV + col];
            }
    }
    for (int c0 = 0; c0 < p.nchunk; c0 += BT) {
        const long long t0 = (long long)c0 * kC;
        const long long left = p.T - t0;
        const int valid = left < BT * kC ? (int)left : BT * kC;
        const int nc = (valid + kC - 1) / kC;
        __syncthreads();
        load_rows<E>(Ks, KP, k + t0 * p.sk[0], p.sk[0], nc * kC, valid, p.DK, DKP, p.vec, 1.f);
        load_rows<E>(Qs, KP, q + t0 * p.sq[0], p.sq[0], nc * kC, valid, p.DK, DKP, p.vec, 1.f);
        __syncthreads();
        for (int c = wave; c < nc; c += nw) {
            double run; int seg;
            chunk_gates(p, b, h, t0 + c * kC, lane, run, seg, cvs + c);
            const f4 D = chunk_decay(run, seg, lane);
            f4 kk = zero4(), qk = zero4();
            const float* kr = Ks + (c * kC + li) * KP + g4;
            const float* qr = Qs + (c * kC + li) * KP + g4;
#pragma unroll
            for (int t = 0; t < DKT; ++t) {
                const f4 a = lds4(kr + 16 * t), e = lds4(qr + 16 * t);
#pragma unroll
                for (int r = 0; r < 4; ++r) { kk = mfma(a[r], a[r], kk); qk = mfma(e[r], a[r], qk); }
            }
            wave_sync();
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = g4 + r;
                Ti[(c * kC + i) * kSP + li] = i > li ? cvs[c].beta[i] * D[r] * kk[r] : 0.f;
                Am[(c * kC + i) * kSP + li] = i >= li ? D[r] * qk[r] : 0.f;
            }
            wave_sync();
            unit_lower_inverse(Ti + c * kC * kSP, lane);
        }
        __syncthreads();
        if (live) {
            for (int c = 0; c < nc; ++c) {
                const long long tc = t0 + c * kC;
                f4 vv;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const long long t = tc + g4 + r;
                    vv[r] = (mine && t < p.T) ? Elem<E>::get(v[t * p.sv[0] + col]) : 0.f;
                }
                if (p.ckpt && mine) {
                    float* ck = p.ckpt + (bh * (p.nchunk + 1) + c0 + c) * sst + col;
#pragma unroll
                    for (int t = 0; t < DKT; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int d = 16 * t + g4 + r;
                            if (d < p.DK) ck[(long long)d * p.DV] = S[t][r];
                        }
                }
                const float* kr = Ks + (c * kC + li) * KP + g4;
                const float* qr = Qs + (c * kC + li) * KP + g4;
                f4 ks = zero4(), qs = zero4();
#pragma unroll
                for (int t = 0; t < DKT; ++t) {
                    const f4 a = lds4(kr + 16 * t), e = lds4(qr + 16 * t);
#pragma unroll
                    for (int r = 0; r < 4; ++r) { ks = mfma(a[r], S[t][r], ks); qs = mfma(e[r], S[t][r], qs); }
                }
                const ChunkVec& cv = cvs[c];
                const f4 be = lds4(cv.beta + g4), ga = lds4(cv.gam + g4), de = lds4(cv.toend + g4);
                f4 rhs, out;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    rhs[r] = be[r] * (vv[r] - (ga[r] == 0.f ? 0.f : ga[r] * ks[r]));
                    out[r] = ga[r] == 0.f ? 0.f : ga[r] * qs[r];
                }
                const f4 ti = lds4(Ti + (c * kC + li) * kSP + g4), am = lds4(Am + (c * kC + li) * kSP + g4);
                f4 u = zero4();
#pragma unroll
                for (int r = 0; r < 4; ++r) u = mfma(ti[r], rhs[r], u);
#pragma unroll
                for (int r = 0; r < 4; ++r) out = mfma(am[r], u[r], out);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const long long t = tc + g4 + r;
                    if (mine && t < p.T) o[t * so + col] = Elem<E>::put(out[r] * p.scale);
                }
                const float ge = cv.gend;
                const float* kc = Ks + (c * kC + g4) * KP + li;
                f4 ud;
#pragma unroll
                for (int r = 0; r < 4; ++r) ud[r] = u[r] * de[r];
#pragma unroll
                for (int t = 0; t < DKT; ++t) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) S[t][r] = ge == 0.f ? 0.f : ge * S[t][r];
#pragma unroll
                    for (int r = 0; r < 4; ++r) S[t] = mfma(kc[r * KP + 16 * t], ud[r], S[t]);
                }
            }
        }
    }
    if (live && mine) {
        float* outs[2] = {p.state_out ? p.state_out + bh * sst + col : nullptr,
                          p.ckpt ? p.ckpt + (bh * (p.nchunk + 1) + p.nchunk) * sst + col : nullptr};
#pragma unroll
        for (int w = 0; w < 2; ++w)
            if (outs[w]) {
#pragma unroll
                for (int t = 0; t < DKT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int d = 16 * t + g4 + r;
                        if (d < p.DK) outs[w][(long long)d * p.DV] = S[t][r];
                    }
            }
    }
}

// ---- backward ------------------------------------------------------------------------------------------------------------------
// One workgroup per (row, head), chunks from the last to the first, d(state) in registers (wave w: value tiles w, w + 4).  Per chunk:
//   dU = A^T do + D_C K dS,  Y = (I + beta N)^-T dU,  X = beta Y,  dV = X,  dbeta = Y . (V - gam K S0 - N U)      (by value columns)
//   dS <- gam_C dS + Q^T (gam do) - K^T (gam X)                                                                    (by value columns)
//   dQ = gam do S0^T + (do U^T . D) K                                                                              (by key columns)
//   dK = (do U^T . D)^T Q + D_C U dS^T - gam X S0^T + (Z + Z^T) K,   Z = -(X U^T . D), strictly lower              (by key columns)
//   dg_t = sum over s >= t of the same segment (q_s.dq_s - v_s.dv_s), + <dS_C, S_C> if no restart follows in the chunk
// (the last line sums <dS', S'> from the chunk's end, where it is taken whole: no running sum crosses a chunk).  S0 comes from the
// checkpoints of the forward pass; U, X, dS pass through LDS where the contraction changes from key to value columns.
template <typename E, int DKT, int DVT>
__global__ __launch_bounds__(256) void delta_bwd_k(const Seq p) {
    constexpr int DKP = DKT * 16, KP = DKP + 4, DVP = DVT * 16, VP = DVP + 4;
    constexpr int TPW = (DVT + kMaxWaves - 1) / kMaxWaves, KPW = (DKT + kMaxWaves - 1) / kMaxWaves;
    extern __shared__ float sh[];
    float* Ks = sh;
    float* Qs = Ks + kC * KP;
    float* Us = Qs + kC * KP;
    float* Xs = Us + kC * VP;
    float* Os = Xs + kC * VP;                   // scale * do
    float* dSs = Os + kC * VP;                  // [DKP][VP]
    float* Ti = dSs + DKP * VP;
    float* Am = Ti + kC * kSP;
    float* Nm = Am + kC * kSP;
    float* Dm = Nm + kC * kSP;
    float* Bm = Dm + kC * kSP;                  // (do U^T) . D
    float* Zm = Bm + kC * kSP;                  // Z + Z^T
    float* red = Zm + kC * kSP;                 // [3][4][16]: dbeta, v.dv, q.dq by wave; [4]: <dS, S>
    ChunkVec& cv = *reinterpret_cast<ChunkVec*>(red + 3 * 64 + 4);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int li = lane & 15, g4 = (lane >> 4) << 2;
    const long long bh = blockIdx.x, b = bh / p.H;
    const int h = (int)(bh - b * p.H), hk = h / p.rep;
    const E* q = reinterpret_cast<const E*>(p.q) + b * p.sq[1] + hk * p.sq[2];
    const E* k = reinterpret_cast<const E*>(p.k) + b * p.sk[1] + hk * p.sk[2];
    const E* v = reinterpret_cast<const E*>(p.v) + b * p.sv[1] + h * p.sv[2];
    const E* dou = reinterpret_cast<const E*>(p.dout) + b * p.sdo[1] + h * p.sdo[2];
    const long long sst = (long long)p.DK * p.DV, st = p.B * p.H;

    f4 dS[TPW][DKT], Sn[TPW][DKT];              // d(state after the chunk), state after the chunk
#pragma unroll
    for (int w = 0; w < TPW; ++w) {
        const int col = (wave + w * kMaxWaves) * 16 + li;
#pragma unroll
        for (int t = 0; t < DKT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = 16 * t + g4 + r;
                const bool in = d < p.DK && col < p.DV;
                const long long at = (long long)d * p.DV + col;
                dS[w][t][r] = (in && p.dstate1) ? p.dstate1[bh * sst + at] : 0.f;
                Sn[w][t][r] = in ? p.ckpt[(bh * (p.nchunk + 1) + p.nchunk) * sst + at] : 0.f;
            }
    }
    for (int c = p.nchunk - 1; c >= 0; --c) {
        const long long t0 = (long long)c * kC;
        const long long left = p.T - t0;
        const int valid = left < kC ? (int)left : kC;
        const float* ck = p.ckpt + (bh * (p.nchunk + 1) + c) * sst;
        __syncthreads();
        load_rows<E>(Ks, KP, k + t0 * p.sk[0], p.sk[0], kC, valid, p.DK, DKP, p.vec, 1.f);
        load_rows<E>(Qs, KP, q + t0 * p.sq[0], p.sq[0], kC, valid, p.DK, DKP, p.vec, 1.f);
        load_rows<E>(Os, VP, dou + t0 * p.sdo[0], p.sdo[0], kC, valid, p.DV, DVP, p.vec, p.scale);
        __syncthreads();
        if (wave == 0) {
            double run; int seg;
            chunk_gates(p, b, h, t0, lane, run, seg, &cv);
            const f4 D = chunk_decay(run, seg, lane);
            f4 kk = zero4(), qk = zero4();
            const float* kr = Ks + li * KP + g4;
            const float* qr = Qs + li * KP + g4;
#pragma unroll
            for (int t = 0; t < DKT; ++t) {
                const f4 a = lds4(kr + 16 * t), e = lds4(qr + 16 * t);
#pragma unroll
                for (int r = 0; r < 4; ++r) { kk = mfma(a[r], a[r], kk); qk = mfma(e[r], a[r], qk); }
            }
            wave_sync();
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = g4 + r;
                const float n = i > li ? D[r] * kk[r] : 0.f;
                Nm[i * kSP + li] = n;
                Ti[i * kSP + li] = cv.beta[i] * n;
                Am[i * kSP + li] = i >= li ? D[r] * qk[r] : 0.f;
                Dm[i * kSP + li] = D[r];
            }
            wave_sync();
            unit_lower_inverse(Ti, lane);
        }
        __syncthreads();
        const f4 be = lds4(cv.beta + g4), ga = lds4(cv.gam + g4), de = lds4(cv.toend + g4);
        const float ge = cv.gend;
        float db[4] = {0.f, 0.f, 0.f, 0.f}, vd[4] = {0.f, 0.f, 0.f, 0.f}, dots = 0.f;
#pragma unroll
        for (int w = 0; w < TPW; ++w) {
            const int tile = wave + w * kMaxWaves, col = tile * 16 + li;
            if (tile >= DVT) continue;
            const bool mine = col < p.DV;
            f4 vv, dd;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const long long t = t0 + g4 + r;
                vv[r] = (mine && t < p.T) ? Elem<E>::get(v[t * p.sv[0] + col]) : 0.f;
                dd[r] = Os[(g4 + r) * VP + tile * 16 + li];
            }
#pragma unroll
            for (int t = 0; t < DKT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int d = 16 * t + g4 + r;
                    dots += dS[w][t][r] * Sn[w][t][r];
                    Sn[w][t][r] = (d < p.DK && mine) ? ck[(long long)d * p.DV + col] : 0.f;
                    dSs[d * VP + tile * 16 + li] = dS[w][t][r];
                }
            f4 ks = zero4(), kd = zero4();
            const float* kr = Ks + li * KP + g4;
#pragma unroll
            for (int t = 0; t < DKT; ++t) {
                const f4 a = lds4(kr + 16 * t);
#pragma unroll
                for (int r = 0; r < 4; ++r) { ks = mfma(a[r], Sn[w][t][r], ks); kd = mfma(a[r], dS[w][t][r], kd); }
            }
            f4 rhat, rhs, u = zero4(), y = zero4(), x, rres;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                rhat[r] = vv[r] - (ga[r] == 0.f ? 0.f : ga[r] * ks[r]);
                rhs[r] = be[r] * rhat[r];
                kd[r] *= de[r];
            }
            const f4 ti = lds4(Ti + li * kSP + g4), nm = lds4(Nm + li * kSP + g4);
#pragma unroll
            for (int r = 0; r < 4; ++r) u = mfma(ti[r], rhs[r], u);
#pragma unroll
            for (int r = 0; r < 4; ++r) kd = mfma(Am[(g4 + r) * kSP + li], dd[r], kd);           // dU
#pragma unroll
            for (int r = 0; r < 4; ++r) y = mfma(Ti[(g4 + r) * kSP + li], kd[r], y);
            f4 nu = zero4();
#pragma unroll
            for (int r = 0; r < 4; ++r) nu = mfma(nm[r], u[r], nu);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                x[r] = be[r] * y[r];
                rres[r] = rhat[r] - nu[r];
                db[r] += y[r] * rres[r];
                vd[r] += vv[r] * x[r];
                Us[(g4 + r) * VP + tile * 16 + li] = u[r];
                Xs[(g4 + r) * VP + tile * 16 + li] = x[r];
                const long long t = t0 + g4 + r;
                if (mine && t < p.T) reinterpret_cast<E*>(p.dv)[(t * st + bh) * p.DV + col] = Elem<E>::put(x[r]);
                dd[r] *= ga[r];
                x[r] = ga[r] == 0.f ? 0.f : -ga[r] * x[r];
            }
            const float* kc = Ks + g4 * KP + li;
            const float* qc = Qs + g4 * KP + li;
#pragma unroll
            for (int t = 0; t < DKT; ++t) {
#pragma unroll
                for (int r = 0; r < 4; ++r) dS[w][t][r] = ge == 0.f ? 0.f : ge * dS[w][t][r];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    dS[w][t] = mfma(qc[r * KP + 16 * t], dd[r], dS[w][t]);
                    dS[w][t] = mfma(kc[r * KP + 16 * t], x[r], dS[w][t]);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            db[r] = row_sum(db[r]);
            vd[r] = row_sum(vd[r]);
            if (li == 0) { red[wave * 16 + g4 + r] = db[r]; red[64 + wave * 16 + g4 + r] = vd[r]; }
        }
        dots = wave_sum(dots);
        if (lane == 0) red[192 + wave] = dots;
        __syncthreads();
        if (wave < 2) {         // wave 0: do U^T, wave 1: X U^T
            const float* ar = (wave == 0 ? Os : Xs) + li * VP + g4;
            const float* ur = Us + li * VP + g4;
            f4 m = zero4();
#pragma unroll
            for (int t = 0; t < DVT; ++t) {
                const f4 a = lds4(ar + 16 * t), e = lds4(ur + 16 * t);
#pragma unroll
                for (int r = 0; r < 4; ++r) m = mfma(a[r], e[r], m);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = g4 + r;
                const float D = Dm[i * kSP + li];
                if (wave == 0) {
                    Bm[i * kSP + li] = i >= li ? D * m[r] : 0.f;
                } else if (i > li) {
                    const float z = -D * m[r];
                    Zm[i * kSP + li] = z;
                    Zm[li * kSP + i] = z;
                } else if (i == li) {
                    Zm[i * kSP + li] = 0.f;
                }
            }
        }
        __syncthreads();
        float qd[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < KPW; ++w) {
            const int tile = wave + w * kMaxWaves, kcol = tile * 16 + li;
            if (tile >= DKT) continue;
            const bool mine = kcol < p.DK;
            f4 gq = zero4(), gu = zero4(), gx = zero4();
#pragma unroll
            for (int t = 0; t < DVT; ++t) {
                const int c4 = 16 * t + g4;
                f4 s;
#pragma unroll
                for (int r = 0; r < 4; ++r) s[r] = (mine && c4 + r < p.DV) ? ck[(long long)kcol * p.DV + c4 + r] : 0.f;
                const f4 e = lds4(dSs + kcol * VP + c4);
                const f4 od = lds4(Os + li * VP + c4), uu = lds4(Us + li * VP + c4), xx = lds4(Xs + li * VP + c4);
#pragma unroll
                for (int r = 0; r < 4; ++r) { gq = mfma(od[r], s[r], gq); gu = mfma(uu[r], e[r], gu); gx = mfma(xx[r], s[r], gx); }
            }
            const f4 bm = lds4(Bm + li * kSP + g4), zm = lds4(Zm + li * kSP + g4);
            f4 dq, dk;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                dq[r] = ga[r] == 0.f ? 0.f : ga[r] * gq[r];
                dk[r] = de[r] * gu[r] - (ga[r] == 0.f ? 0.f : ga[r] * gx[r]);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float kv = Ks[(g4 + r) * KP + kcol], qv = Qs[(g4 + r) * KP + kcol];
                dq = mfma(bm[r], kv, dq);
                dk = mfma(Bm[(g4 + r) * kSP + li], qv, dk);
                dk = mfma(zm[r], kv, dk);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                qd[r] += dq[r] * Qs[(g4 + r) * KP + kcol];
                const long long t = t0 + g4 + r;
                if (mine && t < p.T) {
                    if (p.dq32) {       // heads that share a key head: summed afterwards, in a fixed order
                        p.dq32[(t * st + bh) * p.DK + kcol] = dq[r];
                        p.dk32[(t * st + bh) * p.DK + kcol] = dk[r];
                    } else {
                        reinterpret_cast<E*>(p.dq)[(t * st + bh) * p.DK + kcol] = Elem<E>::put(dq[r]);
                        reinterpret_cast<E*>(p.dk)[(t * st + bh) * p.DK + kcol] = Elem<E>::put(dk[r]);
                    }
                }
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            qd[r] = row_sum(qd[r]);
            if (li == 0) red[128 + wave * 16 + g4 + r] = qd[r];
        }
        __syncthreads();
        if (wave == 0) {
            float sb = 0.f, w = 0.f, dot = 0.f;
#pragma unroll
            for (int i = 0; i < kMaxWaves; ++i) {
                sb += red[i * 16 + li];
                w += red[128 + i * 16 + li] - red[64 + i * 16 + li];
                dot += red[192 + i];
            }
            const float sraw = cv.seg[li];
            const bool cut = sraw < 0.f;
            const float seg = cut ? -1.f - sraw : sraw;
            const float send = __shfl(seg, 15, 16);
            float acc = seg == send ? dot : 0.f;
#pragma unroll
            for (int s = kC - 1; s >= 0; --s) {
                const float ws = __shfl(w, s, 16), ss = __shfl(seg, s, 16);
                if (s >= li && ss == seg) acc += ws;
            }
            const long long t = t0 + li;
            if (lane < kC && t < p.T) {
                p.dbeta[t * st + bh] = sb;
                p.dg[t * st + bh] = cut ? 0.f : acc;
            }
        }
    }
    if (p.dstate0) {
#pragma unroll
        for (int w = 0; w < TPW; ++w) {
            const int col = (wave + w * kMaxWaves) * 16 + li;
#pragma unroll
            for (int t = 0; t < DKT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int d = 16 * t + g4 + r;
                    if (d < p.DK && col < p.DV) p.dstate0[bh * sst + (long long)d * p.DV + col] = dS[w][t][r];
                }
        }
    }
}

// dq, dk of a key head = the sum over its value heads, in head order
template <typename E>
__global__ __launch_bounds__(256) void delta_fold_k(const float* __restrict__ a, const float* __restrict__ b, E* __restrict__ oa,
                                                    E* __restrict__ ob, long long n, int rep, int DK) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        const long long row = i / DK;               // (t, b, key head)
        const int d = (int)(i - row * DK);
        float sa = 0.f, sb = 0.f;
        for (int r = 0; r < rep; ++r) {
            const long long at = (row * rep + r) * DK + d;
            sa += a[at];
            sb += b[at];
        }
        oa[i] = Elem<E>::put(sa);
        ob[i] = Elem<E>::put(sb);
    }
}

// ---- one token -----------------------------------------------------------------------------------------------------------------
// Bound by reading and writing the state once.  A wave owns one (row, head) and 16 * VEC value columns; lane l holds columns
// VEC * (l % 16).. of the key rows 4 i + l / 16, all of them loaded before the first use.
template <typename E, int R, int VEC>
__global__ __launch_bounds__(256) void delta_step_k(const Seq p, int slices) {
    const int lane = threadIdx.x & 63;
    const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const long long bh = w / slices;
    if (bh >= p.B * p.H) return;
    const long long b = bh / p.H;
    const int h = (int)(bh - b * p.H), hk = h / p.rep;
    const int col = (int)(w - bh * slices) * 16 * VEC + (lane & 15) * VEC, grp = lane >> 4;
    const bool mine = col < p.DV;
    const E* q = reinterpret_cast<const E*>(p.q) + b * p.sq[1] + hk * p.sq[2];
    const E* k = reinterpret_cast<const E*>(p.k) + b * p.sk[1] + hk * p.sk[2];
    const E* v = reinterpret_cast<const E*>(p.v) + b * p.sv[1] + h * p.sv[2];
    const long long sst = (long long)p.DK * p.DV;
    const float* s0 = p.state0 + bh * sst + col;
    float* s1 = p.state_out + bh * sst + col;
    float S[R][VEC];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int d = 4 * i + grp;
#pragma unroll
        for (int e = 0; e < VEC; ++e) S[i][e] = 0.f;
        if (mine && d < p.DK) {
            if constexpr (VEC == 4) {
                const float4 x = *reinterpret_cast<const float4*>(s0 + (long long)d * p.DV);
                S[i][0] = x.x; S[i][1] = x.y; S[i][2] = x.z; S[i][3] = x.w;
            } else {
                S[i][0] = s0[(long long)d * p.DV];
            }
        }
    }
    float kr[R], qr[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int d = 4 * i + grp;
        kr[i] = d < p.DK ? Elem<E>::get(k[d]) : 0.f;
        qr[i] = d < p.DK ? Elem<E>::get(q[d]) : 0.f;
    }
    const float g = p.g[b * p.sg[1] + h * p.sg[2]], be = p.beta[b * p.sb[1] + h * p.sb[2]];
    const bool cut = (p.masks && p.masks[b * p.sm[1]] == 0.f) || g < kDead;
    const float al = expf(g);
    float u[VEC], oo[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        float acc = 0.f;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            S[i][e] = cut ? 0.f : al * S[i][e];
            acc += kr[i] * S[i][e];
        }
        acc += __shfl_xor(acc, 16, 64);
        acc += __shfl_xor(acc, 32, 64);
        const float vv = mine ? Elem<E>::get(v[col + e]) : 0.f;
        u[e] = be * (vv - acc);
        float o = 0.f;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            S[i][e] += kr[i] * u[e];
            o += qr[i] * S[i][e];
        }
        o += __shfl_xor(o, 16, 64);
        o += __shfl_xor(o, 32, 64);
        oo[e] = o * p.scale;
    }
    if (!mine) return;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int d = 4 * i + grp;
        if (d < p.DK) {
            if constexpr (VEC == 4) *reinterpret_cast<float4*>(s1 + (long long)d * p.DV) = make_float4(S[i][0], S[i][1], S[i][2], S[i][3]);
            else s1[(long long)d * p.DV] = S[i][0];
        }
    }
    if (grp == 0) {
        E* o = reinterpret_cast<E*>(p.o) + bh * p.DV + col;
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] = Elem<E>::put(oo[e]);
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------
bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
size_t esize(int dtype) { return dtype == DCC_DELTA_F32 ? 4 : 2; }
const char* sizes_error(const dcc_delta_seq* s) {
    if (!s) return "null argument";
    if (s->T < 0 || s->B < 0) return "T and B must not be negative";
    if (s->HK < 1 || s->H < 1 || s->H % s->HK != 0) return "H must be a positive multiple of HK";
    if (s->DK < 1 || s->DV < 1 || s->DK > DCC_DELTA_MAX_DIM || s->DV > DCC_DELTA_MAX_DIM) return "DK and DV must lie in 1..128";
    if (s->dtype < DCC_DELTA_F32 || s->dtype > DCC_DELTA_F16) return "dtype must be float32, bfloat16 or float16";
    if (s->T > (1ll << 31) || (double)s->B * s->H > 2147483647.0) return "more than 2^31 tokens or (row, head) pairs";
    return nullptr;
}
bool rows_vec(const void* p, const long long* st, int dtype) {
    return aligned(p, 4 * esize(dtype)) && st[0] % 4 == 0 && st[1] % 4 == 0 && st[2] % 4 == 0;
}
Seq base(const dcc_delta_seq* s) {
    Seq p = {};
    p.T = s->T; p.B = s->B; p.HK = s->HK; p.H = s->H; p.DK = s->DK; p.DV = s->DV; p.rep = s->H / s->HK;
    p.nchunk = (int)((s->T + kC - 1) / kC);
    p.scale = s->scale;
    p.q = s->q; p.k = s->k; p.v = s->v; p.g = s->g; p.beta = s->beta; p.masks = s->masks; p.state0 = s->state0;
    for (int i = 0; i < 3; ++i) { p.sq[i] = s->st_q[i]; p.sk[i] = s->st_k[i]; p.sv[i] = s->st_v[i]; p.sg[i] = s->st_g[i]; p.sb[i] = s->st_beta[i]; }
    for (int i = 0; i < 2; ++i) p.sm[i] = s->st_masks[i];
    p.o = s->o; p.state_out = s->state1; p.ckpt = s->ckpt;
    p.vec = rows_vec(s->q, p.sq, s->dtype) && rows_vec(s->k, p.sk, s->dtype);
    return p;
}
int done(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : dcc_fail(kEHIP, std::string(what) + ": " + hipGetErrorString(e));
}
int refuse(const char* what, const char* why) { return dcc_fail(kEINVAL, std::string(what) + ": " + why); }

// a workgroup may ask for more than the 64 KB that a launch allows by itself (a CU has 160)
template <typename K>
bool allow_lds(K kernel, size_t bytes) {
    return bytes <= 65536 || hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) == hipSuccess;
}

template <typename E, int DKT, int BT>
int launch_fwd(const Seq& p, hipStream_t st) {
    constexpr int KP = DKT * 16 + 4;
    const size_t lds = sizeof(float) * (2 * BT * kC * KP + 2 * BT * kC * kSP) + BT * sizeof(ChunkVec);
    const int nt = (p.DV + 15) / 16, nw = nt < kMaxWaves ? nt : kMaxWaves;
    if (!allow_lds(delta_fwd_k<E, DKT, BT>, lds)) return dcc_fail(kEHIP, "dcc_delta_fwd: shared memory refused");
    hipLaunchKernelGGL((delta_fwd_k<E, DKT, BT>), dim3((unsigned)(p.B * p.H), (nt + nw - 1) / nw), dim3(64 * nw), lds, st, p);
    return done("dcc_delta_fwd");
}
template <typename E>
int fwd_typed(const Seq& p, hipStream_t st) {
    const int t = (p.DK + 15) / 16;
    if (p.nchunk == 1) return t <= 2 ? launch_fwd<E, 2, 1>(p, st) : t <= 4 ? launch_fwd<E, 4, 1>(p, st) : launch_fwd<E, 8, 1>(p, st);
    return t <= 2 ? launch_fwd<E, 2, 4>(p, st) : t <= 4 ? launch_fwd<E, 4, 4>(p, st) : launch_fwd<E, 8, 4>(p, st);
}

template <typename E, int DKT, int DVT>
int launch_bwd(const Seq& p, hipStream_t st) {
    constexpr int KP = DKT * 16 + 4, VP = DVT * 16 + 4;
    const size_t lds = sizeof(float) * (2 * kC * KP + 3 * kC * VP + DKT * 16 * VP + 6 * kC * kSP + 3 * 64 + 4) + sizeof(ChunkVec);
    if (!allow_lds(delta_bwd_k<E, DKT, DVT>, lds)) return dcc_fail(kEHIP, "dcc_delta_bwd: shared memory refused");
    hipLaunchKernelGGL((delta_bwd_k<E, DKT, DVT>), dim3((unsigned)(p.B * p.H)), dim3(64 * kMaxWaves), lds, st, p);
    return done("dcc_delta_bwd");
}
template <typename E, int DKT>
int bwd_dv(const Seq& p, hipStream_t st) {
    const int t = (p.DV + 15) / 16;
    return t <= 2 ? launch_bwd<E, DKT, 2>(p, st) : t <= 4 ? launch_bwd<E, DKT, 4>(p, st) : launch_bwd<E, DKT, 8>(p, st);
}
template <typename E>
int bwd_typed(const Seq& p, hipStream_t st) {
    const int t = (p.DK + 15) / 16;
    const int rc = t <= 2 ? bwd_dv<E, 2>(p, st) : t <= 4 ? bwd_dv<E, 4>(p, st) : bwd_dv<E, 8>(p, st);
    if (rc != 0 || !p.dq32) return rc;
    const long long n = p.T * p.B * p.HK * (long long)p.DK;
    const long long nb = (n + 255) / 256;
    hipLaunchKernelGGL((delta_fold_k<E>), dim3((unsigned)(nb < 8192 ? nb : 8192)), dim3(256), 0, st, p.dq32, p.dk32,
                       reinterpret_cast<E*>(p.dq), reinterpret_cast<E*>(p.dk), n, p.rep, p.DK);
    return done("dcc_delta_bwd");
}

template <typename E, int R>
int step_rows(const Seq& p, hipStream_t st) {
    // four columns per lane where the state's rows allow it; one where that would leave the chip empty (under 1024 waves)
    const bool vec = p.DV % 4 == 0 && aligned(p.state0, 16) && aligned(p.state_out, 16) && p.B * p.H * ((p.DV + 63) / 64) >= 1024;
    const int slices = vec ? (p.DV + 63) / 64 : (p.DV + 15) / 16;
    const long long blocks = (p.B * p.H * slices + 3) / 4;
    if (vec) hipLaunchKernelGGL((delta_step_k<E, R, 4>), dim3((unsigned)blocks), dim3(256), 0, st, p, slices);
    else hipLaunchKernelGGL((delta_step_k<E, R, 1>), dim3((unsigned)blocks), dim3(256), 0, st, p, slices);
    return done("dcc_delta_step");
}
template <typename E>
int step_typed(const Seq& p, hipStream_t st) {
    return p.DK <= 32 ? step_rows<E, 8>(p, st) : p.DK <= 64 ? step_rows<E, 16>(p, st) : step_rows<E, 32>(p, st);
}

}  // namespace

extern "C" {

DCC_API int64_t dcc_delta_ckpt_floats(const dcc_delta_seq* s) {
    if (sizes_error(s)) return 0;
    return s->B * s->H * ((s->T + kC - 1) / kC + 1) * (int64_t)s->DK * s->DV;
}
DCC_API int64_t dcc_delta_fwd_workspace_floats(const dcc_delta_seq* s) { (void)s; return 0; }
DCC_API int64_t dcc_delta_bwd_workspace_floats(const dcc_delta_seq* s) {
    if (sizes_error(s) || s->H == s->HK) return 0;
    return 2 * s->T * s->B * s->H * (int64_t)s->DK;
}

DCC_API int dcc_delta_fwd(const dcc_delta_seq* s, float* workspace, void* stream) {
    (void)workspace;
    if (const char* e = sizes_error(s)) return refuse("dcc_delta_fwd", e);
    if (s->B == 0) return 0;
    if (s->T > 0 && (!s->q || !s->k || !s->v || !s->g || !s->beta || !s->o)) return refuse("dcc_delta_fwd", "null pointer");
    const Seq p = base(s);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    switch (s->dtype) {
        case DCC_DELTA_F32: return fwd_typed<float>(p, st);
        case DCC_DELTA_BF16: return fwd_typed<__hip_bfloat16>(p, st);
        default: return fwd_typed<__half>(p, st);
    }
}

DCC_API int dcc_delta_bwd(const dcc_delta_seq* s, const dcc_delta_grad* d, float* workspace, void* stream) {
    if (const char* e = sizes_error(s)) return refuse("dcc_delta_bwd", e);
    if (!d) return refuse("dcc_delta_bwd", "null argument");
    if (s->B == 0) return 0;
    if (!d->ckpt) return refuse("dcc_delta_bwd", "null checkpoint");
    if (s->T > 0 && (!s->q || !s->k || !s->v || !s->g || !s->beta || !d->dout || !d->dq || !d->dk || !d->dv || !d->dg || !d->dbeta))
        return refuse("dcc_delta_bwd", "null pointer");
    Seq p = base(s);
    if (dcc_delta_bwd_workspace_floats(s) > 0) {
        if (!workspace) return refuse("dcc_delta_bwd", "null workspace");
        p.dq32 = workspace;
        p.dk32 = workspace + s->T * s->B * s->H * (int64_t)s->DK;
    }
    p.dout = d->dout; p.dstate1 = d->dstate1; p.ckpt = const_cast<float*>(d->ckpt);
    for (int i = 0; i < 3; ++i) p.sdo[i] = d->st_do[i];
    p.dq = d->dq; p.dk = d->dk; p.dv = d->dv; p.dg = d->dg; p.dbeta = d->dbeta; p.dstate0 = d->dstate0;
    p.vec = p.vec && rows_vec(d->dout, p.sdo, s->dtype);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    switch (s->dtype) {
        case DCC_DELTA_F32: return bwd_typed<float>(p, st);
        case DCC_DELTA_BF16: return bwd_typed<__hip_bfloat16>(p, st);
        default: return bwd_typed<__half>(p, st);
    }
}

DCC_API int dcc_delta_step(const dcc_delta_seq* s, void* stream) {
    if (const char* e = sizes_error(s)) return refuse("dcc_delta_step", e);
    if (s->T != 1) return refuse("dcc_delta_step", "T must be 1");
    if (s->B == 0) return 0;
    if (!s->q || !s->k || !s->v || !s->g || !s->beta || !s->o || !s->state0 || !s->state1) return refuse("dcc_delta_step", "null pointer");
    const Seq p = base(s);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    switch (s->dtype) {
        case DCC_DELTA_F32: return step_typed<float>(p, st);
        case DCC_DELTA_BF16: return step_typed<__hip_bfloat16>(p, st);
        default: return step_typed<__half>(p, st);
    }
}

}  // extern "C"
