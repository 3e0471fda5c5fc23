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

#include <algorithm>
#include <cstdint>
#include <string>

#include "dcc_delta.h"
#include "dcc_internal.h"

#pragma clang fp contract(fast)

namespace {

constexpr int kEINVAL = -1, kEHIP = -2;
constexpr int kC = 16;                  // tokens per chunk
constexpr int64_t kSegBelow = 128, kSegFill = 512, kSegMin = 16;      // segments of long sequences: see segments_of
constexpr float kDead = -103.98f;       // exp() below this is 0 in float32: a restart

typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned int u4 __attribute__((ext_vector_type(4)));

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
    int nseg, seglen;            // the chunks in segments of `seglen` (a multiple of the block) that run side by side; nseg 1: one
    int* cuts;                   // [nseg - 1] does the summarised segment hold a restart?
    float *sumN, *sumP, *segS;   // [nseg - 1] segment summaries N [DK, DV], P [DK, DK]; [nseg] states at segment starts (all per (row, head))
    long long first;             // this launch's first (row, head) pair (delta_step_k: first workgroup)
    int vec;        // rows of q, k (and dout, v) may be read four elements at a time
};

// lanes of one wave exchange values through LDS between the two sides of this (a wave's LDS operations complete in order)
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ f4 mfma(float a, float b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4 zero4() { f4 z = {0.f, 0.f, 0.f, 0.f}; return z; }
// x, of which the compiler knows nothing: comparisons with it are made where they stand.  (What is compared with the lane's number is the
// same for all chunks, and would be kept for the whole kernel, as a mask of 64 bits each: more than there are scalar registers.)
__device__ __forceinline__ int fresh(int x) {
    asm volatile("" : "+v"(x));
    return x;
}
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

// A state [DK, DV] through a buffer descriptor: 32-bit offsets, rows and columns outside it read 0 and write nothing.
constexpr unsigned kOutside = 0x40000000u;      // byte offset of lanes without a column
__device__ __forceinline__ __amdgpu_buffer_rsrc_t state_rsrc(const float* base, int rows, int cols) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(base), 0, rows * cols * 4, 0x00027000);
}
__device__ __forceinline__ float state_load(__amdgpu_buffer_rsrc_t rs, unsigned off) {
    return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, off, 0, 0));
}
__device__ __forceinline__ void state_store(float v, __amdgpu_buffer_rsrc_t rs, unsigned off) {
    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), rs, off, 0, 0);
}

// A lane's entries of a state, element (16 t + r, 0) at byte offset off + (16 t + r) * row.  The offsets are counted up here each time: the
// compiler would otherwise keep all of them in registers for the whole kernel, and spill.
template <int T, typename F>
__device__ __forceinline__ void for_state(unsigned off, unsigned row, F f) {
    off = fresh(off);
#pragma unroll
    for (int t = 0; t < T; ++t) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            f(t, r, off);
            off += r < 3 ? row : 13 * row;
        }
    }
}
template <int T>
__device__ __forceinline__ void state_load_all(f4 (&s)[T], __amdgpu_buffer_rsrc_t rs, unsigned off, unsigned row) {
    for_state<T>(off, row, [&](int t, int r, unsigned o) { s[t][r] = state_load(rs, o); });
}
template <int T>
__device__ __forceinline__ void state_store_all(const f4 (&s)[T], __amdgpu_buffer_rsrc_t rs, unsigned off, unsigned row) {
    for_state<T>(off, row, [&](int t, int r, unsigned o) { state_store(s[t][r], rs, o); });
}

// ROWS rows of DIMP columns from global memory (row i: base + i * stride; rows >= valid and columns >= dim are zero; valid >= 1) to LDS
// rows of `pitch` floats, in two halves: all loads are under way before the first is waited for, and other work fits in between.
// Out-of-range places read a valid one instead and are cleared afterwards: no branches.  VEC: dim, strides and base are multiples of four.
template <typename E, int ROWS, int DIMP, int NTHR, bool VEC>
struct RowTile {
    static constexpr int C4 = DIMP / 4, N = (ROWS * C4 + NTHR - 1) / NTHR;
    typename Elem<E>::vec raw[N];
    __device__ __forceinline__ void issue(const E* base, long long stride, int valid, int dim) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int e = threadIdx.x + n * NTHR, i = e / C4, c = (e % C4) * 4;
            const E* row = base + (long long)(i < valid ? i : valid - 1) * stride;
            if constexpr (VEC) {
                raw[n] = *reinterpret_cast<const typename Elem<E>::vec*>(row + (c < dim ? c : 0));
            } else {
                E* x = reinterpret_cast<E*>(&raw[n]);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = row[c + j < dim ? c + j : 0];
            }
        }
    }
    __device__ __forceinline__ void commit(float* dst, int pitch, int valid, int dim, float mul) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int e = threadIdx.x + n * NTHR, i = e / C4, c = (e % C4) * 4;
            if (N * NTHR == ROWS * C4 || e < ROWS * C4) {
                const float4 x = Elem<E>::get4(raw[n]);
                f4 y = {x.x * mul, x.y * mul, x.z * mul, x.w * mul};
                const bool in = i < valid;
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = in && c + (VEC ? 0 : j) < dim ? y[j] : 0.f;
                *reinterpret_cast<f4*>(dst + i * pitch + c) = y;
            }
        }
    }
};

constexpr int kSP = 20;                         // pitch of the 16x16 tiles in LDS (rows 16-byte aligned)
struct ChunkVec { float beta[kC], gam[kC], toend[kC], seg[kC], g[kC], gend; int odd; float pad[2]; };     // per chunk: gates as the products use them

// The gates of one token as they come from memory (nothing is computed from them here: that would wait for them, and with them for all
// loads before them) ...
struct RawGate { float g, beta, m; };
__device__ __forceinline__ RawGate load_gate(const Seq& p, long long b, int h, long long t) {
    RawGate x;
    const float* g = p.g + b * p.sg[1] + h * p.sg[2];
    const float* be = p.beta + b * p.sb[1] + h * p.sb[2];
    const float* m = p.masks ? p.masks + b * p.sm[1] : p.g;             // (a select of addresses: no branch)
    const long long sm = p.masks ? p.sm[0] : 0;
    t = t < p.T ? t : p.T - 1;
    x.g = g[t * p.sg[0]];
    x.beta = be[t * p.sb[0]];
    x.m = m[t * sm];
    return x;
}
// ... and as they are used: token t >= T does nothing
struct Gate { float g, beta; int cut; };
__device__ __forceinline__ Gate gate_of(const Seq& p, const RawGate& raw, long long t) {
    const bool in = t < p.T;
    Gate x;
    x.cut = in && ((p.masks && raw.m == 0.f) || raw.g < kDead);
    x.g = x.cut || !in ? 0.f : raw.g;
    x.beta = in ? raw.beta : 0.f;
    return x;
}

// Decays of one chunk, by one wave: lane l works on token l % 16 (the four groups repeat each other).  Running sums in double: the
// difference of two float sums would carry the error of the larger one into every D_ij.  Returns this lane's running sum and segment.
__device__ __forceinline__ void chunk_gates(const Gate& x, int lane, double& run, int& seg, ChunkVec* cv) {
    const int i = fresh(lane) & 15;
    double s = (double)x.g;
    int c = x.cut;
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
    if (fresh(lane) < 16) {
        const float e = c == 0 ? expf((float)s) : 0.f;
        cv->beta[i] = x.beta;
        cv->gam[i] = e;
        cv->toend[i] = c == cend ? expf((float)(send - s)) : 0.f;
        cv->seg[i] = x.cut ? -1.f - c : (float)c;         // sign: a restart at this token
        cv->g[i] = x.g;
        if (i == 15) cv->gend = e;
    }
}

// D_ij of this lane's four entries (row i = 4*(lane/16) + r, column j = lane % 16), 0 above the diagonal
__device__ __forceinline__ f4 chunk_decay(double run, int seg, int lane) {
    lane = fresh(lane);
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

// (I + L)^-1 -> `t` [16][kSP]; this lane holds L[4*(lane/16) + r][lane % 16], strictly lower triangular.  Lane l solves column l % 16 by
// forward substitution; the entries of L come by lane reads, so nothing waits on memory.
__device__ __forceinline__ void unit_lower_inverse(const f4& L, float* t, int lane) {
    lane = fresh(lane);
    const int c = lane & 15;
    float x[kC];
#pragma unroll
    for (int i = 0; i < kC; ++i) {
        float a = i == c ? 1.f : 0.f;
#pragma unroll
        for (int j = 0; j < kC; ++j)
            if (j < i) a -= __int_as_float(__builtin_amdgcn_readlane(__float_as_int(L[i & 3]), 16 * (i >> 2) + j)) * x[j];
        x[i] = a;
        __builtin_amdgcn_sched_barrier(0);      // or all 120 lane reads are taken first, and spilled
    }
    if (lane < 16) {
#pragma unroll
        for (int i = 0; i < kC; ++i) t[i * kSP + c] = x[i];
    }
}

// K K^T and (HASQ) Q K^T of one chunk from its LDS rows
template <int DKT, bool HASQ>
__device__ __forceinline__ void chunk_products(const float* kr, const float* qr, f4& kk, f4& qk) {
    f4 k0 = zero4(), k1 = zero4(), q0 = zero4(), q1 = zero4();
#pragma unroll
    for (int t = 0; t < DKT; ++t) {
        const f4 a = lds4(kr + 16 * t);
        f4 e = zero4();
        if (HASQ) e = lds4(qr + 16 * t);
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
            k0 = mfma(a[r], a[r], k0);
            if (HASQ) q0 = mfma(e[r], a[r], q0);
            k1 = mfma(a[r + 1], a[r + 1], k1);
            if (HASQ) q1 = mfma(e[r + 1], a[r + 1], q1);
        }
    }
    kk = k0 + k1;
    qk = q0 + q1;
}

// ---- values that are not finite ------------------------------------------------------------------------------------------------
// The products of a chunk meet every token with every other: what is not finite would reach tokens before it and tokens behind a restart,
// by way of 0 * NaN.  Where a chunk holds such values, what they reach is taken token by token instead: forward and in the summaries, by
// column, the tokens that they reach; in the gradient, the whole chunk.  These are its pieces, for a lane's part of a state, rows 16 t + 4 *
// (lane / 16) + r of one column.  The barriers to the scheduler keep the registers of these rare paths few.
__device__ __forceinline__ float not_finite(const f4& x) { return (x[0] * 0.f + x[1] * 0.f) + (x[2] * 0.f + x[3] * 0.f); }      // 0, or NaN
template <int T>
__device__ __forceinline__ float token_dot(const f4 (&S)[T], const float* row) {         // S^T row; row: LDS, at + 4 * (lane / 16)
    float a = 0.f;
#pragma unroll
    for (int t = 0; t < T; ++t) {
        const f4 x = lds4(row + 16 * t);
#pragma unroll
        for (int r = 0; r < 4; ++r) a += x[r] * S[t][r];
        __builtin_amdgcn_sched_barrier(0);
    }
    a += __shfl_xor(a, 16, 64);
    return a + __shfl_xor(a, 32, 64);
}
template <int T>
__device__ __forceinline__ void token_add(f4 (&S)[T], const float* row, float u) {        // S += row u^T
#pragma unroll
    for (int t = 0; t < T; ++t) {
        const f4 x = lds4(row + 16 * t);
#pragma unroll
        for (int r = 0; r < 4; ++r) S[t][r] += x[r] * u;
        __builtin_amdgcn_sched_barrier(0);
    }
}
template <int T>
__device__ __forceinline__ void token_decay(f4 (&S)[T], const ChunkVec& cv, int i) {
    const bool cut = cv.seg[i] < 0.f;
    const float al = expf(cv.g[i]);
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[t][r] = cut ? 0.f : al * S[t][r];
}

// ---- forward -------------------------------------------------------------------------------------------------------------------
// One workgroup per (row, head) and NW tiles of 16 value columns; each wave keeps its [DK, 16] slice of the state in registers and
// walks the chunks.  Blocks of BT chunks are staged in LDS: the waves first split the state-free part (K K^T, Q K^T, gates, inverse) of
// the BT chunks among them, then every wave runs the BT chunks on its own columns without a barrier, while the next block is loading.
//
// Few long sequences are cut into segments that run side by side.  A segment maps its start state S to P S + N: SUM_FWD runs it from
// zero on the value columns (N) and from the identity on DK more (P), delta_join_k chains the segments, and FULL runs each from its
// own start.  SUM_BWD does the same for d(state), which runs the other way: dS <- gam_C dS + Q^T (gam do) - K^T (gam X) needs no state.
//
// Bound by the issue of instructions in chains of small products, with two to four waves a SIMD.  8192 (row, head) pairs of 150 tokens,
// 64 x 64 float32, with checkpoints: 800 - 830 us, 2.9 GB at 3.5 TB/s, fp32 MFMA busy 37 % of the time.  8 heads of 16384 tokens, 128 x 128
// bfloat16: 190 - 205 us in 32 segments and 250 - 265 us for their summaries, where one after the other they would take some 6 ms.  Blocks of four chunks
// against one: the preparation of a chunk is a chain of 5 us for one wave, and four waves do one each; a sequence of one chunk takes the
// block of one (960 x 4 pairs of 10 tokens: 59 us, 220 MB).
enum { FULL = 0, SUM_FWD = 1, SUM_BWD = 2 };

// (waves a SIMD: what the loop itself has room for; the rare path must not take it)
template <typename E, int DKT, int BT, int NW, bool VEC, int MODE>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu((DKT > 4 ? 2 : DKT > 2 && BT > 1 ? 3 : 4) + (DKT > 2 && MODE == SUM_FWD && BT > 1 ? 1 : 0)))) void delta_fwd_k(const Seq p) {
    constexpr int DKP = DKT * 16, KP = DKP + 4, CPW = (BT + NW - 1) / NW;
    constexpr bool HASQ = MODE != SUM_FWD;
    extern __shared__ float sh[];
    float* Ks = sh;
    float* Ti = Ks + BT * kC * KP;              // [BT][16][kSP] inverse
    ChunkVec* cvs = reinterpret_cast<ChunkVec*>(Ti + BT * kC * kSP);
    float* Qs = reinterpret_cast<float*>(cvs + BT);
    float* Am = Qs + BT * kC * KP;              // [BT][16][kSP] (Q K^T) . D
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 15, g4 = (lane >> 4) << 2;
    const long long bh = p.first + blockIdx.x, b = bh / p.H;
    const int h = (int)(bh - b * p.H), hk = h / p.rep;
    const int nt = (p.DV + 15) / 16, tile0 = blockIdx.y * NW + wave;
    // (SUM_BWD leaves out segment 0, the others the last one)
    const int seg = MODE == SUM_BWD ? blockIdx.z + 1 : blockIdx.z;
    const bool unit = MODE != FULL && tile0 >= nt;              // a tile of the identity's columns
    const int tile = unit ? tile0 - nt : tile0, col = tile * 16 + li, ncol = unit ? p.DK : p.DV;
    const bool live = tile * 16 < ncol, mine = col < ncol, full = !unit && mine;
    const E* q = reinterpret_cast<const E*>(p.q) + b * p.sq[1] + hk * p.sq[2];
    const E* k = reinterpret_cast<const E*>(p.k) + b * p.sk[1] + hk * p.sk[2];
    const E* v = MODE == SUM_BWD ? reinterpret_cast<const E*>(p.dout) + b * p.sdo[1] + h * p.sdo[2] : reinterpret_cast<const E*>(p.v) + b * p.sv[1] + h * p.sv[2];
    const long long sv0 = MODE == SUM_BWD ? p.sdo[0] : p.sv[0];
    v += full ? col : 0;
    E* o = reinterpret_cast<E*>(p.o) + bh * (long long)p.DV + col;
    const long long so = p.B * p.H * (long long)p.DV, sst = (long long)p.DK * p.DV;
    const unsigned srow = 4u * ncol, soff = mine ? 4u * (g4 * ncol + col) : kOutside;   // state element (16 t + 4 g + r, col): soff + (16 t + r) * srow
    const int cbeg = seg * p.seglen, cend = cbeg + p.seglen < p.nchunk ? cbeg + p.seglen : p.nchunk;

    f4 S[DKT];
#pragma unroll
    for (int t = 0; t < DKT; ++t) S[t] = zero4();
    {
        const float* from = nullptr;
        if (MODE == FULL) from = seg == 0 ? p.state0 ? p.state0 + bh * sst : nullptr : p.segS + (bh * p.nseg + seg) * sst;
        if (MODE == SUM_FWD && !unit && seg == 0 && p.state0) from = p.state0 + bh * sst;
        if (MODE == SUM_BWD && !unit && seg == p.nseg - 1 && p.dstate1) from = p.dstate1 + bh * sst;
        if (from) {
            const __amdgpu_buffer_rsrc_t rs = state_rsrc(from, p.DK, p.DV);
#pragma unroll
            for (int t = 0; t < DKT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) S[t][r] = state_load(rs, soff + (16 * t + r) * srow);
        } else if (unit) {
#pragma unroll
            for (int t = 0; t < DKT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) S[t][r] = 16 * t + g4 + r == col ? 1.f : 0.f;
        }
    }
    auto store_state = [&](float* base) {
        const __amdgpu_buffer_rsrc_t rs = state_rsrc(base, p.DK, ncol);
#pragma unroll
        for (int t = 0; t < DKT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) state_store(S[t][r], rs, soff + (16 * t + r) * srow);
    };
    RowTile<E, BT * kC, DKP, 64 * NW, VEC> rk, rq;
    RawGate gate[CPW];
    E vnext[4];
    auto valid_of = [&](int c0) {
        const long long left = p.T - (long long)c0 * kC;
        return left < BT * kC ? (int)left : BT * kC;
    };
    auto fetch = [&](int c0) {
        const long long t0 = (long long)c0 * kC;
        const int valid = valid_of(c0);
        rk.issue(k + t0 * p.sk[0], p.sk[0], valid, p.DK);
        if (HASQ) rq.issue(q + t0 * p.sq[0], p.sq[0], valid, p.DK);
#pragma unroll
        for (int n = 0; n < CPW; ++n) gate[n] = load_gate(p, b, h, t0 + (wave + n * NW) * kC + li);
    };
    auto fetch_v = [&](long long t0) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const long long t = t0 + g4 + r;
            vnext[r] = v[(t < p.T ? t : p.T - 1) * sv0];
        }
    };
    bool cutseg = false;
    const int nblk = (cend - cbeg + BT - 1) / BT;
    auto block = [&](int i) { return cbeg + BT * (MODE == SUM_BWD ? nblk - 1 - i : i); };
    if (nblk > 0) {
        fetch(block(0));
        fetch_v((long long)(MODE == SUM_BWD ? cend - 1 : cbeg) * kC);
    }
    for (int i = 0; i < nblk; ++i) {
        const int c0 = block(i);
        const long long t0 = (long long)c0 * kC;
        const int nc = cend - c0 < BT ? cend - c0 : BT, valid = valid_of(c0);
        __syncthreads();
        rk.commit(Ks, KP, valid, p.DK, 1.f);
        if (HASQ) rq.commit(Qs, KP, valid, p.DK, 1.f);
        Gate now[CPW];
#pragma unroll
        for (int n = 0; n < CPW; ++n) now[n] = gate_of(p, gate[n], t0 + (wave + n * NW) * kC + li);
        __syncthreads();
        if (i + 1 < nblk) fetch(block(i + 1));
#pragma unroll
        for (int n = 0; n < CPW; ++n) {
            const int c = wave + n * NW;
            if (c >= nc) continue;
            double run; int sg;
            chunk_gates(now[n], lane, run, sg, cvs + c);
            const f4 D = chunk_decay(run, sg, lane);
            f4 kk, qk, L;
            chunk_products<DKT, HASQ>(Ks + (c * kC + li) * KP + g4, Qs + (c * kC + li) * KP + g4, kk, qk);
            wave_sync();
            const f4 be = lds4(cvs[c].beta + g4);
            float amod = 0.f;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int j = g4 + r;
                L[r] = j > li ? be[r] * D[r] * kk[r] : 0.f;
                if (HASQ) {
                    const float a = j >= li ? D[r] * qk[r] : 0.f;
                    Am[(c * kC + j) * kSP + li] = a;
                    if (MODE == SUM_BWD) amod += a * 0.f;
                }
            }
            // (forward, a query reaches its own token's row only)
            const bool odd = __any(not_finite(L) + amod != 0.f);
            if (lane == 0) cvs[c].odd = odd;
            unit_lower_inverse(L, Ti + c * kC * kSP, lane);
        }
        __syncthreads();
        if (live) {
#pragma unroll 1
            for (int n = 0; n < nc; ++n) {
                const int c = MODE == SUM_BWD ? nc - 1 - n : n;
                const long long tc = t0 + c * kC;
                f4 vv;
#pragma unroll
                for (int r = 0; r < 4; ++r) vv[r] = full && tc + g4 + r < p.T ? Elem<E>::get(vnext[r]) : 0.f;
                if (MODE == SUM_BWD ? c0 + c > cbeg : c0 + c + 1 < cend) fetch_v(MODE == SUM_BWD ? tc - kC : tc + kC);
                if (MODE == FULL && p.ckpt) store_state(p.ckpt + (bh * p.nchunk + c0 + c) * sst);
                const float* kr = Ks + (c * kC + li) * KP + g4;
                const float* qr = Qs + (c * kC + li) * KP + g4;
                const ChunkVec& cv = cvs[c];
                const f4 be = lds4(cv.beta + g4), ga = lds4(cv.gam + g4);
                f4 de = lds4(cv.toend + g4);
                float ge = cv.gend;
                const int odd = __builtin_amdgcn_readfirstlane(cv.odd);
                if (MODE != FULL) cutseg |= cv.seg[kC - 1] != 0.f;
                const float* kc = Ks + (c * kC + g4) * KP + li;
                const float* qc = Qs + (c * kC + g4) * KP + li;
                f4 ks = zero4(), qs = zero4();
                if (MODE == SUM_BWD) {
                    // dU = A^T do + D_C K dS, Y = (I + beta N)^-T dU, dS <- gam_C dS + Q^T (gam do) - K^T (gam beta Y)
#pragma unroll
                    for (int r = 0; r < 4; ++r) vv[r] *= p.scale;
#pragma unroll
                    for (int t = 0; t < DKT; ++t) {
                        const f4 a = lds4(kr + 16 * t);
#pragma unroll
                        for (int r = 0; r < 4; r += 2) { ks = mfma(a[r], S[t][r], ks); qs = mfma(a[r + 1], S[t][r + 1], qs); }
                    }
                    f4 y = zero4();
#pragma unroll
                    for (int r = 0; r < 4; ++r) ks[r] = (ks[r] + qs[r]) * de[r];
                    if (__builtin_expect(odd | __any(not_finite(ks) + not_finite(vv) != 0.f), 0)) {
#pragma unroll 1
                        for (int at = (valid - c * kC < kC ? valid - c * kC : kC) - 1; at >= 0; --at) {
                            const float* kt = Ks + (c * kC + at) * KP + g4;
                            const int r = at & 3;
                            const float x = __shfl(r == 0 ? vv[0] : r == 1 ? vv[1] : r == 2 ? vv[2] : vv[3], 4 * (at - r) + li, 64);
                            if (!unit) token_add(S, Qs + (c * kC + at) * KP + g4, x);
                            token_add(S, kt, -cv.beta[at] * token_dot(S, kt));
                            token_decay(S, cv, at);
                        }
                        continue;
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) ks = mfma(Am[(c * kC + g4 + r) * kSP + li], vv[r], ks);
#pragma unroll
                    for (int r = 0; r < 4; ++r) y = mfma(Ti[(c * kC + g4 + r) * kSP + li], ks[r], y);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        vv[r] *= ga[r];
                        y[r] = ga[r] == 0.f ? 0.f : -ga[r] * (be[r] * y[r]);
                    }
#pragma unroll
                    for (int t = 0; t < DKT; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r) S[t][r] = ge == 0.f ? 0.f : ge * S[t][r];
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int t = 0; t < DKT; ++t) S[t] = mfma(qc[r * KP + 16 * t], vv[r], S[t]);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int t = 0; t < DKT; ++t) S[t] = mfma(kc[r * KP + 16 * t], y[r], S[t]);
                    continue;
                }
#pragma unroll
                for (int t = 0; t < DKT; ++t) {
                    const f4 a = lds4(kr + 16 * t);
                    if (MODE == FULL) {
                        const f4 e = lds4(qr + 16 * t);
#pragma unroll
                        for (int r = 0; r < 4; ++r) { ks = mfma(a[r], S[t][r], ks); qs = mfma(e[r], S[t][r], qs); }
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; r += 2) { ks = mfma(a[r], S[t][r], ks); qs = mfma(a[r + 1], S[t][r + 1], qs); }
                    }
                }
                if (MODE != FULL) ks += qs;
                f4 rhs, out;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    rhs[r] = be[r] * (vv[r] - (ga[r] == 0.f ? 0.f : ga[r] * ks[r]));
                    out[r] = ga[r] == 0.f ? 0.f : ga[r] * qs[r];
                }
                const bool rare = odd | __any(not_finite(rhs) != 0.f);
                unsigned met;                   // rare: this lane's tokens that what is not finite reaches, bit r; bit 4: the chunk's end
                f4 walked;
                if (__builtin_expect(rare, 0)) {
                    // By column: what is not finite reaches the tokens from its right-hand side to the end of the stretch between restarts.  They
                    // and, if the last is among them, the state come from the walk; all else keeps the bits that it has without.  (odd: K, the
                    // gates or beta are not finite, and all tokens are walked.)
                    unsigned bad = odd ? 0xffffu : 0u, reach = 0;
                    walked = zero4();
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (rhs[r] * 0.f != 0.f) { bad |= 1u << (g4 + r); rhs[r] = 0.f; }
                    bad |= __shfl_xor(bad, 16, 64);
                    bad |= __shfl_xor(bad, 32, 64);
#pragma unroll 1
                    for (int at = 0; at < kC; ++at) reach |= ((cv.seg[at] < 0.f ? 0u : reach << 1) | bad) & (1u << at);
                    met = (reach >> g4 & 15u) | (reach >> 11 & 16u);
                    if (reach) {
#pragma unroll 1
                        for (int at = 0; at < valid - c * kC && at < kC; ++at) {
                            const float* kt = Ks + (c * kC + at) * KP + g4;
                            const int r = at & 3;
                            const float x = __shfl(r == 0 ? vv[0] : r == 1 ? vv[1] : r == 2 ? vv[2] : vv[3], 4 * (at - r) + li, 64);
                            token_decay(S, cv, at);
                            token_add(S, kt, cv.beta[at] * (x - token_dot(S, kt)));
                            if (MODE == FULL) {
                                const float y = token_dot(S, Qs + (c * kC + at) * KP + g4);
#pragma unroll
                                for (int e = 0; e < 4; ++e) walked[e] = g4 + e == at ? y : walked[e];
                            }
                        }
                    }
                    if (met & 16u) {            // the products leave this state as it is
                        de = zero4();
                        ge = 1.f;
                    }
                }
                if (!odd) {
                    const f4 ti = lds4(Ti + (c * kC + li) * kSP + g4);
                    f4 u = zero4();
#pragma unroll
                    for (int r = 0; r < 4; ++r) u = mfma(ti[r], rhs[r], u);
                    f4 ud;
#pragma unroll
                    for (int r = 0; r < 4; ++r) ud[r] = u[r] * de[r];
                    if (MODE == FULL) {
                        const f4 am = lds4(Am + (c * kC + li) * kSP + g4);
#pragma unroll
                        for (int r = 0; r < 4; ++r) out = mfma(am[r], u[r], out);
                    }
#pragma unroll
                    for (int t = 0; t < DKT; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r) S[t][r] = ge == 0.f ? 0.f : ge * S[t][r];
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int t = 0; t < DKT; ++t) S[t] = mfma(kc[r * KP + 16 * t], ud[r], S[t]);
                }
                if (MODE == FULL && __builtin_expect(rare, 0)) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) out[r] = met >> r & 1u ? walked[r] : out[r];
                }
                if (MODE == FULL) {
                    E* oc = o + (tc + g4) * so;
                    if (mine && tc + kC <= p.T) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) oc[r * so] = Elem<E>::put(out[r] * p.scale);
                    } else if (mine) {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (tc + g4 + r < p.T) oc[r * so] = Elem<E>::put(out[r] * p.scale);
                    }
                }
            }
        }
    }
    if (!live) return;
    if (MODE != FULL) {
        const long long at = bh * (p.nseg - 1) + blockIdx.z;
        store_state(unit ? p.sumP + at * p.DK * p.DK : p.sumN + at * sst);
        if (tile0 == 0 && lane == 0) p.cuts[at] = cutseg;
    } else if (seg == p.nseg - 1) {
        if (p.state_out) store_state(p.state_out + bh * sst);
    }
}

// States at the segment starts from the segments' summaries: S <- P S + N, one 16-column tile per workgroup, wave w the rows 16 w..;
// the state passes through LDS (one barrier a segment) while the next P and N are loading.  `back`: from the last segment to the first.
// A chain of 32 products per segment, 2.2 us each: 31 segments of 128 x 128 for 8 heads 70 us (232 with P loaded in the step that uses it).
template <int DKT, bool VEC>
__global__ __launch_bounds__(64 * DKT) void delta_join_k(const Seq p, int back) {
    __shared__ float sh[2][DKT * 16][17];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, g4 = (lane >> 4) << 2;
    const long long bh = blockIdx.x, sst = (long long)p.DK * p.DV, spp = (long long)p.DK * p.DK;
    const int col = blockIdx.y * 16 + li, n = p.nseg - 1;
    const unsigned srow = 4u * p.DV, off = col < p.DV ? 4u * ((16 * wave + g4) * p.DV + col) : kOutside;
    const int prow = 16 * wave + li;
    // summary i belongs to segment i (forward) or i + 1 (backward)
    struct Sum { f4 P[DKT], N; int cut; };
    auto fetch = [&](Sum& s, int i) {
        i = back ? n - 1 - i : i;
        i = i < 0 ? 0 : i < n ? i : n - 1;
        s.cut = p.cuts[bh * n + i];
        const __amdgpu_buffer_rsrc_t rn = state_rsrc(p.sumN + (bh * n + i) * sst, p.DK, p.DV), rp = state_rsrc(p.sumP + (bh * n + i) * spp, p.DK, p.DK);
#pragma unroll
        for (int r = 0; r < 4; ++r) s.N[r] = state_load(rn, off + r * srow);
#pragma unroll
        for (int t = 0; t < DKT; ++t) {
            const int k = 16 * t + g4;
            if constexpr (VEC) {        // DK a multiple of four
                s.P[t] = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(rp, k < p.DK ? 4u * (prow * p.DK + k) : kOutside, 0, 0));
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r) s.P[t][r] = state_load(rp, k + r < p.DK ? 4u * (prow * p.DK + k + r) : kOutside);
            }
        }
    };
    f4 S;
    auto leave = [&](int i) {           // the state after i + 1 summaries, to LDS and to its segment
        float (*x)[17] = sh[i & 1];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[16 * wave + g4 + r][li] = S[r];
        const __amdgpu_buffer_rsrc_t ro = state_rsrc(p.segS + (bh * p.nseg + (back ? n - 1 - i : i + 1)) * sst, p.DK, p.DV);
#pragma unroll
        for (int r = 0; r < 4; ++r) state_store(S[r], ro, off + r * srow);
        __syncthreads();
    };
    auto step = [&](const Sum& s, int i) {
        const float (*x)[17] = sh[i & 1];
        // behind a restart what the state held before (NaN included) is gone: not multiplied by P == 0.  (P may be 0 by decay alone, which is
        // no restart: NaN stays NaN.)
        if (s.cut) { S = s.N; return; }
        f4 a = s.N, c = zero4();
#pragma unroll
        for (int t = 0; t < DKT; ++t)
#pragma unroll
            for (int r = 0; r < 4; r += 2) {
                a = mfma(s.P[t][r], x[16 * t + g4 + r][li], a);
                c = mfma(s.P[t][r + 1], x[16 * t + g4 + r + 1][li], c);
            }
        S = a + c;
    };
    Sum s0, s1;                         // one on its way while the other is used
    fetch(s1, 0);
    fetch(s0, 1);
    S = s1.N;
    for (int i = 0; i < n; i += 2) {
        leave(i);
        if (i + 1 == n) break;
        fetch(s1, i + 2);
        step(s0, i);
        leave(i + 1);
        if (i + 2 == n) break;
        fetch(s0, i + 3);
        step(s1, i + 1);
    }
}

// ---- backward ------------------------------------------------------------------------------------------------------------------
// One workgroup per (row, head), chunks from the last to the first, d(state) in registers (wave w: value tiles w, w + NW).  Per chunk:
//   dU = A^T do + D_C K dS,  Y = (I + beta N)^-T dU,  X = beta Y,  dV = X,  dbeta = Y . (V - gam K S0 - N U)      (by value columns)
//   dS <- gam_C dS + Q^T (gam do) - K^T (gam X)                                                                    (by value columns)
//   dQ = gam do S0^T + (do U^T . D) K                                                                              (by key columns)
//   dK = (do U^T . D)^T Q + D_C U dS^T - gam X S0^T + (Z + Z^T) K,   Z = -(X U^T . D), strictly lower              (by key columns)
//   dg_t = <dS'_t, S'_t> = gam_C <dS_C, S0> + sum over s >= t of gam_s (q_s.(S0 do_s) - k_s.(S0 x_s)) + sum over j < t of D_Cj k_j.(dS_C u_j)
//          + sum over s >= t > j of D_sj ((q_s.k_j)(do_s.u_j) - (k_s.k_j)(x_s.u_j))
// (every term holds the decay of token t: dg_t of a head that forgets fast is as small as exp(g_t), and a difference of larger sums, such as
// q.dq - v.dv, would have no digits of it left.)  S0 comes from the checkpoints of the forward pass; U, X, dS pass through LDS where the contraction changes from key to value columns.  Between the two
// halves, waves 0 and 1 form do U^T and X U^T while waves 2 and 3 prepare the state-free part of the chunk that comes next; its rows were
// loaded one chunk ahead.  Three barriers per chunk.
// Bound by the chains between those barriers, with two workgroups a compute unit (LDS: 68 KB at 64 x 64) and some 30 thousand cycles a chunk, of
// which waits for memory are below 1.  8192 pairs of 150 tokens, 64 x 64 float32: 2.0 - 2.1 ms, 4.8 GB, fp32 MFMA busy 34 % of the time.  (Two
// more waves that only prepare leave room for one workgroup: 2.6 ms.)
struct ChunkTiles { float Ti[kC * kSP], Am[kC * kSP], Nm[kC * kSP], Dm[kC * kSP]; ChunkVec cv; };

template <typename E, int DKT, int DVT, int NW, bool VEC>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2))) void delta_bwd_k(const Seq p) {
    constexpr int DKP = DKT * 16, KP = DKP + 4, DVP = DVT * 16, VP = DVP + 4;
    constexpr int TPW = (DVT + NW - 1) / NW, KPW = (DKT + NW - 1) / NW;
    extern __shared__ float sh[];
    float* Kb = sh;                             // [2][16][KP], by parity of the chunk
    float* Qb = Kb + 2 * kC * KP;
    float* Ob = Qb + 2 * kC * KP;               // [2][16][VP]: scale * do
    float* Us = Ob + 2 * kC * VP;
    float* Xs = Us + kC * VP;
    float* dSs = Xs + kC * VP;                  // [DKP][VP]
    float* Bm = dSs + DKP * VP;                 // (do U^T) . D
    float* Zm = Bm + kC * kSP;                  // Z + Z^T
    float* redb = Zm + kC * kSP;                // [2][4][NW][16] by wave: dbeta; dg's pairs (waves 0 and 1), terms of s, terms of j
    float* dotb = redb + 2 * 4 * NW * 16;       // [2][NW]: <dS_C, S0>
    int* oddb = reinterpret_cast<int*>(dotb + 2 * NW);                      // [2] (of 4): not all of a chunk's results are finite
    ChunkTiles* tiles = reinterpret_cast<ChunkTiles*>(oddb + 4);            // [2]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 15, g4 = (lane >> 4) << 2;
    const long long bh = p.first + blockIdx.x, b = bh / p.H;
    const int h = (int)(bh - b * p.H), hk = h / p.rep;
    const E* q = reinterpret_cast<const E*>(p.q) + b * p.sq[1] + hk * p.sq[2];
    const E* k = reinterpret_cast<const E*>(p.k) + b * p.sk[1] + hk * p.sk[2];
    const E* v = reinterpret_cast<const E*>(p.v) + b * p.sv[1] + h * p.sv[2];
    const E* dou = reinterpret_cast<const E*>(p.dout) + b * p.sdo[1] + h * p.sdo[2];
    const long long sst = (long long)p.DK * p.DV, st = p.B * p.H;
    const unsigned srow = 4u * p.DV;
    const float* ck0 = p.ckpt + bh * p.nchunk * sst;
    const int seg = blockIdx.y, cbeg = seg * p.seglen, cend = cbeg + p.seglen < p.nchunk ? cbeg + p.seglen : p.nchunk;
    unsigned soff[TPW];
#pragma unroll
    for (int w = 0; w < TPW; ++w) {
        const int col = (wave + w * NW) * 16 + li;
        soff[w] = col < p.DV ? 4u * (g4 * p.DV + col) : kOutside;
    }

    f4 dS[TPW][DKT], S0[TPW][DKT];              // d(state after the chunk); state before the chunk
    E vnext[TPW][4];
    RowTile<E, kC, DKP, 64 * NW, VEC> rk, rq;
    RowTile<E, kC, DVP, 64 * NW, VEC> ro;
    RawGate gate;
    auto valid_of = [&](int c) {
        const long long left = p.T - (long long)c * kC;
        return left < kC ? (int)left : kC;
    };
    auto fetch_state = [&](int c) {
        const __amdgpu_buffer_rsrc_t rs = state_rsrc(ck0 + c * sst, p.DK, p.DV);
#pragma unroll
        for (int w = 0; w < TPW; ++w)
            state_load_all(S0[w], rs, soff[w], srow);
    };
    auto fetch_v = [&](int c) {
#pragma unroll
        for (int w = 0; w < TPW; ++w) {
            const int col = (wave + w * NW) * 16 + li;
            const E* pv = v + (col < p.DV ? col : 0);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const long long t = (long long)c * kC + g4 + r;
                vnext[w][r] = pv[(t < p.T ? t : p.T - 1) * p.sv[0]];
            }
        }
    };
    auto fetch_rows = [&](int c) {
        const long long t0 = (long long)c * kC;
        const int valid = valid_of(c);
        rk.issue(k + t0 * p.sk[0], p.sk[0], valid, p.DK);
        rq.issue(q + t0 * p.sq[0], p.sq[0], valid, p.DK);
        ro.issue(dou + t0 * p.sdo[0], p.sdo[0], valid, p.DV);
        gate = load_gate(p, b, h, t0 + li);
    };
    auto commit_rows = [&](int c) {
        const int valid = valid_of(c), par = c & 1;
        rk.commit(Kb + par * kC * KP, KP, valid, p.DK, 1.f);
        rq.commit(Qb + par * kC * KP, KP, valid, p.DK, 1.f);
        ro.commit(Ob + par * kC * VP, VP, valid, p.DV, p.scale);
    };
    // the state-free part of chunk c, by two waves: `part` 0 gates, K K^T, inverse; 1: Q K^T
    auto prepare = [&](int c, int part, const Gate& gt) {
        ChunkTiles& ct = tiles[c & 1];
        double run; int seg;
        ChunkVec dump;
        if (part == 0) chunk_gates(gt, lane, run, seg, &ct.cv);
        else chunk_gates(gt, lane, run, seg, &dump);
        const f4 D = chunk_decay(run, seg, lane);
        const float* kr = Kb + (c & 1) * kC * KP + li * KP + g4;
        const float* lr = part == 0 ? kr : Qb + (c & 1) * kC * KP + li * KP + g4;
        f4 m0 = zero4(), m1 = zero4();
#pragma unroll
        for (int t = 0; t < DKT; ++t) {
            const f4 a = lds4(lr + 16 * t), e = lds4(kr + 16 * t);
#pragma unroll
            for (int r = 0; r < 4; r += 2) { m0 = mfma(a[r], e[r], m0); m1 = mfma(a[r + 1], e[r + 1], m1); }
        }
        m0 = m0 + m1;
        if (part == 0) {
            wave_sync();
            const f4 be = lds4(ct.cv.beta + g4);
            f4 L;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = g4 + r;
                const float n = i > li ? D[r] * m0[r] : 0.f;
                ct.Nm[i * kSP + li] = n;
                ct.Dm[i * kSP + li] = D[r];
                L[r] = be[r] * n;
            }
            unit_lower_inverse(L, ct.Ti, lane);
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) ct.Am[(g4 + r) * kSP + li] = g4 + r >= li ? D[r] * m0[r] : 0.f;
        }
    };
    auto dot_state = [&](int par) {             // this wave's part of <dS_C, S0> -> dotb[par]
        float d = 0.f;
#pragma unroll
        for (int w = 0; w < TPW; ++w)
#pragma unroll
            for (int t = 0; t < DKT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) d += dS[w][t][r] * S0[w][t][r];
        d = wave_sum(d);
        if (lane == 0) dotb[par * NW + wave] = d;
    };

#pragma unroll
    for (int w = 0; w < TPW; ++w)
#pragma unroll
        for (int t = 0; t < DKT; ++t) dS[w][t] = zero4();
    const float* from = seg == p.nseg - 1 ? p.dstate1 ? p.dstate1 + bh * sst : nullptr : p.segS + (bh * p.nseg + seg) * sst;
    if (from) {
        const __amdgpu_buffer_rsrc_t rs = state_rsrc(from, p.DK, p.DV);
#pragma unroll
        for (int w = 0; w < TPW; ++w)
            state_load_all(dS[w], rs, soff[w], srow);
    }
    // The chunk token by token, all waves together (see "values that are not finite"): results over those that are there, and dS anew.
    auto walk = [&](int c) {
        const long long t0 = (long long)c * kC;
        const int n = valid_of(c);
        const float* Ks = Kb + (c & 1) * kC * KP;
        const float* Qs = Qb + (c & 1) * kC * KP;
        const float* Os = Ob + (c & 1) * kC * VP;
        const ChunkVec& cv = tiles[c & 1].cv;
        static_assert(TPW == 1, "one tile of value columns a wave");
        const int col = wave * 16 + li;
        const bool mine = col < p.DV;
        float* part = dSs;                      // [2][NW][DKP]: dq, dk by wave; the space of d(state), which is taken first
        float* sums = redb + (c & 1) * 4 * NW * 16;             // [2][NW]: dbeta, dg
        if (wave < DVT) {
#pragma unroll
            for (int t = 0; t < DKT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) dS[0][t][r] = dSs[(16 * t + g4 + r) * VP + col];
        }
        __syncthreads();
#pragma unroll 1
        for (int i = n - 1; i >= 0; --i) {
            const float* kt = Ks + i * KP + g4;
            const float* qt = Qs + i * KP + g4;
            const E* pv = v + t0 * p.sv[0] + (mine ? col : 0);
            float db = 0.f, dg = 0.f;
            fetch_state(c);
#pragma unroll 1
            for (int j = 0; j < i; ++j) {
                const float x = mine ? Elem<E>::get(pv[j * p.sv[0]]) : 0.f;
                token_decay(S0[0], cv, j);
                token_add(S0[0], Ks + j * KP + g4, cv.beta[j] * (x - token_dot(S0[0], Ks + j * KP + g4)));
            }
            token_decay(S0[0], cv, i);
            const float be = cv.beta[i], d = mine ? Os[i * VP + col] : 0.f;
            const float rr = (mine ? Elem<E>::get(pv[i * p.sv[0]]) : 0.f) - token_dot(S0[0], kt), u = be * rr;
            token_add(dS[0], qt, d);
            const float du = token_dot(dS[0], kt), dr = be * du;
#pragma unroll
            for (int t = 0; t < DKT; ++t) {
                const f4 x = lds4(kt + 16 * t);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float a = row_sum(mine ? (S0[0][t][r] + x[r] * u) * d : 0.f);
                    const float b = row_sum(mine ? dS[0][t][r] * u - S0[0][t][r] * dr : 0.f);
                    if (li == 0) { part[wave * DKP + 16 * t + g4 + r] = a; part[(NW + wave) * DKP + 16 * t + g4 + r] = b; }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            token_add(dS[0], kt, -dr);
#pragma unroll
            for (int t = 0; t < DKT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) dg += mine && 16 * t + g4 + r < p.DK ? dS[0][t][r] * S0[0][t][r] : 0.f;
            db = row_sum(mine ? du * rr : 0.f);
            dg = wave_sum(dg);
            if (lane == 0) { sums[wave] = db; sums[NW + wave] = dg; }
            if (mine && g4 == 0) (reinterpret_cast<E*>(p.dv) + ((t0 + i) * st + bh) * p.DV)[col] = Elem<E>::put(dr);
            token_decay(dS[0], cv, i);
            __syncthreads();
            for (int e = threadIdx.x; e < p.DK; e += 64 * NW) {
                float a = 0.f, b = 0.f;
                for (int w = 0; w < NW; ++w) { a += part[w * DKP + e]; b += part[(NW + w) * DKP + e]; }
                const long long at = ((t0 + i) * st + bh) * p.DK + e;
                if (p.dq32) {
                    p.dq32[at] = a;
                    p.dk32[at] = b;
                } else {
                    reinterpret_cast<E*>(p.dq)[at] = Elem<E>::put(a);
                    reinterpret_cast<E*>(p.dk)[at] = Elem<E>::put(b);
                }
            }
            if (threadIdx.x == 0) {
                float a = 0.f, b = 0.f;
                for (int w = 0; w < NW; ++w) { a += sums[w]; b += sums[NW + w]; }
                p.dbeta[(t0 + i) * st + bh] = a;
                p.dg[(t0 + i) * st + bh] = cv.seg[i] < 0.f ? 0.f : b;
            }
            __syncthreads();
        }
    };
    const int last = cend - 1;
    if (threadIdx.x < 2) oddb[threadIdx.x] = 0;
    if (last >= cbeg) {
        fetch_rows(last);
        commit_rows(last);
        const Gate gt = gate_of(p, gate, (long long)last * kC + li);
        __syncthreads();
        fetch_state(last);
        fetch_v(last);
        if (last > cbeg) fetch_rows(last - 1);
        if (wave >= 2 && wave < 4) prepare(last, wave - 2, gt);
        __syncthreads();
    }
#pragma unroll 1
    for (int c = last; c >= cbeg; --c) {
        const long long t0 = (long long)c * kC;
        const int par = c & 1;
        const float* Ks = Kb + par * kC * KP;
        const float* Qs = Qb + par * kC * KP;
        const float* Os = Ob + par * kC * VP;
        const ChunkTiles& ct = tiles[par];
        float* red = redb + par * 4 * NW * 16;
        const Gate gnext = gate_of(p, gate, t0 - kC + li);
        if (c > cbeg) commit_rows(c - 1);
        if (c > cbeg + 1) fetch_rows(c - 2);
        const f4 be = lds4(ct.cv.beta + g4), ga = lds4(ct.cv.gam + g4), de = lds4(ct.cv.toend + g4);
        const float ge = ct.cv.gend;
        float db[4] = {0.f, 0.f, 0.f, 0.f};
        dot_state(par);
#pragma unroll
        for (int w = 0; w < TPW; ++w) {
            const int tile = wave + w * NW, col = tile * 16 + li;
            if (tile >= DVT) continue;
            const bool mine = col < p.DV;
            f4 vv, dd;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                vv[r] = mine && t0 + g4 + r < p.T ? Elem<E>::get(vnext[w][r]) : 0.f;
                dd[r] = Os[(g4 + r) * VP + tile * 16 + li];
            }
#pragma unroll
            for (int t = 0; t < DKT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) dSs[(16 * t + g4 + r) * VP + tile * 16 + li] = dS[w][t][r];
            f4 ks = zero4(), kd = zero4();
            const float* kr = Ks + li * KP + g4;
#pragma unroll
            for (int t = 0; t < DKT; ++t) {
                const f4 a = lds4(kr + 16 * t);
#pragma unroll
                for (int r = 0; r < 4; ++r) { kd = mfma(a[r], dS[w][t][r], kd); ks = mfma(a[r], S0[w][t][r], ks); }
            }
            f4 rhat, rhs, u = zero4(), y = zero4(), x;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                rhat[r] = vv[r] - (ga[r] == 0.f ? 0.f : ga[r] * ks[r]);
                rhs[r] = be[r] * rhat[r];
                kd[r] *= de[r];
            }
            const f4 ti = lds4(ct.Ti + li * kSP + g4), nm = lds4(ct.Nm + li * kSP + g4);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                kd = mfma(ct.Am[(g4 + r) * kSP + li], dd[r], kd);            // dU
                u = mfma(ti[r], rhs[r], u);
            }
            f4 nu = zero4();
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                y = mfma(ct.Ti[(g4 + r) * kSP + li], kd[r], y);
                nu = mfma(nm[r], u[r], nu);
            }
            if (__any(not_finite(u) + not_finite(y) != 0.f) && lane == 0) oddb[par] = 1;
            E* dv = reinterpret_cast<E*>(p.dv) + ((t0 + g4) * st + bh) * p.DV + col;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                x[r] = be[r] * y[r];
                db[r] += y[r] * (rhat[r] - nu[r]);
                Us[(g4 + r) * VP + tile * 16 + li] = u[r];
                Xs[(g4 + r) * VP + tile * 16 + li] = x[r];
                if (mine && t0 + g4 + r < p.T) dv[r * st * p.DV] = Elem<E>::put(x[r]);
                dd[r] *= ga[r];
                x[r] = ga[r] == 0.f ? 0.f : -ga[r] * x[r];
            }
            const float* kc = Ks + g4 * KP + li;
            const float* qc = Qs + g4 * KP + li;
#pragma unroll
            for (int t = 0; t < DKT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) dS[w][t][r] = ge == 0.f ? 0.f : ge * dS[w][t][r];
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int t = 0; t < DKT; ++t) dS[w][t] = mfma(qc[r * KP + 16 * t], dd[r], dS[w][t]);
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int t = 0; t < DKT; ++t) dS[w][t] = mfma(kc[r * KP + 16 * t], x[r], dS[w][t]);
        }
        if (c > cbeg) { fetch_state(c - 1); fetch_v(c - 1); }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            db[r] = row_sum(db[r]);
            if (li == 0) red[wave * 16 + g4 + r] = db[r];
        }
        __syncthreads();
        if (threadIdx.x == 0) oddb[par ^ 1] = 0;        // (all have read it before this barrier; the next chunk writes it behind the next)
        if (wave < 2) {         // wave 0: do U^T, wave 1: X U^T
            const float* ar = (wave == 0 ? Os : Xs) + li * VP + g4;
            const float* ur = Us + li * VP + g4;
            f4 m0 = zero4(), m1 = zero4();
#pragma unroll
            for (int t = 0; t < DVT; ++t) {
                const f4 a = lds4(ar + 16 * t), e = lds4(ur + 16 * t);
#pragma unroll
                for (int r = 0; r < 4; r += 2) { m0 = mfma(a[r], e[r], m0); m1 = mfma(a[r + 1], e[r + 1], m1); }
            }
            m0 = m0 + m1;
            const int lc = fresh(li);
            f4 pair, sum = zero4();     // the pairs (s, j) of dg; their sums over s >= t
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = g4 + r;
                const float D = ct.Dm[i * kSP + li];
                const float w = wave == 0 ? ct.Am[i * kSP + li] : -ct.Nm[i * kSP + li];
                pair[r] = i > lc ? w * m0[r] : 0.f;
                if (wave == 0) {
                    Bm[i * kSP + li] = i >= li ? D * m0[r] : 0.f;
                } else if (i >= li) {
                    const float z = i > li ? -D * m0[r] : 0.f;
                    Zm[i * kSP + li] = z;
                    Zm[li * kSP + i] = z;
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) sum = mfma(g4 + r >= lc ? 1.f : 0.f, pair[r], sum);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float w = row_sum(lc < g4 + r ? sum[r] : 0.f);
                if (li == 0) red[(NW + wave) * 16 + g4 + r] = w;
            }
        } else if (wave < 4 && c > cbeg) {
            prepare(c - 1, wave - 2, gnext);
        }
        __syncthreads();
        const __amdgpu_buffer_rsrc_t rs = state_rsrc(ck0 + c * sst, p.DK, p.DV);
        float ps[4] = {0.f, 0.f, 0.f, 0.f}, pj[4] = {0.f, 0.f, 0.f, 0.f};     // dg's terms of s and of j
#pragma unroll
        for (int w = 0; w < KPW; ++w) {
            const int tile = wave + w * NW, kcol = tile * 16 + li;
            if (tile >= DKT) continue;
            const bool mine = kcol < p.DK;
            f4 gq = zero4(), gu = zero4(), gx = zero4();
            f4 s[DVT];
            // (a piece that ends behind DV meets zero columns of do and X; rows behind DK read 0)
#pragma unroll
            for (int t = 0; t < DVT; ++t) {
                const unsigned off = (unsigned)kcol * srow + 4u * (16 * t + g4);
                if constexpr (VEC) {
                    s[t] = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0));
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[t][r] = state_load(rs, off + 4 * r);
                }
            }
#pragma unroll
            for (int t = 0; t < DVT; ++t) {
                const int c4 = 16 * t + g4;
                const f4 e = lds4(dSs + kcol * VP + c4), uu = lds4(Us + li * VP + c4);
#pragma unroll
                for (int r = 0; r < 4; ++r) gu = mfma(uu[r], e[r], gu);
            }
#pragma unroll
            for (int t = 0; t < DVT; ++t) {
                const int c4 = 16 * t + g4;
                const f4 od = lds4(Os + li * VP + c4), xx = lds4(Xs + li * VP + c4);
#pragma unroll
                for (int r = 0; r < 4; ++r) { gq = mfma(od[r], s[t][r], gq); gx = mfma(xx[r], s[t][r], gx); }
            }
            const f4 bm = lds4(Bm + li * kSP + g4), zm = lds4(Zm + li * kSP + g4);
            f4 dq, dk;
            float kvs[4], qvs[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float kv = kvs[r] = Ks[(g4 + r) * KP + kcol], qv = qvs[r] = Qs[(g4 + r) * KP + kcol];
                const float u = de[r] * gu[r], x = ga[r] == 0.f ? 0.f : ga[r] * gx[r];
                dq[r] = ga[r] == 0.f ? 0.f : ga[r] * gq[r];
                dk[r] = u - x;
                ps[r] += dq[r] * qv - x * kv;
                pj[r] += u * kv;
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float kv = kvs[r], qv = qvs[r];
                dq = mfma(bm[r], kv, dq);
                dk = mfma(Bm[(g4 + r) * kSP + li], qv, dk);
                dk = mfma(zm[r], kv, dk);
            }
            const long long at = ((t0 + g4) * st + bh) * p.DK + kcol;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (mine && t0 + g4 + r < p.T) {
                    const long long i = at + r * st * p.DK;
                    if (p.dq32) {       // heads that share a key head: summed afterwards, in a fixed order
                        p.dq32[i] = dq[r];
                        p.dk32[i] = dk[r];
                    } else {
                        reinterpret_cast<E*>(p.dq)[i] = Elem<E>::put(dq[r]);
                        reinterpret_cast<E*>(p.dk)[i] = Elem<E>::put(dk[r]);
                    }
                }
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            ps[r] = row_sum(ps[r]);
            pj[r] = row_sum(pj[r]);
            if (li == 0) { red[(2 * NW + wave) * 16 + g4 + r] = ps[r]; red[(3 * NW + wave) * 16 + g4 + r] = pj[r]; }
        }
        __syncthreads();
        if (__builtin_expect(oddb[par], 0)) {
            walk(c);
            if (c > cbeg) fetch_state(c - 1);
            continue;
        }
        if (wave == 0) {        // (the others go on: red, dotb and the tiles alternate)
            float sb = 0.f, ws = 0.f, wj = 0.f, dot = 0.f;
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                sb += red[i * 16 + li];
                ws += red[(2 * NW + i) * 16 + li];
                wj += red[(3 * NW + i) * 16 + li];
                dot += dotb[par * NW + i];
            }
            const bool cut = ct.cv.seg[li] < 0.f;
            float acc = red[NW * 16 + li] + red[(NW + 1) * 16 + li] + (ge == 0.f ? 0.f : ge * dot);
            const int lc = fresh(li);
#pragma unroll
            for (int s = kC - 1; s >= 0; --s) {
                const float a = __shfl(ws, s, 16), b = __shfl(wj, s, 16);
                acc += s >= lc ? a : b;
            }
            const long long t = t0 + li;
            if (lane < kC && t < p.T) {
                p.dbeta[t * st + bh] = sb;
                p.dg[t * st + bh] = cut ? 0.f : acc;
            }
        }
    }
    if (seg == 0 && p.dstate0) {
        const __amdgpu_buffer_rsrc_t rs = state_rsrc(p.dstate0 + bh * sst, p.DK, p.DV);
#pragma unroll
        for (int w = 0; w < TPW; ++w)
            if (wave + w * NW < DVT) state_store_all(dS[w], rs, soff[w], srow);
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
// Bound by reading and writing the state once: 32768 x 4 states of 64 x 64 in 845 us, 5.2 TB/s, where a large copy reaches 4.8 and an addition in
// place 5.9; 1000 x 6 states of 96 x 80 in 70 us.  64 x 4 states take 4.5 us.  A wave owns one (row, head) and 16 * VEC value columns; lane l holds columns
// VEC * (l % 16).. of the key rows 4 i + l / 16, all of them loaded before the first use.
template <typename E, int R, int VEC>
__global__ __launch_bounds__(256) void delta_step_k(const Seq p, int slices) {
    const int lane = threadIdx.x & 63;
    const long long w = (p.first + blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long bh = w / slices;
    if (bh >= p.B * p.H) return;
    const long long b = bh / p.H;
    const int h = (int)(bh - b * p.H), hk = h / p.rep;
    const int col = (int)(w - bh * slices) * 16 * VEC + (lane & 15) * VEC, grp = lane >> 4;
    const bool mine = col < p.DV;
    const E* q = reinterpret_cast<const E*>(p.q) + b * p.sq[1] + hk * p.sq[2];
    const E* k = reinterpret_cast<const E*>(p.k) + b * p.sk[1] + hk * p.sk[2];
    const E* v = reinterpret_cast<const E*>(p.v) + b * p.sv[1] + h * p.sv[2] + (mine ? col : 0);
    const long long sst = (long long)p.DK * p.DV;
    const __amdgpu_buffer_rsrc_t r0 = state_rsrc(p.state0 + bh * sst, p.DK, p.DV), r1 = state_rsrc(p.state_out + bh * sst, p.DK, p.DV);
    const unsigned off = mine ? 4u * (grp * p.DV + col) : kOutside, srow = 16u * p.DV;     // row 4 i + grp: off + i * srow
    float S[R][VEC];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if constexpr (VEC == 4) {
            const f4 x = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(r0, off + i * srow, 0, 0));
            S[i][0] = x[0]; S[i][1] = x[1]; S[i][2] = x[2]; S[i][3] = x[3];
        } else {
            S[i][0] = state_load(r0, off + i * srow);
        }
    }
    float kr[R], qr[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int d = 4 * i + grp, dc = d < p.DK ? d : 0;
        kr[i] = Elem<E>::get(k[dc]);
        qr[i] = Elem<E>::get(q[dc]);
        if (d >= p.DK) kr[i] = qr[i] = 0.f;
    }
    float vv[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) vv[e] = Elem<E>::get(v[e]);
    const float g = p.g[b * p.sg[1] + h * p.sg[2]], be = p.beta[b * p.sb[1] + h * p.sb[2]];
    const bool cut = (p.masks && p.masks[b * p.sm[1]] == 0.f) || g < kDead;
    const float al = expf(g);
    float oo[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        float a0 = 0.f, a1 = 0.f;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            S[i][e] = cut ? 0.f : al * S[i][e];
            (i & 1 ? a1 : a0) += kr[i] * S[i][e];
        }
        float acc = a0 + a1;
        acc += __shfl_xor(acc, 16, 64);
        acc += __shfl_xor(acc, 32, 64);
        const float u = be * (vv[e] - acc);
        a0 = a1 = 0.f;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            S[i][e] += kr[i] * u;
            (i & 1 ? a1 : a0) += qr[i] * S[i][e];
        }
        float o = a0 + a1;
        o += __shfl_xor(o, 16, 64);
        o += __shfl_xor(o, 32, 64);
        oo[e] = o * p.scale;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if constexpr (VEC == 4) {
            const f4 x = {S[i][0], S[i][1], S[i][2], S[i][3]};
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, x), r1, off + i * srow, 0, 0);
        } else {
            state_store(S[i][0], r1, off + i * srow);
        }
    }
    if (mine && grp == 0) {
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
// rows of `dim` elements that may be read four at a time
bool rows_vec(const void* p, const long long* st, int dim, int dtype) {
    return aligned(p, 4 * esize(dtype)) && st[0] % 4 == 0 && st[1] % 4 == 0 && st[2] % 4 == 0 && dim % 4 == 0;
}
// Segments of a call whose workgroups (row, head and, forward, 64 value columns) leave most of the chip idle: enough to fill it, none
// shorter than 16 chunks.  The summaries cost about what the pass itself does, so a chip that is half full is left alone.
int segments_of(const dcc_delta_seq* s, bool backward, int& seglen) {
    const int64_t nchunk = (s->T + kC - 1) / kC, wgs = s->B * s->H * (backward ? 1 : (s->DV + 63) / 64);
    int64_t n = 1;
    if (wgs > 0 && wgs <= kSegBelow) n = std::max<int64_t>(1, std::min<int64_t>(kSegFill / wgs, nchunk / kSegMin));
    int64_t len = (nchunk + n - 1) / n;
    len = (len + 3) / 4 * 4;            // whole blocks
    seglen = (int)std::max<int64_t>(len, 4);
    return (int)std::max<int64_t>(1, (nchunk + seglen - 1) / seglen);
}
int64_t segment_floats(const dcc_delta_seq* s, int nseg) {
    if (nseg <= 1) return 0;
    return s->B * s->H * ((int64_t)(nseg - 1) * (s->DK * (s->DV + s->DK) + 1) + (int64_t)nseg * s->DK * s->DV);
}
void place_segments(Seq& p, float* ws) {
    if (p.nseg <= 1) return;
    const int64_t bh = p.B * p.H;
    p.sumN = ws;
    p.sumP = p.sumN + bh * (p.nseg - 1) * p.DK * p.DV;
    p.segS = p.sumP + bh * (p.nseg - 1) * p.DK * p.DK;
    p.cuts = reinterpret_cast<int*>(p.segS + bh * p.nseg * p.DK * p.DV);
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
    p.vec = rows_vec(s->q, p.sq, s->DK, s->dtype) && rows_vec(s->k, p.sk, s->DK, s->dtype);
    return p;
}
int done(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : dcc_fail_nothrow(kEHIP, what, ": ", hipGetErrorString(e));
}
int refuse(const char* what, const char* why) { return dcc_fail_nothrow(kEINVAL, what, ": ", why); }

// a workgroup may ask for more than the 64 KB that a launch allows by itself (a CU has 160)
template <typename K>
bool allow_lds(K kernel, size_t bytes) {
    return bytes <= 65536 || hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) == hipSuccess;
}

// A launch holds less than 2^32 threads in a direction: n workgroups of at most 512 in as many launches as that takes
template <typename F>
int in_launches(Seq& p, int64_t n, const char* what, F launch) {
    constexpr int64_t kMost = 1 << 22;
    for (p.first = 0; p.first < n; p.first += kMost) launch((unsigned)std::min(n - (int64_t)p.first, kMost));
    return done(what);
}

template <typename E, int DKT, int BT, int NW, bool VEC, int MODE>
int launch_walk(Seq& p, hipStream_t st) {
    constexpr int KP = DKT * 16 + 4, TILES = MODE == SUM_FWD ? 1 : 2;
    const size_t lds = sizeof(float) * TILES * (BT * kC * KP + BT * kC * kSP) + BT * sizeof(ChunkVec);
    const int nt = (p.DV + 15) / 16 + (MODE == FULL ? 0 : (p.DK + 15) / 16);
    if (!allow_lds(delta_fwd_k<E, DKT, BT, NW, VEC, MODE>, lds)) return dcc_fail_nothrow(kEHIP, "gated delta rule: shared memory refused");
    return in_launches(p, p.B * p.H, "gated delta rule", [&](unsigned pairs) {
        hipLaunchKernelGGL((delta_fwd_k<E, DKT, BT, NW, VEC, MODE>), dim3(pairs, (nt + NW - 1) / NW, MODE == FULL ? p.nseg : p.nseg - 1), dim3(64 * NW), lds, st, p);
    });
}
// segment summaries and the states at the segments' starts (dir SUM_FWD) or ends (SUM_BWD)
template <typename E, int DKT, int DIR>
int segments(Seq& p, hipStream_t st) {
    const int rc = p.vec ? launch_walk<E, DKT, 4, 4, true, DIR>(p, st) : launch_walk<E, DKT, 1, 4, false, DIR>(p, st);
    if (rc != 0) return rc;
    const dim3 grid((unsigned)(p.B * p.H), (p.DV + 15) / 16);
    if (p.DK % 4 == 0) hipLaunchKernelGGL((delta_join_k<DKT, true>), grid, dim3(64 * DKT), 0, st, p, DIR == SUM_BWD);
    else hipLaunchKernelGGL((delta_join_k<DKT, false>), grid, dim3(64 * DKT), 0, st, p, DIR == SUM_BWD);
    return done("gated delta rule");
}
template <typename E, int DKT>
int fwd_dk(Seq& p, hipStream_t st) {
    if (p.nseg > 1)
        if (const int rc = segments<E, DKT, SUM_FWD>(p, st)) return rc;
    if (!p.vec) return launch_walk<E, DKT, 1, 4, false, FULL>(p, st);
    if (p.nchunk <= 1) return p.DV <= 32 ? launch_walk<E, DKT, 1, 2, true, FULL>(p, st) : launch_walk<E, DKT, 1, 4, true, FULL>(p, st);
    return p.DV <= 32 ? launch_walk<E, DKT, 2, 2, true, FULL>(p, st) : launch_walk<E, DKT, 4, 4, true, FULL>(p, st);
}
template <typename E>
int fwd_typed(Seq& p, hipStream_t st) {
    const int t = (p.DK + 15) / 16;
    return t <= 2 ? fwd_dk<E, 2>(p, st) : t <= 4 ? fwd_dk<E, 4>(p, st) : fwd_dk<E, 8>(p, st);
}

template <typename E, int DKT, int DVT, int NW, bool VEC>
int launch_bwd(Seq& p, hipStream_t st) {
    constexpr int KP = DKT * 16 + 4, VP = DVT * 16 + 4;
    const size_t lds = sizeof(float) * (4 * kC * KP + 4 * kC * VP + DKT * 16 * VP + 2 * kC * kSP + 8 * NW * 16 + 2 * NW + 4) + 2 * sizeof(ChunkTiles);
    if (!allow_lds(delta_bwd_k<E, DKT, DVT, NW, VEC>, lds)) return dcc_fail_nothrow(kEHIP, "dcc_delta_bwd: shared memory refused");
    return in_launches(p, p.B * p.H, "dcc_delta_bwd", [&](unsigned pairs) {
        hipLaunchKernelGGL((delta_bwd_k<E, DKT, DVT, NW, VEC>), dim3(pairs, p.nseg), dim3(64 * NW), lds, st, p);
    });
}
template <typename E, int DKT>
int bwd_dv(Seq& p, hipStream_t st) {
    const int t = (p.DV + 15) / 16;
    constexpr int NW = DKT > 4 ? 8 : 4;
    if (p.nseg > 1)
        if (const int rc = segments<E, DKT, SUM_BWD>(p, st)) return rc;
    if (!p.vec) return launch_bwd<E, DKT, 8, 8, false>(p, st);
    return t <= 2 ? launch_bwd<E, DKT, 2, NW, true>(p, st) : t <= 4 ? launch_bwd<E, DKT, 4, NW, true>(p, st) : launch_bwd<E, DKT, 8, 8, true>(p, st);
}
template <typename E>
int bwd_typed(Seq& p, hipStream_t st) {
    const int t = (p.DK + 15) / 16;
    const int rc = t <= 2 ? bwd_dv<E, 2>(p, st) : t <= 4 ? bwd_dv<E, 4>(p, st) : bwd_dv<E, 8>(p, st);
    if (rc != 0 || !p.dq32) return rc;
    const long long n = p.T * p.B * p.HK * (long long)p.DK;
    const long long nb = (n + 255) / 256;
    hipLaunchKernelGGL((delta_fold_k<E>), dim3((unsigned)(nb < 8192 ? nb : 8192)), dim3(256), 0, st, p.dq32, p.dk32,
                       reinterpret_cast<E*>(p.dq), reinterpret_cast<E*>(p.dk), n, p.rep, p.DK);
    return done("dcc_delta_bwd");
}

// Do the results of a step share bytes with what it reads, or with each other?  (Workgroups read the same operands at their own time.)
bool step_overlaps(const dcc_delta_seq* s) {
    struct Range { uintptr_t a, b; };
    auto range = [](const void* p, int64_t last, int64_t bytes) {           // `last`: the highest element's index
        const uintptr_t a = reinterpret_cast<uintptr_t>(p);
        return Range{a, a + (uintptr_t)((last + 1) * bytes)};
    };
    auto meet = [](const Range& x, const Range& y) { return x.a < y.b && y.a < x.b; };
    const int64_t e = esize(s->dtype), b = s->B - 1, state = s->B * s->H * s->DK * s->DV;
    const Range o = range(s->o, s->B * s->H * s->DV - 1, e), s0 = range(s->state0, state - 1, 4), s1 = range(s->state1, state - 1, 4);
    const Range in[] = {range(s->q, b * s->st_q[1] + (s->HK - 1) * s->st_q[2] + s->DK - 1, e), range(s->k, b * s->st_k[1] + (s->HK - 1) * s->st_k[2] + s->DK - 1, e),
                        range(s->v, b * s->st_v[1] + (s->H - 1) * s->st_v[2] + s->DV - 1, e), range(s->g, b * s->st_g[1] + (s->H - 1) * s->st_g[2], 4),
                        range(s->beta, b * s->st_beta[1] + (s->H - 1) * s->st_beta[2], 4),
                        s->masks ? range(s->masks, b * s->st_masks[1], 4) : Range{0, 0}};
    for (const Range& x : in)
        if (meet(o, x) || meet(s1, x)) return true;
    return meet(o, s0) || meet(o, s1) || (s->state1 != s->state0 && meet(s1, s0));
}
template <typename E, int R>
int step_rows(Seq& p, hipStream_t st) {
    // four columns per lane where the state's rows allow it; one where that would leave the chip empty (under 1024 waves)
    const bool vec = p.DV % 4 == 0 && aligned(p.state0, 16) && aligned(p.state_out, 16) && p.B * p.H * ((p.DV + 63) / 64) >= 1024;
    const int slices = vec ? (p.DV + 63) / 64 : (p.DV + 15) / 16;
    return in_launches(p, (p.B * p.H * slices + 3) / 4, "dcc_delta_step", [&](unsigned blocks) {
        if (vec) hipLaunchKernelGGL((delta_step_k<E, R, 4>), dim3(blocks), dim3(256), 0, st, p, slices);
        else hipLaunchKernelGGL((delta_step_k<E, R, 1>), dim3(blocks), dim3(256), 0, st, p, slices);
    });
}
template <typename E>
int step_typed(Seq& p, hipStream_t st) {
    return p.DK <= 32 ? step_rows<E, 8>(p, st) : p.DK <= 64 ? step_rows<E, 16>(p, st) : p.DK <= 96 ? step_rows<E, 24>(p, st) : step_rows<E, 32>(p, st);
}

}  // namespace

extern "C" {

DCC_API int64_t dcc_delta_ckpt_floats(const dcc_delta_seq* s) {
    if (sizes_error(s)) return 0;
    return s->B * s->H * ((s->T + kC - 1) / kC) * (int64_t)s->DK * s->DV;
}
DCC_API int64_t dcc_delta_fwd_workspace_floats(const dcc_delta_seq* s) {
    int len;
    return sizes_error(s) ? 0 : segment_floats(s, segments_of(s, false, len));
}
DCC_API int64_t dcc_delta_bwd_workspace_floats(const dcc_delta_seq* s) {
    int len;
    if (sizes_error(s)) return 0;
    return segment_floats(s, segments_of(s, true, len)) + (s->H == s->HK ? 0 : 2 * s->T * s->B * s->H * (int64_t)s->DK);
}

DCC_API int dcc_delta_fwd(const dcc_delta_seq* s, float* workspace, void* stream) {
    if (const char* e = sizes_error(s)) return refuse("dcc_delta_fwd", e);
    if (s->B == 0) return 0;
    if (s->T > 0 && (!s->q || !s->k || !s->v || !s->g || !s->beta || !s->o)) return refuse("dcc_delta_fwd", "null pointer");
    if (dcc_delta_fwd_workspace_floats(s) > 0 && !workspace) return refuse("dcc_delta_fwd", "null workspace");
    Seq p = base(s);
    p.nseg = segments_of(s, false, p.seglen);
    place_segments(p, workspace);
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
        if (s->H != s->HK) {
            p.dq32 = workspace + segment_floats(s, segments_of(s, true, p.seglen));
            p.dk32 = p.dq32 + s->T * s->B * s->H * (int64_t)s->DK;
        }
    }
    p.nseg = segments_of(s, true, p.seglen);
    place_segments(p, workspace);
    p.dout = d->dout; p.dstate1 = d->dstate1; p.ckpt = const_cast<float*>(d->ckpt);
    for (int i = 0; i < 3; ++i) p.sdo[i] = d->st_do[i];
    p.dq = d->dq; p.dk = d->dk; p.dv = d->dv; p.dg = d->dg; p.dbeta = d->dbeta; p.dstate0 = d->dstate0;
    p.vec = p.vec && rows_vec(d->dout, p.sdo, s->DV, s->dtype);
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
    if (step_overlaps(s)) return refuse("dcc_delta_step", "o and state1 must lie apart from the operands and from each other (state1 may be state0)");
    Seq p = base(s);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    switch (s->dtype) {
        case DCC_DELTA_F32: return step_typed<float>(p, st);
        case DCC_DELTA_BF16: return step_typed<__hip_bfloat16>(p, st);
        default: return step_typed<__half>(p, st);
    }
}

}  // extern "C"
