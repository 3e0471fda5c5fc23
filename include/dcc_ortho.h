/*
 * dcc_ortho.h -- C-ABI of the orthogonalised update (Newton-Schulz products, as the Muon optimiser takes them) in libdcc_hip.so.
 *
 * The reference trains every parameter with Adam (uav_dcc_control/algos/mappo.py:27-37); FlatMuon (algos/algo_utils/optim.py) stands
 * beside it: the update of a weight matrix is its momentum G [M, N] with all singular values drawn towards 1.  With m = min(M, N),
 * X [m, n] = G, transposed when M > N:
 *
 *     X <- X / (|X|_F + eps);      `steps` times:   A = X X^T,   X <- (a I + b A + c A^2) X
 *
 * for every matrix of the list, all matrices of the list together in each launch (a network has a handful of small ones).
 * For small m and for n much longer than m the steps are taken on the m x m side in float64, which is the same polynomial of X in another
 * order.  Large, nearly square matrices are taken step by step: float32 and float16 in products of 24 bits summed in float32, bfloat16 in
 * products of 16 bits on a float32 X (3e-5 of the result or less, like float32 throughout).  The norm is summed in float64, so any
 * finite G has one; G == 0 gives 0.
 *
 * Calls are asynchronous on `stream`, use only `workspace`, keep nothing, and return 0 or a negative DCC_E* code with the message in
 * dcc_last_error().  in[i] and out[i] are contiguous row-major device arrays of `dtype`; an output must not
 * overlap any input or other output.  Matrices with M == 0 or N == 0 are skipped.  Results do not depend on scheduling: no atomics.
 */
#ifndef DCC_ORTHO_H
#define DCC_ORTHO_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#ifndef DCC_API
#if defined(__GNUC__)
#define DCC_API __attribute__((visibility("default")))
#else
#define DCC_API
#endif
#endif

#define DCC_ORTHO_F32 0
#define DCC_ORTHO_BF16 1
#define DCC_ORTHO_F16 2
#define DCC_ORTHO_MAX_STEPS 32

typedef struct {
    const void* in;
    void* out;
    int64_t M, N;
} dcc_ortho_mat;

/* Bytes of `workspace` (256-byte aligned) that dcc_orthogonalize needs for this list; 0 for a list that is refused or empty. */
DCC_API int64_t dcc_ortho_workspace_bytes(const dcc_ortho_mat* mats, int32_t count, int32_t dtype, int32_t steps);

DCC_API int dcc_orthogonalize(const dcc_ortho_mat* mats, int32_t count, int32_t dtype, int32_t steps, float a, float b, float c,
                              float eps, void* workspace, void* stream);

/* The two element-wise ends of a Muon step on flat float32 arrays (16-byte aligned, apart from each other):
 *   dcc_muon_momentum   g = clip * grad;  buf = momentum * buf + g;  dir = nesterov ? g + momentum * buf : buf
 *                       (clip: device pointer to the scale of the gradient, NULL = 1; dcc_grad_norm_clip leaves it)
 *   dcc_muon_apply      param = keep * param - segs[i].scale * dir on every range of the list (ranges must not overlap) */
typedef struct {
    int64_t offset, numel;       /* in elements; the offset a multiple of 4 */
    float scale;
} dcc_muon_seg;
DCC_API int dcc_muon_momentum(const float* grad, float* buf, float* dir, int64_t n, float momentum, int32_t nesterov, const float* clip,
                              void* stream);
DCC_API int dcc_muon_apply(float* param, const float* dir, const dcc_muon_seg* segs, int32_t count, float keep, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* DCC_ORTHO_H */
