// Internal host-side interface between the layer operators' entry points
// (capi_layers.cu) and their kernels.  Not installed; the public ABI is
// include/spmm_b200.h.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/spmm_b200.h"
#include "engine.h"

namespace spmmb {

// A value per device that is computed once (a kernel's launch attributes).
// Racing threads compute the same value.
template <typename T> struct PerDevice {
    static constexpr int kDevices = 64;
    T value[kDevices] = {};
    T *here()   // nullptr: no device, or one out of range
    {
        int dev = 0;
        return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < kDevices ? value + dev : nullptr;
    }
};

// ---- layer normalisation (norm.cu) ---------------------------------------
struct NormLaunch {
    const void *x;
    const void *weight;   // may be null: ones
    const void *bias;     // may be null: zeros
    void *out;            // y (forward) or dx (backward; may be null)
    float *mean, *rstd;   // forward: written when not null; backward: read
    int64_t rows, width;
    float eps;
    int dtype;            // of x, out and the gradient
    int param_dtype;      // of weight, bias and their gradients
};
cudaError_t launch_norm_forward(const NormLaunch &n, cudaStream_t stream);
// Blocks that write a partial row of dw and db each (2 * width floats in the
// workspace).
int64_t norm_backward_blocks(int64_t rows, int64_t width);
cudaError_t launch_norm_backward(const NormLaunch &n, const void *grad, void *dweight, void *dbias, float *workspace,
                                 cudaStream_t stream);

// ---- products grouped by row ranges (grouped.cu) ---------------------------
struct GroupedLaunch {
    const void *x;        // [rows, k] (rows product) or [rows, K] (weight gradient)
    const void *w;        // weight [groups, K, N] or, for the weight gradient, grad [rows, N]
    const void *ptr;      // [groups + 1]
    void *out;
    int64_t rows, groups, K, N;   // K, N: the weight's
    bool transposed;      // rows product: x [rows, N] times the transposed weight
    int itype, dtype;
    DevStatus *status;
};
size_t grouped_rows_workspace(int64_t rows, int64_t groups, int64_t K, int64_t N, bool transposed, int dtype);
cudaError_t launch_grouped_rows(const GroupedLaunch &a, void *workspace, cudaStream_t stream);
size_t grouped_weight_grad_workspace(int64_t rows, int64_t groups, int64_t K, int64_t N, int dtype);
cudaError_t launch_grouped_weight_grad(const GroupedLaunch &a, void *workspace, cudaStream_t stream);

// ---- orthogonalised updates (ortho.cu) --------------------------------------
struct OrthoLaunch {
    const void *update;   // [batch, m, n]
    void *out;            // bf16 [batch, m, n]
    int64_t batch, m, n;
    int steps;
    float a, b, c, eps;
    int dtype;
    DevStatus *status;
};
size_t ortho_workspace(int64_t batch, int64_t m, int64_t n, int dtype);
// A shorter side of at most 128 and steps that its form computes accurately
// (ortho_small.cu): its scale of Q, else 0.
float ortho_small_scale(const OrthoLaunch &o);
size_t ortho_small_workspace(int64_t batch, int64_t m, int64_t n);
cudaError_t launch_ortho_small(const OrthoLaunch &o, float scale_q, void *workspace, cudaStream_t stream);
// Sums of squares of each matrix in parts (ortho.cu): squares [batch][parts].
int ortho_square_parts(int64_t batch, int64_t m, int64_t n);
cudaError_t launch_ortho_squares(const OrthoLaunch &o, double *squares, cudaStream_t stream);
cudaError_t launch_ortho(const OrthoLaunch &o, void *workspace, cudaStream_t stream);

}  // namespace spmmb
