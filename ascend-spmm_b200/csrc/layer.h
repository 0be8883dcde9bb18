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

// ---- routing to experts (route.cu) ------------------------------------------
struct RouteLaunch {
    const void *logits;   // [tokens, n]
    const float *bias;    // [n], may be null
    float *weights;       // [tokens, k]
    int *experts;         // [tokens, k]; read by the backward pass
    int64_t tokens;
    int n, k, groups, top_groups, group_best;
    bool sigmoid, renormalize;
    float scale;
    int dtype;
};
constexpr int kMostExperts = 1024, kMostChosen = 32, kMostGroups = 32;
cudaError_t launch_route(const RouteLaunch &r, cudaStream_t stream);
cudaError_t launch_route_backward(const RouteLaunch &r, const float *grad, void *dlogits, DevStatus *status,
                                  cudaStream_t stream);

// ---- stable counting sort (bucket.cu) ---------------------------------------
struct BucketSort {
    const void *keys;       // [n] int32 or int64, or instead of them
    bool wide;
    const int2 *pairs_in;   // [n] inputs and their keys in the order to keep (an earlier pass's), -1: none
    int64_t n;
    int buckets;            // at most kMostBuckets; a key's bucket is (key >> shift) & mask
    int shift, mask;
    int64_t limit;          // keys outside [0, limit) raise the status and are left out
    int64_t skip;           // this key is left out
    int *ptr;               // [buckets + 1] first place of each bucket; may be null
    int *position;          // [n] place of each input, -1 where it is left out; may be null
    int *order;             // [n] input of each place, -1 past the last, or instead of it
    int2 *pairs;            // [n] input and key of each place
    int *counts;            // workspace: bucket_workspace bytes
    int *clear;             // two integers to set to 0; may be null
    void *zero;             // 16-byte vectors to zero meanwhile
    int64_t zero_vectors;
    DevStatus *status;
};
constexpr int kBucketBits = 10, kMostBuckets = 1 << kBucketBits;
// Passes of a sort by more bits, the lowest first; of the same n and numbers of buckets.
struct BucketPasses {
    BucketSort pass[4];
    int passes;
};
size_t bucket_workspace(int64_t n, int buckets);
cudaError_t launch_bucket_sort(const BucketPasses &a, cudaStream_t stream);

// ---- rows to their experts and back (routed.cu) -------------------------------
struct RoutedLaunch {
    const void *x;          // dispatch: [tokens, width]; combine: rows [tokens * k, width]
    const void *grad;       // combine's backward: [tokens, width]
    void *out;
    const int *position;    // [tokens, k]
    const int *source;      // [tokens * k]
    const float *weights;   // [tokens, k], may be null: ones
    float *dweights;        // combine's backward, may be null
    int64_t tokens, width;
    int k, dtype;
    DevStatus *status;
};
cudaError_t launch_dispatch(const RoutedLaunch &r, cudaStream_t stream);
cudaError_t launch_combine(const RoutedLaunch &r, cudaStream_t stream);
cudaError_t launch_combine_backward(const RoutedLaunch &r, cudaStream_t stream);

// ---- rows of a table (embedding.cu) -------------------------------------------
struct EmbeddingLaunch {
    const void *ids;        // [n]
    const void *in;         // the table [rows, width]; backward: the gradient [n, width]
    void *out;              // [n, width]; backward: the table's gradient [rows, width]
    int64_t n, rows, width;
    float scale;
    int itype, dtype;
    DevStatus *status;
};
cudaError_t launch_embedding(const EmbeddingLaunch &l, cudaStream_t stream);
size_t embedding_backward_workspace(int64_t n, int64_t width);
cudaError_t launch_embedding_backward(const EmbeddingLaunch &l, int64_t skip, void *workspace, cudaStream_t stream);

// ---- 8-bit floating point with block scales (fp8.cu) ----------------------------
struct Fp8Launch {
    const void *x;          // [rows, K] e4m3
    const float *x_scale;   // [ceil(K / 128), rows]
    const void *w;          // [groups, N, K] e4m3
    const float *w_scale;   // [groups, ceil(N / 128), ceil(K / 128)]
    const void *ptr;        // [groups + 1]
    void *out;              // [rows, N]
    int64_t rows, groups, K, N;
    int itype, out_dtype;
    DevStatus *status;
};
cudaError_t launch_quantize_rows(const void *x, void *q, float *scale, int64_t rows, int64_t width, int dtype,
                                 cudaStream_t stream);
cudaError_t launch_quantize_weight(const void *w, void *q, float *scale, int64_t groups, int64_t K, int64_t N, int dtype,
                                   cudaStream_t stream);
cudaError_t launch_grouped_fp8(const Fp8Launch &a, cudaStream_t stream);

}  // namespace spmmb
