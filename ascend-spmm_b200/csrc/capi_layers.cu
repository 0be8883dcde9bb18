// extern "C" entry points of the layer operators (declared in
// include/spmm_b200.h): argument contract, workspace check and launch.
#include <cmath>
#include <cstdint>
#include <initializer_list>

#include "../../include/spmm_b200.h"
#include "common.cuh"
#include "engine.h"
#include "layer.h"

namespace {

using spmmb::capi_error;

int elem_bytes(int dtype) { return dtype == SPMM_F32 ? 4 : 2; }

int check_dtype(int dtype, const char *op)
{
    if (dtype != SPMM_F16 && dtype != SPMM_BF16 && dtype != SPMM_F32)
        return capi_error(SPMM_ERR_ARG, "%s supports only FP16, BF16 and FP32 tensors", op);
    return SPMM_OK;
}

bool misaligned(const void *p) { return ((uintptr_t)p & 15u) != 0; }

int cuda_error(cudaError_t e, const char *op) { return capi_error(SPMM_ERR_CUDA, "%s: %s", op, cudaGetErrorString(e)); }

int check_workspace(const void *ws, size_t have, size_t need, const char *op)
{
    if (misaligned(ws)) return capi_error(SPMM_ERR_ARG, "%s: workspace must be 16-byte aligned", op);
    if (have < need || (need > 0 && !ws))
        return capi_error(SPMM_ERR_WORKSPACE, "%s: workspace of %zu bytes is smaller than the %zu required", op, have,
                          need);
    return SPMM_OK;
}

// Sizes whose product, in bytes, fits 63 bits with room for the offsets.
int check_size(int64_t a, int64_t b, int64_t c, const char *op)
{
    if (a < 0 || b < 0 || c < 0) return capi_error(SPMM_ERR_ARG, "%s: negative size", op);
    if ((double)a * (double)b * (double)c > 1e17) return capi_error(SPMM_ERR_ARG, "%s: size too large", op);
    return SPMM_OK;
}

int check_norm(const void *x, const void *weight, const void *bias, const void *out, int64_t rows, int64_t width,
               int dtype, int param_dtype, const char *op)
{
    int rc = check_dtype(dtype, op);
    if (rc) return rc;
    if (param_dtype != dtype && param_dtype != SPMM_F32)
        return capi_error(SPMM_ERR_ARG, "%s: weight and bias must have the dtype of x or FP32", op);
    if ((rc = check_size(rows, width, 1, op))) return rc;
    if (width < 1) return capi_error(SPMM_ERR_ARG, "%s requires a feature width of at least 1", op);
    if (rows > 0 && !x) return capi_error(SPMM_ERR_ARG, "%s: null array", op);
    if (misaligned(x) || misaligned(weight) || misaligned(bias) || misaligned(out))
        return capi_error(SPMM_ERR_ARG, "%s: arrays must be 16-byte aligned", op);
    return SPMM_OK;
}

int check_grouped(const void *x, const void *w, const void *ptr, const void *out, int64_t rows, int64_t groups,
                  int64_t K, int64_t N, int itype, int dtype, const char *op)
{
    int rc = check_dtype(dtype, op);
    if (rc) return rc;
    if (itype != SPMM_I32 && itype != SPMM_I64)
        return capi_error(SPMM_ERR_ARG, "%s: index arrays must be int32 or int64", op);
    if ((rc = check_size(rows, K, N, op)) || (rc = check_size(groups, K, N, op))) return rc;
    const int64_t unit = 32 / elem_bytes(dtype);
    for (const int64_t width : {K, N}) {
        if (width <= 0) return capi_error(SPMM_ERR_ARG, "%s requires 0 < feature width", op);
        if (width % unit != 0)
            return capi_error(SPMM_ERR_ARG,
                              "%s requires feature width divisible by %lld, but got %lld. Pad and crop the tensors.",
                              op, (long long)unit, (long long)width);
        if (width > INT32_MAX) return capi_error(SPMM_ERR_ARG, "%s: size too large", op);
    }
    if (rows > INT32_MAX || groups > (1 << 24)) return capi_error(SPMM_ERR_ARG, "%s: size too large", op);
    if (!ptr || (rows > 0 && !x)) return capi_error(SPMM_ERR_ARG, "%s: null array", op);
    if (misaligned(x) || misaligned(w) || misaligned(out))
        return capi_error(SPMM_ERR_ARG, "%s: arrays must be 16-byte aligned", op);
    return SPMM_OK;
}

int check_route(const void *logits, const void *bias, const void *weights, const void *experts, int64_t tokens,
                int64_t num_experts, int64_t k, int scoring, double scale, int dtype, const char *op)
{
    int rc = check_dtype(dtype, op);
    if (rc) return rc;
    if (num_experts < 1 || num_experts > spmmb::kMostExperts)
        return capi_error(SPMM_ERR_ARG, "%s: the number of experts must be in [1, %d]", op, spmmb::kMostExperts);
    if (k < 1 || k > spmmb::kMostChosen || k > num_experts)
        return capi_error(SPMM_ERR_ARG, "%s: top_k must be in [1, min(%d, number of experts)]", op, spmmb::kMostChosen);
    if (scoring != SPMM_SCORE_SOFTMAX && scoring != SPMM_SCORE_SIGMOID)
        return capi_error(SPMM_ERR_ARG, "%s: unknown scoring", op);
    if (!std::isfinite((float)scale)) return capi_error(SPMM_ERR_ARG, "%s: scale must be finite", op);
    if ((rc = check_size(tokens, num_experts, 1, op))) return rc;
    if (tokens > 0 && (!logits || !weights || !experts)) return capi_error(SPMM_ERR_ARG, "%s: null array", op);
    if (misaligned(logits) || misaligned(bias) || misaligned(weights) || misaligned(experts))
        return capi_error(SPMM_ERR_ARG, "%s: arrays must be 16-byte aligned", op);
    return SPMM_OK;
}

// Arrays of dispatch_rows, combine_rows and its backward pass; those in `opt` may be null.
int check_routed(std::initializer_list<const void *> arrays, std::initializer_list<const void *> opt, int64_t tokens,
                 int64_t k, int64_t width, int dtype, const char *op)
{
    int rc = check_dtype(dtype, op);
    if (rc) return rc;
    if ((rc = check_size(tokens, k, width, op))) return rc;
    if (k < 1) return capi_error(SPMM_ERR_ARG, "%s requires at least one choice per row", op);
    if (width < 1) return capi_error(SPMM_ERR_ARG, "%s requires a feature width of at least 1", op);
    if (tokens > INT32_MAX / k) return capi_error(SPMM_ERR_ARG, "%s: size too large", op);
    for (const void *p : arrays)
        if (tokens > 0 && !p) return capi_error(SPMM_ERR_ARG, "%s: null array", op);
    for (const auto &list : {arrays, opt})
        for (const void *p : list)
            if (misaligned(p)) return capi_error(SPMM_ERR_ARG, "%s: arrays must be 16-byte aligned", op);
    return SPMM_OK;
}

int check_embedding(const void *ids, const void *in, const void *out, int64_t n, int64_t rows, int64_t width,
                    double scale, int itype, int dtype, const char *op)
{
    int rc = check_dtype(dtype, op);
    if (rc) return rc;
    if (itype != SPMM_I32 && itype != SPMM_I64)
        return capi_error(SPMM_ERR_ARG, "%s: index arrays must be int32 or int64", op);
    if ((rc = check_size(n, width, 1, op)) || (rc = check_size(rows, width, 1, op))) return rc;
    if (width < 1) return capi_error(SPMM_ERR_ARG, "%s requires a feature width of at least 1", op);
    if (n > INT32_MAX || rows > INT32_MAX || width > (1 << 24))
        return capi_error(SPMM_ERR_ARG, "%s: size too large", op);
    if (!std::isfinite((float)scale)) return capi_error(SPMM_ERR_ARG, "%s: scale must be finite", op);
    if (n > 0 && (!ids || !in)) return capi_error(SPMM_ERR_ARG, "%s: null array", op);
    if (misaligned(in) || misaligned(out)) return capi_error(SPMM_ERR_ARG, "%s: arrays must be 16-byte aligned", op);
    return SPMM_OK;
}

int check_fp8(int64_t rows, int64_t groups, int64_t K, int64_t N, std::initializer_list<const void *> arrays,
              const char *op)
{
    int rc;
    if ((rc = check_size(rows, K, N, op)) || (rc = check_size(groups, K, N, op))) return rc;
    for (const int64_t width : {K, N}) {
        if (width <= 0) return capi_error(SPMM_ERR_ARG, "%s requires 0 < feature width", op);
        if (width % 16 != 0)
            return capi_error(SPMM_ERR_ARG,
                              "%s requires feature width divisible by 16, but got %lld. Pad and crop the tensors.", op,
                              (long long)width);
        if (width > INT32_MAX) return capi_error(SPMM_ERR_ARG, "%s: size too large", op);
    }
    if (rows > INT32_MAX || groups > (1 << 24)) return capi_error(SPMM_ERR_ARG, "%s: size too large", op);
    for (const void *p : arrays)
        if (misaligned(p)) return capi_error(SPMM_ERR_ARG, "%s: arrays must be 16-byte aligned", op);
    return SPMM_OK;
}

spmmb::DevStatus *status_or_error(const char *op, int *rc)
{
    cudaError_t e;
    spmmb::DevStatus *s = spmmb::device_status_ptr(&e);
    *rc = s ? SPMM_OK : cuda_error(e, op);
    return s;
}

}  // namespace

extern "C" {

int spmm_layer_norm_launch(const void *x, const void *weight, const void *bias, void *y, float *mean, float *rstd,
                           int64_t rows, int64_t width, double eps, int dtype, int param_dtype, void *stream)
{
    const char *op = "layer_norm";
    int rc = check_norm(x, weight, bias, y, rows, width, dtype, param_dtype, op);
    if (rc) return rc;
    if (!(eps >= 0)) return capi_error(SPMM_ERR_ARG, "%s: eps must not be negative", op);
    if (rows == 0) return SPMM_OK;
    if (!y || !mean != !rstd) return capi_error(SPMM_ERR_ARG, "%s: null array", op);
    spmmb::NormLaunch n{};
    n.x = x; n.weight = weight; n.bias = bias; n.out = y; n.mean = mean; n.rstd = rstd;
    n.rows = rows; n.width = width; n.eps = (float)eps; n.dtype = dtype; n.param_dtype = param_dtype;
    const cudaError_t e = spmmb::launch_norm_forward(n, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? SPMM_OK : cuda_error(e, op);
}

size_t spmm_layer_norm_backward_workspace_bytes(int64_t rows, int64_t width)
{
    if (rows <= 0 || width <= 0) return 0;
    return (size_t)spmmb::norm_backward_blocks(rows, width) * 2 * (size_t)width * sizeof(float);
}

int spmm_layer_norm_backward_launch(const void *grad, const void *x, const float *mean, const float *rstd,
                                    const void *weight, void *dx, void *dweight, void *dbias, int64_t rows,
                                    int64_t width, int dtype, int param_dtype, void *workspace,
                                    size_t workspace_bytes, void *stream)
{
    const char *op = "layer_norm_backward";
    int rc = check_norm(x, weight, nullptr, dx, rows, width, dtype, param_dtype, op);
    if (rc) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (rows == 0) {
        const size_t bytes = (size_t)width * elem_bytes(param_dtype);
        cudaError_t e = dweight ? cudaMemsetAsync(dweight, 0, bytes, s) : cudaSuccess;
        if (e == cudaSuccess && dbias) e = cudaMemsetAsync(dbias, 0, bytes, s);
        return e == cudaSuccess ? SPMM_OK : cuda_error(e, op);
    }
    if (!grad || !mean || !rstd) return capi_error(SPMM_ERR_ARG, "%s: null array", op);
    if (misaligned(grad)) return capi_error(SPMM_ERR_ARG, "%s: arrays must be 16-byte aligned", op);
    if (!dx && !dweight && !dbias) return SPMM_OK;
    if (dweight || dbias)
        if ((rc = check_workspace(workspace, workspace_bytes, spmm_layer_norm_backward_workspace_bytes(rows, width),
                                  op)))
            return rc;
    spmmb::NormLaunch n{};
    n.x = x; n.weight = weight; n.out = dx; n.mean = const_cast<float *>(mean); n.rstd = const_cast<float *>(rstd);
    n.rows = rows; n.width = width; n.dtype = dtype; n.param_dtype = param_dtype;
    const cudaError_t e = spmmb::launch_norm_backward(n, grad, dweight, dbias, static_cast<float *>(workspace), s);
    return e == cudaSuccess ? SPMM_OK : cuda_error(e, op);
}

size_t spmm_grouped_matmul_workspace_bytes(int64_t rows, int64_t groups, int64_t K, int64_t N, int transposed,
                                           int dtype)
{
    if (rows <= 0 || groups < 0 || K <= 0 || N <= 0) return 0;
    return spmmb::grouped_rows_workspace(rows, groups, K, N, transposed != 0, dtype);
}

int spmm_grouped_matmul_launch(const void *x, const void *weight, const void *group_ptr, void *out, int64_t rows,
                               int64_t groups, int64_t K, int64_t N, int transposed, int itype, int dtype,
                               void *workspace, size_t workspace_bytes, void *stream)
{
    const char *op = "grouped_matmul";
    int rc = check_grouped(x, weight, group_ptr, out, rows, groups, K, N, itype, dtype, op);
    if (rc || rows == 0) return rc;
    if (!out || (groups > 0 && !weight)) return capi_error(SPMM_ERR_ARG, "%s: null array", op);
    if ((rc = check_workspace(workspace, workspace_bytes,
                              spmmb::grouped_rows_workspace(rows, groups, K, N, transposed != 0, dtype), op)))
        return rc;
    cudaError_t e;
    spmmb::GroupedLaunch a{};
    a.status = spmmb::device_status_ptr(&e);
    if (!a.status) return cuda_error(e, op);
    a.x = x; a.w = weight; a.ptr = group_ptr; a.out = out; a.rows = rows; a.groups = groups; a.K = K; a.N = N;
    a.transposed = transposed != 0; a.itype = itype; a.dtype = dtype;
    e = spmmb::launch_grouped_rows(a, workspace, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? SPMM_OK : cuda_error(e, op);
}

size_t spmm_grouped_weight_grad_workspace_bytes(int64_t rows, int64_t groups, int64_t K, int64_t N, int dtype)
{
    if (rows < 0 || groups <= 0 || K <= 0 || N <= 0) return 0;
    return spmmb::grouped_weight_grad_workspace(rows, groups, K, N, dtype);
}

int spmm_grouped_weight_grad_launch(const void *x, const void *grad, const void *group_ptr, void *dweight,
                                    int64_t rows, int64_t groups, int64_t K, int64_t N, int itype, int dtype,
                                    void *workspace, size_t workspace_bytes, void *stream)
{
    const char *op = "grouped_weight_grad";
    int rc = check_grouped(x, grad, group_ptr, dweight, rows, groups, K, N, itype, dtype, op);
    if (rc || groups == 0) return rc;
    if (!dweight || (rows > 0 && !grad)) return capi_error(SPMM_ERR_ARG, "%s: null array", op);
    if ((rc = check_workspace(workspace, workspace_bytes,
                              spmmb::grouped_weight_grad_workspace(rows, groups, K, N, dtype), op)))
        return rc;
    cudaError_t e;
    spmmb::GroupedLaunch a{};
    a.status = spmmb::device_status_ptr(&e);
    if (!a.status) return cuda_error(e, op);
    a.x = x; a.w = grad; a.ptr = group_ptr; a.out = dweight; a.rows = rows; a.groups = groups; a.K = K; a.N = N;
    a.itype = itype; a.dtype = dtype;
    e = spmmb::launch_grouped_weight_grad(a, workspace, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? SPMM_OK : cuda_error(e, op);
}

size_t spmm_orthogonalize_workspace_bytes(int64_t batch, int64_t m, int64_t n, int dtype)
{
    if (batch <= 0 || m <= 0 || n <= 0) return 0;
    return spmmb::ortho_workspace(batch, m, n, dtype);
}

int spmm_orthogonalize_launch(const void *update, void *out, int64_t batch, int64_t m, int64_t n, int steps, double a,
                              double b, double c, double eps, int dtype, void *workspace, size_t workspace_bytes,
                              void *stream)
{
    const char *op = "orthogonalize";
    int rc = check_dtype(dtype, op);
    if (rc) return rc;
    if ((rc = check_size(batch, m, n, op))) return rc;
    if (m > (1 << 20) || n > (1 << 20) || batch > 65535) return capi_error(SPMM_ERR_ARG, "%s: size too large", op);
    if (steps < 0 || steps > 100) return capi_error(SPMM_ERR_ARG, "%s: steps must be in [0, 100]", op);
    if (!(eps >= 0)) return capi_error(SPMM_ERR_ARG, "%s: eps must not be negative", op);
    if (!std::isfinite((float)a) || !std::isfinite((float)b) || !std::isfinite((float)c))
        return capi_error(SPMM_ERR_ARG, "%s: coefficients must be finite", op);
    if (batch == 0 || m == 0 || n == 0) return SPMM_OK;
    if (!update || !out) return capi_error(SPMM_ERR_ARG, "%s: null array", op);
    if (misaligned(update) || misaligned(out))
        return capi_error(SPMM_ERR_ARG, "%s: arrays must be 16-byte aligned", op);
    if ((rc = check_workspace(workspace, workspace_bytes, spmmb::ortho_workspace(batch, m, n, dtype), op))) return rc;
    cudaError_t e;
    spmmb::OrthoLaunch o{};
    o.status = spmmb::device_status_ptr(&e);
    if (!o.status) return cuda_error(e, op);
    o.update = update; o.out = out; o.batch = batch; o.m = m; o.n = n; o.steps = steps;
    o.a = (float)a; o.b = (float)b; o.c = (float)c; o.eps = (float)eps; o.dtype = dtype;
    e = spmmb::launch_ortho(o, workspace, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? SPMM_OK : cuda_error(e, op);
}

int spmm_route_experts_launch(const void *logits, const float *bias, float *weights, int32_t *experts, int64_t tokens,
                              int64_t num_experts, int64_t top_k, int scoring, int64_t groups, int64_t top_groups,
                              int group_best, int renormalize, double scale, int dtype, void *stream)
{
    const char *op = "route_experts";
    int rc = check_route(logits, bias, weights, experts, tokens, num_experts, top_k, scoring, scale, dtype, op);
    if (rc) return rc;
    if (groups < 1 || groups > spmmb::kMostGroups || num_experts % groups != 0)
        return capi_error(SPMM_ERR_ARG, "%s: groups must be in [1, %d] and divide the number of experts", op,
                          spmmb::kMostGroups);
    if (top_groups < 1 || top_groups > groups)
        return capi_error(SPMM_ERR_ARG, "%s: top_groups must be in [1, groups]", op);
    if (group_best < 1 || group_best > 2 || (top_groups < groups && group_best > num_experts / groups))
        return capi_error(SPMM_ERR_ARG, "%s: group_best must be 1 or 2, and at most a group's experts", op);
    if (top_k > top_groups * (num_experts / groups))
        return capi_error(SPMM_ERR_ARG, "%s: the groups that are kept have fewer than top_k experts", op);
    if (tokens == 0) return SPMM_OK;
    spmmb::RouteLaunch r{};
    r.logits = logits; r.bias = bias; r.weights = weights; r.experts = experts; r.tokens = tokens;
    r.n = (int)num_experts; r.k = (int)top_k; r.groups = (int)groups; r.top_groups = (int)top_groups;
    r.group_best = group_best; r.sigmoid = scoring == SPMM_SCORE_SIGMOID; r.renormalize = renormalize != 0;
    r.scale = (float)scale; r.dtype = dtype;
    const cudaError_t e = spmmb::launch_route(r, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? SPMM_OK : cuda_error(e, op);
}

int spmm_route_experts_backward_launch(const void *logits, const int32_t *experts, const float *grad, void *dlogits,
                                       int64_t tokens, int64_t num_experts, int64_t top_k, int scoring,
                                       int renormalize, double scale, int dtype, void *stream)
{
    const char *op = "route_experts_backward";
    int rc = check_route(logits, dlogits, grad, experts, tokens, num_experts, top_k, scoring, scale, dtype, op);
    if (rc || tokens == 0) return rc;
    if (!dlogits) return capi_error(SPMM_ERR_ARG, "%s: null array", op);
    spmmb::DevStatus *status = status_or_error(op, &rc);
    if (rc) return rc;
    spmmb::RouteLaunch r{};
    r.logits = logits; r.experts = const_cast<int32_t *>(experts); r.tokens = tokens; r.n = (int)num_experts;
    r.k = (int)top_k; r.sigmoid = scoring == SPMM_SCORE_SIGMOID; r.renormalize = renormalize != 0;
    r.scale = (float)scale; r.dtype = dtype;
    const cudaError_t e = spmmb::launch_route_backward(r, grad, dlogits, status, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? SPMM_OK : cuda_error(e, op);
}

size_t spmm_expert_plan_workspace_bytes(int64_t n, int64_t num_experts)
{
    if (n <= 0 || num_experts <= 0 || num_experts > spmmb::kMostBuckets) return 0;
    return spmmb::bucket_workspace(n, (int)num_experts);
}

int spmm_expert_plan_launch(const void *experts, int32_t *group_ptr, int32_t *position, int32_t *source, int64_t n,
                            int64_t num_experts, int itype, void *workspace, size_t workspace_bytes, void *stream)
{
    const char *op = "expert_plan";
    if (itype != SPMM_I32 && itype != SPMM_I64)
        return capi_error(SPMM_ERR_ARG, "%s: index arrays must be int32 or int64", op);
    if (num_experts < 1 || num_experts > spmmb::kMostBuckets)
        return capi_error(SPMM_ERR_ARG, "%s: the number of experts must be in [1, %d]", op, spmmb::kMostBuckets);
    if (n < 0) return capi_error(SPMM_ERR_ARG, "%s: negative size", op);
    if (n > INT32_MAX) return capi_error(SPMM_ERR_ARG, "%s: size too large", op);
    if (!group_ptr || (n > 0 && (!experts || !position || !source)))
        return capi_error(SPMM_ERR_ARG, "%s: null array", op);
    int rc = check_workspace(workspace, workspace_bytes, spmm_expert_plan_workspace_bytes(n, num_experts), op);
    if (rc) return rc;
    spmmb::BucketPasses sort{};
    sort.passes = 1;
    spmmb::BucketSort &b = sort.pass[0];
    b.status = status_or_error(op, &rc);
    if (rc) return rc;
    b.keys = experts; b.wide = itype == SPMM_I64; b.n = n; b.buckets = (int)num_experts; b.mask = -1;
    b.limit = num_experts; b.skip = -1; b.ptr = group_ptr; b.position = position; b.order = source;
    b.counts = static_cast<int *>(workspace);
    const cudaError_t e = spmmb::launch_bucket_sort(sort, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? SPMM_OK : cuda_error(e, op);
}

int spmm_dispatch_rows_launch(const void *x, const int32_t *position, const int32_t *source, void *rows, int64_t tokens,
                              int64_t k, int64_t width, int dtype, void *stream)
{
    const char *op = "dispatch_rows";
    int rc = check_routed({x, position, source, rows}, {}, tokens, k, width, dtype, op);
    if (rc || tokens == 0) return rc;
    spmmb::RoutedLaunch r{};
    r.status = status_or_error(op, &rc);
    if (rc) return rc;
    r.x = x; r.position = position; r.source = source; r.out = rows; r.tokens = tokens; r.k = (int)k; r.width = width;
    r.dtype = dtype;
    const cudaError_t e = spmmb::launch_dispatch(r, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? SPMM_OK : cuda_error(e, op);
}

int spmm_combine_rows_launch(const void *rows, const int32_t *position, const float *weights, void *y, int64_t tokens,
                             int64_t k, int64_t width, int dtype, void *stream)
{
    const char *op = "combine_rows";
    int rc = check_routed({rows, position, y}, {weights}, tokens, k, width, dtype, op);
    if (rc || tokens == 0) return rc;
    spmmb::RoutedLaunch r{};
    r.status = status_or_error(op, &rc);
    if (rc) return rc;
    r.x = rows; r.position = position; r.weights = weights; r.out = y; r.tokens = tokens; r.k = (int)k; r.width = width;
    r.dtype = dtype;
    const cudaError_t e = spmmb::launch_combine(r, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? SPMM_OK : cuda_error(e, op);
}

int spmm_combine_rows_backward_launch(const void *grad, const void *rows, const int32_t *position,
                                      const int32_t *source, const float *weights, void *drows, float *dweights,
                                      int64_t tokens, int64_t k, int64_t width, int dtype, void *stream)
{
    const char *op = "combine_rows_backward";
    int rc = check_routed({grad, position, source}, {rows, weights, drows, dweights}, tokens, k, width, dtype, op);
    if (rc || tokens == 0 || (!drows && !dweights)) return rc;
    if (dweights && !rows) return capi_error(SPMM_ERR_ARG, "%s: null array", op);
    spmmb::RoutedLaunch r{};
    r.status = status_or_error(op, &rc);
    if (rc) return rc;
    r.x = rows; r.grad = grad; r.position = position; r.source = source; r.weights = weights; r.out = drows;
    r.dweights = dweights; r.tokens = tokens; r.k = (int)k; r.width = width; r.dtype = dtype;
    const cudaError_t e = spmmb::launch_combine_backward(r, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? SPMM_OK : cuda_error(e, op);
}

int spmm_embedding_launch(const void *ids, const void *table, void *y, int64_t n, int64_t rows, int64_t width,
                          double scale, int itype, int dtype, void *stream)
{
    const char *op = "embedding";
    int rc = check_embedding(ids, table, y, n, rows, width, scale, itype, dtype, op);
    if (rc || n == 0) return rc;
    if (!y) return capi_error(SPMM_ERR_ARG, "%s: null array", op);
    spmmb::EmbeddingLaunch l{};
    l.status = status_or_error(op, &rc);
    if (rc) return rc;
    l.ids = ids; l.in = table; l.out = y; l.n = n; l.rows = rows; l.width = width; l.scale = (float)scale;
    l.itype = itype; l.dtype = dtype;
    const cudaError_t e = spmmb::launch_embedding(l, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? SPMM_OK : cuda_error(e, op);
}

size_t spmm_embedding_backward_workspace_bytes(int64_t n, int64_t width)
{
    if (n <= 0 || width <= 0) return 0;
    return spmmb::embedding_backward_workspace(n, width);
}

int spmm_embedding_backward_launch(const void *ids, const void *grad, void *dtable, int64_t n, int64_t rows,
                                   int64_t width, double scale, int64_t padding_id, int itype, int dtype,
                                   void *workspace, size_t workspace_bytes, void *stream)
{
    const char *op = "embedding_backward";
    int rc = check_embedding(ids, grad, dtable, n, rows, width, scale, itype, dtype, op);
    if (rc) return rc;
    if (rows > 0 && !dtable) return capi_error(SPMM_ERR_ARG, "%s: null array", op);
    if ((rc = check_workspace(workspace, workspace_bytes, spmm_embedding_backward_workspace_bytes(n, width), op)))
        return rc;
    spmmb::EmbeddingLaunch l{};
    l.status = status_or_error(op, &rc);
    if (rc) return rc;
    l.ids = ids; l.in = grad; l.out = dtable; l.n = n; l.rows = rows; l.width = width; l.scale = (float)scale;
    l.itype = itype; l.dtype = dtype;
    const cudaError_t e = spmmb::launch_embedding_backward(l, padding_id < 0 ? INT64_MIN : padding_id, workspace,
                                                           static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? SPMM_OK : cuda_error(e, op);
}

int spmm_quantize_fp8_launch(const void *x, void *q, float *scale, int64_t rows, int64_t width, int dtype, void *stream)
{
    const char *op = "quantize_fp8";
    int rc = check_dtype(dtype, op);
    if (rc || (rc = check_fp8(rows, 1, width, 16, {x, q}, op)) || rows == 0) return rc;
    if (!x || !q || !scale) return capi_error(SPMM_ERR_ARG, "%s: null array", op);
    const cudaError_t e = spmmb::launch_quantize_rows(x, q, scale, rows, width, dtype, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? SPMM_OK : cuda_error(e, op);
}

int spmm_quantize_weight_fp8_launch(const void *weight, void *q, float *scale, int64_t groups, int64_t K, int64_t N,
                                    int dtype, void *stream)
{
    const char *op = "quantize_weight_fp8";
    int rc = check_dtype(dtype, op);
    if (rc || (rc = check_fp8(1, groups, K, N, {weight, q}, op)) || groups == 0) return rc;
    if (!weight || !q || !scale) return capi_error(SPMM_ERR_ARG, "%s: null array", op);
    const cudaError_t e =
        spmmb::launch_quantize_weight(weight, q, scale, groups, K, N, dtype, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? SPMM_OK : cuda_error(e, op);
}

int spmm_grouped_matmul_fp8_launch(const void *x, const float *x_scale, const void *weight, const float *weight_scale,
                                   const void *group_ptr, void *out, int64_t rows, int64_t groups, int64_t K, int64_t N,
                                   int itype, int out_dtype, void *stream)
{
    const char *op = "grouped_matmul_fp8";
    int rc = check_dtype(out_dtype, op);
    if (rc || (rc = check_fp8(rows, groups, K, N, {x, weight, out}, op))) return rc;
    if (itype != SPMM_I32 && itype != SPMM_I64)
        return capi_error(SPMM_ERR_ARG, "%s: index arrays must be int32 or int64", op);
    if (rows == 0) return SPMM_OK;
    if (!x || !x_scale || !out || !group_ptr || (groups > 0 && (!weight || !weight_scale)))
        return capi_error(SPMM_ERR_ARG, "%s: null array", op);
    spmmb::Fp8Launch a{};
    a.status = status_or_error(op, &rc);
    if (rc) return rc;
    a.x = x; a.x_scale = x_scale; a.w = weight; a.w_scale = weight_scale; a.ptr = group_ptr; a.out = out;
    a.rows = rows; a.groups = groups; a.K = K; a.N = N; a.itype = itype; a.out_dtype = out_dtype;
    const cudaError_t e = spmmb::launch_grouped_fp8(a, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? SPMM_OK : cuda_error(e, op);
}

}  // extern "C"
