// extern "C" entry points of the layer operators (declared in
// include/spmm_b200.h): argument contract, workspace check and launch.
#include <cmath>
#include <cstdint>

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

}  // extern "C"
