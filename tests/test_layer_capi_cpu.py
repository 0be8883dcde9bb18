"""CPU checks of the layer operators' entry points: contract violations are
refused on the host with a message, sizes of zero return before any launch,
workspace queries answer without a device."""

import ctypes

import pytest
import torch

V, I64, INT, SZ, F64 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_size_t, ctypes.c_double
F16, F32, FP64, BF16 = 0, 1, 2, 3
PTR = 4096   # an aligned address that is never read


@pytest.fixture(scope="module")
def lib():
    import build

    build.build()
    L = ctypes.CDLL(str(build.LIB))
    L.spmm_last_error.restype = ctypes.c_char_p
    L.spmm_layer_norm_launch.argtypes = [V] * 6 + [I64, I64, F64, INT, INT, V]
    L.spmm_layer_norm_backward_workspace_bytes.restype = SZ
    L.spmm_layer_norm_backward_workspace_bytes.argtypes = [I64, I64]
    L.spmm_layer_norm_backward_launch.argtypes = [V] * 8 + [I64, I64, INT, INT, V, SZ, V]
    L.spmm_grouped_matmul_launch.argtypes = [V] * 4 + [I64] * 4 + [INT] * 3 + [V, SZ, V]
    L.spmm_grouped_matmul_workspace_bytes.restype = SZ
    L.spmm_grouped_matmul_workspace_bytes.argtypes = [I64] * 4 + [INT] * 2
    L.spmm_grouped_weight_grad_launch.argtypes = [V] * 4 + [I64] * 4 + [INT] * 2 + [V, SZ, V]
    L.spmm_grouped_weight_grad_workspace_bytes.restype = SZ
    L.spmm_grouped_weight_grad_workspace_bytes.argtypes = [I64] * 4 + [INT]
    L.spmm_orthogonalize_launch.argtypes = [V, V] + [I64] * 3 + [INT] + [F64] * 4 + [INT, V, SZ, V]
    L.spmm_orthogonalize_workspace_bytes.restype = SZ
    L.spmm_orthogonalize_workspace_bytes.argtypes = [I64] * 3 + [INT]
    return L


def refused(lib, rc, text):
    assert rc == 1 and text in lib.spmm_last_error().decode(), (rc, lib.spmm_last_error())


def test_layer_norm(lib):
    f = lambda **k: lib.spmm_layer_norm_launch(  # noqa: E731
        k.get("x", PTR), None, None, k.get("y", PTR), k.get("mean"), None, k.get("rows", 4), k.get("width", 32),
        k.get("eps", 1e-5), k.get("dtype", F16), k.get("params", F16), None)
    refused(lib, f(dtype=FP64), "supports only FP16, BF16 and FP32")
    refused(lib, f(dtype=7), "supports only FP16, BF16 and FP32")
    refused(lib, f(params=BF16), "dtype of x or FP32")
    refused(lib, f(dtype=F32, params=F16), "dtype of x or FP32")
    refused(lib, f(rows=-1), "negative size")
    refused(lib, f(width=0), "at least 1")
    refused(lib, f(x=None), "null array")
    refused(lib, f(y=None), "null array")
    refused(lib, f(mean=PTR), "null array")
    refused(lib, f(x=PTR + 2), "16-byte aligned")
    refused(lib, f(eps=-1.0), "eps must not be negative")
    refused(lib, f(eps=float("nan")), "eps must not be negative")
    refused(lib, f(rows=1 << 60), "size too large")
    assert f(rows=0) == 0
    assert lib.spmm_layer_norm_backward_workspace_bytes(0, 64) == 0
    need = lib.spmm_layer_norm_backward_workspace_bytes(1000, 64)
    assert need >= 2 * 64 * 4
    g = lambda ws, n, dw=PTR: lib.spmm_layer_norm_backward_launch(  # noqa: E731
        PTR, PTR, PTR, PTR, None, PTR, dw, PTR, 1000, 64, F16, F16, ws, n, None)
    assert g(PTR, need - 1) == 6 and g(None, need) == 6
    refused(lib, g(PTR + 4, need), "16-byte aligned")


def test_grouped(lib):
    f = lambda **k: lib.spmm_grouped_matmul_launch(  # noqa: E731
        k.get("x", PTR), k.get("w", PTR), k.get("ptr", PTR), k.get("out", PTR), k.get("rows", 4), k.get("groups", 2),
        k.get("K", 32), k.get("N", 32), 0, k.get("itype", 0), k.get("dtype", F16), None, 0, None)
    refused(lib, f(dtype=FP64), "supports only FP16, BF16 and FP32")
    refused(lib, f(itype=2), "int32 or int64")
    refused(lib, f(K=24), "divisible by 16, but got 24")
    refused(lib, f(N=8, dtype=BF16), "divisible by 16, but got 8")
    refused(lib, f(N=12, dtype=F32), "divisible by 8, but got 12")
    refused(lib, f(K=0), "0 < feature width")
    refused(lib, f(rows=-1), "negative size")
    refused(lib, f(groups=-1), "negative size")
    refused(lib, f(rows=1 << 40), "size too large")
    refused(lib, f(ptr=None), "null array")
    refused(lib, f(x=None), "null array")
    refused(lib, f(w=None), "null array")
    refused(lib, f(out=None), "null array")
    refused(lib, f(w=PTR + 8), "16-byte aligned")
    assert f(rows=0) == 0
    g = lambda **k: lib.spmm_grouped_weight_grad_launch(  # noqa: E731
        PTR, k.get("grad", PTR), PTR, k.get("out", PTR), k.get("rows", 4), k.get("groups", 2), k.get("K", 32), 32, 0,
        k.get("dtype", F16), None, 0, None)
    refused(lib, g(K=40), "divisible by 16, but got 40")
    refused(lib, g(grad=None), "null array")
    refused(lib, g(out=None), "null array")
    assert g(groups=0) == 0


def test_orthogonalize(lib):
    f = lambda **k: lib.spmm_orthogonalize_launch(  # noqa: E731
        k.get("u", PTR), PTR, k.get("batch", 1), k.get("m", 8), 8, k.get("steps", 5), k.get("a", 3.4), -4.7, 2.0,
        k.get("eps", 1e-7), k.get("dtype", F32), None, 0, None)
    refused(lib, f(dtype=FP64), "supports only FP16, BF16 and FP32")
    refused(lib, f(steps=-1), "steps must be")
    refused(lib, f(steps=101), "steps must be")
    refused(lib, f(a=float("inf")), "finite")
    refused(lib, f(eps=-1e-9), "eps must not be negative")
    refused(lib, f(m=-1), "negative size")
    refused(lib, f(m=1 << 40), "size too large")
    refused(lib, f(u=None), "null array")
    assert f() == 6 and "workspace" in lib.spmm_last_error().decode()
    assert f(batch=0) == 0 and f(m=0) == 0
    assert lib.spmm_orthogonalize_workspace_bytes(0, 8, 8, F32) == 0
    assert lib.spmm_orthogonalize_workspace_bytes(2, 300, 200, F16) > 0


def test_python_operators_refuse_cpu_tensors(lib):
    import spmm_npu

    for name in ("grouped_matmul", "grouped_weight_grad", "layer_norm", "layer_norm_backward", "layer_norm_forward",
                 "orthogonalize"):
        assert name in spmm_npu.__all__
    x = torch.zeros(4, 32)
    ptr = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: spmm_npu.layer_norm(x), lambda: spmm_npu.grouped_matmul(x, torch.zeros(1, 32, 16), ptr),
                 lambda: spmm_npu.grouped_weight_grad(x, x, ptr), lambda: spmm_npu.orthogonalize(x)):
        with pytest.raises(RuntimeError, match="must be CUDA tensor"):
            call()
