"""CPU checks of the entry points around routed experts, embeddings and 8-bit
products: contract violations are refused on the host with a message, sizes of
zero return before any launch."""

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
    L.spmm_route_experts_launch.argtypes = [V] * 4 + [I64] * 3 + [INT] + [I64] * 2 + [INT] * 2 + [F64, INT, V]
    L.spmm_route_experts_backward_launch.argtypes = [V] * 4 + [I64] * 3 + [INT] * 2 + [F64, INT, V]
    L.spmm_expert_plan_workspace_bytes.restype = SZ
    L.spmm_expert_plan_workspace_bytes.argtypes = [I64] * 2
    L.spmm_expert_plan_launch.argtypes = [V] * 4 + [I64] * 2 + [INT, V, SZ, V]
    L.spmm_dispatch_rows_launch.argtypes = [V] * 4 + [I64] * 3 + [INT, V]
    L.spmm_combine_rows_launch.argtypes = [V] * 4 + [I64] * 3 + [INT, V]
    L.spmm_combine_rows_backward_launch.argtypes = [V] * 7 + [I64] * 3 + [INT, V]
    L.spmm_embedding_launch.argtypes = [V] * 3 + [I64] * 3 + [F64, INT, INT, V]
    L.spmm_embedding_backward_workspace_bytes.restype = SZ
    L.spmm_embedding_backward_workspace_bytes.argtypes = [I64] * 2
    L.spmm_embedding_backward_launch.argtypes = [V] * 3 + [I64] * 3 + [F64, I64, INT, INT, V, SZ, V]
    L.spmm_quantize_fp8_launch.argtypes = [V] * 3 + [I64] * 2 + [INT, V]
    L.spmm_quantize_weight_fp8_launch.argtypes = [V] * 3 + [I64] * 3 + [INT, V]
    L.spmm_grouped_matmul_fp8_launch.argtypes = [V] * 6 + [I64] * 4 + [INT, INT, V]
    return L


def refused(lib, rc, text):
    assert rc == 1 and text in lib.spmm_last_error().decode(), (rc, lib.spmm_last_error())


def test_route_experts(lib):
    f = lambda **k: lib.spmm_route_experts_launch(  # noqa: E731
        k.get("x", PTR), k.get("bias"), k.get("w", PTR), k.get("e", PTR), k.get("tokens", 4), k.get("n", 12), k.get("k", 2),
        k.get("scoring", 0), k.get("groups", 1), k.get("top_groups", 1), k.get("best", 1), 1, k.get("scale", 1.0),
        k.get("dtype", F32), None)
    refused(lib, f(dtype=FP64), "supports only FP16, BF16 and FP32")
    refused(lib, f(n=0), "number of experts must be in [1, 1024]")
    refused(lib, f(n=1025), "number of experts must be in [1, 1024]")
    refused(lib, f(k=0), "top_k must be in")
    refused(lib, f(k=13), "top_k must be in")
    refused(lib, f(n=100, k=33), "top_k must be in")
    refused(lib, f(scoring=2), "unknown scoring")
    refused(lib, f(scale=float("inf")), "scale must be finite")
    refused(lib, f(scale=1e300), "scale must be finite")
    refused(lib, f(tokens=-1), "negative size")
    refused(lib, f(tokens=1 << 60), "size too large")
    refused(lib, f(groups=0), "divide the number of experts")
    refused(lib, f(groups=5), "divide the number of experts")
    refused(lib, f(n=66, groups=33), "groups must be in [1, 32]")
    refused(lib, f(groups=3, top_groups=0), "top_groups must be")
    refused(lib, f(groups=3, top_groups=4), "top_groups must be")
    refused(lib, f(groups=12, top_groups=6, best=2), "group_best must be")
    refused(lib, f(groups=3, top_groups=2, best=0), "group_best must be")
    refused(lib, f(groups=6, top_groups=1, k=3), "fewer than top_k experts")
    refused(lib, f(x=None), "null array")
    refused(lib, f(w=None), "null array")
    refused(lib, f(e=None), "null array")
    refused(lib, f(x=PTR + 2), "16-byte aligned")
    refused(lib, f(bias=PTR + 4), "16-byte aligned")
    assert f(tokens=0, x=None, w=None, e=None) == 0
    g = lambda **k: lib.spmm_route_experts_backward_launch(  # noqa: E731
        PTR, PTR, k.get("grad", PTR), k.get("dx", PTR), k.get("tokens", 4), 12, k.get("k", 2), 0, 1, 1.0, F32, None)
    refused(lib, g(grad=None), "null array")
    refused(lib, g(dx=None), "null array")
    refused(lib, g(k=40), "top_k must be in")
    assert g(tokens=0) == 0


def test_expert_plan(lib):
    f = lambda **k: lib.spmm_expert_plan_launch(  # noqa: E731
        k.get("e", PTR), k.get("ptr", PTR), PTR, k.get("s", PTR), k.get("n", 8), k.get("num", 4), k.get("itype", 0), k.get("ws"), k.get("bytes", 0), None)
    refused(lib, f(itype=2), "int32 or int64")
    refused(lib, f(num=0), "number of experts must be in [1, 1024]")
    refused(lib, f(num=1025), "number of experts must be in [1, 1024]")
    refused(lib, f(n=-1), "negative size")
    refused(lib, f(n=1 << 31), "size too large")
    refused(lib, f(e=None), "null array")
    refused(lib, f(s=None), "null array")
    refused(lib, f(ptr=None, n=0), "null array")
    assert lib.spmm_expert_plan_workspace_bytes(0, 4) == 0
    need = lib.spmm_expert_plan_workspace_bytes(1 << 20, 64)
    assert need > 0 and f(n=1 << 20, num=64, ws=PTR, bytes=need - 1) == 6 and f(n=1 << 20, num=64, bytes=need) == 6
    refused(lib, f(n=1 << 20, num=64, ws=PTR + 8, bytes=need), "16-byte aligned")


def test_rows(lib):
    d = lambda **k: lib.spmm_dispatch_rows_launch(  # noqa: E731
        k.get("x", PTR), PTR, k.get("s", PTR), PTR, k.get("tokens", 4), k.get("k", 2), k.get("width", 8), k.get("dtype", F16), None)
    refused(lib, d(dtype=FP64), "supports only FP16, BF16 and FP32")
    refused(lib, d(k=0), "at least one choice")
    refused(lib, d(width=0), "feature width of at least 1")
    refused(lib, d(tokens=-1), "negative size")
    refused(lib, d(tokens=1 << 30), "size too large")
    refused(lib, d(x=None), "null array")
    refused(lib, d(s=None), "null array")
    refused(lib, d(x=PTR + 8), "16-byte aligned")
    assert d(tokens=0) == 0
    c = lambda **k: lib.spmm_combine_rows_launch(PTR, k.get("p", PTR), k.get("w"), k.get("y", PTR), 4, 2, 8, F16, None)  # noqa: E731
    refused(lib, c(p=None), "null array")
    refused(lib, c(y=None), "null array")
    refused(lib, c(w=PTR + 4), "16-byte aligned")
    b = lambda **k: lib.spmm_combine_rows_backward_launch(  # noqa: E731
        k.get("dy", PTR), k.get("rows", PTR), PTR, PTR, None, k.get("dr", PTR), k.get("dw", PTR), k.get("tokens", 4), 2, 8, F16, None)
    refused(lib, b(dy=None), "null array")
    refused(lib, b(rows=None), "null array")
    refused(lib, b(dr=PTR + 2), "16-byte aligned")
    assert b(dr=None, dw=None) == 0 and b(tokens=0) == 0


def test_embedding(lib):
    f = lambda **k: lib.spmm_embedding_launch(  # noqa: E731
        k.get("ids", PTR), PTR, k.get("y", PTR), k.get("n", 4), k.get("rows", 9), k.get("width", 8), k.get("scale", 1.0),
        k.get("itype", 0), k.get("dtype", F16), None)
    refused(lib, f(dtype=FP64), "supports only FP16, BF16 and FP32")
    refused(lib, f(itype=3), "int32 or int64")
    refused(lib, f(n=-1), "negative size")
    refused(lib, f(rows=-1), "negative size")
    refused(lib, f(n=1 << 31), "size too large")
    refused(lib, f(width=0), "feature width of at least 1")
    refused(lib, f(scale=float("nan")), "scale must be finite")
    refused(lib, f(ids=None), "null array")
    refused(lib, f(y=None), "null array")
    refused(lib, f(y=PTR + 4), "16-byte aligned")
    assert f(n=0) == 0
    assert lib.spmm_embedding_backward_workspace_bytes(0, 8) == 0
    need = lib.spmm_embedding_backward_workspace_bytes(1000, 64)
    assert need >= 2 * 4 * 1000
    g = lambda ws, n, **k: lib.spmm_embedding_backward_launch(  # noqa: E731
        PTR, k.get("dy", PTR), k.get("d", PTR), 1000, 50, 64, 1.0, -1, 0, F16, ws, n, None)
    assert g(PTR, need - 1) == 6 and g(None, need) == 6
    refused(lib, g(PTR + 4, need), "16-byte aligned")
    refused(lib, g(PTR, need, dy=None), "null array")
    refused(lib, g(PTR, need, d=None), "null array")


def test_fp8(lib):
    q = lambda **k: lib.spmm_quantize_fp8_launch(  # noqa: E731
        k.get("x", PTR), PTR, k.get("s", PTR), k.get("rows", 4), k.get("width", 32), k.get("dtype", F16), None)
    refused(lib, q(dtype=FP64), "supports only FP16, BF16 and FP32")
    refused(lib, q(width=24), "divisible by 16, but got 24")
    refused(lib, q(width=0), "0 < feature width")
    refused(lib, q(rows=-1), "negative size")
    refused(lib, q(x=None), "null array")
    refused(lib, q(s=None), "null array")
    refused(lib, q(x=PTR + 8), "16-byte aligned")
    assert q(rows=0) == 0
    w = lambda **k: lib.spmm_quantize_weight_fp8_launch(PTR, PTR, k.get("s", PTR), k.get("groups", 2), k.get("K", 32), 48, F16, None)  # noqa: E731
    refused(lib, w(K=8), "divisible by 16, but got 8")
    refused(lib, w(s=None), "null array")
    assert w(groups=0) == 0
    f = lambda **k: lib.spmm_grouped_matmul_fp8_launch(  # noqa: E731
        k.get("x", PTR), k.get("xs", PTR), k.get("w", PTR), PTR, k.get("ptr", PTR), k.get("out", PTR), k.get("rows", 4),
        k.get("groups", 2), k.get("K", 32), k.get("N", 48), k.get("itype", 0), k.get("dtype", BF16), None)
    refused(lib, f(dtype=FP64), "supports only FP16, BF16 and FP32")
    refused(lib, f(itype=5), "int32 or int64")
    refused(lib, f(K=40), "divisible by 16, but got 40")
    refused(lib, f(N=8), "divisible by 16, but got 8")
    refused(lib, f(rows=1 << 40), "size too large")
    refused(lib, f(groups=-1), "negative size")
    refused(lib, f(xs=None), "null array")
    refused(lib, f(w=None), "null array")
    refused(lib, f(ptr=None), "null array")
    refused(lib, f(out=None), "null array")
    refused(lib, f(w=PTR + 8), "16-byte aligned")
    assert f(rows=0) == 0


def test_python_operators_refuse_cpu_tensors(lib):
    import spmm_npu

    x, i = torch.zeros(4, 32), torch.zeros(4, 2, dtype=torch.int32)
    calls = {"route_experts": lambda: spmm_npu.route_experts(x, 2), "expert_plan": lambda: spmm_npu.expert_plan(i, 4),
             "dispatch_rows": lambda: spmm_npu.dispatch_rows(x, i, i.view(-1)),
             "combine_rows": lambda: spmm_npu.combine_rows(x, i, i.view(-1)),
             "embedding": lambda: spmm_npu.embedding(i, x), "embedding_grad": lambda: spmm_npu.embedding_grad(i, torch.zeros(4, 2, 8), 4),
             "quantize_fp8": lambda: spmm_npu.quantize_fp8(x), "quantize_weight_fp8": lambda: spmm_npu.quantize_weight_fp8(x[None]),
             "grouped_matmul_fp8": lambda: spmm_npu.grouped_matmul_fp8(x, x, x, x, i)}
    for name, call in calls.items():
        assert name in spmm_npu.__all__
        with pytest.raises(RuntimeError, match="must be CUDA tensor"):
            call()
