"""layer_norm on the GPU against its definition in 64 bits: every team shape
(widths from one element to rows wider than a block's registers, rows that
start at any element), the gradients against the formula and against
differences, types, row counts, constant and extreme rows, refusals."""

import pytest
import torch

from layer_reference import assert_within, norm_reference

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def lib():
    import build

    build.build()
    import spmm_npu

    return spmm_npu


def make(rows, width, dtype, params, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x = (n(rows, width) * torch.exp(0.5 * n(rows, 1)) + n(rows, 1)).to(dtype)
    return x, (1 + 0.3 * n(width)).to(params), (0.3 * n(width)).to(params), n(rows, width).to(dtype)


def check(lib, x, w, b, grad, eps=1e-5):
    y = lib.layer_norm(x, w, b, eps)
    leaves = [t.detach().clone().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    yt = lib.layer_norm(*leaves, eps)
    assert torch.equal(y, yt)
    got = torch.autograd.grad(yt, [t for t in leaves if t is not None], grad)
    (ry, sy), (rdx, sdx), (rdw, sdw), (rdb, sdb) = norm_reference(x, w, b, eps, grad)
    assert_within(y, ry, sy, "y")
    assert_within(got[0], rdx, sdx, "dx")
    if w is not None:
        assert got[1].dtype == w.dtype
        assert_within(got[1], rdw, sdw, "dweight")
    if b is not None:
        assert got[-1].dtype == b.dtype
        assert_within(got[-1], rdb, sdb, "dbias")


@pytest.mark.parametrize("dtype,params", [(F16, F16), (BF16, F32), (F32, F32)])
@pytest.mark.parametrize("width", [1, 2, 7, 16, 31, 33, 64, 100, 129, 256, 264, 500, 512, 1001, 1024, 1025, 2048, 2056,
                                   4000, 4097, 8192, 8200, 16384, 16392, 33000])
def test_every_width(lib, width, dtype, params):
    check(lib, *make(37, width, dtype, params, seed=width))


@pytest.mark.parametrize("dtype,params", [(F16, F32), (BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("rows", [1, 2, 15, 17, 1000, 20011])
def test_row_counts(lib, rows, dtype, params):
    for width in (48, 200, 1024):
        check(lib, *make(rows, width, dtype, params, seed=rows))


def test_without_parameters(lib):
    x, w, b, grad = make(65, 96, F32, F32)
    check(lib, x, None, None, grad)
    check(lib, x, w, None, grad)
    check(lib, x, None, b, grad)


def test_gradient_against_differences(lib):
    """Central differences of sum(grad * y) along random directions, in 64 bits
    on the definition; the kernel's gradients give the same slopes."""
    x, w, b, grad = make(11, 40, F32, F32, seed=4)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    got = torch.autograd.grad(lib.layer_norm(*leaves), leaves, grad)
    g = torch.Generator(device="cuda").manual_seed(5)
    f = lambda *p: float((norm_reference(*p, 1e-5)[0][0] * grad.double()).sum())  # noqa: E731
    at = [t.double() for t in (x, w, b)]
    for k in range(3):
        d = torch.randn(at[k].shape, generator=g, device="cuda", dtype=torch.float64)
        h = 1e-6
        hi, lo = [list(at) for _ in range(2)]
        hi[k], lo[k] = at[k] + h * d, at[k] - h * d
        slope = (f(*hi) - f(*lo)) / (2 * h)
        # differences: h^2 times a third derivative of order 10; fp32 gradients: 1e-6 of their magnitudes
        scale = float((got[k].double().abs() * d.abs()).sum())
        assert abs(float((got[k].double() * d).sum()) - slope) <= 1e-5 * scale + 1e-6


@pytest.mark.parametrize("dtype", [F16, F32])
def test_constant_rows_and_large_means(lib, dtype):
    # zero variance: y is the bias, dx has the factor 1 / sqrt(eps)
    x = torch.full((5, 128), 3.0, device="cuda", dtype=dtype)
    b = torch.randn(128, device="cuda").to(dtype)
    assert torch.equal(lib.layer_norm(x, None, b), b.expand(5, 128))
    # a mean a thousand times the spread: E[x^2] - E[x]^2 in fp32 would lose the variance
    g = torch.Generator(device="cuda").manual_seed(1)
    x = (1000 + torch.randn(9, 512, generator=g, device="cuda")).to(dtype)
    (ry, sy), = norm_reference(x, None, None, 1e-5)
    assert_within(lib.layer_norm(x), ry, sy)


def test_non_finite_rows_stay_alone(lib):
    x, w, b, grad = make(40, 264, F16, F16)
    good = lib.layer_norm(x, w, b)
    x2 = x.clone()
    x2[3, 7], x2[20, 0] = float("nan"), float("inf")
    y = lib.layer_norm(x2, w, b)
    keep = torch.ones(40, dtype=torch.bool, device="cuda")
    keep[[3, 20]] = False
    assert torch.equal(y[keep], good[keep]) and bool(y[3].isnan().all()) and bool(y[20].isnan().all())


def test_shapes_strides_and_views(lib):
    x, w, b, grad = make(24, 96, F32, F32)
    want = lib.layer_norm(x, w, b)
    assert torch.equal(lib.layer_norm(x.view(2, 3, 4, 96), w, b).view(24, 96), want)
    wide = torch.zeros(24, 200, device="cuda")
    wide[:, 50:146] = x
    assert torch.equal(lib.layer_norm(wide[:, 50:146], w, b), want)
    assert torch.equal(lib.layer_norm(x.t().contiguous().t(), w, b), want)
    odd = torch.zeros(24 * 96 + 1, device="cuda")
    odd[1:] = x.reshape(-1)
    assert torch.equal(lib.layer_norm(odd[1:].view(24, 96), w, b), want)
    # an expanded gradient (sum of the outputs)
    leaf = x.clone().requires_grad_(True)
    lib.layer_norm(leaf, w, b).sum().backward()
    ref = norm_reference(x, w, b, 1e-5, torch.ones_like(x))[1]
    assert_within(leaf.grad, *ref, "dx of a sum")


def test_empty(lib):
    w = torch.ones(32, device="cuda", requires_grad=True)
    x = torch.zeros(0, 32, device="cuda", requires_grad=True)
    y = lib.layer_norm(x, w)
    assert y.shape == (0, 32)
    dx, dw = torch.autograd.grad(y, [x, w], torch.zeros(0, 32, device="cuda"))
    assert dx.shape == (0, 32) and not bool(dw.any())


def test_only_wanted_gradients(lib):
    x, w, b, grad = make(70, 136, BF16, F32)
    y, mean, rstd = lib.layer_norm_forward(x, w, b, 1e-5, True)
    full = lib.layer_norm_backward(grad, x, mean, rstd, w)
    for k in range(3):
        want = [i == k for i in range(3)]
        part = lib.layer_norm_backward(grad, x, mean, rstd, w, *want, True)
        assert [p is not None for p in part] == want
        assert torch.equal(part[k], full[k]) if k < 2 else torch.equal(part[2].float(), full[2].float())


def test_same_result_twice_and_on_another_stream(lib):
    x, w, b, grad = make(5000, 1024, F16, F32)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    run = lambda: torch.autograd.grad(lib.layer_norm(*leaves), leaves, grad)  # noqa: E731
    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(first, second))


def test_graph_capture(lib):
    x, w, b, _ = make(33, 256, F16, F16)
    want = lib.layer_norm(x, w, b)
    graph = torch.cuda.CUDAGraph()
    static = torch.zeros_like(x)
    with torch.cuda.graph(graph):
        y = lib.layer_norm(static, w, b)
    static.copy_(x)
    graph.replay()
    assert torch.equal(y, want)


def test_offsets_beyond_32_bits(lib):
    """2.2 M rows of 1024 features: element offsets pass 2^31."""
    rows, width = (1 << 21) + 70001, 1024
    x = torch.zeros(rows, width, dtype=F16, device="cuda")
    tail, w, b, grad = make(64, width, F16, F16, seed=3)
    x[-64:] = tail
    y = lib.layer_norm(x, w, b)
    (ry, sy), = norm_reference(tail, w, b, 1e-5)
    assert_within(y[-64:], ry, sy)
    assert torch.equal(y[: 1 << 10], b.expand(1 << 10, width))
    y, mean, rstd = lib.layer_norm_forward(x, w, b, 1e-5, True)
    full = torch.zeros_like(x)
    full[-64:] = grad
    dx, dw, db = lib.layer_norm_backward(full, x, mean, rstd, w)
    _, (rdx, sdx), (rdw, sdw), (rdb, sdb) = norm_reference(tail, w, b, 1e-5, grad)
    assert_within(dx[-64:], rdx, sdx)
    assert_within(dw, rdw, sdw)
    assert_within(db, rdb, sdb)


def test_refusals(lib):
    x, w, b, grad = make(4, 32, F16, F16)
    with pytest.raises(RuntimeError, match="must be CUDA tensor"):
        lib.layer_norm(x.cpu())
    with pytest.raises(RuntimeError, match="supports only FP16, BF16 and FP32"):
        lib.layer_norm(x.double())
    with pytest.raises(RuntimeError, match="must have shape"):
        lib.layer_norm(x, w[:16])
    with pytest.raises(RuntimeError, match="dtype of x or FP32"):
        lib.layer_norm(x, w.bfloat16())
    with pytest.raises(RuntimeError, match="same dtype"):
        lib.layer_norm(x, w, b.float())
    with pytest.raises(RuntimeError, match="eps must not be negative"):
        lib.layer_norm(x, w, b, -1.0)
    with pytest.raises(RuntimeError, match="at least 1"):
        lib.layer_norm(torch.zeros(4, 0, device="cuda"))
    _, mean, rstd = lib.layer_norm_forward(x, w, b, 1e-5, True)
    with pytest.raises(RuntimeError, match="shape and dtype of x"):
        lib.layer_norm_backward(grad[:, :16], x, mean, rstd, w)
    with pytest.raises(RuntimeError, match="one value per row"):
        lib.layer_norm_backward(grad, x, mean[:2], rstd, w)


def test_differentiable_once(lib):
    x, w, b, grad = make(4, 32, F32, F32)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    first = torch.autograd.grad(lib.layer_norm(*leaves), leaves, grad, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        first[0].sum().backward()
    # a frozen parameter gets no gradient, the others keep theirs
    y = lib.layer_norm(x, w.detach(), b)
    dx, db = torch.autograd.grad(y, [x, b], grad)
    assert torch.equal(dx, first[0].detach()) and torch.equal(db, first[2].detach())
