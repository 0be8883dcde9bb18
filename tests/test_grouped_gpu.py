"""grouped_matmul and its gradients on the GPU against a product per group in
64 bits: ragged, empty and single-row groups, rows outside every group, types,
widths, non-finite neighbours, malformed ranges, refusals."""

import pytest
import torch

from layer_reference import assert_within, grouped_reference, weight_grad_reference

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def lib():
    import build

    build.build()
    import spmm_npu

    spmm_npu.device_status(True)
    yield spmm_npu
    assert spmm_npu.device_status(True)[0] == 0


def make(sizes, K, N, dtype, seed=0, before=0, after=0, idt=torch.int32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    ptr = torch.zeros(len(sizes) + 1, dtype=torch.int64)
    ptr[1:] = torch.cumsum(torch.tensor(sizes, dtype=torch.int64), 0)
    rows = int(ptr[-1]) + before + after
    return (n(rows, K).to(dtype), (n(len(sizes), K, N) / K ** 0.5).to(dtype), (ptr + before).to(idt).cuda(),
            n(rows, N).to(dtype))


def check(lib, x, w, ptr, grad):
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = lib.grouped_matmul(xl, wl, ptr)
    dx, dw = torch.autograd.grad(y, [xl, wl], grad)
    assert torch.equal(lib.grouped_matmul(x, w, ptr), y)
    assert_within(y.detach(), *grouped_reference(x, w, ptr), "y")
    assert_within(dx, *grouped_reference(grad, w, ptr, True), "dx")
    assert_within(dw, *weight_grad_reference(x, grad, ptr), "dw")


SIZES = [[1], [5], [128], [129], [0, 0, 7], [64, 0, 1, 200, 0], [1] * 40, [300, 3, 17, 0, 131, 64, 63, 65, 127],
         [0] * 70 + [9, 0, 33] + [0] * 50]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("sizes", SIZES, ids=range(len(SIZES)))
def test_ragged_groups(lib, sizes, dtype):
    check(lib, *make(sizes, 64, 48, dtype, seed=len(sizes)))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("K,N", [(16, 16), (16, 272), (80, 16), (128, 128), (48, 320), (256, 512), (1040, 144),
                                 (144, 1040), (512, 256)])
def test_widths(lib, K, N, dtype):
    check(lib, *make([70, 0, 131, 1, 260], K, N, dtype, seed=K + N))


@pytest.mark.parametrize("K,N", [(8, 8), (24, 264), (264, 40)])
def test_fp32_widths_of_eight(lib, K, N):
    check(lib, *make([70, 0, 131, 1], K, N, F32, seed=K))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("idt", [torch.int32, torch.int64])
def test_long_groups(lib, dtype, idt):
    check(lib, *make([5000, 1, 9001, 0, 333], 144, 272, dtype, seed=2, idt=idt))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_rows_outside_every_group_are_zero(lib, dtype):
    x, w, ptr, grad = make([33, 0, 150], 64, 80, dtype, before=140, after=301)
    lo, hi = int(ptr[0]), int(ptr[-1])
    x[:lo], x[hi:] = float("nan"), float("inf")       # never read into a result
    grad[:lo], grad[hi:] = float("inf"), float("nan")
    y = lib.grouped_matmul(x, w, ptr)
    dx = lib.grouped_matmul(grad, w, ptr, transposed=True)
    dw = lib.grouped_weight_grad(x, grad, ptr)
    for t in (y, dx):
        assert not bool(t[:lo].any()) and not bool(t[hi:].any())
    assert_within(y[lo:hi], *(t[lo:hi] for t in grouped_reference(x, w, ptr)))
    assert_within(dx[lo:hi], *(t[lo:hi] for t in grouped_reference(grad, w, ptr, True)))
    assert_within(dw, *weight_grad_reference(x, grad, ptr))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_non_finite_values_stay_in_their_group(lib, dtype):
    """A group's NaN and infinite rows and weights reach no other group, though tiles of rows and of the
    reduction end inside a group and would take in its neighbours."""
    x, w, ptr, grad = make([37, 41, 90, 13], 48, 80, dtype, seed=9)
    want = (lib.grouped_matmul(x, w, ptr), lib.grouped_matmul(grad, w, ptr, transposed=True),
            lib.grouped_weight_grad(x, grad, ptr))
    b, e = int(ptr[1]), int(ptr[2])
    x[b:e], grad[b:e], w[1] = float("nan"), float("inf"), float("nan")
    got = (lib.grouped_matmul(x, w, ptr), lib.grouped_matmul(grad, w, ptr, transposed=True),
           lib.grouped_weight_grad(x, grad, ptr))
    rows = torch.ones(x.shape[0], dtype=torch.bool, device="cuda")
    rows[b:e] = False
    groups = torch.tensor([True, False, True, True], device="cuda")
    assert torch.equal(got[0][rows], want[0][rows]) and torch.equal(got[1][rows], want[1][rows])
    assert torch.equal(got[2][groups], want[2][groups])
    assert bool(got[0][b:e].isnan().all()) and bool(got[1][b:e].isnan().all()) and bool(got[2][1].isnan().all())


@pytest.mark.parametrize("dtype", [F16, F32])
def test_gradient_against_differences(lib, dtype):
    """The product is bilinear: f(x + d) - f(x - d) = 2 <df/dx, d> exactly, up to rounding."""
    x, w, ptr, grad = make([20, 0, 45], 32, 48, dtype, seed=6)
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(lib.grouped_matmul(xl, wl, ptr), [xl, wl], grad)
    g = torch.Generator(device="cuda").manual_seed(7)
    f = lambda a, b: float((grouped_reference(a, b, ptr)[0] * grad.double()).sum())  # noqa: E731
    for t, d_t, put in ((x, dx, lambda v: (v, w)), (w, dw, lambda v: (x, v))):
        d = torch.randn(t.shape, generator=g, device="cuda", dtype=torch.float64)
        slope = (f(*put(t.double() + d)) - f(*put(t.double() - d))) / 2
        # each gradient element is rounded once to its type (u relative) and summed in fp32
        scale = float((d_t.double().abs() * d.abs()).sum())
        assert abs(float((d_t.double() * d).sum()) - slope) <= (2.0 ** -10 if dtype == F16 else 2.0 ** -18) * scale


def test_no_rows_and_no_groups(lib):
    w = torch.randn(3, 32, 16, device="cuda", dtype=F16)
    x = torch.zeros(0, 32, device="cuda", dtype=F16)
    ptr = torch.zeros(4, dtype=torch.int32, device="cuda")
    assert lib.grouped_matmul(x, w, ptr).shape == (0, 16)
    dw = lib.grouped_weight_grad(x, torch.zeros(0, 16, device="cuda", dtype=F16), ptr)
    assert dw.shape == (3, 32, 16) and not bool(dw.any())
    none = lib.grouped_matmul(torch.randn(5, 32, device="cuda").half(), w[:0], ptr[:1])
    assert none.shape == (5, 16) and not bool(none.any())
    assert lib.grouped_weight_grad(x, torch.zeros(0, 16, device="cuda", dtype=F16), ptr[:1]).shape == (0, 32, 16)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_malformed_ranges_are_reported(lib, dtype):
    x, w, ptr, grad = make([30, 30, 30], 32, 32, dtype)
    for bad in ([0, 30, 20, 90], [0, 30, 60, 400], [-5, 30, 60, 90]):
        p = torch.tensor(bad, dtype=torch.int32, device="cuda")
        for call in (lambda: lib.grouped_matmul(x, w, p), lambda: lib.grouped_weight_grad(x, grad, p)):
            lib.device_status(True)
            call()
            assert lib.device_status(True)[0] == 2
    # the well-formed groups beside a malformed one are right
    p = torch.tensor([0, 30, 60, 400], dtype=torch.int64, device="cuda")
    y = lib.grouped_matmul(x, w, p)
    assert_within(y[:60], *(t[:60] for t in grouped_reference(x, w, ptr)))
    assert lib.device_status(True)[0] == 2


def test_strided_inputs(lib):
    x, w, ptr, grad = make([20, 33], 48, 64, F16)
    want = lib.grouped_matmul(x, w, ptr)
    wide = torch.zeros(53, 100, device="cuda", dtype=F16)
    wide[:, 30:78] = x
    assert torch.equal(lib.grouped_matmul(wide[:, 30:78], w, ptr), want)
    assert torch.equal(lib.grouped_matmul(x, w.transpose(1, 2).contiguous().transpose(1, 2), ptr), want)
    # an expanded gradient
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    lib.grouped_matmul(xl, wl, ptr).sum().backward()
    one = torch.ones(53, 64, device="cuda", dtype=F16)
    assert_within(xl.grad, *grouped_reference(one, w, ptr, True))
    assert_within(wl.grad, *weight_grad_reference(x, one, ptr))


def test_same_result_twice_on_another_stream_and_in_a_graph(lib):
    x, w, ptr, grad = make([1000, 3, 0, 2500, 40], 256, 128, BF16, seed=3)
    run = lambda: (lib.grouped_matmul(x, w, ptr), lib.grouped_matmul(grad, w, ptr, transposed=True),  # noqa: E731
                   lib.grouped_weight_grad(x, grad, ptr))
    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = run()
    graph.replay()
    assert all(torch.equal(p, q) for p, q in zip(first, third))
    # the ranges are read by the launch, not kept: new ones take effect in a replay
    ptr.copy_(torch.tensor([0, 7, 1007, 1010, 1010, 3543], dtype=torch.int32))
    graph.replay()
    assert_within(third[0], *grouped_reference(x, w, ptr))
    assert_within(third[2], *weight_grad_reference(x, grad, ptr))


def test_offsets_beyond_32_bits(lib):
    """2.2 M rows of 1024 features: element offsets of x pass 2^31; the last groups are checked."""
    rows, K, N = (1 << 21) + 70001, 1024, 16
    x = torch.zeros(rows, K, dtype=F16, device="cuda")
    tail, w, p, grad = make([100, 57], K, N, F16, seed=5)
    x[-157:] = tail
    ptr = torch.tensor([0, rows - 57, rows], dtype=torch.int64, device="cuda")
    y = lib.grouped_matmul(x, w, ptr)
    ref, slack = grouped_reference(tail, w, p)
    assert_within(y[-157:], ref, slack)
    assert not bool(y[: rows - 157].any())
    full = torch.zeros(rows, N, dtype=F16, device="cuda")
    full[-157:] = grad
    dw, sdw = weight_grad_reference(tail, grad, p)
    assert_within(lib.grouped_weight_grad(x, full, ptr), dw, sdw)
    dx = lib.grouped_matmul(full, w, ptr, transposed=True)
    assert_within(dx[-157:], *grouped_reference(grad, w, p, True))


def test_refusals(lib):
    x, w, ptr, grad = make([4, 4], 32, 32, F16)
    with pytest.raises(RuntimeError, match="must be CUDA tensor"):
        lib.grouped_matmul(x.cpu(), w, ptr)
    with pytest.raises(RuntimeError, match="group_ptr must be CUDA tensor"):
        lib.grouped_matmul(x, w, ptr.cpu())
    with pytest.raises(RuntimeError, match="supports only FP16, BF16 and FP32"):
        lib.grouped_matmul(x.double(), w.double(), ptr)
    with pytest.raises(RuntimeError, match="same dtype as x"):
        lib.grouped_matmul(x, w.float(), ptr)
    with pytest.raises(RuntimeError, match="features"):
        lib.grouped_matmul(x[:, :16], w, ptr)
    with pytest.raises(RuntimeError, match="groups \\+ 1"):
        lib.grouped_matmul(x, w, ptr[:2])
    with pytest.raises(RuntimeError, match="int32 or int64"):
        lib.grouped_matmul(x, w, ptr.float())
    with pytest.raises(RuntimeError, match="divisible by 16, but got 24"):
        lib.grouped_matmul(x[:, :24], w[:, :24], ptr)
    with pytest.raises(RuntimeError, match="divisible by 8, but got 12"):
        lib.grouped_matmul(x[:, :16].float(), w[:, :16, :12].float(), ptr)
    with pytest.raises(RuntimeError, match="same number of rows"):
        lib.grouped_weight_grad(x, grad[:4], ptr)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("groups", [255, 256, 257, 3000])
def test_many_groups(lib, groups, dtype):
    """More groups than the weight gradient sorts, some of them long enough to be summed in parts."""
    g = torch.Generator().manual_seed(groups)
    sizes = torch.randint(0, 7, (groups,), generator=g)
    sizes[groups // 3], sizes[groups - 2] = 3000, 2100
    check(lib, *make(sizes.tolist(), 48, 32, dtype, seed=groups))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_pairs_of_blocks(lib, dtype):
    """Long groups and wide weights, where two blocks share a tile of 256 rows; groups that end anywhere in it."""
    check(lib, *make([5000, 3000, 129, 0, 1, 255, 12000, 257], 512, 1024, dtype, seed=11))
    x, w, ptr, grad = make([9001, 9007], 1024, 512, dtype, seed=12, before=300, after=77)
    x[:300], x[-77:] = float("nan"), float("inf")
    y = lib.grouped_matmul(x, w, ptr)
    assert not bool(y[:300].any()) and not bool(y[-77:].any())
    assert_within(y[300:-77], *(t[300:-77] for t in grouped_reference(x, w, ptr)))
    dx = lib.grouped_matmul(grad, w, ptr, transposed=True)
    assert_within(dx, *grouped_reference(grad, w, ptr, True))


def test_one_long_group_and_wide_weights(lib):
    """A weight gradient in many parts, tiles of several widths."""
    for K, N in ((16, 544), (272, 80), (1024, 256)):
        x, w, ptr, grad = make([40000, 0, 5], K, N, F16, seed=K)
        assert_within(lib.grouped_weight_grad(x, grad, ptr), *weight_grad_reference(x, grad, ptr))


def test_fp32_extremes(lib):
    """Values over fp32's range: the planes of a split operand keep its exponents; infinities and NaN give
    non-finite results in their rows alone."""
    x, w, ptr, grad = make([40, 30], 64, 48, F32, seed=13)
    big = x * 1e30
    assert_within(lib.grouped_matmul(big, w, ptr), *grouped_reference(big, w, ptr))
    small = x * 1e-25
    assert_within(lib.grouped_matmul(small, w, ptr), *grouped_reference(small, w, ptr))
    top = torch.full((70, 64), 3.4028234e38, device="cuda")
    one = torch.zeros(2, 64, 48, device="cuda")
    one[:, 0] = 0.5
    assert torch.equal(lib.grouped_matmul(top, one, ptr), torch.full((70, 48), 1.7014117e38, device="cuda"))
    x[3, 5] = float("inf")
    y = lib.grouped_matmul(x, w, ptr)
    rows = torch.arange(70, device="cuda") != 3
    assert not bool(y[3].isfinite().any()) and bool(y[rows].isfinite().all())
