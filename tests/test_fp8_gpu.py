"""quantize_fp8, quantize_weight_fp8 and grouped_matmul_fp8 on the GPU: bits of
the quantised values, products against 64 bits of what 8 bits hold."""

import pytest
import torch

import routed_reference as ref
from layer_reference import assert_within, grouped_reference
from test_grouped_gpu import SIZES, lib  # noqa: F401

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def normal(*shape, dtype=F32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def same_bits(q, want):
    """8-bit tensors against values (zeros of either sign are told apart, NaNs are not)."""
    got = q.float()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    ok = ~torch.isnan(want)
    assert torch.equal(got[ok], want[ok]) and torch.equal(torch.signbit(got[ok]), torch.signbit(want[ok]))


def check_rows(lib, x):  # noqa: F811
    q, scale = lib.quantize_fp8(x)
    want, wscale = ref.quantize_reference(x.reshape(-1, x.shape[-1]))
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and scale.shape == (*x.shape[:-1], wscale.shape[1])
    assert torch.equal(scale.reshape(wscale.shape), wscale)
    same_bits(q.reshape(want.shape), want)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("width", [16, 32, 112, 128, 144, 256, 400, 1024, 2064])
@pytest.mark.parametrize("rows", [1, 7, 130])
def test_rows_in_8_bits(lib, rows, width, dtype):  # noqa: F811
    x = normal(rows, width, seed=width) * torch.exp(2 * normal(rows, 1, seed=1))
    check_rows(lib, x.to(dtype))
    check_rows(lib, x.to(dtype).view(1, rows, width))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_rows_of_special_values(lib, dtype):  # noqa: F811
    x = normal(12, 256, dtype=dtype)
    x[1] = 0
    x[2] = -0.0
    x[3, 5], x[3, 140], x[3, 141] = float("inf"), -float("inf"), float("nan")
    x[4, :128] = float("nan")
    x[5] *= torch.finfo(dtype).max / 8
    x[6] = torch.finfo(dtype).tiny
    x[7] = torch.finfo(dtype).smallest_normal
    x[8] = torch.finfo(dtype).max
    x[9, ::2] *= 2.0 ** -12            # e4m3's subnormals
    x[10] = torch.arange(256, device="cuda").to(dtype) * 0.0625   # values between two of e4m3
    check_rows(lib, x)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("groups,K,N", [(1, 16, 16), (3, 128, 128), (2, 144, 272), (5, 400, 112), (2, 1024, 48)])
def test_weights_in_8_bits(lib, groups, K, N, dtype):  # noqa: F811
    w = normal(groups, K, N, dtype=dtype, seed=K)
    w[0, 3, 5] = float("nan")
    w[0, 4, 5] = -float("inf")
    if groups > 1:
        w[1] = 0
    q, scale = lib.quantize_weight_fp8(w)
    want, wscale = ref.quantize_weight_reference(w)
    assert q.shape == (groups, N, K) and torch.equal(scale, wscale)
    same_bits(q, want)


def make(lib, sizes, K, N, dtype, seed=0, before=0, after=0, idt=torch.int32):  # noqa: F811
    ptr = torch.zeros(len(sizes) + 1, dtype=torch.int64)
    ptr[1:] = torch.cumsum(torch.tensor(sizes, dtype=torch.int64), 0)
    rows = int(ptr[-1]) + before + after
    x = (normal(rows, K, seed=seed) * torch.exp(normal(rows, 1, seed=seed + 1))).to(dtype)
    w = (normal(len(sizes), K, N, seed=seed + 2) / K ** 0.5).to(dtype)
    return x, w, (ptr + before).to(idt).cuda()


def check(lib, x, w, ptr, out_dtype=None):  # noqa: F811
    q, s = lib.quantize_fp8(x)
    wq, ws = lib.quantize_weight_fp8(w)
    out_dtype = out_dtype or x.dtype
    y = lib.grouped_matmul_fp8(q, s, wq, ws, ptr, out_dtype)
    assert y.dtype == out_dtype
    assert_within(y, *ref.fp8_reference(q, s, wq, ws, ptr), "y")
    return y


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("sizes", SIZES, ids=range(len(SIZES)))
def test_ragged_groups(lib, sizes, dtype):  # noqa: F811
    check(lib, *make(lib, sizes, 144, 48, dtype, seed=len(sizes)))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("K,N", [(16, 16), (16, 272), (80, 16), (128, 128), (48, 320), (256, 512), (1040, 144), (144, 1040),
                                 (512, 256), (400, 272), (2048, 96)])
def test_widths(lib, K, N, dtype):  # noqa: F811
    check(lib, *make(lib, [70, 0, 131, 9], K, N, dtype, seed=K + N))


@pytest.mark.parametrize("rows,groups,K,N", [(9, 32, 1024, 512), (3000, 4, 512, 512), (5003, 46, 400, 272), (9000, 6, 1024, 512)])
def test_sizes_of_use(lib, rows, groups, K, N):  # noqa: F811
    g = torch.Generator().manual_seed(rows)
    sizes = torch.bincount(torch.randint(0, groups, (rows,), generator=g), minlength=groups).tolist()
    check(lib, *make(lib, sizes, K, N, BF16, seed=1))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("sizes,N", [([6000, 0, 9003, 4097], 256), ([257, 255, 256, 1, 5000, 4, 0, 4000], 512),
                                     ([3] * 30 + [5000, 4700], 512), ([0, 0, 19500, 0], 256)])
def test_many_rows(lib, sizes, N, dtype):  # noqa: F811
    """Groups that end inside a pair's tile of 256 rows, rows before the first one and behind the last."""
    x, w, ptr = make(lib, sizes, 144, N, dtype, seed=2, before=77, after=133)
    y = check(lib, x, w, ptr)
    assert bool((y[:77] == 0).all()) and bool((y[len(y) - 133:] == 0).all())


def test_rows_outside_every_group_and_index_types(lib):  # noqa: F811
    for idt in (torch.int32, torch.int64):
        x, w, ptr = make(lib, [40, 3], 64, 32, BF16, before=5, after=9, idt=idt)
        y = check(lib, x, w, ptr)
        assert bool((y[:5] == 0).all()) and bool((y[48:] == 0).all())
        check(lib, x, w, ptr, F32)
        check(lib, x, w, ptr, F16)


def test_a_value_that_is_not_finite_stays_in_its_row(lib):  # noqa: F811
    x, w, ptr = make(lib, [20, 30], 256, 48, F32)
    x[3, 200], x[25, 1] = float("inf"), float("nan")
    q, s = lib.quantize_fp8(x)
    wq, ws = lib.quantize_weight_fp8(w)
    y = lib.grouped_matmul_fp8(q, s, wq, ws, ptr, F32)
    bad = torch.isnan(y).all(1)
    assert bad.nonzero().flatten().tolist() == [3, 25] and int((~torch.isfinite(y)).sum()) == 2 * 48


def test_how_far_8_bits_are_from_the_product(lib):  # noqa: F811
    """Each operand is off by at most 2^-4 of itself (or, below e4m3's normal range, 2^-10 of a scale): the sum of the
    products' magnitudes times 2^-3 + 2^-8 bounds the difference."""
    x, w, ptr = make(lib, [100, 50, 7], 384, 64, F32, seed=3)
    q, s = lib.quantize_fp8(x)
    wq, ws = lib.quantize_weight_fp8(w)
    y = lib.grouped_matmul_fp8(q, s, wq, ws, ptr, F32)
    want, _ = grouped_reference(x, w, ptr)
    most, _ = grouped_reference(x.abs() + s.repeat_interleave(128, 1), w.abs() + w.abs().amax() / 448, ptr)
    assert bool(((y.double() - want).abs() <= (2.0 ** -3 + 2.0 ** -8) * most).all())
    assert float((y.double() - want).norm()) < 0.06 * float(want.norm())   # 2^-4 / sqrt(3) of each of the two, summed


def test_no_rows_no_groups(lib):  # noqa: F811
    x, w, ptr = make(lib, [0, 0], 32, 32, BF16)
    assert check(lib, x, w, ptr).shape == (0, 32)
    q, s = lib.quantize_fp8(normal(6, 32, dtype=BF16))
    wq, ws = lib.quantize_weight_fp8(torch.empty(0, 32, 48, device="cuda"))
    y = lib.grouped_matmul_fp8(q, s, wq, ws, torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert y.shape == (6, 48) and bool((y == 0).all())


def test_captured_and_on_another_stream(lib):  # noqa: F811
    x, w, ptr = make(lib, [100, 0, 60], 256, 128, BF16)
    wq, ws = lib.quantize_weight_fp8(w)

    def call():
        q, s = lib.quantize_fp8(x)
        return lib.grouped_matmul_fp8(q, s, wq, ws, ptr)

    want = call()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = call()
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for sizes in ([100, 0, 60], [0, 160, 0], [1, 100, 59]):
        x.copy_(normal(160, 256, seed=sizes[0]))
        ptr[1:] = torch.cumsum(torch.tensor(sizes), 0).to(torch.int32)
        graph.replay()
        assert torch.equal(got, call())


def test_refusals(lib):  # noqa: F811
    x, w, ptr = make(lib, [4, 3], 32, 48, BF16)
    q, s = lib.quantize_fp8(x)
    wq, ws = lib.quantize_weight_fp8(w)
    f = lib.grouped_matmul_fp8
    for call, text in ((lambda: lib.quantize_fp8(normal(4, 24)), "divisible by 16, but got 24"),
                       (lambda: lib.quantize_fp8(normal(4, 32).double()), "supports only FP16, BF16 and FP32"),
                       (lambda: lib.quantize_fp8(normal(4, 32).requires_grad_(True)), "not differentiable"),
                       (lambda: lib.quantize_weight_fp8(w[0]), "three-dimensional"),
                       (lambda: lib.quantize_weight_fp8(normal(1, 32, 8)), "divisible by 16, but got 8"),
                       (lambda: f(x, s, wq, ws, ptr), "float8_e4m3fn"),
                       (lambda: f(q, s, w, ws, ptr), "float8_e4m3fn"),
                       (lambda: f(q[:, :16], s, wq, ws, ptr), "features"),
                       (lambda: f(q, s[:6], wq, ws, ptr), "x_scale must have shape"),
                       (lambda: f(q, s, wq, ws[:1], ptr), "weight_scale must have shape"),
                       (lambda: f(q, s.half(), wq, ws, ptr), "scales must be FP32"),
                       (lambda: f(q, s, wq, ws, ptr[:2]), "groups \\+ 1 entries"),
                       (lambda: f(q, s, wq, ws, ptr.float()), "int32 or int64"),
                       (lambda: f(q, s, wq, ws, ptr, torch.float64), "FP16, BF16 and FP32 results"),
                       (lambda: f(q.cpu(), s, wq, ws, ptr), "must be CUDA tensor")):
        with pytest.raises(RuntimeError, match=text):
            call()
