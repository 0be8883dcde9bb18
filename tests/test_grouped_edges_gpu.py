"""grouped_matmul and its gradients at the limits of their forms: infinities
in fp32, long sums, the number of groups that a weight gradient sorts, pairs
of blocks in both directions."""

import pytest
import torch

from layer_reference import assert_within, grouped_reference
from test_grouped_gpu import check, lib, make  # noqa: F401

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def same_kind(got, want, what):
    """NaN where the reference has NaN, the same infinities; finite values to fp32's accuracy."""
    got, want = got.cpu().double(), want.cpu()
    assert torch.equal(got.isnan(), want.isnan()), what
    assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got[got.isinf()], want[want.isinf()]), what
    ok = want.isfinite()
    assert bool(((got - want)[ok].abs() <= 1e-5 * (1 + want[ok].abs())).all()), what


def test_fp32_infinities(lib):  # noqa: F811
    """An infinity gives what fp32 arithmetic gives: infinities of the products' signs, NaN for infinity times zero,
    for infinities of both signs and for NaN."""
    x, w, ptr, grad = make([40, 30], 64, 48, F32, seed=13)
    inf = float("inf")
    x[3, 5], x[50, 7] = inf, -inf
    x[9, 1], x[9, 2] = inf, inf                  # of one sign or of both, by the weight's signs
    w[0, 5, 11] = 0.0                            # inf * 0
    w[0, 20, 3], x[4, 20], x[5, 20] = -inf, 0.0, inf
    w[1, 30, 40], x[60, 30] = float("nan"), 2.0
    w[0, 5, 12] = 0.5                            # nothing below the highest of its three parts
    ref = lambda a, b: (a.cpu().double()[:, :, None] * b.cpu().double()[None]).sum(1)  # noqa: E731
    want = torch.cat([ref(x[:40], w[0]), ref(x[40:], w[1])])
    assert bool(want[3].isinf().any()) and bool(want[3].isnan().any()) and bool(want[50, :40].isinf().all())
    same_kind(lib.grouped_matmul(x, w, ptr), want, "y")
    grad[2, 3], grad[45, 9], grad[33, 3] = inf, -inf, 0.0
    want = torch.cat([ref(grad[:40], w[0].T), ref(grad[40:], w[1].T)])
    same_kind(lib.grouped_matmul(grad, w, ptr, transposed=True), want, "dx")
    want = torch.stack([ref(x[:40].T, grad[:40]), ref(x[40:].T, grad[40:])])
    same_kind(lib.grouped_weight_grad(x, grad, ptr), want, "dw")


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_million_rows_of_one_group(lib, dtype):  # noqa: F811
    """A sum of 2^20 products of one sign.  A matrix unit truncates its accumulator in every step of 16 products, by
    at most 2^-22 of what it holds; over a part of 16384 rows that is at most 1024 steps at half of the final sum on
    average, 2^-13, and the parts are added with fp32's rounding.  The result's own rounding has either sign: over
    4096 elements its mean is below 2^-9 / 64 = 2^-15 for bf16."""
    rows, width = 1 << 20, 2048
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.rand(rows, width, generator=g, device="cuda", dtype=dtype).add_(0.5).mul_(0.125)
    grad = torch.rand(rows, width, generator=g, device="cuda", dtype=dtype).add_(0.5).mul_(0.125)
    ptr = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    dw = lib.grouped_weight_grad(x, grad, ptr)[0]
    for at in (slice(0, 64), slice(width - 64, width)):
        want = x[:, at].double().T @ grad[:, at].double()
        mean = float(((dw[at, at].double() - want) / want).mean())
        assert abs(mean) <= 2.0 ** -13 + 2.0 ** -15, mean


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("groups", [127, 128, 129])
def test_groups_around_the_sorted_ones(lib, groups, dtype):  # noqa: F811
    """A weight gradient sorts up to 128 groups; the others are walked in their order."""
    g = torch.Generator().manual_seed(groups)
    sizes = torch.randint(0, 7, (groups,), generator=g)
    sizes[groups // 3], sizes[groups - 2], sizes[groups - 1] = 3000, 2100, 1
    check(lib, *make(sizes.tolist(), 48, 32, dtype, seed=groups))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("transposed", [False, True])
def test_pairs_of_blocks_beside_rows_of_no_group(lib, dtype, transposed):  # noqa: F811
    """Tiles of 256 rows shared by two blocks (rows / 256 * width / 256 of at least two turns of the GPU, groups of
    512 rows on average, 512 deep), in both directions, with rows outside every group."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    K, N, width = 512, 768, 512 if transposed else 768
    rows = -(-2 * sms // (width // 256)) * 256 + 1000
    sizes = [5000, 0, 1, 129, 255, 257, rows - 300 - 77 - 5642]
    x, w, ptr, grad = make(sizes, K, N, dtype, seed=12, before=300, after=77)
    a = grad if transposed else x
    assert a.shape[0] == rows and rows // 256 * (width // 256) >= 2 * sms and rows >= 512 * len(sizes)
    a[:300], a[-77:] = float("nan"), float("inf")
    y = lib.grouped_matmul(a, w, ptr, transposed=transposed)
    assert not bool(y[:300].any()) and not bool(y[-77:].any())
    ref, slack = grouped_reference(a, w, ptr, transposed)
    assert_within(y[300:-77], ref[300:-77], slack[300:-77])
    # a group's values reach no other: those of the first as NaN
    a[300:5300] = float("nan")
    again = lib.grouped_matmul(a, w, ptr, transposed=transposed)
    assert torch.equal(again[5300:], y[5300:]) and bool(again[300:5300].isnan().all())
