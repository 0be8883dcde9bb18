"""grouped_matmul and its gradients at the limits of their forms: long sums."""

import pytest
import torch

from test_grouped_gpu import lib  # noqa: F401

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


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
