"""Plain 64-bit forms of the layer operators and the error bounds their tests
hold the kernels to.

Bounds.  A result rounded once to its type is off by at most u |r| (u the
type's unit roundoff: half a unit in the last place), plus the fp32 error of
the sum behind it.  A sum of n products, added in any order in fp32 (also by
a matrix unit that truncates each step), is off by at most n 2^-23 times the
sum of the products' magnitudes; ``sum_bound`` takes n = length / 8 + 16,
since every kernel adds at least eight products before it rounds into a
running sum or runs several sums side by side.  fp16 results below 2^-14 are
subnormal: 2^-25 absolute.
"""

import torch

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -140}


def sum_bound(length):
    return (length / 8 + 16) * 2.0 ** -23


def assert_within(actual, expected, slack, what=""):
    """|actual - expected| <= u |expected| + slack, element by element."""
    assert actual.shape == expected.shape, (what, tuple(actual.shape), tuple(expected.shape))
    err = (actual.double() - expected).abs()
    bound = UNIT[actual.dtype] * expected.abs() * 1.0001 + slack + TINY[actual.dtype]
    bad = ~(err <= bound)
    if bool(bad.any()):
        i = tuple(torch.nonzero(bad)[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: {actual[i].item()} vs "
                             f"{expected[i].item()}, bound {bound.expand_as(err)[i].item()}")


def norm_reference(x, weight, bias, eps, grad=None):
    """y (and dx, dw, db) with each one's fp32 slack, all in 64 bits."""
    x = x.double()
    width = x.shape[-1]
    w = torch.ones(width, dtype=torch.float64, device=x.device) if weight is None else weight.double()
    b = torch.zeros(width, dtype=torch.float64, device=x.device) if bias is None else bias.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    xhat = (x - mean) * rstd
    y = xhat * w + b
    # xhat's error: the mean's (sum of |x|) and rstd's relative one
    s = sum_bound(width)
    dxhat = s * (x.abs().mean(-1, keepdim=True) + x.abs()) * rstd + 4 * s * xhat.abs()
    dxhat = dxhat + s * xhat.abs() * (x.abs().mean(-1, keepdim=True) * rstd) * xhat.abs().mean(-1, keepdim=True)
    out = [(y, dxhat * w.abs() + 2.0 ** -22 * (y.abs() + b.abs()))]
    if grad is not None:
        grad = grad.double()
        g = grad * w
        c1, c2 = g.mean(-1, keepdim=True), (g * xhat).mean(-1, keepdim=True)
        dx = rstd * (g - c1 - xhat * c2)
        a2 = (g * xhat).abs().mean(-1, keepdim=True)
        slack = rstd * (s * (g.abs() + g.abs().mean(-1, keepdim=True) + xhat.abs() * a2) + dxhat * a2
                        + xhat.abs() * (dxhat * g.abs()).mean(-1, keepdim=True)) + 4 * s * dx.abs()
        out.append((dx, slack))
        rows = x.reshape(-1, width).shape[0]
        flat = lambda t: t.reshape(-1, width)  # noqa: E731
        n = sum_bound(rows)
        out.append((flat(grad * xhat).sum(0), n * flat(grad * xhat).abs().sum(0) + flat(dxhat * grad.abs()).sum(0)))
        out.append((flat(grad).sum(0), n * flat(grad).abs().sum(0)))
    return out


def grouped_reference(x, weight, ptr, transposed=False):
    """Rows product in 64 bits and its slack (rows outside every group are zero)."""
    ptr = [int(p) for p in ptr.tolist()]
    groups, K, N = weight.shape
    width, depth = (K, N) if transposed else (N, K)
    y = torch.zeros(x.shape[0], width, dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(y)
    for g in range(groups):
        r = slice(ptr[g], ptr[g + 1])
        w = weight[g].double().T if transposed else weight[g].double()
        y[r] = x[r].double() @ w
        mag[r] = x[r].double().abs() @ w.abs()
    return y, sum_bound(depth) * mag


def weight_grad_reference(x, grad, ptr):
    ptr = [int(p) for p in ptr.tolist()]
    groups = len(ptr) - 1
    dw = torch.zeros(groups, x.shape[1], grad.shape[1], dtype=torch.float64, device=x.device)
    slack = torch.zeros_like(dw)
    for g in range(groups):
        r = slice(ptr[g], ptr[g + 1])
        a, b = x[r].double(), grad[r].double()
        dw[g] = a.T @ b
        slack[g] = sum_bound(max(0, ptr[g + 1] - ptr[g])) * (a.abs().T @ b.abs())
    return dw, slack


def ortho_reference(update, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7):
    """The polynomial a s + b s^3 + c s^5 applied to the singular values."""
    a, b, c = coefficients
    u, s, vh = torch.linalg.svd(update.double(), full_matrices=False)
    s = s / (torch.sqrt((s * s).sum(-1, keepdim=True)) + eps)
    for _ in range(steps):
        s = a * s + b * s ** 3 + c * s ** 5
    return u @ (s[..., None] * vh)
