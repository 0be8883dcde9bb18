"""orthogonalize on the GPU where rounding could grow: many steps on low rank
and steep spectra, the 22-bit form of thin matrices, coefficients that take
the operands out of the range of the default ones."""

import pytest
import torch

from layer_reference import ortho_reference
from test_ortho_gpu import check, gradient, lib  # noqa: F401

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def low_rank(m, n, rank, noise, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return r(m, rank) @ r(rank, n) + noise * r(m, n)


@pytest.mark.parametrize("steps", [5, 6, 7, 8, 9])
@pytest.mark.parametrize("m,n", [(100, 200), (128, 256), (1024, 128)])
def test_steps_on_low_rank_and_steep_spectra(lib, m, n, steps):  # noqa: F811
    """Small singular values grow by a factor of 3.4 a step, and so does what was rounded along them."""
    for rank in (1, 4):
        for noise in (1e-2, 1e-3):
            check(lib, low_rank(m, n, rank, noise), steps=steps)
    check(lib, gradient(1, m, n, F32, decay=3.0), steps=steps)


@pytest.mark.parametrize("batch,m,n", [(1, 128, 64), (2, 100, 200), (1, 128, 128), (2, 64, 2000), (1, 4000, 30)])
def test_thin_matrices_keep_their_low_parts(lib, batch, m, n):  # noqa: F811
    """A side of at most 128, default steps: the error before the result's rounding stays below 2.5e-4 in the norm
    (operands of two fp16 parts, 22 bits; 11-bit operands alone give 1.5e-3 and more).  The rounding to bf16 is
    independent of it, so the squares add up; 2 % of the rounding's for the chance of it."""
    u = gradient(batch, m, n, F32, seed=m)
    ref = ortho_reference(u)
    norm = lambda t: t.flatten(-2).norm(dim=-1)  # noqa: E731
    rounding = norm(ref.to(BF16).double() - ref)
    err = norm(lib.orthogonalize(u).double() - ref)
    assert bool((err ** 2 <= 1.02 * rounding ** 2 + (2.5e-4 * norm(ref)) ** 2).all()), (err / norm(ref), rounding / norm(ref))


@pytest.mark.parametrize("m,n", [(24, 40), (300, 100), (200, 136), (130, 400)])
@pytest.mark.parametrize("coefficients,steps", [((1.0, 300.0, -200.0), 1), ((1.0, 6.0, 0.0), 2), ((200.0, 0.0, 0.0), 2)])
def test_coefficients_beyond_the_operands_range(lib, m, n, coefficients, steps):  # noqa: F811
    """One dominant element, so that elements reach what the polynomials of the singular values reach: hundreds
    for b G + c G G, a X + P X and a I + b G + c G G."""
    g = torch.Generator(device="cuda").manual_seed(m)
    u = 0.01 * torch.randn(2, m, n, generator=g, device="cuda")
    u[:, 3, 5] = 10.0
    check(lib, u, steps=steps, coefficients=coefficients)


def test_coefficients_that_fp32_cannot_hold_are_refused(lib):  # noqa: F811
    with pytest.raises(RuntimeError, match="finite"):
        lib.orthogonalize(torch.zeros(8, 8, device="cuda"), coefficients=(1.0, 1e300, 0.0))


@pytest.mark.parametrize("m,n", [(136, 1 << 20), (1 << 18, 200)])
def test_a_long_side_of_a_million(lib, m, n):  # noqa: F811
    """G sums squares along the long side; a matrix unit truncates its accumulator towards zero.  The result's
    rounding (1.7e-3) and the 11-bit operands' 2e-3 leave the norm of the error below 2^-8."""
    g = torch.Generator(device="cuda").manual_seed(m)
    side = min(m, n)
    u = torch.randn(side, max(m, n), generator=g, device="cuda") * torch.logspace(0, -1, side, device="cuda")[:, None]
    u = (u if m < n else u.T).to(F16)
    y = lib.orthogonalize(u)
    # the polynomial of the eigenvalues of X X^T, in 64 bits
    x = (u if m < n else u.T).double()
    gram = x @ x.T
    norm = gram.trace().sqrt() + 1e-7
    value, basis = torch.linalg.eigh(gram / norm ** 2)
    factor = torch.ones_like(value)
    for _ in range(5):
        t = 3.4445 - 4.7750 * value + 2.0315 * value ** 2
        factor, value = factor * t, value * t * t
    ref = (basis * (factor / norm)) @ (basis.T @ x)
    assert float(((y if m < n else y.T).double() - ref).norm()) <= 2.0 ** -8 * float(ref.norm())
