"""orthogonalize on the GPU where rounding could grow: many steps on low rank
and steep spectra, coefficients that take the operands out of the range of the
default ones."""

import pytest
import torch

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
