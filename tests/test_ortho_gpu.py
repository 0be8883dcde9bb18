"""orthogonalize on the GPU against its polynomial applied to the singular
values in 64 bits: sizes from one element on, tall, wide and odd ones, batches,
types, degenerate updates, refusals."""

import pytest
import torch

from layer_reference import ortho_reference

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32

# bf16 result: at most 2^-8 per element; the products' operands are held to at
# least 11 bits, each of the fifteen products adds a relative 2^-12 at most to
# the matrix (in the Frobenius norm): 15 * 2^-12
TOLERANCE = 2.0 ** -8 + 15 * 2.0 ** -12


@pytest.fixture(scope="module")
def lib():
    import build

    build.build()
    import spmm_npu

    return spmm_npu


def gradient(batch, m, n, dtype, seed=0, decay=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = 2 * min(m, n) + 16
    left = torch.randn(batch, rows, m, generator=g, device="cuda") * torch.logspace(0, -decay, m, device="cuda")
    right = torch.randn(batch, rows, n, generator=g, device="cuda") * torch.logspace(0, -decay, n, device="cuda")
    return (left.transpose(1, 2) @ right / rows).to(dtype)


def check(lib, u, **kw):
    y = lib.orthogonalize(u, **kw)
    assert y.dtype == BF16 and y.shape == u.shape and y.is_contiguous()
    ref = ortho_reference(u, **kw)
    err = (y.double() - ref).flatten(-2).norm(dim=-1)
    assert bool((err <= TOLERANCE * ref.flatten(-2).norm(dim=-1) + 1e-30).all()), (
        err / ref.flatten(-2).norm(dim=-1)).max()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("m,n", [(1, 1), (1, 40), (40, 1), (2, 3), (16, 16), (31, 33), (64, 128), (128, 64), (65, 64),
                                 (127, 129), (128, 128), (200, 136), (257, 384), (384, 257), (601, 130), (130, 1023),
                                 (512, 1024), (1024, 1024)])
def test_sizes(lib, m, n, dtype):
    check(lib, gradient(1, m, n, dtype, seed=m + n))


@pytest.mark.parametrize("batch,m,n", [(2, 48, 80), (7, 129, 64), (46, 256, 128), (3, 300, 301), (65, 16, 24)])
def test_batches(lib, batch, m, n):
    u = gradient(batch, m, n, F32, seed=batch)
    check(lib, u)
    y = lib.orthogonalize(u)
    check(lib, u[batch - 1])
    assert torch.equal(lib.orthogonalize(u.view(1, batch, m, n))[0], y)


@pytest.mark.parametrize("batch,m,n", [(1, 250, 1030), (1, 1031, 250), (5, 512, 500), (5, 500, 510), (2, 1024, 1000),
                                       (12, 700, 697), (30, 200, 900), (20, 900, 200), (1, 1100, 9000),
                                       (1, 9001, 1100)])
def test_tile_widths(lib, batch, m, n):
    """Sizes on both sides of the rules that choose a product's tiles: one turn of narrow tiles or mirrored ones,
    updates of 64 to 256 columns, alone and in pairs of SMs."""
    check(lib, gradient(batch, m, n, BF16, seed=m))


@pytest.mark.parametrize("decay", [0.0, 3.0])
def test_spectra(lib, decay):
    """Flat and steep spectra; low rank plus noise, where an operand's rounding could grow with the small
    singular values."""
    check(lib, gradient(1, 256, 320, F32, decay=decay))
    g = torch.Generator(device="cuda").manual_seed(1)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    check(lib, n(300, 4) @ n(4, 200) + 0.05 * n(300, 200))


@pytest.mark.parametrize("scale", [1e-30, 1e-6, 1.0, 1e6, 1e30])
def test_scale_does_not_matter(lib, scale):
    u = gradient(2, 96, 160, F32, seed=3) * scale
    check(lib, u, eps=0.0)
    if scale >= 1e-6:   # below, the default eps leaves a matrix of almost zero
        check(lib, u)


def test_steps_and_coefficients(lib):
    u = gradient(1, 100, 70, F32, seed=8)
    for steps in (0, 1, 2, 7):
        check(lib, u, steps=steps)
    check(lib, u, steps=3, coefficients=(1.5, -0.5, 0.0))


def test_degenerate_updates(lib):
    assert not bool(lib.orthogonalize(torch.zeros(2, 40, 30, device="cuda")).any())
    assert lib.orthogonalize(torch.zeros(0, 8, 8, device="cuda")).shape == (0, 8, 8)
    assert lib.orthogonalize(torch.zeros(3, 0, 8, device="cuda")).shape == (3, 0, 8)
    # a non-finite matrix does not reach its neighbours
    u = gradient(3, 64, 96, F32)
    want = lib.orthogonalize(u)
    for bad in (float("nan"), float("inf")):
        v = u.clone()
        v[1, 3, 5] = bad
        y = lib.orthogonalize(v)
        assert torch.equal(y[0], want[0]) and torch.equal(y[2], want[2]) and not bool(y[1].isfinite().any())


def test_strided_update_other_stream_and_graph(lib):
    u = gradient(2, 100, 140, F16, seed=2)
    want = lib.orthogonalize(u)
    assert torch.equal(lib.orthogonalize(u.transpose(1, 2).contiguous().transpose(1, 2)), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = lib.orthogonalize(u)
    side.synchronize()
    assert torch.equal(again, want)
    graph = torch.cuda.CUDAGraph()
    static = torch.zeros_like(u)
    with torch.cuda.graph(graph):
        y = lib.orthogonalize(static)
    static.copy_(u)
    graph.replay()
    assert torch.equal(y, want)


def test_refusals(lib):
    u = torch.zeros(8, 8, device="cuda")
    with pytest.raises(RuntimeError, match="must be CUDA tensor"):
        lib.orthogonalize(u.cpu())
    with pytest.raises(RuntimeError, match="supports only FP16, BF16 and FP32"):
        lib.orthogonalize(u.double())
    with pytest.raises(RuntimeError, match="at least two dimensions"):
        lib.orthogonalize(u[0])
    with pytest.raises(RuntimeError, match="steps must be"):
        lib.orthogonalize(u, steps=-1)
    with pytest.raises(RuntimeError, match="finite"):
        lib.orthogonalize(u, coefficients=(float("nan"), 0.0, 0.0))
    with pytest.raises(RuntimeError, match="eps must not be negative"):
        lib.orthogonalize(u, eps=-1.0)


@pytest.mark.parametrize("m,n", [(8, 300), (128, 257), (513, 128), (100, 2000), (4096, 32), (64, 4097), (129, 600)])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_thin_matrices(lib, m, n, dtype):
    """A short side of at most 128, in several chunks of the long one, and just past both limits."""
    check(lib, gradient(2, m, n, dtype, seed=m))


@pytest.mark.parametrize("batch,m,n", [(1, 30, 4000), (3, 769, 128), (2, 17, 20000), (90, 40, 1100), (2, 1, 5000)])
def test_long_thin_matrices(lib, batch, m, n):
    """One matrix over many blocks, and many matrices over one block each."""
    check(lib, gradient(batch, m, n, F32, seed=m))
    check(lib, gradient(batch, m, n, BF16, seed=m), steps=1)
    check(lib, gradient(batch, m, n, F16, seed=m), steps=0)


@pytest.mark.parametrize("steps", [1, 2, 8, 9])
def test_step_counts_of_thin_matrices(lib, steps):
    check(lib, gradient(2, 96, 300, F32, seed=steps, decay=0.5), steps=steps)
    check(lib, gradient(2, 30, 20, F32, seed=steps, decay=0.5), steps=steps)
