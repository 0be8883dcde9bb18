"""grouped_matmul_fp8 with scales whose product leaves fp32's range: results that
fp32 holds are as exact as any others, and rows do not depend on their neighbours'."""

import pytest
import torch

import routed_reference as ref
from test_grouped_gpu import lib  # noqa: F401

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
MAX = torch.finfo(F32).max
# rows of the groups, K, N: tiles of 64 and of 128 columns, and of 256 x 256 on pairs of blocks
SHAPES = [([20, 0, 33], 272, 48), ([1500] * 6 + [3], 400, 544), ([9000, 10500], 272, 256)]


def normal(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda")


def ptr_of(sizes):
    return torch.tensor([0, *torch.tensor(sizes).cumsum(0).tolist()], dtype=torch.int32, device="cuda")


def check(lib, q, s, wq, ws, ptr, least=2.0 ** -149):  # noqa: F811
    """The results that fp32 holds, and whose terms it holds.  Slack: that of the sum; a block's product with the scales
    rounds once more than there, by 2^-23 of itself (part of that sum's 2^-23 a step); 2^-150 for each rounding of a
    subnormal term or sum."""
    y = lib.grouped_matmul_fp8(q, s, wq, ws, ptr, F32)
    want, slack = ref.fp8_reference(q, s, wq, ws, ptr)
    size = slack / ref.sum_bound(q.shape[1])   # the sum of the products' magnitudes
    held = size < MAX / 2
    err = (y.double() - want).abs()
    bound = 2.0 ** -24 * want.abs() + slack + (2 * s.shape[1] + 1) * 2.0 ** -150
    bad = held & ~(err <= bound)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[0].tolist(), y[bad][0].item(), want[bad][0].item())
    some = held & (want.abs() > 2.0 ** 20 * least)
    return y, held, int(some.sum())


@pytest.mark.parametrize("sizes,K,N", SHAPES)
@pytest.mark.parametrize("row,weight", [(-55, -55), (-64, -60), (-20, -100), (-90, -45), (-70, -72), (-98, -98)])
def test_small_operands(lib, sizes, K, N, row, weight):  # noqa: F811
    """Block maxima whose product is 2^-105 to 2^-190: the scales' is subnormal or zero in fp32, the result is not at first."""
    x = normal(sum(sizes), K) * 2.0 ** row
    w = normal(len(sizes), K, N, seed=1) * 2.0 ** weight
    (q, s), (wq, ws) = lib.quantize_fp8(x), lib.quantize_weight_fp8(w)
    assert float((q.float() != 0).float().mean()) > 0.9 and float((wq.float() != 0).float().mean()) > 0.9
    *_, some = check(lib, q, s, wq, ws, ptr_of(sizes))
    assert some > 0 or row + weight < -125


@pytest.mark.parametrize("sizes,K,N", SHAPES)
@pytest.mark.parametrize("power", [61, 57])
def test_large_operands(lib, sizes, K, N, power):  # noqa: F811
    """Block maxima of 2^73 on either side that do not meet: the scales' product is infinite, the sums are 0 or fit."""
    x, w = normal(sum(sizes), K) * 2.0 ** power, normal(len(sizes), K, N, seed=1) * 2.0 ** power
    x[:, 5::128], w[:, 5::128] = 2.0 ** 73, 0
    w[:, 9::128, 3::128], x[:, 9::128] = 2.0 ** 73, 0
    x[1::7] = 0
    x[1::7, 5::128] = 2.0 ** 73      # nothing meets a weight
    (q, s), (wq, ws) = lib.quantize_fp8(x), lib.quantize_weight_fp8(w)
    assert bool((s[:, :1, None] * ws[:1].flatten() > MAX).any())
    y, held, some = check(lib, q, s, wq, ws, ptr_of(sizes))
    assert bool((y[1::7] == 0).all())
    if power < 61:   # of 61, the magnitudes sum up to K 2^122 2 / pi and may leave fp32: K 2^114 2 / pi does not
        assert bool(held.all()) and some > 0


@pytest.mark.parametrize("sizes,K,N", SHAPES)
def test_scales_of_any_size(lib, sizes, K, N):  # noqa: F811
    """Blocks of a row from one end to the other, of either sign."""
    g = torch.Generator(device="cuda").manual_seed(7)
    rows, G = sum(sizes), len(sizes)
    kb, nb = -(-K // 128), -(-N // 128)
    q = (8 * normal(rows, K)).to(torch.float8_e4m3fn)
    wq = (8 * normal(G, N, K, seed=1)).to(torch.float8_e4m3fn)
    power = lambda *s: torch.exp2(torch.rand(*s, generator=g, device="cuda") * 210 - 108) * normal(*s, seed=3)  # noqa: E731
    s, ws = power(rows, kb), power(G, nb, kb)
    s[::5] = normal(rows, kb)[::5] * 1e-3
    *_, some = check(lib, q, s, wq, ws, ptr_of(sizes))
    assert some > 100


@pytest.mark.parametrize("sizes,K,N", SHAPES)
def test_rows_do_not_depend_on_their_neighbours(lib, sizes, K, N):  # noqa: F811
    rows, G = sum(sizes), len(sizes)
    x, w = normal(rows, K), normal(G, K, N, seed=1)
    (q, s), (wq, ws) = lib.quantize_fp8(x), lib.quantize_weight_fp8(w)
    want = lib.grouped_matmul_fp8(q, s, wq, ws, ptr_of(sizes), BF16)
    far = s.clone()
    far[3::11] = 2.0 ** -140
    far[4::11] = float("inf")
    far[5::11] = 0
    far[6::11] = float("nan")
    y = lib.grouped_matmul_fp8(q, far, wq, ws, ptr_of(sizes), BF16)
    index = torch.arange(rows, device="cuda") % 11
    same = (index < 3) | (index > 6)
    assert torch.equal(y[same], want[same])
    assert bool((y[index == 5] == 0).all()) and bool(torch.isnan(y[index == 6]).all())
    assert bool((~torch.isfinite(y[index == 4])).all())
    assert bool((y[index == 3].float().abs() < 2.0 ** -110).all()) and bool((y[index == 3] != 0).any())


@pytest.mark.parametrize("sizes,K,N", SHAPES)
def test_captured_and_on_two_streams(lib, sizes, K, N):  # noqa: F811
    """One graph replayed with ordinary and far scales; calls with either at once."""
    (q, near), (wq, ws) = lib.quantize_fp8(normal(sum(sizes), K)), lib.quantize_weight_fp8(normal(len(sizes), K, N, seed=1))
    far = near.clone()
    far[::3] = 2.0 ** -140
    call = lambda s: lib.grouped_matmul_fp8(q, s, wq, ws, ptr, BF16)  # noqa: E731
    ptr, s = ptr_of(sizes), far.clone()
    want = [call(far), call(near)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call(s)
    for i in (0, 1, 0, 1):
        s.copy_((far, near)[i])
        graph.replay()
        assert torch.equal(y, want[i])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got.append(call((far, near)[i]))
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
