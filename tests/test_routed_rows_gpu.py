"""expert_plan, dispatch_rows and combine_rows on the GPU against a stable sort
and sums in 64 bits: sizes from one row up, rows without an expert, widths of
every alignment, gradients, plans that are not one."""

import pytest
import torch

import routed_reference as ref
from layer_reference import UNIT, assert_within, sum_bound
from test_grouped_gpu import lib  # noqa: F401

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
SPMM_DEV_BAD_COLUMN = 1


def experts_of(tokens, k, num, seed=0, dropped=0.1, dtype=torch.int32):
    g = torch.Generator().manual_seed(seed)
    e = torch.randint(0, num, (tokens, k), generator=g)
    e[torch.rand(tokens, k, generator=g) < dropped] = -1
    return e.to(dtype).cuda()


def normal(*shape, dtype=F32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def check_plan(lib, e, num):  # noqa: F811
    got = lib.expert_plan(e, num)
    for a, b, name in zip(got, ref.plan_reference(e, num), ("group_ptr", "position", "source")):
        assert a.dtype == torch.int32 and torch.equal(a.cpu(), b), name
    return got


@pytest.mark.parametrize("tokens,k,num", [(1, 1, 1), (1, 4, 32), (9, 4, 32), (31, 1, 5), (32, 1, 5), (33, 2, 1024), (1000, 4, 3),
                                          (1024, 4, 64), (1025, 4, 64), (4099, 2, 46), (5001, 7, 1023), (70000, 8, 256)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_plan(lib, tokens, k, num, dtype):  # noqa: F811
    check_plan(lib, experts_of(tokens, k, num, seed=tokens, dtype=dtype), num)


@pytest.mark.parametrize("n", [2047, 2048, 2049, 8191, 8192, 8193, 10240, 10241, 131072, 131073, 524288, 524289])
@pytest.mark.parametrize("num", [64, 257, 1024])
def test_plan_where_its_blocks_change(lib, n, num):  # noqa: F811
    check_plan(lib, experts_of(n, 1, num, seed=n), num)


@pytest.mark.parametrize("tokens", [50, 6000])
def test_plan_of_unequal_loads(lib, tokens):  # noqa: F811
    """One expert has every row; none has any; experts without rows between others."""
    check_plan(lib, torch.full((tokens, 2), 6, dtype=torch.int32, device="cuda"), 9)
    ptr, position, source = check_plan(lib, torch.full((tokens, 2), -1, dtype=torch.int32, device="cuda"), 9)
    assert int(ptr[-1]) == 0 and bool((position == -1).all()) and bool((source == -1).all())
    check_plan(lib, 3 * experts_of(tokens, 2, 3, dropped=0.0), 9)


def test_plan_without_rows(lib):  # noqa: F811
    ptr, position, source = lib.expert_plan(torch.empty(0, 3, dtype=torch.int32, device="cuda"), 5)
    assert torch.equal(ptr.cpu(), torch.zeros(6, dtype=torch.int32)) and position.shape == (0, 3) and source.shape == (0,)


@pytest.mark.parametrize("tokens", [40, 3000])
def test_experts_out_of_range_raise_the_status(lib, tokens):  # noqa: F811
    e = experts_of(tokens, 2, 8, seed=1, dropped=0.0, dtype=torch.int64)
    e[7, 1], e[9, 0], e[11, 0] = 8, -2, 1 << 40
    check_plan(lib, e, 8)
    code, detail = lib.device_status(True)
    assert code == SPMM_DEV_BAD_COLUMN and detail in (15, 18, 22)


def check_rows(lib, e, num, width, dtype, seed=0):  # noqa: F811
    tokens, k = e.shape
    _, position, source = lib.expert_plan(e, num)
    x, out = normal(tokens, width, dtype=dtype, seed=seed), normal(tokens * k, width, dtype=dtype, seed=seed + 1)
    w, dy = normal(tokens, k, seed=seed + 2), normal(tokens, width, dtype=dtype, seed=seed + 3)
    drows = normal(tokens * k, width, dtype=dtype, seed=seed + 4)
    live = (source >= 0)[:, None]
    token = source.clamp(min=0).long() // k

    xl, ol, wl = (t.clone().requires_grad_(True) for t in (x, out, w))
    rows = lib.dispatch_rows(xl, position, source)
    assert torch.equal(rows.detach(), torch.where(live, x[token], torch.zeros_like(out)))
    y = lib.combine_rows(ol, position, source, wl)
    assert_within(y.detach(), *ref.combine_reference(out, position, w), "y")
    plain = lib.combine_rows(out, position, source)
    assert_within(plain, *ref.combine_reference(out, position), "y without weights")

    (dx,) = torch.autograd.grad(rows, xl, drows)
    assert_within(dx, *ref.combine_reference(drows, position), "dx")
    dout, dw = torch.autograd.grad(y, [ol, wl], dy)
    each = w.double().reshape(-1)[source.clamp(min=0).long()][:, None] * dy.double()[token]
    each = torch.where(live, each, torch.zeros_like(each))
    assert_within(dout, each, 2.0 ** -24 * each.abs(), "drows")   # the product's fp32 rounding
    r = torch.where((position >= 0)[:, :, None], out.double()[position.clamp(min=0).long()], 0.0)
    terms = r * dy.double()[:, None, :]
    assert_within(dw, terms.sum(2), sum_bound(width) * terms.abs().sum(2), "dw")
    # one gradient at a time, and the unweighted combine's
    assert torch.equal(torch.autograd.grad(lib.combine_rows(ol, position, source, w), ol, dy)[0], dout)
    assert torch.equal(torch.autograd.grad(lib.combine_rows(out, position, source, wl), wl, dy)[0], dw)
    (du,) = torch.autograd.grad(lib.combine_rows(ol, position, source), ol, dy)
    assert torch.equal(du, torch.where(live, dy[token], torch.zeros_like(out)))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("width", [1, 2, 3, 4, 6, 7, 8, 12, 31, 64, 100, 129, 256, 1000, 1001, 1023, 1024, 2050, 4096, 5000])
def test_widths(lib, width, dtype):  # noqa: F811
    check_rows(lib, experts_of(37, 3, 6, seed=width), 6, width, dtype, seed=width)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("tokens,k,num", [(1, 1, 1), (1, 8, 16), (2, 1, 3), (9, 4, 32), (33, 5, 7), (300, 1, 4), (2100, 6, 64),
                                          (17, 40, 50)])
@pytest.mark.parametrize("width", [72, 57])
def test_numbers_of_rows(lib, tokens, k, num, width, dtype):  # noqa: F811
    check_rows(lib, experts_of(tokens, k, num, seed=tokens), num, width, dtype, seed=k)


@pytest.mark.parametrize("width", [64, 65])
def test_rows_without_any_expert(lib, width):  # noqa: F811
    check_rows(lib, torch.full((40, 3), -1, dtype=torch.int32, device="cuda"), 4, width, BF16)
    e = experts_of(100, 2, 4, seed=3)
    e[20:70] = -1
    check_rows(lib, e, 4, width, BF16)


def test_no_rows(lib):  # noqa: F811
    ptr, position, source = lib.expert_plan(torch.empty(0, 2, dtype=torch.int32, device="cuda"), 3)
    x = torch.empty(0, 16, device="cuda", requires_grad=True)
    rows = lib.dispatch_rows(x, position, source)
    y = lib.combine_rows(rows, position, source, torch.empty(0, 2, device="cuda"))
    assert rows.shape == y.shape == (0, 16)
    y.sum().backward()
    assert x.grad.shape == (0, 16)


def test_values_that_are_not_finite_stay_where_they_are(lib):  # noqa: F811
    e = experts_of(64, 2, 4, seed=5, dropped=0.3)
    _, position, source = lib.expert_plan(e, 4)
    out, w = normal(128, 24), normal(64, 2)
    out[source < 0] = float("nan")          # behind the last row: read by nobody
    hit = int(position[position >= 0][0])
    out[hit, 3] = float("inf")
    w = torch.where(position < 0, torch.full_like(w, float("nan")), w)   # weights of choices without an expert
    y = lib.combine_rows(out, position, source, w)
    bad = ~torch.isfinite(y)
    token = int(source[hit]) // 2
    assert bool(bad[token, 3]) and int(bad.sum()) == 1


@pytest.mark.parametrize("width", [32, 33])
def test_positions_out_of_range_raise_the_status(lib, width):  # noqa: F811
    e = experts_of(50, 2, 4, seed=6, dropped=0.0)
    _, position, source = lib.expert_plan(e, 4)
    x, out, w, dy = normal(50, width), normal(100, width), normal(50, 2), normal(50, width)
    bad = position.clone()
    bad[3, 1], bad[4, 0] = 100, -7
    as_none = position.clone()
    as_none[3, 1] = as_none[4, 0] = -1
    assert_within(lib.combine_rows(out, bad, source, w), *ref.combine_reference(out, as_none, w))
    assert lib.device_status(True)[0] == SPMM_DEV_BAD_COLUMN
    lib.dispatch_rows(x, bad, source)
    assert lib.device_status(True)[0] == SPMM_DEV_BAD_COLUMN
    wl = w.clone().requires_grad_(True)
    (dw,) = torch.autograd.grad(lib.combine_rows(out, bad, source, wl), wl, dy)
    assert lib.device_status(True)[0] == SPMM_DEV_BAD_COLUMN
    assert float(dw[3, 1]) == 0 and float(dw[4, 0]) == 0


def test_strided_and_misaligned_inputs(lib):  # noqa: F811
    e = experts_of(60, 2, 4, seed=2)
    _, position, source = lib.expert_plan(e.T.contiguous().T, 4)
    for a, b in zip((position, source), lib.expert_plan(e, 4)[1:]):
        assert torch.equal(a, b)
    base = normal(60, 200, dtype=F16)
    want = lib.dispatch_rows(base[:, 3:99].contiguous(), position, source)
    assert torch.equal(lib.dispatch_rows(base[:, 3:99], position, source), want)
    odd = torch.empty(60 * 96 + 1, dtype=F16, device="cuda")[1:].view(60, 96)
    odd.copy_(base[:, 3:99])
    assert torch.equal(lib.dispatch_rows(odd, position, source), want)
    y = lib.combine_rows(want, position, source, normal(2, 60).T)
    assert torch.equal(y, lib.combine_rows(want, position, source, normal(2, 60).T.contiguous()))


def test_another_stream_and_captured(lib):  # noqa: F811
    e, x, w = experts_of(500, 4, 16, seed=1), normal(500, 96, dtype=BF16), normal(500, 4)

    def call():
        ptr, position, source = lib.expert_plan(e, 16)
        rows = lib.dispatch_rows(x, position, source)
        return ptr, position, source, rows, lib.combine_rows(rows, position, source, w)

    want = call()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = call()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for seed in (1, 2, 3):
        e.copy_(experts_of(500, 4, 16, seed=seed, dropped=0.2 * seed))
        x.copy_(normal(500, 96, dtype=BF16, seed=seed))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, call()))


def test_refusals(lib):  # noqa: F811
    e = experts_of(6, 2, 4)
    _, position, source = lib.expert_plan(e, 4)
    x, out, w = normal(6, 16), normal(12, 16), normal(6, 2)
    for call, text in ((lambda: lib.expert_plan(e.float(), 4), "int32 or int64"),
                       (lambda: lib.expert_plan(e, 0), "number of experts"),
                       (lambda: lib.expert_plan(e, 1025), "number of experts"),
                       (lambda: lib.expert_plan(e.cpu(), 4), "must be CUDA tensor"),
                       (lambda: lib.dispatch_rows(x.double(), position, source), "supports only FP16, BF16 and FP32"),
                       (lambda: lib.dispatch_rows(x[:5], position, source), "same number of rows"),
                       (lambda: lib.dispatch_rows(x, position.long(), source), "contiguous int32"),
                       (lambda: lib.dispatch_rows(x, position, source[:11]), "one entry per position"),
                       (lambda: lib.dispatch_rows(x, position.view(-1), source), "must have shape"),
                       (lambda: lib.dispatch_rows(x[:, :0], position, source), "feature width"),
                       (lambda: lib.combine_rows(x, position, source), "one row per position"),
                       (lambda: lib.combine_rows(out, position, source, w.half()), "weights must be FP32"),
                       (lambda: lib.combine_rows(out, position, source, w[:, :1]), "weights must be FP32"),
                       (lambda: lib.combine_rows(out.cpu(), position, source), "must be CUDA tensor")):
        with pytest.raises(RuntimeError, match=text):
            call()
    wl = w.clone().requires_grad_(True)
    (dw,) = torch.autograd.grad(lib.combine_rows(out, position, source, wl).sum(), wl, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        dw.sum().backward()


def test_gradients_against_differences(lib):  # noqa: F811
    """combine is linear in rows and in weights: a difference of two calls in fp32 is its derivative."""
    e = experts_of(30, 3, 5, seed=8)
    _, position, source = lib.expert_plan(e, 5)
    out, w, dy, v, u = normal(90, 20), normal(30, 3, seed=1), normal(30, 20, seed=2), normal(90, 20, seed=3), normal(30, 3, seed=4)
    ol, wl = out.clone().requires_grad_(True), w.clone().requires_grad_(True)
    do, dw = torch.autograd.grad(lib.combine_rows(ol, position, source, wl), [ol, wl], dy)
    f = lambda o, ws: float((lib.combine_rows(o, position, source, ws).double() * dy.double()).sum())  # noqa: E731
    size = float((ref.combine_reference(out, position, w)[0].abs() * dy.double().abs()).sum())
    slack = 64 * UNIT[F32] * 8 * size + 1e-3   # roundings of the two calls and of out +- v
    assert abs(float((do.double() * v.double()).sum()) - (f(out + v, w) - f(out - v, w)) / 2) < slack
    assert abs(float((dw.double() * u.double()).sum()) - (f(out, w + u) - f(out, w - u)) / 2) < slack
