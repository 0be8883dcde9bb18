"""Arrays of more than 2^31 elements, two calls at once on two streams, and the
last rows of what the operators around routed experts read and write."""

import pytest
import torch

from test_grouped_gpu import lib  # noqa: F401

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def last_rows(t, n=3):
    return t[-n:].clone()


@pytest.mark.parametrize("width", [1024, 1021])
def test_rows_past_32_bits(lib, width):  # noqa: F811
    tokens, k = 1_100_000, 2   # 2.2 million rows: 2.25e9 elements
    assert tokens * k * width > 1 << 31
    e = torch.arange(tokens * k, device="cuda").view(tokens, k).remainder(7).int()
    _, position, source = lib.expert_plan(e, 7)
    x = torch.randn(tokens, width, device="cuda", dtype=BF16)
    w = torch.rand(tokens, k, device="cuda")
    rows = lib.dispatch_rows(x, position, source)
    for r in (0, tokens * k // 2, tokens * k - 1):
        assert torch.equal(rows[r], x[int(source[r]) // k])
    y = lib.combine_rows(rows, position, source, w)
    for t in (0, tokens - 1):
        want = (w[t, 0] * x[t].float() + w[t, 1] * x[t].float())
        assert float((y[t].float() - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max()) + 1e-6
    wl = w.clone().requires_grad_(True)
    rl = rows.requires_grad_(True)
    dr, dw = torch.autograd.grad(lib.combine_rows(rl, position, source, wl), [rl, wl], x)
    t = tokens - 1
    p = position[t].long()
    want = (w[t][:, None] * x[t].float()).to(BF16)
    assert torch.equal(dr[p], want)
    dots = (rows.detach()[p].double() * x[t].double()).sum(1)
    assert float((dw[t].double() - dots).abs().max()) < 1e-4 * width


def test_a_table_past_32_bits(lib):  # noqa: F811
    rows, width = 2_200_000, 1000
    assert rows * width > 1 << 31
    table = torch.randn(rows, width, device="cuda", dtype=BF16)
    ids = torch.tensor([0, rows - 1, 5, rows - 1, rows // 2], device="cuda")
    y = lib.embedding(ids, table)
    assert torch.equal(y, table[ids])
    dy = torch.randn(5, width, device="cuda", dtype=BF16)
    d = lib.embedding_grad(ids, dy, rows)
    assert torch.equal(d[rows - 1], (dy[1].float() + dy[3].float()).to(BF16)) and torch.equal(d[0], dy[0])
    assert bool((d[1:5] == 0).all()) and bool((d[rows - 100:rows - 1] == 0).all())


def test_products_past_32_bits(lib):  # noqa: F811
    rows, K, N = 1_100_000, 128, 2048
    assert rows * N > 1 << 31
    ptr = torch.tensor([0, 700_001, rows], dtype=torch.int32, device="cuda")
    x = torch.randn(rows, K, device="cuda", dtype=BF16)
    wq, ws = lib.quantize_weight_fp8(torch.randn(2, K, N, device="cuda", dtype=BF16))
    q, s = lib.quantize_fp8(x)
    y = lib.grouped_matmul_fp8(q, s, wq, ws, ptr)
    for r in (0, 700_000, 700_001, rows - 1):
        g = int(r >= 700_001)
        w = wq[g].double() * ws[g].double().repeat_interleave(128, 0)
        want = (q[r].double() * s[r].double()) @ w.T
        mag = (q[r].double() * s[r].double()).abs() @ w.abs().T
        assert bool(((y[r].double() - want).abs() <= 2.0 ** -8 * want.abs() + 32 * 2.0 ** -23 * mag).all())


def test_scores_past_32_bits(lib):  # noqa: F811
    tokens, experts = 8_500_000, 256
    assert tokens * experts > 1 << 31
    x = torch.randn(tokens, experts, device="cuda", dtype=BF16)
    w, e = lib.route_experts(x, 4)
    last = lib.route_experts(last_rows(x), 4)
    assert torch.equal(w[-3:], last[0]) and torch.equal(e[-3:], last[1])
    xl = x.requires_grad_(True)
    w, _ = lib.route_experts(xl, 4)
    (dx,) = torch.autograd.grad(w, xl, torch.ones_like(w[:1]).expand_as(w) * torch.arange(4, device="cuda"))
    ll = last_rows(x.detach()).requires_grad_(True)
    wl, _ = lib.route_experts(ll, 4)
    (dl,) = torch.autograd.grad(wl, ll, torch.arange(4, device="cuda", dtype=F32).expand(3, 4))
    assert torch.equal(dx[-3:], dl)


def test_two_streams_at_once(lib):  # noqa: F811
    """Each call has its own workspace: results of calls that overlap are those of calls one after the other."""
    g = torch.Generator(device="cuda").manual_seed(0)
    ids = [torch.randint(0, 3000, (60000,), generator=g, device="cuda") for _ in range(2)]
    dy = [torch.randn(60000, 96, generator=g, device="cuda") for _ in range(2)]
    e = [torch.randint(0, 64, (30000, 2), generator=g, device="cuda", dtype=torch.int32) for _ in range(2)]
    want = [(lib.embedding_grad(ids[i], dy[i], 3000), *lib.expert_plan(e[i], 64)) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i] = (lib.embedding_grad(ids[i], dy[i], 3000), *lib.expert_plan(e[i], 64))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want[i]))
