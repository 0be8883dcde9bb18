"""Groups of experts under biases that are large against the scores: a group's
two best values nearly cancel, so that the order of the sums hangs on what each
term lost.  The choice is that of 64-bit scores, row by row."""

import pytest
import torch

from test_grouped_gpu import lib  # noqa: F401

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def chosen(x, k, bias, scoring, groups, top_groups, best):
    """[T, k] from 64-bit scores; equal values to the lowest index."""
    c = (torch.softmax if scoring == "softmax" else lambda v, _: torch.sigmoid(v))(x.double(), 1) + bias.double()
    T, E = c.shape
    score = c.view(T, groups, -1).topk(best, 2).values.sum(2)
    kept = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :top_groups]
    out = torch.ones(T, groups, dtype=torch.bool, device=x.device).scatter_(1, kept, False)
    c = c.masked_fill(out.repeat_interleave(E // groups, 1), -float("inf"))
    return torch.sort(c, dim=1, descending=True, stable=True).indices[:, :k]


def rows_of(tokens, experts, dtype=F32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (1.5 * torch.randn(tokens, experts, generator=g, device="cuda")).to(dtype)


def opposite(experts, groups, size):
    """+size for one expert of each group, -size for the others."""
    g = torch.Generator().manual_seed(experts)
    b = torch.full((groups, experts // groups), -size)
    b[torch.arange(groups), torch.randint(0, experts // groups, (groups,), generator=g)] = size
    return b.view(-1).cuda()


def check(lib, x, k, bias, scoring, groups, top_groups, best=2):  # noqa: F811
    w, e = lib.route_experts(x, k, bias, scoring, groups, top_groups, best)
    off = (e.long() != chosen(x, k, bias, scoring, groups, top_groups, best)).any(1)
    assert not bool(off.any()), (int(off.sum()), off.nonzero().flatten().tolist()[:5])
    assert bool(torch.isfinite(w).all())


@pytest.mark.parametrize("size", [1.0, 2.0, 8.0, 64.0, 100.0])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens,experts,groups,top_groups", [(65537, 256, 8, 4), (65537, 64, 32, 8), (65537, 64, 8, 4),
                                                              (16411, 1024, 8, 4), (16411, 512, 4, 3), (65537, 60, 5, 2),
                                                              (65537, 32, 16, 5), (65537, 96, 32, 7)])
def test_biases_that_cancel(lib, tokens, experts, groups, top_groups, scoring, size):  # noqa: F811
    x = rows_of(tokens, experts, seed=groups)
    check(lib, x, min(8, top_groups * (experts // groups)), opposite(experts, groups, size), scoring, groups, top_groups)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("best", [1, 2])
def test_biases_of_any_size(lib, dtype, scoring, best):  # noqa: F811
    """16-bit logits, biases from small to large in the same row."""
    g = torch.Generator(device="cuda").manual_seed(5)
    for experts, groups, top_groups in ((256, 8, 4), (40, 5, 2), (1024, 32, 9)):
        bias = torch.randn(experts, generator=g, device="cuda")
        bias = bias * torch.exp(2 * torch.randn(experts, generator=g, device="cuda"))
        check(lib, rows_of(16411, experts, dtype, seed=best), 4, bias, scoring, groups, top_groups, best)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_groups_shut_out_by_their_bias(lib, scoring):  # noqa: F811
    """Groups whose experts all have a far lower bias, or an infinite one, beside groups that cancel."""
    for low in (-1e9, -3e38, -float("inf")):
        bias = opposite(256, 8, 8.0)
        bias[32:96] = low
        bias[200:224] = low
        check(lib, rows_of(4099, 256, seed=3), 8, bias, scoring, 8, 4)


def test_bias_near_the_end_of_fp32(lib):  # noqa: F811
    """Sums that leave fp32 are compared in 64 bits."""
    size = torch.finfo(F32).max
    bias = torch.full((64,), size)
    bias[::3] = size * 0.75
    bias[40:48] = size * 0.5
    check(lib, rows_of(300, 64), 4, bias.cuda(), "sigmoid", 8, 3)
    check(lib, rows_of(300, 64), 4, -bias.cuda(), "sigmoid", 8, 3)
