"""route_experts on the GPU against a 64-bit reference: numbers of experts and
choices, ties, masks, groups, biases, types, non-finite values, gradients."""

import pytest
import torch

import routed_reference as ref
from layer_reference import UNIT, assert_within
from test_grouped_gpu import lib  # noqa: F401

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def logits_of(tokens, experts, dtype, seed=0, spread=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (spread * torch.randn(tokens, experts, generator=g, device="cuda")).to(dtype)


def bias_of(experts, seed=1, size=0.1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return size * torch.randn(experts, generator=g, device="cuda")


def same(experts, want):
    off = (experts.cpu().long() != want).any(1)
    assert not bool(off.any()), (off.nonzero().flatten().tolist()[:5], experts[off.cuda()][:2].tolist(), want[off][:2].tolist())


def check(lib, x, k, bias=None, scoring="softmax", groups=1, top_groups=1, group_best=1, renormalize=True,  # noqa: F811
          scale=1.0, grad=True):
    choice = dict(bias=bias, scoring=scoring, groups=groups, top_groups=top_groups, group_best=group_best)
    xl = x.clone().requires_grad_(grad)
    w, e = lib.route_experts(xl, k, renormalize=renormalize, scale=scale, **choice)
    assert w.dtype == torch.float32 and e.dtype == torch.int32 and not e.requires_grad
    same(e, ref.route_choice(x, k, **choice))
    xd = x.double().requires_grad_(True)
    want = ref.route_weights(xd, e, scoring, renormalize, scale)
    rel = 2 * ref.score_error(x, e, scoring)
    assert_within(w.detach(), want.detach(), rel * want.detach().abs() + 2.0 ** -120, "weights")
    if not grad:
        return w, e
    g = logits_of(*e.shape, F32, seed=9)
    (dx,) = torch.autograd.grad(w, xl, g)
    (dwant,) = torch.autograd.grad(want, xd, g.double())
    assert_within(dx, dwant, ref.route_gradient_slack(x, e, g, scoring, renormalize, scale) + 2.0 ** -120, "gradient")
    w2, e2 = lib.route_experts(x, k, renormalize=renormalize, scale=scale, **choice)
    assert torch.equal(w2, w.detach()) and torch.equal(e2, e)
    return w, e


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("experts,k", [(1, 1), (2, 1), (3, 3), (16, 4), (31, 8), (32, 32), (33, 2), (60, 5), (64, 6), (65, 1),
                                       (127, 8), (128, 16), (129, 3), (256, 8), (257, 32), (512, 7), (1000, 10), (1024, 32)])
def test_numbers_of_experts(lib, experts, k, dtype):  # noqa: F811
    check(lib, logits_of(67, experts, dtype, seed=experts), k)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("biased", [False, True])
def test_scores(lib, dtype, scoring, renormalize, biased):  # noqa: F811
    x = logits_of(301, 72, dtype, seed=5)
    check(lib, x, 6, bias=bias_of(72) if biased else None, scoring=scoring, renormalize=renormalize, scale=2.5)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups,top_groups", [(256, 8, 4), (64, 4, 1), (60, 5, 2), (96, 32, 7), (30, 3, 3),
                                                       (1024, 32, 31), (8, 4, 2)])
@pytest.mark.parametrize("best", [1, 2])
@pytest.mark.parametrize("biased", [False, True])
def test_groups(lib, dtype, scoring, experts, groups, top_groups, best, biased):  # noqa: F811
    x = logits_of(130, experts, dtype, seed=groups)
    check(lib, x, min(4, top_groups * (experts // groups)), bias=bias_of(experts) if biased else None, scoring=scoring,
          groups=groups, top_groups=top_groups, group_best=best)


@pytest.mark.parametrize("tokens", [1, 2, 7, 8, 9, 5003])
def test_numbers_of_rows(lib, tokens):  # noqa: F811
    check(lib, logits_of(tokens, 64, BF16, seed=tokens), 4)


def test_no_rows_and_leading_dimensions(lib):  # noqa: F811
    w, e = lib.route_experts(logits_of(0, 8, F32).requires_grad_(True), 2)
    assert w.shape == e.shape == (0, 2)
    w.sum().backward()
    x = logits_of(24, 40, F16)
    w, e = lib.route_experts(x.view(2, 3, 4, 40), 3)
    assert w.shape == e.shape == (2, 3, 4, 3)
    flat = lib.route_experts(x, 3)
    assert torch.equal(w.view(24, 3), flat[0]) and torch.equal(e.view(24, 3), flat[1])


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("options", [{}, {"groups": 8, "top_groups": 3}, {"groups": 8, "top_groups": 3, "group_best": 2}])
@pytest.mark.parametrize("bias", [None, 0.0, 0.25])
def test_ties_go_to_the_lowest_index(lib, dtype, scoring, options, bias):  # noqa: F811
    """Logits of few values; with a bias that is alike everywhere the scores tie as they do."""
    x = torch.round(2 * logits_of(200, 128, F32, seed=3)).to(dtype) / 2
    b = None if bias is None else torch.full((128,), bias, device="cuda")
    check(lib, x, 8, bias=b, scoring=scoring, **options)
    same = torch.zeros(3, 128, dtype=dtype, device="cuda")
    _, e = check(lib, same, 8, bias=b, scoring=scoring, **options)
    assert torch.equal(e.cpu(), torch.arange(8, dtype=torch.int32).expand(3, 8))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_neighbouring_scores_are_told_apart(lib, scoring, biased):  # noqa: F811
    """fp32 logits one unit in the last place apart, in shuffled order: what 64-bit scores say."""
    g = torch.Generator().manual_seed(2)
    steps = torch.stack([torch.randperm(96, generator=g) for _ in range(150)]).double()
    x = (1.0 + steps * 2.0 ** -23).float().cuda()
    check(lib, x, 8, bias=torch.full((96,), 0.125, device="cuda") if biased else None, scoring=scoring)
    b = bias_of(96, size=2.0 ** -22)   # biases as small as the steps
    check(lib, x, 8, bias=b if biased else None, scoring=scoring, groups=6, top_groups=2, group_best=2)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("spread", [20.0, 60.0])
def test_far_logits(lib, scoring, spread):  # noqa: F811
    """Scores down to the end of fp32 and past it."""
    x = logits_of(120, 64, F32, seed=8, spread=spread)
    for renormalize in (False, True):
        w, e = lib.route_experts(x, 6, scoring=scoring, renormalize=renormalize)
        same(e, ref.route_choice(x, 6, scoring=scoring))
        want = ref.route_weights(x.double(), e, scoring, renormalize, 1.0)
        assert_within(w, want, 2 * ref.score_error(x, e, scoring) * want + 2.0 ** -120)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_masked_experts(lib, dtype, scoring):  # noqa: F811
    """Logits of -infinity: chosen last, with a weight of zero and no gradient; rows that leave nothing."""
    x = logits_of(60, 40, dtype, seed=4)
    x[:, 5] = -float("inf")
    x[10:20, 3:] = -float("inf")     # fewer experts than choices
    x[20:25] = -float("inf")         # none
    xl = x.clone().requires_grad_(True)
    w, e = lib.route_experts(xl, 4, scoring=scoring)
    same(e, ref.route_choice(x, 4, scoring=scoring))
    want = ref.route_weights(x.double(), e, scoring, True, 1.0)
    assert_within(w.detach(), want, 2 * ref.score_error(x, e, scoring) * want + 2.0 ** -120)
    assert bool((w[20:25] == 0).all()) and torch.equal(e[20].cpu(), torch.arange(4, dtype=torch.int32))
    (dx,) = torch.autograd.grad(w, xl, torch.ones_like(w))
    assert bool(torch.isfinite(dx).all()) and bool((dx[torch.isneginf(x)] == 0).all())
    lowest = x.clone()
    lowest[torch.isneginf(x)] = torch.finfo(dtype).min   # masks of the type's lowest value
    w2, e2 = lib.route_experts(lowest, 4, scoring=scoring)
    same(e2, ref.route_choice(lowest, 4, scoring=scoring))
    assert bool(torch.isfinite(w2).all())


@pytest.mark.parametrize("options", [{}, {"groups": 5, "top_groups": 2}, {"groups": 5, "top_groups": 2, "group_best": 2}])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_values_that_are_not_finite(lib, options, scoring, biased):  # noqa: F811
    """NaN is chosen last; choices stay in range, distinct and those of the reference; other rows are not touched."""
    x = logits_of(50, 40, F32, seed=6)
    clean = lib.route_experts(x, 4, bias_of(40) if biased else None, scoring, **options)
    x[3, 7] = float("nan")
    x[4, 2:38] = float("nan")
    x[5] = float("nan")
    b = bias_of(40) if biased else None
    w, e = lib.route_experts(x, 4, b, scoring, **options)
    rows = [3, 4, 5] if scoring == "sigmoid" or not (biased or options.get("group_best") == 2) else [5]
    want = ref.route_choice(x, 4, bias=b, scoring=scoring, **options)
    assert torch.equal(e.cpu().long()[rows], want[rows])
    for row in e.tolist():
        assert len(set(row)) == 4 and all(0 <= i < 40 for i in row)
    others = [t for t in range(50) if t not in (3, 4, 5)]
    assert torch.equal(w[others], clean[0][others]) and torch.equal(e[others], clean[1][others])
    if biased:   # a bias of +-infinity forces the choice
        b = b.clone()
        b[11], b[12] = float("inf"), -float("inf")
        y = logits_of(50, 40, F32, seed=6)
        w, e = lib.route_experts(y, 4, b, scoring, **options)
        same(e, ref.route_choice(y, 4, bias=b, scoring=scoring, **options))
        assert bool((e[:, 0] == 11).all()) and not bool((e == 12).any()) and bool(torch.isfinite(w).all())


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_gradient_against_differences(lib, scoring, renormalize):  # noqa: F811
    """<dx, v> is the derivative along v of the weights with the choice fixed (central differences in 64 bits)."""
    x, v, g = logits_of(40, 33, F32, seed=1), logits_of(40, 33, F32, seed=2).double(), logits_of(40, 5, F32, seed=3)
    xl = x.clone().requires_grad_(True)
    w, e = lib.route_experts(xl, 5, scoring=scoring, renormalize=renormalize, scale=1.5)
    (dx,) = torch.autograd.grad(w, xl, g)
    f = lambda y: (ref.route_weights(y, e, scoring, renormalize, 1.5) * g.double()).sum(1)  # noqa: E731
    h = 1e-5
    want = (f(x.double() + h * v) - f(x.double() - h * v)) / (2 * h)
    slack = ref.route_gradient_slack(x, e, g, scoring, renormalize, 1.5) + UNIT[F32] * dx.double().abs()
    # the differences: h^2 of third derivatives (below 100 |g| |v|^3), 2^-52 / h of the values
    slack = (slack * v.abs()).sum(1) + h * h * 100 * g.double().abs().sum(1) * v.abs().amax(1) ** 3 + 1e-9
    assert bool(((dx.double() * v).sum(1) - want).abs().le(slack).all())


def test_strided_and_misaligned_logits(lib):  # noqa: F811
    x = logits_of(33, 129, BF16, seed=7)
    want = lib.route_experts(x[:, 1:65].contiguous(), 3)
    for view in (x[:, 1:65], x[:, 1:65].contiguous().T.contiguous().T):
        got = lib.route_experts(view, 3)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = torch.empty(33 * 64 + 1, dtype=BF16, device="cuda")[1:].view(33, 64)
    odd.copy_(x[:, 1:65])
    got = lib.route_experts(odd, 3)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_captured_and_replayed(lib):  # noqa: F811
    x = logits_of(100, 64, F32, seed=1)
    bias = bias_of(64)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        lib.route_experts(x, 4, bias, "sigmoid", 8, 4, 2)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w, e = lib.route_experts(x, 4, bias, "sigmoid", 8, 4, 2)
    for seed in (1, 2, 3):
        x.copy_(logits_of(100, 64, F32, seed=seed))
        graph.replay()
        want = lib.route_experts(x, 4, bias, "sigmoid", 8, 4, 2)
        assert torch.equal(w, want[0]) and torch.equal(e, want[1])


def test_refusals(lib):  # noqa: F811
    x = logits_of(4, 12, F32)
    for call, text in ((lambda: lib.route_experts(x.double(), 2), "supports only FP16, BF16 and FP32"),
                       (lambda: lib.route_experts(x, 0), "top_k must be"),
                       (lambda: lib.route_experts(x, 13), "top_k must be"),
                       (lambda: lib.route_experts(logits_of(2, 1025, F32), 2), "number of experts"),
                       (lambda: lib.route_experts(x, 2, scoring="tanh"), "softmax or sigmoid"),
                       (lambda: lib.route_experts(x, 2, groups=5), "divide the number of experts"),
                       (lambda: lib.route_experts(x, 2, groups=0), "divide the number of experts"),
                       (lambda: lib.route_experts(x, 2, groups=3, top_groups=4), "top_groups"),
                       (lambda: lib.route_experts(x, 5, groups=3, top_groups=1), "fewer than top_k"),
                       (lambda: lib.route_experts(x, 2, groups=12, top_groups=4, group_best=2), "group_best"),
                       (lambda: lib.route_experts(x, 2, groups=3, top_groups=2, group_best=3), "group_best"),
                       (lambda: lib.route_experts(x, 2, scale=float("nan")), "scale must be finite"),
                       (lambda: lib.route_experts(x, 2, bias=bias_of(11)), "bias must have shape"),
                       (lambda: lib.route_experts(x, 2, bias=bias_of(12).half()), "bias must be FP32"),
                       (lambda: lib.route_experts(x, 2, bias=bias_of(12).cpu()), "must be CUDA tensor")):
        with pytest.raises(RuntimeError, match=text):
            call()
    w, _ = lib.route_experts(x.requires_grad_(True), 2)
    (dx,) = torch.autograd.grad(w.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        dx.sum().backward()


@pytest.mark.parametrize("options", [{}, {"groups": 8, "top_groups": 3}, {"groups": 8, "top_groups": 3, "group_best": 2}])
def test_scores_that_saturate(lib, options):  # noqa: F811
    """Sigmoids that round to 1 (or 0) in 64 bits: without a bias, and with no sums of groups, the logits decide; a bias,
    of zeros too, or such sums compare the scores, which are equal there."""
    x = torch.linspace(40, 60, 64, device="cuda").repeat(5, 1)
    x[1] = 50 + torch.arange(64, device="cuda").flip(0) * 2.0 ** -18
    x[2:] = torch.stack([x[0, torch.randperm(64, generator=torch.Generator().manual_seed(s))] for s in range(3)])
    by_score = torch.arange(4, device="cuda", dtype=torch.int32).expand(5, 4)
    for logits in (x, x - 900):   # scores of 1, and scores of 0
        _, e = lib.route_experts(logits, 4, scoring="sigmoid", **options)
        by_logit = ref.route_choice(logits, 4, scoring="sigmoid", **{**options, "group_best": 1})
        want = by_score.cpu().long() if options.get("group_best") == 2 else by_logit
        assert torch.equal(e.cpu().long(), want)
        _, e = lib.route_experts(logits, 4, torch.zeros(64, device="cuda"), "sigmoid", **options)
        assert torch.equal(e, by_score)
    assert not torch.equal(by_score.cpu().long(), by_logit)
