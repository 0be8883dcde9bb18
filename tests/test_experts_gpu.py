"""Node features, a typed-edge layer and a routed-expert layer in one training
step, and the expert layer served in 8 bits."""

import pytest
import torch

from test_grouped_gpu import lib  # noqa: F401
from test_relational_gpu import edges, relational  # noqa: F401

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


@pytest.fixture(scope="module")
def experts(lib):  # noqa: F811
    import experts

    return experts


def plain(layer, x):
    """The layer's formula expert by expert in 64 bits, for the choice that the layer's own router makes."""
    import spmm_npu

    r = layer.router
    logits = x.detach().float() @ r.gate.detach()
    w, e = spmm_npu.route_experts(logits, bias=r.bias, **r.options)
    up, down = layer.up.double(), layer.down.double()
    y = torch.zeros(x.shape[0], down.shape[2], dtype=torch.float64, device=x.device)
    for t in range(x.shape[0]):
        for j in range(e.shape[1]):
            y[t] = y[t] + w[t, j].double() * (torch.relu(x[t].double() @ up[e[t, j]]) @ down[e[t, j]])
    return y


@pytest.mark.parametrize("options", [{}, {"scoring": "sigmoid", "groups": 4, "top_groups": 2, "group_best": 2, "scale": 1.5}])
def test_layer(experts, options):
    torch.manual_seed(0)
    layer = experts.ExpertLayer(32, 48, 8, 2, **options).cuda()
    x = torch.randn(50, 32, device="cuda", requires_grad=True)
    y = layer(x)
    want = plain(layer, x)
    assert float((y.detach().double() - want.detach()).norm()) < 1e-5 * float(want.detach().norm())
    dy = torch.randn_like(y)
    got = torch.autograd.grad(y, [layer.up, layer.down], dy)
    ref = torch.autograd.grad(want, [layer.up, layer.down], dy.double())
    for a, b in zip(got, ref):
        assert float((a - b).norm()) < 1e-5 * float(b.norm())
    load = layer.router.group_ptr.diff()
    assert int(load.sum()) == 100
    layer.balance(0.01)
    assert torch.equal(layer.router.bias, 0.01 * torch.sign(load.float().mean() - load.float()))


def test_gradients_against_differences(experts):
    """Of the gate and of x, where the choice and the relus' signs do not change."""
    torch.manual_seed(1)
    layer = experts.ExpertLayer(16, 24, 6, 2).cuda()
    x = torch.randn(20, 16, device="cuda", requires_grad=True)
    dy = torch.randn(20, 16, device="cuda")
    dx, dgate = torch.autograd.grad(layer(x), [x, layer.router.gate], dy)

    def f(xv, gate):
        up, down = layer.up.detach().double(), layer.down.detach().double()
        logits = xv @ gate
        w, e = torch.softmax(logits, 1).topk(2, 1)
        w = w / w.sum(1, keepdim=True)
        h = torch.relu(torch.einsum("tk,tjkh->tjh", xv, up[e]))
        return (torch.einsum("tj,tjh,tjhn->tn", w, h, down[e]) * dy.double()).sum()

    g = layer.router.gate.detach().double()
    xd = x.detach().double()
    for grad, at in ((dx, 0), (dgate, 1)):
        v = torch.randn_like(grad).double()
        h = 1e-6
        move = [(xd + s * h * v, g) if at == 0 else (xd, g + s * h * v) for s in (1, -1)]
        want = float(f(*move[0]) - f(*move[1])) / (2 * h)
        assert abs(float((grad.double() * v).sum()) - want) < 1e-4 * float((grad.double() * v).abs().sum())


def test_served_in_8_bits(experts):
    torch.manual_seed(2)
    layer = experts.ExpertLayer(64, 128, 16, 4, dtype=torch.bfloat16).cuda()
    served = layer.quantized()
    for rows in (1, 9, 300):
        x = torch.randn(rows, 64, device="cuda").bfloat16()
        want, got = layer(x).detach(), served(x)
        assert got.dtype == torch.bfloat16 and not got.requires_grad
        # two products whose operands are off by up to 2^-4 / sqrt(3) each, in the root mean square
        assert float((got.float() - want.float()).norm()) < 0.1 * float(want.float().norm())
    state = served.state_dict()
    assert {"up", "up_scale", "down", "down_scale", "router.bias"} <= set(state)


def test_the_state_of_a_served_layer(experts):
    """All of it: another served layer that loads it answers alike; the gate moves with the rest."""
    torch.manual_seed(7)
    served = experts.ExpertLayer(32, 48, 8, 2, scoring="sigmoid", dtype=torch.bfloat16).cuda().quantized()
    other = experts.ExpertLayer(32, 48, 8, 2, scoring="sigmoid", dtype=torch.bfloat16).cuda().quantized()
    x = torch.randn(40, 32, device="cuda").bfloat16()
    want = served(x)
    assert not torch.equal(other(x), want)
    other.load_state_dict(served.state_dict())
    assert torch.equal(other(x), want)
    assert not any(p.requires_grad for p in served.parameters())
    served.cpu()
    assert all(t.device.type == "cpu" for t in (served.router.gate, *served.state_dict().values()))
    assert torch.equal(served.cuda()(x), want)


def test_a_layer_cast_to_16_bits(experts):
    """Its scores stay fp32: those of the rounded gate and bias, so the same experts as the uncast layer that holds them."""
    torch.manual_seed(5)
    layer = experts.ExpertLayer(32, 48, 8, 2, scoring="sigmoid").cuda()
    layer.router.bias.normal_()
    layer.bfloat16()
    x = torch.randn(60, 32, device="cuda").bfloat16()
    y = layer(x)
    assert y.dtype == torch.bfloat16
    twin = experts.ExpertLayer(32, 48, 8, 2, dtype=torch.bfloat16, scoring="sigmoid").cuda()
    with torch.no_grad():
        for name in ("up", "down"):
            getattr(twin, name).copy_(getattr(layer, name))
        twin.router.gate.copy_(layer.router.gate)
        twin.router.bias.copy_(layer.router.bias)
    assert torch.equal(twin(x), y) and torch.equal(layer.router.group_ptr, twin.router.group_ptr)
    y.float().sum().backward()
    assert all(p.grad.dtype == torch.bfloat16 and bool(torch.isfinite(p.grad).all()) for p in layer.parameters())


@pytest.mark.parametrize("cast", [lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.to(torch.bfloat16),
                                  lambda m: m.to("cpu", torch.float16).cuda(), lambda m: torch.nn.Sequential(m).half()[0]])
def test_a_served_layer_cast_to_16_bits(experts, cast):
    """Its 8-bit weights and their scales stay as they are; it answers as the layer of the cast gate."""
    torch.manual_seed(6)
    layer = experts.ExpertLayer(32, 48, 8, 2, dtype=torch.bfloat16).cuda()
    served, twin = layer.quantized(), layer.quantized()
    names = ["up", "up_scale", "down", "down_scale"]
    before = {name: served.state_dict()[name].clone() for name in names}
    order = list(served.state_dict())
    served = cast(served)
    assert list(served.state_dict()) == order
    for name in names:
        now = served.state_dict()[name]
        assert now.dtype == before[name].dtype and now.is_cuda and torch.equal(now.float(), before[name].float()), name
    assert served.router.gate.dtype in (torch.float16, torch.bfloat16)
    twin.router.gate.copy_(served.router.gate)
    x = torch.randn(40, 32, device="cuda").bfloat16()
    assert torch.equal(served(x), twin(x))


def test_balance_of_a_layer_cast_to_16_bits(experts):
    """The bias stays fp32: small steps add up at any size of it."""
    torch.manual_seed(8)
    layer = experts.ExpertLayer(32, 48, 8, 2, scoring="sigmoid").cuda().bfloat16()
    layer.router.bias.copy_(torch.linspace(-3, 3, 8, device="cuda"))
    x = torch.randn(60, 32, device="cuda").bfloat16()
    want = layer.router.bias.double()
    for _ in range(5):
        layer(x)
        load = layer.router.group_ptr.diff().double()
        want = want + 1e-3 * torch.sign(load.mean() - load)
        layer.balance(1e-3)
    # five sums and their step, each off by at most 2^-24 of 4
    assert float((layer.router.bias.double() - want).abs().max()) <= 6 * 2.0 ** -22
    assert layer.router.bias.dtype == torch.float32 and layer.half().quantized().bfloat16().router.bias.dtype == torch.float32


def test_a_bias_that_was_saved_in_16_bits(experts):
    """Copied into the fp32 one, or put in its place: the layer answers alike."""
    torch.manual_seed(10)
    layer, other = (experts.ExpertLayer(32, 48, 8, 2, scoring="sigmoid").cuda() for _ in range(2))
    layer.router.bias.copy_(torch.randn(8, device="cuda").bfloat16())
    state = layer.state_dict()
    state["router.bias"] = state["router.bias"].bfloat16()
    x = torch.randn(60, 32, device="cuda")
    want = layer(x)
    other.load_state_dict(state)
    assert other.router.bias.dtype == torch.float32 and torch.equal(other(x), want)
    other.load_state_dict(state, assign=True)
    assert other.router.bias.dtype == torch.bfloat16 and torch.equal(other(x), want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_under_autocast(experts, dtype):
    """The scores stay fp32: the same experts, results and gradients as without it."""
    torch.manual_seed(9)
    layer = experts.ExpertLayer(64, 48, 32, 4, scoring="sigmoid").cuda()
    x = torch.randn(300, 64, device="cuda", requires_grad=True)
    dy = torch.randn(300, 64, device="cuda")
    want = layer(x)
    want_ptr = layer.router.group_ptr
    want_grads = torch.autograd.grad(want, [x, *layer.parameters()], dy)
    with torch.autocast("cuda", dtype=dtype):
        got = layer(x)
        served = layer.quantized()(x.detach())
    assert torch.equal(got, want) and torch.equal(layer.router.group_ptr, want_ptr)
    for a, b in zip(torch.autograd.grad(got, [x, *layer.parameters()], dy), want_grads):
        assert torch.equal(a, b)
    assert torch.equal(served, layer.quantized()(x.detach()))


def test_no_rows(experts):
    layer = experts.ExpertLayer(32, 48, 8, 2).cuda()
    x = torch.empty(0, 32, device="cuda", requires_grad=True)
    y = layer(x)
    assert y.shape == (0, 32) and layer.router.group_ptr.tolist() == [0] * 9
    y.sum().backward()
    assert x.grad.shape == x.shape and all(bool((p.grad == 0).all()) for p in layer.parameters())
    layer.balance()
    assert layer.quantized()(x.detach()).shape == (0, 32)
    ids = torch.empty(0, dtype=torch.int64, device="cuda")
    features = experts.NodeFeatures(10, 32).cuda()
    features(ids).sum().backward()
    assert bool((features.table.grad == 0).all())


def test_a_training_step_of_them_together(experts, relational):  # noqa: F811
    torch.manual_seed(3)
    n, relations = 80, 3
    graph = relational.RelationalGraph(*edges(n, relations, 400, seed=7), n, relations)
    model = torch.nn.ModuleDict({
        "features": experts.NodeFeatures(200, 32, scale=2.0, padding_id=0),
        "edges": relational.RelationalLayer(graph, 32, 32),
        "experts": experts.ExpertLayer(32, 64, 8, 2, scoring="sigmoid", out_features=16),
    }).cuda()
    ids = torch.randint(0, 200, (n,), device="cuda")
    optimiser = relational.OrthogonalMomentum(model.parameters(), lr=0.01)

    def loss_of():
        h = model["edges"](model["features"](ids))
        return (model["experts"](h) ** 2).mean()

    loss = loss_of()
    loss.backward()
    for name, p in model.named_parameters():
        assert p.grad is not None and bool(torch.isfinite(p.grad).all()) and p.grad.shape == p.shape, name
    table = model["features"].table.grad
    seen = torch.zeros(200, dtype=torch.bool, device="cuda")
    seen[ids] = True
    seen[0] = False
    assert bool((table[~seen] == 0).all()) and float(table.abs().sum()) > 0
    # the whole gradient against a difference along itself
    params = [p for p in model.parameters() if p.requires_grad]
    grads = [p.grad.clone() for p in params]
    size = sum(float((g.double() ** 2).sum()) for g in grads)
    h = 1e-3 / size ** 0.5
    values = []
    for s in (1, -1):
        with torch.no_grad():
            for p, g in zip(params, grads):
                p.add_(g, alpha=s * h)
            values.append(float(loss_of().double()))
            for p, g in zip(params, grads):
                p.add_(g, alpha=-s * h)
    assert abs((values[0] - values[1]) / (2 * h) - size) < 0.05 * size
    optimiser.step()
    model["experts"].balance()
    assert torch.isfinite(loss_of())


def test_a_captured_backward_pass(experts):
    """A captured step of the operators, replayed with new rows."""
    import spmm_npu

    torch.manual_seed(4)
    x = torch.randn(40, 32, device="cuda", requires_grad=True)
    logits = torch.randn(40, 8, device="cuda", requires_grad=True)

    def step(xl, ll):
        w, e = spmm_npu.route_experts(ll, 2)
        ptr, position, source = spmm_npu.expert_plan(e, 8)
        y = spmm_npu.combine_rows(spmm_npu.dispatch_rows(xl, position, source), position, source, w)
        return torch.autograd.grad(y, [xl, ll], torch.ones_like(y))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(x, logits)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, logits)
    for seed in range(3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        with torch.no_grad():
            x.copy_(torch.randn(40, 32, generator=g, device="cuda"))
        graph.replay()
        want = step(x.detach().requires_grad_(True), logits.detach().requires_grad_(True))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
