"""The typed-edge layer (ascend-spmm_b200/relational.py): layer_norm, SpMM,
grouped_matmul, SpMM forward and backward against dense 64-bit torch, and a
few training steps with orthogonalised updates."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def relational():
    import build

    build.build()
    import relational

    return relational


def edges(num_nodes, num_relations, count, seed):
    g = torch.Generator().manual_seed(seed)
    key = torch.randperm(num_relations * num_nodes * num_nodes, generator=g)[:count]
    relation = key // (num_nodes * num_nodes)
    keep = relation != 1   # one relation without edges
    relation = relation[keep]
    rest = key[keep] % (num_nodes * num_nodes)
    return relation, rest // num_nodes, rest % num_nodes, torch.rand(relation.numel(), generator=g) - 0.5


def dense(relation, src, dst, values, num_nodes, num_relations):
    a = torch.zeros(num_relations, num_nodes, num_nodes, dtype=torch.float64)
    a[relation, dst, src] = values.double()
    return a.cuda()


# fp32: sums of at most 60 terms of order one through two SpMMs, a product and
# their backward passes, each at 2^-20 of their magnitudes or better; fp16:
# each intermediate is rounded to 11 bits
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.float16, 2e-2)])
def test_layer_and_gradients(relational, dtype, tol):
    n, R, K, N = 60, 5, 48, 32
    e = edges(n, R, 900, seed=1)
    graph = relational.RelationalGraph(*e[:3], e[3].to(dtype), n, R)
    assert graph.num_pairs <= R * n and int(graph.group_ptr[-1]) == graph.num_pairs
    assert int(graph.group_ptr[1]) == int(graph.group_ptr[2])
    layer = relational.RelationalLayer(graph, K, N, dtype).cuda()
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(n, K, generator=g, device="cuda").to(dtype).requires_grad_(True)
    gy = torch.randn(n, N, generator=g, device="cuda").to(dtype)
    y = layer(x)
    got = torch.autograd.grad(y, [x, layer.weight, layer.norm_weight, layer.norm_bias], gy)

    a = dense(*e[:3], e[3].to(dtype), n, R)
    leaves = [t.detach().double().requires_grad_(True) for t in (x, layer.weight, layer.norm_weight, layer.norm_bias)]
    h = torch.nn.functional.layer_norm(leaves[0], (K,), leaves[2], leaves[3])
    ref = torch.relu(torch.einsum("rvu,uk,rkn->vn", a, h, leaves[1]))
    # the relu's slope is taken where the kernel's own output is positive
    ref_grads = torch.autograd.grad(torch.einsum("rvu,uk,rkn->vn", a, h, leaves[1]), leaves,
                                    gy.double() * (y.detach() > 0))
    assert float((y.detach().double() - ref.detach()).abs().max()) <= tol * float(ref.detach().abs().max())
    for k, r in zip(got, ref_grads):
        assert float((k.double() - r).norm()) <= tol * float(r.norm())
    assert not bool(got[1][1].any())   # the relation without edges


def test_training_step_reduces_the_loss(relational):
    n, R, K, N = 200, 4, 64, 64
    e = edges(n, R, 3000, seed=3)
    graph = relational.RelationalGraph(*e, n, R)
    torch.manual_seed(0)
    layer = relational.RelationalLayer(graph, K, N).cuda()
    optimiser = relational.OrthogonalMomentum(layer.parameters(), lr=0.02)
    x = torch.randn(n, K, device="cuda")
    target = torch.relu(torch.randn(n, N, device="cuda"))
    losses = []
    for _ in range(30):
        optimiser.zero_grad()
        loss = (layer(x) - target).square().mean()
        loss.backward()
        optimiser.step()
        losses.append(float(loss.detach()))
    assert losses[-1] < 0.7 * losses[0] and all(l == l for l in losses)


def test_refusals(relational):
    e = edges(20, 3, 50, seed=4)
    with pytest.raises(ValueError, match="must lie in"):
        relational.RelationalGraph(*e, 20, 2)
    with pytest.raises(ValueError, match="one length"):
        relational.RelationalGraph(e[0][:3], *e[1:], 20, 3)
    graph = relational.RelationalGraph(*e, 20, 3)
    with pytest.raises(ValueError, match="20 nodes"):
        graph.propagate(torch.zeros(21, 16, device="cuda"), torch.zeros(3, 16, 16, device="cuda"))
