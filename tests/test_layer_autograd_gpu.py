"""What the layer operators do with gradients beyond the plain backward pass:
the transposed product's, an orthogonalised update's, forward-mode tangents,
second derivatives of the sparse products, edge weights."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from layer_reference import assert_within, grouped_reference, weight_grad_reference
from test_grouped_gpu import lib, make  # noqa: F401
from test_relational_gpu import edges, relational  # noqa: F401

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [F16, F32])
def test_gradient_of_the_transposed_product(lib, dtype):  # noqa: F811
    """y = g W^T: dg = dy W and dW = dy^T g per group."""
    x, w, ptr, grad = make([37, 0, 150], 64, 80, dtype, seed=3, before=5, after=9)
    gl, wl = grad.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = lib.grouped_matmul(gl, wl, ptr, transposed=True)
    assert torch.equal(y.detach(), lib.grouped_matmul(grad, w, ptr, transposed=True))
    dg, dw = torch.autograd.grad(y, [gl, wl], x)
    assert_within(dg, *grouped_reference(x, w, ptr))
    assert_within(dw, *weight_grad_reference(x, grad, ptr))


def test_an_orthogonalised_update_refuses_its_backward_pass(lib):  # noqa: F811
    u = torch.randn(40, 30, device="cuda", requires_grad=True)
    y = lib.orthogonalize(u)
    assert y.requires_grad and torch.equal(y.detach(), lib.orthogonalize(u.detach()))
    for call in (lambda: y.float().sum().backward(), lambda: torch.autograd.grad(y.sum(), [u], allow_unused=True)):
        with pytest.raises(RuntimeError, match="orthogonalize is not differentiable"):
            call()
    with torch.no_grad():
        assert not lib.orthogonalize(u).requires_grad


def test_forward_mode_tangents_are_refused(lib):  # noqa: F811
    x, w, ptr, grad = make([8, 8], 32, 32, F32)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        dw = forward_ad.make_dual(w, torch.ones_like(w))
        for call in (lambda: lib.layer_norm(d), lambda: lib.layer_norm(x, d[0]), lambda: lib.grouped_matmul(d, w, ptr),
                     lambda: lib.grouped_matmul(x, dw, ptr), lambda: lib.grouped_matmul(d, w, ptr, True),
                     lambda: lib.grouped_weight_grad(x, d, ptr), lambda: lib.orthogonalize(d),
                     lambda: lib.layer_norm_forward(d, None, None)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            lib.layer_norm(d)
    lib.layer_norm(x)


def test_sparse_products_are_differentiable_twice(relational):  # noqa: F811
    """f(x) = |A x|^2: the gradient 2 A^T A x has its own, 2 A^T A v."""
    n, R = 30, 3
    graph = relational.RelationalGraph(*edges(n, R, 200, seed=5), n, R)
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(n, 16, generator=g, device="cuda", requires_grad=True)
    v = torch.randn(n, 16, generator=g, device="cuda")
    y = graph.gather @ x
    (first,) = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    (second,) = torch.autograd.grad(first, x, v)
    (want,) = torch.autograd.grad(graph.gather @ x, x, 2 * (graph.gather @ v))
    assert float((second - want).norm()) <= 1e-5 * float(want.norm()) and float(want.norm()) > 0


def test_edge_weights_that_want_a_gradient_are_refused(relational):  # noqa: F811
    e = edges(20, 3, 50, seed=4)
    with pytest.raises(ValueError, match="no gradient"):
        relational.RelationalGraph(*e[:3], e[3].requires_grad_(True), 20, 3)
    relational.RelationalGraph(*e[:3], e[3].detach(), 20, 3)
