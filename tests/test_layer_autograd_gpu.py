"""What the layer operators do with gradients beyond the plain backward pass:
the transposed product's, an orthogonalised update's."""

import pytest
import torch

from layer_reference import assert_within, grouped_reference, weight_grad_reference
from test_grouped_gpu import lib, make  # noqa: F401

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
