"""Public Python API of the B200 SpMM engine (drop-in for the reference's
``spmm_npu`` module, IDMG-Lab/Ascend-SpMM spmm_npu.py:1-78).

Every operator and layout function runs as hand-written CUDA through
``custom_ops_lib`` (the torch-facing module over ``libspmm_b200.so``).  There
is no CPU fallback: importing this module fails if the extension is missing,
and the operators require CUDA tensors, as the reference requires NPU tensors.

For fixed square graphs, ``preprocess(..., graph_layout=True)`` returns
``P A P^T`` mappings; pack node tensors once with ``P`` and restore original
ids only when needed.
"""

import torch

from custom_ops_lib import (  # noqa: F401  (re-exported API)
    device_status,
    spmm_ascend_cube,
    spmm_ascend_cube_aic_without_pipeline,
    spmm_ascend_cube_aiv_mb,
    spmm_ascend_cube_tiles,
    spmm_csr,
    spmm_csr_aiv_mb_batch,
    spmm_cube,
)

from custom_ops_lib import (  # noqa: F401  (GPU layout builders)
    block_level_split,
    csr_to_ascend_cube,
    csr_to_bcsr,
    csr_to_spmm_cube,
    preprocess,
)
from custom_ops_lib import pack_rows as _pack_rows, restore_rows as _restore_rows
from custom_ops_lib import (  # noqa: F401  (layer operators)
    grouped_matmul as _grouped_matmul,
    grouped_weight_grad,
    layer_norm as _layer_norm,
    layer_norm_backward,
    layer_norm_forward,
    orthogonalize as _orthogonalize,
)


def _index(inv_permutation, device):
    return inv_permutation.to(device=device, dtype=torch.long).reshape(-1).contiguous()


# Row scatter / gather on the GPU, differentiable like the reference's
# index_copy_ / index_select (the gradient of one is the other).
class _PackRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tensor, index, packed_rows):
        ctx.save_for_backward(index)
        return _pack_rows(tensor.contiguous(), index, packed_rows)

    @staticmethod
    def backward(ctx, grad):
        (index,) = ctx.saved_tensors
        return _restore_rows(grad.contiguous(), index), None, None


class _RestoreRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, packed, index):
        ctx.save_for_backward(index)
        ctx.rows = packed.size(0)
        return _restore_rows(packed.contiguous(), index)

    @staticmethod
    def backward(ctx, grad):
        (index,) = ctx.saved_tensors
        return _pack_rows(grad.contiguous(), index, ctx.rows), None


def pack_node_tensor(tensor, inv_permutation, packed_rows=None):
    """Apply ``P`` once to a tensor whose leading dimension is original node id.

    Same contract as the reference (spmm_npu.py:22-47): padding rows are
    zero, and errors are raised as ValueError with the reference's messages.
    This helper belongs in graph preprocessing, not in the per-layer loop.
    """
    if tensor.ndim < 1:
        raise ValueError("a node tensor must have at least one dimension")
    index = _index(inv_permutation, tensor.device)
    if tensor.size(0) != index.numel():
        raise ValueError("inv_permutation must contain one entry per original node")
    if index.numel() and bool((index < 0).any().item()):
        raise ValueError("inv_permutation does not map every original node")
    minimum_rows = int(index.max().item()) + 1 if index.numel() else 0
    if packed_rows is None:
        packed_rows = minimum_rows
    elif torch.is_tensor(packed_rows):
        packed_rows = int(packed_rows.item())
    else:
        packed_rows = int(packed_rows)
    if packed_rows < minimum_rows:
        raise ValueError("packed_rows is smaller than the permutation extent")
    return _PackRows.apply(tensor, index, packed_rows)


def restore_node_tensor(packed_tensor, inv_permutation):
    """Apply ``P^T`` once and return rows in original node-id order
    (reference spmm_npu.py:50-61)."""
    if packed_tensor.ndim < 1:
        raise ValueError("a packed node tensor must have at least one dimension")
    index = _index(inv_permutation, packed_tensor.device)
    if index.numel() and (
        bool((index < 0).any().item())
        or int(index.max().item()) >= packed_tensor.size(0)
    ):
        raise ValueError("inv_permutation contains an invalid packed node id")
    return _RestoreRows.apply(packed_tensor, index)


# --------------------------------------------------------------------------
# Layer operators around the SpMM (no counterpart in the reference)
# --------------------------------------------------------------------------
def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension
    of a CUDA tensor x (fp16, bf16 or fp32, any width), differentiable in x,
    weight and bias.

    ``weight`` and ``bias`` ([width], or None for ones and zeros) share one
    dtype, x's or fp32; their gradients have that dtype.  Sums are fp32 and
    run in a fixed order.  ``layer_norm_forward`` / ``layer_norm_backward`` are
    the two passes by themselves.
    """
    return _layer_norm(x, weight, bias, eps)


def grouped_matmul(x, weight, group_ptr, transposed=False):
    """Row ranges of x times one matrix each: ``y[r] = x[r] @ weight[g]`` for
    ``group_ptr[g] <= r < group_ptr[g + 1]``; rows outside every group are zero.

    ``x`` [rows, K], ``weight`` [groups, K, N] (fp16, bf16 or fp32; widths
    divisible by 16, fp32 by 8), ``group_ptr`` [groups + 1] int32 or int64 on
    the device, like a CSR row pointer (the relations of a typed graph's
    messages, the experts of routed rows).  ``transposed`` takes x [rows, N] to
    [rows, K] by ``weight[g].T``.  Both are differentiable in x and weight;
    ``grouped_weight_grad`` is the weight's gradient by itself, without a
    gradient of its own.  A malformed range raises the device status instead of
    a fault.
    """
    return _grouped_matmul(x, weight, group_ptr, transposed)


def orthogonalize(update, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7):
    """An update's matrices [..., m, n] with their singular values driven
    towards one: divided by the Frobenius norm + eps, then ``steps`` times
    ``G = X X^T; X = a X + (b G + c G G) X`` (the step of an optimiser that
    orthogonalises its momentum before it is applied to a weight matrix).

    ``update`` is fp16, bf16 or fp32; the result is bf16.  The products run on
    16-bit operands, so fp32 would hold no more of it: with five steps it is off
    by 1.7e-3 to 2.5e-3 of its norm (the rounding alone is 1.7e-3), with ten by
    up to 5e-3, and more with many.  It has no derivative: a backward pass
    through it raises an error.
    """
    a, b, c = coefficients
    return _orthogonalize(update, steps, a, b, c, eps)


__all__ = [
    "block_level_split",
    "csr_to_ascend_cube",
    "csr_to_bcsr",
    "csr_to_spmm_cube",
    "grouped_matmul",
    "grouped_weight_grad",
    "layer_norm",
    "layer_norm_backward",
    "layer_norm_forward",
    "orthogonalize",
    "pack_node_tensor",
    "preprocess",
    "restore_node_tensor",
    "spmm_ascend_cube",
    "spmm_ascend_cube_aic_without_pipeline",
    "spmm_ascend_cube_aiv_mb",
    "spmm_ascend_cube_tiles",
    "spmm_csr",
    "spmm_csr_aiv_mb_batch",
    "spmm_cube",
]
