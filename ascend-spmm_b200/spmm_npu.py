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
    combine_rows as _combine_rows,
    dispatch_rows,
    embedding as _embedding,
    embedding_grad,
    expert_plan as _expert_plan,
    grouped_matmul as _grouped_matmul,
    grouped_matmul_fp8 as _grouped_matmul_fp8,
    grouped_weight_grad,
    layer_norm as _layer_norm,
    layer_norm_backward,
    layer_norm_forward,
    orthogonalize as _orthogonalize,
    quantize_fp8 as _quantize_fp8,
    quantize_weight_fp8 as _quantize_weight_fp8,
    route_experts as _route_experts,
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


# --------------------------------------------------------------------------
# Routed experts and learned features (no counterpart in the reference)
# --------------------------------------------------------------------------
def route_experts(logits, top_k, bias=None, scoring="softmax", groups=1, top_groups=1, group_best=1,
                  renormalize=True, scale=1.0):
    """The ``top_k`` experts of each row of logits [..., num_experts] (fp16,
    bf16 or fp32) and their weights: ``(weights, experts)``, fp32 and int32
    [..., top_k], in descending order.

    The scores are the row's softmax or sigmoid (``scoring``).  ``bias`` (fp32
    [num_experts], for balance) is added to them for the choice alone.  With
    ``groups`` > ``top_groups`` the experts are that many ranges of equal size,
    and only those of the ``top_groups`` ranges with the largest sums of their
    ``group_best`` (1 or 2) largest values can be chosen.  Values are compared
    as 64-bit scores, or, where nothing is added to a score (no ``bias``, and no
    sums of two by ``groups``), as the logits, in whose order the scores are:
    scores that round to the same number, as of sigmoid 1 above 37, tie with a
    bias of zeros and not with None.  Equal values go to the lowest index, NaN
    below all.  ``renormalize`` divides the chosen scores by their sum + 1e-20;
    ``scale`` multiplies them; sigmoids below 2^-126 count as 0 in the weights.
    At most 1024 experts, 32 chosen ones, 32 groups.

    The weights are differentiable in the logits; the choice is a constant.
    """
    return _route_experts(logits, top_k, bias, scoring, groups, top_groups, group_best, renormalize, scale)


def expert_plan(experts, num_experts):
    """The order that brings the rows of each expert together, as int32 tensors
    on the device: ``(group_ptr, position, source)``.

    ``experts`` (int32 or int64, [rows, choices]; -1: none) is sorted stably.
    ``group_ptr`` [num_experts + 1] is ``grouped_matmul``'s, ``position`` (like
    ``experts``) the row of each choice or -1, ``source`` [rows * choices] the
    choice of each row, -1 behind the last.  ``group_ptr`` differences are the
    experts' loads.  An expert outside [-1, num_experts) counts as -1 and raises
    the device status.  At most 1024 experts.
    """
    return _expert_plan(experts, num_experts)


def combine_rows(rows, position, source, weights=None):
    """``y[t] = sum_j weights[t, j] * rows[position[t, j]]``: the results of each
    row's experts added up, in fp32.  ``weights`` is fp32 [rows, choices]
    (``route_experts``'s) or None for ones; choices without a position add
    nothing.  Differentiable in rows and weights.

    ``dispatch_rows(x, position, source)`` is the way there: the rows of x in
    the plan's order, one per choice, zeros behind the last (differentiable).
    """
    return _combine_rows(rows, position, source, weights)


def embedding(ids, table, scale=1.0, padding_id=None):
    """``scale * table[ids]`` for ids (int32 or int64, any shape) and a table
    [rows, width] in fp16, bf16 or fp32, differentiable in table.

    The gradient adds the rows of each id up in fp32 in the order of the ids
    (no atomics: the same bits every time); the id ``padding_id`` gets none.
    An id outside the table gives zeros and raises the device status.
    ``embedding_grad(ids, grad, num_rows, scale, padding_id)`` is the gradient by
    itself.
    """
    return _embedding(ids, table, scale, padding_id)


def quantize_fp8(x):
    """x [..., width] in 8-bit floating point: ``(q, scale)``, q e4m3 like x and
    fp32 scales [..., ceil(width / 128)], one per block of 128 elements.

    A block's scale is its largest finite magnitude (at least 2^-100) / 448, q
    the values x / scale rounded to nearest; infinities and NaN become NaN.
    Widths are divisible by 16.  Not differentiable.
    """
    return _quantize_fp8(x)


def quantize_weight_fp8(weight):
    """Weights [groups, K, N] for ``grouped_matmul_fp8``, laid out once: ``(q,
    scale)``, q e4m3 [groups, N, K] (transposed) and fp32 scales [groups,
    ceil(N / 128), ceil(K / 128)] of blocks of 128 x 128, as ``quantize_fp8``."""
    return _quantize_weight_fp8(weight)


def grouped_matmul_fp8(x, x_scale, weight, weight_scale, group_ptr, out_dtype=torch.bfloat16):
    """``grouped_matmul`` of operands in 8 bits (``quantize_fp8``'s rows,
    ``quantize_weight_fp8``'s weights): each block of 128 products is summed on
    the tensor cores, the blocks in fp32 times their scales, and the result
    rounded to ``out_dtype`` (fp16, bf16 or fp32) once.  K and N are divisible
    by 16.  For serving: not differentiable.
    """
    return _grouped_matmul_fp8(x, x_scale, weight, weight_scale, group_ptr, out_dtype)


__all__ = [
    "block_level_split",
    "combine_rows",
    "csr_to_ascend_cube",
    "csr_to_bcsr",
    "csr_to_spmm_cube",
    "dispatch_rows",
    "embedding",
    "embedding_grad",
    "expert_plan",
    "grouped_matmul",
    "grouped_matmul_fp8",
    "grouped_weight_grad",
    "layer_norm",
    "layer_norm_backward",
    "layer_norm_forward",
    "orthogonalize",
    "pack_node_tensor",
    "preprocess",
    "quantize_fp8",
    "quantize_weight_fp8",
    "restore_node_tensor",
    "route_experts",
    "spmm_ascend_cube",
    "spmm_ascend_cube_aic_without_pipeline",
    "spmm_ascend_cube_aiv_mb",
    "spmm_ascend_cube_tiles",
    "spmm_csr",
    "spmm_csr_aiv_mb_batch",
    "spmm_cube",
]
