"""Layers of routed experts, and a table of learned node features.

``ExpertLayer`` sends each row of x to ``top_k`` of its experts, two-layer
networks of their own, and adds their results up:

    y[t] = sum over the chosen experts e of w[t, e] relu(x[t] A_e) B_e

The rows are put in the order of their experts, so that the products of all
experts are two ``grouped_matmul`` calls:

    layer = ExpertLayer(256, 512, num_experts=32, top_k=4).cuda()
    loss = criterion(layer(x)); loss.backward(); optimiser.step()
    layer.balance()                     # moves the bias of the choice against the last loads
    served = layer.quantized()          # the same layer with its products in 8 bits

``NodeFeatures`` holds a learned row per node (or per node type) and looks it up:

    features = NodeFeatures(num_nodes, 256).cuda()
    h = relational_layer(features(node_ids))
"""

from __future__ import annotations

import torch

import spmm_npu


class _KeepsTypes(torch.nn.Module):
    """A module whose buffers named in ``kept`` go where it goes, and keep their types when it is cast."""

    kept = ()

    def _apply(self, fn, recurse=True):
        kept = {name: self._buffers[name] for name in self.kept}
        self._buffers.update(dict.fromkeys(kept))
        try:
            super()._apply(fn, recurse)
        finally:
            self._buffers.update(kept)
        for name, buffer in kept.items():
            as_cast = fn(buffer.new_empty(0))
            self._buffers[name] = fn(buffer) if as_cast.dtype == buffer.dtype else buffer.to(as_cast.device)
        return self


class _Router(_KeepsTypes):
    """Scores of the experts, their choice, and the way of the rows to the experts and back.  The bias stays fp32 in a module
    that is cast to 16 bits, where the steps of ``balance`` would be rounded away."""

    kept = ("bias",)

    def __init__(self, gate, bias, options):
        super().__init__()
        if isinstance(gate, torch.nn.Parameter):
            self.gate = gate
        else:   # of a layer that does not train
            self.register_buffer("gate", gate)
        self.register_buffer("bias", bias)
        self.options = dict(options)
        self.group_ptr = None   # of the last call: group_ptr[e + 1] - group_ptr[e] rows went to expert e

    def forward(self, x, products):
        """x [rows, in] -> [rows, out]; ``products(rows, group_ptr)`` are the experts'."""
        with torch.autocast(x.device.type, enabled=False):   # scores are fp32, also in a module that was cast to 16 bits
            logits = x.float() @ self.gate.float()
        weights, experts = spmm_npu.route_experts(logits, bias=self.bias.float(), **self.options)
        group_ptr, position, source = spmm_npu.expert_plan(experts, self.gate.size(1))
        self.group_ptr = group_ptr
        rows = spmm_npu.dispatch_rows(x, position, source)
        return spmm_npu.combine_rows(products(rows, group_ptr), position, source, weights)


class ExpertLayer(torch.nn.Module):
    """``top_k`` of ``num_experts`` two-layer networks per row.  ``routing``: further arguments of
    ``route_experts`` (scoring, groups, top_groups, group_best, renormalize, scale)."""

    def __init__(self, in_features: int, hidden: int, num_experts: int, top_k: int, out_features: int | None = None,
                 dtype=torch.float32, **routing):
        super().__init__()
        out_features = in_features if out_features is None else out_features
        gate = torch.nn.Parameter(torch.randn(in_features, num_experts) / in_features ** 0.5)
        self.router = _Router(gate, torch.zeros(num_experts), {"top_k": top_k, **routing})
        up = torch.randn(num_experts, in_features, hidden) / in_features ** 0.5
        down = torch.randn(num_experts, hidden, out_features) / hidden ** 0.5
        self.up, self.down = torch.nn.Parameter(up.to(dtype)), torch.nn.Parameter(down.to(dtype))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        def products(rows, group_ptr):
            return spmm_npu.grouped_matmul(torch.relu(spmm_npu.grouped_matmul(rows, self.up, group_ptr)), self.down, group_ptr)

        return self.router(x, products)

    @torch.no_grad()
    def balance(self, rate: float = 1e-3):
        """Moves the bias of each expert by ``rate`` towards the average load of the last call."""
        if self.router.group_ptr is None:
            raise RuntimeError("balance needs a call of the layer before it")
        load = self.router.group_ptr.diff().float()
        self.router.bias.add_(torch.sign(load.mean() - load), alpha=rate)

    def quantized(self) -> "QuantizedExpertLayer":
        """A layer for serving, with the experts' weights in 8 bits."""
        return QuantizedExpertLayer(self)


class QuantizedExpertLayer(_KeepsTypes):
    """An ``ExpertLayer`` whose products run in 8-bit floating point (not differentiable).  Cast to another type, it keeps
    its 8-bit weights and their fp32 scales."""

    kept = ("up", "up_scale", "down", "down_scale")

    @torch.no_grad()
    def __init__(self, layer: ExpertLayer):
        super().__init__()
        self.router = _Router(layer.router.gate.detach().clone(), layer.router.bias.clone(), layer.router.options)
        for name in ("up", "down"):
            q, scale = spmm_npu.quantize_weight_fp8(getattr(layer, name).detach())
            self.register_buffer(name, q)
            self.register_buffer(name + "_scale", scale)

    @torch.no_grad()
    def forward(self, x: torch.Tensor) -> torch.Tensor:
        def products(rows, group_ptr):
            q, scale = spmm_npu.quantize_fp8(rows)
            hidden = torch.relu(spmm_npu.grouped_matmul_fp8(q, scale, self.up, self.up_scale, group_ptr, rows.dtype))
            q, scale = spmm_npu.quantize_fp8(hidden)
            return spmm_npu.grouped_matmul_fp8(q, scale, self.down, self.down_scale, group_ptr, rows.dtype)

        return self.router(x, products)


class NodeFeatures(torch.nn.Module):
    """A learned row of ``width`` features per id, times ``scale``."""

    def __init__(self, num_rows: int, width: int, scale: float = 1.0, padding_id: int | None = None, dtype=torch.float32):
        super().__init__()
        self.table = torch.nn.Parameter(torch.randn(num_rows, width).to(dtype))
        self.scale, self.padding_id = scale, padding_id

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        return spmm_npu.embedding(ids, self.table, self.scale, self.padding_id)


__all__ = ["ExpertLayer", "NodeFeatures", "QuantizedExpertLayer"]
