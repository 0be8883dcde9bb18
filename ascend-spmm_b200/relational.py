"""Message passing over typed edges, and a training step for it.

A graph whose edges have one of R relations computes, for every node,

    y[v] = sum over relations r of (sum over edges u -> v of r of a_uv x[u]) W_r

The inner sums are one SpMM whose rows are the (relation, node) pairs that
have an edge, ordered by relation; the products with the R matrices are one
``grouped_matmul`` over those rows, with as many rows per relation as it has
receiving nodes; the outer sum is a second SpMM:

    g = RelationalGraph(relation, src, dst, values, num_nodes, num_relations)
    layer = RelationalLayer(g, 256, 128).cuda()     # layer_norm, messages, relu
    optimiser = OrthogonalMomentum(layer.parameters())
    loss = criterion(layer(x)); loss.backward(); optimiser.step()

Every part is differentiable: the backward pass of an SpMM is the SpMM with
the transposed matrix, laid out once with the graph.
"""

from __future__ import annotations

import torch

import spmm_npu


def _csr(row, col, val, rows):
    """CSR (int32) of coordinate triples, sorted by (row, col) as given."""
    ptr = torch.zeros(rows + 1, dtype=torch.int64, device=row.device)
    ptr[1:] = torch.cumsum(torch.bincount(row, minlength=rows), 0)
    return ptr.to(torch.int32), col.to(torch.int32).contiguous(), val.contiguous()


class _SparseMatrix:
    """A CSR matrix and its transpose."""

    def __init__(self, row, col, val, rows, cols):
        order = torch.argsort(row * cols + col)
        self.forward_csr = _csr(row[order], col[order], val[order], rows)
        order = torch.argsort(col * rows + row)
        self.transpose_csr = _csr(col[order], row[order], val[order], cols)
        self._start = torch.zeros(40, dtype=torch.int32, device=row.device)

    def __matmul__(self, x):
        return _Spmm.apply(x, self, False)

    def run(self, csr, x):
        ptr, col, val = csr
        return spmm_npu.spmm_csr(ptr, col, val.to(x.dtype), x.contiguous(), self._start)


class _Spmm(torch.autograd.Function):
    """A @ x, or with ``transposed`` A^T @ x: each is the other's gradient, to any order."""

    @staticmethod
    def forward(ctx, x, matrix, transposed):
        ctx.matrix, ctx.transposed = matrix, transposed
        return matrix.run(matrix.transpose_csr if transposed else matrix.forward_csr, x)

    @staticmethod
    def backward(ctx, grad):
        return _Spmm.apply(grad, ctx.matrix, not ctx.transposed), None, None


class RelationalGraph:
    """Edges ``src[i] -> dst[i]`` of relation ``relation[i]`` with weight
    ``values[i]`` (fp16 or fp32; distinct triples), on ``num_nodes`` nodes.  The
    weights are constants of the graph: they get no gradient."""

    def __init__(self, relation, src, dst, values, num_nodes: int, num_relations: int, device=None):
        if values.requires_grad:
            raise ValueError("values get no gradient: pass them detached")
        device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        relation, src, dst = (t.to(device=device, dtype=torch.int64) for t in (relation, src, dst))
        values = values.to(device)
        if not (relation.shape == src.shape == dst.shape == values.shape) or relation.dim() != 1:
            raise ValueError("relation, src, dst and values must be one-dimensional and of one length")
        for name, t, size in (("relation", relation, num_relations), ("src", src, num_nodes), ("dst", dst, num_nodes)):
            if t.numel() and (int(t.min()) < 0 or int(t.max()) >= size):
                raise ValueError(f"{name} must lie in [0, {size})")
        pairs, row = torch.unique(relation * num_nodes + dst, return_inverse=True)   # sorted by relation, node
        self.num_nodes, self.num_relations, self.num_pairs = num_nodes, num_relations, int(pairs.numel())
        self.gather = _SparseMatrix(row, src, values, self.num_pairs, num_nodes)
        self.scatter = _SparseMatrix(pairs % num_nodes, torch.arange(self.num_pairs, device=device),
                                     torch.ones(self.num_pairs, dtype=values.dtype, device=device), num_nodes,
                                     self.num_pairs)
        bounds = torch.arange(num_relations + 1, device=device) * num_nodes
        self.group_ptr = torch.searchsorted(pairs, bounds).to(torch.int32)

    def propagate(self, x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
        """``y[v] = sum_r (A_r x)[v] W_r`` for x [num_nodes, K], weight [num_relations, K, N]."""
        if x.size(0) != self.num_nodes:
            raise ValueError(f"expected features of {self.num_nodes} nodes, got {x.size(0)}")
        messages = self.gather @ x
        return self.scatter @ spmm_npu.grouped_matmul(messages, weight, self.group_ptr)


class RelationalLayer(torch.nn.Module):
    """relu(propagate(layer_norm(x)))."""

    def __init__(self, graph: RelationalGraph, in_features: int, out_features: int, dtype=torch.float32):
        super().__init__()
        self.graph = graph
        self.norm_weight = torch.nn.Parameter(torch.ones(in_features))
        self.norm_bias = torch.nn.Parameter(torch.zeros(in_features))
        w = torch.randn(graph.num_relations, in_features, out_features) / in_features ** 0.5
        self.weight = torch.nn.Parameter(w.to(dtype))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        h = spmm_npu.layer_norm(x, self.norm_weight, self.norm_bias)
        return torch.relu(self.graph.propagate(h, self.weight))


class OrthogonalMomentum(torch.optim.Optimizer):
    """Momentum whose matrices (parameters of two or more dimensions) are
    orthogonalised before they are applied; other parameters take the plain
    momentum step."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.9, vector_lr: float = 0.01):
        super().__init__(params, {"lr": lr, "momentum": momentum, "vector_lr": vector_lr})

    def load_state_dict(self, state_dict):
        """As the base class, which takes saved tensors to their parameter's type; the momentum stays fp32."""
        super().load_state_dict(state_dict)
        params = [p for group in self.param_groups for p in group["params"]]
        names = [name for group in state_dict["param_groups"] for name in group["params"]]
        for name, p in zip(names, params):
            saved = state_dict["state"].get(name, {}).get("momentum")
            if saved is not None:
                self.state[p]["momentum"] = saved.detach().to(device=p.device, dtype=torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if "momentum" not in state:
                    state["momentum"] = torch.zeros_like(p, dtype=torch.float32)
                m = state["momentum"].mul_(group["momentum"]).add_(p.grad)
                if p.dim() < 2:
                    p.add_(m, alpha=-group["vector_lr"])
                else:   # unit singular values: scaled so that a tall matrix's rows move as far as a square one's
                    scale = max(1.0, p.size(-2) / p.size(-1)) ** 0.5
                    p.add_(spmm_npu.orthogonalize(m), alpha=-group["lr"] * scale)
        return loss


__all__ = ["OrthogonalMomentum", "RelationalGraph", "RelationalLayer"]
