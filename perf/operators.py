"""Measured cases of the layer operators that stand around an SpMM in a training step.

A graph layer reads ``A @ X`` and then normalises the node rows
(``layer_norm``), multiplies each relation's (or expert's) rows with that
relation's matrix (``grouped_matmul``: the rows of group g are
``group_ptr[g] .. group_ptr[g + 1]``, as in a CSR row pointer), and its weight
matrices are updated with an orthogonalised step (``orthogonalize``: five
Newton-Schulz products on a matrix of unit Frobenius norm).

``listed()`` and ``draw()`` give cases, ``prepare()`` the inputs, ``run()`` one
pass (the formulas in elementary torch operations, or this repository's
operators where ``own`` is set), ``work()`` the bytes and operations a pass
cannot do without and ``exact()`` the definition in 64 bits.
"""

import math
import sys
from pathlib import Path

import torch

own = False

EPS_NORM = 1e-5
EPS_ORTHO = 1e-7
STEPS = 5
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one decoding step of a served model: nine rows of 256 features, the cost is the call itself
        {"name": "norm_few_rows", "op": "layer_norm", "rows": 9, "width": 256, "dtype": "fp16", "params": "fp16",
         "train": False},
        # fp32 node features of a mid-sized graph, forward and backward
        {"name": "norm_graph_fp32_train", "op": "layer_norm", "rows": 100003, "width": 256, "dtype": "fp32",
         "params": "fp32", "train": True},
        # rows that are not 16-byte aligned, parameters kept in fp32
        {"name": "norm_odd_width", "op": "layer_norm", "rows": 16411, "width": 1001, "dtype": "bf16",
         "params": "fp32", "train": False},
        # the widest features of this repository's benchmark, forward and backward
        {"name": "norm_wide_train", "op": "layer_norm", "rows": 524287, "width": 1024, "dtype": "fp16",
         "params": "fp16", "train": True},
        # nine routed rows over 32 experts: bound by reading the experts that have a row
        {"name": "grouped_few_rows", "op": "grouped_matmul", "rows": 9, "groups": 32, "k": 1024, "n": 512,
         "dtype": "bf16", "skew": False, "train": False},
        # edge messages of a graph with 46 relations of very unequal sizes, forward and backward
        {"name": "grouped_relations_train", "op": "grouped_matmul", "rows": 100003, "groups": 46, "k": 256, "n": 128,
         "dtype": "fp16", "skew": True, "train": True},
        # the same in fp32, where the products keep fp32's accuracy
        {"name": "grouped_fp32_train", "op": "grouped_matmul", "rows": 20011, "groups": 8, "k": 256, "n": 264,
         "dtype": "fp32", "skew": True, "train": True},
        # a large expert layer, forward and backward: bound by the products
        {"name": "grouped_experts_train", "op": "grouped_matmul", "rows": 65537, "groups": 64, "k": 1024, "n": 2048,
         "dtype": "bf16", "skew": True, "train": True},
        # one small weight matrix: fifteen dependent products, the cost is their latency
        {"name": "ortho_small", "op": "orthogonalize", "batch": 1, "m": 128, "n": 64, "dtype": "fp32"},
        # the matrices of 46 relations at once
        {"name": "ortho_relations", "op": "orthogonalize", "batch": 46, "m": 256, "n": 128, "dtype": "fp16"},
        # odd sizes, wider than tall
        {"name": "ortho_odd", "op": "orthogonalize", "batch": 3, "m": 601, "n": 1023, "dtype": "bf16"},
        # one large matrix: bound by the products
        {"name": "ortho_large", "op": "orthogonalize", "batch": 1, "m": 4096, "n": 2048, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same operators: the smallest call to one that costs no more than the largest listed one."""
    op = rng.choice(("layer_norm", "grouped_matmul", "orthogonalize"))
    dtype = rng.choice(("fp16", "bf16", "fp32"))
    if op == "layer_norm":
        while True:
            rows, width = _log_int(rng, 1, 524287), _log_int(rng, 8, 8191)
            if rows * width <= 524287 * 1024 // (2 if dtype == "fp32" else 1) and width != 3072:
                break
        return {"op": op, "rows": rows, "width": width, "dtype": dtype, "params": rng.choice((dtype, "fp32")),
                "train": rng.random() < 0.5}
    if op == "grouped_matmul":
        heavy = 4 if dtype == "fp32" else 1
        while True:
            rows, groups = _log_int(rng, 1, 65537), _log_int(rng, 1, 128)
            k, n = 16 * _log_int(rng, 1, 128), 16 * _log_int(rng, 1, 128)
            if heavy * rows * k * n <= 65537 * 1024 * 2048 and groups * k * n <= 64 * 1024 * 2048 and 3072 not in (k, n):
                break
        return {"op": op, "rows": rows, "groups": groups, "k": k, "n": n, "dtype": dtype, "skew": rng.random() < 0.5,
                "train": rng.random() < 0.5}
    while True:
        batch, m, n = _log_int(rng, 1, 64), _log_int(rng, 1, 4096), _log_int(rng, 1, 4096)
        if batch * _ortho_products(m, n) <= _ortho_products(4096, 2048) and 3072 not in (m, n):
            break
    return {"op": op, "batch": batch, "m": m, "n": n, "dtype": dtype}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    state = dict(case)
    if case["op"] == "layer_norm":
        # node rows differ in level and spread, as aggregated features do
        level, spread = normal(case["rows"], 1), torch.exp(0.5 * normal(case["rows"], 1))
        x = (normal(case["rows"], case["width"]) * spread).add_(level).to(dtype)
        params = DTYPES[case["params"]]
        state.update(x=x, weight=(1 + 0.2 * normal(case["width"])).to(params),
                     bias=(0.2 * normal(case["width"])).to(params))
        if case["train"]:
            state["grad"] = normal(case["rows"], case["width"]).to(dtype)
            for name in ("x", "weight", "bias"):
                state[name].requires_grad_(own)
    elif case["op"] == "grouped_matmul":
        M, G, K, N = case["rows"], case["groups"], case["k"], case["n"]
        share = torch.rand(G, generator=g, device="cuda") ** (4.0 if case["skew"] else 0.5) + 1e-4
        owner = torch.multinomial(share, M, replacement=True, generator=g)
        ptr = torch.zeros(G + 1, dtype=torch.int64, device="cuda")
        ptr[1:] = torch.cumsum(torch.bincount(owner, minlength=G), 0)
        state.update(x=normal(M, K).to(dtype), weight=(normal(G, K, N) / math.sqrt(K)).to(dtype),
                     ptr=ptr.to(torch.int32))
        if case["train"]:
            state["grad"] = normal(M, N).to(dtype)
            for name in ("x", "weight"):
                state[name].requires_grad_(own)
        # the plain form's row tiles: about two for each group of even size
        state["tile"] = max(16, 1 << max(0, (M // max(1, G)).bit_length() - 1))
    else:
        # a weight gradient X^T dY over features of unequal strength
        m, n = case["m"], case["n"]
        rows = 2 * min(m, n) + 16
        left = normal(case["batch"], rows, m) * torch.logspace(0, -1, m, device="cuda")
        right = normal(case["batch"], rows, n) * torch.logspace(0, -1, n, device="cuda")
        state["update"] = (torch.bmm(left.transpose(1, 2), right) / rows).to(dtype)
    return state


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

def _operators():
    at = str(Path(__file__).resolve().parents[1] / "ascend-spmm_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import spmm_npu

    return spmm_npu


def run(state):
    if own:
        return _run_own(state)
    return {"layer_norm": _plain_norm, "grouped_matmul": _plain_grouped, "orthogonalize": _plain_ortho}[state["op"]](state)


def _run_own(state):
    lib = _operators()
    if state["op"] == "orthogonalize":
        return [lib.orthogonalize(state["update"])]
    if state["op"] == "layer_norm":
        inputs = [state["x"], state["weight"], state["bias"]]
        y = lib.layer_norm(*inputs, EPS_NORM)
    else:
        inputs = [state["x"], state["weight"]]
        y = lib.grouped_matmul(*inputs, state["ptr"])
    if not state["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, inputs, state["grad"])]


def _plain_norm(s):
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    centred = x - x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + EPS_NORM)
    xhat = centred * rstd
    y = (xhat * w + b).to(s["x"].dtype)
    if not s["train"]:
        return [y]
    grad = s["grad"].float()
    gw = grad * w
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - xhat * (gw * xhat).mean(-1, keepdim=True))
    return [y, dx.to(s["x"].dtype), (grad * xhat).sum(0).to(s["weight"].dtype), grad.sum(0).to(s["bias"].dtype)]


def _plain_grouped(s):
    """Rows in tiles that belong to one group each (a tile's missing rows are zero), one batched product over the tiles."""
    dtype, (M, K), (G, _, N) = s["x"].dtype, s["x"].shape, s["weight"].shape
    ptr, tile, dev = s["ptr"].long(), s["tile"], s["x"].device
    first = torch.zeros(G + 1, dtype=torch.int64, device=dev)
    first[1:] = torch.cumsum((ptr[1:] - ptr[:-1] + tile - 1) // tile, 0)
    t = torch.arange(-(-M // tile) + G, device=dev)
    group = torch.searchsorted(first[1:], t, right=True).clamp(max=G - 1)
    row = (ptr[group] + (t - first[group]) * tile)[:, None] + torch.arange(tile, device=dev)
    valid = (row < ptr[group + 1][:, None]) & (t < first[G])[:, None]
    take, put = torch.where(valid, row, 0), torch.where(valid, row, M)
    weight = s["weight"].float()[group]

    def tiles(a):
        return torch.where(valid[:, :, None], a[take], 0).float()

    def rows(a):
        out = torch.zeros(M + 1, a.shape[-1], device=dev)
        out[put] = a
        return out[:M].to(dtype)

    x = tiles(s["x"])
    y = rows(torch.bmm(x, weight))
    if not s["train"]:
        return [y]
    grad = tiles(s["grad"])
    dx = rows(torch.bmm(grad, weight.transpose(1, 2)))
    dw = torch.zeros(G, K, N, device=dev).index_add_(0, group, torch.bmm(x.transpose(1, 2), grad))
    return [y, dx, dw.to(dtype)]


def _plain_ortho(s):
    a, b, c = COEFFICIENTS
    x = s["update"].float()
    tall = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2) if tall else x
    x = x / (torch.sqrt((x * x).sum((1, 2), keepdim=True)) + EPS_ORTHO)
    for _ in range(STEPS):
        gram = torch.bmm(x, x.transpose(1, 2))
        x = a * x + torch.bmm(b * gram + c * torch.bmm(gram, gram), x)
    return [(x.transpose(1, 2) if tall else x).contiguous().to(torch.bfloat16)]


# --------------------------------------------------------------------------
# floors and the definition in 64 bits
# --------------------------------------------------------------------------

def _ortho_products(m, n):
    """Operations of one matrix: each of the five steps has two symmetric products (half of their tiles) and a full one."""
    s, r = min(m, n), max(m, n)
    return STEPS * (s * s * r + s * s * s + 2 * s * s * r)


def _bytes(name):
    return 4 if name == "fp32" else 2


def work(case):
    size = _bytes(case["dtype"])
    if case["op"] == "layer_norm":
        tensor, params = case["rows"] * case["width"], 2 * case["width"] * _bytes(case["params"])
        if case["train"]:   # x and the gradient read; y, dx and the parameters' gradients written
            return {"bytes": 4 * tensor * size + 2 * params, "flops": 20 * tensor}
        return {"bytes": 2 * tensor * size + params, "flops": 8 * tensor}
    if case["op"] == "grouped_matmul":
        M, G, K, N = case["rows"], case["groups"], case["k"], case["n"]
        x, y = M * K * size, M * N * size
        w = G * (1 - (1 - 1 / G) ** M) * K * N * size   # the groups that M rows meet
        if case["train"]:   # x, weight and the gradient read; y, dx and every group's gradient written
            return {"bytes": 2 * x + 2 * y + w + G * K * N * size, "flops": 6 * M * K * N}
        return {"bytes": x + w + y, "flops": 2 * M * K * N}
    elements = case["batch"] * case["m"] * case["n"]
    return {"bytes": elements * (size + 2), "flops": case["batch"] * _ortho_products(case["m"], case["n"])}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "layer_norm":
        with torch.no_grad():
            return _exact_norm(s)
    if case["op"] == "grouped_matmul":
        with torch.no_grad():
            return _exact_grouped(s)
    return [torch.stack([_exact_ortho(u) for u in s["update"]])]


def _exact_norm(s):
    """Row by row from var = E[(x - mean)^2] and dx = J^T (w dy), J the derivative of the normalised row."""
    rows, width = s["x"].shape
    w, b = s["weight"].double(), s["bias"].double()
    y, dx = [], []
    dw, db = torch.zeros_like(w), torch.zeros_like(w)
    step = max(1, (1 << 27) // width)
    for r in range(0, rows, step):
        x = s["x"][r:r + step].double()
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        sd = torch.sqrt(var + EPS_NORM)
        xhat = (x - mean) / sd
        y.append(torch.addcmul(b, xhat, w))
        if s["train"]:
            dy = s["grad"][r:r + step].double()
            t = dy * w
            along = torch.einsum("rd,rd->r", t, xhat)[:, None] / width
            dx.append((t - t.sum(1, keepdim=True) / width - along * xhat) / sd)
            dw += torch.einsum("rd,rd->d", dy, xhat)
            db += dy.sum(0)
    return [torch.cat(y), torch.cat(dx), dw, db] if s["train"] else [torch.cat(y)]


def _exact_grouped(s):
    ptr = s["ptr"].tolist()
    M, (G, K, N) = s["x"].shape[0], s["weight"].shape
    y = torch.zeros(M, N, dtype=torch.float64, device="cuda")
    dx = torch.zeros(M, K, dtype=torch.float64, device="cuda")
    dw = torch.zeros(G, K, N, dtype=torch.float64, device="cuda")
    for g in range(G):
        r = slice(ptr[g], ptr[g + 1])
        if r.start == r.stop:
            continue
        x, w = s["x"][r].double(), s["weight"][g].double()
        y[r] = x @ w
        if s["train"]:
            dy = s["grad"][r].double()
            dx[r], dw[g] = dy @ w.T, x.T @ dy
    return [y, dx, dw] if s["train"] else [y]


def _exact_ortho(update):
    """The polynomial a s + b s^3 + c s^5, applied five times to the singular values of the normalised matrix."""
    a, b, c = COEFFICIENTS
    x = update.double()
    x = x / (torch.linalg.norm(x) + EPS_ORTHO)
    for _ in range(STEPS):
        small = x.T @ x if x.shape[0] > x.shape[1] else x @ x.T
        poly = a * torch.eye(small.shape[0], dtype=torch.float64, device=x.device) + b * small + c * small @ small
        x = x @ poly if x.shape[0] > x.shape[1] else poly @ x
    return x
