"""Measured cases of the operators around routed experts and learned node features.

A model that sends each node (or token) to a few experts computes the experts
of a row from its scores (``route_experts``), sorts the rows by expert so that
one ``grouped_matmul`` multiplies them (``expert_plan``, ``dispatch_rows``) and
adds the experts' results of a row up again (``combine_rows``).  Served, the
products run in 8-bit floating point with a scale for each block of 128
(``quantize_fp8``, ``grouped_matmul_fp8``).  In front of the layers stands a
table of learned features (``embedding``), whose gradient adds the rows of each
id up.

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

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BLOCK = 128          # elements that share a scale
LARGEST = 448.0      # of e4m3
TINY = 2.0 ** -100   # least block maximum that sets a scale


def listed():
    return [
        # one decoding step of a served model: nine rows, the cost is the call itself
        {"name": "route_few_rows", "op": "route", "tokens": 9, "experts": 32, "k": 4, "scoring": "softmax",
         "bias": False, "groups": 1, "top_groups": 1, "group_best": 1, "renormalize": True, "scale": 1.0,
         "dtype": "bf16", "train": False},
        # a training batch, softmax scores as they are, forward and backward
        {"name": "route_softmax_train", "op": "route", "tokens": 16411, "experts": 64, "k": 6, "scoring": "softmax",
         "bias": False, "groups": 1, "top_groups": 1, "group_best": 1, "renormalize": False, "scale": 1.0,
         "dtype": "bf16", "train": True},
        # sigmoid scores, a balance bias and half of eight groups of experts, forward and backward
        {"name": "route_groups_train", "op": "route", "tokens": 65537, "experts": 256, "k": 8, "scoring": "sigmoid",
         "bias": True, "groups": 8, "top_groups": 4, "group_best": 2, "renormalize": True, "scale": 2.5,
         "dtype": "fp32", "train": True},
        # the rows of the decoding step to their experts and back
        {"name": "rows_few", "op": "rows", "tokens": 9, "experts": 32, "k": 4, "width": 1024, "dtype": "bf16",
         "padded": False, "train": False},
        # rows that are not 16-byte aligned and a padded batch (a part of the rows has no expert)
        {"name": "rows_odd_train", "op": "rows", "tokens": 4099, "experts": 46, "k": 2, "width": 1001,
         "dtype": "fp16", "padded": True, "train": True},
        # the rows of a large expert layer, forward and backward: bound by memory
        {"name": "rows_train", "op": "rows", "tokens": 32771, "experts": 64, "k": 8, "width": 1024, "dtype": "bf16",
         "padded": False, "train": True},
        # features of nine nodes of a served model
        {"name": "embed_few_rows", "op": "embedding", "ids": 9, "table": 32003, "width": 256, "dtype": "fp16",
         "train": False},
        # a training batch whose ids follow a power law, forward and backward
        {"name": "embed_train", "op": "embedding", "ids": 16411, "table": 50021, "width": 1024, "dtype": "bf16",
         "train": True},
        # as many ids as this repository's widest layer case has rows, fp32 table of a large graph
        {"name": "embed_wide_train", "op": "embedding", "ids": 524287, "table": 131071, "width": 512,
         "dtype": "fp32", "train": True},
        # nine routed rows over 32 experts in 8 bits: bound by reading the experts that have a row
        {"name": "fp8_few_rows", "op": "fp8", "rows": 9, "groups": 32, "k": 1024, "n": 512, "dtype": "bf16",
         "skew": False},
        # experts of odd widths whose last blocks are short, very unequal groups
        {"name": "fp8_odd", "op": "fp8", "rows": 5003, "groups": 46, "k": 400, "n": 272, "dtype": "fp16",
         "skew": True},
        # a large expert layer served in 8 bits: bound by the products
        {"name": "fp8_experts", "op": "fp8", "rows": 65537, "groups": 64, "k": 1024, "n": 2048, "dtype": "bf16",
         "skew": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same operators: the smallest call to one that costs no more than the largest listed one."""
    op = rng.choice(("route", "rows", "embedding", "fp8"))
    dtype = rng.choice(("fp16", "bf16", "fp32"))
    wide = 2 if dtype == "fp32" else 1
    if op == "route":
        while True:
            tokens = _log_int(rng, 1, 65537)
            groups = rng.choice((1, 1, 1, 2, 4, 8))
            each = _log_int(rng, 2, 512 // groups)
            if tokens * groups * each <= 65537 * 256:
                break
        top_groups = rng.randint(1, groups)
        return {"op": op, "tokens": tokens, "experts": groups * each,
                "k": rng.randint(1, min(16, top_groups * each)), "scoring": rng.choice(("softmax", "sigmoid")),
                "bias": rng.random() < 0.5, "groups": groups, "top_groups": top_groups,
                "group_best": rng.choice((1, 2)), "renormalize": rng.random() < 0.5, "scale": rng.choice((1.0, 2.5)),
                "dtype": dtype, "train": rng.random() < 0.5}
    if op == "rows":
        while True:
            tokens, experts, width = _log_int(rng, 1, 65537), _log_int(rng, 1, 256), _log_int(rng, 8, 4096)
            k = rng.randint(1, min(8, experts))
            if wide * tokens * k * width <= 32771 * 8 * 1024:
                break
        return {"op": op, "tokens": tokens, "experts": experts, "k": k, "width": width, "dtype": dtype,
                "padded": rng.random() < 0.5, "train": rng.random() < 0.5}
    if op == "embedding":
        while True:
            ids, table, width = _log_int(rng, 1, 524287), _log_int(rng, 2, 1000003), _log_int(rng, 8, 4096)
            if wide * (ids + table) * width <= 2 * (524287 + 131071) * 512:
                break
        return {"op": op, "ids": ids, "table": table, "width": width, "dtype": dtype, "train": rng.random() < 0.5}
    while True:
        rows, groups = _log_int(rng, 1, 65537), _log_int(rng, 1, 128)
        k, n = 16 * _log_int(rng, 1, 128), 16 * _log_int(rng, 1, 128)
        if rows * k * n <= 65537 * 1024 * 2048 and groups * k * n <= 64 * 1024 * 2048:
            break
    return {"op": op, "rows": rows, "groups": groups, "k": k, "n": n, "dtype": dtype, "skew": rng.random() < 0.5}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    state = dict(case)
    if case["op"] == "route":
        T, E = case["tokens"], case["experts"]
        # experts differ in how much they are liked, and the bias works against it
        liked = 0.5 * normal(E)
        state["logits"] = (1.5 * normal(T, E) + liked).to(dtype)
        state["bias"] = (0.05 * normal(E) - 0.1 * liked) if case["bias"] else None
        if case["train"]:
            state["grad"] = normal(T, case["k"])
            state["logits"].requires_grad_(own)
    elif case["op"] == "rows":
        T, E, k, D = case["tokens"], case["experts"], case["k"], case["width"]
        liked = torch.exp(normal(E))
        experts = torch.topk(torch.log(uniform(T, E) + 1e-9) / liked, k, dim=1).indices.to(torch.int32)
        if case["padded"]:
            experts[uniform(T) < 0.125] = -1
        w = uniform(T, k) + 0.05
        state.update(x=normal(T, D).to(dtype), expert=experts, weights=w / w.sum(1, keepdim=True),
                     out=normal(T * k, D).to(dtype))
        if case["train"]:
            state.update(grad=normal(T, D).to(dtype), grad_rows=normal(T * k, D).to(dtype))
            for name in ("x", "weights", "out"):
                state[name].requires_grad_(own)
    elif case["op"] == "embedding":
        N, V, D = case["ids"], case["table"], case["width"]
        rank = torch.exp(uniform(N).double() * math.log(V + 1)).long().clamp(1, V) - 1   # density 1 / rank
        state.update(id=torch.randperm(V, generator=g, device="cuda")[rank], table=(normal(V, D) / math.sqrt(D)).to(dtype),
                     scale=math.sqrt(D))
        if case["train"]:
            state["grad"] = normal(N, D).to(dtype)
            state["table"].requires_grad_(own)
    else:
        M, G, K, N = case["rows"], case["groups"], case["k"], case["n"]
        share = uniform(G) ** (4.0 if case["skew"] else 0.5) + 1e-4
        owner = torch.multinomial(share, M, replacement=True, generator=g)
        ptr = torch.zeros(G + 1, dtype=torch.int64, device="cuda")
        ptr[1:] = torch.cumsum(torch.bincount(owner, minlength=G), 0)
        # rows of unequal size; the weights are laid out once, as a served model keeps them: [G, N, K] in 8 bits
        x = normal(M, K) * torch.exp(normal(M, 1))
        kb, nb = -(-K // BLOCK), -(-N // BLOCK)
        w = torch.zeros(G, nb * BLOCK, kb * BLOCK, device="cuda")
        w[:, :N, :K] = normal(G, N, K) / math.sqrt(K)
        w = w.view(G, nb, BLOCK, kb, BLOCK)
        scale = w.abs().amax((2, 4)).clamp(min=TINY) / LARGEST
        q = (w / scale[:, :, None, :, None]).view(G, nb * BLOCK, kb * BLOCK)[:, :N, :K]
        state.update(x=x.to(dtype), weight=q.contiguous().to(torch.float8_e4m3fn), weight_scale=scale,
                     ptr=ptr.to(torch.int32))
        # the plain form's row tiles: about two for each group of even size
        state["tile"] = max(16, 1 << max(0, (M // max(1, G)).bit_length() - 1))
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
    return {"route": _plain_route, "rows": _plain_rows, "embedding": _plain_embedding, "fp8": _plain_fp8}[state["op"]](state)


def _run_own(s):
    lib = _operators()
    if s["op"] == "route":
        weights, experts = lib.route_experts(s["logits"], s["k"], bias=s["bias"], scoring=s["scoring"],
                                             groups=s["groups"], top_groups=s["top_groups"],
                                             group_best=s["group_best"], renormalize=s["renormalize"],
                                             scale=s["scale"])
        if not s["train"]:
            return [weights, experts]
        return [weights.detach(), experts, *torch.autograd.grad(weights, [s["logits"]], s["grad"])]
    if s["op"] == "rows":
        group_ptr, position, source = lib.expert_plan(s["expert"], s["experts"])
        rows = lib.dispatch_rows(s["x"], position, source)
        y = lib.combine_rows(s["out"], position, source, s["weights"])
        if not s["train"]:
            return [group_ptr, position, source, rows, y]
        dout, dw = torch.autograd.grad(y, [s["out"], s["weights"]], s["grad"])
        (dx,) = torch.autograd.grad(rows, [s["x"]], s["grad_rows"])
        return [group_ptr, position, source, rows.detach(), y.detach(), dx, dout, dw]
    if s["op"] == "embedding":
        y = lib.embedding(s["id"], s["table"], scale=s["scale"])
        if not s["train"]:
            return [y]
        return [y.detach(), *torch.autograd.grad(y, [s["table"]], s["grad"])]
    q, scale = lib.quantize_fp8(s["x"])
    return [lib.grouped_matmul_fp8(q, scale, s["weight"], s["weight_scale"], s["ptr"], out_dtype=s["x"].dtype)]


def _plain_route(s):
    """The choice in 64 bits (scores next to each other decide it), ties to the lowest index by a stable sort."""
    x, k, G = s["logits"].double(), s["k"], s["groups"]
    T, E = x.shape
    if s["scoring"] == "softmax":
        score = torch.exp(x - x.amax(1, keepdim=True))
        score = score / score.sum(1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-x))
    choice = score if s["bias"] is None else score + s["bias"].double()
    if G > 1:
        best = torch.sort(choice.view(T, G, E // G), dim=2, descending=True).values[:, :, :s["group_best"]].sum(2)
        kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :s["top_groups"]]
        out = torch.ones(T, G, dtype=torch.bool, device=x.device)
        out[torch.arange(T, device=x.device)[:, None], kept] = False
        choice = choice.masked_fill(out.repeat_interleave(E // G, dim=1), -math.inf)
    experts = torch.sort(choice, dim=1, descending=True, stable=True).indices[:, :k]
    score = score.float()
    chosen = torch.gather(score, 1, experts)
    total = chosen.sum(1, keepdim=True) + 1e-20
    weights = (chosen / total if s["renormalize"] else chosen) * s["scale"]
    if not s["train"]:
        return [weights, experts.int()]
    d = s["grad"] * s["scale"]
    if s["renormalize"]:
        d = (d - (d * chosen / total).sum(1, keepdim=True)) / total
    dscore = torch.zeros_like(score)
    dscore[torch.arange(T, device=x.device)[:, None], experts] = d
    if s["scoring"] == "softmax":
        dx = score * (dscore - (dscore * score).sum(1, keepdim=True))
    else:
        dx = dscore * score * (1 - score)
    return [weights, experts.int(), dx.to(s["logits"].dtype)]


def _plain_rows(s):
    e, (T, k), E = s["expert"].long(), s["expert"].shape, s["experts"]
    dtype, dev, D = s["x"].dtype, s["x"].device, s["x"].shape[1]
    key = torch.where(e < 0, E, e).reshape(-1)
    order = torch.sort(key, stable=True).indices
    group_ptr = torch.zeros(E + 1, dtype=torch.int64, device=dev)
    group_ptr[1:] = torch.cumsum((key[order][:, None] == torch.arange(E, device=dev)).sum(0), 0)
    row = torch.arange(T * k, device=dev)
    position = torch.empty(T * k, dtype=torch.int64, device=dev)
    position[order] = row
    position = torch.where(e < 0, -1, position.view(T, k))
    source = torch.where(row < group_ptr[E], order, -1)
    here, there = (position >= 0)[:, :, None], (source >= 0)[:, None]
    take, put = position.clamp(min=0), source.clamp(min=0)
    rows = torch.where(there, s["x"].float()[put // k], 0)
    out = torch.where(here, s["out"].float()[take], 0)
    y = (s["weights"][:, :, None] * out).sum(1)
    found = [group_ptr.int(), position.int(), source.int(), rows.to(dtype), y.to(dtype)]
    if not s["train"]:
        return found
    grad = s["grad"].float()
    dw = (out * grad[:, None, :]).sum(2)
    dout = torch.where(there, s["weights"].reshape(-1)[put][:, None] * grad[put // k], 0)
    dx = torch.where(here, s["grad_rows"].float()[take], 0).sum(1)
    return found + [dx.to(dtype), dout.to(dtype), dw]


def _plain_embedding(s):
    table = s["table"].float()
    y = (table[s["id"]] * s["scale"]).to(s["table"].dtype)
    if not s["train"]:
        return [y]
    d = torch.zeros_like(table).index_add_(0, s["id"], s["grad"].float())
    return [y, (d * s["scale"]).to(s["table"].dtype)]


def _plain_fp8(s):
    """Each row's blocks of 128 rounded to 8 bits with a scale; then rows in tiles that belong to one group each (a
    tile's missing rows are zero), one batched product over the tiles."""
    dtype, (M, K), (G, N, _) = s["x"].dtype, s["x"].shape, s["weight"].shape
    kb, nb, dev = s["weight_scale"].shape[2], s["weight_scale"].shape[1], s["x"].device
    x = torch.zeros(M, kb * BLOCK, device=dev)
    x[:, :K] = s["x"].float()
    x = x.view(M, kb, BLOCK)
    scale = x.abs().amax(2, keepdim=True).clamp(min=TINY) / LARGEST
    x = ((x / scale).to(torch.float8_e4m3fn).float() * scale).view(M, kb * BLOCK)[:, :K]
    at_n, at_k = torch.arange(N, device=dev) // BLOCK, torch.arange(K, device=dev) // BLOCK
    weight = s["weight"].float() * s["weight_scale"][:, at_n][:, :, at_k]
    ptr, tile = s["ptr"].long(), s["tile"]
    first = torch.zeros(G + 1, dtype=torch.int64, device=dev)
    first[1:] = torch.cumsum((ptr[1:] - ptr[:-1] + tile - 1) // tile, 0)
    t = torch.arange(-(-M // tile) + G, device=dev)
    group = torch.searchsorted(first[1:], t, right=True).clamp(max=G - 1)
    row = (ptr[group] + (t - first[group]) * tile)[:, None] + torch.arange(tile, device=dev)
    valid = (row < ptr[group + 1][:, None]) & (t < first[G])[:, None]
    take, put = torch.where(valid, row, 0), torch.where(valid, row, M)
    out = torch.zeros(M + 1, N, device=dev)
    out[put] = torch.bmm(torch.where(valid[:, :, None], x[take], 0), weight[group].transpose(1, 2))
    return [out[:M].to(dtype)]


# --------------------------------------------------------------------------
# floors and the definition in 64 bits
# --------------------------------------------------------------------------

def _bytes(name):
    return 4 if name == "fp32" else 2


def work(case):
    size = _bytes(case["dtype"])
    if case["op"] == "route":
        scores, chosen = case["tokens"] * case["experts"], case["tokens"] * case["k"]
        b = scores * size + chosen * 8 + (4 * case["experts"] if case["bias"] else 0)
        if case["train"]:   # the weights' gradient read, the logits' written
            return {"bytes": b + chosen * 4 + scores * size, "flops": 8 * scores}
        return {"bytes": b, "flops": 4 * scores}
    if case["op"] == "rows":
        T, k, D = case["tokens"], case["k"], case["width"]
        live = 0.875 if case["padded"] else 1.0   # choices that have an expert
        token, row = T * D * size, T * k * D * size
        # every row of a result is written, those without a source as zeros; only the others are read
        b = T * k * 16 + 4 * (case["experts"] + 1) + live * token + row + live * row + token
        f = 2 * live * T * k * D
        if case["train"]:   # both gradients read, those of x, the experts' results and the weights written
            b += live * token + live * row + token + row + 4 * T * k
            f *= 3
        return {"bytes": b, "flops": f}
    if case["op"] == "embedding":
        N, V, D = case["ids"], case["table"], case["width"]
        seen = _distinct(N, V)
        b = 8 * N + (seen + N) * D * size
        if case["train"]:
            return {"bytes": b + (N + V) * D * size, "flops": 2 * N * D}
        return {"bytes": b, "flops": N * D}
    M, G, K, N = case["rows"], case["groups"], case["k"], case["n"]
    w = G * (1 - (1 - 1 / G) ** M) * (K * N + 4 * -(-K // BLOCK) * -(-N // BLOCK))   # the groups that M rows meet
    return {"bytes": M * K * size + w + M * N * size, "flops": 2 * M * K * N}


def _distinct(ids, table):
    """Expected distinct ones of `ids` ranks of density 1 / rank (rank r has the share log(1 + 1 / r) / log(table + 1))."""
    r = torch.arange(1, table + 1, dtype=torch.float64)
    return float(-torch.expm1(ids * torch.log1p(-torch.log1p(1 / r) / math.log(table + 1))).sum()) if table > 1 else 1.0


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"route": _exact_route, "rows": _exact_rows, "embedding": _exact_embedding, "fp8": _exact_fp8}[s["op"]](s)


def _first_largest(c):
    """Index of each row's largest value, the lowest of equal ones."""
    at = torch.arange(c.shape[1], device=c.device)
    return torch.where(c == c.amax(1, keepdim=True), at, c.shape[1]).amin(1)


def _exact_route(s):
    """Pick by pick; the gradient from the derivative of log weights."""
    x = s["logits"].detach().double()
    T, E = x.shape
    G, row = s["groups"], torch.arange(T, device=x.device)
    log_score = torch.log_softmax(x, 1) if s["scoring"] == "softmax" else torch.nn.functional.logsigmoid(x)
    score = log_score.exp()
    choice = score.clone() if s["bias"] is None else score + s["bias"].double()
    if G > 1:
        left, best = choice.reshape(T * G, E // G).clone(), torch.zeros(T * G, dtype=torch.float64, device=x.device)
        for _ in range(s["group_best"]):
            best += left.amax(1)
            left[torch.arange(T * G, device=x.device), _first_largest(left)] = -math.inf
        best, kept = best.view(T, G), torch.zeros(T, G, dtype=torch.bool, device=x.device)
        for _ in range(s["top_groups"]):
            at = _first_largest(best)
            kept[row, at] = True
            best[row, at] = -math.inf
        choice[~kept[:, torch.arange(E, device=x.device) // (E // G)]] = -math.inf
    picks = []
    for _ in range(s["k"]):
        picks.append(_first_largest(choice))
        choice[row, picks[-1]] = -math.inf
    experts = torch.stack(picks, 1)
    chosen = score.gather(1, experts)
    total = chosen.sum(1, keepdim=True) + 1e-20 if s["renormalize"] else torch.ones_like(chosen[:, :1])
    weights = s["scale"] * chosen / total
    if not s["train"]:
        return [weights, experts.int()]
    # d weight_j = weight_j (d log score_j - sum_i (chosen_i / total) d log score_i)
    gw = s["grad"].double() * weights
    u = gw - gw.sum(1, keepdim=True) * chosen / total if s["renormalize"] else gw
    if s["scoring"] == "softmax":   # d log score_j / d x_i = [i == j] - score_i
        dx = -score * u.sum(1, keepdim=True)
        dx.scatter_add_(1, experts, u)
    else:                           # 1 - score_j
        dx = torch.zeros_like(x).scatter_add_(1, experts, u * torch.sigmoid(-x).gather(1, experts))
    return [weights, experts.int(), dx]


def _exact_rows(s):
    """Expert by expert, from the places where its number stands."""
    e, k, E = s["expert"].reshape(-1), s["expert"].shape[1], s["experts"]
    places = [torch.nonzero(e == g).flatten() for g in range(E)]
    ptr, places = [0] + [p.numel() for p in places], torch.cat(places)
    live, total = places.numel(), e.numel()
    source = torch.full((total,), -1, dtype=torch.int64, device=e.device)
    source[:live] = places
    position = torch.full((total,), -1, dtype=torch.int64, device=e.device)
    position[places] = torch.arange(live, device=e.device)
    group_ptr = torch.tensor(ptr, device=e.device).cumsum(0)
    dtype, token, rank = torch.float64, places // k, places % k
    D = s["x"].shape[1]
    w = s["weights"].double()[token, rank][:, None]

    def to_rows(v):
        out = torch.zeros(total, D, dtype=dtype, device=e.device)
        out[:live] = v
        return out

    def to_tokens(v):
        return torch.zeros(s["x"].shape[0], D, dtype=dtype, device=e.device).index_add_(0, token, v)

    rows, out = to_rows(s["x"].double()[token]), s["out"][:live].double()
    found = [group_ptr.int(), position.view(-1, k).int(), source.int(), rows, to_tokens(w * out)]
    if not s["train"]:
        return found
    grad = s["grad"].double()[token]
    dw = torch.zeros(total, dtype=dtype, device=e.device)
    dw[places] = torch.einsum("rd,rd->r", out, grad)
    return found + [to_tokens(s["grad_rows"][:live].double()), to_rows(w * grad), dw.view(-1, k)]


def _exact_embedding(s):
    V, D = s["table"].shape
    y = s["table"].double().mul_(s["scale"])[s["id"]]
    if not s["train"]:
        return [y]
    order = torch.argsort(s["id"])
    ids, counts = torch.unique_consecutive(s["id"][order], return_counts=True)
    d = torch.zeros(V, D, dtype=torch.float64, device=y.device)
    d[ids] = torch.segment_reduce(s["grad"].double()[order], "sum", lengths=counts, axis=0)
    return [y, d.mul_(s["scale"])]


def _exact_fp8(s):
    """Group by group and block by block.  The scales are what fp32 holds of them, as a user is given them."""
    x, (G, N, K) = s["x"].double(), s["weight"].shape
    y = torch.zeros(x.shape[0], N, dtype=torch.float64, device=x.device)
    ptr = s["ptr"].tolist()
    for b in range(0, K, BLOCK):
        part = x[:, b:b + BLOCK]
        scale = (part.abs().amax(1, keepdim=True).clamp(min=TINY) / LARGEST).float().double()
        q = (part / scale).to(torch.float8_e4m3fn).double() * scale
        for g in range(G):
            w = s["weight"][g, :, b:b + BLOCK].double()
            w = w * s["weight_scale"][g, :, b // BLOCK].double().repeat_interleave(BLOCK)[:N, None]
            y[ptr[g]:ptr[g + 1]] += q[ptr[g]:ptr[g + 1]] @ w.T
    return [y]
