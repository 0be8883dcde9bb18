"""Plain 64-bit forms of the operators around routed experts, embeddings and
8-bit products, and the error bounds their tests hold the kernels to (beside
those of layer_reference).

Routing.  A score's fp32 error, relative: the argument x - max rounds by
2^-24 |x - max|, the exponential by 2 ulp (2^-22), the row's sum of E
exponentials by ``sum_bound(E)`` and 2^-22 of its terms, the two divisions by
2^-24 each.  ``score_error`` is their sum with the exponent's part at the
largest distance of a chosen expert; a renormalised weight has it twice.
"""

import numpy as np
import torch

from layer_reference import sum_bound

BLOCK, LARGEST, TINY = 128, 448.0, 2.0 ** -100


def _descending(values):
    """Indexes in descending order, the lowest first among equal ones, NaN last."""
    return np.lexsort((np.arange(values.size), -np.where(np.isnan(values), -np.inf, values), np.isnan(values)))


def route_choice(logits, k, bias=None, scoring="softmax", groups=1, top_groups=1, group_best=1):
    """experts [T, k] of logits [T, E] (numpy, row by row)."""
    x = logits.double().cpu().numpy()
    T, E = x.shape
    by_logit = bias is None and (groups == top_groups or group_best == 1)
    with np.errstate(all="ignore"):
        if by_logit:
            c = x.copy()
        elif scoring == "sigmoid":
            c = 1 / (1 + np.exp(-x))
        else:
            m = x.max(1, keepdims=True)
            e = np.exp(x - np.where(np.isneginf(m), 0, m))
            z = e.sum(1, keepdims=True)
            c = np.where(z == 0, 0, e / z)
        if bias is not None:
            c = c + bias.double().cpu().numpy()
        out = np.empty((T, k), dtype=np.int64)
        for t in range(T):
            allowed = np.ones(E, dtype=bool)
            if top_groups < groups:
                per = c[t].reshape(groups, -1)
                score = np.array([g[_descending(g)[:group_best]].sum() for g in per])
                allowed = np.isin(np.arange(E) // (E // groups), _descending(score)[:top_groups])
            order = _descending(c[t])
            out[t] = order[allowed[order]][:k]
    return torch.from_numpy(out)


def route_weights(logits, experts, scoring, renormalize, scale):
    """weights of the given experts in 64 bits, differentiable (logits double)."""
    if scoring == "softmax":
        m = logits.amax(1, keepdim=True)
        e = torch.exp(logits - torch.where(torch.isneginf(m), torch.zeros_like(m), m).detach())
        z = e.sum(1, keepdim=True)
        score = torch.where(z == 0, torch.zeros_like(e), e / torch.where(z == 0, torch.ones_like(z), z))
    else:
        score = torch.sigmoid(logits)
    s = score.gather(1, experts.long())
    return scale * (s / (s.sum(1, keepdim=True) + 1e-20) if renormalize else s)


def score_error(logits, experts, scoring):
    """Relative error [T, 1] of the chosen experts' fp32 scores."""
    x = logits.double()
    far = x.gather(1, experts.long())
    far = x.amax(1, keepdim=True) - far if scoring == "softmax" else far.abs()
    far = torch.where(torch.isfinite(far), far, torch.zeros_like(far)).amax(1, keepdim=True)
    return far * 2.0 ** -24 + 2.0 ** -21 + sum_bound(logits.shape[1])


def route_gradient_slack(logits, experts, grad, scoring, renormalize, scale):
    """fp32 error of the logits' gradient [T, E]: the score error on every term of its formula, each taken with its
    magnitude (d has two differences, the row's sum and the product one more each)."""
    x = logits.double()
    score = torch.softmax(x, 1) if scoring == "softmax" else torch.sigmoid(x)
    score = torch.nan_to_num(score)
    s = score.gather(1, experts.long())
    g = grad.double().abs() * abs(scale)
    S = s.sum(1, keepdim=True) + 1e-20 if renormalize else torch.ones_like(s[:, :1])
    d = (g + (g * s).sum(1, keepdim=True) / S) / S if renormalize else g
    rel = 6 * score_error(logits, experts, scoring)
    own = torch.zeros_like(x).scatter_(1, experts.long(), d)
    if scoring == "softmax":
        return rel * score * (own + (d * s).sum(1, keepdim=True))
    return rel * own * score


def plan_reference(experts, num_experts):
    """(group_ptr, position, source) of a stable sort."""
    e = experts.reshape(-1).cpu().numpy().astype(np.int64)
    key = np.where((e < 0) | (e >= num_experts), num_experts, e)
    order = np.argsort(key, kind="stable")
    counts = np.bincount(key, minlength=num_experts + 1)[:num_experts]
    ptr = np.concatenate([[0], np.cumsum(counts)])
    position, source = np.full(e.size, -1), np.full(e.size, -1)
    live = order[:ptr[-1]]
    source[:live.size] = live
    position[live] = np.arange(live.size)
    as_int = lambda a: torch.from_numpy(a.astype(np.int32))  # noqa: E731
    return as_int(ptr), as_int(position).view(experts.shape), as_int(source)


def combine_reference(rows, position, weights=None):
    """y and its fp32 slack in 64 bits."""
    p = position.long()
    here = (p >= 0)[:, :, None]
    r = torch.where(here, rows.double()[p.clamp(min=0)], torch.zeros((), dtype=torch.float64, device=rows.device))
    if weights is not None:
        r = torch.where(here, r * weights.double()[:, :, None], torch.zeros_like(r))
    return r.sum(1), sum_bound(p.shape[1]) * r.abs().sum(1)


def embedding_grad_reference(ids, grad, rows, scale, padding_id=None):
    ids, g = ids.reshape(-1).long(), grad.reshape(-1, grad.shape[-1]).double()
    keep = (ids >= 0) & (ids < rows)
    if padding_id is not None:
        keep &= ids != padding_id
    ids, g = ids[keep], g[keep]
    zero = torch.zeros(rows, g.shape[1], dtype=torch.float64, device=g.device)
    count = torch.bincount(ids, minlength=rows).double()[:, None]
    total, mag = zero.index_add(0, ids, g) * scale, zero.index_add(0, ids, g.abs()) * abs(scale)
    return total, (count / 8 + 16) * 2.0 ** -23 * mag


def _largest(m):
    """Scales of blocks; by a tensor, since torch multiplies by a number's rounded reciprocal."""
    return m.clamp(min=TINY) / torch.full_like(m, LARGEST)


def quantize_reference(x):
    """(q as fp32 values, scale) of the rows of x [rows, width], in fp32 arithmetic: both are defined by it."""
    rows, width = x.shape
    blocks = -(-width // BLOCK)
    f = torch.zeros(rows, blocks * BLOCK, device=x.device)
    f[:, :width] = x.float()
    f = f.view(rows, blocks, BLOCK)
    finite = torch.where(torch.isfinite(f), f, torch.zeros_like(f))
    scale = _largest(finite.abs().amax(2))
    q = (finite / scale[:, :, None]).clamp(-LARGEST, LARGEST).to(torch.float8_e4m3fn).float()
    q = torch.where(torch.isfinite(f), q, torch.full_like(q, float("nan")))
    return q.view(rows, -1)[:, :width], scale


def quantize_weight_reference(w):
    """(q [G, N, K] as fp32 values, scale [G, N blocks, K blocks]) of w [G, K, N]."""
    G, K, N = w.shape
    kb, nb = -(-K // BLOCK), -(-N // BLOCK)
    f = torch.zeros(G, nb * BLOCK, kb * BLOCK, device=w.device)
    f[:, :N, :K] = w.float().transpose(1, 2)
    f = f.view(G, nb, BLOCK, kb, BLOCK)
    finite = torch.where(torch.isfinite(f), f, torch.zeros_like(f))
    scale = _largest(finite.abs().amax((2, 4)))
    q = (finite / scale[:, :, None, :, None]).clamp(-LARGEST, LARGEST).to(torch.float8_e4m3fn).float()
    q = torch.where(torch.isfinite(f), q, torch.full_like(q, float("nan")))
    return q.view(G, nb * BLOCK, kb * BLOCK)[:, :N, :K], scale


def fp8_reference(q, scale, wq, wscale, ptr):
    """The product in 64 bits of what is held in 8, and its slack: sums of blocks as any sum of K products."""
    ptr = [int(p) for p in ptr.tolist()]
    G, N, K = wq.shape
    at_n, at_k = torch.arange(N, device=q.device) // BLOCK, torch.arange(K, device=q.device) // BLOCK
    x = q.double() * scale.double()[:, at_k]
    y = torch.zeros(q.shape[0], N, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(y)
    for g in range(G):
        r = slice(ptr[g], ptr[g + 1])
        w = wq[g].double() * wscale[g].double()[at_n][:, at_k]
        y[r] = x[r] @ w.T
        mag[r] = x[r].abs() @ w.abs().T
    return y, sum_bound(K) * mag
