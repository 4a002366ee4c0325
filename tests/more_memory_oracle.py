"""The memory layer's further operators in float64 on the CPU, token by token and
action by action: what the kernels are compared with."""

from __future__ import annotations

import math

import torch


def decay(q, k, v, g, state, resets, scale):
    """Linear attention with a decay for each head by its definition: (out, state),
    float64, differentiable.  q, k [T, N, Hk, DK]; g [Hv]; state or None."""
    T, N, hk, dk = q.shape
    hv, dv = v.shape[-2:]
    q, k, v, g = (x.double() for x in (q, k, v, g))
    S = torch.zeros(N, hv, dk, dv, dtype=torch.float64) if state is None else state.double()
    which = torch.arange(hv) // (hv // hk)
    out = []
    for t in range(T):
        S = S * torch.exp(g)[:, None, None]
        if resets is not None:
            S = torch.where(resets[t].bool()[:, None, None, None], torch.zeros_like(S), S)
        S = S + k[t][:, which][..., None] * v[t][..., None, :]
        out.append(scale * (S * q[t][:, which][..., None]).sum(-2))
    return (torch.stack(out) if out else v.new_zeros(v.shape)), S


def layer_norm(x, weight, bias, eps):
    x = x.double()
    off = x - x.mean(-1, keepdim=True)
    y = off / torch.sqrt((off * off).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.double()
    return y if bias is None else y + bias.double()


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(action, logprob) of one row, lists of Python floats."""
    top = max(logits)
    if any(math.isnan(x) or x == math.inf for x in logits) or top == -math.inf or math.isnan(u):
        return -1, math.nan
    if temperature == 0.0:
        return logits.index(top), 0.0
    w = [math.exp((x - top) / temperature) if x > -math.inf else 0.0 for x in logits]
    order = sorted(range(len(w)), key=lambda i: (-logits[i], i))
    if top_k:
        for i in order[top_k:]:
            w[i] = 0.0
    share, before = top_p * math.fsum(w), []
    for i in order:
        if top_p < 1.0 and not math.fsum(before) < share:
            w[i] = 0.0
        before.append(w[i])
    w = [x if x >= min_p else 0.0 for x in w]
    total, run = math.fsum(w), []
    last = max(i for i, x in enumerate(w) if x > 0.0)
    for i, x in enumerate(w):
        run.append(x)
        if x > 0.0 and (math.fsum(run) > max(u, 0.0) * total or i == last):
            return i, math.log(x / total)
    raise AssertionError
