"""The memory operators in float64 on the CPU, token by token and element by
element: what the kernels are compared with."""

from __future__ import annotations

import torch


def delta(q, k, v, g, beta, state, resets, scale):
    """The gated delta rule by its definition: (out, state), float64,
    differentiable.  q, k [T, N, Hk, DK]; state [N, Hv, DK, DV] or None."""
    T, N, hk, dk = q.shape
    hv, dv = v.shape[-2:]
    q, k, v, g, beta = (x.double() for x in (q, k, v, g, beta))
    S = torch.zeros(N, hv, dk, dv, dtype=torch.float64) if state is None else state.double()
    which = torch.arange(hv) // (hv // hk)
    out = []
    for t in range(T):
        S = S * torch.exp(g[t])[..., None, None]
        if resets is not None:
            S = torch.where(resets[t].bool()[:, None, None, None], torch.zeros_like(S), S)
        kt, qt = k[t][:, which], q[t][:, which]
        u = beta[t][..., None] * (v[t] - (S * kt[..., None]).sum(-2))
        S = S + kt[..., None] * u[..., None, :]
        out.append(scale * (S * qt[..., None]).sum(-2))
    return (torch.stack(out) if out else v.new_zeros(v.shape)), S


def rotate(x, w, positions, table, eps, unit, interleaved):
    """Norm and rotation of one kind of head, float64, differentiable."""
    x = x.double()
    square = (x * x).sum(-1, keepdim=True)
    y = x / torch.sqrt((square if unit else square / x.shape[-1]) + eps)
    if w is not None:
        y = y * w.double()
    if table is None:
        return y
    R = table.shape[1]
    turn = table.double()[positions.long()][..., None, :]
    c, s = turn[..., :R // 2], turn[..., R // 2:]
    a, b = (y[..., 0:R:2], y[..., 1:R:2]) if interleaved else (y[..., :R // 2], y[..., R // 2:R])
    a, b = a * c - b * s, a * s + b * c
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, y[..., R:]), -1)


def off(got, want) -> float:
    """2-norm of the difference over 2-norm of the result (0 / 0 is 0), the
    definition's rounded to the result's type."""
    want = want.detach().to(got.dtype).double()
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    d, n = float((got - want).norm()), float(want.norm())
    return d if n == 0.0 else d / n
