"""Operators of a policy with memory, as HIP kernels (include/nesle_memory.h).

A console's RAM or frame shows one instant.  These operators give a policy a
memory of the episode that acts one token at a time for every console and
trains on whole rollouts with gradients:

* ``qk_norm_rotate``    norms of queries and keys for each head with the
  position rotation, in one pass;
* ``gated_delta``       the gated delta rule over a rollout [T, N], memory
  dropped where an episode ends;
* ``gated_delta_step``  one token of it for every console, states in place;
* ``rotation_table``    cosines and sines for the rotation.

Tensors are time-major, [T, N, heads, dim] (a step's: [N, heads, dim]), float32
or bfloat16, on the GPU.  Queries, keys and values may be slices of one
projection's output: only the elements of a head have to lie next to each
other.  Arguments that do not fit raise ValueError.  Work is enqueued on the
current stream; nothing synchronises, so calls may be captured in a graph.
"""

from __future__ import annotations

import ctypes

import torch

from nesle_amd import abi

_DTYPES = {torch.float32: abi.MEM_F32, torch.bfloat16: abi.MEM_BF16}


def rotation_table(positions: int, rotated: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """float32 [positions, rotated]: row p has the cosines, then the sines, of
    p * base^(-2i / rotated), i = 0 .. rotated/2 - 1 (computed in float64)."""
    if positions < 1 or rotated < 8 or rotated % 8:
        raise ValueError(f"rotation_table: needs at least one position and a multiple of 8 elements, got {positions} "
                         f"and {rotated}")
    dev = device if device is not None else torch.device("cuda")
    rate = torch.pow(base, -torch.arange(0, rotated, 2, dtype=torch.float64, device=dev) / rotated)
    turn = torch.arange(positions, dtype=torch.float64, device=dev)[:, None] * rate
    return torch.cat((turn.cos(), turn.sin()), -1).float()


# ---- arguments ---------------------------------------------------------------------

def _need(ok: bool, who: str, name: str, want: str, t) -> None:
    if not ok:
        got = f"{tuple(t.shape)} {t.dtype} on {t.device}, strides {t.stride()}" if isinstance(t, torch.Tensor) else repr(t)
        raise ValueError(f"{who}: {name} must be {want}, got {got}")


def _check_heads(t, who: str, name: str, lead: tuple, dtype, dev) -> None:
    """A [*lead, heads, dim] tensor whose heads' elements lie next to each other."""
    _need(isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == dtype and t.device == dev
          and t.dim() == len(lead) + 2 and tuple(t.shape[:-2]) == lead and (t.stride(-1) == 1 or t.shape[-1] <= 1),
          who, name, f"a {dtype} tensor [{', '.join(map(str, lead))}, heads, dim] on {dev}, elements of a head next to "
          "each other", t)


def _check_plain(t, who: str, name: str, shape: tuple, dtype, dev) -> None:
    _need(isinstance(t, torch.Tensor) and t.dtype == dtype and t.device == dev and tuple(t.shape) == shape
          and t.is_contiguous(), who, name, f"a contiguous {dtype} tensor of shape {shape} on {dev}", t)


def _heads(t) -> abi.Heads:
    s = t.stride()
    return abi.Heads(t.data_ptr(), s[0] if len(s) == 4 else 0, s[-3], s[-2])


def _unit_last(t):
    """A gradient as autograd hands it over, made readable where it is not."""
    return t if t.stride(-1) == 1 else t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(name: str, args, dev) -> None:
    fn = getattr(abi.lib(), name)
    if torch.cuda.current_device() == dev.index:
        rc = fn(ctypes.byref(args), torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(ctypes.byref(args), torch.cuda.current_stream(dev).cuda_stream)
    abi._check(rc)


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---- norm and rotation --------------------------------------------------------------

def qk_norm_rotate(q, k, q_weight=None, k_weight=None, *, positions=None, table=None, eps: float = 1e-6,
                   unit: bool = False, interleaved: bool = False):
    """(q, k) normed for each head and rotated by position.

    q [..., q_heads, dim] and k [..., k_heads, dim] have one or two leading
    dimensions ([N] or [T, N]).  Each head x becomes
    x * weight / sqrt(mean(x^2) + eps) (``unit``: the sum of squares instead of
    the mean), weights float32 [dim] or None; then the pairs (i, i + R/2)
    (``interleaved``: (2i, 2i + 1)) of its first R elements are turned by the
    angles in row ``positions`` (int32, the leading shape) of ``table``
    (float32 [rows, R], ``rotation_table``).  Without a table nothing is
    turned.  A position outside the table makes its heads NaN.  dim and R are
    multiples of 8, dim at most 256.  Differentiable in q, k and the weights."""
    who = "qk_norm_rotate"
    _need(isinstance(q, torch.Tensor) and q.is_cuda and q.dtype in _DTYPES and q.dim() in (3, 4), who, "q",
          "a float32 or bfloat16 GPU tensor [N, heads, dim] or [T, N, heads, dim]", q)
    lead, dim, dev = tuple(q.shape[:-2]), q.shape[-1], q.device
    _check_heads(q, who, "q", lead, q.dtype, dev)
    _check_heads(k, who, "k", lead, q.dtype, dev)
    _need(k.shape[-1] == dim, who, "k", f"of q's head dimension {dim}", k)
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None:
            _check_plain(w, who, name, (dim,), torch.float32, dev)
            _need(w.data_ptr() % 16 == 0, who, name, "on a 16-byte boundary", w)
    rotated = 0
    if table is not None:
        _need(isinstance(table, torch.Tensor) and table.dim() == 2 and table.shape[0] > 0
              and table.shape[1] % 8 == 0 and table.shape[1] <= dim, who, "table",
              f"a float32 tensor [rows, R], R a multiple of 8 up to {dim}", table)
        _check_plain(table, who, "table", tuple(table.shape), torch.float32, dev)
        _need(table.data_ptr() % 16 == 0, who, "table", "on a 16-byte boundary", table)
        _check_plain(positions, who, "positions", lead, torch.int32, dev)
        rotated = table.shape[1]
    elif positions is not None:
        raise ValueError(f"{who}: positions need a table")
    how = (positions, table, rotated, float(eps), bool(unit), bool(interleaved))
    if _wants_grad(q, k, q_weight, k_weight):
        return _QkNormRotate.apply(q, k, q_weight, k_weight, how)
    return _qk_forward(q, k, q_weight, k_weight, how)


def _qk_args(q, k, q_weight, k_weight, how) -> abi.QkArgs:
    positions, table, rotated, eps, unit, interleaved = how
    a = abi.QkArgs(_DTYPES[q.dtype], q.shape[0] if q.dim() == 4 else 1, q.shape[-3], q.shape[-2], k.shape[-2],
                   q.shape[-1], rotated, unit, interleaved, eps)
    a.q, a.k = _heads(q), _heads(k)
    a.q_weight, a.k_weight = _ptr(q_weight), _ptr(k_weight)
    if rotated:
        a.positions, a.table, a.table_rows = positions.data_ptr(), table.data_ptr(), table.shape[0]
    return a


def _qk_forward(q, k, q_weight, k_weight, how):
    a = _qk_args(q, k, q_weight, k_weight, how)
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    a.q_out, a.k_out = q_out.data_ptr(), k_out.data_ptr()
    _call("nesle_qk_norm_rotate", a, q.device)
    return q_out, k_out


class _QkNormRotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, how):
        ctx.save_for_backward(q, k, q_weight, k_weight, how[0], how[1])
        ctx.how = how[2:]
        return _qk_forward(q, k, q_weight, k_weight, how)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, positions, table = ctx.saved_tensors
        a = _qk_args(q, k, q_weight, k_weight, (positions, table, *ctx.how))
        dq_out, dk_out = _unit_last(dq_out), _unit_last(dk_out)
        a.dq_out, a.dk_out = _heads(dq_out), _heads(dk_out)
        dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        dk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        dwq = None if q_weight is None else torch.empty_like(q_weight)
        dwk = None if k_weight is None else torch.empty_like(k_weight)
        a.dq, a.dk, a.dq_weight, a.dk_weight = dq.data_ptr(), dk.data_ptr(), _ptr(dwq), _ptr(dwk)
        floats = int(abi.lib().nesle_qk_scratch_floats(ctypes.byref(a)))
        scratch = torch.empty(floats, dtype=torch.float32, device=q.device) if floats else None
        a.scratch = _ptr(scratch)
        _call("nesle_qk_norm_rotate_grad", a, q.device)
        return dq, dk, dwq, dwk, None


# ---- the gated delta rule -----------------------------------------------------------

def _check_delta(who: str, q, k, v, g, beta, state, resets, lead: int):
    _need(isinstance(q, torch.Tensor) and q.is_cuda and q.dtype in _DTYPES and q.dim() == lead + 2, who, "q",
          f"a float32 or bfloat16 GPU tensor [{'T, ' if lead == 2 else ''}N, heads, dim]", q)
    shape, dev = tuple(q.shape[:-2]), q.device
    _check_heads(q, who, "q", shape, q.dtype, dev)
    _check_heads(k, who, "k", shape, q.dtype, dev)
    _check_heads(v, who, "v", shape, q.dtype, dev)
    _need(k.shape == q.shape, who, "k", f"of q's shape {tuple(q.shape)}", k)
    hk, dk = q.shape[-2:]
    hv, dv = v.shape[-2:]
    _need(hk > 0 and hv > 0 and hv % hk == 0, who, "v", f"of a multiple of {hk} heads", v)
    for name, d in (("q", dk), ("v", dv)):
        if d % 8 or not 8 <= d <= abi.DELTA_MAX_DIM:
            raise ValueError(f"{who}: {name}'s head dimension must be a multiple of 8 up to {abi.DELTA_MAX_DIM}, got {d}")
    _check_plain(g, who, "g", (*shape, hv), torch.float32, dev)
    _check_plain(beta, who, "beta", (*shape, hv), torch.float32, dev)
    if state is not None:
        _check_plain(state, who, "state", (shape[-1], hv, dk, dv), torch.float32, dev)
        _need(state.data_ptr() % 16 == 0, who, "state", "on a 16-byte boundary", state)
    if resets is not None:
        _check_plain(resets, who, "resets", shape, torch.bool if getattr(resets, "dtype", None) == torch.bool else torch.uint8,
                     dev)


def _delta_args(q, k, v, g, beta, state, resets, scale) -> abi.DeltaArgs:
    a = abi.DeltaArgs(_DTYPES[q.dtype], q.shape[0] if q.dim() == 4 else 1, q.shape[-3], q.shape[-2], v.shape[-2],
                      q.shape[-1], v.shape[-1], scale)
    a.q, a.k, a.v = _heads(q), _heads(k), _heads(v)
    a.g, a.beta, a.resets, a.state = g.data_ptr(), beta.data_ptr(), _ptr(resets), _ptr(state)
    return a


def gated_delta_step(q, k, v, g, beta, state, *, resets=None, scale: float | None = None):
    """One token of the gated delta rule for every console (``gated_delta``):
    q, k [N, k_heads, k_dim], v [N, v_heads, v_dim], g, beta [N, v_heads],
    resets [N]; ``state`` [N, v_heads, k_dim, v_dim] is updated in place.
    Returns the output [N, v_heads, v_dim].  Not differentiable: acting."""
    who = "gated_delta_step"
    _check_delta(who, q, k, v, g, beta, state, resets, 1)
    _need(state is not None, who, "state", "a tensor", state)
    if _wants_grad(q, k, v, g, beta, state):
        raise ValueError(f"{who} has no gradient: use gated_delta, or torch.no_grad()")
    a = _delta_args(q, k, v, g, beta, state, resets, q.shape[-1] ** -0.5 if scale is None else float(scale))
    out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    a.out, a.state_out = out.data_ptr(), a.state
    _call("nesle_delta_step", a, q.device)
    return out


def gated_delta(q, k, v, g, beta, *, state=None, resets=None, scale: float | None = None):
    """The gated delta rule over a rollout: (output, state after it).

    Each head of each console keeps a float32 state S [k_dim, v_dim].  A token
    first lets it decay, S <- exp(g) S, or drops it where ``resets`` is set
    (an episode's first token), then writes what the state gets wrong about its
    key, S <- S + k (beta (v - S^T k))^T, and reads out = scale S^T q.

    q, k [T, N, k_heads, k_dim] (keys of about unit length), v [T, N, v_heads,
    v_dim], g and beta float32 [T, N, v_heads] (g <= 0; -inf drops the state),
    resets bool or uint8 [T, N], state float32 [N, v_heads, k_dim, v_dim]
    (None: zeros).  v_heads is a multiple of k_heads: value head h goes with
    key head h // (v_heads // k_heads).  Head dimensions are multiples of 8 up
    to 128; T and N may be 0; scale defaults to k_dim ** -0.5.  A padded token
    is one with g = 0 and beta = 0.  The output has q's type; the new state is
    float32, a tensor of its own.  Differentiable in q, k, v, g, beta and
    state.  No value of a dropped state, and nothing that is not finite in a
    later token, reaches an output it does not belong to; the gradient of
    inputs that are not finite is unspecified."""
    who = "gated_delta"
    _check_delta(who, q, k, v, g, beta, state, resets, 2)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if _wants_grad(q, k, v, g, beta, state):
        return _GatedDelta.apply(q, k, v, g, beta, state, resets, scale)
    return _delta_forward(q, k, v, g, beta, state, resets, scale, False)[:2]


def _delta_forward(q, k, v, g, beta, state, resets, scale, keep: bool):
    a = _delta_args(q, k, v, g, beta, state, resets, scale)
    out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    after = torch.empty((v.shape[1], v.shape[2], q.shape[3], v.shape[3]), dtype=torch.float32, device=v.device)
    a.out, a.state_out = out.data_ptr(), after.data_ptr()
    saved = None
    if keep:
        floats = int(abi.lib().nesle_delta_saved_floats(ctypes.byref(a)))
        if floats:
            saved = torch.empty(floats, dtype=torch.float32, device=v.device)
            a.saved = saved.data_ptr()
    _call("nesle_delta_forward", a, q.device)
    return out, after, saved


class _GatedDelta(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, state, resets, scale):
        out, after, saved = _delta_forward(q, k, v, g, beta, state, resets, scale, True)
        ctx.save_for_backward(q, k, v, g, beta, state, resets, saved)
        ctx.scale = scale
        return out, after

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dafter):
        q, k, v, g, beta, state, resets, saved = ctx.saved_tensors
        a = _delta_args(q, k, v, g, beta, state, resets, ctx.scale)
        a.saved = _ptr(saved)
        dout, dafter = _unit_last(dout), dafter.contiguous()
        a.dout, a.dstate_out = _heads(dout), dafter.data_ptr()
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        dg, dbeta = torch.empty_like(g), torch.empty_like(beta)
        dstate = torch.empty_like(state) if state is not None and ctx.needs_input_grad[5] else None
        a.dq, a.dk, a.dv, a.dg, a.dbeta, a.dstate = (dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dg.data_ptr(),
                                                     dbeta.data_ptr(), _ptr(dstate))
        floats = int(abi.lib().nesle_delta_scratch_floats(ctypes.byref(a)))
        scratch = torch.empty(floats, dtype=torch.float32, device=q.device) if floats else None
        a.scratch = _ptr(scratch)
        _call("nesle_delta_backward", a, q.device)
        return dq, dk, dv, dg, dbeta, dstate, None, None
