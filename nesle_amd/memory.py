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
# Acting calls these for one token at a time, where the host's time is the
# call's: messages are only made for an argument that is refused.

def _refuse(who: str, name: str, want: str, t) -> None:
    got = f"{tuple(t.shape)} {t.dtype} on {t.device}, strides {t.stride()}" if isinstance(t, torch.Tensor) else repr(t)
    raise ValueError(f"{who}: {name} must be {want}, got {got}")


def _check_first(t, who: str, name: str, dims: tuple) -> None:
    """The tensor that says type, device and leading dimensions."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in _DTYPES and t.dim() in dims and t.stride(-1) == 1):
        shapes = {3: "[N, heads, dim]", 4: "[T, N, heads, dim]"}
        _refuse(who, name, f"a float32 or bfloat16 GPU tensor {' or '.join(shapes[d] for d in dims)}, elements of a head "
                "next to each other", t)


def _check_heads(t, who: str, name: str, first) -> None:
    """A [..., heads, dim] tensor that goes with ``first``, whose heads'
    elements lie next to each other."""
    if not (isinstance(t, torch.Tensor) and t.dtype == first.dtype and t.device == first.device
            and t.dim() == first.dim() and t.shape[:-2] == first.shape[:-2] and t.stride(-1) == 1):
        _refuse(who, name, f"a {first.dtype} tensor [{', '.join(map(str, first.shape[:-2]))}, heads, dim] on "
                f"{first.device}, elements of a head next to each other", t)


def _check_plain(t, who: str, name: str, shape: tuple, dtype, dev, aligned: bool = False) -> None:
    if not (isinstance(t, torch.Tensor) and t.dtype == dtype and t.device == dev and t.shape == shape
            and t.is_contiguous()):
        _refuse(who, name, f"a contiguous {dtype} tensor of shape {tuple(shape)} on {dev}", t)
    if aligned and t.data_ptr() % 16:
        _refuse(who, name, "on a 16-byte boundary", t)


def _heads(t) -> tuple:
    """nesle_heads of a [N, heads, dim] or [T, N, heads, dim] tensor."""
    s = t.stride()
    return (t.data_ptr(), s[0], s[1], s[2]) if len(s) == 4 else (t.data_ptr(), 0, s[0], s[1])


def _unit_last(t):
    """A gradient as autograd hands it over, made readable where it is not."""
    return t if t.stride(-1) == 1 else t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _like(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _call(name: str, args, dev) -> None:
    fn = getattr(abi.lib(), name)
    if torch.cuda.current_device() == dev.index:
        rc = fn(ctypes.byref(args), torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(ctypes.byref(args), torch.cuda.current_stream(dev).cuda_stream)
    if rc:
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
    _check_first(q, who, "q", (3, 4))
    _check_heads(k, who, "k", q)
    dim, dev = q.shape[-1], q.device
    if k.shape[-1] != dim:
        _refuse(who, "k", f"of q's head dimension {dim}", k)
    if q_weight is not None:
        _check_plain(q_weight, who, "q_weight", (dim,), torch.float32, dev, True)
    if k_weight is not None:
        _check_plain(k_weight, who, "k_weight", (dim,), torch.float32, dev, True)
    if table is not None:
        if not (isinstance(table, torch.Tensor) and table.dim() == 2 and table.shape[0] > 0 and table.shape[1] > 0
                and table.shape[1] % 8 == 0 and table.shape[1] <= dim):
            _refuse(who, "table", f"a float32 tensor [rows, R], R a multiple of 8 up to {dim}", table)
        _check_plain(table, who, "table", table.shape, torch.float32, dev, True)
        _check_plain(positions, who, "positions", q.shape[:-2], torch.int32, dev)
    elif positions is not None:
        raise ValueError(f"{who}: positions need a table")
    how = (positions, table, float(eps), bool(unit), bool(interleaved))
    if _wants_grad(q, k, q_weight, k_weight):
        return _QkNormRotate.apply(q, k, q_weight, k_weight, how)
    return _qk_forward(q, k, q_weight, k_weight, how)


def _qk_args(q, k, q_weight, k_weight, how, *out) -> abi.QkArgs:
    positions, table, eps, unit, interleaved = how
    shape = q.shape
    rows, rotated = (0, 0) if table is None else table.shape
    return abi.QkArgs(_DTYPES[q.dtype], shape[0] if len(shape) == 4 else 1, shape[-3], shape[-2], k.shape[-2],
                      shape[-1], rotated, unit, interleaved, eps, _heads(q), _heads(k), _ptr(q_weight),
                      _ptr(k_weight), _ptr(positions), _ptr(table), rows, *out)


def _qk_forward(q, k, q_weight, k_weight, how):
    q_out, k_out = _like(q), _like(k)
    _call("nesle_qk_norm_rotate", _qk_args(q, k, q_weight, k_weight, how, q_out.data_ptr(), k_out.data_ptr()), q.device)
    return q_out, k_out


class _QkNormRotate(torch.autograd.Function):
    # The gradient's arguments are made with the forward's: autograd runs the
    # backward on a thread of its own, where the same lines take several times
    # as long.
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, how):
        q_out, k_out = _like(q), _like(k)
        a = _qk_args(q, k, q_weight, k_weight, how, q_out.data_ptr(), k_out.data_ptr())
        _call("nesle_qk_norm_rotate", a, q.device)
        ctx.save_for_backward(q, k, q_weight, k_weight, how[0], how[1])
        ctx.args, ctx.floats = a, int(abi.lib().nesle_qk_scratch_floats(ctypes.byref(a)))
        return q_out, k_out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight = ctx.saved_tensors[:4]
        a = abi.QkArgs.from_buffer_copy(ctx.args)
        dq_out, dk_out = _unit_last(dq_out), _unit_last(dk_out)
        a.dq_out, a.dk_out = _heads(dq_out), _heads(dk_out)
        dq, dk = _like(q), _like(k)
        a.dq, a.dk = dq.data_ptr(), dk.data_ptr()
        dwq = dwk = None
        if q_weight is not None:
            dwq = _like(q_weight)
            a.dq_weight = dwq.data_ptr()
        if k_weight is not None:
            dwk = _like(k_weight)
            a.dk_weight = dwk.data_ptr()
        if ctx.floats:
            scratch = torch.empty(ctx.floats, dtype=torch.float32, device=q.device)
            a.scratch = scratch.data_ptr()
        _call("nesle_qk_norm_rotate_grad", a, q.device)
        return dq, dk, dwq, dwk, None


# ---- the gated delta rule -----------------------------------------------------------

def _check_delta(who: str, q, k, v, g, beta, state, resets, dims: tuple) -> None:
    _check_first(q, who, "q", dims)
    _check_heads(k, who, "k", q)
    _check_heads(v, who, "v", q)
    if k.shape != q.shape:
        _refuse(who, "k", f"of q's shape {tuple(q.shape)}", k)
    lead, dev = q.shape[:-2], q.device
    hk, dk = q.shape[-2:]
    hv, dv = v.shape[-2:]
    if hk == 0 or hv == 0 or hv % hk:
        _refuse(who, "v", f"of a multiple of {hk} heads", v)
    if dk % 8 or dv % 8 or not (8 <= dk <= abi.DELTA_MAX_DIM and 8 <= dv <= abi.DELTA_MAX_DIM):
        raise ValueError(f"{who}: head dimensions must be multiples of 8 up to {abi.DELTA_MAX_DIM}, got {dk} and {dv}")
    gates = (*lead, hv)
    _check_plain(g, who, "g", gates, torch.float32, dev)
    _check_plain(beta, who, "beta", gates, torch.float32, dev)
    if state is not None:
        _check_plain(state, who, "state", (lead[-1], hv, dk, dv), torch.float32, dev, True)
    if resets is not None:
        dtype = torch.uint8 if getattr(resets, "dtype", None) == torch.uint8 else torch.bool
        _check_plain(resets, who, "resets", lead, dtype, dev)


def _delta_args(q, k, v, g, beta, state, resets, scale, *out) -> abi.DeltaArgs:
    shape, values = q.shape, v.shape
    return abi.DeltaArgs(_DTYPES[q.dtype], shape[0] if len(shape) == 4 else 1, shape[-3], shape[-2], values[-2],
                         shape[-1], values[-1], scale, _heads(q), _heads(k), _heads(v), g.data_ptr(), beta.data_ptr(),
                         _ptr(resets), _ptr(state), *out)


def gated_delta_step(q, k, v, g, beta, state, *, resets=None, scale: float | None = None):
    """One token of the gated delta rule for every console (``gated_delta``):
    q, k [N, k_heads, k_dim], v [N, v_heads, v_dim], g, beta [N, v_heads],
    resets [N]; ``state`` [N, v_heads, k_dim, v_dim] is updated in place.
    Returns the output [N, v_heads, v_dim].  Not differentiable: acting."""
    who = "gated_delta_step"
    _check_delta(who, q, k, v, g, beta, state, resets, (3,))
    if state is None:
        _refuse(who, "state", "a tensor", state)
    if _wants_grad(q, k, v, g, beta, state):
        raise ValueError(f"{who} has no gradient: use gated_delta, or torch.no_grad()")
    out = _like(v)
    _call("nesle_delta_step", _delta_args(q, k, v, g, beta, state, resets, _scale(q, scale), out.data_ptr(),
                                          state.data_ptr()), q.device)
    return out


def _scale(q, scale) -> float:
    return q.shape[-1] ** -0.5 if scale is None else float(scale)


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
    _check_delta(who, q, k, v, g, beta, state, resets, (4,))
    scale = _scale(q, scale)
    if _wants_grad(q, k, v, g, beta, state):
        return _GatedDelta.apply(q, k, v, g, beta, state, resets, scale)
    return _delta_forward(q, k, v, g, beta, state, resets, scale, False)[:2]


def _delta_forward(q, k, v, g, beta, state, resets, scale, keep: bool):
    out = _like(v)
    after = torch.empty((v.shape[1], v.shape[2], q.shape[3], v.shape[3]), dtype=torch.float32, device=v.device)
    a = _delta_args(q, k, v, g, beta, state, resets, scale, out.data_ptr(), after.data_ptr())
    saved = scratch = None
    floats = abi.lib().nesle_delta_forward_scratch_floats(ctypes.byref(a))
    if floats:
        scratch = torch.empty(floats, dtype=torch.float32, device=v.device)
        a.scratch = scratch.data_ptr()
    if keep:
        floats = int(abi.lib().nesle_delta_saved_floats(ctypes.byref(a)))
        if floats:
            saved = torch.empty(floats, dtype=torch.float32, device=v.device)
            a.saved = saved.data_ptr()
    _call("nesle_delta_forward", a, q.device)
    return out, after, saved, a


class _GatedDelta(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, state, resets, scale):
        out, after, saved, a = _delta_forward(q, k, v, g, beta, state, resets, scale, True)
        ctx.save_for_backward(q, k, v, g, beta, state, resets, saved)
        ctx.args, ctx.floats = a, int(abi.lib().nesle_delta_scratch_floats(ctypes.byref(a)))
        return out, after

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dafter):
        q, k, v, g, beta, state = ctx.saved_tensors[:6]
        a = abi.DeltaArgs.from_buffer_copy(ctx.args)
        dout, dafter = _unit_last(dout), dafter.contiguous()
        a.dout, a.dstate_out = _heads(dout), dafter.data_ptr()
        dq, dk, dv, dg, dbeta = _like(q), _like(k), _like(v), _like(g), _like(beta)
        a.dq, a.dk, a.dv, a.dg, a.dbeta = dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dg.data_ptr(), dbeta.data_ptr()
        dstate = None
        if ctx.needs_input_grad[5]:
            dstate = _like(state)
            a.dstate = dstate.data_ptr()
        if ctx.floats:
            scratch = torch.empty(ctx.floats, dtype=torch.float32, device=q.device)
            a.scratch = scratch.data_ptr()
        _call("nesle_delta_backward", a, q.device)
        return dq, dk, dv, dg, dbeta, dstate, None, None
