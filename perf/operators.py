"""What the operators of a policy with memory are timed on.

Three entry points of ``nesle_amd.memory``: the per-head norm of queries and
keys with the position rotation (``qk_norm_rotate``), the gated delta rule
over a rollout (``gated_delta``) and one token of it for every console
(``gated_delta_step``).  Sizes follow the trainer's: rollouts of 128 steps,
up to 8,192 consoles, a hidden width of 256 as 4 heads of 64; the odd ones are
sizes nobody rounded.  Tensors are time-major, [T, N, heads, head dimension].
"""

from __future__ import annotations

import math

import torch

own = False

TABLE_ROWS = 4096       # positions of the rotation table: steps of an episode
EPS = 1e-6


def listed() -> list[dict]:
    return [
        # Acting, 16 consoles: one token's queries and keys, where the call's
        # latency is what counts.
        {"name": "rotate_act_16", "op": "rotate", "T": 1, "N": 16, "Hq": 4, "Hk": 4, "D": 64, "R": 64,
         "dtype": "float32", "unit": True, "weights": False, "interleaved": False, "train": False, "fused": True},
        # The trainer's minibatch of whole consoles in bfloat16, forward and
        # gradient, queries and keys cut out of one projection.
        {"name": "rotate_train_512", "op": "rotate", "T": 128, "N": 512, "Hq": 4, "Hk": 4, "D": 64, "R": 64,
         "dtype": "bfloat16", "unit": True, "weights": True, "interleaved": False, "train": True, "fused": True},
        # A size nobody rounded: shared key heads, part of the head rotated,
        # neighbouring pairs, float32.
        {"name": "rotate_ragged", "op": "rotate", "T": 77, "N": 301, "Hq": 6, "Hk": 2, "D": 40, "R": 16,
         "dtype": "float32", "unit": False, "weights": True, "interleaved": True, "train": True, "fused": False},
        # A whole rollout of 4,096 consoles, forward only (values and log
        # probabilities of the old policy).
        {"name": "rotate_rollout_4096", "op": "rotate", "T": 128, "N": 4096, "Hq": 4, "Hk": 4, "D": 64, "R": 64,
         "dtype": "bfloat16", "unit": True, "weights": True, "interleaved": False, "train": False, "fused": True},
        # Watching one console play: one token.
        {"name": "step_1", "op": "step", "N": 1, "Hk": 4, "Hv": 4, "DK": 64, "DV": 64, "dtype": "float32",
         "resets": 0.0, "fused": True},
        # An odd batch with two value heads for each key head and odd head
        # sizes, episodes ending.
        {"name": "step_1000_odd", "op": "step", "N": 1000, "Hk": 3, "Hv": 6, "DK": 48, "DV": 40, "dtype": "float32",
         "resets": 0.01, "fused": False},
        # The trainer's rollout step of 8,192 consoles.
        {"name": "step_8192", "op": "step", "N": 8192, "Hk": 4, "Hv": 4, "DK": 64, "DV": 64, "dtype": "bfloat16",
         "resets": 0.005, "fused": True},
        # Recorded evaluation episodes of 16 consoles, forward only: few heads,
        # a long axis.
        {"name": "delta_eval_1024x16", "op": "delta", "T": 1024, "N": 16, "Hk": 4, "Hv": 4, "DK": 64, "DV": 64,
         "dtype": "bfloat16", "resets": 0.002, "train": False, "fused": True},
        # One very long recording, an odd length, two consoles.
        {"name": "delta_long_8191x2", "op": "delta", "T": 8191, "N": 2, "Hk": 4, "Hv": 4, "DK": 64, "DV": 64,
         "dtype": "bfloat16", "resets": 0.0005, "train": False, "fused": True},
        # A training minibatch of 512 consoles, 128 steps, episodes ending
        # inside, forward and gradient in bfloat16.
        {"name": "delta_train_512", "op": "delta", "T": 128, "N": 512, "Hk": 4, "Hv": 4, "DK": 64, "DV": 64,
         "dtype": "bfloat16", "resets": 0.005, "train": True, "fused": True},
        # The trainer's own type, a small minibatch (8,192 samples).
        {"name": "delta_train_64_f32", "op": "delta", "T": 128, "N": 64, "Hk": 4, "Hv": 4, "DK": 64, "DV": 64,
         "dtype": "float32", "resets": 0.005, "train": True, "fused": True},
        # Ragged: odd length and batch, shared key heads, odd head sizes.
        {"name": "delta_ragged", "op": "delta", "T": 77, "N": 61, "Hk": 2, "Hv": 4, "DK": 48, "DV": 24,
         "dtype": "float32", "resets": 0.02, "train": True, "fused": False},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng) -> dict:
    op = rng.choice(["rotate", "step", "delta", "delta"])
    dtype = rng.choice(["float32", "bfloat16"])
    fused = rng.random() < 0.5
    if op == "rotate":
        Hk = rng.choice([1, 2, 4])
        D = rng.choice([16, 32, 40, 64, 64, 80, 128])
        T = _log_int(rng, 1, 256)
        train = rng.random() < 0.5
        room = (128 * 512 * 8 * 64 if train else 128 * 4096 * 8 * 64) // 4
        N = _log_int(rng, 1, max(1, min(4096, room // (T * Hk * 2 * D))))
        return {"op": op, "T": T, "N": N, "Hq": Hk * rng.choice([1, 1, 2]), "Hk": Hk, "D": D,
                "R": rng.choice([D, D, D // 16 * 8]), "dtype": dtype, "unit": rng.random() < 0.5,
                "weights": rng.random() < 0.5, "interleaved": rng.random() < 0.3, "train": train, "fused": fused}
    Hk = rng.choice([1, 2, 4])
    Hv = Hk * rng.choice([1, 1, 2])
    DK = rng.choice([16, 32, 48, 64, 64, 128])
    DV = rng.choice([DK, DK, DK, 24, 64])
    if op == "step":
        N = _log_int(rng, 1, max(1, min(8192, 8192 * 4 * 64 * 64 // (Hv * DK * DV))))
        return {"op": op, "N": N, "Hk": Hk, "Hv": Hv, "DK": DK, "DV": DV, "dtype": dtype,
                "resets": rng.choice([0.0, 0.005, 0.05]), "fused": fused}
    train = rng.random() < 0.6
    T = _log_int(rng, 1, 256 if train else 4096)
    room = 128 * 512 * 4 * 64 * 64 // (8 if train else 2)
    N = _log_int(rng, 1, max(1, min(2048, room // (T * Hv * DK * DV))))
    return {"op": op, "T": T, "N": N, "Hk": Hk, "Hv": Hv, "DK": DK, "DV": DV, "dtype": dtype,
            "resets": rng.choice([0.0, 0.002, 0.02]), "train": train, "fused": fused}


# ---- inputs ----------------------------------------------------------------------

def _cut(parts: list, lead: tuple, fused: bool, make) -> list:
    """Tensors of shape lead + (heads, dim): cut out of one projection's output
    (``fused``: strided views, as a model that projects once has them), or
    each its own."""
    sizes = [h * d for h, d in parts]
    if fused:
        return [t.unflatten(-1, p) for t, p in zip(make((*lead, sum(sizes))).split(sizes, -1), parts)]
    return [make((*lead, *p)) for p in parts]


def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = getattr(torch, case["dtype"])

    def normal(shape, dt=torch.float32):
        return torch.randn(shape, generator=gen, device=dev).to(dt)

    def uniform(shape):
        return torch.rand(shape, generator=gen, device=dev)

    st = {"case": case}
    if case["op"] == "rotate":
        lead, D, R = (case["T"], case["N"]), case["D"], case["R"]
        st["q"], st["k"] = _cut([(case["Hq"], D), (case["Hk"], D)], lead, case["fused"], lambda s: normal(s, dtype))
        st["wq"], st["wk"] = [1.0 + 0.1 * normal((D,)) if case["weights"] else None for _ in "qk"]
        # Step of the episode: consoles start anywhere and count on.
        first = torch.randint(0, TABLE_ROWS, (case["N"],), generator=gen, device=dev)
        steps = torch.arange(case["T"], device=dev)[:, None]
        st["positions"] = ((first + steps) % TABLE_ROWS).to(torch.int32)
        turn = torch.arange(TABLE_ROWS, device=dev, dtype=torch.float64)[:, None] * torch.pow(
            10000.0, -torch.arange(0, R, 2, device=dev, dtype=torch.float64) / max(R, 1))
        st["table"] = torch.cat((turn.cos(), turn.sin()), -1).float()
        if case["train"]:
            st["dq"], st["dk"] = normal(st["q"].shape, dtype), normal(st["k"].shape, dtype)
        return st
    Hk, Hv, DK, DV, N = case["Hk"], case["Hv"], case["DK"], case["DV"], case["N"]
    lead = (N,) if case["op"] == "step" else (case["T"], N)
    # Queries and keys of unit length with a part that a console keeps from
    # step to step, as neighbouring frames look alike.
    base = normal((N, 2 * Hk, DK))

    def project(shape):
        x = normal(shape)
        n = Hk * DK
        for j in range(2):
            h = x[..., j * n:(j + 1) * n].unflatten(-1, (Hk, DK))
            h += base[:, j * Hk:(j + 1) * Hk]
            h /= h.norm(dim=-1, keepdim=True)
        return x.to(dtype)

    flat = project((*lead, 2 * Hk * DK + Hv * DV))
    q, k, v = [t.unflatten(-1, p) for t, p in zip(flat.split([Hk * DK, Hk * DK, Hv * DV], -1),
                                                  [(Hk, DK), (Hk, DK), (Hv, DV)])]
    if not case["fused"]:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    st["q"], st["k"], st["v"] = q, k, v
    # Log decays of a learned gate (half lives of about 10 to 700 steps) and
    # write strengths.
    rate = torch.exp(torch.linspace(math.log(0.001), math.log(0.07), Hv, device=dev))
    st["g"] = -rate * 2.0 * torch.sigmoid(normal((*lead, Hv)))
    st["beta"] = torch.sigmoid(normal((*lead, Hv)))
    st["state"] = 0.3 * normal((N, Hv, DK, DV))
    st["resets"] = uniform(lead) < case["resets"]
    st["scale"] = DK ** -0.5
    if case.get("train"):
        st["dout"] = normal((*lead, Hv, DV), dtype)
        st["dstate"] = 0.1 * normal((N, Hv, DK, DV))
    return st


# ---- one pass ---------------------------------------------------------------------

def run(st: dict):
    op = st["case"]["op"]
    if op == "rotate":
        return _run_rotate(st, _own_rotate if own else _plain_rotate)
    if op == "step":
        return _own_step(st) if own else _plain_step(st)
    return _run_delta(st, _own_delta if own else _plain_delta)


def _run_rotate(st, forward):
    if not st["case"]["train"]:
        with torch.no_grad():
            q, k = forward(st, st["q"], st["k"], st["wq"], st["wk"])
        return {"q": q, "k": k}
    leaves = {n: st[n].detach().requires_grad_() for n in ("q", "k", "wq", "wk") if st[n] is not None}
    q, k = forward(st, leaves["q"], leaves["k"], leaves.get("wq"), leaves.get("wk"))
    grads = torch.autograd.grad((q, k), list(leaves.values()), (st["dq"], st["dk"]))
    return {"q": q.detach(), "k": k.detach(), **{"d" + n: g for n, g in zip(leaves, grads)}}


def _run_delta(st, forward):
    names = ("q", "k", "v", "g", "beta", "state")
    if not st["case"]["train"]:
        with torch.no_grad():
            out, state = forward(st, *(st[n] for n in names))
        return {"out": out, "state": state}
    leaves = [st[n].detach().requires_grad_() for n in names]
    out, state = forward(st, *leaves)
    grads = torch.autograd.grad((out, state), leaves, (st["dout"], st["dstate"]))
    return {"out": out.detach(), "state": state.detach(), **{"d_" + n: g for n, g in zip(names, grads)}}


def _own_rotate(st, q, k, wq, wk):
    from nesle_amd import memory

    return memory.qk_norm_rotate(q, k, wq, wk, positions=st["positions"], table=st["table"], eps=EPS,
                                 unit=st["case"]["unit"], interleaved=st["case"]["interleaved"])


def _own_delta(st, q, k, v, g, beta, state):
    from nesle_amd import memory

    return memory.gated_delta(q, k, v, g, beta, state=state, resets=st["resets"], scale=st["scale"])


def _own_step(st):
    from nesle_amd import memory

    out = memory.gated_delta_step(st["q"], st["k"], st["v"], st["g"], st["beta"], st["state"], resets=st["resets"],
                                  scale=st["scale"])
    return {"out": out, "state": st["state"]}


def _plain_rotate(st, q, k, wq, wk):
    case, R = st["case"], st["case"]["R"]
    turn = st["table"][st["positions"].long()].unsqueeze(-2)     # [T, N, 1, R]
    c, s = turn[..., :R // 2], turn[..., R // 2:]

    def one(x, w):
        x32 = x.float()
        square = (x32 * x32).sum(-1, keepdim=True)
        y = x32 / torch.sqrt((square if case["unit"] else square / case["D"]) + EPS)
        if w is not None:
            y = y * w
        if case["interleaved"]:
            a, b = y[..., 0:R:2], y[..., 1:R:2]
            turned = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
        else:
            a, b = y[..., :R // 2], y[..., R // 2:R]
            turned = torch.cat((a * c - b * s, a * s + b * c), -1)
        return torch.cat((turned, y[..., R:]), -1).to(x.dtype)

    return one(q, wq), one(k, wk)


def _token(q, k, v, g, beta, state, reset, scale):
    """One token of the rule, everything float32: (output, new state)."""
    decayed = state * torch.exp(g)[..., None, None]
    state = torch.where(reset[:, None, None, None], 0.0, decayed)
    held = torch.matmul(k.unsqueeze(-2), state).squeeze(-2)
    u = beta.unsqueeze(-1) * (v - held)
    state = state + k.unsqueeze(-1) * u.unsqueeze(-2)
    return scale * torch.matmul(q.unsqueeze(-2), state).squeeze(-2), state


def _plain_step(st):
    r = st["case"]["Hv"] // st["case"]["Hk"]
    q, k = [st[n].float().repeat_interleave(r, -2) for n in "qk"]
    out, state = _token(q, k, st["v"].float(), st["g"], st["beta"], st["state"], st["resets"], st["scale"])
    st["state"].copy_(state)
    return {"out": out.to(st["v"].dtype), "state": st["state"]}


def _plain_delta(st, q, k, v, g, beta, state):
    r = st["case"]["Hv"] // st["case"]["Hk"]
    q32, k32, v32 = q.float().repeat_interleave(r, -2), k.float().repeat_interleave(r, -2), v.float()
    outs = []
    # The rule is a recurrence: its plain form goes token by token.
    for t in range(st["case"]["T"]):
        out, state = _token(q32[t], k32[t], v32[t], g[t], beta[t], state, st["resets"][t], st["scale"])
        outs.append(out)
    return torch.stack(outs).to(v.dtype), state


# ---- sizes ------------------------------------------------------------------------

def work(case: dict) -> dict:
    item = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "rotate":
        rows = case["T"] * case["N"]
        values = rows * (case["Hq"] + case["Hk"]) * case["D"]
        table = min(rows, TABLE_ROWS) * case["R"] * 4
        # forward: x in, y out; gradient: the outputs' gradients in, dx out
        moved = values * item * (4 if case["train"] else 2) + rows * 4 + table
        return {"bytes": moved, "flops": values * (22 if case["train"] else 8)}
    tokens = case["N"] * case.get("T", 1)
    wide = 2 * case["Hk"] * case["DK"] + 2 * case["Hv"] * case["DV"]      # q, k, v, out
    state = case["N"] * case["Hv"] * case["DK"] * case["DV"] * 4
    moved = tokens * (wide * item + 8 * case["Hv"] + 1) + 2 * state
    flops = 7 * tokens * case["Hv"] * case["DK"] * case["DV"]
    if case.get("train"):
        # out's gradient in; dq, dk, dv, dg, dbeta and both states' gradients out
        moved += tokens * (wide * item + 8 * case["Hv"]) + 2 * state
        flops *= 3
    return {"bytes": moved, "flops": flops}


# ---- the definition in 64 bits ------------------------------------------------------

def exact(case: dict, seed: int):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "rotate":
            return _exact_rotate(st)
        return _exact_delta(st)


def _exact_rotate(st):
    """The rotation as a matrix for each pair, the norm by its definition, the
    gradient from the formulas."""
    case, R, D = st["case"], st["case"]["R"], st["case"]["D"]
    count = D if not case["unit"] else 1
    pos = st["positions"].long().reshape(-1)
    angle_c, angle_s = st["table"].double()[pos][:, None].chunk(2, -1)
    first = torch.arange(0, R, 2, device=pos.device) if case["interleaved"] else torch.arange(R // 2, device=pos.device)
    second = first + (1 if case["interleaved"] else R // 2)
    result = {}
    for n in "qk":
        x = st[n].double().reshape(pos.numel(), -1, D)
        w = torch.ones(D, dtype=torch.float64, device=pos.device) if st["w" + n] is None else st["w" + n].double()
        inv = torch.rsqrt(x.pow(2).sum(-1, keepdim=True) / count + EPS)
        y = x * inv * w
        out = y.clone()
        out[..., first] = y[..., first] * angle_c - y[..., second] * angle_s
        out[..., second] = y[..., second] * angle_c + y[..., first] * angle_s
        result[n] = out.reshape(st[n].shape)
        if case["train"]:
            d = st["d" + n].double().reshape(x.shape)
            dy = d.clone()
            dy[..., first] = d[..., first] * angle_c + d[..., second] * angle_s
            dy[..., second] = d[..., second] * angle_c - d[..., first] * angle_s
            dn = dy * w
            result["d" + n] = (inv * dn - x * inv.pow(3) * (x * dn).sum(-1, keepdim=True) / count).reshape(st[n].shape)
            if st["w" + n] is not None:
                result["dw" + n] = (x * inv * dy).sum((0, 1))
    order = ("q", "k") if not case["train"] else ("q", "k", "dq", "dk", "dwq", "dwk")
    return {n: result[n] for n in order if n in result}


def _exact_delta(st):
    """Forward recurrence with every state kept, then the adjoint recurrence."""
    case = st["case"]
    step = case["op"] == "step"
    T = 1 if step else case["T"]
    r = case["Hv"] // case["Hk"]

    def steps(n):
        return (st[n][None] if step else st[n]).double()

    q, k = steps("q").repeat_interleave(r, -2), steps("k").repeat_interleave(r, -2)
    v, g, beta, resets = steps("v"), steps("g"), steps("beta"), (st["resets"][None] if step else st["resets"])
    a = torch.exp(g) * (~resets)[..., None]
    S = st["state"].double()
    keep, us, outs = [], [], []
    for t in range(T):
        D = S * a[t, ..., None, None]
        u = beta[t, ..., None] * (v[t] - torch.einsum("nhk,nhkv->nhv", k[t], D))
        if case.get("train"):
            keep.append(S)
        us.append(u)
        S = D + torch.einsum("nhk,nhv->nhkv", k[t], u)
        outs.append(st["scale"] * torch.einsum("nhk,nhkv->nhv", q[t], S))
    out = torch.stack(outs)
    if step:
        return {"out": out[0], "state": S}
    if not case["train"]:
        return {"out": out, "state": S}
    dq, dk, dv, dg, db = (torch.zeros_like(x) for x in (q, k, v, g, beta))
    dS, after = st["dstate"].double(), S
    for t in range(T - 1, -1, -1):
        do = st["scale"] * st["dout"][t].double()
        dq[t] = torch.einsum("nhkv,nhv->nhk", after, do)
        dS = dS + torch.einsum("nhk,nhv->nhkv", q[t], do)
        du = torch.einsum("nhk,nhkv->nhv", k[t], dS)
        D = keep[t] * a[t, ..., None, None]
        err = v[t] - torch.einsum("nhk,nhkv->nhv", k[t], D)
        de = beta[t, ..., None] * du
        dv[t], db[t] = de, (du * err).sum(-1)
        dk[t] = torch.einsum("nhkv,nhv->nhk", dS, us[t]) - torch.einsum("nhkv,nhv->nhk", D, de)
        dD = dS - torch.einsum("nhk,nhv->nhkv", k[t], de)
        dg[t] = (dD * D).sum((-1, -2))
        dS = dD * a[t, ..., None, None]
        after = keep[t]
    dq, dk = [x.unflatten(-2, (case["Hk"], r)).sum(-2) for x in (dq, dk)]
    return {"out": out, "state": S, "d_q": dq, "d_k": dk, "d_v": dv, "d_g": dg, "d_beta": db, "d_state": dS}
