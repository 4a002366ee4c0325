"""Operators of a policy with memory, as HIP kernels (include/nesle_memory.h).

A console's RAM or frame shows one instant.  These operators give a policy a
memory of the episode that acts one token at a time for every console and
trains on whole rollouts with gradients:

* ``qk_norm_rotate``    norms of queries and keys for each head with the
  position rotation, in one pass;
* ``gated_delta``       the gated delta rule over a rollout [T, N], memory
  dropped where an episode ends;
* ``gated_delta_step``  one token of it for every console, states in place;
* ``decay_attention``   linear attention with a decay for each head over a
  rollout, the plainer memory: nothing is taken out but by the decay;
* ``decay_attention_step``  one token of it for every console, states in place;
* ``layer_norm``        the layer norm of features or of a memory's heads;
* ``sample_actions``    actions drawn from logits by given random numbers, with
  temperature, top-k, top-p and min-p, and their log probabilities;
* ``rotation_table``    cosines and sines for the rotation.

Tensors are time-major, [T, N, heads, dim] (a step's: [N, heads, dim]), float32
or bfloat16, on the GPU.  Queries, keys and values may be slices of one
projection's output: only the elements of a head have to lie next to each
other.  Arguments that do not fit raise ValueError.  Work is enqueued on the
current stream; nothing synchronises, so calls may be captured in a graph.
First derivatives in reverse mode only: forward-mode derivatives are refused,
and so is a call under a tracer (``torch.jit.trace``, ``make_fx``), whose record
would hold the outputs without the launch.
"""

from __future__ import annotations

import torch

from nesle_amd import abi

abi.lib()      # before the binding below, which is linked against it
from nesle_amd import _memory_native as _native  # noqa: E402  (built by `python -m nesle_amd.build`)


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


def _called(fn, *args):
    """A binding's answer; an argument of a type it does not take is refused as
    every other is."""
    try:
        return fn(*args)
    except TypeError as exc:
        raise ValueError(f"{fn.__name__}: an argument has a type that it does not take\n{exc}") from None


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
    return _called(_native.qk_norm_rotate, q, k, q_weight, k_weight, positions, table, eps, unit, interleaved)


# ---- the gated delta rule -----------------------------------------------------------

def gated_delta_step(q, k, v, g, beta, state, *, resets=None, scale: float | None = None):
    """One token of the gated delta rule for every console (``gated_delta``):
    q, k [N, k_heads, k_dim], v [N, v_heads, v_dim], g, beta [N, v_heads],
    resets [N]; ``state`` [N, v_heads, k_dim, v_dim] is updated in place.
    Returns the output [N, v_heads, v_dim].  Not differentiable: acting."""
    return _called(_native.gated_delta_step, q, k, v, g, beta, state, resets, scale)


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
    inputs that are not finite is unspecified, and so is a chunk of 32 tokens of a
    head in which finite inputs overflow float32.  Products keep float32 precision
    for either type: bfloat16 results are rounded once."""
    return _called(_native.gated_delta, q, k, v, g, beta, state, resets, scale)


# ---- linear attention with a decay for each head --------------------------------------

def decay_attention_step(q, k, v, g, state, *, resets=None, scale: float | None = None):
    """One token of ``decay_attention`` for every console: q, k [N, k_heads,
    k_dim], v [N, v_heads, v_dim], g [v_heads], resets [N]; ``state`` [N, v_heads,
    k_dim, v_dim] is updated in place.  Returns the output [N, v_heads, v_dim].
    Not differentiable: acting."""
    return _called(_native.decay_attention_step, q, k, v, g, state, resets, scale)


def decay_attention(q, k, v, g, *, state=None, resets=None, scale: float | None = None):
    """Linear attention with a decay for each head over a rollout: (output, state
    after it).

    Each head of each console keeps a float32 state S [k_dim, v_dim].  A token
    first lets it decay, S <- exp(g) S, or drops it where ``resets`` is set (an
    episode's first token), then writes, S <- S + k v^T, and reads
    out = scale S^T q: all tokens of the episode up to its own, each weighed by
    scale exp(g)^distance (q . k).  Nothing is normalised (``layer_norm``).

    q, k [T, N, k_heads, k_dim], v [T, N, v_heads, v_dim], g float32 [v_heads]
    (the logarithm of a head's decay, g <= 0; -inf: a token sees itself alone),
    resets bool or uint8 [T, N], state float32 [N, v_heads, k_dim, v_dim] (None:
    zeros).  v_heads is a multiple of k_heads: value head h goes with key head
    h // (v_heads // k_heads).  Head dimensions are multiples of 8 up to 128; T and
    N may be 0; scale defaults to k_dim ** -0.5.  A padded token at the end of a
    rollout still lets the state decay; its key, or value, of zeros writes nothing.
    The output has q's type; the new state is float32, a tensor of its own.
    Differentiable in q, k, v, g and state.  No value of a dropped state, and
    nothing that is not finite in a later token, reaches an output it does not
    belong to; the gradient of inputs that are not finite is unspecified, and so is
    a chunk of 64 tokens of a head in which finite inputs overflow float32.  A g above
    0 is taken as it is, and the state grows; from where exp(n g) overflows float32, for
    n tokens of a chunk, or of the few chunks that a long walk is cut into, without an
    episode's end among them, results are unspecified until one ends.  Products
    keep float32 precision for either type: bfloat16 results are rounded once."""
    return _called(_native.decay_attention, q, k, v, g, state, resets, scale)


# ---- layer norm -------------------------------------------------------------------------

def layer_norm(x, weight=None, bias=None, *, eps: float = 1e-5):
    """(x - mean) / sqrt(mean((x - mean)^2) + eps) * weight + bias over the last
    dimension.

    x float32 or bfloat16, one to four dimensions, the last of 1 to 16,384 elements
    next to each other (leading ones may be strided: a slice of one projection's
    output); weight and bias float32 [dim] or None.  Statistics and the gradients of
    weight and bias are float32; the result has x's type, rounded once.
    Differentiable in x, weight and bias."""
    return _called(_native.layer_norm, x, weight, bias, eps)


# ---- sampling ---------------------------------------------------------------------------

def sample_actions(logits, uniform, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Actions drawn from ``logits`` [N, actions] or [T, N, actions] (float32 or
    bfloat16, at most 1,024 actions) by one random number a row, ``uniform``
    (float32 [N] or [T, N], in [0, 1)): (actions int64, log probabilities float32).

    With w = exp(logits / temperature) relative to the largest, and actions in order
    of falling logits (equal ones by rising index): the ``top_k`` first stay (0:
    all); of these the ones before which less than ``top_p`` of their sum lies; of
    these the ones with w >= ``min_p``.  The action is the first by index at which
    the running sum of what stays exceeds ``uniform`` times all of it, its log
    probability that of w among what stays.  Temperature 0 takes the largest logit,
    the first of equal ones, with log probability 0.

    The four settings are numbers, or tensors with each row's own (float32, top_k
    int32, of uniform's shape).  Sums are float64.  Logits of -inf are never taken.
    A row without an answer (NaN or +inf among its logits, nothing above -inf, NaN
    as its number, a setting of its own out of range) gets action -1 and NaN.  Not
    differentiable: acting."""
    return _called(_native.sample_actions, logits, uniform, temperature, top_k, top_p, min_p)
