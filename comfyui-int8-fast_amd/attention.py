"""Between the projections of an attention block: the norms of queries and keys for each head, the rotation by positions of several
axes, and the attention over an encoder's states.

The layers around them are quantised (Int8TensorwiseOps.Linear); what lies between is in 16 bits, since the scores and the rotation do not
bear the steps of int8 rows.  forward_cross_attention is the whole path, projections included.
"""
from __future__ import annotations

import math
import operator

import torch
from torch import Tensor

from . import _lib
from ._comfy_compat import compute_device
from .int8_quant import forward_fanout


class RotaryAxes:
    """The rotation of heads by positions of one to four axes (time, height and width of a video, say), on one device.

    dims:        how many elements of a head each axis turns, even numbers; elements behind their sum are left as they are.
    theta:       base of the frequencies, one number or one for each axis: pair j of an axis with d elements turns by theta^(-2j/d) radians to a unit.
    interleaved: pairs of neighbours, (2j, 2j + 1); False: (j, j + sum(dims) / 2), as models that rotate halves have them.
    device:      where the heads are (default: ComfyUI's compute device).

    Laid out once: assigning to its attributes is refused."""

    def __init__(self, dims, theta=10000.0, *, interleaved: bool = True, device=None):
        dims = tuple(operator.index(n) for n in dims)
        if not 1 <= len(dims) <= _lib.MAX_AXES or any(n < 2 or n % 2 for n in dims):
            raise ValueError(f"dims must be one to {_lib.MAX_AXES} even numbers from 2 on, got {list(dims)}")
        thetas = tuple(float(t) for t in theta) if isinstance(theta, (tuple, list)) else (float(theta),) * len(dims)
        if len(thetas) != len(dims) or any(not 0.0 < t < math.inf for t in thetas):
            raise ValueError(f"theta must be positive, one number or one for each of {len(dims)} axes, got {theta}")
        rates = [t ** (-2 * j / n) / (2 * math.pi) for t, n in zip(thetas, dims) for j in range(n // 2)]   # turns to a unit
        self.dims, self.theta, self.interleaved = dims, thetas, bool(interleaved)
        self.rates = torch.tensor(rates, dtype=torch.float64, device=compute_device() if device is None else device)
        self._laid_out = True

    def __setattr__(self, name, value):
        if "_laid_out" in self.__dict__:
            raise AttributeError(f"a rotation is laid out once: make another one instead of assigning {name}")
        super().__setattr__(name, value)


def norm_heads(xs, weights=None, *, eps: float = 1e-6, rotary: RotaryAxes | None = None, positions: Tensor | None = None):
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension of every head, turned by its token's positions where `rotary` is given.

    xs:        heads [batch, tokens, heads, width] or [tokens, heads, width], or a list of tensors of the same tokens (queries and keys, of
               unlike numbers of heads; then the result is a list).  bfloat16, float16 or float32, width up to 256.  Views of a fused
               projection are taken as they are.
    weights:   [width] of their type or float32, one for each of xs (None for none), or None for none at all.
    positions: [tokens, axes], or [batch, tokens, axes] (a batch of 1 for all), int32, int64, float32 or float64, on xs' device.

    Everything is computed in binary32 (squares too, whose sum must stay within it), the angles in binary64, and rounded once.  The results are contiguous.  No gradients: under grad
    mode an input that asks for one is refused, one with a tangent always."""
    single = isinstance(xs, Tensor)
    xs = (xs,) if single else tuple(xs)
    weights = (None,) * len(xs) if weights is None else (weights,) if single and isinstance(weights, Tensor) else tuple(weights)
    if len(weights) != len(xs):
        raise ValueError(f"{len(xs)} tensors of heads and {len(weights)} weights")
    outs = _norm_rotate(xs, weights, True, eps, rotary, positions)
    return outs[0] if single else outs


def rotate_heads(xs, rotary: RotaryAxes, positions: Tensor):
    """Heads turned by their tokens' positions, without a norm: norm_heads describes xs, positions and the result."""
    single = isinstance(xs, Tensor)
    xs = (xs,) if single else tuple(xs)
    if rotary is None:
        raise ValueError("a rotation needs its axes")
    outs = _norm_rotate(xs, (None,) * len(xs), False, 0.0, rotary, positions)
    return outs[0] if single else outs


def _norm_rotate(xs, weights, norm, eps, rotary, positions):
    if (rotary is None) != (positions is None):
        raise ValueError("rotary and positions go together")
    if rotary is not None and not isinstance(rotary, RotaryAxes):
        raise TypeError(f"rotary must be a RotaryAxes, not {type(rotary).__name__}")
    for x in xs:
        if not isinstance(x, Tensor):
            raise TypeError(f"heads must be tensors, not {type(x).__name__}")
    rates, dims, apart = (None, (), False) if rotary is None else (rotary.rates, rotary.dims, not rotary.interleaved)
    compiling = torch.compiler.is_compiling()
    if xs and xs[0].is_cuda and not compiling:
        outs = _lib.host().norm_rotate(xs, weights, norm, eps, rates, dims, apart, positions)
        if outs is not None:
            return outs
    _lib.refuse_gradients(**{f"xs[{i}]": x for i, x in enumerate(xs)}, **{f"weights[{i}]": w for i, w in enumerate(weights)}, positions=positions)
    if compiling:
        return torch.ops.i8f.norm_rotate_heads(list(xs), list(weights), norm, eps, rates, list(dims), apart, positions)
    return _lib.norm_rotate(xs, weights, norm, eps, rates, dims, apart, positions)


def cross_attention(q: Tensor, k: Tensor, v: Tensor, *, key_lengths: Tensor | None = None, key_mask: Tensor | None = None, scale: float | None = None) -> Tensor:
    """softmax(scale * q k^T + mask) v for every head: queries over the keys and values of as many states as there are.

    q:    [batch, queries, heads, width], k, v: [batch, keys, kv heads, width], bfloat16 or float16, width up to 256; heads a multiple of
          kv heads, consecutive ones sharing one.  Views (of a fused projection, of a cache, expanded) are taken as they are.
    key_lengths: int32 or int64 [batch]: only the first so many states count (all of them for a larger number, none for a negative one).
    key_mask:    [batch, keys], bool (True: the state counts) or bfloat16, float16, float32 added to the scores; a state whose addend is -inf
                 or the lowest value of its type does not count.  With lengths both hold.
    scale:       positive, at most 2^126; width ** -0.5 by default.

    -> [batch, queries, heads, width], contiguous.  A query over which no state counts, or a finite one whose scores all are -inf, gets zeros, and what
    the states that do not count hold (NaN, infinities) reaches nothing.  Scores (with their addends), maximum and sums are in binary32, and finite
    scores of any size are the formula's; one that passes binary32 upwards gives NaN.  The weights are rounded to q's type for the second product, the
    result is rounded once; bfloat16 values up to 2^127 / keys cannot overflow its sums.  A row's bits do not depend on the rows beside it.  key_lengths
    and key_mask are read on the device: a captured graph follows what is written into them.  No gradients: under grad mode an input that asks for
    one is refused, one with a tangent always."""
    compiling = torch.compiler.is_compiling()
    if type(q) is Tensor and q.is_cuda and not compiling:
        out = _lib.host().attention(q, k, v, key_lengths, key_mask, scale)
        if out is not None:
            return out
    _lib.refuse_gradients(q=q, k=k, v=v, key_mask=key_mask)
    if compiling:
        return torch.ops.i8f.cross_attention(q, k, v, key_lengths, key_mask, scale)
    return _lib.attention(q, k, v, key_lengths, key_mask, scale)


def forward_cross_attention(x: Tensor, context: Tensor | None, to_q, to_k, to_v, to_out=None, *, heads: int, kv_heads: int | None = None,
                            q_weight: Tensor | None = None, k_weight: Tensor | None = None, eps: float = 1e-6, rotary: RotaryAxes | None = None,
                            positions: Tensor | None = None, context_positions: Tensor | None = None, key_lengths: Tensor | None = None,
                            key_mask: Tensor | None = None, scale: float | None = None, gate: Tensor | None = None, residual: Tensor | None = None) -> Tensor:
    """An attention block from its quantised projections to the residual stream: to_out(attention(to_q(x), to_k(context), to_v(context))).

    x [batch, queries, features], context [batch, keys, features] or None for x itself, in the types of the attention (bfloat16 or float16: float32 is
    refused behind the projections); layers that read one tensor quantise it once
    (int8_quant.forward_fanout).  q_weight, k_weight [head width]: the norms of the heads (both or neither); rotary with `positions` of x's tokens
    and `context_positions` of the context's (None: its keys are not turned; without a context those of x).  gate and residual as
    Linear.forward takes them, applied behind to_out; without to_out the heads side by side are returned.  No gradients: under grad mode an
    input that asks for one is refused, and layers of queries, keys and values with trainable parameters; an input with a tangent always."""
    _lib.refuse_gradients(x=x, context=context, gate=gate, residual=residual)
    kv_heads = heads if kv_heads is None else kv_heads
    if (q_weight is None) != (k_weight is None):
        raise ValueError("the norms of queries and keys go together")
    if rotary is None and (positions is not None or context_positions is not None) or rotary is not None and positions is None:
        raise ValueError("rotary and positions go together")
    if context is None and context_positions is not None:
        raise ValueError("context_positions without a context")
    if to_out is None and (gate is not None or residual is not None):
        raise ValueError("gate and residual go behind to_out")
    if context is None:
        q, k, v = forward_fanout([to_q, to_k, to_v], x)
        context_positions = positions
    else:
        q = to_q(x)
        k, v = forward_fanout([to_k, to_v], context)
    for name, t, n in (("queries", q, heads), ("keys", k, kv_heads), ("values", v, kv_heads)):
        if n < 1 or t.shape[-1] % n or t.dim() != 3:
            raise ValueError(f"the {name} must be [batch, tokens, features] of {n} heads, got {list(t.shape)}")
    q, k, v = q.unflatten(-1, (heads, -1)), k.unflatten(-1, (kv_heads, -1)), v.unflatten(-1, (kv_heads, -1))
    norm = q_weight is not None
    if context is None and (norm or rotary is not None):
        q, k = _norm_rotate((q, k), (q_weight, k_weight), norm, eps, rotary, positions)
    else:
        if norm or positions is not None:
            q, = _norm_rotate((q,), (q_weight,), norm, eps, rotary, positions)
        if norm or context_positions is not None:
            k, = _norm_rotate((k,), (k_weight,), norm, eps, rotary if context_positions is not None else None, context_positions)
    out = cross_attention(q, k, v, key_lengths=key_lengths, key_mask=key_mask, scale=scale).flatten(-2)
    return out if to_out is None else to_out(out) if gate is None and residual is None else to_out(out, gate=gate, residual=residual)
