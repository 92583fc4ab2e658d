"""Between two blocks of a model that normalises a block's output: the norm behind the block, its gate and scale, the
residual stream, and the norm and modulation in front of the next block, in one pass.

The prologues of a layer (_lib.PRO_RMS_NORM, _lib.PRO_NORM_MODULATE) normalise what goes INTO it and its epilogue gates what comes
out; a norm between the projection and the gate, x + tanh(g) * norm(block(...)), needs the whole row of the block's output and is a
pass of its own, which then may as well leave the next block's input.
"""
from __future__ import annotations

import torch
from torch import Tensor

from . import _lib, compile_ops, int8_fused_kernel
from .adapters import _quantised_here
from .int8_quant import SMALL_BATCH_ROWS, _layers_in_place, _project_quantised, _scale_on, forward_fanout


def block_norm(y: Tensor, residual: Tensor, *, post_norm: str | None = None, post_weight: Tensor | None = None, post_bias: Tensor | None = None,
               post_eps: float = 1e-6, gate: Tensor | None = None, gate_tanh: bool = False, residual_scale: float = 1.0, branch_scale: float = 1.0,
               pre_norm: str | None = None, pre_weight: Tensor | None = None, pre_bias: Tensor | None = None, pre_eps: float = 1e-6,
               mod_scale: Tensor | None = None, mod_shift: Tensor | None = None):
    """(x, h) behind a block that computed y on the residual stream `residual`:

        x = residual_scale * residual + branch_scale * gate * norm_post(y)      (tanh(gate) with gate_tanh; without a gate 1)
        h = norm_pre(x) * (1 + mod_scale) + mod_shift                           (each part where it is given; None without any)

    Norms: "rms", "layer" or None over the last dimension, with weight and bias [K] of y's dtype or float32.
    y, residual: tensors alike, bfloat16, float16 or float32.  gate, mod_scale, mod_shift: of y's dtype, [K] or y's shape with ones from
    some leading dimension on ([batch, 1, K] for one vector to an image).  Everything is computed in binary32, h from x before its
    rounding; x and h are rounded once.  No gradients: under grad mode an input that asks for one is refused, one with a
    tangent always."""
    if type(y) is Tensor and y.is_cuda and not torch.compiler.is_compiling():
        out = _lib.host().block_norm(y, residual, post_norm, post_weight, post_bias, post_eps, gate, gate_tanh, residual_scale, branch_scale, pre_norm,
                                     pre_weight, pre_bias, pre_eps, mod_scale, mod_shift, None, None, None, None, False, 0, None)
        if out is not None:
            return out
    operands = dict(post_norm=post_norm, post_weight=post_weight, post_bias=post_bias, post_eps=post_eps, gate=gate, gate_tanh=gate_tanh,
                    residual_scale=residual_scale, branch_scale=branch_scale, pre_norm=pre_norm, pre_weight=pre_weight, pre_bias=pre_bias,
                    pre_eps=pre_eps, mod_scale=mod_scale, mod_shift=mod_shift)
    _refuse_gradients(y, residual, operands)
    return _block_norm(y, residual, operands)


def _block_norm(y, residual, operands):
    if not torch.compiler.is_compiling():
        return _lib.block_norm(y, residual, **operands)
    x, h = torch.ops.i8f.block_norm(y, residual, **operands)
    return x, None if all(operands.get(name) is None for name in ("pre_norm", "mod_scale", "mod_shift")) else h


def _forward_native(layers, y, residual, post_norm=None, post_weight=None, post_bias=None, post_eps=1e-6, gate=None, gate_tanh=False, residual_scale=1.0,
                    branch_scale=1.0, pre_norm=None, pre_weight=None, pre_bias=None, pre_eps=1e-6, mod_scale=None, mod_shift=None):
    """forward_block_norm() without the interpreter's part of it, for layers of one rotation flag on the W8A8 path with everything in place;
    None for everything else."""
    parts = _layers_in_place(layers)
    if parts is None:
        return None
    work = _lib._splitk_workspace if y.shape[-1] >= _lib.SPLITK_MIN_K else None
    return _lib.host().block_norm(y, residual, post_norm, post_weight, post_bias, post_eps, gate, gate_tanh, residual_scale, branch_scale, pre_norm, pre_weight,
                                  pre_bias, pre_eps, mod_scale, mod_shift, *parts, int8_fused_kernel.DEFAULT_EPILOGUE, work)


def forward_block_norm(layers, y: Tensor, residual: Tensor, **operands):
    """(x, [layer(h) for layer in layers]) of block_norm(y, residual, **operands), which has to have an h: the next block's first projections
    along with the step in front of them.  Where the layers are on the W8A8 path (as for forward_fanout) h is quantised where it is computed
    and never stored; the results are those of block_norm and the layers' own forward bit for bit."""
    layers = list(layers)
    if type(y) is Tensor and y.is_cuda and 0 < len(layers) <= 8 and y.numel() // max(1, y.shape[-1]) > SMALL_BATCH_ROWS and not torch.compiler.is_compiling():
        out = _forward_native(layers, y, residual, **operands)
        if out is not None:
            return out
    _refuse_gradients(y, residual, operands)
    if operands.get("pre_norm") is None and operands.get("mod_scale") is None and operands.get("mod_shift") is None:
        raise ValueError("the layers need an h: give pre_norm, mod_scale or mod_shift")
    rotate = bool(getattr(layers[0], "_use_quarot", False)) if layers else False
    if (layers and y.is_cuda and y.dim() >= 2 and y.numel() // max(1, y.shape[-1]) > SMALL_BATCH_ROWS
            and y.dtype in (torch.float16, torch.bfloat16)
            and all(_quantised_here(lin, y) and bool(getattr(lin, "_use_quarot", False)) == rotate and lin.weight.shape[1] == y.shape[-1] for lin in layers)):
        if torch.compiler.is_compiling():
            x, q, s = torch.ops.i8f.block_norm_quantised(y, residual, rotate, **operands)
            scales = [compile_ops.split_scale(_scale_on(lin, y.device)) for lin in layers]
            outs = [torch.ops.i8f.linear_w8a8(q, s, lin.weight, t, v, lin.bias, y.dtype, int8_fused_kernel.DEFAULT_EPILOGUE) for lin, (t, v) in zip(layers, scales)]
            return x, [o.reshape(*y.shape[:-1], o.shape[-1]) for o in outs]
        x, q, s = _lib.block_norm(y, residual, quantise=True, rotate=rotate, **operands)
        return x, [o.reshape(*y.shape[:-1], o.shape[-1]) for o in _project_quantised(layers, q, s, y.dtype)]
    x, h = _block_norm(y, residual, operands)
    return x, forward_fanout(layers, h)


def _refuse_gradients(y, residual, operands):
    _lib.refuse_gradients(y=y, residual=residual, **{k: v for k, v in operands.items() if isinstance(v, Tensor)})
