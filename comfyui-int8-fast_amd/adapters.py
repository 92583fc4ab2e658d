"""Low-rank adapters of many requests at once beside quantised projections that all of them share.

`Int8TensorwiseOps.Linear` carries one dynamic LoRA for everything that goes through it (dynamic_lora.py).  A program that
serves several users from one model has another one for each request of a batch, which changes from call to call: here the
adapters of a layer lie in an `AdapterBank`, and a call names the adapter of every request.
"""
from __future__ import annotations

import math

import torch
from torch import Tensor, nn

from . import _lib, compile_ops
from ._comfy_compat import compute_device
from .dynamic_lora import _factors
from .int8_quant import SMALL_BATCH_ROWS, _layers_in_place, _scale_on


def _second_factor_exponent(top: float, scale: float) -> int:
    """e for which up * 2^e and scale * 2^-e are laid out in float16, top being the largest element of up: it comes to between 1 and 2.

    The kernels round t = scale * down @ x to 16 bits for the matrix unit, and float16 ends at 65504 above and has fewer bits below 2^-14.
    With up near 1 a t is beyond the type only where its share of an output is as well (in a rank whose column of up is as large as the
    others'), and what a t below 2^-14 loses is at most 2^-25 of up: r * 2^-24 of an output, steps of the smallest numbers.  Powers of
    two change no other rounding."""
    if not 0.0 < top < math.inf:
        return 0
    e = 1 - math.frexp(top)[1]
    if scale != 0.0 and math.isfinite(scale):   # (which stays a normal float32)
        at = math.frexp(scale)[1]
        e = min(max(e, at - 128), at + 125)
    return min(max(e, -126), 126)


class AdapterBank:
    """The adapters of ONE layer on one device, laid out for the kernels.

    adapters: one entry for each adapter number, (down [r, in features], up [out features, r]) or (down, up, scale); None for an
              adapter that leaves this layer alone.  Ranks may differ.  An adapter adds scale * up @ down to the layer's weight.
    dtype:    torch.bfloat16 or torch.float16, the activations' (default: the first factor's); factors are rounded to it once.
    device:   where the layer runs (default: the first factor's device if that is a GPU, else ComfyUI's compute device).
    in_features / out_features: needed where no entry has factors.

    In float16 an adapter's up is kept times a power of two and its scale times the inverse (_second_factor_exponent).
    A bank is laid out once.  Its tensors may be written into (captured graphs follow that too); assigning another one to an attribute of
    the layout is refused, because the host path keeps the tensors that the kernels are given.
    """

    def __init__(self, adapters, dtype: torch.dtype | None = None, device=None, in_features: int | None = None, out_features: int | None = None):
        entries = []
        for i, entry in enumerate(adapters):
            if entry is None:
                entries.append(None)
                continue
            if not 2 <= len(entry) <= 3:
                raise ValueError(f"adapter {i}: expected (down, up) or (down, up, scale)")
            down, up, scale = (*entry, 1.0)[:3]
            if down.dim() != 2 or up.dim() != 2 or down.shape[0] != up.shape[1]:
                raise ValueError(f"adapter {i}: down is {list(down.shape)} and up {list(up.shape)}, expected [r, in features] and [out features, r]")
            if in_features not in (None, down.shape[1]) or out_features not in (None, up.shape[0]):
                raise ValueError(f"adapter {i} is for a layer of {down.shape[1]} inputs and {up.shape[0]} outputs, expected {in_features} and {out_features}")
            in_features, out_features = down.shape[1], up.shape[0]
            entries.append((down, up, float(scale)))
        if in_features is None or out_features is None:
            raise ValueError("a bank without factors needs in_features and out_features")
        first = next((e for e in entries if e is not None), None)
        if dtype is None:
            dtype = torch.bfloat16 if first is None else first[0].dtype
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"adapters are kept in bfloat16 or float16, not {dtype}: give the activations' dtype")
        if device is None:
            device = first[0].device if first is not None and first[0].is_cuda else compute_device()
        self.dtype, self.count, self.in_features, self.out_features = dtype, len(entries), in_features, out_features
        self.ranks = [0 if e is None else e[0].shape[0] for e in entries]
        padded = [-(-r // 16) * 16 for r in self.ranks]
        self.max_rank = max(padded, default=0)
        offsets = [0]
        for r in padded:
            offsets.append(offsets[-1] + r)
        if offsets[-1] >= 1 << 31 or self.max_rank > 65536:
            raise ValueError(f"the ranks of a bank add up to less than 2^31 and stay within 65536, got {offsets[-1]} and {self.max_rank}")
        scales = [0.0 if e is None else e[2] for e in entries]
        with torch.no_grad():
            down_all = torch.zeros((offsets[-1], -(-in_features // 8) * 8), dtype=dtype, device=device)   # (whole 16-byte pieces)
            # (float16 factors are scaled before they are rounded)
            wide = dtype == torch.float16 and any(e is not None and e[1].dtype != torch.float16 for e in entries)
            up_all = torch.zeros((offsets[-1] * out_features,), dtype=torch.float32 if wide else dtype, device=device)
            for entry, at, r in zip(entries, offsets, padded):
                if entry is not None and entry[0].shape[0]:
                    down, up, _ = entry
                    down_all[at:at + down.shape[0], :in_features] = down.detach().to(device=device, dtype=dtype)
                    up_all[at * out_features:(at + r) * out_features].view(out_features, r)[:, :up.shape[1]] = up.detach().to(device=device, dtype=up_all.dtype)
            if dtype == torch.float16 and up_all.numel() and not up_all.is_meta:
                pieces = up_all.view(-1, 16 * out_features)   # (each of one adapter)
                tops = torch.maximum(pieces.amax(1), -pieces.amin(1)).tolist()
                exponents = [_second_factor_exponent(max(tops[at // 16:(at + r) // 16], key=lambda v: (v != v, v)), scale) if r else 0
                             for at, r, scale in zip(offsets, padded, scales)]
                if any(exponents):
                    scales = [math.ldexp(scale, -e) for scale, e in zip(scales, exponents)]
                    pieces.mul_(torch.tensor([2.0 ** e for e, r in zip(exponents, padded) for _ in range(r // 16)], dtype=torch.float32, device=device)[:, None])
            up_all = up_all.to(dtype)
        self.down, self.up = down_all, up_all
        self.scale = torch.tensor(scales, dtype=torch.float32, device=device)
        self.first_rank = torch.tensor(offsets, dtype=torch.int32, device=device)
        self.device = down_all.device
        # (as the host path takes it)
        self._native = (self.down, self.up, self.scale, self.first_rank, self.count, self.max_rank, self.in_features, self.out_features)

    _LAID_OUT = frozenset(("down", "up", "scale", "first_rank", "count", "max_rank", "in_features", "out_features", "dtype", "device", "ranks", "_native"))

    def __setattr__(self, name, value):
        if name in self._LAID_OUT and "_native" in self.__dict__:
            raise AttributeError(f"a bank is laid out once: make another one instead of assigning {name}")
        super().__setattr__(name, value)

    @classmethod
    def from_patches(cls, patches, **kwargs):
        """A bank of ComfyUI LoRA patches of one layer: (adapter, strength) for each adapter number or None, as the entries of
        the dynamic LoRA loaders hold them; alpha, rank and strength make the scale, which stays out of the rounded factors."""
        return cls([None if p is None else _factors(*p) for p in patches], **kwargs)


def _adapter_rows(x: Tensor, ids: Tensor) -> tuple[Tensor, int]:
    """(ids as the kernels take them, rows of x to each) of adapter numbers shaped like some leading dimensions of x."""
    _lib._dev(ids, "ids")
    lead = tuple(x.shape[:-1])
    if ids.dtype != torch.int32 or ids.device != x.device:
        raise TypeError(f"ids must be int32 on {x.device}, got {ids.dtype} on {ids.device}")
    if ids.dim() > len(lead) or tuple(ids.shape) != lead[:ids.dim()]:
        raise ValueError(f"ids must have the shape of leading dimensions of x, {list(lead)}, got {list(ids.shape)}")
    rows = 1
    for n in lead[ids.dim():]:
        rows *= n
    return ids.contiguous(), max(1, rows)


def _quantised_here(layer, x: Tensor) -> bool:
    """Whether the layer's own kernels can take the adapters: quantised weights in place, nothing else attached to it."""
    return bool(getattr(layer, "_is_quantized", False) and layer.lora_A is None and layer.weight.device == x.device
                and not (layer.comfy_cast_weights or len(layer.weight_function) > 0 or len(layer.bias_function) > 0)
                and (layer.bias is None or layer.bias.device == x.device))


def _forward_native(layers, x, banks, ids):
    """forward_adapters() without the interpreter's part of it, for layers of one rotation flag whose own kernels take the adapters, with
    everything in place; None for everything else.  (Four rows into 4096 columns: 31 us a call on the general path.)"""
    parts = _layers_in_place(layers)
    if parts is None:
        return None
    return _lib.host().adapters(x, ids, *parts, SMALL_BATCH_ROWS, tuple([getattr(bank, "_native", None) for bank in banks]))


def forward_adapters(layers, x: Tensor, banks, ids: Tensor):
    """layer(x) + scale_a * up_a @ down_a @ x with the adapter a of each row, for one layer or for several that read the same x.

    layers, banks: an Int8TensorwiseOps.Linear and its AdapterBank, or lists of them (then the result is a list).
    x:    [..., in features], bfloat16 or float16, the banks' dtype.
    ids:  int32 tensor on x's device, the adapter number of each request: of the shape of x's leading dimensions, all of them (one number
          for each token) or fewer ([batch] for x [batch, tokens, features]).  A number that is not one of the bank's (-1, say) is a
          request without an adapter.  The numbers are read by the kernels, so a captured graph follows what is written into the tensor.

    One rounding at the end: the projection stays in binary32 (in the order of _lib.EPI_FUSED) until the adapter's share has been
    added; down @ x is rounded to x's dtype for the matrix unit.  x is quantised once for all layers; which layers go together may change the
    order of binary32 sums, and so may the way a call goes: for 17 to 128 rows with more than 16 numbers the native path sums the adapters'
    share for itself, in a launch of its own, which contiguous ids of up to four layers of one rotation flag take in eager mode.
    A row without an adapter is the layer's result in that order, not layer(x) bit for bit.  The adapter acts on x itself,
    also where the layer rotates its activations (a dynamic LoRA of the layer gets them rotated).  Layers whose own kernels cannot take
    the adapters (not quantised, weights that ComfyUI casts or moves for the call, a dynamic LoRA attached) run by themselves, and
    their rounded result gets the adapters' share.  No gradients: under grad mode an input that asks for one is refused, and so is a layer
    with trainable parameters that goes alone; an input with a tangent always."""
    single = isinstance(layers, nn.Module)
    layers, banks = ([layers], [banks]) if single else (list(layers), list(banks))
    if type(x) is Tensor and x.is_cuda and 0 < len(layers) == len(banks) <= _lib.MAX_ADAPTED_LAYERS and not torch.compiler.is_compiling():
        outs = _forward_native(layers, x, banks, ids)
        if outs is not None:
            return outs[0] if single else outs
    if len(layers) != len(banks):
        raise ValueError(f"{len(layers)} layers and {len(banks)} banks")
    _lib._dev(x, "x")
    if x.dim() < 1:
        raise ValueError("x must have a feature dimension")
    _lib.refuse_gradients(x=x)
    for layer, bank in zip(layers, banks):
        if x.dtype != bank.dtype or x.device != bank.device:
            raise TypeError(f"x is {x.dtype} on {x.device}, the adapters are {bank.dtype} on {bank.device}")
        if x.shape[-1] != bank.in_features or getattr(layer, "out_features", bank.out_features) != bank.out_features:
            raise ValueError(f"x has {x.shape[-1]} features and the layer {getattr(layer, 'out_features', '?')} outputs, the adapters are for "
                             f"{bank.in_features} and {bank.out_features}")
    ids, per = _adapter_rows(x, ids)
    lead = x.shape[:-1]
    x2 = x.reshape(-1, x.shape[-1])
    rows = x2.shape[0]
    outs = [None] * len(layers)
    # under torch.compile the calls go through the registered operators, in eager mode they go past the dispatcher
    compiling = torch.compiler.is_compiling()
    add_adapters = torch.ops.i8f.add_adapters if compiling else compile_ops.add_adapters_eager
    linear_adapters = torch.ops.i8f.linear_adapters if compiling else compile_ops.linear_adapters_eager
    # layers of one rotation flag go together, as many as a launch takes: x quantised (or rotated) once, the adapters' first products in
    # one launch, the layers in another
    together = {}
    for i, layer in enumerate(layers):
        together.setdefault(bool(layer._use_quarot) if _quantised_here(layer, x) else None, []).append(i)
    for rotate, members in together.items():
        if rotate is None:   # layers that go alone
            for i in members:
                base = layers[i](x)
                _lib.refuse_gradients(**{"the layer's result": base})   # (of trainable parameters: it would end here)
                outs[i] = add_adapters(base.reshape(rows, banks[i].out_features), x2, ids, per, *compile_ops.bank_args(banks[i]))
            continue
        scales = [compile_ops.split_scale(_scale_on(layers[i], x.device)) for i in members]
        parts = zip(*[compile_ops.bank_args(banks[i]) for i in members])
        got = linear_adapters(x2, ids, per, rotate, [layers[i].weight for i in members], [t for t, _ in scales], [v for _, v in scales],
                                  [layers[i].bias for i in members], *[list(p) for p in parts])
        for i, y in zip(members, got):
            outs[i] = y
    outs = [y.reshape(*lead, y.shape[-1]) for y in outs]
    return outs[0] if single else outs
