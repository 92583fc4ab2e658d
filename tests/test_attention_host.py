"""Host side of the heads' norms and rotations and of the attention over other states: the C interface and its refusals, the rotation's layout,
shapes under a tracer (no GPU)."""
import ctypes
import math
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, UNSUPPORTED = -1, -2


def test_the_header_declares_what_the_binding_names(L):
    text = open(os.path.join(ROOT, "include", "i8f_attention.h")).read()
    names = set(re.findall(r"\b(i8f_[a-z0-9_]+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S)))
    assert names == set(L.ATTENTION_EXPORTS)
    for name in names:
        assert getattr(L.lib(), name) is not None


def _heads(L, args=None, *groups, n=None):
    """i8f_norm_rotate of valid arguments with these fields instead."""
    base = {"batch": 1, "tokens": 2, "width": 8, "dtype": L.BF16, "norm": 1, "eps": 1e-6, "axes": 2, "first_pair": (0, 1, 4, 0, 0), "positions_type": 0, "rates": 1 << 20,
            "positions": 1 << 21, "position_token": 2, "position_axis": 1, **(args or {})}
    a = L._NormRotateArgs()
    for k, v in base.items():
        setattr(a, k, (ctypes.c_int * 5)(*v) if k == "first_pair" else v)
    arr = (L._Heads * max(1, len(groups)))()
    for i, (e, over) in enumerate(zip(arr, groups)):
        for k, v in {"x": 1 << 22, "out": (1 << 24) + (i << 20), "heads": 3, "batch_stride": 48, "token_stride": 24, "head_stride": 8, **over}.items():
            setattr(e, k, v)
    return L.lib().i8f_norm_rotate(ctypes.byref(a), arr, len(groups) if n is None else n, None)


def test_norm_rotate_arguments_are_checked_before_any_launch(L):
    assert L.lib().i8f_norm_rotate(None, None, 0, None) == INVALID
    for bad in ({"batch": -1}, {"tokens": -1}, {"width": 0}, {"width": -8}, {"dtype": 3}, {"eps": -1.0}, {"eps": float("nan")}, {"axes": -1}, {"positions_type": 4},
                {"positions_type": -1}, {"first_pair": (1, 2, 4, 0, 0)}, {"first_pair": (0, 2, 2, 0, 0)}, {"first_pair": (0, 3, 1, 0, 0)}, {"first_pair": (0, 1, 5, 0, 0)},
                {"rates": None}, {"positions": None}, {"position_batch": -1}, {"position_token": -1}, {"position_axis": -1}):
        assert _heads(L, bad, {}) == INVALID, bad
    for bad in ({"x": None}, {"out": None}, {"heads": -1}, {"batch_stride": -1}, {"token_stride": -1}, {"head_stride": -1}, {"x": (1 << 22) + 1}, {"weight": 16, "weight_dtype": L.F16},
                {"out": 1 << 22}, {"out": (1 << 22) + 94}, {"out": (1 << 22) - 94}):
        assert _heads(L, None, bad) == INVALID, bad
        assert _heads(L, None, {}, bad) == INVALID, bad
    assert _heads(L, {"norm": 0}, {"weight": 16, "weight_dtype": L.BF16}) == INVALID     # a weight without a norm
    assert _heads(L, None, {"out": 1 << 24}, {"out": (1 << 24) + 94}) == INVALID          # outputs that overlap
    assert _heads(L, None, {}, {}, n=-1) == INVALID and L.lib().i8f_norm_rotate(ctypes.byref(L._NormRotateArgs(width=8)), None, 1, None) == INVALID
    assert _heads(L, {"axes": 5}, {}) == UNSUPPORTED and _heads(L, {"width": 257}, {}) == UNSUPPORTED and _heads(L, None, *[{}] * 5) == UNSUPPORTED
    assert _heads(L, {"batch": 1 << 31}, {}) == UNSUPPORTED and _heads(L, {"tokens": 1 << 31}, {}) == UNSUPPORTED
    assert _heads(L, None, {"token_stride": 1 << 62}) == UNSUPPORTED
    for empty in ({"batch": 0}, {"tokens": 0}):
        assert _heads(L, {**empty, "rates": None, "positions": None}, {"x": None, "out": None}) == 0
    assert _heads(L, None, {"heads": 0, "x": None, "out": None}) == 0 and _heads(L) == 0


def _attention_args(L, **over):
    base = {"q": 1 << 20, "k": 1 << 22, "v": 1 << 23, "out": 1 << 24, "batch": 2, "queries": 3, "keys": 5, "heads": 4, "kv_heads": 2, "width": 8, "q_batch": 96, "q_token": 32,
            "q_head": 8, "k_batch": 80, "k_token": 16, "k_head": 8, "v_batch": 80, "v_token": 16, "v_head": 8, "dtype": L.BF16, "scale": 0.5, **over}
    a = L._AttentionArgs()
    for k, v in base.items():
        setattr(a, k, v)
    return a


def _attention(L, **over):
    return L.lib().i8f_attention(ctypes.byref(_attention_args(L, **over)), None)


def test_attention_arguments_are_checked_before_any_launch(L):
    assert L.lib().i8f_attention(None, None) == INVALID
    for bad in (*({n: -1} for n in ("batch", "queries", "keys", "heads", "kv_heads", "width", "q_batch", "q_token", "q_head", "k_batch", "k_token", "k_head", "v_batch",
                                    "v_token", "v_head")),
                {"width": 0}, {"dtype": 9}, {"kv_heads": 0}, {"kv_heads": 3}, {"scale": 0.0}, {"scale": -1.0}, {"scale": float("inf")}, {"scale": float("nan")}, {"scale": 2.0 ** 127}, {"q": (1 << 20) + 1}, {"v": (1 << 23) + 1},
                {"q": None}, {"k": None}, {"v": None}, {"out": None}, {"key_lengths": 16, "lengths_type": 2}, {"key_mask": 16, "mask_type": 4}, {"key_mask": 16, "mask_type": -1},
                {"key_mask": 16, "mask_batch": -1}, {"key_mask": 16, "mask_key": -1}, {"out": 1 << 20}, {"out": (1 << 22) + 16}, {"out": (1 << 23) - 16}):
        assert _attention(L, **bad) == INVALID, bad
    for bad in ({"dtype": L.F32}, {"width": 257}, {"batch": 1 << 31}, {"queries": 1 << 31}, {"keys": 1 << 31}, {"heads": 1 << 31}, {"k_token": 1 << 61}):
        assert _attention(L, **bad) == UNSUPPORTED, bad
    assert _attention(L, batch=0, q=None, out=None) == 0 and _attention(L, queries=0) == 0 and _attention(L, heads=0, kv_heads=0) == 0
    size = lambda **over: L.lib().i8f_attention_workspace_bytes(ctypes.byref(_attention_args(L, **over)))  # noqa: E731
    for bad in ({}, {"batch": 0}, {"queries": 0}, {"heads": 0, "kv_heads": 0}, {"keys": 0, "width": 7}, {"batch": -1}, {"kv_heads": 3}, {"width": 300}):
        assert size(**bad) == 0, bad
    assert L.lib().i8f_attention_workspace_bytes(None) == 0
    # rows that are not whole aligned pieces are copied: q [2, 3, 4, 8], k and v [2, 5, 2, 8]
    assert size(q=(1 << 20) + 2) == 2 * 3 * 4 * 16 and size(k=(1 << 22) + 8) == size(v_head=9) == 2 * 5 * 2 * 16 and size(width=5) == 2 * 3 * 4 * 16 + 2 * 2 * 5 * 2 * 16
    assert size(k_token=(1 << 22) + 8, k_batch=1 << 40, out=1 << 50) == 2 * 5 * 2 * 16
    assert _attention(L, width=5) == INVALID and _attention(L, width=5, workspace=16, workspace_bytes=1023) == INVALID and _attention(L, width=5, workspace=24, workspace_bytes=1 << 20) == INVALID
    long = {"keys": 100000, "k_batch": 1600000, "v_batch": 1600000, "v": 1 << 30, "out": 1 << 40}
    assert size(**long) > 0 and _attention(L, **long) == INVALID and _attention(L, **long, workspace=16, workspace_bytes=size(**long) - 1) == INVALID


def test_a_rotation_keeps_turns_to_a_unit(pkg):
    r = pkg.RotaryAxes((4, 2, 6), 100.0, device="cpu")
    want = [1.0, 100 ** -0.5, 1.0, 1.0, 100 ** (-1 / 3), 100 ** (-2 / 3)]
    assert r.rates.dtype == torch.float64 and torch.allclose(r.rates * 2 * math.pi, torch.tensor(want, dtype=torch.float64), rtol=1e-15, atol=0)
    assert r.dims == (4, 2, 6) and r.interleaved and r.theta == (100.0, 100.0, 100.0)
    assert torch.equal(pkg.RotaryAxes((4, 2), (100.0, 7.0), device="cpu").rates, r.rates[:3])
    for name in ("dims", "theta", "rates", "interleaved", "other"):
        with pytest.raises(AttributeError, match="laid out once"):
            setattr(r, name, None)


def test_rotations_refuse_what_is_none(pkg):
    with pytest.raises(TypeError):
        pkg.RotaryAxes((2.0, 4), device="cpu")
    for dims in ((), (2, 2, 2, 2, 2), (3,), (0,), (-2,)):
        with pytest.raises(ValueError, match="even numbers"):
            pkg.RotaryAxes(dims, device="cpu")
    for theta in (0.0, -1.0, math.inf, math.nan, (10.0,), (10.0, 0.0)):
        with pytest.raises(ValueError, match="theta"):
            pkg.RotaryAxes((2, 2), theta, device="cpu")


def test_there_is_no_cpu_path(pkg):
    x, r = torch.zeros(1, 2, 3, 8).bfloat16(), pkg.RotaryAxes((4, 4), device="cpu")
    with pytest.raises(RuntimeError, match="no CPU path"):
        pkg.norm_heads(x)
    with pytest.raises(RuntimeError, match="no CPU path"):
        pkg.rotate_heads([x, x], r, torch.zeros(2, 2))
    with pytest.raises(RuntimeError, match="no CPU path"):
        pkg.cross_attention(x, x, x)


def test_arguments_that_do_not_go_together(pkg):
    x, r = torch.zeros(1, 2, 3, 8).bfloat16(), pkg.RotaryAxes((4, 4), device="cpu")
    lin = torch.nn.Linear(8, 8)
    with pytest.raises(ValueError, match="go together"):
        pkg.norm_heads(x, rotary=r)
    with pytest.raises(ValueError, match="go together"):
        pkg.norm_heads(x, positions=torch.zeros(2, 2))
    with pytest.raises(ValueError, match="its axes"):
        pkg.rotate_heads(x, None, torch.zeros(2, 2))
    with pytest.raises(TypeError, match="RotaryAxes"):
        pkg.rotate_heads(x, (4, 4), torch.zeros(2, 2))
    with pytest.raises(TypeError, match="tensors"):
        pkg.norm_heads([1.0])
    with pytest.raises(ValueError, match="weights"):
        pkg.norm_heads([x, x], [None])
    for bad in ({"q_weight": torch.ones(8)}, {"rotary": r}, {"positions": torch.zeros(2, 2)}, {"context_positions": torch.zeros(2, 2)}, {"gate": torch.ones(8)},
                {"residual": torch.ones(8)}):
        with pytest.raises(ValueError):
            pkg.forward_cross_attention(x[0], None, lin, lin, lin, heads=1, **bad)


def test_gradients_are_refused(pkg):
    x = torch.zeros(1, 2, 3, 8, requires_grad=True)
    for call in (lambda: pkg.norm_heads(x), lambda: pkg.norm_heads(x.detach(), x[0, 0, 0]), lambda: pkg.rotate_heads(x, pkg.RotaryAxes((8,), device="cpu"), torch.zeros(2, 1)),
                 lambda: pkg.cross_attention(x, x.detach(), x.detach()), lambda: pkg.cross_attention(x.detach(), x.detach(), x)):
        with pytest.raises(RuntimeError, match="gradient"):
            call()


def test_operators_of_a_traced_graph_give_shapes(pkg):
    x = torch.empty(2, 3, 4, 16, device="meta", dtype=torch.bfloat16)
    for y in torch.ops.i8f.norm_rotate_heads([x[:, :, :3], x], [None, torch.empty(16, device="meta")], True, 1e-6, None, [], False, None):
        assert y.shape[-1] == 16 and y.is_contiguous() and y.dtype == torch.bfloat16
    o = torch.ops.i8f.cross_attention(x.transpose(1, 2), torch.empty(2, 7, 1, 16, device="meta", dtype=torch.bfloat16), torch.empty(2, 7, 1, 16, device="meta", dtype=torch.bfloat16))
    assert o.shape == (2, 4, 3, 16) and o.is_contiguous()
