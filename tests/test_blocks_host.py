"""Host side of the adapters of many requests and the norms between blocks: the C interface and its refusals, the banks' layout (no GPU)."""
import ctypes
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, UNSUPPORTED = -1, -2


def test_the_header_declares_what_the_binding_names(L):
    text = open(os.path.join(ROOT, "include", "i8f_blocks.h")).read()
    names = set(re.findall(r"\b(i8f_[a-z0-9_]+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S)))
    assert names == set(L.BLOCK_EXPORTS)
    for name in names:
        assert getattr(L.lib(), name) is not None


BANK = {"down": 16, "up": 16, "scale": 16, "first_rank": 16, "ids": 16, "rows_per_id": 1, "count": 2, "max_rank": 32}
LAYER = {"w": 16, "w_scale": 16, "w_scale_host": 1.0, "scale_mode": 0, "N": 8, "t": 16, "out": 16}


def _bank(L, **over):
    return ctypes.byref(L._Adapters(*({**BANK, **over}[n] for n, _ in L._Adapters._fields_)))


def _layers(L, *overs):
    """An array of layers, each with the fields of its dict (of the layer or of its adapters) instead of the usual ones."""
    arr = (L._AdaptedLayer * max(1, len(overs)))()
    for e, over in zip(arr, overs):
        e.adapters = L._Adapters(*({**BANK, **over}[n] for n, _ in L._Adapters._fields_))
        for k, v in {**LAYER, **over}.items():
            if k not in BANK:
                setattr(e, k, v)
    return arr


def test_adapters_arguments_are_checked_before_any_launch(L):
    lib, null, one = L.lib(), ctypes.c_void_p(None), ctypes.c_void_p(16)

    def down(*overs, dt=L.BF16, M=4, K=64, ld=64, x=one, n=None, rb=0, q=null, s=null, work=null):
        return lib.i8f_adapters_down(x, dt, M, K, ld, _layers(L, *overs), len(overs) if n is None else n, rb, q, s, work, 0, null)

    for bad in ({"count": -1}, {"max_rank": 24}, {"max_rank": -16}, {"rows_per_id": 0}, {"ids": None}, {"first_rank": None}, {"scale": None}, {"down": None},
                {"up": None}, {"up": 8}, {"t": None}, {"t": 24}):
        assert down(bad) == INVALID, bad
        assert down({}, bad) == INVALID, bad
    assert down({"max_rank": 1 << 20}) == UNSUPPORTED and down(*[{}] * 5) == UNSUPPORTED and down({}, n=-1) == INVALID
    assert lib.i8f_adapters_down(one, L.BF16, 4, 64, 64, None, 1, 0, null, null, null, 0, null) == INVALID
    assert down({}, {"ids": 32}) == INVALID and down({}, {"rows_per_id": 2}) == INVALID     # layers of one call have the same requests
    assert down({}, dt=L.F32) == INVALID and down({}, dt=9) == INVALID
    assert down({}, M=-1) == INVALID and down({}, ld=32) == INVALID and down({}, x=null) == INVALID
    assert down({}, q=one) == INVALID and down({}, s=one) == INVALID and down({}, rb=64) == UNSUPPORTED and down({}, rb=128) == INVALID
    assert down({}, work=ctypes.c_void_p(8)) == INVALID
    size = lib.i8f_adapters_down_workspace_bytes
    assert size(16, 4096, 32, 1) == size(0, 64, 16, 1) == size(4096, 0, 16, 1) == size(4096, 64, 0, 1) == size(1 << 31, 64, 16, 1) == 0
    assert size(4096, 4096, 32, 1) % (4096 * 32 * 4) == 0 and size(4096, 4096, 32, 1) > 0
    assert size(4096, 4096, 32, 0) == size(4096, 4096, 32, 1) + 4096 * 4096 * 2 and size(4096, 4089, 32, 1) == size(4096, 4089, 32, 0)
    assert size(200, 4096, 128, 1) == 0 < size(200, 4096, 192, 1) and size(1000, 4096, 16, 1) == 0 < size(1100, 4096, 16, 1)
    assert down({}, M=1 << 31) == UNSUPPORTED and down({}, K=(1 << 30) + 8, ld=(1 << 30) + 8) == UNSUPPORTED
    assert down({"ids": None, "t": None}, M=0) == 0

    def up(base=one, bd=L.F32, dt=L.BF16, out=ctypes.c_void_p(32), M=4, N=8, t=one):
        return lib.i8f_adapters_up(base, bd, _bank(L), t, out, dt, M, N, null)

    assert up(bd=L.F16) == INVALID and up(dt=L.F32) == INVALID and up(base=null) == INVALID and up(t=null) == INVALID
    assert up(out=one) == INVALID           # binary32 read where 16 bits are written
    assert up(N=-1) == INVALID and up(M=0) == 0 and up(N=0) == 0
    assert lib.i8f_linear_w8a8_adapters_workspace_bytes(20, 8, 64) == 0 and lib.i8f_linear_w8a8_adapters_workspace_bytes(0, 9, 63) == 0
    assert lib.i8f_linear_w8a8_adapters_workspace_bytes(20, 9, 64) == 20 * 9 * 4

    def linear(*overs, M=20, K=64, work=null, nbytes=0, dt=L.BF16, a=one, s=one):
        return lib.i8f_linear_w8a8_adapters(a, s, _layers(L, *overs), len(overs), dt, M, K, work, nbytes, null)

    for bad in ({"t": None}, {"scale_mode": 7}, {"scale_mode": 1, "w_scale": None}, {"N": -1}, {"w": None}, {"out": None}, {"bias": 16, "bias_dtype": 9}, {"ids": None}):
        assert linear(bad) == INVALID, bad
    assert linear({}, dt=L.F32) == INVALID and linear({}, K=-1) == INVALID and linear({}, s=null) == INVALID and linear({}, a=null) == INVALID
    assert linear({}, work=ctypes.c_void_p(24)) == INVALID
    assert linear({"N": 9}) == INVALID and linear({"N": 9}, work=one, nbytes=20 * 9 * 4 - 1) == INVALID     # needs a workspace
    assert linear({"w": 24}) == UNSUPPORTED and linear({"out": 18}) == UNSUPPORTED and linear({}, a=ctypes.c_void_p(20)) == UNSUPPORTED
    assert linear({}, M=0) == 0 and linear() == 0
    by_side = lib.i8f_adapters_by_side
    assert by_side(64, 512, 256, 1) and by_side(34, 512, 256, 2) and not by_side(34, 512, 256, 34) and not by_side(64, 512, 256, 0)
    assert not by_side(16, 512, 256, 1) and not by_side(4096, 512, 256, 1) and not by_side(64, 511, 256, 1) and not by_side(64, 512, 250, 1)
    assert linear({"side": 24}) == INVALID and linear({"side": 16}, {}) == INVALID and linear({"side": 16, "N": 9}) == UNSUPPORTED
    assert down({"side": 24}) == INVALID and down({}, {"side": 16}) == INVALID

    def small(*overs, M=4, K=64, ld=64, dt=L.BF16, x=one):
        return lib.i8f_linear_w8a16_small_m_adapters(x, dt, M, K, ld, _layers(L, *overs), len(overs), null)

    for bad in ({"t": None}, {"scale_mode": 3}, {"scale_mode": 1, "w_scale": None}, {"w": None}, {"out": None}, {"N": -1}):
        assert small(bad) == INVALID, bad
    assert small({"side": 16}) == UNSUPPORTED
    assert small({}, M=17) == UNSUPPORTED and small({}, ld=32) == INVALID and small({}, dt=L.F32) == INVALID and small({}, x=null) == INVALID
    assert small({}, M=0) == 0 and small() == 0


def _norm(L, **over):
    a = L._BlockNormArgs()
    base = {"y": 16, "residual": 16, "M": 4, "K": 128, "ldy": 128, "ldr": 128, "dtype": L.BF16, "x_out": 32, "rows_per_gate": 1, "rows_per_scale": 1,
            "rows_per_shift": 1, "residual_scale": 1.0, "branch_scale": 1.0, "post_eps": 1e-6, "pre_eps": 1e-6}
    for k, v in {**base, **over}.items():
        setattr(a, k, v)
    return L.lib().i8f_block_norm(ctypes.byref(a), None)


def test_block_norm_arguments_are_checked_before_any_launch(L):
    assert L.lib().i8f_block_norm(None, None) == INVALID
    q = {"q": 64, "scale": 16}
    for bad in ({"M": -1}, {"K": -1}, {"dtype": 5}, {"y": None}, {"residual": None}, {"x_out": None}, {"ldy": 64}, {"ldr": 64}, {"post_norm": 3}, {"pre_norm": -1, "h": 48},
                {"post_norm": 1, "post_eps": -1.0}, {"post_norm": 1, "post_eps": float("nan")}, {"post_weight": 16}, {"pre_bias": 16, "h": 48},
                {"post_norm": 1, "post_weight": 16, "post_dtype": L.F16}, {"gate": 16, "rows_per_gate": 0}, {"mod_scale": 16, "rows_per_scale": 0, "h": 48},
                {"mod_shift": 16, "rows_per_shift": -1, "h": 48}, {"pre_norm": 1}, {"mod_scale": 16}, {"h": 48, **q}, {"q": 64}, {"scale": 16}, {"rotate_block": 128},
                {"rotate_block": 128, "K": 100, **q}):
        assert _norm(L, **bad) == INVALID, bad
    for alias in ({"x_out": 16}, {"h": 16}, {"h": 32}, {"q": 16, "scale": 96}, {"q": 32, "scale": 96}):
        assert _norm(L, **alias) == INVALID, alias
    assert _norm(L, rotate_block=64, **q) == UNSUPPORTED
    assert _norm(L, M=1 << 31, ldy=128) == UNSUPPORTED
    assert _norm(L, M=0, y=None, residual=None, x_out=None) == 0


def test_a_bank_keeps_its_factors_padded_to_sixteen_ranks(pkg):
    g = torch.Generator().manual_seed(1)
    factors = [(torch.randn(3, 10, generator=g), torch.randn(6, 3, generator=g), 0.5), None, (torch.randn(16, 10, generator=g), torch.randn(6, 16, generator=g)),
               (torch.randn(20, 10, generator=g), torch.randn(6, 20, generator=g), 2)]
    bank = pkg.AdapterBank(factors, dtype=torch.bfloat16, device="cpu")
    assert bank.count == 4 and bank.ranks == [3, 0, 16, 20] and bank.max_rank == 32 and (bank.in_features, bank.out_features) == (10, 6)
    assert bank.first_rank.tolist() == [0, 16, 16, 32, 64] and bank.first_rank.dtype == torch.int32
    assert bank.scale.tolist() == [0.5, 0.0, 1.0, 2.0]
    for i, f in enumerate(factors):
        first, r = int(bank.first_rank[i]), int(bank.first_rank[i + 1] - bank.first_rank[i])
        down, up = bank.down[first:first + r], bank.up[first * 6:(first + r) * 6].view(6, r)
        if f is None:
            assert r == 0
            continue
        n = f[0].shape[0]
        assert torch.equal(down[:n, :10], f[0].bfloat16()) and torch.equal(up[:, :n], f[1].bfloat16())
        assert down.shape[1] == 16 and not down[:, 10:].any() and not down[n:].any() and not up[:, n:].any()


def test_banks_refuse_what_is_no_adapter(pkg):
    z, d = torch.zeros, {"dtype": torch.bfloat16, "device": "cpu"}
    for bad in ([(z(4, 8),)], [(z(4, 8), z(6, 5))], [(z(4, 8, 1), z(6, 4))], [(z(4, 8), z(6, 4)), (z(4, 9), z(6, 4))], [(z(4, 8), z(6, 4)), (z(4, 8), z(7, 4))], [None]):
        with pytest.raises(ValueError):
            pkg.AdapterBank(bad, **d)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        pkg.AdapterBank([(z(4, 8), z(6, 4))], device="cpu")
    assert pkg.AdapterBank([None], in_features=8, out_features=6, **d).max_rank == 0


def test_there_is_no_cpu_path(pkg):
    bank = pkg.AdapterBank([(torch.zeros(4, 8), torch.zeros(6, 4))], dtype=torch.bfloat16, device="cpu")
    lin = torch.nn.Linear(8, 6)
    with pytest.raises(RuntimeError, match="no CPU path"):
        pkg.forward_adapters(lin, torch.zeros(2, 8).bfloat16(), bank, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        pkg.block_norm(torch.zeros(2, 8), torch.zeros(2, 8))
    with pytest.raises(RuntimeError, match="no CPU path"):
        pkg.forward_block_norm([lin], torch.zeros(2, 8), torch.zeros(2, 8), pre_norm="rms")


def test_operators_of_a_traced_graph_give_shapes(pkg):
    ops, meta = torch.ops.i8f, dict(device="meta", dtype=torch.bfloat16)
    bank = pkg.AdapterBank([(torch.zeros(5, 40), torch.zeros(24, 5))], dtype=torch.bfloat16, device="meta")
    x, ids = torch.empty(6, 40, **meta), torch.empty(3, dtype=torch.int32, device="meta")
    down, up, scale, first, count, most = pkg.compile_ops.bank_args(bank)
    w = torch.empty(24, 40, dtype=torch.int8, device="meta")
    y, z = ops.linear_adapters(x, ids, 2, False, [w, w], [None, torch.empty(24, 1, device="meta")], [0.5, 0.0], [None, None], [down] * 2, [up] * 2,
                               [scale] * 2, [first] * 2, [count] * 2, [most] * 2)
    assert y.shape == z.shape == (6, 24) and y.dtype == torch.bfloat16
    assert ops.add_adapters(y, x, ids, 2, down, up, scale, first, count, most).shape == (6, 24)
    v = torch.empty(2, 3, 40, **meta)
    out, h = ops.block_norm(v, v, post_norm="rms")
    assert out.shape == v.shape and h.numel() == 0
    assert ops.block_norm(v, v, mod_scale=torch.empty(40, **meta))[1].shape == v.shape
    out, q, s = ops.block_norm_quantised(v, v, False, pre_norm="layer")
    assert out.shape == v.shape and q.shape == (6, 40) and q.dtype == torch.int8 and s.shape == (6, 1) and s.dtype == torch.float32
