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


def _bank(L, **over):
    fields = {"down": 16, "up": 16, "scale": 16, "first_rank": 16, "ids": 16, "rows_per_id": 1, "count": 2, "max_rank": 32, **over}
    return ctypes.byref(L._Adapters(*(fields[n] for n, _ in L._Adapters._fields_)))


def test_adapters_arguments_are_checked_before_any_launch(L):
    lib, null, one = L.lib(), ctypes.c_void_p(None), ctypes.c_void_p(16)
    down = lambda b, dt=L.BF16, M=4, K=64, ld=64, x=one, t=one: lib.i8f_adapters_down(x, dt, M, K, ld, b, t, null)  # noqa: E731
    assert down(None) == INVALID
    for bad in ({"count": -1}, {"max_rank": 24}, {"max_rank": -16}, {"rows_per_id": 0}, {"ids": None}, {"first_rank": None}, {"scale": None}, {"down": None},
                {"up": None}, {"up": 8}):
        assert down(_bank(L, **bad)) == INVALID, bad
    assert down(_bank(L, max_rank=1 << 20)) == UNSUPPORTED
    assert down(_bank(L), dt=L.F32) == INVALID and down(_bank(L), dt=9) == INVALID
    assert down(_bank(L), M=-1) == INVALID and down(_bank(L), ld=32) == INVALID and down(_bank(L), x=null) == INVALID and down(_bank(L), t=null) == INVALID
    assert down(_bank(L), t=ctypes.c_void_p(24)) == INVALID
    assert down(_bank(L), M=1 << 31) == UNSUPPORTED
    assert down(_bank(L, ids=None), M=0) == 0 and down(_bank(L, count=0), t=null) == 0 and down(_bank(L, max_rank=0, down=None, up=None), t=null) == 0
    up = lambda b, base=one, bd=L.F32, dt=L.BF16, out=ctypes.c_void_p(32), M=4, N=8, t=one: lib.i8f_adapters_up(base, bd, b, t, out, dt, M, N, null)  # noqa: E731
    assert up(_bank(L), bd=L.F16) == INVALID and up(_bank(L), dt=L.F32) == INVALID and up(_bank(L), base=null) == INVALID and up(_bank(L), t=null) == INVALID
    assert up(_bank(L), out=one) == INVALID           # binary32 read where 16 bits are written
    assert up(_bank(L), N=-1) == INVALID and up(_bank(L), M=0) == 0 and up(_bank(L), N=0) == 0
    need = lib.i8f_linear_w8a8_adapters_workspace_bytes(20, 8, 64)
    assert need >= 0 and lib.i8f_linear_w8a8_adapters_workspace_bytes(0, 8, 64) == 0

    def linear(b, M=20, N=8, K=64, t=one, work=one, nbytes=None, dt=L.BF16, mode=0, ws=one):
        return lib.i8f_linear_w8a8_adapters(one, one, one, ws, 1.0, mode, null, 0, b, t, one, dt, M, N, K, work, 1 << 40 if nbytes is None else nbytes, null)

    assert linear(_bank(L), dt=L.F32) == INVALID and linear(_bank(L), t=null) == INVALID and linear(_bank(L), K=-1) == INVALID
    assert linear(_bank(L), mode=7) == INVALID and linear(_bank(L), mode=1, ws=null) == INVALID
    assert linear(_bank(L), work=ctypes.c_void_p(24)) == INVALID
    if need:
        assert linear(_bank(L), nbytes=need - 1) == INVALID and linear(_bank(L), work=null) == INVALID
    assert linear(_bank(L), M=0) == 0 and linear(_bank(L), N=0) == 0

    def small(b, M=4, N=8, K=64, ld=64, t=one, dt=L.BF16, mode=0, ws=one):
        return lib.i8f_linear_w8a16_small_m_adapters(one, dt, M, K, ld, one, ws, 1.0, mode, null, 0, b, t, one, N, null)

    assert small(_bank(L), M=17) == UNSUPPORTED and small(_bank(L), ld=32) == INVALID and small(_bank(L), t=null) == INVALID
    assert small(_bank(L), dt=L.F32) == INVALID and small(_bank(L), mode=3) == INVALID and small(_bank(L), mode=1, ws=null) == INVALID
    assert small(_bank(L), M=0) == 0


def _norm(L, **over):
    a = L._BlockNormArgs()
    base = {"y": 16, "residual": 16, "M": 4, "K": 128, "ldy": 128, "ldr": 128, "dtype": L.BF16, "x_out": 16, "rows_per_gate": 1, "rows_per_scale": 1,
            "rows_per_shift": 1, "residual_scale": 1.0, "branch_scale": 1.0, "post_eps": 1e-6, "pre_eps": 1e-6}
    for k, v in {**base, **over}.items():
        setattr(a, k, v)
    return L.lib().i8f_block_norm(ctypes.byref(a), None)


def test_block_norm_arguments_are_checked_before_any_launch(L):
    assert L.lib().i8f_block_norm(None, None) == INVALID
    q = {"q": 16, "scale": 16}
    for bad in ({"M": -1}, {"K": -1}, {"dtype": 5}, {"y": None}, {"residual": None}, {"x_out": None}, {"ldy": 64}, {"ldr": 64}, {"post_norm": 3}, {"pre_norm": -1, "h": 16},
                {"post_norm": 1, "post_eps": -1.0}, {"post_norm": 1, "post_eps": float("nan")}, {"post_weight": 16}, {"pre_bias": 16, "h": 16},
                {"post_norm": 1, "post_weight": 16, "post_dtype": L.F16}, {"gate": 16, "rows_per_gate": 0}, {"mod_scale": 16, "rows_per_scale": 0, "h": 16},
                {"mod_shift": 16, "rows_per_shift": -1, "h": 16}, {"pre_norm": 1}, {"mod_scale": 16}, {"h": 16, **q}, {"q": 16}, {"scale": 16}, {"rotate_block": 128},
                {"rotate_block": 128, "K": 100, **q}):
        assert _norm(L, **bad) == INVALID, bad
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
        assert torch.equal(down[:n], f[0].bfloat16()) and torch.equal(up[:, :n], f[1].bfloat16())
        assert not down[n:].any() and not up[:, n:].any()


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
