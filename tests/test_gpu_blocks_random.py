"""Adapters and block norms at sizes, layouts and options drawn at random (the same ones in every run), against the formulas in 64 bits."""
import random

import pytest
import torch

from test_gpu_adapters import check, expected, factors_of, layer_of
from test_gpu_block_norm import check as check_norm, expected as expected_norm

pytestmark = pytest.mark.gpu


def size(rng, most, multiple=1):
    """1 to most, spread over the logarithm, in multiples of `multiple` where there are any."""
    n = int(round(most ** rng.random()))
    return max(multiple, n // multiple * multiple)


def rows_in_memory(rng, rows, K, dtype, dev):
    """[rows, K] contiguous, as part of a wider tensor, or from an odd address."""
    g = torch.Generator(device="cuda").manual_seed(rng.randrange(1 << 30))
    kind = rng.choice(("plain", "plain", "wide", "odd"))
    if kind == "wide":
        pad = rng.choice((1, 8, 24))
        return torch.randn(rows, K + pad, generator=g, device=dev).to(dtype)[:, pad // 2:pad // 2 + K]
    if kind == "odd":
        return torch.randn(rows * K + 1, generator=g, device=dev).to(dtype)[1:].view(rows, K)
    return torch.randn(rows, K, generator=g, device=dev).to(dtype)


@pytest.mark.parametrize("seed", range(150))
def test_adapters(pkg, dev, seed):
    rng = random.Random(seed)
    dtype = rng.choice((torch.bfloat16, torch.float16))
    rows, K = size(rng, 2500), size(rng, 5000, rng.choice((1, 8, 16, 64, 128)))
    rotate = K % 128 == 0 and rng.random() < 0.5
    layers, adapters = [], []
    count = size(rng, 40)
    for i in range(rng.choice((1, 1, 2, 3, 4, 6))):
        N = size(rng, 2500, rng.choice((1, 8, 8, 64)))
        layers.append(layer_of(pkg, K, N, dtype, bias=rng.random() < 0.5, rotate=rotate, per_row=rng.random() < 0.7, seed=i))
        ranks = [None if rng.random() < 0.1 else size(rng, 100) for _ in range(max(1, count - rng.randrange(3)))]
        adapters.append(factors_of(K, N, ranks, dtype, seed + i))
    banks = [pkg.AdapterBank(a, dtype=dtype, device=dev, in_features=K, out_features=lin.out_features) for a, lin in zip(adapters, layers)]
    x = rows_in_memory(rng, rows, K, dtype, dev)
    batch = rng.choice([b for b in (1, 2, 3, 5, rows) if rows % b == 0])
    numbers = torch.tensor([rng.choice((-1, rng.randrange(count), rng.randrange(count), count)) for _ in range(batch)], dtype=torch.int32, device=dev)
    each = numbers.repeat_interleave(rows // batch)
    if rng.random() < 0.5 and x.is_contiguous():   # one number for a request
        outs = pkg.forward_adapters(layers, x.view(batch, rows // batch, K), banks, numbers)
    else:
        outs = pkg.forward_adapters(layers, x, banks, each)
    for lin, some, y in zip(layers, adapters, outs):
        check(y.reshape(rows, -1), *expected(pkg, lin, x.contiguous(), some, each))


@pytest.mark.parametrize("seed", range(150))
def test_block_norms(pkg, L, dev, seed):
    rng = random.Random(1000 + seed)
    dtype = rng.choice((torch.bfloat16, torch.float16, torch.float32))
    batch, tokens, K = size(rng, 8), size(rng, 300), size(rng, 20000, rng.choice((1, 1, 8, 16, 128)))
    y, r = (rows_in_memory(rng, batch * tokens, K, dtype, dev).view(batch, tokens, K) for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(seed)

    def vector(*lead, of=dtype, about=0.0):
        return (torch.randn(*lead, K, generator=g, device=dev) * 0.5 + about).to(of)

    ops = {"post_eps": 10.0 ** rng.uniform(-6, -2), "pre_eps": 10.0 ** rng.uniform(-6, -2), "residual_scale": rng.choice((1.0, 0.7)), "branch_scale": rng.choice((1.0, -0.4))}
    for name in ("post", "pre"):
        kind = rng.choice((None, "rms", "layer")) if name == "post" else rng.choice((None, "rms", "layer", "rms"))
        ops[f"{name}_norm"] = kind
        of = rng.choice((dtype, torch.float32))
        if kind and rng.random() < 0.7:
            ops[f"{name}_weight"] = vector(of=of, about=1.0)
        if kind and rng.random() < 0.3:
            ops[f"{name}_bias"] = vector(of=of)
    for name in ("gate", "mod_scale", "mod_shift"):
        lead = rng.choice((None, (), (1, 1), (batch, 1), (batch, tokens)))
        if lead is not None:
            ops[name] = vector(*lead)
    ops["gate_tanh"] = rng.random() < 0.5
    x, h = pkg.block_norm(y, r, **ops)
    want_x, want_h = expected_norm(y, r, **ops)
    check_norm(x, want_x, "x")
    assert (h is None) == (want_h is None)
    if h is not None:
        check_norm(h, want_h, "h")
        rotate = K % 128 == 0 and rng.random() < 0.5
        x8, q, s = L.block_norm(y, r, quantise=True, rotate=rotate, **ops)
        want_q, want_s = L.quant_rowwise(h.view(-1, K), rotate=rotate)
        assert torch.equal(x, x8) and torch.equal(q, want_q) and torch.equal(s, want_s)
