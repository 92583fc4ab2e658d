"""Norms and rotations of heads and the attention at sizes, layouts and options drawn at random (the same ones in every run), against the formulas
in 64 bits."""
import random

import pytest
import torch

from test_gpu_attention import check, expected
from test_gpu_norm_heads import check as check_heads, expected as expected_heads

pytestmark = pytest.mark.gpu


def size(rng, most):
    return max(1, int(round(most ** rng.random())))


def heads_in_memory(rng, batch, tokens, heads, width, dtype):
    """[batch, tokens, heads, width] contiguous, heads first, part of a wider projection, from an odd address, or one batch for all."""
    g = torch.Generator(device="cuda").manual_seed(rng.randrange(1 << 30))
    make = lambda *s: (torch.randn(*s, generator=g, device="cuda") * 1.5).to(dtype)  # noqa: E731
    kind = rng.choice(("plain", "plain", "fused", "heads first", "odd", "wide", "expanded"))
    if kind == "fused":
        return make(batch, tokens, heads + 3, width)[:, :, 1:1 + heads]
    if kind == "heads first":
        return make(batch, heads, tokens, width).transpose(1, 2)
    if kind == "odd":
        return make(batch * tokens * heads * width + 1)[1:].view(batch, tokens, heads, width)
    if kind == "wide":
        return make(batch, tokens, heads, width + rng.choice((1, 8)))[..., :width]
    if kind == "expanded":
        return make(1, tokens, heads, width).expand(batch, -1, -1, -1)
    return make(batch, tokens, heads, width)


@pytest.mark.parametrize("seed", range(150))
def test_heads(pkg, dev, seed):
    rng = random.Random(seed)
    dtype = rng.choice((torch.bfloat16, torch.float16, torch.float32))
    batch, tokens, width = size(rng, 6), size(rng, 1500), rng.choice((64, 128, rng.randint(2, 256), 8 * rng.randint(1, 32)))
    xs = [heads_in_memory(rng, batch, tokens, size(rng, 24), width, dtype) for _ in range(rng.choice((1, 2, 2, 3, 5)))]
    ws = [rng.choice((None, (1 + 0.3 * torch.randn(width, device="cuda")).to(rng.choice((dtype, torch.float32))))) for _ in xs]
    pairs = rng.randint(1, width // 2)
    axes = rng.randint(1, min(4, pairs))
    cuts = sorted(rng.sample(range(1, pairs), axes - 1))
    dims = tuple(2 * (b - a) for a, b in zip([0, *cuts], [*cuts, pairs]))
    theta = tuple(rng.choice((10000.0, 256.0, 3.0)) for _ in dims)
    interleaved = rng.random() < 0.5
    r = pkg.RotaryAxes(dims, theta, interleaved=interleaved)
    p = torch.randint(-3000, 100000, (*([rng.choice((1, batch))] if rng.random() < 0.5 else []), tokens, axes), device="cuda")
    p = p.to(rng.choice((torch.int32, torch.int64, torch.float32, torch.float64)))
    p = p / 7 if p.is_floating_point() else p
    if rng.random() < 0.7:
        for got, x, w in zip(pkg.norm_heads(xs, ws, eps=1e-5, rotary=r, positions=p), xs, ws):
            check_heads(got, expected_heads(x, w, True, 1e-5, dims, theta, interleaved, p))
    else:
        for got, x in zip(pkg.rotate_heads(xs, r, p), xs):
            check_heads(got, expected_heads(x, None, False, 0.0, dims, theta, interleaved, p))


@pytest.mark.parametrize("seed", range(200))
def test_attention(pkg, dev, seed):
    rng = random.Random(1000 + seed)
    dtype = rng.choice((torch.bfloat16, torch.float16))
    batch, kv_heads, width = size(rng, 5), size(rng, 6), rng.choice((64, 128, rng.randint(1, 256), 8 * rng.randint(1, 32)))
    share, queries, keys = rng.choice((1, 1, 2, 5)), rng.choice((1, size(rng, 700))), size(rng, rng.choice((300, 5000)))
    q = heads_in_memory(rng, batch, queries, kv_heads * share, width, dtype)
    k, v = (heads_in_memory(rng, batch, keys, kv_heads, width, dtype) for _ in range(2))
    options = {}
    g = torch.Generator(device="cuda").manual_seed(seed)
    if rng.random() < 0.4:
        options["key_lengths"] = torch.randint(-2, keys + 3, (batch,), generator=g, device="cuda", dtype=rng.choice((torch.int32, torch.int64)))
    kind = rng.choice(("", "", "bool", "few", "float"))
    on = torch.rand(batch, keys, generator=g, device="cuda") < (0.02 if kind == "few" else 0.7)
    if kind in ("bool", "few"):
        options["key_mask"] = on
    elif kind == "float":
        m = torch.randn(batch, keys, generator=g, device="cuda").to(rng.choice((torch.bfloat16, torch.float16, torch.float32)))
        options["key_mask"] = torch.where(on, m, torch.full((), rng.choice((-float("inf"), torch.finfo(m.dtype).min)), dtype=m.dtype, device="cuda"))
    if rng.random() < 0.3:
        options["scale"] = rng.choice((0.02, 0.5))
    check(pkg.cross_attention(q, k, v, **options), expected(q, k, v, **options), (batch, queries, keys, kv_heads, share, width, kind))
