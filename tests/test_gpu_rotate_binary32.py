"""Rotations of heads in binary32: sine and cosine as exact as the type, over whole turns and far positions.

Bounds: the turns t are off by |t| 2^-51 with the rate's own rounding, 2 pi |t| 2^-51 < |t| 2^-48 of an angle.  What is left of them behind quarters is exact in
binary64, at most pi/4 as an angle, and rounded to binary32 by 2^-25; a series of which x and 1 - x^2 / 2 are the first parts has its last sum rounded
by 2^-25, x^2 by 2^-25 of itself and what follows it, below 0.09, by a few 2^-24 of itself: 2^-25 at the most; the terms left out are below 2^-28 together.
So sine and cosine are within 3 2^-25 + 2^-28 + |t| 2^-48.  An element of a turned pair adds its two products, each rounded, and their sum: 3 2^-24 of both."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 3 * 2.0 ** -25 + 2.0 ** -28


def turned(pkg, positions, rate, interleaved=True):
    """(cosine, sine) that the rotation has for one pair at each position: the pair (1, 0) turned.  theta^(-2/4) = rate for the second pair of an axis."""
    x = torch.zeros(1, positions.shape[0], 1, 4, device="cuda")
    x[..., 2 if interleaved else 1] = 1.0
    y = pkg.rotate_heads(x, pkg.RotaryAxes((4,), rate ** -2.0, interleaved=interleaved), positions[:, None])[0, :, 0]
    return (y[:, 2], y[:, 3]) if interleaved else (y[:, 1], y[:, 3])


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("kind", ["turn", "far", "negative", "integers"])
def test_sine_and_cosine(pkg, dev, kind, interleaved):
    n = 1 << 20
    g = torch.Generator(device="cuda").manual_seed(7)
    p = {"turn": torch.arange(n, device="cuda", dtype=torch.float64) * (2 * math.pi / n), "far": torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * 2.0 ** 31,
         "negative": -torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * 1e5, "integers": torch.randint(-(2 ** 31) + 1, 2 ** 31 - 1, (n,), generator=g, device="cuda")}[kind]
    for rate in (1.0, 0.01, 0.37):
        c, s = turned(pkg, p, rate, interleaved)
        angle = p.double().cpu().numpy() * (rate ** -2.0) ** -0.5
        for got, want in ((c, np.cos(angle)), (s, np.sin(angle))):
            off = np.abs(got.double().cpu().numpy() - want) - (E + np.abs(angle) / (2 * math.pi) * 2.0 ** -48)
            assert off.max() <= 0, (kind, rate, off.max())


def test_quarter_turns_and_eighths(pkg, dev):
    """Where quarters meet and where they begin, on either side."""
    turns = torch.arange(-64, 65, device="cuda", dtype=torch.float64) / 8
    p = (turns[:, None] + torch.tensor([-1e-9, 0.0, 1e-9], device="cuda", dtype=torch.float64)).flatten() * (2 * math.pi)
    c, s = turned(pkg, p, 1.0)
    assert (c.double() - p.cos()).abs().max() <= E + 2.0 ** -44 and (s.double() - p.sin()).abs().max() <= E + 2.0 ** -44


def test_turned_heads(pkg, dev):
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(2, 500, 3, 64, generator=g, device="cuda")
    p = torch.randint(0, 5000, (500, 2), generator=g, device="cuda")
    y = pkg.rotate_heads(x, pkg.RotaryAxes((32, 32), 10000.0), p).double()
    angle = torch.cat([p[:, a:a + 1].double() * 10000.0 ** (-torch.arange(0, 32, 2, device="cuda", dtype=torch.float64) / 32) for a in range(2)], 1)[None, :, None]
    a, b = x[..., 0::2].double(), x[..., 1::2].double()
    slack = (a.abs() + b.abs()) * (E + angle.abs() / (2 * math.pi) * 2.0 ** -48 + 3 * 2.0 ** -24)
    assert ((y[..., 0::2] - (a * angle.cos() - b * angle.sin())).abs() <= slack).all() and ((y[..., 1::2] - (a * angle.sin() + b * angle.cos())).abs() <= slack).all()


def test_positions_that_are_no_numbers(pkg, dev):
    p = torch.tensor([math.nan, math.inf, -math.inf, 1.0], device="cuda")
    c, s = turned(pkg, p, 1.0)
    assert torch.isnan(c[:3]).all() and torch.isnan(s[:3]).all() and torch.isfinite(c[3]) and torch.isfinite(s[3])
