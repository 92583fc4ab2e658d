"""Norms and rotations of heads against the formula in 64 bits, element by element.

Bounds, with v = 2^-24 and u half a step of the type:
    norm      a head's sum of squares has positive terms and goes through at most 14 sums in a row (eight elements of a lane, a tree over its
              lanes): 14 v of it; mean, eps, root and reciprocal a rounding each, half of that carried through the root; two products:
              (7 + 1/2 + 1/2 + 1 + 1 + 2) v < 14 v of the result.
    rotation  the angle is t turns in binary64, |t| 2^-51 off with the rate's own rounding, and at most half a turn in binary32: 2^-25 of a half turn;
              cosine and sine of that are two steps off, 2^-22.  Together e = 2^-22 + pi 2^-25 + 2 pi |t| 2^-51 < 2^-21 + |t| 2^-48.
              A turned element is off by (|x0| + |x1|) (e + 14 v + 2 v).
    both      and by u of itself, rounded once."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

V = 2.0 ** -24


def expected(x, weight, norm, eps, dims=(), theta=10000.0, interleaved=True, positions=None):
    """(value, bound) in float64 for heads [batch, tokens, heads, width]."""
    z = x.double()
    if norm:
        z = z / (z.square().mean(-1, keepdim=True) + eps).sqrt()
        if weight is not None:
            z = z * weight.double()
    slack = 14 * V * z.abs()
    if positions is not None:
        p = positions.double().cpu()
        p = (p[None] if p.dim() == 2 else p).expand(x.shape[0], -1, -1)
        thetas = theta if isinstance(theta, tuple) else (theta,) * len(dims)
        rate = [torch.tensor([t ** (-2 * j / n) for j in range(n // 2)], dtype=torch.float64) for t, n in zip(thetas, dims)]
        angle = torch.cat([p[..., a:a + 1] * r for a, r in enumerate(rate)], -1)[:, :, None].to(x.device)
        cos, sin, e = angle.cos(), angle.sin(), 2.0 ** -21 + angle.abs() / (2 * math.pi) * 2.0 ** -48
        n = sum(dims) // 2
        i0 = torch.arange(n, device=x.device) * (2 if interleaved else 1)
        i1 = i0 + (1 if interleaved else n)
        a, b = z[..., i0], z[..., i1]
        both = (a.abs() + b.abs()) * (e + 16 * V)
        z, slack = z.clone(), slack.clone()
        z[..., i0], z[..., i1] = a * cos - b * sin, a * sin + b * cos
        slack[..., i0], slack[..., i1] = both, both
    f = torch.finfo(x.dtype)
    return z, slack + f.eps / 2 * (z.abs() + slack) + f.smallest_normal * f.eps


def check(got, want, what=""):
    value, bound = want
    assert got.shape == value.shape and got.is_contiguous() and torch.isfinite(got.float()).all(), what
    worst = ((got.double() - value).abs() / bound).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} of the bound"


def heads(*shape, dtype=torch.bfloat16, seed=0, std=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed + shape[-1])
    x = torch.randn(shape, generator=g, device="cuda") * std
    x[..., :: max(1, shape[-1] // 3)] *= 8
    return x.to(dtype)


def weight(width, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(99 + seed)
    return (1 + 0.3 * torch.randn(width, generator=g, device="cuda")).to(dtype)


def grid(tokens, axes, dtype=torch.int64):
    i = torch.arange(tokens, device="cuda")
    return torch.stack([i // 5 ** (axes - 1 - a) % (5 if a else 1 << 30) for a in range(axes)], 1).to(dtype)


# (batch, tokens, heads of each tensor, width, elements to an axis)
SHAPES = [(1, 1, (1,), 1, ()), (2, 1, (3,), 2, (2,)), (1, 5, (1, 2), 7, (2, 4)), (3, 4, (5,), 16, (8, 8)), (1, 77, (5, 5), 37, (10, 14)), (2, 33, (4, 1), 64, (20, 22, 22)),
          (1, 9, (3,), 64, (2, 2, 2, 58)), (2, 130, (16,), 72, (16, 20)), (1, 64, (7, 7), 96, (32, 32, 32)), (2, 300, (6, 2), 128, (16, 56, 56)), (1, 3000, (10, 10), 128, (44, 42, 42)),
          (1, 40, (3, 3), 120, (40,)), (1, 17, (2,), 130, (60, 70)), (2, 21, (3, 1), 256, (64, 64)), (1, 10, (2,), 255, (250,)), (1, 6, (2, 2), 256, (62, 64, 128)), (1, 6, (2,), 255, (2,)), (2, 5, (3,), 256, (254,)), (1, 9, (2, 5), 64, (62,)), (1, 9, (2,), 66, (64,)),
          (1, 3, (70, 3), 128, (64, 32, 32)), (40000, 1, (1,), 8, (8,))]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_the_formula(pkg, dev, shape, dtype):
    batch, tokens, sizes, width, dims = shape
    xs = [heads(batch, tokens, n, width, dtype=dtype, seed=i) for i, n in enumerate(sizes)]
    ws = [weight(width, dtype if i else torch.float32, i) for i in range(len(xs))]
    for got, x, w in zip(pkg.norm_heads(xs, ws, eps=1e-5), xs, ws):
        check(got, expected(x, w, True, 1e-5), "norm")
    for got, x in zip(pkg.norm_heads(xs, eps=0.0), xs):
        check(got, expected(x, None, True, 0.0), "norm without a weight")
    if not dims:
        return
    for i, interleaved in enumerate((True, False)):
        theta = (10000.0, 256.0)[i]
        r, p = pkg.RotaryAxes(dims, theta, interleaved=interleaved), grid(tokens, len(dims), (torch.int64, torch.int32)[i])
        for got, x, w in zip(pkg.norm_heads(xs, ws, rotary=r, positions=p), xs, ws):
            check(got, expected(x, w, True, 1e-6, dims, theta, interleaved, p), f"norm and rotation, {interleaved}")
        for got, x in zip(pkg.rotate_heads(xs, r, p), xs):
            check(got, expected(x, None, False, 0.0, dims, theta, interleaved, p), f"rotation, {interleaved}")


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("kind", ["i32", "i64", "f32", "f64", "batch", "one batch", "strided"])
def test_positions(pkg, dev, kind, interleaved):
    """Far, negative and fractional ones, of every type and layout."""
    x, dims = heads(3, 20, 4, 64, dtype=torch.float32), (20, 22, 20)
    g = torch.Generator(device="cuda").manual_seed(5)
    far = torch.randint(-(2 ** 31) + 1, 2 ** 31 - 1, (20, 3), generator=g, device="cuda")
    p = {"i32": far.int(), "i64": far, "f32": far.float() / 4096, "f64": far.double() / 1000003}.get(kind)
    if p is None:
        p = torch.randint(-9, 3000, (1 if kind == "one batch" else 3, 20, 3), generator=g, device="cuda")
        p = p.transpose(1, 2).contiguous().transpose(1, 2) if kind == "strided" else p
    r = pkg.RotaryAxes(dims, (10000.0, 7.0, 2.0), interleaved=interleaved)
    check(pkg.rotate_heads(x, r, p), expected(x, None, False, 0.0, dims, (10000.0, 7.0, 2.0), interleaved, p), kind)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("width,dims", [(128, (16, 56, 56)), (72, (16, 20)), (37, (10, 14))])
def test_strides(pkg, dev, width, dims, dtype):
    """Views of a fused projection, heads in front of tokens, expanded batches, odd offsets."""
    p, r, w = grid(12, len(dims)), pkg.RotaryAxes(dims), weight(width, dtype)
    fused = heads(2, 12, 9, width, dtype=dtype)
    swapped = heads(2, 3, 12, width, dtype=dtype).transpose(1, 2)
    offset = torch.empty(2 * 12 * 3 * width + 3, dtype=dtype, device="cuda")[3:].view(2, 12, 3, width).copy_(swapped)
    for x in (fused[:, :, 2:5], swapped, fused[:1, :, :3].expand(2, -1, -1, -1), fused[:, :, ::3], offset, fused[:, :, :3].transpose(-1, -2).contiguous().transpose(-1, -2),
              fused[:, :1, :3].expand(-1, 12, -1, -1)):
        check(pkg.norm_heads(x, w, rotary=r, positions=p), expected(x, w, True, 1e-6, dims, 10000.0, True, p))
        check(pkg.rotate_heads(x, r, p), expected(x, None, False, 0.0, dims, 10000.0, True, p))
    three = pkg.norm_heads(fused[0], w, rotary=r, positions=p)
    assert torch.equal(three, pkg.norm_heads(fused[:1], w, rotary=r, positions=p)[0])


def test_heads_do_not_depend_on_what_is_beside_them(pkg, dev):
    """A head's bits: alone, in a large batch, beside other tensors."""
    dims, p = (16, 56, 56), grid(600, 3)
    x, y, w = heads(1, 600, 10, 128), heads(1, 600, 30, 128, seed=3), weight(128, torch.bfloat16)
    r = pkg.RotaryAxes(dims)
    whole = pkg.norm_heads([x, y, x, y, y], [w, None, w, None, w], rotary=r, positions=p)
    assert torch.equal(whole[0], whole[2]) and torch.equal(whole[1], whole[3])
    for t in (0, 599):
        one = pkg.norm_heads(x[:, t:t + 1, 3:4], w, rotary=r, positions=p[t:t + 1])
        assert torch.equal(one, whole[0][:, t:t + 1, 3:4])
    assert torch.equal(pkg.norm_heads(y, None, rotary=r, positions=p), whole[1])


def test_values_that_are_not_finite_stay_in_their_head(pkg, dev):
    for width, dims in ((128, (32, 32)), (37, (10,))):
        x = heads(2, 30, 4, width)
        r, p = pkg.RotaryAxes(dims), grid(30, len(dims))
        want = pkg.rotate_heads(x, r, p), pkg.norm_heads(x, rotary=r, positions=p)
        x[1, 3, 2, 0], x[0, 29, 3, width - 1], x[0, 5, 0, 3] = float("nan"), float("inf"), -float("inf")
        for i, got in enumerate((pkg.rotate_heads(x, r, p), pkg.norm_heads(x, rotary=r, positions=p))):
            same = torch.ones(2, 30, 4, dtype=torch.bool, device="cuda")
            same[1, 3, 2] = same[0, 29, 3] = same[0, 5, 0] = False
            assert torch.equal(got[same], want[i][same])
            if i == 0:   # without a norm a pair at the most
                assert torch.isinf(got[0, 29, 3, -1]) and torch.isfinite(got[0, 29, 3, :-1].float()).all() and (~torch.isfinite(got[1, 3, 2].float())).sum() == 2


def test_zero_heads_and_empty_tensors(pkg, dev):
    r = pkg.RotaryAxes((8,))
    z = torch.zeros(2, 3, 4, 16, device="cuda", dtype=torch.bfloat16)
    assert not pkg.norm_heads(z).any()
    for shape in ((0, 3, 4, 16), (2, 0, 4, 16), (2, 3, 0, 16), (0, 4, 16)):
        x = torch.empty(shape, device="cuda", dtype=torch.bfloat16)
        tokens = shape[-3]
        assert pkg.norm_heads(x, rotary=r, positions=torch.zeros(tokens, 1, device="cuda")).shape == shape
        assert pkg.rotate_heads([x, x], r, torch.zeros(tokens, 1, device="cuda"))[1].shape == shape
    assert pkg.norm_heads([]) == []


def test_refusals(pkg, dev):
    x, r, p = heads(2, 3, 4, 16), pkg.RotaryAxes((8, 4)), grid(3, 2)
    ok = dict(rotary=r, positions=p)
    for bad in (lambda: pkg.norm_heads(x[0, 0]), lambda: pkg.norm_heads([x, x[:1]]), lambda: pkg.norm_heads([x, x[..., :8]]), lambda: pkg.norm_heads(x, eps=-1.0),
                lambda: pkg.norm_heads(x, weight(8, x.dtype)), lambda: pkg.norm_heads(x, weight(16, torch.float16)), lambda: pkg.norm_heads(x, weight(16, x.dtype).cpu()),
                lambda: pkg.rotate_heads(x, r, p[:2]), lambda: pkg.rotate_heads(x, r, p[:, :1]), lambda: pkg.rotate_heads(x, r, p[None].expand(3, -1, -1)),
                lambda: pkg.rotate_heads(x, r, p.half()), lambda: pkg.rotate_heads(x, r, p.cpu()), lambda: pkg.rotate_heads(x, pkg.RotaryAxes((8, 10)), p),
                lambda: pkg.rotate_heads(x, pkg.RotaryAxes((8, 4), device="cpu"), p), lambda: pkg.norm_heads([x, x.half()], **ok), lambda: pkg.norm_heads(x.double(), **ok),
                lambda: pkg.norm_heads(torch.zeros(1, 1, 1, 257, device="cuda")), lambda: pkg.norm_heads(torch.zeros(1, 1, 1, 0, device="cuda"))):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            bad()


def test_captured_call_follows_positions_and_heads(pkg, dev):
    dims = (16, 56, 56)
    x, p, w, r = heads(1, 50, 6, 128), grid(50, 3), weight(128, torch.bfloat16), pkg.RotaryAxes(dims)
    pkg.norm_heads(x, w, rotary=r, positions=p)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.norm_heads(x, w, rotary=r, positions=p)
    for i in range(3):
        x.copy_(heads(1, 50, 6, 128, seed=i + 10))
        p.add_(7)
        graph.replay()
        assert torch.equal(out, pkg.norm_heads(x, w, rotary=r, positions=p))


def test_on_another_stream_and_under_the_compiler(pkg, dev):
    dims = (16, 56, 56)
    x, p, w, r = heads(2, 50, 6, 128), grid(50, 3), weight(128, torch.bfloat16), pkg.RotaryAxes(dims)
    want = pkg.norm_heads([x, x], [w, None], rotary=r, positions=p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pkg.norm_heads([x, x], [w, None], rotary=r, positions=p)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    compiled = torch.compile(lambda a, q: pkg.norm_heads([a, a], [w, None], rotary=r, positions=q), backend="eager", fullgraph=True)
    assert all(torch.equal(a, b) for a, b in zip(compiled(x, p), want))
