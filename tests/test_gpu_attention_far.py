"""Attention over scores, addends and values far from one: what a running maximum may lose there and the formula does not.

Bounds, with V = 2^-24 and u half a step of the type:
    a score is off by at most E = scale (D + 4) V sum |q_e k_e| + 4 V (|s| + |m|), as in test_gpu_attention; where the largest one of a row is more than
    2 E + 40 above every other, those others' weights are below e^-40 each, and the result is that state's value: off by u of it and n e^-40 2 max|v|.
    Where it is not, weights are positive and sum to one, each rounded by u: the result lies within the values, by (2 u + 2 n V + 2^-17) of the largest.
    Equal scores are equal in binary32 too, whatever their rounding: the weights are 1/n, each off by u and 2^-21 of itself, and the result their mean."""
import math

import pytest
import torch

from test_gpu_attention import V, check, counts_of, expected, inputs

pytestmark = pytest.mark.gpu

# (batch, queries, keys, heads, kv heads, width): apart, over few states and over many (split); 128 rows together, split, whole; 256 rows
FORMS = [(2, 3, 300, 2, 2, 128), (1, 1, 1, 2, 2, 64), (1, 2, 3000, 4, 2, 72), (2, 70, 300, 4, 4, 200), (1, 300, 4000, 1, 1, 128), (1, 700, 333, 8, 8, 128), (1, 700, 129, 8, 8, 96), (1, 8200, 4113, 32, 32, 64), (1, 8150, 4113, 32, 32, 128)]


def masked(kind, batch, keys):
    on = torch.arange(keys, device="cuda").expand(batch, -1) % 3 != 1
    return {"none": {}, "lengths": {"key_lengths": torch.tensor([keys - keys // 3, keys][:batch], device="cuda")}, "bool": {"key_mask": on},
            "addends": {"key_mask": torch.where(on, 0.0, -math.inf)}}[kind]


def some(size):
    """Rows and heads that are compared: all, or a part of a large call's."""
    queries, heads = size[1], size[3]
    if queries * heads < 20000:
        return torch.arange(queries, device="cuda"), range(heads)
    return torch.cat([torch.arange(a, a + 40, device="cuda") for a in (0, 230, queries // 2, queries - 40)]), (0, heads // 2, heads - 1)


def compare(got, q, k, v, size, scale, mask):
    batch, queries, keys, heads, kv_heads, width = size
    scale = width ** -0.5 if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    rows, picked = some(size)
    single = total = 0
    for b in range(batch):
        on = torch.ones(keys, dtype=torch.bool, device="cuda")
        add = torch.zeros(keys, dtype=torch.float64, device="cuda")
        if "key_mask" in mask:
            on, add = counts_of(mask["key_mask"][b])
        if "key_lengths" in mask:
            on = on & (torch.arange(keys, device="cuda") < mask["key_lengths"][b])
        for h in picked:
            g = h // (heads // kv_heads)
            qq, kk, vv = q[b, rows, h].double(), k[b, on, g].double(), v[b, on, g].double()
            n, m = vv.shape[0], add[on]
            s = scale * (qq @ kk.t()) + m
            off = scale * (width + 4) * V * (qq.abs() @ kk.abs().t()) + 4 * V * (s.abs() + m.abs())
            order = s.sort(-1, descending=True)
            gap = order.values[:, 0] - (order.values[:, 1] if n > 1 else -math.inf)
            clear = gap > 2 * off.amax(-1) + 40
            best, most = vv[order.indices[:, 0]], vv.abs().amax(0)
            o = got[b, rows, h].double()
            assert torch.isfinite(o).all()
            d = (o - best).abs() - (u * best.abs() + 2 * n * math.exp(-40) * most + 2.0 ** -130)
            assert (d[clear] <= 0).all()
            slack = (2 * u + 2 * n * V + 2.0 ** -17) * most
            assert (o >= vv.amin(0) - slack).all() and (o <= vv.amax(0) + slack).all()
            single, total = single + int(clear.sum()), total + clear.numel()
    return single, total


# scores of about 2^12, 2^19, 2^22, 2^24, 2^28, 2^33, 2^60 and 2^100 with queries and states of about one
@pytest.mark.parametrize("scale", [300.0, 4e4, 3e5, 1.1e6, 1e7, 1e8, 0.7e17, 1e29])
@pytest.mark.parametrize("size", FORMS, ids=str)
def test_large_scales(pkg, dev, size, scale):
    for dtype in (torch.bfloat16, torch.float16):
        q, k, v = inputs(*size, dtype)
        for kind in ("none", "lengths", "bool", "addends"):
            mask = masked(kind, size[0], size[2])
            single, total = compare(pkg.cross_attention(q, k, v, scale=scale, **mask), q, k, v, size, scale, mask)
            assert single > total // 2, (single, total)   # (most rows have one state that wins by more than the roundings)


@pytest.mark.parametrize("size", FORMS, ids=str)
def test_large_heads(pkg, dev, size):
    """The default scale, over queries and states that are large themselves."""
    for dtype, std in ((torch.bfloat16, 3e4), (torch.bfloat16, 1e9), (torch.bfloat16, 1e17), (torch.float16, 700.0), (torch.float16, 7000.0)):
        q, k, v = inputs(*size, torch.float32, std=1.0)
        q, k, v = (q * std).to(dtype), (k * std).to(dtype), v.to(dtype)
        for kind in ("none", "bool", "addends"):
            mask = masked(kind, size[0], size[2])
            single, total = compare(pkg.cross_attention(q, k, v, **mask), q, k, v, size, None, mask)
            assert single > total // 2, (single, total)


@pytest.mark.parametrize("dtype, value", [(torch.bfloat16, 3e4), (torch.bfloat16, 1e5), (torch.bfloat16, -1.3e15), (torch.float16, 7000.0), (torch.float16, 30000.0), (torch.float16, -1234.0)])
@pytest.mark.parametrize("size", FORMS, ids=str)
def test_equal_large_scores(pkg, dev, size, dtype, value):
    """Either sign: the result is the mean of the values that count."""
    q, k, v = inputs(*size, dtype)
    rows, picked = some(size)
    u = torch.finfo(dtype).eps / 2
    for sign in (1.0, -1.0):
        for kind in ("none", "lengths", "bool", "addends"):
            mask = masked(kind, size[0], size[2])
            got = pkg.cross_attention(torch.full_like(q, sign * value), torch.full_like(k, abs(value)), v, **mask)
            for b in range(size[0]):
                on = torch.ones(size[2], dtype=torch.bool, device="cuda")
                if "key_mask" in mask:
                    on = counts_of(mask["key_mask"][b])[0]
                if "key_lengths" in mask:
                    on = on & (torch.arange(size[2], device="cuda") < mask["key_lengths"][b])
                for h in picked:
                    vv = v[b, on, h // (size[3] // size[4])].double()
                    mean, n = vv.mean(0), vv.shape[0]
                    bound = (u + 2.0 ** -21 + 2 * n * V + 2.0 ** -17) * (vv.abs().mean(0) + mean.abs()) + u * mean.abs()
                    if dtype == torch.float16:   # (weights of one at the least, rounded to steps of 2^-24 below 2^-14)
                        bound = bound + 2.0 ** -24 * vv.abs().amax(0)
                    assert ((got[b, rows, h].double() - mean).abs() <= bound).all(), (kind, sign, b, h)


def test_scores_that_pass_the_bound_on_the_way(pkg, dev):
    """Rows that begin with small scores and end with large ones, or the other way, beside rows that stay small: the large one wins, the small rows are as without them."""
    for dtype in (torch.bfloat16, torch.float16):
        for size in ((1, 40, 700, 2, 2, 64), (1, 1, 3000, 2, 2, 64), (1, 700, 900, 8, 8, 128)):
            q, k, v = inputs(*size, dtype)
            for at in (0, size[2] // 2, size[2] - 1):
                kk, qq = k.clone(), q.clone()
                kk[:, at, :, 0] = 27000.0
                qq[..., 0] = 0.0
                small = pkg.cross_attention(qq, kk, v)
                qq[:, ::3, :, 0] = 23000.0       # scores of 6e8 / 8 and more, no powers of two
                single, total = compare(pkg.cross_attention(qq, kk, v), qq, kk, v, size, None, {})
                assert single >= total // 3
                got = pkg.cross_attention(qq, kk, v)
                rest = torch.arange(size[1], device="cuda") % 3 != 0
                # with every score close to the others the two ways of forming the exponent differ by its roundings only
                d = (got[:, rest].double() - small[:, rest].double()).abs()
                assert (d <= 2 * torch.finfo(dtype).eps * v.abs().max().double()).all()


@pytest.mark.parametrize("scale", [0.7, 1.0, 2.0, 3.0, 4.6, 5.5, 7.0])
@pytest.mark.parametrize("size", [(1, 3, 300, 2, 2, 64), (1, 1, 3000, 2, 2, 64), (1, 700, 300, 8, 8, 128)], ids=str)
def test_scores_a_step_of_binary32_apart(pkg, dev, size, scale):
    """Scores 2^24 and the next larger ones, which the products give exactly: the steps between them are the formula's, whatever tile they are in.  Only the weights'
    own roundings remain: u and 2^-21 of each, binary16's fixed step of 2^-24 beside a largest of one or more, n sums of each."""
    for dtype in (torch.bfloat16, torch.float16):
        q, k, v = inputs(*size, dtype)
        u, n = torch.finfo(dtype).eps / 2, size[2]
        q.zero_(), k.zero_()
        q[..., 0], q[..., 1] = 4096.0, 1.0
        for steps in ((1,), (2, 1), (1, 2, 3, 4), (7, 6, 5)):
            k.zero_()
            k[..., 0] = 4096.0
            for i, step in enumerate(steps):
                k[:, (i + 1) * n // (len(steps) + 1), :, 1] = 2.0 * step
            w = torch.softmax(scale * k[0, :, 0, 1].double(), 0)
            got = pkg.cross_attention(q, k, v, scale=scale)
            for h in range(size[3]):
                vv = v[0, :, h].double()
                o, a = w @ vv, w @ vv.abs()
                bound = (u + 2.0 ** -21 + 2 * n * V + 2.0 ** -17) * (a + o.abs()) + u * o.abs() + (2.0 ** -24 * n * vv.abs().amax() if dtype == torch.float16 else 0.0)
                assert ((got[0, :, h].double() - o).abs() <= bound).all(), (dtype, steps, h)


def test_scores_without_a_maximum_beside_far_ones(pkg, dev):
    """Rows whose scores are all -inf, or no numbers, in one wave with rows near and far: zeros, NaN, and the others as they are without them."""
    for dtype, size in ((torch.bfloat16, (1, 40, 700, 2, 2, 64)), (torch.bfloat16, (1, 700, 300, 8, 8, 128)), (torch.bfloat16, (1, 5, 3000, 2, 2, 64))):
        q, k, v = inputs(*size, dtype)
        k[..., 0] = 2.0 ** 64
        q[..., 0] = 0.0
        for far in (0.0, 3e5):
            q[:, 2::5, :, 1] = far
            want = pkg.cross_attention(q, k, v)
            compare(want, q, k, v, size, None, {})
            bad = q.clone()
            bad[:, 1::5] = 0.0
            bad[:, 1::5, :, 0] = -2.0 ** 64
            got = pkg.cross_attention(bad, k, v)
            rest = torch.arange(size[1], device="cuda") % 5 != 1
            assert torch.equal(got[:, rest], want[:, rest]) and not got[:, ~rest].any()
            bad[:, 1::5, :, 0] = math.nan
            got = pkg.cross_attention(bad, k, v)
            assert torch.equal(got[:, rest], want[:, rest]) and torch.isnan(got[:, ~rest]).all()
            bad[:, 1::5, :, 0] = 2.0 ** 64   # +inf: the formula has no value
            assert torch.isnan(pkg.cross_attention(bad, k, v)[:, ~rest]).all()


@pytest.mark.parametrize("kind, large", [(torch.float32, 3.3e38), (torch.float32, 2.4e38), (torch.bfloat16, 3.3e38), (torch.bfloat16, 2.4e38), (torch.float16, 65504.0)])
@pytest.mark.parametrize("size", [(2, 3, 300, 2, 2, 128), (1, 1, 3000, 4, 2, 72), (1, 700, 333, 8, 8, 128), (1, 300, 4000, 1, 1, 128)], ids=str)
def test_addends_at_the_ends_of_their_type(pkg, dev, size, kind, large):
    """A state whose finite addend is far above the others' is the result, bit for bit; below all of them it has no part; one for all states changes nothing but by
    the roundings of sums of that size, which leave the result within the values."""
    batch, keys = size[0], size[2]
    for dtype in (torch.bfloat16, torch.float16):
        q, k, v = inputs(*size, dtype)
        picked = v[:, 77].repeat_interleave(size[3] // size[4], 1)[:, None]
        near = torch.finfo(kind).max if kind == torch.float16 else large
        m = torch.zeros(batch, keys, dtype=kind, device="cuda")
        m[:, 77] = near
        assert torch.equal(pkg.cross_attention(q, k, v, key_mask=m), picked.expand_as(q)), "above zeros"
        m.fill_(-0.99 * near)
        m[:, 77] = -0.9 * near
        assert torch.equal(pkg.cross_attention(q, k, v, key_mask=m), picked.expand_as(q)), "above others as low"
        m.fill_(0.9 * near)
        m[:, 77] = near
        assert torch.equal(pkg.cross_attention(q, k, v, key_mask=m), picked.expand_as(q)), "above others as high"
        m.zero_()
        m[:, 77] = -0.99 * near
        off = torch.arange(keys, device="cuda") != 77
        compared = pkg.cross_attention(q, k, v, key_mask=m)
        assert torch.equal(compared, pkg.cross_attention(q, k, v, key_mask=torch.where(off, torch.zeros_like(m), -math.inf))), "below all"
        u = torch.finfo(dtype).eps / 2
        for every in (0.97 * near, -0.97 * near):
            got = pkg.cross_attention(q, k, v, key_mask=torch.full_like(m, every)).double()
            assert torch.isfinite(got).all()
            wide = v.double().repeat_interleave(size[3] // size[4], 2)
            slack = (2 * u + 2 * keys * V + 2.0 ** -17) * wide.abs().amax(1, keepdim=True)
            assert (got >= wide.amin(1, keepdim=True) - slack).all() and (got <= wide.amax(1, keepdim=True) + slack).all()
        m.fill_(-math.inf)
        m[:, 5], m[:, 200] = math.inf, 0.0      # an infinite addend has no weight that is a number
        assert torch.isnan(pkg.cross_attention(q, k, v, key_mask=m)).all()


@pytest.mark.parametrize("queries, keys", [(200, 300), (3, 300), (1, 1), (1, 3000), (700, 333)])
def test_values_at_the_ends_of_bfloat16(pkg, dev, queries, keys):
    """Values of 2^127 / keys whose weights grow by just less than the running maximum lets them, equal ones (their mean is themselves, but for keys roundings of
    2^-24 in two sums and 2^-8 at the end); and values around 2^-122, whose products with weights reach below binary32's normal numbers."""
    q, k, v = inputs(2, queries, keys, 4, 2, 64, torch.bfloat16)
    on = torch.arange(keys, device="cuda").expand(2, -1) % 3 != 1
    for mask in (None, on, torch.where(on, 0.25, -math.inf)):
        grow = torch.linspace(0.0, 1.0, keys, device="cuda")[None, :, None, None] * 5.0
        large = torch.full_like(v, 2.0 ** 127 / 2 ** math.ceil(math.log2(keys)))
        got = pkg.cross_attention(torch.ones_like(q), (grow / 8).expand(2, -1, 2, 64).bfloat16(), large, key_mask=mask)
        off = ((got.double() / large[0, 0, 0, 0].double()) - 1.0).abs().max().item()
        assert off <= 2.0 ** -8 + 2 * keys * V + 2.0 ** -20, off
        tiny = (v.double() * 2.0 ** -122).bfloat16()
        check(pkg.cross_attention(q, k, tiny, key_mask=mask), expected(q, k, tiny, key_mask=mask))


@pytest.mark.parametrize("size", [(1, 3, 300, 2, 2, 64), (1, 1, 3000, 2, 2, 64), (1, 700, 300, 8, 8, 128)], ids=str)
def test_scales_at_the_ends_of_binary32(pkg, dev, size):
    """The largest scale over heads whose products are small, the smallest over ones whose products are large, with scores of about one either way, and of nothing."""
    for scale, std in ((2.0 ** 126, 2.0 ** -61), (2.0 ** 126, 2.0 ** -60), (2.0 ** -126, 2.0 ** 61), (2.0 ** -120, 2.0 ** 58), (2.0 ** -149, 1.0), (2.0 ** -140, 2.0 ** 10)):
        q, k, v = inputs(*size, torch.float32, std=1.0)
        q, k, v = (q * std).bfloat16(), (k * std).bfloat16(), v.bfloat16()
        for mask in ({}, masked("bool", size[0], size[2]), {"key_mask": torch.linspace(-1, 1, size[2], device="cuda").expand(size[0], -1)}):
            check(pkg.cross_attention(q, k, v, scale=scale, **mask), expected(q, k, v, scale=scale, **mask), (scale, std))
