"""Attention over an encoder's states against the formula in 64 bits, element by element.

Bounds, with v = 2^-24, u half a step of the type, w_j the weights (their sum 1), A = sum w_j |v_j|:
    scores    a product of D terms in binary32: D v of sum |q_e k_e|, times the scale; two roundings behind it.  ds = (D + 4) v max_j scale sum |q_e k_e|
              + 4 v max_j (|s_j| + |m_j|), the larger one of a row for all its weights
    weights   e^s by the hardware's exp2, off by 2^-22 of itself besides e^ds - 1 < 2 ds, and rounded to the type: u.  Binary16 has no more than a fixed
              step below 2^-14: the weights are kept at 2^6 to 2^14 for the largest, so that is 2^-31 of it and 2^-31 max|v| n of a result
    sums      of weights and of their products with v, n terms in binary32 and rescaled a few times: 2 (n v + 2^-18) of A and of |o|
    result    rounded once: u
so |error| <= (u + 2^-21 + 2 ds + 2 n v + 2^-17) (A + |o|) + u |o| + (binary16: 2^-31 n max|v|)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

V = 2.0 ** -24


def counts_of(mask):
    """(which states count, their addends) of a mask."""
    if mask.dtype == torch.bool:
        return mask, torch.zeros(mask.shape, dtype=torch.float64, device=mask.device)
    on = mask > torch.finfo(mask.dtype).min
    return on, torch.where(on, mask.double(), 0.0)


def expected(q, k, v, key_lengths=None, key_mask=None, scale=None):
    """(value, bound) in float64; rows without states are zeros."""
    batch, queries, heads, width = q.shape
    keys, kv_heads = k.shape[1:3]
    scale = width ** -0.5 if scale is None else scale
    f = torch.finfo(q.dtype)
    u = f.eps / 2
    value, bound = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    for b in range(batch):
        on, add = counts_of(key_mask[b]) if key_mask is not None else (torch.ones(keys, dtype=torch.bool, device=q.device), torch.zeros(keys, dtype=torch.float64, device=q.device))
        if key_lengths is not None:
            on = on & (torch.arange(keys, device=q.device) < key_lengths[b])
        n = int(on.sum())
        if n == 0:
            continue
        m = add[on]
        for h in range(heads):
            g = h // (heads // kv_heads)
            qq, kk, vv = q[b, :, h].double(), k[b, on, g].double(), v[b, on, g].double()
            s = scale * (qq @ kk.t()) + m
            w = torch.softmax(s, -1)
            o, A = w @ vv, w @ vv.abs()
            ds = (width + 4) * V * scale * (qq.abs() @ kk.abs().t()).amax(-1, keepdim=True) + 4 * V * (s.abs() + m.abs()).amax(-1, keepdim=True)
            value[b, :, h] = o
            bound[b, :, h] = (u + 2.0 ** -21 + 2 * ds + 2 * n * V + 2.0 ** -17) * (A + o.abs()) + u * o.abs() + f.smallest_normal * f.eps
            if q.dtype == torch.float16:
                bound[b, :, h] += 2.0 ** -31 * n * vv.abs().amax()
    return value, bound


def check(got, want, what=""):
    value, bound = want
    assert got.shape == value.shape and got.is_contiguous() and torch.isfinite(got.float()).all(), what
    off = (got.double() - value).abs()
    worst = torch.where(bound > 0, off / bound.clamp_min(1e-300), torch.where(off > 0, math.inf, 0.0)).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} of the bound"


def inputs(batch, queries, keys, heads, kv_heads, width, dtype, seed=0, std=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed + queries + keys + width)
    q, k, v = (torch.randn(*s, generator=g, device="cuda") * std for s in ((batch, queries, heads, width), (batch, keys, kv_heads, width), (batch, keys, kv_heads, width)))
    v = v + 0.5
    return q.to(dtype), k.to(dtype), v.to(dtype)


# (batch, queries, keys, heads, kv heads, width)
SIZES = [(1, 1, 1, 1, 1, 1), (1, 1, 1, 1, 1, 64), (2, 1, 3, 2, 1, 8), (1, 3, 31, 2, 2, 33), (1, 5, 32, 3, 3, 64), (2, 33, 33, 4, 2, 40), (1, 7, 63, 2, 2, 72), (1, 64, 64, 2, 2, 128),
         (1, 129, 65, 2, 1, 128), (3, 77, 100, 5, 5, 96), (1, 128, 127, 2, 2, 80), (1, 130, 128, 2, 2, 128), (2, 257, 333, 4, 4, 64), (1, 300, 512, 6, 6, 128), (1, 200, 1000, 2, 2, 256),
         (1, 70, 200, 3, 3, 160), (1, 65, 129, 2, 2, 192), (1, 66, 90, 2, 2, 200), (1, 40, 150, 2, 2, 255), (1, 1, 4097, 8, 8, 64), (1, 1, 5000, 32, 8, 128), (2, 2, 3000, 12, 3, 72),
         (1, 1, 2500, 4, 4, 256), (1, 4, 2049, 6, 2, 37), (1, 1000, 77, 3, 3, 128), (1, 513, 2050, 2, 2, 128), (4, 1, 257, 16, 16, 64), (1, 16, 700, 40, 1, 64), (1, 33, 1, 4, 4, 128),
         (1, 1, 20000, 1, 1, 128), (300, 3, 20, 2, 2, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_against_the_formula(pkg, dev, size, dtype):
    q, k, v = inputs(*size, dtype)
    check(pkg.cross_attention(q, k, v), expected(q, k, v))


@pytest.mark.parametrize("scale", [1e-30, 0.01, 1.0, 3.0])
def test_scales(pkg, dev, scale):
    """From weights that are all alike to ones that leave a single state."""
    q, k, v = inputs(1, 70, 300, 2, 2, 128, torch.bfloat16)
    check(pkg.cross_attention(q, k, v, scale=scale), expected(q, k, v, scale=scale))


def masks(kind, batch, keys, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + keys)
    on = torch.rand(batch, keys, generator=g, device="cuda") < 0.6
    if kind == "lengths":
        given = torch.tensor([keys, keys // 2, 0, -5, 10 ** 6, 1, 64, 63][:batch] * (batch // 8 + 1), device="cuda")[:batch]
        return {"key_lengths": given}
    if kind == "lengths32":
        return {"key_lengths": masks("lengths", batch, keys, dtype)["key_lengths"].flip(0).int()}
    if kind == "bool":
        return {"key_mask": on}
    if kind == "sparse":      # whole tiles without a state, a row of the batch without any
        on = torch.zeros(batch, keys, dtype=torch.bool, device="cuda")
        on[:, keys // 3] = True
        on[0, :] = False
        on[-1, -1] = True
        return {"key_mask": on}
    if kind == "strided":
        wide = torch.zeros(keys, batch * 3, dtype=torch.bool, device="cuda")
        wide[:, ::3] = on.t()
        return {"key_mask": wide.t()[::3]}
    if kind == "one for all":
        return {"key_mask": on[:1].expand(batch, -1)}
    if kind == "both":
        return {"key_mask": on, "key_lengths": masks("lengths", batch, keys, dtype)["key_lengths"]}
    add = torch.randn(batch, keys, generator=g, device="cuda") * 2
    kinds = {"added": dtype, "added32": torch.float32, "added other": torch.float16 if dtype == torch.bfloat16 else torch.bfloat16, "added infinities": dtype}
    add = add.to(kinds[kind])
    off = torch.full((), -math.inf if kind == "added infinities" else torch.finfo(add.dtype).min, dtype=add.dtype, device="cuda")
    add = torch.where(on, add, off)
    add[0] = off
    return {"key_mask": add}


KINDS = ["lengths", "lengths32", "bool", "sparse", "strided", "one for all", "both", "added", "added32", "added other", "added infinities"]
MASKED = [(3, 40, 130, 4, 2, 128), (2, 1, 500, 3, 3, 64), (5, 130, 77, 2, 2, 72), (2, 300, 1000, 2, 2, 128), (8, 3, 2100, 8, 2, 96), (2, 34, 70, 2, 2, 33), (3, 1, 3000, 4, 4, 256), (2, 150, 200, 1, 1, 130)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", MASKED, ids=str)
def test_masks(pkg, dev, size, kind):
    for dtype in (torch.bfloat16, torch.float16):
        q, k, v = inputs(*size, dtype)
        mask = masks(kind, size[0], size[2], dtype)
        got = pkg.cross_attention(q, k, v, **mask)
        check(got, expected(q, k, v, **mask), kind)
        # what does not count is not looked at
        on = torch.ones(size[0], size[2], dtype=torch.bool, device="cuda")
        if "key_mask" in mask:
            on &= counts_of(mask["key_mask"])[0]
        if "key_lengths" in mask:
            on &= torch.arange(size[2], device="cuda") < mask["key_lengths"][:, None]
        for bad in (math.nan, math.inf):
            kb, vb = (torch.where(on[:, :, None, None], t, torch.full((), bad, dtype=dtype, device="cuda")) for t in (k, v))
            assert torch.equal(pkg.cross_attention(q, kb, vb, **mask), got), (kind, bad)
        empty = ~on.any(1)
        assert not got[empty].any()


@pytest.mark.parametrize("size", [(2, 130, 200, 4, 2, 128), (2, 1, 900, 4, 2, 128), (2, 40, 100, 4, 4, 72), (2, 33, 70, 2, 2, 37)], ids=str)
def test_strides(pkg, dev, size):
    """Views of fused projections, heads in front of tokens, expanded and odd ones: as their copies, bit for bit."""
    batch, queries, keys, heads, kv_heads, width = size
    for dtype in (torch.bfloat16, torch.float16):
        q, k, v = inputs(*size, dtype)
        want = pkg.cross_attention(q, k, v)
        check(want, expected(q, k, v))
        both = torch.stack((k, v), 2)
        assert torch.equal(pkg.cross_attention(q, both[:, :, 0], both[:, :, 1]), want)
        ahead = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
        assert torch.equal(pkg.cross_attention(*ahead), want)
        wide = [torch.cat((t, t), -1)[..., :width] for t in (q, k, v)]
        assert torch.equal(pkg.cross_attention(*wide), want)
        last = [t.transpose(1, 3).contiguous().transpose(1, 3) for t in (q, k, v)]
        assert torch.equal(pkg.cross_attention(*last), want)
        for off in (1, 3, 4):   # first elements at odd places: other loads, the same products
            moved = [torch.empty(t.numel() + off, dtype=dtype, device="cuda")[off:].view(t.shape).copy_(t) for t in (q, k, v)]
            assert torch.equal(pkg.cross_attention(*moved), want), off
        assert torch.equal(pkg.cross_attention(q[:1].expand(batch, -1, -1, -1), k[:1].expand(batch, -1, -1, -1), v[:1].expand(batch, -1, -1, -1))[-1], want[0])
        check(pkg.cross_attention(q, k[:, :1].expand(-1, keys, -1, -1), v), expected(q, k[:, :1].expand(-1, keys, -1, -1), v))


def test_scores_that_grow_and_fall(pkg, dev):
    """States in order of their scores, either way, far apart: the running maximum moves with every tile, or never again."""
    for dtype in (torch.bfloat16, torch.float16):
        for queries, keys in ((40, 700), (1, 3000), (200, 300)):
            q, k, v = inputs(1, queries, keys, 2, 2, 64, dtype)
            q = q.abs() + 0.5
            slope = torch.linspace(-3, 3, keys, device="cuda")[None, :, None, None]
            for s in (slope, -slope, torch.where(torch.arange(keys, device="cuda")[None, :, None, None] == keys // 2, 4.0, -4.0)):
                kk = (k * 0.1 + s).to(dtype)
                check(pkg.cross_attention(q, kk, v), expected(q, kk, v))


def test_addends_that_are_large_but_count(pkg, dev):
    q, k, v = inputs(2, 50, 200, 2, 2, 128, torch.bfloat16)
    for dtype, big in ((torch.float32, -1e6), (torch.bfloat16, -2.0 ** 20), (torch.float16, -60000.0), (torch.float32, 1e6)):
        m = torch.zeros(2, 200, dtype=dtype, device="cuda")
        m[:, 50:] = big
        check(pkg.cross_attention(q, k, v, key_mask=m), expected(q, k, v, key_mask=m))
        check(pkg.cross_attention(q, k, v, key_mask=torch.full_like(m, big)), expected(q, k, v, key_mask=torch.full_like(m, big)))


def test_an_addend_that_is_no_number_ends_its_batch_only(pkg, dev):
    q, k, v = inputs(2, 50, 200, 2, 2, 128, torch.bfloat16)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        m = torch.zeros(2, 200, dtype=dtype, device="cuda")
        want = pkg.cross_attention(q, k, v, key_mask=m)
        m[1, 77] = math.nan
        got = pkg.cross_attention(q, k, v, key_mask=m)
        assert torch.equal(got[0], want[0]) and torch.isnan(got[1]).all()


def test_values_that_are_not_finite_stay_in_their_rows(pkg, dev):
    """A query that is no number ends itself, a state that counts ends the queries of its batch and head."""
    for queries, keys in ((200, 300), (3, 300), (1, 3000)):
        q, k, v = inputs(2, queries, keys, 2, 2, 64, torch.bfloat16)
        want = pkg.cross_attention(q, k, v)
        bad = q.clone()
        bad[0, queries // 2, 1, 5] = math.nan
        got = pkg.cross_attention(bad, k, v)
        same = torch.ones(q.shape[:3], dtype=torch.bool, device="cuda")
        same[0, queries // 2, 1] = False
        assert torch.equal(got[same], want[same]) and torch.isnan(got[~same]).all()
        bad = v.clone()
        bad[1, keys - 1, 0, 3] = math.inf
        got = pkg.cross_attention(q, k, bad)
        same = torch.ones(q.shape, dtype=torch.bool, device="cuda")
        same[1, :, 0, 3] = False
        assert torch.equal(got[same], want[same]) and not torch.isfinite(got[~same].float()).any()


@pytest.mark.parametrize("queries, keys", [(200, 300), (3, 300), (1, 3000)])
def test_scores_and_values_at_the_ends_of_binary32(pkg, dev, queries, keys):
    q, k, v = inputs(2, queries, keys, 2, 2, 64, torch.bfloat16)
    some = torch.arange(keys, device="cuda").expand(2, -1) % 3 > 0
    for mask in (None, some, some.float() - 1.0):
        got = pkg.cross_attention(torch.full_like(q, -2.0 ** 64), torch.full_like(k, 2.0 ** 64), v, key_mask=mask)
        assert torch.equal(got, torch.zeros_like(got))   # (every score is -inf)
        # scores that grow by just less than the running maximum lets them, values as large as the documentation has them: equal ones are their mean
        grow = torch.linspace(0.0, 1.0, keys, device="cuda")[None, :, None, None] * 5.0
        large = torch.full_like(v, 2.0 ** 119 / 2 ** math.ceil(math.log2(keys)))
        got = pkg.cross_attention(torch.ones_like(q), (grow / 8).expand(2, -1, 2, 64).bfloat16(), large, key_mask=mask)
        # sums and weights in binary32 cancel but for keys roundings of 2^-24 each in two sums, the result is rounded by 2^-8
        off = ((got.double() / large[0, 0, 0, 0].double()) - 1.0).abs().max().item()
        assert off <= 2.0 ** -8 + 2 * keys * 2.0 ** -24 + 2.0 ** -20, off


def test_rows_of_nothing(pkg, dev):
    for shape in ((0, 3, 5, 2, 2, 64), (2, 0, 5, 2, 2, 64), (2, 3, 5, 0, 0, 64)):
        q, k, v = inputs(*shape, torch.bfloat16)
        assert pkg.cross_attention(q, k, v).shape == q.shape
    for width in (64, 37, 256):
        for queries in (3, 500):
            q, k, v = inputs(2, queries, 0, 4, 2, width, torch.bfloat16)
            torch.empty_like(q).fill_(7.0)   # (what the result's memory may have held)
            got = pkg.cross_attention(q[..., :], k, v)
            assert got.shape == q.shape and torch.equal(got, torch.zeros_like(q))
    q, k, v = inputs(2, 3, 0, 4, 2, 64, torch.bfloat16)
    assert not pkg.cross_attention(q, k, v, key_mask=torch.zeros(2, 0, dtype=torch.bool, device="cuda"), key_lengths=torch.ones(2, dtype=torch.int64, device="cuda")).any()


def test_states_whose_offsets_pass_32_bits(pkg, dev):
    """Tokens 2 MiB apart: the last ones lie behind 2^31 and 2^32 bytes."""
    space = torch.empty(2200 << 20, dtype=torch.bfloat16, device="cuda")
    q, k, v = inputs(1, 3, 2200, 2, 1, 64, torch.bfloat16)
    far = space.as_strided((1, 2200, 1, 64), (0, 1 << 20, 64, 1))
    far.copy_(k)
    far_v = space[1024:].as_strided((1, 2200, 1, 64), (0, 1 << 20, 64, 1))
    far_v.copy_(v)
    for queries in (3, 200):
        q = inputs(1, queries, 2200, 2, 1, 64, torch.bfloat16)[0]
        assert torch.equal(pkg.cross_attention(q, far, far_v), pkg.cross_attention(q, k, v))
    del space


def test_refusals(pkg, dev):
    q, k, v = inputs(2, 3, 5, 4, 2, 64, torch.bfloat16)
    call = pkg.cross_attention
    for bad in (lambda: call(q[0], k, v), lambda: call(q, k[0], v[0]), lambda: call(q, k, v[:, :4]), lambda: call(q, k[:1], v[:1]), lambda: call(q, k[..., :32], v[..., :32]),
                lambda: call(q[:, :, :3], k, v), lambda: call(q, k[:, :, :0], v[:, :, :0]), lambda: call(q.half(), k, v), lambda: call(q, k, v.half()),
                lambda: call(q.float(), k.float(), v.float()), lambda: call(q, k.cpu(), v), lambda: call(q, k, v, scale=0.0), lambda: call(q, k, v, scale=-1.0),
                lambda: call(q, k, v, scale=math.inf), lambda: call(q, k, v, scale=math.nan), lambda: call(q, k, v, scale=1e39), lambda: call(q, k, v, scale=1e-60), lambda: call(q[..., :0], k[..., :0], v[..., :0]),
                lambda: call(*(torch.zeros(1, 1, 1, 257, device="cuda", dtype=torch.bfloat16) for _ in range(3))),
                lambda: call(q, k, v, key_lengths=torch.ones(3, dtype=torch.int32, device="cuda")), lambda: call(q, k, v, key_lengths=torch.ones(2, device="cuda")),
                lambda: call(q, k, v, key_lengths=torch.ones(2, dtype=torch.int32)), lambda: call(q, k, v, key_mask=torch.ones(2, 4, dtype=torch.bool, device="cuda")),
                lambda: call(q, k, v, key_mask=torch.ones(5, dtype=torch.bool, device="cuda")), lambda: call(q, k, v, key_mask=torch.ones(2, 5, dtype=torch.uint8, device="cuda")),
                lambda: call(q, k, v, key_mask=torch.ones(2, 5, dtype=torch.float64, device="cuda")), lambda: call(q, k, v, key_mask=torch.ones(2, 5, dtype=torch.bool))):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            bad()


@pytest.mark.parametrize("size", [(1, 1, 5000, 8, 2, 128), (2, 200, 300, 4, 4, 64), (1, 300, 4000, 1, 1, 128)], ids=str)
def test_calls_agree_bit_for_bit(pkg, dev, size):
    """Twice, on another stream beside the first, captured and replayed with the program's own calls between, under the compiler."""
    q, k, v = inputs(*size, torch.bfloat16)
    lengths = torch.full((size[0],), size[2], dtype=torch.int32, device="cuda")
    call = lambda: pkg.cross_attention(q, k, v, key_lengths=lengths)  # noqa: E731
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    both = []
    for _ in range(4):
        with torch.cuda.stream(side):
            both.append(call())
        both.append(call())
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(o, want) for o in both)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    for n in (size[2], size[2] // 2, 1, 0):
        lengths.fill_(n)
        eager = call()
        for graph, out in graphs:
            graph.replay()
        again = call()
        torch.cuda.synchronize()
        assert torch.equal(eager, again) and all(torch.equal(out, eager) for _, out in graphs), n
    lengths.fill_(size[2])
    compiled = torch.compile(lambda a: pkg.cross_attention(a, k, v, key_lengths=lengths), backend="eager", fullgraph=True)
    assert torch.equal(compiled(q), want)

