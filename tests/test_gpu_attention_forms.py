"""Every form of the attention (which sizes reach which is asked of the library): masks, what masked states hold, and layouts, for every width of a kernel."""
import math

import pytest
import torch

from attention_forms import SIZES, form_of
from test_gpu_attention import KINDS, check, counts_of, expected, inputs, masks

pytestmark = pytest.mark.gpu

ALL = [(form, size) for form, sizes in SIZES.items() for size in sizes]


def some(size):
    """Rows and heads that are compared with the formula: all, or a part of a large call's, from all its waves and its last rows."""
    batch, queries, keys, heads, kv_heads, width = size
    if queries * heads < 20000:
        return torch.arange(queries, device="cuda"), torch.arange(heads, device="cuda")
    return torch.cat([torch.arange(a, a + 40, device="cuda") for a in (0, 130, 236, queries // 2, queries - 40)]), torch.tensor([0, heads // 2 + 1, heads - 1], device="cuda")


def compare(got, q, k, v, size, what="", **mask):
    rows, heads = some(size)
    if len(heads) < size[3]:   # (such calls have as many heads of states)
        got, q, k, v = got[:, rows][:, :, heads], q[:, rows][:, :, heads], k[:, :, heads], v[:, :, heads]
    check(got.contiguous(), expected(q, k, v, **mask), what)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("form, size", ALL, ids=str)
def test_masks_in_every_form(pkg, L, dev, form, size, dtype):
    """Against the formula under every mask; and what the states that do not count hold reaches nothing."""
    assert form_of(L, size)[0] == form
    q, k, v = inputs(*size, dtype)
    compare(pkg.cross_attention(q, k, v), q, k, v, size)
    for kind in KINDS if form != "eight" else ("lengths", "bool", "sparse", "both", "added", "added32", "added infinities"):
        mask = masks(kind, size[0], size[2], dtype)
        got = pkg.cross_attention(q, k, v, **mask)
        compare(got, q, k, v, size, kind, **mask)
        on = torch.ones(size[0], size[2], dtype=torch.bool, device="cuda")
        if "key_mask" in mask:
            on &= counts_of(mask["key_mask"])[0]
        if "key_lengths" in mask:
            on &= torch.arange(size[2], device="cuda") < mask["key_lengths"][:, None]
        for bad in (math.nan, math.inf):
            kb, vb = (torch.where(on[:, :, None, None], t, torch.full((), bad, dtype=dtype, device="cuda")) for t in (k, v))
            assert torch.equal(pkg.cross_attention(q, kb, vb, **mask), got), (kind, bad)
        assert not got[~on.any(1)].any()


@pytest.mark.parametrize("form, size", ALL, ids=str)
def test_layouts_in_every_form(pkg, L, dev, form, size):
    """Views of fused projections, heads in front of tokens, elements at odd addresses, expanded: as their copies, bit for bit."""
    assert form_of(L, size)[0] == form
    width = size[-1]
    for dtype in (torch.bfloat16, torch.float16):
        q, k, v = inputs(*size, dtype)
        want = pkg.cross_attention(q, k, v)
        both = torch.stack((k, v), 2)
        assert torch.equal(pkg.cross_attention(q, both[:, :, 0], both[:, :, 1]), want)
        assert torch.equal(pkg.cross_attention(*(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))), want)
        assert torch.equal(pkg.cross_attention(*(torch.cat((t, t), -1)[..., :width] for t in (q, k, v))), want)
        for off in (1, 4):
            assert torch.equal(pkg.cross_attention(*(torch.empty(t.numel() + off, dtype=dtype, device="cuda")[off:].view(t.shape).copy_(t) for t in (q, k, v))), want), off
        one = [t[:1].expand(size[0], -1, -1, -1) for t in (q, k, v)]
        assert torch.equal(pkg.cross_attention(*one)[-1], want[0])
        mask = masks("bool", size[0], size[2], dtype)
        masked = pkg.cross_attention(q, k, v, **mask)
        assert torch.equal(pkg.cross_attention(q, both[:, :, 0], both[:, :, 1], **mask), masked)


@pytest.mark.parametrize("form, size", [(form, size) for form, size in ALL if size[-1] in (64, 128, 200, 37)], ids=str)
def test_calls_of_every_form_agree_bit_for_bit(pkg, L, dev, form, size):
    """Twice, on another stream at the same time, and captured and replayed between the program's own calls."""
    assert form_of(L, size)[0] == form
    q, k, v = inputs(*size, torch.bfloat16)
    lengths = torch.full((size[0],), size[2], dtype=torch.int32, device="cuda")
    call = lambda: pkg.cross_attention(q, k, v, key_lengths=lengths)  # noqa: E731
    want, side = call(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    both = []
    for _ in range(3):
        with torch.cuda.stream(side):
            both.append(call())
        both.append(call())
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(o, want) for o in both)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for n in (size[2], size[2] // 2, 1, 0):
        lengths.fill_(n)
        eager = call()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), n


@pytest.mark.parametrize("size", [(1, 1, 1536, 1, 1, 37), (1, 1, 4097, 1, 1, 37), (1, 3, 5000, 1, 1, 33), (1, 5, 3000, 3, 1, 199)], ids=str)
def test_copies_behind_an_odd_number_of_split_rows(pkg, dev, size):
    for dtype in (torch.bfloat16, torch.float16):
        q, k, v = inputs(*size, dtype)
        got = pkg.cross_attention(q, k, v)
        check(got, expected(q, k, v))
        wide = -(-size[-1] // 8) * 8
        whole = [torch.nn.functional.pad(t, (0, wide - size[-1])) for t in (q, k, v)]
        assert torch.equal(pkg.cross_attention(*whole, scale=size[-1] ** -0.5)[..., :size[-1]], got)


def test_copies_of_more_heads_than_a_tile_reaches_over(pkg, L, dev):
    """Odd widths of so many heads that 63 tokens of all of them are more than 2^31 bytes: tiles of 64 states reach over them by 32-bit offsets."""
    size = (1, 33, 64, 67000, 67000, 255)
    assert form_of(L, size)[0] == "together" and 63 * 67000 * 256 * 2 > 1 << 31
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.empty(1, n, 67000, 255, dtype=torch.bfloat16, device="cuda").normal_(generator=g) for n in (33, 64, 64))
    got = pkg.cross_attention(q, k, v)
    for heads in (slice(0, 2), slice(40000, 40002), slice(66998, 67000)):
        part = [t[:, :, heads] for t in (q, k, v)]
        check(got[:, :, heads].contiguous(), expected(*part))
