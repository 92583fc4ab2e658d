"""Block norms of more rows than a launch has workgroups for (fewer than 2^32 threads): the rows at the ends and on both sides of a border
between launches are those of a call with these rows alone, bit for bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,K,border", [((1 << 24) + 70, 4, 1 << 23), ((1 << 26) + 6, 16, 1 << 25)])   # a workgroup to a row, four rows to one
def test_rows_in_several_launches(pkg, dev, rows, K, border):
    g = torch.Generator(device="cuda").manual_seed(K)
    y = torch.randn(rows, K, generator=g, device=dev, dtype=torch.bfloat16)
    w, gate = torch.rand(K, generator=g, device=dev) + 0.5, torch.randn(K, generator=g, device=dev).bfloat16()
    ops = dict(post_norm="rms", post_weight=w, gate=gate, gate_tanh=True, pre_norm="layer", residual_scale=0.5)
    x, h = pkg.block_norm(y, y, **ops)
    for first in (0, border - 200, 2 * border - 200, rows - 400):
        part = slice(first, min(first + 400, rows))
        want_x, want_h = pkg.block_norm(y[part], y[part], **ops)
        assert torch.equal(x[part], want_x) and torch.equal(h[part], want_h), f"rows from {first}"
    assert torch.isfinite(x.sum()) and torch.isfinite(h.sum())


def test_int8_rows_in_several_launches(pkg, L, dev):
    rows, K = (1 << 24) + 70, 3
    y = torch.randn(rows, K, generator=torch.Generator(device="cuda").manual_seed(K), device=dev, dtype=torch.float16)
    x, q, s = L.block_norm(y, y, pre_norm="rms", quantise=True)
    for first in (0, (1 << 23) - 200, (1 << 24) - 200, rows - 400):
        part = slice(first, min(first + 400, rows))
        want_x, want_h = pkg.block_norm(y[part], y[part], pre_norm="rms")
        want_q, want_s = L.quant_rowwise(want_h)
        assert torch.equal(x[part], want_x) and torch.equal(q[part], want_q) and torch.equal(s[part], want_s), f"rows from {first}"


def test_vectors_of_a_row_each_in_several_launches(pkg, dev):
    """The number of a row's gate counts from the first launch's first row."""
    rows, K = (1 << 24) + 70, 4
    g = torch.Generator(device="cuda").manual_seed(5)
    y, gate = (torch.randn(rows, K, generator=g, device=dev, dtype=torch.bfloat16) for _ in range(2))
    x, _ = pkg.block_norm(y, y, gate=gate)
    for first in (0, (1 << 23) - 200, (1 << 24) - 200, rows - 400):
        part = slice(first, min(first + 400, rows))
        assert torch.equal(x[part], pkg.block_norm(y[part], y[part], gate=gate[part])[0]), f"rows from {first}"
