"""Adapters in binary16 whose first product alone leaves the type's range.

t = s A x is an operand of the matrix unit in 16 bits.  The result depends on t B alone, so the range that s and B take of it is
the bank's to choose: a large scale over small second factors, and a small one over large ones, are as good as any other pair.
The bound is the one of test_gpu_adapters.py, and half a step of the smallest numbers, 2^-25, of every t times the largest
element of B as the bank holds it, below 2: ranks * 2^-24."""
import pytest
import torch

from test_gpu_adapters import check, expected, ids_of, layer_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,K,N", [(1, 256, 128), (9, 250, 33), (64, 256, 192), (100, 200, 101), (300, 1024, 384), (700, 512, 200), (700, 515, 201), (1100, 512, 2304)])
@pytest.mark.parametrize("up_size,scale", [(2.0 ** -12, 2.0 ** 19), (200.0, 1e-6), (2.0 ** -18, 3e7), (5e-3, 0.7)])
def test_scales_and_factors_far_from_one(pkg, dev, rows, K, N, up_size, scale):
    ranks, dtype = (16, 40, 5), torch.float16
    lin = layer_of(pkg, K, N, dtype, bias=False)
    if scale < 1e-3:
        lin.weight.zero_()   # (the adapters' share alone)
    g = torch.Generator(device="cuda").manual_seed(rows)
    adapters = [((torch.randn(r, K, generator=g, device=dev) * K ** -0.5).to(dtype), (torch.randn(N, r, generator=g, device=dev) * up_size).to(dtype), scale * (1 + i))
                for i, r in enumerate(ranks)]
    x = torch.randn(rows, K, generator=g, device=dev).to(dtype)
    for kind in ("tokens", "runs", "one"):
        ids = ids_of(kind, rows, len(ranks))
        want, bound = expected(pkg, lin, x, adapters, ids)
        check(pkg.forward_adapters(lin, x, pkg.AdapterBank(adapters), ids), want, bound + max(ranks) * 2.0 ** -24, kind)
