"""Adapters in every tile configuration, over long rows, over slices of a few K-tiles and for several layers in every form.  The bound is
the one of test_gpu_adapters.py; every call is made twice and has to repeat itself."""
import ctypes

import pytest
import torch

from test_gpu_adapters import check, expected, factors_of, ids_of, layer_of

pytestmark = pytest.mark.gpu


def run(pkg, dev, layers, adapters, x, ids):
    """forward_adapters of one or several layers against the formula."""
    banks = [pkg.AdapterBank(a, dtype=x.dtype, device=dev) for a in adapters]
    outs = pkg.forward_adapters(layers, x, banks, ids)
    again = pkg.forward_adapters(layers, x, banks, ids)
    for lin, some, y, z in zip(layers, adapters, outs, again):
        check(y, *expected(pkg, lin, x, some, ids))
        assert torch.equal(y, z)


TILES = [((64, 64, 4), 131, 264), ((128, 64, 4), 400, 3000), ((128, 96, 4), 330, 6664), ((128, 128, 4), 140, 12504), ((128, 128, 2), 257, 12504),
         ((256, 96, 3), 270, 11192), ((256, 192, 2), 518, 13160), ((256, 256, 2), 1544, 6928), ((256, 288, 2), 1755, 9224), ((288, 256, 2), 1544, 9224)]


@pytest.mark.parametrize("kind", ["one", "runs", "tokens"])
@pytest.mark.parametrize("ranks", [(20, 32), (8, 40, 160), (64, 16, 48, 128)])
@pytest.mark.parametrize("tile,rows,N", TILES)
def test_every_tile(pkg, L, dev, tile, rows, N, ranks, kind):
    """One adapter in a wave, two where a request ends, and more, of ranks up to one that is taken a part at a time."""
    K, dtype = (128, torch.bfloat16) if len(ranks) == 3 else (208, torch.float16)   # (whole K-tiles, and one that ends inside)
    dims = [ctypes.c_int() for _ in range(3)]
    assert L.lib().i8f_gemm_tile(rows, N, K, *map(ctypes.byref, dims)) == 0 and tuple(v.value for v in dims) == tile
    lin, adapters = layer_of(pkg, K, N, dtype, per_row=len(ranks) != 2), [factors_of(K, N, ranks, dtype, rows)]
    x = torch.randn(rows, K, generator=torch.Generator(device="cuda").manual_seed(rows), device=dev).to(dtype)
    run(pkg, dev, [lin], adapters, x, ids_of(kind, rows, len(ranks)))


@pytest.mark.parametrize("kind", ["tokens", "runs"])
@pytest.mark.parametrize("rows", [3, 40, 300, 700])
@pytest.mark.parametrize("K,dtype,opts", [(5120, torch.bfloat16, {"rotate": True}), (6144, torch.float16, {}), (9216, torch.bfloat16, {}), (12288, torch.float16, {"rotate": True}),
                                          (5003, torch.bfloat16, {}), (8198, torch.float16, {}), (16400, torch.bfloat16, {}), (20011, torch.float16, {})])
def test_rows_of_more_than_4096_columns(pkg, dev, K, dtype, opts, rows, kind):
    """Several trips of a wave over its row, and the quantisers of longer rows beside it, at sizes of every form of the first product."""
    N, ranks = 136, (16, 40, 64)
    x = torch.randn(rows, K, generator=torch.Generator(device="cuda").manual_seed(rows), device=dev).to(dtype)
    run(pkg, dev, [layer_of(pkg, K, N, dtype, **opts)], [factors_of(K, N, ranks, dtype, rows)], x, ids_of(kind, rows, len(ranks)))


@pytest.mark.parametrize("kind", ["tokens", "runs", "one"])
@pytest.mark.parametrize("ranks", [(64, 32, 48), (96, 16, 80), (128, 112, 200, 8)])
@pytest.mark.parametrize("K", [64, 192, 320, 800, 1152])
def test_slices_that_are_shorter_than_the_loads_reach_ahead(pkg, dev, K, ranks, kind):
    """One K-tile to five in a slice, one slice and several: the passes drain between them."""
    rows, N, dtype = 700, 264, torch.bfloat16
    x = torch.randn(rows, K, generator=torch.Generator(device="cuda").manual_seed(K), device=dev).to(dtype)
    run(pkg, dev, [layer_of(pkg, K, N, dtype)], [factors_of(K, N, ranks, dtype, K)], x, ids_of(kind, rows, len(ranks)))


@pytest.mark.parametrize("kind", ["tokens", "runs"])
@pytest.mark.parametrize("rows,K,rotate", [(12, 512, False), (64, 1024, False), (100, 640, True), (128, 200, False), (300, 1536, False), (700, 2048, True), (700, 1003, False), (2100, 1024, False)])
def test_several_layers_of_unequal_widths_ranks_and_banks(pkg, dev, rows, K, rotate, kind):
    """q, k and v: one call in every form; one bank has fewer adapters than the others and one nothing at all."""
    dtype, widths = torch.bfloat16, (520, 136, 264, 72)
    layers = [layer_of(pkg, K, N, dtype, bias=i != 1, per_row=i != 2, rotate=rotate, seed=i) for i, N in enumerate(widths)]
    ranks = [(40, 8, 16), (16, None, 72), (8, 100), (None, None, None)]
    adapters = [factors_of(K, N, r, dtype, 10 * rows + i) for i, (N, r) in enumerate(zip(widths, ranks))]
    banks = [pkg.AdapterBank(a, dtype=dtype, device=dev, in_features=K, out_features=N) for a, N in zip(adapters, widths)]
    x = torch.randn(rows, K, generator=torch.Generator(device="cuda").manual_seed(rows), device=dev).to(dtype)
    ids = ids_of(kind, rows, 3)
    outs, again = (pkg.forward_adapters(layers, x, banks, ids) for _ in range(2))
    for lin, some, y, z in zip(layers, adapters, outs, again):
        check(y, *expected(pkg, lin, x, some, ids))
        assert torch.equal(y, z)


@pytest.mark.parametrize("rows", [3, 20])
def test_rows_of_eight_million_columns(pkg, dev, rows):
    """Beyond the 32-bit offsets of 64 rows of them: by waves, whatever the rows."""
    K, N, dtype = (1 << 23) + 16, 8, torch.bfloat16
    x = torch.randn(rows, K, generator=torch.Generator(device="cuda").manual_seed(rows), device=dev).to(dtype)
    run(pkg, dev, [layer_of(pkg, K, N, dtype)], [factors_of(K, N, (3, 16), dtype, rows)], x, ids_of("tokens", rows, 2))


def test_a_row_of_almost_2_to_the_30_columns(pkg, L, dev):
    """The first product alone, of an x with three values: exact."""
    K = (1 << 30) - 5
    down = torch.zeros(1, K, dtype=torch.bfloat16, device=dev)
    at = torch.tensor([0, (1 << 29) + 3, K - 1], device=dev)
    down[0, at] = torch.tensor([1.0, 0.5, 2.0], device=dev).bfloat16()
    bank = pkg.AdapterBank([(down, torch.ones(4, 1, device=dev).bfloat16(), 3.0)])
    del down
    x = torch.zeros(2, K, dtype=torch.bfloat16, device=dev)
    x[0, at] = torch.tensor([2.0, 8.0, -5.0], device=dev).bfloat16()
    x[1, K - 1] = 7.0
    t, = L.adapters_down(x, [bank], torch.zeros(2, dtype=torch.int32, device=dev))
    assert t[:, 0].tolist() == [-12.0, 42.0]


def test_more_activations_than_a_descriptor_addresses(pkg, L, dev):
    """M K >= 2^31: the projection goes in blocks of rows and through binary32; rows at the ends and around the blocks' borders."""
    rows, K, N, dtype = (1 << 17) + 200, 16384, 64, torch.bfloat16
    lin, adapters = layer_of(pkg, K, N, dtype), factors_of(K, N, (16, 40), dtype)
    x = torch.randn(rows, K, generator=torch.Generator(device="cuda").manual_seed(1), device=dev, dtype=dtype)
    ids = ids_of("runs", rows, 2)
    y = pkg.forward_adapters(lin, x, pkg.AdapterBank(adapters), ids)
    for first in (0, (1 << 16) - 100, (1 << 17) - 356, rows - 300):
        part = slice(first, first + 300)
        check(y[part], *expected(pkg, lin, x[part], adapters, ids[part]), f"rows from {first}")
