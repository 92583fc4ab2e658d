"""A call gives the same results whichever way it goes: the native path, the general one, a compiled program."""
import pytest
import torch

from test_gpu_adapters import check, expected, factors_of, layer_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [9, 40, 64, 128, 200])
def test_the_general_path_and_a_compiled_program_repeat_the_native_one(pkg, dev, rows):
    """One number for each row, as many as rows.  Between 17 and 128 of them the native path adds the adapters' share, summed for itself, to the
    projection, where the others add its terms: the same up to the order of binary32 sums.  Else bit for bit."""
    dtype, K = torch.bfloat16, 512
    layers = [layer_of(pkg, K, N, dtype, seed=N) for N in (384, 136, 72)]
    adapters = [factors_of(K, lin.out_features, (16, 40, None, 8), dtype, seed=i) for i, lin in enumerate(layers)]
    banks = [pkg.AdapterBank(a) for a in adapters]
    x = torch.randn(rows, K, generator=torch.Generator(device="cuda").manual_seed(rows), device=dev).to(dtype)
    ids = (torch.arange(rows, device=dev) % 5 - 1).to(torch.int32)
    spread = torch.stack((ids, ids), 1)[:, 0]   # (not contiguous: the general path)
    native = pkg.forward_adapters(layers, x, banks, ids)
    general = pkg.forward_adapters(layers, x, banks, spread)
    with torch.no_grad():
        compiled = torch.compile(lambda x, ids: pkg.forward_adapters(layers, x, banks, ids), backend="aot_eager", fullgraph=True)(x, ids)
    for lin, some, a, b, c in zip(layers, adapters, native, general, compiled):
        want = expected(pkg, lin, x, some, ids)
        for y in (a, b, c):
            check(y, *want)
        assert torch.equal(b, c) and (16 < rows <= 128 or torch.equal(a, b))
