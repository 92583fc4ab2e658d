"""Adapters and block norms at the edges of what their documentation allows: no rows, banks beyond 2^32 bytes, rows far apart in memory,
operands at odd addresses, int8 rows of values that are not finite."""
import pytest
import torch

from test_gpu_adapters import check, expected, factors_of, ids_of, layer_of
from test_gpu_block_norm import check as check_norm, expected as expected_norm, inputs, layers_of

pytestmark = pytest.mark.gpu


def test_no_rows(pkg, dev):
    layers = layers_of(pkg, 256, (128, 64), torch.bfloat16)
    plain = torch.nn.Linear(256, 128, device=dev, dtype=torch.bfloat16).requires_grad_(False)
    banks = [pkg.AdapterBank(factors_of(256, n, (16,), torch.bfloat16)) for n in (128, 64)]
    for shape in ((0, 256), (3, 0, 256)):
        y = torch.empty(shape, device=dev, dtype=torch.bfloat16)
        x, outs = pkg.forward_block_norm(layers, y, y, pre_norm="rms", mod_scale=torch.ones(256, device=dev).bfloat16())
        assert x.shape == shape and [o.shape for o in outs] == [(*shape[:-1], 128), (*shape[:-1], 64)]
        ids = torch.empty(shape[:-1], dtype=torch.int32, device=dev)
        assert [o.shape for o in pkg.forward_adapters(layers, y, banks, ids)] == [(*shape[:-1], 128), (*shape[:-1], 64)]
        assert pkg.forward_adapters(plain, y, banks[0], ids).shape == (*shape[:-1], 128)
    assert pkg.forward_adapters([], y, [], ids) == []


@pytest.mark.parametrize("kind", ["tokens", "one"])
@pytest.mark.parametrize("rows", [8, 64, 200, 700])
def test_factors_beyond_32_bits_of_offset(pkg, dev, rows, kind):
    """2400 adapters of rank 256, each factor 5 GB in memory; the rows take the first one and the last two."""
    K = N = 4096
    dtype, count = torch.bfloat16, 2400
    some = factors_of(K, N, (256, 250, 64), dtype, rows)
    bank = pkg.AdapterBank([some[0]] * (count - 2) + some[1:])
    assert bank.down.numel() * 2 > 1 << 32 and bank.up.numel() * 2 > 1 << 32
    x = torch.randn(rows, K, generator=torch.Generator(device="cuda").manual_seed(rows), device=dev).to(dtype)
    few = ids_of(kind, rows, 3)
    ids = torch.where((few > 0) & (few < 3), few + (count - 3), few).to(torch.int32)
    ids = torch.where(few >= 3, 2 ** 31 - 1, ids).to(torch.int32)
    lin = layer_of(pkg, K, N, dtype)
    check(pkg.forward_adapters(lin, x, bank, ids), *expected(pkg, lin, x, some, few))


@pytest.mark.parametrize("rows", [5, 40, 200, 300])
def test_rows_eight_million_elements_apart(pkg, dev, rows):
    K, N, dtype = 512, 264, torch.bfloat16
    wide = torch.zeros(rows, (1 << 23) + 8, dtype=dtype, device=dev)
    x = wide[:, 64:64 + K]
    x.copy_(torch.randn(rows, K, generator=torch.Generator(device="cuda").manual_seed(rows), device=dev))
    lin, adapters = layer_of(pkg, K, N, dtype), factors_of(K, N, (64, 100), dtype)
    ids = ids_of("tokens", rows, 2)
    check(pkg.forward_adapters(lin, x, pkg.AdapterBank(adapters), ids), *expected(pkg, lin, x.contiguous(), adapters, ids))
    y, h = pkg.block_norm(x, x, pre_norm="rms")
    want, want_h = pkg.block_norm(x.contiguous(), x.contiguous(), pre_norm="rms")
    assert torch.equal(y, want) and torch.equal(h, want_h)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [96, 640, 1001, 4096])
def test_norm_operands_at_odd_addresses(pkg, dev, K, dtype):
    """Each operand alone one element off."""
    y, r = inputs((2, 9, K), dtype)
    g = torch.Generator(device="cuda").manual_seed(K)
    names = ("post_weight", "post_bias", "pre_weight", "pre_bias", "gate", "mod_scale", "mod_shift")
    flat = {n: (torch.randn(K + 1, generator=g, device=dev) * 0.5 + 1).to(torch.float32 if "weight" in n or "bias" in n else dtype) for n in names}
    for odd in (*names, "all"):
        ops = {n: v[1:] if odd in (n, "all") else v[:K] for n, v in flat.items()}
        x, h = pkg.block_norm(y, r, post_norm="layer", pre_norm="layer", **ops)
        want_x, want_h = expected_norm(y, r, post_norm="layer", pre_norm="layer", **ops)
        check_norm(x, want_x, odd)
        check_norm(h, want_h, odd)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("K,rotate", [(10, False), (24, False), (384, False), (1000, False), (1001, False), (4096, False), (20000, False), (384, True), (4096, True), (16512, True)])
def test_int8_rows_of_values_that_are_not_finite(pkg, L, dev, K, rotate, dtype):
    """What the quantiser makes of the stored h, in these rows too."""
    y, r = inputs((40, K), dtype)
    y[3, K // 2], r[9, 1], r[11], y[20] = float("nan"), float("inf"), float("nan"), 0.0
    r[20] = 0.0
    for ops in (dict(pre_norm="rms"), dict(mod_shift=torch.zeros(K, device=dev).to(dtype))):   # (without a norm one element of the row is not finite)
        x, h = L.block_norm(y, r, **ops)
        x8, q, s = L.block_norm(y, r, quantise=True, rotate=rotate, **ops)
        want_q, want_s = L.quant_rowwise(h, rotate=rotate)
        assert torch.equal(x.nan_to_num(1.0), x8.nan_to_num(1.0))
        off = ((s != want_s) & ~(s.isnan() & want_s.isnan())).view(-1) | (q != want_q).any(1)
        assert not off.any(), f"rows {off.nonzero().view(-1).tolist()}"


def test_threads_with_and_without_streams_of_their_own(pkg, dev):
    """The host path gives the interpreter's lock back while it launches."""
    import concurrent.futures

    layers = layers_of(pkg, 1024, (512, 264), torch.bfloat16)
    banks = [pkg.AdapterBank(factors_of(1024, n, (16, 40), torch.bfloat16)) for n in (512, 264)]
    cases = []
    for rows in (4, 60, 300):
        x = torch.randn(rows, 1024, device=dev).bfloat16()
        ids = (torch.arange(rows, device=dev) % 3 - 1).to(torch.int32)
        cases.append((x, ids, pkg.forward_adapters(layers, x, banks, ids), pkg.forward_block_norm(layers, x, x, post_norm="rms", pre_norm="layer")))
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream() if i % 2 else torch.cuda.default_stream()):
            for k in range(12):
                x, ids, want, (want_x, want_h) = cases[(i + k) % len(cases)]
                got, (got_x, got_h) = pkg.forward_adapters(layers, x, banks, ids), pkg.forward_block_norm(layers, x, x, post_norm="rms", pre_norm="layer")
                if not all(torch.equal(a, b) for a, b in zip((*got, got_x, *got_h), (*want, want_x, *want_h))):
                    return f"thread {i}, call {k}"
        return None

    with concurrent.futures.ThreadPoolExecutor(max_workers=6) as pool:
        assert [r for r in pool.map(work, range(6)) if r] == []
