"""Adapters of many requests beside shared projections against the formula in 64 bits, element by element.

The bound counts what the operator rounds.  With u = half a step of the output type and v = 2^-24, and t = s A x:
    the result once                                     u |out|
    each t once, to the factors' type                   u sum_j |t_j B_nj|
    binary32 sums of K, r and a few more terms          v times (terms) times the sum of the terms' magnitudes
(int8 products are exact; the int8 rows and their scales are the quantiser's, which has tests of its own)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

V = 2.0 ** -24


def layer_of(pkg, K, N, dtype, bias=True, rotate=False, per_row=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + K + N)
    lin = pkg.Int8TensorwiseOps.Linear(K, N, bias=bias, device="meta")
    state = {"weight": torch.randint(-127, 128, (N, K), dtype=torch.int8, generator=g, device="cuda"),
             "weight_scale": (torch.rand(N, 1, generator=g, device="cuda") + 0.5) / (73.0 * K ** 0.5) if per_row else torch.tensor(1.0 / (73.0 * K ** 0.5))}
    if bias:
        state["bias"] = torch.randn(N, generator=g, device="cuda").to(dtype)
    lin._load_from_state_dict(state, "", {}, True, [], [], [])
    lin._use_quarot = rotate
    return lin


def factors_of(K, N, ranks, dtype, seed=0, zero_scale=()):
    g = torch.Generator(device="cuda").manual_seed(1000 + seed)
    out = []
    for i, r in enumerate(ranks):
        if r is None:
            out.append(None)
            continue
        out.append(((torch.randn(r, K, generator=g, device="cuda") * K ** -0.5).to(dtype), torch.randn(N, r, generator=g, device="cuda").to(dtype) * 0.5,
                    0.0 if i in zero_scale else 0.25 + 0.5 * i))
    return out


def expected(pkg, lin, x, adapters, row_ids, rounded_base=None):
    """(results, bounds) [M,N] in float64; rounded_base: the layer's own rounded result, where the operator adds to that."""
    L, dtype = pkg._lib, x.dtype
    u = torch.finfo(dtype).eps / 2
    M, K = x.shape
    w, b = lin.weight.double(), None if lin.bias is None else lin.bias.double()
    ws = lin._get_weight_scale()
    ws = ws.double().view(1, -1) if isinstance(ws, torch.Tensor) else float(torch.tensor(ws, dtype=torch.float32))
    if rounded_base is not None:
        base, size, terms = rounded_base.double(), rounded_base.double().abs(), 1
    elif M > 16:
        q, s = L.quant_rowwise(x, rotate=lin._use_quarot)
        base = (q.double() @ w.t()) * s.double() * ws
        size, terms = base.abs(), 4   # (the sum to binary32, two products of scales, the bias)
    else:
        xr = (L.rotate128(x) if lin._use_quarot else x).double()
        wr = (lin.weight.float() * (ws.float().view(-1, 1) if isinstance(ws, torch.Tensor) else ws)).to(dtype).double()
        base, size, terms = xr @ wr.t(), xr.abs() @ wr.abs().t(), K + 4
    if b is not None and rounded_base is None:
        base, size = base + b, size + b.abs()
    side, t_size, a_size = torch.zeros_like(base), torch.zeros_like(base), torch.zeros_like(base)
    ranks = torch.zeros(M, 1, dtype=torch.float64, device=x.device)
    for a, f in enumerate(adapters):
        rows = row_ids == a
        if f is None or not rows.any():
            continue
        down, up, scale = f[0].double(), f[1].double(), f[2]
        t = scale * (x[rows].double() @ down.t())
        side[rows] = t @ up.t()
        t_size[rows] = t.abs() @ up.abs().t()
        a_size[rows] = (abs(scale) * (x[rows].double().abs() @ down.abs().t())) @ up.abs().t()
        ranks[rows] = float(down.shape[0])
    out = base + side
    inner = u * t_size + V * ((K + 4) * a_size + terms * size + (ranks + 4) * (t_size * (1 + u) + size))
    return out, inner + u * (out.abs() + inner) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def check(got, want, bound, what=""):
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    assert torch.isfinite(got.float()).all(), what
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} of the bound"


CASES = [
    # rows, K, N, ranks of the adapters, dtype, options
    (1, 64, 16, (8,), torch.bfloat16, {}),
    (1, 4096, 512, (16, 3), torch.float16, {"per_row": False}),
    (5, 1000, 77, (1, 7, None, 20), torch.bfloat16, {}),             # K no multiple of 16: no vector loads of the weight
    (16, 512, 1536, (4, 64, 128), torch.float16, {"rotate": True}),
    (16, 2560, 2048, (16, 32), torch.bfloat16, {"bias": False}),
    (17, 256, 64, (8, 16, 24), torch.bfloat16, {}),                  # the first size of the int8 path
    (33, 200, 100, (5, 40), torch.float16, {}),                      # K % 16: the ragged GEMM
    (40, 1024, 1001, (9, 33), torch.bfloat16, {"bias": False}),      # N % 8
    (64, 4096, 1024, (16, 8, 64, None, 32), torch.bfloat16, {"bias": False}),
    (100, 1040, 776, (8, 1100, 40), torch.float16, {"bias": False}),  # a rank beyond every other
    (128, 2048, 4104, (32, 16, 8), torch.bfloat16, {"rotate": True}),
    (130, 384, 264, (100, 17), torch.float16, {"per_row": False}),
    (257, 640, 528, (16, 48), torch.bfloat16, {"rotate": True}),
    (300, 1536, 1536, (64,), torch.float16, {"bias": False}),
    (513, 2048, 4096, (128, 4, 72), torch.bfloat16, {}),
    (1100, 512, 2304, (32, 16), torch.bfloat16, {}),
    (4200, 256, 3840, (32, 160, 16), torch.float16, {}),             # several rounds of large tiles
    (2100, 384, 4608, (20, 64), torch.bfloat16, {"bias": False}),
    (700, 1003, 96, (9, 33, 16), torch.bfloat16, {}),                # odd rows: copied for the first product
    (900, 700, 1001, (130,), torch.float16, {"bias": False}),        # K % 8 of them
    (1500, 2048, 264, (40, 16, 256), torch.bfloat16, {"rotate": True}),
    (8300, 264, 512, (16, 100), torch.float16, {}),
]


def ids_of(kind, rows, count, seed=0):
    g = torch.Generator().manual_seed(seed + rows)
    if kind == "tokens":       # every row another one, some of them no adapter, some no number of the bank
        ids = torch.randint(-1, count + 1, (rows,), generator=g)
        if rows > 2:
            ids[rows // 2] = 2 ** 31 - 1
    elif kind == "runs":       # requests of unequal lengths
        ids = torch.randint(-1, count, (rows,), generator=g)
        ids = ids[torch.cummax(torch.where(torch.rand(rows, generator=g) < 0.02, torch.arange(rows), 0), 0)[0]]
    elif kind == "none":
        ids = torch.full((rows,), -1)
    else:
        ids = torch.full((rows,), count - 1)
    return ids.to(torch.int32).cuda()


@pytest.mark.parametrize("kind", ["tokens", "runs", "one", "none"])
@pytest.mark.parametrize("rows,K,N,ranks,dtype,opts", CASES)
def test_against_the_formula(pkg, dev, rows, K, N, ranks, dtype, opts, kind):
    lin = layer_of(pkg, K, N, dtype, **opts)
    adapters = factors_of(K, N, ranks, dtype, rows)
    bank = pkg.AdapterBank(adapters, dtype=dtype, device=dev)
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, K, generator=g, device=dev).to(dtype)
    ids = ids_of(kind, rows, len(ranks))
    y = pkg.forward_adapters(lin, x, bank, ids)
    assert y.dtype == dtype and y.shape == (rows, N)
    want, bound = expected(pkg, lin, x, adapters, ids)
    check(y, want, bound, kind)
    assert torch.equal(y, pkg.forward_adapters(lin, x, bank, ids))   # nothing depends on timing


def test_rows_without_an_adapter_are_the_layer_in_the_fused_order(pkg, L, dev):
    for rows in (7, 300):
        lin = layer_of(pkg, 512, 768, torch.bfloat16)
        bank = pkg.AdapterBank(factors_of(512, 768, (16, 40), torch.bfloat16))
        x = torch.randn(rows, 512, device=dev).bfloat16()
        ids = torch.randint(-1, 2, (rows,), device=dev, dtype=torch.int32)
        y = pkg.forward_adapters(lin, x, bank, ids)
        if rows > 16:
            q, s = L.quant_rowwise(x)
            plain = L.linear_w8a8(q, s, lin.weight, lin.weight_scale, lin.bias, torch.bfloat16, L.EPI_FUSED)
        else:
            plain = lin(x)
        assert torch.equal(y[ids < 0], plain[ids < 0])
        assert not torch.equal(y[ids >= 0], plain[ids >= 0])


@pytest.mark.parametrize("tokens", [1, 3, 200])
def test_one_number_per_request_and_several_layers(pkg, dev, tokens):
    """ids of the batch, of every token and of the whole call; q, k and v on one x, one of them rotated."""
    batch, K = 4, 256
    lins = [layer_of(pkg, K, n, torch.bfloat16, rotate=r, bias=b) for n, r, b in ((384, False, False), (128, True, True), (128, False, True))]
    adapters = [factors_of(K, lin.weight.shape[0], (16, None, 40), torch.bfloat16, i) for i, lin in enumerate(lins)]
    banks = [pkg.AdapterBank(a) for a in adapters]
    x = torch.randn(batch, tokens, K, device=dev).bfloat16()
    ids = torch.tensor([2, -1, 0, 1], dtype=torch.int32, device=dev)
    every = ids[:, None].expand(batch, tokens)
    outs = pkg.forward_adapters(lins, x, banks, ids)
    again = pkg.forward_adapters(lins, x, banks, every)     # (not contiguous)
    assert isinstance(outs, list) and len(outs) == 3
    for lin, a, o, o2, bank in zip(lins, adapters, outs, again, banks):
        assert o.shape == (batch, tokens, lin.weight.shape[0])
        want, bound = expected(pkg, lin, x.view(-1, K), a, every.reshape(-1))
        check(o.view(want.shape), want, bound)
        assert torch.equal(o, o2)
        alone = pkg.forward_adapters(lin, x, bank, ids)   # (tiles of another shape, maybe: other binary32 sums)
        check(alone.view(want.shape), want, bound)
    one = pkg.forward_adapters(lins[0], x, banks[0], torch.tensor(2, dtype=torch.int32, device=dev))
    assert torch.equal(one[0], outs[0][0])


def test_strides_and_offsets(pkg, dev):
    """Rows of a wider tensor, an x that starts at an odd address, a transposed one."""
    K, N = 512, 256
    lin = layer_of(pkg, K, N, torch.float16)
    adapters = factors_of(K, N, (16, 20), torch.float16)
    bank = pkg.AdapterBank(adapters)
    for rows in (6, 90, 1200):
        ids = torch.arange(rows, device=dev, dtype=torch.int32) % 3 - 1
        wide = torch.randn(rows, K + 24, device=dev).half()
        flat = torch.randn(rows * K + 1, device=dev).half()
        for x in (wide[:, 8:8 + K], wide[:, 5:5 + K], flat[1:].view(rows, K), torch.randn(K, rows, device=dev).half().t()):
            want, bound = expected(pkg, lin, x.contiguous(), adapters, ids)
            check(pkg.forward_adapters(lin, x, bank, ids), want, bound)


def test_layers_whose_kernels_cannot_take_them(pkg, dev):
    """A layer that is not quantised, one with a dynamic LoRA of its own: their rounded result and the adapters' share."""
    K, N = 320, 192
    for rows in (9, 120):
        x = torch.randn(rows, K, device=dev).bfloat16()
        ids = torch.arange(rows, device=dev, dtype=torch.int32) % 3 - 1
        adapters = factors_of(K, N, (16, 20), torch.bfloat16)
        bank = pkg.AdapterBank(adapters)
        plain = torch.nn.Linear(K, N, device=dev, dtype=torch.bfloat16).requires_grad_(False)
        lora = layer_of(pkg, K, N, torch.bfloat16)
        lora.lora_A, lora.lora_B = (torch.randn(s, device=dev).bfloat16() * 0.05 for s in ((16, K), (N, 16)))
        for lin in (plain, lora):
            with torch.no_grad():
                base = lin(x)
            kept = base.clone()
            ref = lora   # (only its base is not used)
            want, bound = expected(pkg, ref, x, adapters, ids, rounded_base=base)
            check(pkg.forward_adapters(lin, x, bank, ids), want, bound)
            assert torch.equal(base, kept)


def test_empty_batches_banks_without_factors_and_zero_scales(pkg, dev):
    lin = layer_of(pkg, 256, 128, torch.bfloat16)
    bank = pkg.AdapterBank(factors_of(256, 128, (16,), torch.bfloat16))
    for shape in ((0, 256), (2, 0, 256)):
        y = pkg.forward_adapters(lin, torch.empty(shape, device=dev, dtype=torch.bfloat16), bank, torch.empty(shape[:-1], dtype=torch.int32, device=dev))
        assert y.shape == (*shape[:-1], 128)
    for rows in (3, 50):
        x = torch.randn(rows, 256, device=dev).bfloat16()
        ids = torch.zeros(rows, dtype=torch.int32, device=dev)
        none = pkg.AdapterBank([None, None], in_features=256, out_features=128, device=dev)
        zero = pkg.AdapterBank(factors_of(256, 128, (16,), torch.bfloat16, zero_scale=(0,)))
        nothing = pkg.AdapterBank([], in_features=256, out_features=128, device=dev)
        plain = pkg.forward_adapters(lin, x, bank, ids - 1)
        for b in (none, zero, nothing):
            assert torch.equal(pkg.forward_adapters(lin, x, b, ids), plain)


def test_not_finite_values_stay_in_their_rows(pkg, dev):
    """An adapter with infinite factors and a row of NaN: other rows, of the same tile too, do not see them."""
    K, N = 256, 192
    for rows in (12, 200):
        lin = layer_of(pkg, K, N, torch.bfloat16)
        adapters = factors_of(K, N, (16, 20, 16), torch.bfloat16)
        x = torch.randn(rows, K, device=dev).bfloat16()
        ids = torch.arange(rows, device=dev, dtype=torch.int32) % 4 - 1
        want = pkg.forward_adapters(lin, x, pkg.AdapterBank(adapters), ids)
        adapters[1][0][3, 5] = float("inf")
        adapters[1][1][7] = float("nan")
        x[5] = float("nan")
        got = pkg.forward_adapters(lin, x, pkg.AdapterBank(adapters), ids)
        fine = (ids != 1) & (torch.arange(rows, device=dev) != 5)
        assert torch.equal(got[fine], want[fine])
        assert not torch.isfinite(got[ids == 1][:, 7].float()).any()


def test_a_captured_call_follows_the_numbers_and_the_rows(pkg, dev):
    K, N = 512, 384
    for rows in (8, 70):
        lin = layer_of(pkg, K, N, torch.bfloat16)
        bank = pkg.AdapterBank(factors_of(K, N, (16, 64, 8), torch.bfloat16))
        x, ids = torch.randn(rows, K, device=dev).bfloat16(), torch.zeros(rows, dtype=torch.int32, device=dev)
        pkg.forward_adapters(lin, x, bank, ids)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = pkg.forward_adapters(lin, x, bank, ids)
        for i in range(4):
            x.copy_(torch.randn(rows, K, device=dev))
            ids.copy_(torch.randint(-1, 3, (rows,), device=dev))
            want = pkg.forward_adapters(lin, x, bank, ids)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want), f"replay {i}"


def test_two_streams_at_once(pkg, dev):
    """Calls of one layer and bank that overlap share nothing that they write."""
    lin = layer_of(pkg, 1024, 1024, torch.bfloat16)
    bank = pkg.AdapterBank(factors_of(1024, 1024, (32, 16), torch.bfloat16))
    xs = [torch.randn(n, 1024, device=dev).bfloat16() for n in (200, 16)]
    ids = [torch.arange(x.shape[0], device=dev, dtype=torch.int32) % 2 for x in xs]
    want = [pkg.forward_adapters(lin, x, bank, i) for x, i in zip(xs, ids)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for _ in range(8):
        for s, x, i in zip(streams, xs, ids):
            with torch.cuda.stream(s):
                got.append(pkg.forward_adapters(lin, x, bank, i))
    torch.cuda.synchronize()
    for k, y in enumerate(got):
        assert torch.equal(y, want[k % 2])


def test_refusals(pkg, dev):
    lin = layer_of(pkg, 256, 128, torch.bfloat16)
    bank = pkg.AdapterBank(factors_of(256, 128, (16,), torch.bfloat16))
    x, ids = torch.randn(20, 256, device=dev).bfloat16(), torch.zeros(20, dtype=torch.int32, device=dev)
    f = pkg.forward_adapters
    with pytest.raises(TypeError, match="int32"):
        f(lin, x, bank, ids.long())
    with pytest.raises(RuntimeError, match="GPU"):
        f(lin, x, bank, ids.cpu())
    with pytest.raises(ValueError, match="leading dimensions"):
        f(lin, x, bank, ids[:19])
    with pytest.raises(ValueError, match="leading dimensions"):
        f(lin, x.view(4, 5, 256), bank, ids)
    with pytest.raises(TypeError, match="float16"):
        f(lin, x.half(), bank, ids)
    with pytest.raises(TypeError, match="float32"):
        f(lin, x.float(), bank, ids)
    with pytest.raises(ValueError, match="features"):
        f(lin, x[:, :128], bank, ids)
    with pytest.raises(ValueError, match="banks"):
        f([lin, lin], x, [bank], ids)
    with pytest.raises(ValueError, match="outputs"):
        f(layer_of(pkg, 256, 64, torch.bfloat16), x, bank, ids)
    with pytest.raises(RuntimeError, match="gradient"):
        f(lin, x.clone().requires_grad_(), bank, ids)
    with torch.no_grad():
        f(lin, x.clone().requires_grad_(), bank, ids)


def test_a_bank_of_lora_patches(pkg, dev):
    """(adapter, strength) as the dynamic loaders hold them: what the layer does with the same LoRA attached, up to their roundings."""
    up, down = torch.randn(128, 16, device=dev) * 0.1, torch.randn(16, 256, device=dev) * 0.1
    patch = pkg.INT8LoRAPatchAdapter(set(), (up, down, 8.0, None, None, None), 0.01)
    bank = pkg.AdapterBank.from_patches([None, (patch, 0.5)], dtype=torch.bfloat16)
    assert bank.count == 2 and bank.ranks == [0, 16] and bank.device == up.device
    lin = layer_of(pkg, 256, 128, torch.bfloat16)
    x = torch.randn(50, 256, device=dev).bfloat16()
    ids = torch.ones(50, dtype=torch.int32, device=dev)
    adapters = [None, ((down * 0.25).bfloat16(), up.bfloat16(), 1.0)]
    want, bound = expected(pkg, lin, x, adapters, ids)
    check(pkg.forward_adapters(lin, x, bank, ids), want, bound)


@pytest.mark.parametrize("rows", [8, 200])
def test_in_a_compiled_program(pkg, dev, rows):
    """Traced without a break, also beside a layer that goes alone; more than 128 rows and up to 16 take the eager call's kernels."""
    layers = [layer_of(pkg, 256, N, torch.bfloat16, rotate=True, seed=N) for N in (128, 72)] + [layer_of(pkg, 256, 64, torch.bfloat16, bias=False)]
    alone = layer_of(pkg, 256, 128, torch.bfloat16, seed=9)
    alone.weight_function = [lambda w: w]
    layers.append(alone)
    banks = [pkg.AdapterBank(factors_of(256, lin.out_features, (8, 20), torch.bfloat16, seed=i)) for i, lin in enumerate(layers)]
    x, ids = torch.randn(rows, 256, device=dev).bfloat16(), ids_of("tokens", rows, 2)

    def run(x, ids):
        return pkg.forward_adapters(layers[:3], x, banks[:3], ids), pkg.forward_adapters(layers[3], x, banks[3], ids)

    with torch.no_grad():
        want, want_alone = run(x, ids)
        got, _ = torch.compile(lambda x, ids: (pkg.forward_adapters(layers[:3], x, banks[:3], ids), 0), backend="aot_eager", fullgraph=True)(x, ids)
        _, got_alone = torch.compile(run, backend="aot_eager")(x, ids)
    for a, b in zip((*got, got_alone), (*want, want_alone)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows", [7, 90, 300])
def test_more_layers_than_a_launch_takes_and_one_number_for_all(pkg, dev, rows):
    """Six layers of both rotation flags, one of them twice with one bank; ids without dimensions."""
    dtype = torch.bfloat16
    layers = [layer_of(pkg, 256, N, dtype, rotate=i % 3 == 0, seed=i) for i, N in enumerate((128, 72, 40, 256, 8))]
    made = [factors_of(256, lin.out_features, (8, 20), dtype, seed=i) for i, lin in enumerate(layers)]
    banks = [pkg.AdapterBank(f) for f in made]
    layers, made, banks = layers + layers[1:2], made + made[1:2], banks + banks[1:2]
    x = torch.randn(rows, 256, device=dev).to(dtype)
    outs = pkg.forward_adapters(layers, x, banks, torch.tensor(1, dtype=torch.int32, device=dev))
    for lin, f, y in zip(layers, made, outs):
        check(y, *expected(pkg, lin, x, f, torch.ones(rows, dtype=torch.int32, device=dev)))
    assert torch.equal(outs[1], outs[5])


def test_a_single_row_without_other_dimensions(pkg, dev):
    lin, f = layer_of(pkg, 128, 48, torch.float16), factors_of(128, 48, (8,), torch.float16)
    x = torch.randn(128, device=dev).half()
    y = pkg.forward_adapters(lin, x, pkg.AdapterBank(f), torch.tensor(0, dtype=torch.int32, device=dev))
    assert y.shape == (48,)
    check(y[None], *expected(pkg, lin, x[None], f, torch.zeros(1, dtype=torch.int32, device=dev)))


@pytest.mark.parametrize("kind", ["tokens", "runs"])
@pytest.mark.parametrize("rows,K,N", [(9, 250, 33), (64, 256, 192), (100, 200, 101), (700, 512, 200), (700, 515, 201), (1100, 512, 2304)])
def test_not_finite_values_stay_in_their_rows_in_every_form(pkg, dev, rows, K, N, kind):
    """By waves and by tiles, by way of a side tensor, of the epilogue and of the second product's own launch."""
    lin = layer_of(pkg, K, N, torch.float16)
    adapters = factors_of(K, N, (40, 20, 16, 33), torch.float16)
    x = torch.randn(rows, K, device=dev).half()
    ids = (torch.arange(rows, device=dev) % 5 - 1 if kind == "tokens" else (torch.arange(rows, device=dev) * 9 // rows) % 5 - 1).to(torch.int32)
    want = pkg.forward_adapters(lin, x, pkg.AdapterBank(adapters), ids)
    adapters[1][0][3, 5] = float("inf")
    adapters[1][1][7] = float("nan")
    x[rows // 2] = float("nan")
    got = pkg.forward_adapters(lin, x, pkg.AdapterBank(adapters), ids)
    fine = (ids != 1) & (torch.arange(rows, device=dev) != rows // 2)
    assert torch.equal(got[fine], want[fine]) and torch.isfinite(want.float()).all()
    assert not torch.isfinite(got[ids == 1][:, 7].float()).any()


@pytest.mark.parametrize("rows,K,N,ranks", [(40, 200, 101, (16, 8)), (90, 512, 384, (64, 16)), (400, 1024, 384, (64, 16, 8)), (700, 1003, 96, (40, 16))])
def test_captured_calls_of_the_other_forms(pkg, dev, rows, K, N, ranks):
    lin, bank = layer_of(pkg, K, N, torch.bfloat16), pkg.AdapterBank(factors_of(K, N, ranks, torch.bfloat16))
    x, ids = torch.randn(rows, K, device=dev).bfloat16(), torch.zeros(rows, dtype=torch.int32, device=dev)
    pkg.forward_adapters(lin, x, bank, ids)
    graphs, ys = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g in graphs:
        with torch.cuda.graph(g):
            ys.append(pkg.forward_adapters(lin, x, bank, ids))
    for i in range(4):
        x.copy_(torch.randn(rows, K, device=dev))
        ids.copy_(torch.randint(-1, len(ranks), (rows,), device=dev))
        want = pkg.forward_adapters(lin, x, bank, ids)
        for g, y in zip(graphs, ys):
            y.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want), f"replay {i}"
