"""Norms, gate and scales between two blocks against the formula in 64 bits, element by element.

Bounds: with u = half a step of the type (of a result, rounded once), v = 2^-24 and c = v (K / 64 + 16), which covers a sum of K values
in binary32 by any kernel here (at least 64 partial sums of a row, joined in a tree), relative to the sum of their magnitudes:
    mean    dm  = c mean|z|
    norm    dn  = (dz + dm) rstd + |n| (c + 8 v + rstd (rms(dz) + dm))        dz: the bound of its input
    x       dx  = |g'| (|w| dn + 4 v (|w n| + |b|)) + dg |w n + b| + 4 v (|residual part| + |branch|)
            dg: 2^-21 with the fast tanh of 16-bit rows, a few v else
    h       the norm's bound on dx, times |w2| and |1 + s|, and 6 v of every term"""
import pytest
import torch

pytestmark = pytest.mark.gpu

V = 2.0 ** -24


def norm64(z, dz, kind, w, b, eps):
    """(norm, its bound) in float64."""
    if kind is None:
        return z, dz
    K = z.shape[-1]
    c = V * (K / 64 + 16)
    m, dm = (z.mean(-1, keepdim=True), c * z.abs().mean(-1, keepdim=True)) if kind == "layer" else (0.0, 0.0)
    d = z - m
    rstd = 1.0 / (d.square().mean(-1, keepdim=True) + eps).sqrt()
    n = d * rstd
    dn = (dz + dm) * rstd + n.abs() * (c + 8 * V + rstd * (dz.square().mean(-1, keepdim=True).sqrt() + dm)) + V * z.abs() * rstd
    w = 1.0 if w is None else w.double()
    b = torch.zeros((), dtype=torch.float64, device=z.device) if b is None else b.double()
    out = n * w + b
    return out, torch.as_tensor(w).abs() * dn + 4 * V * ((n * w).abs() + b.abs())


def expected(y, residual, *, post_norm=None, post_weight=None, post_bias=None, post_eps=1e-6, gate=None, gate_tanh=False, residual_scale=1.0,
             branch_scale=1.0, pre_norm=None, pre_weight=None, pre_bias=None, pre_eps=1e-6, mod_scale=None, mod_shift=None):
    u, dtype = torch.finfo(y.dtype).eps / 2, y.dtype
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps

    def rounded(v, d):
        return v, d + u * (v.abs() + d) + tiny

    z = y.double()
    n, dn = norm64(z, torch.zeros_like(z), post_norm, post_weight, post_bias, post_eps)
    g, dg = torch.ones((), dtype=torch.float64, device=y.device), 0.0
    if gate is not None:
        g = gate.double()
        if gate_tanh:
            g, dg = g.tanh(), 2.0 ** -21 if dtype != torch.float32 else 4 * V
    branch, carried = branch_scale * g * n, residual_scale * residual.double()
    x = carried + branch
    dx = abs(branch_scale) * (g.abs() * dn + dg * n.abs()) + 4 * V * (carried.abs() + branch.abs())
    if pre_norm is None and mod_scale is None and mod_shift is None:
        return rounded(x, dx), None
    h, dh = norm64(x, dx, pre_norm, pre_weight, pre_bias, pre_eps)
    size = h.abs()
    if mod_scale is not None:
        f = 1.0 + mod_scale.double()
        h, dh, size = h * f, dh * f.abs(), size * f.abs()
    if mod_shift is not None:
        h, size = h + mod_shift.double(), size + mod_shift.double().abs()
    return rounded(x, dx), rounded(h, dh + 6 * V * size)


def check(got, want, what=""):
    value, bound = want
    assert got.shape == value.shape and torch.isfinite(got.float()).all(), what
    worst = ((got.double() - value).abs() / bound).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} of the bound"


def inputs(shape, dtype, offset=0.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + shape[-1])
    y, r = (torch.randn(shape, generator=g, device="cuda") * 2 + offset for _ in range(2))
    y[..., :: max(1, shape[-1] // 3)] *= 10
    return y.to(dtype), r.to(dtype)


def operands(shape, dtype, post, pre, gate, seed=0, wide=False):
    g = torch.Generator(device="cuda").manual_seed(7 + seed)
    K, lead = shape[-1], shape[:-1]
    vec = (lead[0], *(1,) * (len(lead) - 1), K)
    weight = lambda: (1 + 0.3 * torch.randn(K, generator=g, device="cuda")).to(torch.float32 if wide else dtype)  # noqa: E731
    bias = lambda: (0.3 * torch.randn(K, generator=g, device="cuda")).to(torch.float32 if wide else dtype)  # noqa: E731
    mod = lambda: (0.5 * torch.randn(vec, generator=g, device="cuda")).to(dtype)  # noqa: E731
    ops = {"post_norm": post, "pre_norm": pre, "post_eps": 1e-5, "pre_eps": 1e-3}
    if post:
        ops.update(post_weight=weight())
    if pre:
        ops.update(pre_weight=weight())
    if post == "layer":
        ops.update(post_bias=bias())
    if pre == "layer":
        ops.update(pre_bias=bias())
    if gate:
        ops.update(gate=mod(), gate_tanh=gate == "tanh")
    return ops, mod


SHAPES = [(1, 1), (3, 1, 2), (2, 3, 16), (1, 64), (5, 63), (2, 40, 128), (4, 7, 1000), (1, 1001), (2, 300, 1024), (3, 5, 1040), (2, 2048), (1, 4096), (7, 111, 1001),
          (2, 30, 3840), (1, 9, 4112), (2, 520, 5120), (3, 8192), (2, 16384), (2, 16400), (1, 40000)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_against_the_formula(pkg, dev, shape, dtype):
    for i, (post, pre, gate) in enumerate((("rms", "rms", "tanh"), ("layer", "layer", "plain"), ("rms", None, ""), (None, "layer", "plain"))):
        y, r = inputs(shape, dtype, seed=i)
        ops, mod = operands(shape, dtype, post, pre, gate, i, wide=i % 2 == 1)
        ops.update(residual_scale=(1.0, 0.8)[i % 2], branch_scale=(0.5, 1.0)[i % 2])
        if i != 2:
            ops.update(mod_scale=mod())
        if i in (1, 3):
            ops.update(mod_shift=mod())
        x, h = pkg.block_norm(y, r, **ops)
        assert x.dtype == dtype and (h is None) == (i == 2)
        want_x, want_h = expected(y, r, **ops)
        check(x, want_x, f"x {post} {pre}")
        if h is not None:
            check(h, want_h, f"h {post} {pre}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [1024, 1003, 20000])
def test_rows_far_from_zero(pkg, dev, K, dtype):
    """A mean many times the spread: the variance is that of the differences."""
    y, r = inputs((6, 5, K), dtype, offset=100.0)
    ops, _ = operands((6, 5, K), dtype, "layer", "layer", "plain")
    x, h = pkg.block_norm(y, r, **ops)
    want_x, want_h = expected(y, r, **ops)
    check(x, want_x)
    check(h, want_h)


@pytest.mark.parametrize("K", [256, 264, 3840, 6144])
def test_strides_gates_and_vectors_of_every_shape(pkg, dev, K):
    dtype, lead = torch.bfloat16, (3, 4)
    g = torch.Generator(device="cuda").manual_seed(K)
    wide = torch.randn(*lead, 2 * K + 8, generator=g, device=dev).to(dtype)
    flat = torch.randn(12 * K + 1, generator=g, device=dev).to(dtype)
    sources = [wide[..., :K], wide[..., K:2 * K], wide[..., 3:K + 3], flat[1:].view(*lead, K), torch.randn(4, 3, K, generator=g, device=dev).to(dtype).transpose(0, 1)]
    vec = lambda *s: (torch.randn(*s, K, generator=g, device=dev) * 0.5).to(dtype)  # noqa: E731
    for i, (y, r) in enumerate(zip(sources, sources[1:] + sources[:1])):
        for gate, scale, shift in ((vec(), vec(3, 1), None), (vec(3, 4), vec(1, 1), vec(3, 4)), (vec(3, 1), None, vec())):
            ops = dict(post_norm="rms", pre_norm="rms", gate=gate, mod_scale=scale, mod_shift=shift, pre_weight=vec())
            x, h = pkg.block_norm(y, r, **ops)
            want_x, want_h = expected(y, r, **ops)
            check(x, want_x, str(i))
            check(h, want_h, str(i))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,K,rotate", [(19, 1000, False), *((rows, K, rotate) for rotate in (False, True) for rows, K in
                                           ((1, 128), (40, 384), (300, 1024), (33, 2048), (33, 3840), (1100, 3840), (2300, 4096), (5, 6144), (9, 16384), (3, 16512)))])
def test_int8_rows_are_those_of_the_stored_h(pkg, L, dev, rows, K, dtype, rotate):
    y, r = inputs((rows, K), dtype)
    for post, pre in (("rms", "rms"), ("layer", "layer")):
        ops, mod = operands((rows, K), dtype, post, pre, "tanh")
        ops.update(mod_scale=mod())
        x, h = L.block_norm(y, r, **ops)
        x8, q, s = L.block_norm(y, r, quantise=True, rotate=rotate, **ops)
        want_q, want_s = L.quant_rowwise(h, rotate=rotate)
        assert torch.equal(x, x8) and torch.equal(q, want_q) and torch.equal(s, want_s)


def layers_of(pkg, K, widths, dtype, rotate=False):
    out = []
    for i, n in enumerate(widths):
        g = torch.Generator(device="cuda").manual_seed(i + n)
        lin = pkg.Int8TensorwiseOps.Linear(K, n, bias=i != 1, device="meta")
        state = {"weight": torch.randint(-127, 128, (n, K), dtype=torch.int8, generator=g, device="cuda"),
                 "weight_scale": torch.rand(n, 1, generator=g, device="cuda") * 0.002 + 1e-3}
        if i != 1:
            state["bias"] = torch.randn(n, generator=g, device="cuda").to(dtype)
        lin._load_from_state_dict(state, "", {}, True, [], [], [])
        lin._use_quarot = rotate
        out.append(lin)
    return out


@pytest.mark.parametrize("shape,widths,dtype,rotate", [((2, 100, 512), (384, 384, 128), torch.bfloat16, False), ((1, 16, 512), (384, 128), torch.float16, False),
                                                       ((3, 200, 384), (256,), torch.float16, True), ((1, 30, 200), (96, 100), torch.bfloat16, False),
                                                       ((2, 64, 256), (128,), torch.float32, False), ((4, 1, 256), (128, 64), torch.bfloat16, True)])
def test_into_projections(pkg, dev, shape, widths, dtype, rotate):
    layers = layers_of(pkg, shape[-1], widths, dtype, rotate)
    y, r = inputs(shape, dtype)
    ops, mod = operands(shape, dtype, "rms", "rms", "tanh")
    ops.update(mod_scale=mod())
    x, outs = pkg.forward_block_norm(layers, y, r, **ops)
    want_x, h = pkg.block_norm(y, r, **ops)
    assert torch.equal(x, want_x) and len(outs) == len(widths)
    for lin, o in zip(layers, outs):
        assert torch.equal(o, lin(h))


def test_layers_with_something_attached_go_alone(pkg, dev):
    layers = layers_of(pkg, 256, (128, 64), torch.bfloat16)
    layers[0].lora_A, layers[0].lora_B = (torch.randn(s, device=dev).bfloat16() * 0.05 for s in ((16, 256), (128, 16)))
    y, r = inputs((2, 50, 256), torch.bfloat16)
    x, outs = pkg.forward_block_norm(layers, y, r, pre_norm="rms")
    want_x, h = pkg.block_norm(y, r, pre_norm="rms")
    assert torch.equal(x, want_x)
    for lin, o in zip(layers, outs):
        assert torch.equal(o, lin(h))


def test_not_finite_values_stay_in_their_rows(pkg, L, dev):
    for K in (512, 515):
        y, r = inputs((64, K), torch.bfloat16)
        ops = dict(post_norm="layer", pre_norm="rms")
        x, h = pkg.block_norm(y, r, **ops)
        y[5, 3], r[9, 2], y[20] = float("nan"), float("inf"), 0.0
        x2, h2 = pkg.block_norm(y, r, **ops)
        bad = torch.tensor([5, 9], device=dev)
        fine = torch.ones(64, dtype=torch.bool, device=dev)
        fine[[5, 9, 20]] = False
        assert torch.equal(x[fine], x2[fine]) and torch.equal(h[fine], h2[fine])
        assert not torch.isfinite(h2[bad].float()).all(1).any()
        assert torch.equal(x2[20], r[20])          # a row of one value normalises to zero


def test_empty_batches_and_outputs_of_their_own(pkg, dev):
    x, h = pkg.block_norm(*(torch.empty(0, 64, device=dev).bfloat16() for _ in range(2)), pre_norm="rms")
    assert x.shape == (0, 64) and h.shape == (0, 64)
    y, r = inputs((8, 128), torch.bfloat16)
    kept = y.clone(), r.clone()
    x, h = pkg.block_norm(y, r)
    assert h is None and torch.equal(x, (y.float() + r.float()).bfloat16())
    assert torch.equal(y, kept[0]) and torch.equal(r, kept[1])


def test_a_captured_call_and_another_stream(pkg, dev):
    layers = layers_of(pkg, 512, (256, 256), torch.bfloat16)
    y, r = inputs((2, 40, 512), torch.bfloat16)
    ops, mod = operands((2, 40, 512), torch.bfloat16, "rms", "rms", "tanh")
    pkg.forward_block_norm(layers, y, r, **ops)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x, outs = pkg.forward_block_norm(layers, y, r, **ops)
        x2, h = pkg.block_norm(y, r, **ops)
    for i in range(4):
        y.copy_(torch.randn(y.shape, device=dev))
        want_x, want = pkg.forward_block_norm(layers, y, r, **ops)
        want_h = pkg.block_norm(y, r, **ops)[1]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, want_x) and torch.equal(x2, want_x) and torch.equal(h, want_h), f"replay {i}"
        for a, b in zip(outs, want):
            assert torch.equal(a, b), f"replay {i}"
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        other = pkg.block_norm(y, r, **ops)
    s.synchronize()
    assert torch.equal(other[0], want_x) and torch.equal(other[1], want_h)


def test_refusals(pkg, L, dev):
    y, r = inputs((2, 6, 128), torch.bfloat16)
    f = pkg.block_norm
    w = torch.ones(128, device=dev)
    with pytest.raises(RuntimeError, match="GPU"):
        f(y.cpu(), r)
    with pytest.raises(ValueError, match="alike"):
        f(y, r[:1])
    with pytest.raises(ValueError, match="alike"):
        f(y, r.float())
    with pytest.raises(TypeError, match="dtype"):
        f(y.double(), r.double())
    with pytest.raises(ValueError, match="post_norm"):
        f(y, r, post_norm="batch")
    with pytest.raises(ValueError, match="without a norm"):
        f(y, r, post_weight=w)
    with pytest.raises(ValueError, match="pre_weight"):
        f(y, r, pre_norm="rms", pre_weight=w.half())
    with pytest.raises(ValueError, match="one type"):
        f(y, r, pre_norm="layer", pre_weight=w, pre_bias=w.bfloat16())
    with pytest.raises(ValueError, match="pre_eps"):
        f(y, r, pre_norm="rms", pre_eps=-1.0)
    for bad in (w, w.bfloat16().expand(1, 6, 128), w.bfloat16().expand(6, 128), w.bfloat16()[:64]):   # type, the tokens' dimension alone, fewer dimensions, width
        with pytest.raises(ValueError, match="gate"):
            f(y, r, gate=bad)
    with pytest.raises(ValueError, match="no elements"):
        f(y[..., :0], r[..., :0])
    with pytest.raises(RuntimeError, match="gradient"):
        f(y.clone().requires_grad_(), r)
    with pytest.raises(RuntimeError, match="gradient"):
        f(y, r, pre_norm="rms", pre_weight=torch.nn.Parameter(w))
    with pytest.raises(ValueError, match="need an h"):
        pkg.forward_block_norm(layers_of(pkg, 128, (64,), torch.bfloat16), y, r)


def test_a_run_of_blocks(pkg, L, dev):
    """The two operators as a model uses them: adapted projections, what lies between the blocks, and the feed-forward's projections."""
    from test_gpu_adapters import check as check_adapted, expected as expected_adapted, factors_of

    dtype, batch, tokens, K, hidden = torch.bfloat16, 3, 40, 256, 512
    qkv, proj, up, down = layers_of(pkg, K, (K, K, K), dtype), layers_of(pkg, K, (K,), dtype)[0], layers_of(pkg, K, (hidden, hidden), dtype), layers_of(pkg, hidden, (K,), dtype)[0]
    adapters = [factors_of(K, K, (8, None, 32), dtype, i) for i in range(3)]
    banks = [pkg.AdapterBank(a) for a in adapters]
    ids = torch.tensor([2, -1, 0], dtype=torch.int32, device=dev)
    x, ops = inputs((batch, tokens, K), dtype)[0], operands((batch, tokens, K), dtype, "rms", "rms", "tanh")[0]
    branch = torch.zeros_like(x)
    for _ in range(2):
        x, h = pkg.block_norm(branch, x, **ops)
        q, k, v = pkg.forward_adapters(qkv, h, banks, ids)
        for lin, some, o in zip(qkv, adapters, (q, k, v)):
            want, bound = expected_adapted(pkg, lin, h.view(-1, K), some, ids.repeat_interleave(tokens))
            check_adapted(o.view(-1, K), want, bound)
        mixed = torch.softmax(q.float() @ k.float().transpose(1, 2) / K ** 0.5, -1) @ v.float()
        x_before = x
        x, (a, b) = pkg.forward_block_norm(up, proj(mixed.to(dtype)), x, **ops)
        want_x, want_h = pkg.block_norm(proj(mixed.to(dtype)), x_before, **ops)
        assert torch.equal(x, want_x) and torch.equal(a, up[0](want_h)) and torch.equal(b, up[1](want_h))
        branch = down(a, prologue=L.PRO_SILU_GATE, mod_scale=b)
        assert torch.isfinite(branch.float()).all()


@pytest.mark.parametrize("rows", [8, 40])
def test_in_a_compiled_program(pkg, dev, rows):
    layers = layers_of(pkg, 256, (128, 72), torch.bfloat16)
    y, r = inputs((rows, 256), torch.bfloat16)
    ops, _ = operands((rows, 256), torch.bfloat16, "rms", "layer", True)

    def run(y, r):
        return pkg.block_norm(y, r, **ops), pkg.block_norm(y, r, post_norm="rms"), pkg.forward_block_norm(layers, y, r, **ops)

    with torch.no_grad():
        want = run(y, r)
        got = torch.compile(run, backend="aot_eager", fullgraph=True)(y, r)
    assert got[1][1] is None and want[1][1] is None
    pairs = [*zip(got[0], want[0]), (got[1][0], want[1][0]), (got[2][0], want[2][0]), *zip(got[2][1], want[2][1])]
    assert all(torch.equal(a, b) for a, b in pairs)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_a_tanh_gate_is_as_good_near_zero(pkg, dev, dtype):
    """Relative to the result: half a step, and 4e-6 of the gate in 16 bits (2e-7 absolute from 0.0625 on, the series below), a few units of
    binary32 else."""
    gate = torch.tensor([0.0, 1e-6, -1e-5, 1e-3, 0.03, -0.0624, 0.0626, 0.1, -0.5, 1.0, 4.0, -9.0, 50.0, 1e-4, 0.06, -0.07], device=dev).to(dtype)
    y = torch.linspace(0.5, 900.0, 48, device=dev).view(3, 16).to(dtype)
    x, _ = pkg.block_norm(y, torch.zeros_like(y), gate=gate, gate_tanh=True)
    want = gate.double().tanh() * y.double()
    u = torch.finfo(dtype).eps / 2
    bound = want.abs() * (u + (5e-6 if dtype != torch.float32 else 8 * V)) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert ((x.double() - want).abs() <= bound).all()
