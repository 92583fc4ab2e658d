"""The heads' norms, rotations and the attention together with the projections around them, as a block of a model runs them."""
import threading

import pytest
import torch

from test_gpu_adapters import layer_of
from test_gpu_attention import check as check_attention, expected as expected_attention
from test_gpu_norm_heads import check as check_heads, expected as expected_heads, grid, weight

pytestmark = pytest.mark.gpu


def states(batch, tokens, width, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(batch, tokens, width, generator=g, device="cuda")
    x[..., ::97] *= 8
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rotate", [False, True])
@pytest.mark.parametrize("batch,queries,keys,heads,kv_heads,width", [(2, 300, 77, 4, 4, 128), (1, 40, 200, 6, 2, 64), (3, 1, 130, 4, 4, 72), (1, 130, 512, 2, 1, 256)])
def test_cross_attention_block(pkg, dev, batch, queries, keys, heads, kv_heads, width, dtype, rotate):
    """Every stage is the operator's own result bit for bit, and within its bound of the formula on what the stage before left."""
    features, other = 512, 384
    to_q, to_out = layer_of(pkg, features, heads * width, dtype, bias=True, rotate=rotate), layer_of(pkg, heads * width, features, dtype, bias=True)
    to_k, to_v = (layer_of(pkg, other, kv_heads * width, dtype, bias=i == 1, rotate=rotate, seed=3 + i) for i in range(2))
    x, context = states(batch, queries, features, dtype), states(batch, keys, other, dtype, 1)
    wq, wk = weight(width, dtype), weight(width, dtype, 1)
    dims = (16, 20, width // 2 - 36 + width // 2 % 2) if width > 72 else (16, 20)
    r, p = pkg.RotaryAxes(dims, 256.0), grid(queries, len(dims))
    lengths = torch.tensor([keys, keys // 2, 0][:batch], device="cuda")
    gate, residual = states(batch, 1, features, dtype, 5), states(batch, queries, features, dtype, 6)
    got = pkg.forward_cross_attention(x, context, to_q, to_k, to_v, to_out, heads=heads, kv_heads=kv_heads, q_weight=wq, k_weight=wk, rotary=r, positions=p, key_lengths=lengths,
                                      gate=gate, residual=residual)
    q, k, v = to_q(x).unflatten(-1, (heads, width)), to_k(context).unflatten(-1, (kv_heads, width)), to_v(context).unflatten(-1, (kv_heads, width))
    nq, nk = pkg.norm_heads(q, wq, rotary=r, positions=p), pkg.norm_heads(k, wk)
    check_heads(nq, expected_heads(q, wq, True, 1e-6, dims, 256.0, True, p))
    check_heads(nk, expected_heads(k, wk, True, 1e-6))
    o = pkg.cross_attention(nq, nk, v, key_lengths=lengths)
    check_attention(o, expected_attention(nq, nk, v, key_lengths=lengths))
    assert torch.equal(got, to_out(o.flatten(-2), gate=gate, residual=residual))
    assert torch.equal(pkg.forward_cross_attention(x, context, to_q, to_k, to_v, to_out, heads=heads, kv_heads=kv_heads), to_out(pkg.cross_attention(q, k, v).flatten(-2)))
    assert torch.equal(pkg.forward_cross_attention(x, context, to_q, to_k, to_v, heads=heads, kv_heads=kv_heads, q_weight=wq, k_weight=wk), pkg.cross_attention(
        pkg.norm_heads(q, wq), nk, v).flatten(-2))
    pk = grid(keys, len(dims))
    assert torch.equal(pkg.forward_cross_attention(x, context, to_q, to_k, to_v, heads=heads, kv_heads=kv_heads, rotary=r, positions=p, context_positions=pk, scale=0.3),
                       pkg.cross_attention(pkg.rotate_heads(q, r, p), pkg.rotate_heads(k, r, pk), v, scale=0.3).flatten(-2))


def test_self_attention_block(pkg, dev):
    dtype, heads, width, features = torch.bfloat16, 4, 128, 512
    layers = [layer_of(pkg, features, heads * width, dtype, bias=True, seed=i) for i in range(3)]
    to_out = layer_of(pkg, heads * width, features, dtype, bias=False, seed=9)
    x, w = states(2, 333, features, dtype), [weight(width, dtype, i) for i in range(2)]
    r, p = pkg.RotaryAxes((32, 48, 48), 256.0, interleaved=False), grid(333, 3)
    mask = torch.rand(2, 333, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) < 0.7
    q, k, v = (y.unflatten(-1, (heads, width)) for y in pkg.forward_fanout(layers, x))
    nq, nk = pkg.norm_heads([q, k], w, rotary=r, positions=p)
    want = to_out(pkg.cross_attention(nq, nk, v, key_mask=mask).flatten(-2))
    run = lambda: pkg.forward_cross_attention(x, None, *layers, to_out, heads=heads, q_weight=w[0], k_weight=w[1], rotary=r, positions=p, key_mask=mask)  # noqa: E731
    assert torch.equal(run(), want)
    # captured, replayed with the program's own calls between
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for seed in (11, 12, 13):
        x.copy_(states(2, 333, features, dtype, seed))
        mask.copy_(torch.rand(2, 333, device="cuda") < 0.5)
        eager = run()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
    compiled = torch.compile(lambda y: pkg.forward_cross_attention(y, None, *layers, to_out, heads=heads, q_weight=w[0], k_weight=w[1], rotary=r, positions=p, key_mask=mask),
                             backend="eager")
    assert torch.equal(compiled(x), run())


def test_path_refusals(pkg, dev):
    dtype = torch.bfloat16
    lin = layer_of(pkg, 512, 256, dtype)
    x, r, p = states(2, 20, 512, dtype), pkg.RotaryAxes((64,)), grid(20, 1)
    call = lambda *a, **k: pkg.forward_cross_attention(x, *a, **{"heads": 2, **k})  # noqa: E731
    for bad in (lambda: call(None, lin, lin, lin, heads=3), lambda: call(None, lin, lin, lin, heads=0), lambda: call(None, lin, lin, lin, kv_heads=3),
                lambda: call(None, lin, lin, lin, rotary=r), lambda: call(None, lin, lin, lin, positions=p), lambda: call(None, lin, lin, lin, q_weight=weight(128, dtype)),
                lambda: call(None, lin, lin, lin, rotary=r, positions=p, context_positions=p), lambda: call(x, lin, lin, lin, gate=x), lambda: call(x[:1], lin, lin, lin),
                lambda: pkg.forward_cross_attention(x[0], None, lin, lin, lin, heads=2), lambda: pkg.forward_cross_attention(x.detach().requires_grad_(), None, lin, lin, lin, heads=2)):
        with pytest.raises((ValueError, RuntimeError, TypeError)):
            bad()


def test_from_several_threads(pkg, dev):
    """Each on a stream of its own, calls that need workspaces and calls that need none, at once."""
    g = torch.Generator(device="cuda").manual_seed(8)
    cases = []
    for queries, keys, heads, kv_heads, width in ((1, 5000, 8, 2, 128), (300, 700, 4, 4, 64), (2, 3000, 3, 3, 37), (64, 100, 2, 2, 256)):
        q, k, v = (torch.randn(1, n, m, width, generator=g, device="cuda").bfloat16() for n, m in ((queries, heads), (keys, kv_heads), (keys, kv_heads)))
        r, p = pkg.RotaryAxes((8, 16)), grid(queries, 2)
        cases.append((q, k, v, r, p, pkg.cross_attention(q, k, v), pkg.norm_heads(q, rotary=r, positions=p)))
    torch.cuda.synchronize()
    wrong = []

    def work(case):
        q, k, v, r, p, o, n = case
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                a, b = pkg.cross_attention(q, k, v), pkg.norm_heads(q, rotary=r, positions=p)
                if not (torch.equal(a, o) and torch.equal(b, n)):
                    wrong.append(q.shape)

    threads = [threading.Thread(target=work, args=(c,)) for c in cases * 2]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_more_tokens_than_a_launch_has_threads_for(pkg, dev):
    x = torch.randn(1, (4 << 23) + 1001, 1, 2, device="cuda").bfloat16()
    w, r = weight(2, torch.bfloat16), pkg.RotaryAxes((2,))
    p = torch.arange(x.shape[1], device="cuda", dtype=torch.int32)[:, None] % 1009
    got = pkg.norm_heads(x, w, rotary=r, positions=p)
    for at in (0, (4 << 23) - 500):
        part = slice(at, at + 1000)
        check_heads(got[:, part].contiguous(), expected_heads(x[:, part], w, True, 1e-6, (2,), 10000.0, True, p[part]))


def test_more_workgroups_than_a_launch_has_are_refused(pkg, dev):
    q = torch.zeros(1, 1, 1, 8, device="cuda", dtype=torch.bfloat16).expand(1 << 24, 1, 1, 8)
    with pytest.raises(pkg._lib.I8FError, match="unsupported"):
        pkg.cross_attention(q, q, q)
