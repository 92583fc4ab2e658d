"""Calls that the adapters and the norms between blocks refuse, whichever path takes them."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from test_gpu_adapters import factors_of, layer_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [5, 40, 300])
@pytest.mark.parametrize("width,features", [(250, 256), (256, 250), (255, 249), (249, 256)])
def test_a_bank_of_another_width_that_is_padded_to_the_same(pkg, dev, rows, width, features):
    """Rows of factors are padded to eight elements: the padded width says nothing of the columns."""
    lin, bank = layer_of(pkg, features, 128, torch.bfloat16), pkg.AdapterBank(factors_of(width, 128, (16,), torch.bfloat16))
    x, ids = torch.randn(rows, features, device=dev).bfloat16(), torch.zeros(rows, dtype=torch.int32, device=dev)
    with pytest.raises(ValueError, match=f"{width}"):
        pkg.forward_adapters(lin, x, bank, ids)
    fits = pkg.AdapterBank(factors_of(features, 128, (16,), torch.bfloat16))
    with pytest.raises(ValueError, match=f"{width}"):
        pkg.forward_adapters([lin, lin], x, [fits, bank], ids)


@pytest.mark.parametrize("rows", [5, 40])
def test_a_bank_without_factors_of_another_width(pkg, dev, rows):
    lin = layer_of(pkg, 256, 128, torch.bfloat16)
    x, ids = torch.randn(rows, 256, device=dev).bfloat16(), torch.zeros(rows, dtype=torch.int32, device=dev)
    for inputs, outputs in ((256, 64), (250, 128)):
        with pytest.raises(ValueError, match="features"):
            pkg.forward_adapters(lin, x, pkg.AdapterBank([None], in_features=inputs, out_features=outputs, device=dev), ids)


@pytest.mark.parametrize("rows", [5, 40])
def test_a_gradient_that_a_layer_going_alone_would_have(pkg, dev, rows):
    x, ids = torch.randn(rows, 256, device=dev).bfloat16(), torch.zeros(rows, dtype=torch.int32, device=dev)
    bank = pkg.AdapterBank(factors_of(256, 128, (16,), torch.bfloat16))
    lora = layer_of(pkg, 256, 128, torch.bfloat16)
    lora.lora_A, lora.lora_B = (torch.nn.Parameter(torch.randn(s, device=dev).bfloat16()) for s in ((16, 256), (128, 16)))
    for lin in (torch.nn.Linear(256, 128, device=dev, dtype=torch.bfloat16), lora):
        with torch.no_grad():
            want, base = pkg.forward_adapters(lin, x, bank, ids), lin(x)
        if not lin(x).requires_grad:   # (the layer itself has no gradient to lose)
            continue
        with pytest.raises(RuntimeError, match="gradient"):
            pkg.forward_adapters(lin, x, bank, ids)
        assert want.shape == base.shape
    assert torch.nn.Linear(256, 128, device=dev, dtype=torch.bfloat16)(x).requires_grad


def test_a_layer_with_parameters_that_ask_for_nothing_goes_on(pkg, dev):
    """Frozen parameters, or no grad mode: the call is as before."""
    x, ids = torch.randn(20, 256, device=dev).bfloat16(), torch.zeros(20, dtype=torch.int32, device=dev)
    bank = pkg.AdapterBank(factors_of(256, 128, (16,), torch.bfloat16))
    lin = torch.nn.Linear(256, 128, device=dev, dtype=torch.bfloat16)
    with torch.no_grad():
        want = pkg.forward_adapters(lin, x, bank, ids)
    lin.requires_grad_(False)
    assert torch.equal(pkg.forward_adapters(lin, x, bank, ids), want)


@pytest.mark.parametrize("rows", [5, 40])
def test_a_tangent_is_not_dropped(pkg, dev, rows):
    """Forward-mode derivatives, with and without grad mode, on either path."""
    lin, bank = layer_of(pkg, 256, 128, torch.bfloat16), pkg.AdapterBank(factors_of(256, 128, (16,), torch.bfloat16))
    x, ids = torch.randn(rows, 256, device=dev).bfloat16(), torch.zeros(rows, dtype=torch.int32, device=dev)
    w = torch.ones(256, device=dev).bfloat16()
    want = pkg.forward_adapters(lin, x, bank, ids), pkg.block_norm(x, x, pre_norm="rms", pre_weight=w)
    plain = torch.nn.Linear(256, 128, device=dev, dtype=torch.bfloat16).requires_grad_(False)
    with forward_ad.dual_level():
        dual, dual_w = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(w, torch.ones_like(w))
        calls = [lambda: pkg.forward_adapters(lin, dual, bank, ids), lambda: pkg.forward_adapters(plain, dual, bank, ids),
                 lambda: pkg.forward_adapters(lin, dual, bank, ids.view(rows, 1)[:, 0].expand(rows)), lambda: pkg.block_norm(dual, x), lambda: pkg.block_norm(x, dual),
                 lambda: pkg.block_norm(x, x, gate=dual), lambda: pkg.block_norm(x, x, pre_norm="rms", pre_weight=dual_w),
                 lambda: pkg.forward_block_norm([lin], dual, x, pre_norm="rms"), lambda: pkg.forward_block_norm([lin], x, x, pre_norm="rms", pre_weight=dual_w)]
        for i, call in enumerate(calls):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
                pytest.fail(f"call {i} dropped a tangent")
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):
                call()
        got = pkg.forward_adapters(lin, x, bank, ids), pkg.block_norm(x, x, pre_norm="rms", pre_weight=w)   # (others of the same level go on)
    assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(got[1], want[1]))
