"""Calls that the adapters and the norms between blocks refuse, whichever path takes them."""
import pytest
import torch

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
