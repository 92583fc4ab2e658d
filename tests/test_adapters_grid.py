"""Launches that would need 2^32 threads are refused on the host."""
import pytest
import torch


def test_a_side_tensor_is_chosen_where_its_launch_fits(L):
    """Four layers go into one launch, with a workgroup of 256 for 1024 columns of a row."""
    by_side = L.lib().i8f_adapters_by_side
    assert by_side(128, (1 << 25) - 1024, 16, 1) and not by_side(128, 1 << 25, 16, 1)
    assert by_side(32, 1 << 26, 16, 1) and not by_side(64, 1 << 26, 16, 1)


@pytest.mark.gpu
def test_more_outputs_than_a_launch_has_waves_for(pkg, L, dev):
    """A layer of odd width has a wave for every output."""
    from test_gpu_adapters import check, expected, factors_of, layer_of

    K, dtype = 8, torch.bfloat16
    x, ids = torch.randn(2, K, device=dev).to(dtype), torch.zeros(2, dtype=torch.int32, device=dev)
    for N in ((1 << 26) - 4, 1 << 26):
        lin, adapters = layer_of(pkg, K, N, dtype, bias=False), factors_of(K, N, (1,), dtype)
        bank = pkg.AdapterBank(adapters)
        if N < 1 << 26:
            check(pkg.forward_adapters(lin, x, bank, ids), *expected(pkg, lin, x, adapters, ids))
        else:
            with pytest.raises(L.I8FError, match="unsupported") as refused:
                pkg.forward_adapters(lin, x, bank, ids)
            assert refused.value.status == L.ERR_UNSUPPORTED
