"""An adapter bank keeps what it was laid out with (no GPU)."""
import copy

import pytest
import torch


def bank_of(pkg, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(2)
    return pkg.AdapterBank([(torch.randn(3, 10, generator=g), torch.randn(6, 3, generator=g), 0.5), None], dtype=dtype, device="cpu")


def parts(pkg, bank):
    """What the general path and a compiled program take of a bank."""
    return pkg.compile_ops.bank_args(bank)


def test_the_host_path_and_the_general_one_take_the_same_tensors(pkg):
    for bank in (bank_of(pkg), copy.copy(bank_of(pkg)), copy.deepcopy(bank_of(pkg))):
        assert all(a is b for a, b in zip(bank._native, parts(pkg, bank))) and bank._native[6:] == (10, 6)


@pytest.mark.parametrize("name", ["down", "up", "scale", "first_rank", "count", "max_rank", "in_features", "out_features", "dtype", "device", "ranks", "other"])
def test_nothing_is_assigned_to_a_bank(pkg, name):
    """A tensor that took another's place would be used by one path and not by the other."""
    bank = bank_of(pkg)
    kept = dict(bank.__dict__)
    value = getattr(bank, name, 1)
    with pytest.raises(AttributeError, match=name):
        setattr(bank, name, value.clone() if isinstance(value, torch.Tensor) else value)
    assert bank.__dict__.keys() == kept.keys() and all(bank.__dict__[k] is v for k, v in kept.items())


def test_what_is_written_into_a_bank_is_in_both(pkg):
    bank = bank_of(pkg)
    bank.scale[0] = 4.0
    bank.down.mul_(2)
    assert bank._native[2][0] == 4.0 and torch.equal(bank._native[0], parts(pkg, bank)[0])
