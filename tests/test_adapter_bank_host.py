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


@pytest.mark.parametrize("name", ["down", "up", "scale", "first_rank", "count", "max_rank", "in_features", "out_features", "dtype", "device", "ranks"])
def test_nothing_is_assigned_to_a_bank(pkg, name):
    """A tensor that took another's place would be used by one path and not by the other."""
    bank = bank_of(pkg)
    kept = dict(bank.__dict__)
    value = getattr(bank, name)
    with pytest.raises(AttributeError, match=name):
        setattr(bank, name, value.clone() if isinstance(value, torch.Tensor) else value)
    assert bank.__dict__.keys() == kept.keys() and all(bank.__dict__[k] is v for k, v in kept.items())


def test_what_is_written_into_a_bank_is_in_both(pkg):
    bank = bank_of(pkg)
    bank.scale[0] = 4.0
    bank.down.mul_(2)
    assert bank._native[2][0] == 4.0 and torch.equal(bank._native[0], parts(pkg, bank)[0])


@pytest.mark.parametrize("given", [torch.float16, torch.bfloat16, torch.float32, torch.float64])
@pytest.mark.parametrize("size,scale", [(1.0, 1.0), (2.0 ** -13, 2.0 ** 20), (300.0, 1e-6), (1e-9, 3e9), (1e6, -1e-7), (1e-30, 1e30), (1.0, 1e-38), (1.0, 3e38)])
def test_second_factors_of_a_binary16_bank_are_near_one(pkg, given, size, scale):
    """scale * up is what it was, up to one rounding of up to binary16; up reaches 1 where the scale leaves it room."""
    if given == torch.float16 and not 2.0 ** -14 <= size <= 300:
        pytest.skip("no binary16 number")
    up, down = (torch.linspace(-1.0, 1.7, 60).view(12, 5) * size).to(given), torch.ones(5, 8)
    bank = pkg.AdapterBank([(down, up, scale), None, (down, up * 0, scale), (down, up, 0.0)], dtype=torch.float16, device="cpu")
    got = bank.up.view(-1)[:12 * 16].view(12, 16)[:, :5].double() * bank.scale[0].double()
    want = up.double() * scale
    top = want.abs().max()
    assert torch.isfinite(bank.scale).all() and bank.scale[0] != 0
    assert ((got - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -23 * want.abs() + 2.0 ** -25 * top).all()
    assert 1.0 <= bank.up.abs().max() <= 2.0
    assert not bank.up.view(-1)[12 * 16:2 * 12 * 16].any() and bank.scale[3] == 0


def test_second_factors_of_a_bfloat16_bank_and_of_no_finite_ones_stay(pkg):
    up, down = torch.full((6, 3), 2.0 ** -10), torch.ones(3, 8)
    bank = pkg.AdapterBank([(down, up, 7.0)], dtype=torch.bfloat16, device="cpu")
    assert bank.scale[0] == 7.0 and bank.up.max() == 2.0 ** -10
    for value in (float("inf"), float("nan")):
        up[2, 1] = value
        bank = pkg.AdapterBank([(down, up, 7.0)], dtype=torch.float16, device="cpu")
        assert bank.scale[0] == 7.0 and bank.up[0] == 2.0 ** -10
    bank = pkg.AdapterBank([(torch.ones(0, 8), torch.ones(6, 0), 7.0)], dtype=torch.float16, device="cpu")
    assert bank.max_rank == 0 and bank.scale[0] == 7.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("alpha,strength", [(3.0, 0.7), (None, 1e-5), (None, -1.3)])
def test_a_patch_s_strength_does_not_go_through_16_bits(pkg, dtype, alpha, strength):
    """Factors of a patch in the activations' type are kept as they are; alpha, rank and strength are the scale."""
    g = torch.Generator().manual_seed(5)
    up, down, mid = (torch.randn(s, generator=g).to(dtype) for s in ((6, 4), (4, 10), (4, 4)))
    for middle in (None, mid):
        patch = pkg.INT8LoRAPatchAdapter(set(), (up, down, alpha, middle, None, None), 0.01)
        bank = pkg.AdapterBank.from_patches([None, (patch, strength)], dtype=dtype, device="cpu")
        scale = strength if alpha is None else alpha / 4 * strength
        assert torch.equal(bank.down[:4, :10], down if middle is None else mid @ down) and bank.ranks == [0, 4]
        got = bank.up.view(6, 16)[:, :4].double() * bank.scale[1].double()
        assert (got - up.double() * scale).abs().max() <= 2.0 ** -23 * (up.double() * scale).abs().max()


def test_a_bank_of_one_s_own_kind_has_attributes_of_its_own(pkg):
    class Named(pkg.AdapterBank):
        def __init__(self, *args, **kwargs):
            super().__init__(*args, **kwargs)
            self.name = "a"

    bank = Named([(torch.ones(3, 8), torch.ones(6, 3))], dtype=torch.bfloat16, device="cpu")
    bank.name = "b"
    assert bank.name == "b"
    with pytest.raises(AttributeError, match="up"):
        bank.up = bank.up.clone()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_bank_of_shapes_alone(pkg, dtype):
    """On the meta device there are no values to look at."""
    bank = pkg.AdapterBank([(torch.ones(3, 8, device="meta"), torch.ones(6, 3, device="meta")), None], dtype=dtype, device="meta")
    assert bank.up.is_meta and bank.up.shape == (96,) and bank.up.dtype == dtype and bank.scale.shape == (2,)
