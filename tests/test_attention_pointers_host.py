"""Addresses that the C interface refuses before any launch: off their elements, or inside the results (no GPU)."""
import pytest

from test_attention_host import INVALID, UNSUPPORTED, _attention, _heads


def test_lengths_and_masks_off_their_elements(L):
    for kind, size in ((0, 4), (1, 8)):
        for off in (1, 2, size - 1, size // 2):
            assert _attention(L, key_lengths=(1 << 30) + off, lengths_type=kind) == INVALID, (kind, off)
    for kind, size in ((1, 2), (2, 2), (3, 4)):
        for off in range(1, size):
            assert _attention(L, key_mask=(1 << 30) + off, mask_type=kind, mask_batch=5, mask_key=1) == INVALID, (kind, off)
    assert _attention(L, queries=0, key_lengths=(1 << 30) + 2, lengths_type=0) == INVALID    # (arguments are checked for empty calls too)


def test_results_on_lengths_and_masks(L):
    """out is [2, 3, 4, 8] in 16 bits: 384 bytes from 2^24 on."""
    end = (1 << 24) + 384
    for at in (1 << 24, end - 8, (1 << 24) - 4):
        assert _attention(L, key_lengths=at, lengths_type=0) == INVALID, at
    for at in (1 << 24, end - 16, (1 << 24) - 8):
        assert _attention(L, key_lengths=at, lengths_type=1) == INVALID, at
    for kind, size in ((0, 1), (1, 2), (3, 4)):     # [2, 5] elements, the second row 7 behind the first
        for at in (1 << 24, end - size, (1 << 24) - 11 * size):
            assert _attention(L, key_mask=at, mask_type=kind, mask_batch=7, mask_key=1) == INVALID, (kind, at)
        assert _attention(L, key_mask=(1 << 24) - 40, mask_type=kind, mask_batch=1 << 20, mask_key=1 << 10) == INVALID   # (between its elements as well)


def test_positions_rates_and_weights_off_their_elements(L):
    for kind, size in ((0, 4), (1, 8), (2, 4), (3, 8)):
        for off in (1, size // 2, size - 1):
            assert _heads(L, {"positions_type": kind, "positions": (1 << 21) + off}, {}) == INVALID, (kind, off)
    for off in (1, 4):
        assert _heads(L, {"rates": (1 << 20) + off}, {}) == INVALID, off
    assert _heads(L, None, {"weight": 17, "weight_dtype": L.BF16}) == INVALID
    for off in (1, 2, 3):
        assert _heads(L, None, {}, {"weight": 16 + off, "weight_dtype": L.F32}) == INVALID, off


@pytest.mark.parametrize("first", [True, False])
def test_results_on_positions_rates_and_weights(L, first):
    """Results of [1, 2, 3, 8] in 16 bits, 96 bytes; positions [2, 2], four rates, weights of eight."""
    at = (1 << 24) if first else (1 << 24) + (1 << 20)
    for kind, size in ((0, 4), (1, 8)):
        for p in (at, at + 96 - size, at - 3 * size):
            assert _heads(L, {"positions_type": kind, "positions": p}, {}, {}) == INVALID, (kind, p)
    for r in (at, at + 88, at - 24):
        assert _heads(L, {"rates": r}, {}, {}) == INVALID, r
    for w in (at, at + 92, at - 12):
        for i in range(2):
            groups = [{}, {}]
            groups[i] = {"weight": w, "weight_dtype": L.BF16}
            assert _heads(L, None, *groups) == INVALID, (w, i)
    assert _heads(L, {"norm": 1}, {"weight": at + 64, "weight_dtype": L.F32}, {"weight": at + 64, "weight_dtype": L.F32}) == INVALID


def test_extents_whose_bytes_pass_64_bits(L):
    for over in ({"token_stride": 1 << 59}, {"head_stride": 1 << 58}):
        assert _heads(L, None, over) == UNSUPPORTED, over
    assert _heads(L, {"position_token": 1 << 60}, {}) == UNSUPPORTED and _heads(L, {"position_axis": 1 << 58}, {}) == UNSUPPORTED
    for over in ({"k_token": 1 << 58}, {"q_head": 1 << 58}, {"v_batch": 1 << 60}, {"key_mask": 1 << 30, "mask_type": 3, "mask_batch": 1 << 60}):
        assert _attention(L, **over) == UNSUPPORTED, over
