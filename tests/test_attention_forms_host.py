"""Which form of the attention a size reaches, on the host (no GPU): a rule that changes cannot leave a form without its tests."""
import ctypes

from attention_forms import SIZES, form_of

INVALID = -1


def test_sizes_reach_the_forms_that_they_are_tested_for(L):
    """Every width of a kernel in every form it has."""
    widths = {form: set() for form in SIZES}
    for form, sizes in SIZES.items():
        for size in sizes:
            name, padded = form_of(L, size)
            assert name == form, (size, name)
            widths[form].add(padded)
    assert all(w == {64, 96, 128, 192, 256} for form, w in widths.items() if form != "eight") and widths["eight"] == {128}


def test_a_plan_of_invalid_or_empty_calls_is_refused(L):
    out, plan = [ctypes.byref(ctypes.c_int64()) for _ in range(4)], L.lib().i8f_internal_attention_plan
    valid = dict(q=1 << 20, k=1 << 22, v=1 << 23, out=1 << 24, batch=1, queries=1, keys=1, heads=1, kv_heads=1, width=8, dtype=L.BF16, scale=1.0)
    assert plan(ctypes.byref(L._AttentionArgs(**valid)), *out) == 0
    assert plan(None, *out) == INVALID and plan(ctypes.byref(L._AttentionArgs(**valid)), None, *out[1:]) == INVALID
    for bad in ({"keys": 0}, {"width": 0}, {"scale": 0.0}):
        assert plan(ctypes.byref(L._AttentionArgs(**{**valid, **bad})), *out) == INVALID, bad


def test_eight_waves_take_full_rounds_of_full_workgroups(L):
    """256 rows to a workgroup where they are nearly all a call's own, and one workgroup to a CU where the last round is nearly full."""
    for size in ((1, 8192, 8192, 40, 40, 128), (1, 32768, 4096, 8, 8, 128), (256, 256, 4096, 16, 4, 128), (64, 250, 5000, 16, 16, 120), (9, 65536, 4096, 1, 1, 97)):
        assert form_of(L, size) == ("eight", 128), size
    for size in ((64, 64, 4096, 16, 16, 128), (64, 128, 4096, 16, 16, 128), (64, 300, 4096, 32, 32, 128), (22, 2048, 4096, 8, 8, 128), (57, 2300, 4096, 8, 8, 128), (1, 8192, 4000, 40, 40, 128),
                 (1, 4096, 4096, 40, 40, 128), (1, 8192, 8192, 40, 40, 64), (1, 8192, 8192, 40, 40, 96), (1, 8192, 8192, 40, 40, 256)):
        assert form_of(L, size)[0] == "together", size
