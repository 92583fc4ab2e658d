"""Sizes by the form of the attention that they reach, shared by the host test that asks the library for it and the GPU tests."""
import ctypes

# (batch, queries, keys, heads, kv heads, width)
WIDTHS = (64, 40, 96, 72, 128, 120, 192, 136, 256, 200, 37)
SIZES = {
    "apart": [(2, 9, 200, 6, 3, w) for w in WIDTHS],
    "apart, split": [(2, 2, 3001, 4, 2, w) for w in WIDTHS],
    "together": [(3, 150, 203, 10, 5, w) for w in WIDTHS],
    "together, split": [(3, 150, 705, 10, 5, w) for w in WIDTHS],
    "eight": [(2, 4050, 4113, 32, 32, w) for w in (128, 120, 101)],
}


def form_of(L, size):
    """(name of the form as above, width of its kernel) of a call on contiguous operands."""
    batch, queries, keys, heads, kv_heads, width = size
    a = L._AttentionArgs(q=1 << 20, k=1 << 40, v=1 << 41, out=1 << 42, batch=batch, queries=queries, keys=keys, heads=heads, kv_heads=kv_heads, width=width, q_batch=queries * heads * width,
                         q_token=heads * width, q_head=width, k_batch=keys * kv_heads * width, k_token=kv_heads * width, k_head=width, v_batch=keys * kv_heads * width,
                         v_token=kv_heads * width, v_head=width, dtype=L.BF16, scale=1.0)
    waves, apart, splits, padded = (ctypes.c_int64() for _ in range(4))
    assert L.lib().i8f_internal_attention_plan(ctypes.byref(a), *(ctypes.byref(x) for x in (waves, apart, splits, padded))) == 0
    name = "apart" if apart.value else "eight" if waves.value == 8 else "together"
    return name + (", split" if splits.value > 1 else ""), padded.value
