"""The attention's workspace: every part of it begins at a whole 16-byte piece (no GPU)."""
import ctypes
import random


def args(L, batch, queries, keys, heads, kv_heads, width, **over):
    a = L._AttentionArgs(q=1 << 20, k=1 << 40, v=1 << 41, out=1 << 42, batch=batch, queries=queries, keys=keys, heads=heads, kv_heads=kv_heads, width=width, q_batch=queries * heads * width,
                         q_token=heads * width, q_head=width, k_batch=keys * kv_heads * width, k_token=kv_heads * width, k_head=width, v_batch=keys * kv_heads * width,
                         v_token=kv_heads * width, v_head=width, dtype=L.BF16, scale=1.0)
    for k, v in over.items():
        setattr(a, k, v)
    return a


def size(L, *s, **over):
    return L.lib().i8f_attention_workspace_bytes(ctypes.byref(args(L, *s, **over)))


def test_copies_begin_at_whole_pieces(L):
    """What lies in front of the copies, the splits' results with two statistics to a row, is 8 bytes off for odd numbers of rows if nothing rounds it."""
    for s in ((1, 1, 1536, 1, 1, 37), (1, 1, 4097, 1, 1, 37), (1, 3, 5000, 1, 1, 33), (1, 5, 3000, 3, 1, 199)):
        whole = size(L, *s[:5], -(-s[5] // 8) * 8)   # (the same call over whole pieces: the splits alone)
        copies = 2 * s[0] * -(-s[5] // 8) * 8 * (s[1] * s[3] + 2 * s[2] * s[4])
        assert whole > 0 and whole % 16 == 0 and size(L, *s) == whole + copies, s
    rng = random.Random(3)
    for _ in range(3000):
        kv = rng.randint(1, 9)
        s = (rng.randint(1, 3), rng.choice((1, 1, 3, rng.randint(1, 300))), rng.randint(1, 20000), kv * rng.choice((1, 1, 3)), kv, rng.randint(1, 256))
        assert size(L, *s) % 16 == 0 and size(L, *s, q=(1 << 20) + 2) % 16 == 0, s
