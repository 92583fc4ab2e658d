"""Copies of operands off 16-byte pieces whose size passes what can be counted: refused before anything is launched (no GPU)."""
import ctypes

from test_attention_host import UNSUPPORTED
from test_attention_workspace_host import args


def test_copies_that_no_memory_holds_are_refused(L):
    """Expanded operands have few elements and many states: 2^25 batches of 2^30 states of 512 bytes are 2^64, which 64 bits take for nothing."""
    for batch, keys, width in ((1 << 25, 1 << 30, 250), (1 << 24, 1 << 30, 250), (1 << 27, 1 << 28, 249), (1 << 23, 1 << 29, 255)):
        a = args(L, batch, 1, keys, 1, 1, width, q_batch=0, k_batch=0, k_token=0, v_batch=0, v_token=0)
        assert L.lib().i8f_attention(ctypes.byref(a), None) == UNSUPPORTED, (batch, keys, width)
        assert L.lib().i8f_attention_workspace_bytes(ctypes.byref(a)) == 0
