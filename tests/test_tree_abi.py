"""w8a8_attention_tree_bf16 refuses an output whose heads share rows, on the host (no GPU needed)."""
import ctypes

import pytest

from w8a8 import _lib

F = ctypes.c_void_p(0x100000)     # never dereferenced: the calls are refused


def tree(ohs):
    L = _lib.lib()
    rc = L.w8a8_attention_tree_bf16(F, 1024, 256, F, 25600, 256, F, 25600, 256, 8, 1, 4, 6, 100, 256, F, 94, None, 0, 1.0, F, ohs,
                                    2048, None, F, 1 << 40, None)
    return rc, L.w8a8_last_error().decode()


@pytest.mark.parametrize("ohs", [0, 8, 248])
def test_heads_of_the_output_that_share_rows(ohs):
    rc, msg = tree(ohs)
    assert rc == _lib.W8A8_EINVAL and "o's heads" in msg, (rc, msg)
