"""w8a8_reorder_rows refuses an index that lies in what it changes, on the host (no GPU needed)."""
import ctypes

import pytest

from w8a8 import _lib

BASE = 0x100000     # never dereferenced: the calls are refused first


def reorder(index, n=4, size=8, outer=1, stride=0, **tensor):
    r = dict(data=BASE, outer_stride=1 << 20, axis_stride=4096, run_stride=0, runs=1, run_bytes=4096)
    other = _lib.Rows(0x9000000, 1 << 44, 1 << 41, 0, 1, 1 << 40)           # too large a tensor, which is refused last
    rows = (_lib.Rows * 2)(other, _lib.Rows(*{**r, **tensor}.values()))
    L = _lib.lib()
    rc = L.w8a8_reorder_rows(rows, 2, ctypes.c_void_p(index), stride, n, size, outer, None)
    return rc, L.w8a8_last_error().decode()


@pytest.mark.parametrize("call", [
    dict(index=BASE), dict(index=BASE - 24),                                    # its last entry is the first row's first
    dict(index=BASE + 4 * 4096 - 8),                                            # the last changed row's last bytes
    dict(index=BASE + (1 << 20) + 16, outer=2), dict(index=BASE - 48, outer=2, stride=4),
    dict(index=BASE + 4096 * 3 + 1024, runs=3, run_stride=1024, run_bytes=256),
], ids=str)
def test_an_index_among_the_changed_rows(call):
    rc, msg = reorder(**call)
    assert rc == _lib.W8A8_EINVAL and "index lies in tensor 1" in msg, (rc, msg)


@pytest.mark.parametrize("call", [
    dict(index=BASE - 32), dict(index=BASE + 4 * 4096),                         # before the first, in the first row that is only read
    dict(index=BASE - 64, outer=2, stride=4), dict(index=BASE, runs=0),         # an empty tensor
], ids=str)
def test_an_index_beside_them(call):
    rc, msg = reorder(**call)
    assert rc == _lib.W8A8_ENOTSUP and "tensor 0 too large" in msg, (rc, msg)
