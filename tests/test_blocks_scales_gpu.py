"""Attention over the 8-bit block cache (attention.block_attention) where its blocks' value scales lie far apart, every column
for itself: against its definition in 64 bits, with the tolerance of test_blocks_gpu.check, which is relative to what a column
itself adds up to."""
import math

import pytest
import torch

from test_blocks_gpu import DEV, E4M3, INT8, check, filled, rows
from w8a8 import attention, cache

pytestmark = pytest.mark.gpu

CASES = [  # H, KV, D, N, n, window, sinks: every tile of rows, parts of one block and of many
    (8, 1, 512, 1, 1024, 0, 0), (16, 2, 128, 1, 4096, 0, 0), (8, 1, 256, 1, 960, 512, 64), (8, 1, 256, 4, 1024, 0, 0), (8, 2, 512, 5, 640, 0, 0),
    (24, 2, 128, 5, 1024, 300, 70), (8, 1, 512, 33, 704, 0, 0), (8, 1, 256, 130, 704, 200, 65), (4, 1, 128, 100, 1024, 0, 0), (256, 8, 128, 96, 768, 0, 0),
]


def queries(g, H, N, D):
    return (torch.randn(H, N, D, generator=g, device=DEV) * 2 * D ** -0.5).bfloat16()


@pytest.mark.parametrize("dtype", [INT8, E4M3])
@pytest.mark.parametrize("size", [1e4, 1e6, 1e8])
@pytest.mark.parametrize("H,KV,D,N,n,window,sinks", CASES)
def test_one_value_far_out(H, KV, D, N, n, window, sinks, size, dtype):
    """One value of one row, in the first block, one between or the last: the other columns are those of all the other blocks."""
    g = torch.Generator(device=DEV).manual_seed(H + D + N + n)
    q = queries(g, H, N, D)
    for at in (3, n // 2 + 1, n - 1):
        k, v = rows(g, KV, n, D)
        v[:, at, 5] = -size
        c = filled(KV, n, D, dtype)
        cache.append(c, k, v, 0)
        check(q, c, n, k, v, window, sinks)


@pytest.mark.parametrize("dtype", [INT8, E4M3])
@pytest.mark.parametrize("H,KV,D,N,n,window,sinks", CASES)
def test_blocks_of_their_own_columns(H, KV, D, N, n, window, sinks, dtype):
    """Every block's values lie in columns of its own, of a size of its own (2^-20 .. 2^20, in any order)."""
    g = torch.Generator(device=DEV).manual_seed(H * 3 + D + N + n)
    q = queries(g, H, N, D)
    k, v = rows(g, KV, n, D)
    block = torch.arange(n, device=DEV) // 64
    size = torch.exp2(40.0 * torch.rand(n // 64, generator=g, device=DEV) - 20.0)
    mine = block[:, None] % 16 == torch.arange(D, device=DEV)[None] % 16
    v = (v.float() * size[block][:, None] * mine).bfloat16()
    c = filled(KV, n, D, dtype)
    cache.append(c, k, v, 0)
    check(q, c, n, k, v, window, sinks)
    k2, v2 = rows(g, KV, n + 30, D)  # .. and rows behind the last whole block
    k2[:, :n], v2[:, :n] = k, v
    c = filled(KV, n + 30, D, dtype)
    cache.append(c, k2, v2, 0)
    check(q, c, n + 30, k2, v2, window, sinks)


def test_many_weights_beside_a_large_one():
    """A key with most of the weight, whose value is 0, and a million with 2^-25 of it each, whose values are 1.

    The weights beside the large one are fp16 numbers 2^7 as large, rounded by at most 2^-25: 2^-32 of the large one, 2^-6.5 of
    their own.  The output's rounding adds 2^-8, the sum over p keys in fp32 (64 of them at a time) 2^-9 at most."""
    H, D, N, n = 8, 128, 2112, 1 << 20
    x = 17.625
    q = torch.zeros(H, N, D, device=DEV, dtype=torch.bfloat16)
    q[..., 0] = 1.0
    k = torch.zeros(1, n, D, device=DEV, dtype=torch.bfloat16)
    v = torch.ones(1, n, D, device=DEV, dtype=torch.bfloat16)
    k[0, 0, 0], v[0, 0] = x, 0.0
    c = filled(1, n, D, INT8)
    cache.append(c, k, v, 0)
    w = torch.arange(n - N, n, device=DEV).double() * math.exp(-x)
    want = (w / (1.0 + w))[None, :, None]
    got = attention.block_attention(q, c, n).double()
    assert ((got - want).abs() <= (2.0 ** -6.5 + 2.0 ** -8 + 2.0 ** -9) * want).all()
