"""Lengths that a BlockCache may be taken back to, on the GPU: those possible give what was put there, others raise."""
import pytest
import torch

from test_blocks_gpu import DEV, INT8, check, filled, rows, values
from w8a8 import attention, cache

pytestmark = pytest.mark.gpu


def holds(c, k, v, n):
    a, b = cache.read(c, 0, n)
    assert torch.equal(a, values(k[:, :n], c.dtype).bfloat16()) and torch.equal(b, values(v[:, :n], c.dtype).bfloat16())


def test_back_and_back_again():
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = rows(g, 2, 700, 128)
    c = filled(2, 700, 128, INT8)
    q = (torch.randn(4, 2, 128, generator=g, device=DEV) * 0.1).bfloat16()
    cache.append(c, k[:, :600], v[:, :600], 0)
    for n in (600, 577, 576, 515, 512, 64):
        holds(c, k, v, n)
    x, y = rows(g, 2, 10, 128)
    k2, v2 = k.clone(), v.clone()
    k2[:, 128:138], v2[:, 128:138] = x, y
    cache.append(c, x, y, 128)
    for n in (138, 130, 128, 64):
        holds(c, k2, v2, n)
    before = c.data.clone()
    for f in (lambda: cache.append(c, x, y, 100), lambda: cache.read(c, 0, 100), lambda: attention.block_attention(q, c, 100),
              lambda: attention.block_attention(q, c, 100, out=torch.empty_like(q))):
        with pytest.raises(ValueError, match="block 1"):
            f()
    assert torch.equal(before, c.data)
    for n in (64, 138):
        check(q, c, n, k2, v2)
    cache.append(c, k[:, 64:101], v[:, 64:101], 64)  # block 1 is put there again
    holds(c, k, v, 100)
    check(q, c, 100, k, v)
    cache.append(c, k[:, 100:700], v[:, 100:700], 100)
    holds(c, k, v, 700)


def test_a_copy_of_another_cache():
    """What torch writes into `data` replaces what was known of it."""
    g = torch.Generator(device=DEV).manual_seed(2)
    k, v = rows(g, 1, 600, 256)
    long, short = filled(1, 600, 256, INT8), filled(1, 600, 256, INT8)
    cache.append(long, k, v, 0)
    cache.append(short, k[:, :100], v[:, :100], 0)
    long.data.copy_(short.data)
    holds(long, k, v, 100)
    cache.append(long, k[:, 100:150], v[:, 100:150], 100)
    holds(long, k, v, 150)
    with torch.inference_mode():
        c = cache.BlockCache(1, 600, 256)
        cache.append(c, k, v, 0)
        cache.append(c, k[:, :10], v[:, :10], 0)
        with pytest.raises(ValueError):
            cache.read(c, 0, 70)
        c.data.copy_(short.data)
        holds(c, k, v, 100)


def test_captured_append():
    """A graph's appends happen when it is replayed: lengths of such a cache are the caller's."""
    g = torch.Generator(device=DEV).manual_seed(3)
    k, v = rows(g, 1, 600, 128)
    c = filled(1, 600, 128, INT8)
    cache.append(c, k[:, :100], v[:, :100], 0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(c, k[:, 100:], v[:, 100:], 100)
    for _ in range(3):
        holds(c, k, v, 100)
        graph.replay()
        holds(c, k, v, 600)
        cache.append(c, k[:, :100], v[:, :100], 0)
