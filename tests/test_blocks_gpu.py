"""The 8-bit block cache (cache.BlockCache, append, read) and attention over it (attention.block_attention) against
their definition in 64 bits."""
import math

import pytest
import torch

from w8a8 import attention, cache

DEV = "cuda"
INT8, E4M3 = torch.int8, torch.float8_e4m3fn
pytestmark = pytest.mark.gpu


def values(x, dtype):
    """[KV, n, D] bf16 -> what the cache holds for them, in 64 bits."""
    out = x.double()
    for b in range(x.shape[1] // 64):
        rows = x[:, 64 * b:64 * b + 64].float()
        # (divided by a tensor: by a number torch multiplies with its reciprocal on the GPU)
        s = rows.abs().amax((1, 2), keepdim=True).clamp(min=1e-8)
        s = s / torch.tensor(127.0, device=DEV) if dtype == INT8 else s * torch.tensor(1.0 / 448.0, device=DEV)
        y = rows / s
        if dtype == INT8:
            c = torch.round(y).clamp(-127, 127).nan_to_num(0.0).double()
        else:
            c = y.cpu().to(E4M3).to(DEV).double()
        out[:, 64 * b:64 * b + 64] = c * s.double()
    return out


def filled(KV, capacity, D, dtype):
    """A cache whose memory holds what is none of it."""
    c = cache.BlockCache(KV, capacity, D, dtype)
    c.data.fill_(255)
    return c


def rows(g, KV, n, D, spread=0.0):
    k, v = (torch.randn(KV, n, D, generator=g, device=DEV) for _ in range(2))
    if spread:  # blocks of very different sizes
        f = torch.exp(spread * torch.randn(2, KV, (n + 63) // 64, 1, generator=g, device=DEV)).repeat_interleave(64, 2)[:, :, :n]
        k, v = k * f[0].clamp(max=4.0), v * f[1]
    return k.bfloat16(), v.bfloat16()


def seen(n, N, window, sinks):
    p = torch.arange(n - N, n, device=DEV)[:, None]
    j = torch.arange(n, device=DEV)[None]
    return (j <= p) if not window else (j <= p) & ((p - j < window) | (j < sinks))


def reference(q, k, v, window, sinks, scale):
    """(o, sum of weight x |v|, lse) in 64 bits; k, v: what the cache holds."""
    H, N, _ = q.shape
    KV, n, _ = k.shape
    m = seen(n, N, window, sinks)
    o, a, lse = [], [], []
    for h in range(H):
        g = h // (H // KV)
        x = (scale * (q[h].double() @ k[g].t().contiguous())).masked_fill(~m, -math.inf)
        w = torch.softmax(x, -1)
        o.append(w @ v[g])
        a.append(w @ v[g].abs())
        lse.append(torch.logsumexp(x, -1))
    return torch.stack(o), torch.stack(a), torch.stack(lse)


def check(q, c, n, kx, vx, window=0, sinks=0, scale=1.0, length=None):
    got, lse = attention.block_attention(q, c, n if length is None else length, window, sinks, scale, return_lse=True)
    k, v = values(kx[:, :n], c.dtype), values(vx[:, :n], c.dtype)
    o, a, want = reference(q if q.dim() == 3 else q[:, None], k, v, window, sinks, scale)
    # the output's rounding (bf16: 2^-8), the weights' (bf16 for rows behind the last whole block, else fp16: 2^-11, and
    # 2^-25 of a weight of 1 below its normal numbers, for at most 2^12 such rows of any one row's), and the scores': sums of
    # D <= 512 products of sum |q k| <= 32 in fp32 (2^-10)
    wr = 2.0 ** -8 if n % 64 else 2.0 ** -11
    tol = 2.0 ** -8 * o.abs() + (wr + 2.0 ** -10 + 2.0 ** -13) * a + 1e-30
    err = (got.view(o.shape).double() - o).abs()
    assert bool((err <= tol).all()), (err / tol).max().item()
    assert bool(((lse.view(want.shape).double() - want).abs() <= 2.0 ** -9 + 2.0 ** -22 * want.abs()).all())
    plain = attention.block_attention(q, c, n if length is None else length, window, sinks, scale)
    assert torch.equal(plain, got)
    return got


@pytest.mark.parametrize("dtype", [INT8, E4M3])
@pytest.mark.parametrize("KV,D", [(1, 512), (2, 256), (3, 128)])
def test_rows(KV, D, dtype):
    """What is read back is the definition's, whichever way the rows came; rows past the last are left alone."""
    g = torch.Generator(device=DEV).manual_seed(D)
    k, v = rows(g, KV, 400, D, spread=3.0)
    k[:, 128:192] = 0.0
    for steps in ([400], [1] * 200, [63, 1, 64, 65, 2, 128, 77], [64, 64, 64], [130, 140, 3, 60, 67]):
        c, n = filled(KV, 400, D, dtype), 0
        for m in steps:
            cache.append(c, k[:, n:n + m], v[:, n:n + m], n)
            n += m
            if len(steps) < 10 or n % 61 == 0:
                for start in (0, n // 2, max(0, n - 1), n):
                    a, b = cache.read(c, start, n)
                    assert torch.equal(a, values(k[:, :n], dtype)[:, start:].bfloat16()) and a.shape == (KV, n - start, D)
                    assert torch.equal(b, values(v[:, :n], dtype)[:, start:].bfloat16())


@pytest.mark.parametrize("dtype", [INT8, E4M3])
def test_taken_back(dtype):
    """Rows written, taken back and written anew: as if the first ones had never been."""
    g = torch.Generator(device=DEV).manual_seed(3)
    KV, D = 2, 256
    k, v = rows(g, KV, 500, D)
    dev = torch.zeros(1, dtype=torch.int32, device=DEV)
    c, n = filled(KV, 500, D, dtype), 0
    for m, back, onto in ((100, 0, None), (40, 36, None), (60, 60, None), (30, 29, None), (128, 100, None), (90, 64, None), (1, 1, None),
                          (200, 0, 128), (5, 5, None), (64, 1, None)):
        x, y = rows(g, KV, m, D)
        keep = m - back
        x[:, :keep], y[:, :keep] = k[:, n:n + keep], v[:, n:n + keep]
        dev.fill_(n)
        cache.append(c, x, y, dev if m % 2 else n)
        n += keep
        if onto is not None:  # a whole number of blocks may be any
            n = onto
        a, b = cache.read(c, 0, n)
        assert torch.equal(a, values(k[:, :n], dtype).bfloat16()) and torch.equal(b, values(v[:, :n], dtype).bfloat16())


CASES = [  # H, KV, D, N, n, window, sinks
    (8, 1, 512, 1, 1, 0, 0), (8, 1, 512, 1, 63, 0, 0), (8, 1, 512, 1, 64, 0, 0), (8, 1, 512, 1, 65, 0, 0), (8, 1, 512, 1, 3659, 0, 0),
    (8, 1, 256, 1, 700, 512, 4), (8, 1, 256, 1, 640, 512, 0), (4, 4, 128, 1, 129, 1, 0), (4, 4, 128, 1, 130, 1, 1), (16, 1, 256, 1, 1000, 64, 64),
    (12, 4, 128, 5, 5, 0, 0), (12, 4, 128, 5, 69, 0, 0), (8, 1, 512, 5, 1027, 0, 0), (8, 1, 512, 7, 256, 100, 3), (32, 8, 128, 3, 2000, 0, 0),
    (5, 5, 256, 17, 333, 50, 70), (8, 2, 512, 64, 64, 0, 0), (8, 2, 512, 33, 400, 0, 0), (8, 1, 256, 130, 700, 0, 0), (8, 1, 256, 300, 300, 64, 4),
    (3, 1, 128, 200, 1000, 129, 130), (24, 2, 128, 100, 512, 512, 1), (1, 1, 512, 70, 200, 5, 200), (20, 1, 256, 9, 449, 0, 0),
]


@pytest.mark.parametrize("dtype", [INT8, E4M3])
@pytest.mark.parametrize("H,KV,D,N,n,window,sinks", CASES)
def test_attention(H, KV, D, N, n, window, sinks, dtype):
    g = torch.Generator(device=DEV).manual_seed(H * 7 + D + N * 3 + n)
    k, v = rows(g, KV, n + 100, D)
    c = filled(KV, n + 100, D, dtype)
    cache.append(c, k[:, :n], v[:, :n], 0)
    q = (torch.randn(H, N, D, generator=g, device=DEV) * 2 * D ** -0.5).bfloat16()
    got = check(q, c, n, k, v, window, sinks)
    # the length in device memory; other scales; strided operands; one token without the middle dimension
    dev = torch.tensor([n], dtype=torch.int32, device=DEV)
    check(q, c, n, k, v, window, sinks, length=dev)
    check((q.float() * 8).bfloat16(), c, n, k, v, window, sinks, 0.125)
    wide = torch.zeros(N, H, D + 16, device=DEV, dtype=torch.bfloat16)
    view = wide.transpose(0, 1)[:, :, 8:D + 8]
    view.copy_(q)
    out = torch.full((N, H, D), 7.0, device=DEV, dtype=torch.bfloat16)
    attention.block_attention(view, c, n, window, sinks, out=out.transpose(0, 1))
    assert torch.equal(out.transpose(0, 1), got)
    if N == 1:
        assert torch.equal(attention.block_attention(q[:, 0], c, n, window, sinks), got[:, 0])
        o, lse = attention.block_attention(q[:, 0], c, n, window, sinks, return_lse=True)
        assert lse.shape == (H,) and torch.equal(o, got[:, 0])


@pytest.mark.parametrize("dtype", [INT8, E4M3])
@pytest.mark.parametrize("D", [128, 512])
def test_sizes_of_blocks(D, dtype):
    """Blocks whose values differ by many powers of two, zeros, and queries of any size."""
    g = torch.Generator(device=DEV).manual_seed(D)
    k, v = rows(g, 1, 1000, D, spread=6.0)
    k[:, 64:128] = 0.0
    v[:, 128:192] = 0.0
    c = filled(1, 1000, D, dtype)
    cache.append(c, k, v, 0)
    q = (torch.randn(8, 4, D, generator=g, device=DEV) * D ** -0.5).bfloat16()
    check(q, c, 1000, k, v, scale=0.5)
    check(q, c, 900, k, v, 200, 64, scale=0.5)
    for f in (2.0 ** -60, 2.0 ** 60):  # the same scores from other sizes
        check((q.double() * f).bfloat16(), c, 1000, k, v, scale=0.5 / f)
    check(torch.zeros_like(q), c, 1000, k, v)
    sharp = (q.float() * 30).bfloat16()
    o, _, _ = reference(sharp, values(k, dtype), values(v, dtype), 0, 0, 1.0)
    assert torch.isfinite(attention.block_attention(sharp, c, 1000)).all() and torch.isfinite(o).all()


def test_many_small_weights():
    """One key with most of the weight and 65000 with 2^-17 each of it: their sum counts."""
    D, n = 128, 65000
    g = torch.Generator(device=DEV).manual_seed(1)
    k = torch.zeros(1, n, D, device=DEV, dtype=torch.bfloat16)
    v = (1.0 + 0.25 * torch.randn(1, n, D, generator=g, device=DEV)).bfloat16()
    q = torch.zeros(1, 1, D, device=DEV, dtype=torch.bfloat16)
    q[..., 0] = 1.0
    k[0, :, 0] = -17 * math.log(2.0)
    k[0, 100, 0] = 0.0
    c = filled(1, n, D, INT8)
    cache.append(c, k, v, 0)
    check(q, c, n, k, v)


@pytest.mark.parametrize("dtype", [INT8, E4M3])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_nan_and_infinities(bad, dtype):
    """A block with one reads NaN for the queries that see any of it, and is nothing to the others; in the rows behind the last
    whole block it is what it is."""
    g = torch.Generator(device=DEV).manual_seed(11)
    H, D, n, N = 4, 256, 290, 40
    q = (torch.randn(H, N, D, generator=g, device=DEV) * D ** -0.5).bfloat16()
    clean = rows(g, 2, n, D)
    base = filled(2, n, D, dtype)
    cache.append(base, *clean, 0)
    for which in range(2):
        for at, hit in ((70, 64), (200, 192), (270, 270)):
            kv = [x.clone() for x in clean]
            kv[which][0, at, 3] = bad
            c = filled(2, n, D, dtype)
            cache.append(c, *kv, 0)
            for window, sinks in ((0, 0), (30, 0), (30, 10), (30, 66)):
                m = seen(n, N, window, sinks)
                want = attention.block_attention(q, base, n, window, sinks)
                got = attention.block_attention(q, c, n, window, sinks)
                block = m[:, hit:hit + 64].any(1) if at < 256 else m[:, at]
                assert torch.equal(got[2:], want[2:])                      # the other KV head
                assert torch.equal(got[:2, ~block], want[:2, ~block])      # rows that don't see it
                if at < 256:
                    assert got[:2, block].isnan().all()
                elif which == 1:
                    x = got[:2, block][..., 3]
                    assert (x.isnan() if math.isnan(bad) else x == bad).all()
                    keep = torch.arange(D, device=DEV) != 3
                    assert torch.equal(got[:2][..., keep], want[:2][..., keep])


def test_captured_step():
    """A decoded token's append and attention, captured once and replayed at each new length, eager work between."""
    g = torch.Generator(device=DEV).manual_seed(21)
    H, KV, D, cap = 8, 1, 256, 300
    k, v = rows(g, KV, cap, D)
    for window, sinks in ((0, 0), (100, 4)):
        c, e = filled(KV, cap, D, INT8), filled(KV, cap, D, INT8)
        n0 = 120
        cache.append(c, k[:, :n0], v[:, :n0], 0)
        cache.append(e, k[:, :n0], v[:, :n0], 0)
        q = torch.zeros(H, 1, D, device=DEV, dtype=torch.bfloat16)
        kn, vn = (torch.zeros(KV, 1, D, device=DEV, dtype=torch.bfloat16) for _ in range(2))
        at, length = (torch.tensor([x], dtype=torch.int32, device=DEV) for x in (n0, n0 + 1))
        kn.copy_(k[:, n0:n0 + 1]), vn.copy_(v[:, n0:n0 + 1])
        cache.append(c, kn, vn, at)
        attention.block_attention(q, c, length, window, sinks)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cache.append(c, kn, vn, at)
            o = attention.block_attention(q, c, length, window, sinks)
        for n in range(n0, cap):
            q.copy_((torch.randn(H, 1, D, generator=g, device=DEV) * 0.1).bfloat16())
            kn.copy_(k[:, n:n + 1]), vn.copy_(v[:, n:n + 1])
            at.fill_(n), length.fill_(n + 1)
            graph.replay()
            cache.append(e, kn, vn, n)
            if n % 7 == 0 or n % 64 in (0, 63, 62):
                check(q, e, n + 1, k, v, window, sinks)
                check(q, c, n + 1, k, v, window, sinks)
                check(q, c, n + 1, k, v, window, sinks, length=length)
                err = (o.double() - reference(q, values(k[:, :n + 1], INT8), values(v[:, :n + 1], INT8), window, sinks, 1.0)[0]).abs()
                assert err.max() < 0.05  # (the checks above are the strict ones; the replay's parts are the capacity's)
                assert torch.equal(o, attention.block_attention(q, c, length, window, sinks))


def test_lengths_out_of_range_in_device_memory():
    """Brought into range: nothing outside the cache is read or written."""
    g = torch.Generator(device=DEV).manual_seed(31)
    k, v = rows(g, 1, 200, 128)
    c = filled(1, 200, 128, INT8)
    cache.append(c, k, v, 0)
    q = (torch.randn(4, 3, 128, generator=g, device=DEV) * 0.1).bfloat16()
    short = filled(1, 200, 128, INT8)  # (a length that the cache doesn't hold any more would read other rows' ring)
    cache.append(short, k[:, :3], v[:, :3], 0)
    for of, n, as_if in ((c, 1 << 30, 200), (c, 201, 200), (short, -5, 3), (short, 2, 3)):
        dev = torch.tensor([n], dtype=torch.int32, device=DEV)
        check(q, of, as_if, k, v, length=dev)
    x, y = rows(g, 1, 10, 128)
    cache.append(c, x, y, torch.tensor([10 ** 6], dtype=torch.int32, device=DEV))
    a, _ = cache.read(c, 192, 200)
    assert torch.equal(a[0], x[0, 2:])


def test_another_stream():
    g = torch.Generator(device=DEV).manual_seed(41)
    k, v = rows(g, 2, 1500, 128)
    q = (torch.randn(8, 2, 128, generator=g, device=DEV) * 0.1).bfloat16()
    side = torch.cuda.Stream()
    c = filled(2, 1500, 128, E4M3)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        cache.append(c, k, v, 0)
        o = attention.block_attention(q, c, 1500)
    side.synchronize()
    assert torch.equal(o, attention.block_attention(q, c, 1500))
    check(q, c, 1500, k, v)


def test_refusals():
    c = cache.BlockCache(2, 100, 128)
    k = torch.zeros(2, 10, 128, device=DEV, dtype=torch.bfloat16)
    q = torch.zeros(4, 3, 128, device=DEV, dtype=torch.bfloat16)
    one = torch.zeros(1, dtype=torch.int32, device=DEV)
    for f, args in ((cache.BlockCache, (2, 100, 96)), (cache.BlockCache, (0, 100, 128)), (cache.BlockCache, (2, 0, 128)),
                    (cache.append, (c, k, k, 91)), (cache.append, (c, k, k, -1)), (cache.append, (c, k, k[:, :9], 0)),
                    (cache.append, (c, k[:1], k[:1], 0)), (cache.append, (c, k, k, one.long())), (cache.append, (c, k, k, one.cpu())),
                    (cache.append, (c, k.transpose(1, 2).contiguous().transpose(1, 2), k, 0)),
                    (cache.read, (c, 5, 4)), (cache.read, (c, 0, 101)), (cache.read, (c, -1, 4)),
                    (attention.block_attention, (q, c, 2)), (attention.block_attention, (q, c, 101)), (attention.block_attention, (q, c, 50, -1)),
                    (attention.block_attention, (q, c, 50, 4, -1)), (attention.block_attention, (q[:, :, :64], c, 50)),
                    (attention.block_attention, (q[:3], c, 50)), (attention.block_attention, (q, c, one.cpu()))):
        with pytest.raises(ValueError):
            f(*args)
    for f, args in ((cache.BlockCache, (2, 100, 128, torch.uint8)), (cache.append, (c, k.float(), k, 0)), (cache.append, (k, k, k, 0)),
                    (cache.read, (k, 0, 1)), (attention.block_attention, (q, k, 5)), (attention.block_attention, (q.half(), c, 50))):
        with pytest.raises(TypeError):
            f(*args)
    cache.append(c, k[:, :0], k[:, :0], 7)
    assert cache.read(c, 3, 3)[0].shape == (2, 0, 128)
