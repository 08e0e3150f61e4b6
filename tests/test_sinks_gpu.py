"""attention.sink_attention (a sliding window with the first keys visible beside it) against masked attention in 64 bits."""
import ctypes
import math

import pytest
import torch

from w8a8 import _lib, attention

DEV = "cuda"
pytestmark = pytest.mark.gpu


def seen(start, t, n, window, sinks):
    p = torch.arange(start, start + t, device=DEV)[:, None]
    j = torch.arange(n, device=DEV)[None]
    return (j <= p) if not window else (j <= p) & ((p - j < window) | (j < sinks))


def reference(q, k, v, start, window, sinks, scale):
    """(o, sum of weight x |v|, lse) in 64 bits."""
    H, t, _ = q.shape
    KV, n, _ = k.shape
    m = seen(start, t, n, window, sinks)
    o, a, lse = [], [], []
    for h in range(H):
        g = h // (H // KV)
        x = (scale * (q[h].double() @ k[g].double().t().contiguous())).masked_fill(~m, -math.inf)
        w = torch.softmax(x, -1)
        o.append(w @ v[g].double())
        a.append(w @ v[g].double().abs())
        lse.append(torch.logsumexp(x, -1))
    return torch.stack(o), torch.stack(a), torch.stack(lse)


def check(q, k, v, start, window, sinks, scale=1.0, at=None):
    got, lse = attention.sink_attention(q, k, v, start if at is None else at, window, sinks, scale, return_lse=True)
    n = start + q.shape[1]  # rows behind the last query may hold anything
    o, a, want = reference(q, k[:, :n], v[:, :n], start, window, sinks, scale)
    # the output's rounding and the weights' (bf16: 2^-8 each), and the scores': sums of D <= 512 products of sum |q k| <= 32 in
    # fp32 (2^-10)
    tol = 2.0 ** -8 * o.abs() + (2.0 ** -8 + 2.0 ** -10) * a + 1e-30
    err = (got.double() - o).abs()
    assert bool((err <= tol).all()), (err / tol).max().item()
    assert bool(((lse.double() - want).abs() <= 2.0 ** -9 + 2.0 ** -22 * want.abs()).all())
    assert torch.equal(attention.sink_attention(q, k, v, start if at is None else at, window, sinks, scale), got)
    return got


def make(g, H, KV, D, t, n, behind=40):
    q = (torch.randn(H, t, D, generator=g, device=DEV) * 2 * D ** -0.5).bfloat16()
    k, v = (torch.randn(KV, n + behind, D, generator=g, device=DEV).bfloat16() for _ in range(2))
    k[:, n:], v[:, n:] = math.nan, math.inf
    return q, k, v


CASES = [  # H, KV, D, start, t, window, sinks
    (8, 1, 256, 0, 1, 512, 4), (8, 1, 256, 700, 1, 512, 4), (8, 1, 512, 300, 1, 100, 1), (4, 4, 128, 5000, 1, 1, 1), (4, 4, 128, 5000, 1, 1, 0),
    (8, 1, 256, 3000, 1, 512, 700), (8, 1, 256, 511, 1, 512, 4), (8, 1, 256, 512, 1, 512, 1), (16, 1, 256, 900, 1, 64, 33),
    (12, 4, 128, 500, 5, 64, 3), (8, 1, 512, 1022, 7, 200, 4), (5, 5, 256, 316, 17, 50, 70), (32, 8, 128, 2000, 3, 0, 0), (20, 1, 256, 440, 9, 100, 64),
    (8, 1, 256, 0, 700, 512, 4), (8, 1, 256, 0, 600, 128, 4), (4, 2, 512, 0, 400, 64, 65), (6, 2, 128, 100, 900, 257, 16), (1, 1, 128, 0, 1000, 1, 2),
    (8, 1, 512, 1000, 130, 300, 32), (24, 2, 128, 77, 333, 500, 5), (3, 1, 512, 50, 200, 5, 400), (8, 2, 256, 0, 65, 0, 0), (16, 16, 128, 0, 300, 40, 8),
    (8, 1, 256, 2000, 260, 1024, 4), (128, 1, 128, 300, 2, 90, 4), (200, 1, 128, 10, 3, 8, 4),
]


@pytest.mark.parametrize("H,KV,D,start,t,window,sinks", CASES)
def test_attention(H, KV, D, start, t, window, sinks):
    g = torch.Generator(device=DEV).manual_seed(H * 7 + D + t * 3 + start)
    q, k, v = make(g, H, KV, D, t, start + t)
    got = check(q, k, v, start, window, sinks)
    check(q, k, v, start, window, sinks, at=torch.tensor([start], dtype=torch.int32, device=DEV))
    check((q.float() * 8).bfloat16(), k, v, start, window, sinks, 0.125)
    # strided operands and output
    wq = torch.zeros(t, H, D + 16, device=DEV, dtype=torch.bfloat16).transpose(0, 1)[:, :, 8:D + 8]
    wq.copy_(q)
    wk = torch.zeros(k.shape[1], KV, D + 8, device=DEV, dtype=torch.bfloat16).transpose(0, 1)[:, :, :D]
    wk.copy_(k)
    out = torch.full((t, H, D), 7.0, device=DEV, dtype=torch.bfloat16)
    attention.sink_attention(wq, wk, v, start, window, sinks, out=out.transpose(0, 1))
    assert torch.equal(out.transpose(0, 1), got)
    if t == 1:
        assert torch.equal(attention.sink_attention(q[:, 0], k, v, start, window, sinks), got[:, 0])
        o, lse = attention.sink_attention(q[:, 0], k, v, start, window, sinks, return_lse=True)
        assert lse.shape == (H,) and torch.equal(o, got[:, 0])


def plan(H, KV, Tq, Tk, D, start, window, sinks):
    r, n = ctypes.c_int(), ctypes.c_int()
    _lib.call("w8a8_attention_sinks_plan", H, KV, Tq, Tk, D, start, window, sinks, ctypes.byref(r), ctypes.byref(n))
    return r.value, n.value


@pytest.mark.parametrize("D", [128, 256, 512])
def test_every_tile(D):
    """Every row tile, split and not, against 64 bits."""
    g = torch.Generator(device=DEV).manual_seed(D)
    met = set()
    for H, KV, start, t, window, sinks in ((1, 1, 900, 7, 300, 4), (8, 1, 900, 16, 300, 40), (8, 2, 100, 600, 64, 3), (16, 2, 3000, 30, 0, 0),
                                           (16, 1, 3000, 100, 2500, 4), (8, 1, 0, 1500, 0, 0), (32, 8, 0, 1000, 0, 0), (32, 8, 0, 1000, 100, 4),
                                           (8, 1, 0, 3000, 0, 0)):
        tile = plan(H, KV, t, start + t, D, start, window, sinks)
        met.add((tile[0], tile[1] > 1))
        q, k, v = make(g, H, KV, D, t, start + t)
        check(q, k, v, start, window, sinks)
    assert {r for r, _ in met} == {16, 32, 64, 128} and {s for _, s in met} == {True, False}, met


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_nan_and_infinities(bad):
    """A key or value that a query doesn't see is nothing to it, whatever it holds."""
    g = torch.Generator(device=DEV).manual_seed(11)
    for D, t, start in ((256, 40, 250), (128, 300, 0), (512, 1, 289)):
        q, k, v = make(g, 4, 2, D, t, start + t)
        for which in range(2):
            for at in (5, 70, 200, 270):
                kv = [x.clone() for x in (k, v)]
                kv[which][0, at, 3] = bad
                for window, sinks in ((0, 0), (30, 0), (30, 10), (100, 66)):
                    m = seen(start, t, start + t, window, sinks)[:, at]
                    want, got = (attention.sink_attention(q, *x, start, window, sinks) for x in ((k, v), kv))
                    assert torch.equal(got[2:], want[2:]) and torch.equal(got[:2, ~m], want[:2, ~m])
                    if which == 1:
                        x = got[:2, m][..., 3]
                        assert (x.isnan() if math.isnan(bad) else x == bad).all()
                        keep = torch.arange(D, device=DEV) != 3
                        assert torch.equal(got[:2][..., keep], want[:2][..., keep])
                    elif math.isnan(bad):
                        assert got[:2, m].isnan().all()


def test_window_alone_is_attention():
    """Without sinks, or with all of them inside the window: what attention() gives, within two roundings of each."""
    g = torch.Generator(device=DEV).manual_seed(3)
    q, k, v = make(g, 8, 1, 256, 400, 400, behind=0)
    for window in (0, 64, 512):
        a = attention.attention(q, k, v, 0, window).double()
        b = attention.sink_attention(q, k, v, 0, window, 0).double()
        assert ((a - b).abs() <= 2.0 ** -6 * a.abs().clamp(min=1.0)).all()
    assert torch.equal(attention.sink_attention(q, k, v, 0, 0, 50), attention.sink_attention(q, k, v, 0, 0, 0))


def test_captured_step():
    """A decode step's attention captured once and replayed at each new position, eager work between."""
    g = torch.Generator(device=DEV).manual_seed(21)
    q, k, v = make(g, 8, 1, 256, 1, 400, behind=0)
    at = torch.tensor([3], dtype=torch.int32, device=DEV)
    attention.sink_attention(q, k, v, at, 100, 4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = attention.sink_attention(q, k, v, at, 100, 4)
    for p in (0, 1, 4, 31, 32, 99, 100, 103, 104, 105, 255, 399):
        q.copy_((torch.randn(8, 1, 256, generator=g, device=DEV) * 0.1).bfloat16())
        at.fill_(p)
        graph.replay()
        assert torch.equal(o, check(q, k, v, p, 100, 4, at=at))
    for p, as_if in ((-7, 0), (400, 399), (1 << 30, 399)):  # brought into range
        check(q, k, v, as_if, 100, 4, at=torch.tensor([p], dtype=torch.int32, device=DEV))


def test_far_positions():
    """Offsets past 32 bits: one head's keys are over 4 GiB."""
    D, n = 512, 4_400_000
    k = torch.zeros(1, n, D, device=DEV, dtype=torch.bfloat16)
    v = torch.zeros(1, n, D, device=DEV, dtype=torch.bfloat16)
    g = torch.Generator(device=DEV).manual_seed(5)
    q, kk, vv = make(g, 8, 1, D, 3, 300, behind=0)
    k[:, :4], v[:, :4] = kk[:, :4], vv[:, :4]
    k[:, n - 296:], v[:, n - 296:] = kk[:, 4:], vv[:, 4:]
    got = attention.sink_attention(q, k, v, n - 3, 290, 4)
    want = attention.sink_attention(q, kk, vv, 297, 290, 4)
    assert ((got.double() - want.double()).abs() <= 2.0 ** -6 * want.double().abs().clamp(min=1.0)).all()
    o, a, _ = reference(q, kk, vv, 297, 290, 4, 1.0)
    assert ((got.double() - o).abs() <= 2.0 ** -8 * o.abs() + (2.0 ** -8 + 2.0 ** -10) * a).all()


def test_refusals():
    q = torch.zeros(4, 3, 128, device=DEV, dtype=torch.bfloat16)
    k = torch.zeros(2, 10, 128, device=DEV, dtype=torch.bfloat16)
    one = torch.zeros(1, dtype=torch.int32, device=DEV)
    for args in ((q, k, k, 8), (q, k, k, -1), (q, k, k[:, :9]), (q, k, k[:1]), (q, k[:, :2], k[:, :2]), (q[..., :64], k, k), (q, k, k, one.cpu()),
                 (q, k, k, one.long()), (q.cpu(), k, k), (q.transpose(1, 2).contiguous().transpose(1, 2), k, k)):
        with pytest.raises(ValueError):
            attention.sink_attention(*args)
    for args in ((q, k, k, 0, -1), (q, k, k, 0, 4, -1), (q[:3], k, k), (q[:, :0], k, k), (q[..., :64].contiguous(), k[..., :64].contiguous(), k[..., :64].contiguous())):
        with pytest.raises((ValueError, _lib.W8A8Error)):
            attention.sink_attention(*args)
    with pytest.raises(_lib.W8A8Error):
        attention.sink_attention(q, k, k, 0, 4, 1, 0.0)
    for args in ((q.float(), k, k), (None, k, k), (q, k.half(), k)):
        with pytest.raises(TypeError):
            attention.sink_attention(*args)
