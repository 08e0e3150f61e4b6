"""GPU parity of the keys' accumulated attention weights (attention.add_key_weights) against their definition in
64 bits.

A term exp(s - lse) inherits its score's absolute error as a relative one.  An fp32 sum of D products in any
order is off by at most (D / 2 + 2) 2^-24 of the sum of their magnitudes where additions are spread over a
tree or over D / 2 terms on the mean; the scores here stay below 40, so their magnitudes' sum below 40 sqrt(D).
In practice roundings cancel; the bound taken is 2^-24 (8 + sqrt(D)) max|s| per term plus 8 ulp for exp2, the
subtraction and the sums, and the terms are positive, so their sum keeps the relative bound.  What stood in
`weights` before adds one rounding.
"""
import math

import pytest
import torch

from w8a8 import W8A8Error
from w8a8 import attention as attn

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(H, KV, Tq, Tk, D, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(H, Tq, D, generator=g) * (spread / math.sqrt(D))).bfloat16()
    k = torch.randn(KV, Tk, D, generator=g).bfloat16()
    w = torch.rand(KV, Tk, generator=g)
    return q, k, w


def reference(q, k, q_start, window, scale, lse=None):
    """(lse [H, Tq], sums [KV, Tk], largest |score|) in 64 bits; the sums for the given lse if there is one."""
    H, Tq, D = q.shape
    KV, Tk, _ = k.shape
    p = torch.arange(q_start, q_start + Tq)[:, None]
    j = torch.arange(Tk)[None]
    seen = (j <= p) & ((p - j < window) if window else True)
    total = torch.zeros(KV, Tk, dtype=torch.float64)
    out = torch.empty(H, Tq, dtype=torch.float64)
    top = 0.0
    for h in range(H):
        s = scale * (q[h].double() @ k[h // (H // KV)].double().T)
        top = max(top, float(s[seen].abs().max()))
        s = s.masked_fill(~seen, -math.inf)
        out[h] = torch.logsumexp(s, 1)
        ref = out[h] if lse is None else lse[h].double()
        total[h // (H // KV)] += torch.exp(s - ref[:, None]).masked_fill(~seen, 0.0).sum(0)
    return out, total, top


def check(got, before, sums, top, D, what):
    tol = (2.0 ** -24 * (8 + math.sqrt(D)) * top + 8 * 2.0 ** -24) * sums + 2.0 ** -23 * (before + sums)
    err = (got.double().cpu() - before.double() - sums).abs()
    assert (err <= tol).all(), f"{what}: worst {float((err / tol.clamp(min=1e-300)).max()):.3f} of the tolerance"


CASES = [
    # H, KV, Tq, Tk, D, q_start, window
    (8, 1, 1, 1, 512, 0, 0),
    (8, 1, 1, 4097, 512, 4096, 0),       # one token
    (8, 1, 1, 700, 256, 699, 512),       # one token of a sliding layer
    (8, 1, 1, 700, 256, 300, 512),       # keys behind the query
    (1, 1, 1, 63, 128, 62, 0),
    (16, 1, 1, 130, 128, 129, 0),
    (32, 8, 1, 1000, 128, 999, 0),
    (8, 1, 4, 260, 512, 256, 0),         # 32 rows, the last few-row call
    (8, 1, 5, 261, 512, 256, 0),         # 40 rows, the first of the other kernel
    (12, 4, 3, 129, 256, 100, 7),        # three heads per KV head
    (8, 1, 77, 77, 256, 0, 16),          # a window shorter than a key block
    (8, 1, 300, 300, 512, 0, 0),
    (8, 1, 513, 600, 256, 50, 200),      # ragged
    (4, 2, 1100, 1100, 128, 0, 0),       # several parts per key block
    (6, 2, 200, 900, 128, 650, 0),
    (8, 8, 65, 65, 128, 0, 0),
    (8, 1, 640, 3000, 256, 2000, 300),   # the window's keys start behind row 0
    (64, 1, 33, 97, 128, 64, 0),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c)))
def test_matches_the_definition(case):
    H, KV, Tq, Tk, D, q_start, window = case
    q, k, w = make(H, KV, Tq, Tk, D, seed=sum(case))
    scale = 1.0 if Tq % 2 else 0.8
    lse = reference(q, k, q_start, window, scale)[0].float()
    _, sums, top = reference(q, k, q_start, window, scale, lse)
    got = w.to(DEV)
    r = attn.add_key_weights(q.to(DEV), k.to(DEV), lse.to(DEV), got, q_start, window, scale)
    assert r is got
    check(got, w, sums, top, D, str(case))
    unseen = torch.ones(Tk, dtype=torch.bool)
    unseen[max(0, q_start - window + 1) if window else 0: q_start + Tq] = False
    assert torch.equal(got.cpu()[:, unseen], w[:, unseen])
    # every query spreads a weight of one
    added = (got.double().cpu() - w.double()).sum()
    assert abs(float(added) - H * Tq) <= 1e-4 * H * Tq + 1e-6 * Tk
    again = w.to(DEV)
    attn.add_key_weights(q.to(DEV), k.to(DEV), lse.to(DEV), again, q_start, window, scale)
    assert torch.equal(got, again)


@pytest.mark.parametrize("D", [128, 256, 512])
@pytest.mark.parametrize("window", [0, 100])
def test_with_the_attention_that_gives_the_logsumexp(D, window):
    """A prompt's attention and the tokens after it, their weights summed up call by call."""
    H, KV, T, n = 8, 1, 200, 6
    q, k, _ = make(H, KV, T + n, T + n, D, seed=D)
    v = torch.randn(KV, T + n, D).bfloat16().to(DEV)
    qd, kd = q.to(DEV), k.to(DEV)
    w = torch.zeros(KV, T + n, device=DEV)
    _, lse = attn.attention(qd[:, :T], kd[:, :T], v[:, :T], 0, window, return_lse=True)
    attn.add_key_weights(qd[:, :T], kd[:, :T], lse, w[:, :T], 0, window)
    for t in range(T, T + n):
        _, l1 = attn.decode(qd[:, t], kd, v, t, window, return_lse=True)
        attn.add_key_weights(qd[:, t], kd, l1, w, t, window)
    ref = reference(q, k, 0, window, 1.0)[1]
    # the attention's own lse is off by a few 2^-24 of its size and its hardware logarithm
    assert ((w.double().cpu() - ref).abs() <= 2e-5 * ref + 1e-9).all()


def test_masked_infinities_and_queries_that_saw_nothing():
    """NaN and infinite keys outside the view add nothing anywhere; an lse of -inf adds nothing."""
    for H, Tq, start, window in ((8, 1, 150, 40), (8, 70, 100, 40)):
        q, k, w = make(H, 1, Tq, 260, 128, seed=Tq)
        lse = reference(q, k, start, window, 1.0)[0].float()
        lse[3, 0] = -math.inf
        given = torch.where(torch.isinf(lse), torch.tensor(math.inf), lse)  # exp(s - inf) = 0
        _, sums, top = reference(q, k, start, window, 1.0, given)
        bad = k.clone()
        lo, hi = start - window + 1, start + Tq
        bad[:, :lo] = math.nan
        bad[:, hi:] = math.inf
        got = w.to(DEV)
        attn.add_key_weights(q.to(DEV), bad.to(DEV), lse.to(DEV), got, start, window)
        assert torch.isfinite(got).all()
        check(got, w, sums, top, 128, f"{Tq}")


def test_nan_in_a_masked_tile_of_a_prompt():
    """A NaN key is seen from its position on only."""
    q, k, w = make(8, 1, 96, 96, 256, seed=4)
    lse = reference(q, k, 0, 0, 1.0)[0].float()
    k[0, 50] = math.nan
    got = w.to(DEV)
    attn.add_key_weights(q.to(DEV), k.to(DEV), lse.to(DEV), got, 0)
    assert torch.isnan(got[0, 50]) and torch.isfinite(got[0, :50]).all() and torch.isfinite(got[0, 51:]).all()


def test_position_in_device_memory_and_graph_replay():
    H, KV, D, cap = 8, 1, 256, 900
    q, k, _ = make(H, KV, 1, cap, D, seed=8)
    qd, kd = q.to(DEV), k.to(DEV)
    for window in (0, 512):
        pos = torch.zeros(1, dtype=torch.int32, device=DEV)
        w = torch.zeros(KV, cap, device=DEV)
        lse = torch.zeros(H, 1, device=DEV)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            attn.add_key_weights(qd, kd, lse, w, pos, window)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            attn.add_key_weights(qd, kd, lse, w, pos, window)
        before = torch.zeros(KV, cap)
        w.zero_()
        total, bound = before.double(), 0.0
        for p in (0, 5, 511, 512, 899, 640):
            l = reference(q, k, p, window, 1.0)[0].float()
            pos.fill_(p)
            lse.copy_(l)
            graph.replay()
            torch.cuda.synchronize()
            _, sums, top = reference(q, k, p, window, 1.0, l)
            total = total + sums
            check(w, before, total, top + 8, D, f"replayed at {p}")
        for p in (-3, 900, 1 << 30):     # the caller's error: nothing outside the cache is touched
            pos.fill_(p)
            graph.replay()
        torch.cuda.synchronize()
        assert w.shape == (KV, cap)


def test_strided_operands():
    H, KV, Tq, Tk, D = 8, 2, 40, 120, 128
    q, k, w = make(H, KV, Tq, Tk, D, seed=5)
    lse = reference(q, k, 80, 0, 1.0)[0].float()
    _, sums, top = reference(q, k, 80, 0, 1.0, lse)
    qd = q.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
    kd = torch.full((Tk, KV, D + 8), math.nan, dtype=torch.bfloat16, device=DEV)
    kd[:, :, :D] = k.to(DEV).transpose(0, 1)
    ld = torch.full((H, Tq + 3), math.nan, device=DEV)
    ld[:, :Tq] = lse.to(DEV)
    store = torch.full((KV, Tk + 9), 5.0, device=DEV)
    store[:, :Tk] = w.to(DEV)
    attn.add_key_weights(qd, kd[:, :, :D].transpose(0, 1), ld[:, :Tq], store[:, :Tk], 80)
    check(store[:, :Tk], w, sums, top, D, "strided")
    assert (store[:, Tk:] == 5.0).all()


def test_a_cache_whose_offsets_pass_32_bits():
    """Rows 40 KiB apart: the last key lies more than 4 GiB behind the first."""
    Tk, D, step = 110_000, 128, 20480
    store = torch.empty(Tk * step, dtype=torch.bfloat16, device=DEV)
    rows = store.view(Tk, step)[:, :D]
    g = torch.Generator(device=DEV).manual_seed(1)
    rows.copy_(torch.randn(Tk, D, generator=g, device=DEV))
    for Tq in (1, 20):
        q = (torch.randn(4, Tq, D, generator=g, device=DEV) * 0.2).bfloat16()
        k = rows[None].contiguous().cpu()
        lse = reference(q.cpu(), k, Tk - Tq, 0, 1.0)[0].float()
        _, sums, top = reference(q.cpu(), k, Tk - Tq, 0, 1.0, lse)
        w = torch.zeros(1, Tk, device=DEV)
        attn.add_key_weights(q, rows[None], lse.to(DEV), w, Tk - Tq)
        check(w, torch.zeros(1, Tk), sums, top, D, "far rows")


def test_refusals():
    q, k, w = (t.to(DEV) for t in make(8, 1, 3, 50, 128, seed=1))
    lse = torch.zeros(8, 3, device=DEV)
    ok = dict(q=q, k=k, lse=lse, weights=w, q_start=40)
    attn.add_key_weights(**ok)
    pos = torch.tensor([3], dtype=torch.int32, device=DEV)
    many = torch.zeros(8, 9, 128, dtype=torch.bfloat16, device=DEV)
    for change, error in [
        (dict(q=q.cpu()), ValueError), (dict(q=q.float()), TypeError), (dict(k=k[:, :, :64]), ValueError),
        (dict(lse=lse[:7]), ValueError), (dict(lse=lse.double()), ValueError), (dict(weights=w[:, :49]), ValueError),
        (dict(weights=w.cpu()), ValueError), (dict(q_start=48), ValueError), (dict(q_start=-1), ValueError),
        (dict(q_start=pos.long()), ValueError), (dict(window=-2), W8A8Error), (dict(scale=-1.0), W8A8Error),
        (dict(q=many, lse=torch.zeros(8, 9, device=DEV), q_start=pos), W8A8Error),   # 72 rows with a device position
        (dict(q=torch.zeros(7, 3, 128, dtype=torch.bfloat16, device=DEV), lse=lse[:7], k=torch.cat([k, k]),
              weights=torch.cat([w, w])), W8A8Error),
        (dict(q=q[:, :, :64].contiguous(), k=k[:, :, :64].contiguous()), W8A8Error),
    ]:
        with pytest.raises(error):
            attn.add_key_weights(**{**ok, **change})
