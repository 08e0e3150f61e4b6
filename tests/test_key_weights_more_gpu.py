"""The keys' accumulated attention weights (attention.add_key_weights) where queries are padding, scores are infinite or a
position in device memory is out of range, against their definition in 64 bits.

Tolerance: a term inherits its score's absolute error as a relative one.  An fp32 sum of D products is off by at most
2^-24 (D / 2 + 2) of the sum of their magnitudes where roundings pile up, 2^-24 (8 + sqrt(D)) of the largest score where they
are spread; exp2, the subtraction and the sums add 8 ulp, and what stood in `weights` before one rounding."""
import math

import pytest
import torch

from w8a8 import attention as attn

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(H, KV, Tq, Tk, D, seed):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(H, Tq, D, generator=g) * (2.0 / math.sqrt(D))).bfloat16()
    return q, torch.randn(KV, Tk, D, generator=g).bfloat16(), torch.rand(KV, Tk, generator=g)


def scores(q, k, q_start, window, scale):
    """Masked scores [H, Tq, Tk] in 64 bits."""
    H, Tq, _ = q.shape
    KV, Tk, _ = k.shape
    p, j = torch.arange(q_start, q_start + Tq)[:, None], torch.arange(Tk)[None]
    seen = (j <= p) & ((p - j < window) if window else True)
    s = torch.stack([scale * (q[h].double() @ k[h // (H // KV)].double().T) for h in range(H)])
    return s.masked_fill(~seen, -math.inf)


def check(got, before, s, lse, KV, D, what):
    sums = torch.exp(s - lse.double()[:, :, None]).view(KV, -1, s.shape[-1]).sum(1)
    top = float(s[torch.isfinite(s)].abs().max())
    tol = (2.0 ** -24 * (8 + math.sqrt(D)) * top + 8 * 2.0 ** -24) * sums + 2.0 ** -23 * (before + sums)
    err = (got.double().cpu() - before.double() - sums).abs()
    assert (err <= tol).all(), f"{what}: worst {float((err / tol.clamp(min=1e-300)).max()):.3f} of the tolerance"


# one token, 32 rows, and prompts in one part and in several
SHAPES = [(8, 1, 1, 130, 512, 129), (8, 2, 4, 260, 128, 200), (8, 1, 96, 96, 256, 0), (8, 1, 700, 900, 512, 150), (4, 2, 600, 600, 128, 0)]


@pytest.mark.parametrize("what", [math.nan, math.inf])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_padding_queries_add_nothing_whatever_they_hold(shape, what):
    """An lse of -inf marks a query that adds nothing, also where its own values are not finite."""
    H, KV, Tq, Tk, D, start = shape
    q, k, w = make(H, KV, Tq, Tk, D, seed=sum(shape))
    for window in (0, 40):
        s = scores(q, k, start, window, 1.0)
        lse = torch.logsumexp(s, 2).float()
        pad = torch.zeros(H, Tq, dtype=torch.bool)
        pad[:, Tq // 2:] = True                        # the second half of the queries
        pad[0] = False
        pad[1] = True                                  # and all of one head's
        bad = q.clone()
        bad[pad] = what
        given = torch.where(pad, -math.inf, lse)
        got = w.to(DEV)
        attn.add_key_weights(bad.to(DEV), k.to(DEV), given.to(DEV), got, start, window)
        assert torch.isfinite(got).all()
        check(got, w, s, torch.where(pad, math.inf, lse), KV, D, f"{window}")       # exp(s - inf) = 0


@pytest.mark.parametrize("scale", [1.0, 0.5, 0.8, 0.1, 128 ** -0.5, 0.3])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_a_key_of_score_minus_infinity_draws_nothing(shape, scale):
    """Keys that every query scores with -inf, at any scale: their weights stay, the others' are as without them."""
    H, KV, Tq, Tk, D, start = shape
    q, k, w = make(H, KV, Tq, Tk, D, seed=sum(shape))
    q[:, :, 3] = q[:, :, 3].abs().clamp(min=2.0 ** -10)
    s = scores(q, k, start, 0, scale)
    out = torch.zeros(Tk, dtype=torch.bool)
    out[1::9] = True
    s = s.masked_fill(out, -math.inf)
    lse = torch.logsumexp(s, 2).float()
    k[:, out, 3] = -math.inf
    got = w.to(DEV)
    attn.add_key_weights(q.to(DEV), k.to(DEV), lse.to(DEV), got, start, 0, scale)
    assert torch.equal(got.cpu()[:, out], w[:, out])
    check(got, w, s, lse, KV, D, f"{scale}")


@pytest.mark.parametrize("window", [0, 512])
def test_a_position_out_of_range_is_the_nearest_in_range(window):
    """The caller's error: the weights are added at the nearest position, and nothing beside `weights` is touched."""
    H, D, cap, guard = 8, 256, 900, 64
    q, k, _ = make(H, 1, 1, cap, D, seed=8)
    store = torch.full((3, guard + cap + guard), 7.0, device=DEV)
    w = store[1:2, guard:guard + cap]
    pos = torch.zeros(1, dtype=torch.int32, device=DEV)
    for p, nearest in ((-3, 0), (cap, cap - 1), (1 << 30, cap - 1), (-(1 << 31), 0), (cap - 1, cap - 1), (0, 0)):
        w.zero_()
        pos.fill_(p)
        s = scores(q, k, nearest, window, 1.0)
        lse = torch.logsumexp(s, 2).float()
        attn.add_key_weights(q.to(DEV), k.to(DEV), lse.to(DEV), w, pos, window)
        check(w, torch.zeros(1, cap), s, lse, 1, D, f"{p}")
        assert (store[0] == 7.0).all() and (store[2] == 7.0).all()
        assert (store[1, :guard] == 7.0).all() and (store[1, guard + cap:] == 7.0).all()
