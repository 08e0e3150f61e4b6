"""ops.verify_drafts where a chunk of the statistics is several tiles of 4096 logits, where statistics are staged more than once,
where a request has more than 256 chunks to draw from, on long chains, and at temperatures next to 0: against the rule
in 64 bits (test_verify_gpu.rule).  Each test says first which plan it runs, so that another plan cannot drop it unseen."""
import math

import pytest
import torch

from test_verify_gpu import DEV, check, make
from w8a8 import ops

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32
TILE, DRAW, STAGE = 4096, 2048, 1536
ALMOST = 1.0 - 2.0 ** -24


def plan(b, n, v):
    """(tiles of a chunk of the statistics, chunks of a row, chunks of the draw), from the workspace's size."""
    draws = (v + 7 + DRAW - 1) // DRAW
    chunks, rest = divmod(ops.verify_drafts_workspace_bytes(b, n, v) - b * draws * 8 - b * 128, b * (2 * n + 1) * 16)
    assert rest == 0
    tiles = next(t for t in range(1, 1 << 20) if (v + 7 + TILE * t - 1) // (TILE * t) == chunks)
    return tiles, chunks, draws


def tree(g, n):
    back = torch.randint(0, 6, (n,), generator=g, device=DEV)
    return (torch.arange(n, device=DEV) - 1 - back).clamp(min=-1).int()


def likely(g, x, parents):
    """Tokens that are often accepted: near the largest logits of the rows that they follow."""
    top = x[:, parents.long() + 1].float()
    return (top + torch.randn(top.shape, generator=g, device=DEV)).argmax(-1)


def far_apart(g, x, tiles, lead=0):
    """Rows whose chunks begin with logits far below those of later tiles, in four ways, a few logits of a later tile or all of
    them being the large ones."""
    n, v = x.shape[-2:]
    at = (torch.arange(v, device=DEV) + lead) % (TILE * tiles)
    first = at < TILE
    low = (-1000.0, -math.inf, float(torch.finfo(x.dtype).min), -450.0)
    for i in range(n):
        x[..., i, first] = low[i % 4]
        if i % 3 == 1:  # only these few are large: most threads see none of them
            some = (at >= TILE) & (torch.rand(v, generator=g, device=DEV) > 2e-4)
            x[..., i, some] = -600.0 if i % 2 else low[i % 4]
    return x


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_tiles_of_a_chunk(dtype):
    g = torch.Generator(device=DEV).manual_seed(1)
    b, n, v = 1, 48, 262144
    tiles, chunks, _ = plan(b, n, v)
    assert tiles == 2 and STAGE // chunks < n + 1  # (and the rows' statistics are staged twice)
    x, _, _, u = make(g, b, n, v, dtype)
    parents = tree(g, n)
    check(x, likely(g, x, parents), u, parents=parents)
    check(x, likely(g, x, parents), u * 0.1, parents=parents)
    far_apart(g, x, tiles)
    tok = likely(g, x, parents)
    for f in (1.0, 0.1, 0.0):
        check(x, tok, u * f, parents=parents)
        check(x, tok, u * f, parents=parents, t=2.5)
    chain = torch.arange(-1, n - 1, dtype=torch.int32, device=DEV)
    tok = likely(g, x, chain)
    for k in (0, 1, 2, 3, 4, 5, 24, 47):  # as far as row k, and drawn from it
        w, t = torch.zeros_like(u), tok.clone()
        w[0, k], t[0, k], w[0, n] = ALMOST, 0, u[0, k]
        assert check(x, t, w).tolist() == [k]


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("b,n,v", [(12, 9, 100003), (8, 8, 262144)])
def test_tiles_of_a_batch(b, n, v, dtype):
    g = torch.Generator(device=DEV).manual_seed(b)
    tiles, _, _ = plan(b, n, v)
    assert tiles == {12: 2, 8: 3}[b]
    x, d, tok, u = make(g, b, n, v, dtype, near=0.2)
    lengths = torch.randint(-1, n + 2, (b,), generator=g, device=DEV, dtype=torch.int32)
    check(x, tok, u, d)
    check(x, tok, u, d, lengths=lengths)
    far_apart(g, x, tiles)
    far_apart(g, d, tiles)
    tok = (d.float() + torch.randn(d.shape, generator=g, device=DEV)).argmax(-1)
    check(x, tok, u, d, lengths=lengths)
    check(x, tok, u * 0.3, d, t=0.7)
    # the same rows where they begin behind a whole 16-byte word
    wide = torch.zeros(b, n + 1, v + 13, device=DEV, dtype=dtype)
    wide[:, :, 3:v + 3] = x
    for p, q in zip(ops.verify_drafts(x, tok, u, d, None, lengths), ops.verify_drafts(wide[:, :, 3:v + 3], tok, u, d, None, lengths)):
        assert torch.equal(p, q)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_no_distribution_in_a_later_tile(value):
    g = torch.Generator(device=DEV).manual_seed(3)
    b, n, v = 12, 9, 100003
    tiles, _, _ = plan(b, n, v)
    assert tiles == 2
    x, _, tok, u = make(g, b, n, v, FP32)
    far_apart(g, x, tiles)
    u[:, :n] = 0.0
    for i in range(b):
        row = x[i, i % (n + 1)]
        if value == -math.inf:
            row.fill_(value)
        else:
            row[TILE + 1000 * (i + 1) if i < 3 else 3 * TILE + i] = value
    tok = x[:, :n].nan_to_num(0.0, 1e30, -1e30).argmax(-1)  # with probability where there is any
    assert check(x, tok, u).tolist() == [i % (n + 1) for i in range(b)]


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("v", [524289, 600000, 1100003])
def test_many_chunks_to_draw_from(v, dtype):
    g = torch.Generator(device=DEV).manual_seed(v)
    b, n = 2, 2
    tiles, _, draws = plan(b, n, v)
    assert draws > 256 and tiles >= 2
    x, d, tok, u = make(g, b, n, v, dtype)
    for last in (0.0, 1e-7, 0.25, 0.5, 0.999, ALMOST):  # the first chunk, those between and the last
        u[:, n] = last
        check(x, tok, u, d)
        check(x, tok, u)
    check(x, tok, u * 0.0 + 0.5, parents=torch.tensor([-1, -1], dtype=torch.int32, device=DEV))
    # all of it in the first chunk, in the last, in two far from one another
    for where in ([5, 700], [v - 1], [3, v - 2], [v // 2]):
        y = torch.full_like(x, -math.inf)
        y[..., where] = torch.randn(b, n + 1, len(where), generator=g, device=DEV).to(dtype)
        for last in (0.0, 0.4, 0.6, ALMOST):
            u[:, n] = last
            check(y, tok, u, d)
            check(y, tok, u)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n", [65, 100, 128])
def test_long_chains(n, dtype):
    g = torch.Generator(device=DEV).manual_seed(n)
    for b, v in ((3, 1000), (1, 50000)):
        if v == 50000 and n == 128:
            assert STAGE // plan(b, n, v)[1] < 2 * n + 1  # statistics staged more than once
        x, d, tok, u = make(g, b, n, v, dtype, near=0.05)
        ends = [n] + [k for k in (0, 63, 64, 65, 99, n - 1) if k < n]
        for k in ends:
            w, t = u * 0.0, tok.clone()
            w[:, n] = u[:, n]
            if k < n:
                w[:, k], t[:, k] = ALMOST, x[:, k].argmin(-1)
            assert (check(x, t, w) == k).all()
            check(x, t, w, d)
            check(x, t, w, d, lengths=torch.full((b,), max(0, k - 1), dtype=torch.int32, device=DEV))
            assert (check(x, t, w, lengths=torch.full((b,), min(n, k + 1), dtype=torch.int32, device=DEV)) == k).all()
        parents = torch.arange(-1, n - 1, dtype=torch.int32, device=DEV)
        check(x, tok, u * 1e-6, parents=parents)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_greedy(dtype):
    """A temperature next to 0: the largest logit has all of the probability, tokens are accepted while they are it, and it
    follows; equal ones share it."""
    g = torch.Generator(device=DEV).manual_seed(5)
    T = 1e-30
    for b, n, v in ((1, 4, 262144), (12, 9, 100003), (3, 70, 500)):
        x = 30.0 * torch.tanh(0.1 * torch.randn(b, n + 1, v, generator=g, device=DEV))
        best = torch.randint(0, v, (b, n + 1), generator=g, device=DEV)
        x = x.scatter(2, best[:, :, None], 30.5).to(dtype)
        u = torch.rand(b, n + 1, generator=g, device=DEV)
        for k in range(0, n + 1, max(1, n // 5)):
            tok = best[:, :n].clone()
            if k < n:
                tok[:, k] = (tok[:, k] + 1) % v
            accepted = check(x, tok, u, t=T)
            assert (accepted == k).all()
            a, _, nxt = ops.verify_drafts(x, tok, u, temperature=T)
            assert torch.equal(nxt, best[:, k])
            check(x, tok, u, parents=torch.arange(-1, n - 1, dtype=torch.int32, device=DEV), t=T)
    x[..., 7], x[..., 400] = 31.0, 31.0
    tok = torch.full((b, n), 7, device=DEV)
    accepted = check(x, tok, u, t=T)
    assert torch.equal(accepted, (u[:, :n] < 0.5).long().cumprod(1).sum(1).int())
