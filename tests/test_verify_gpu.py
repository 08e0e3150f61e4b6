"""ops.verify_drafts against the rule written out in 64 bits on the host."""
import math

import pytest
import torch

from w8a8 import ops

DEV = "cuda"
pytestmark = pytest.mark.gpu


def softmax(row, t):
    x = row.double() / t
    return torch.softmax(x, -1)


def rule(logits, tokens, u, draft=None, parents=None, length=None, t=1.0):
    """One request on the CPU: (accepted, path, next)."""
    n = tokens.numel()
    length = n if length is None else max(0, min(int(length), n))
    sound = lambda row: bool((row < math.inf).all()) and bool((row > -math.inf).any())
    at, path, gone, refused, q = -1, [], 0.0, [], None
    for m in range(length):
        parent = m - 1 if parents is None else int(parents[m])
        if parent != at or not -1 <= parent < m:
            if parents is None:
                break
            continue
        row, tok = logits[at + 1], int(tokens[m])
        p = softmax(row, t)
        pt = float(p[tok]) if 0 <= tok < p.numel() and tok not in refused else 0.0
        if not sound(row):
            pt = 0.0
        if parents is not None:
            need = float(u[m]) * (1.0 - gone)
        elif draft is None:
            need = float(u[m]) * (1.0 if 0 <= tok < p.numel() else 0.0)
        else:
            need = float(u[m]) * (float(softmax(draft[m], t)[tok]) if 0 <= tok < p.numel() else 0.0)
        if need < pt:
            at, gone, refused = m, 0.0, []
            path.append(m)
        else:
            gone += pt
            refused.append(tok)
            if parents is None:
                q = m
                break
    row = logits[at + 1]
    if not sound(row):
        return len(path), path, -1
    p = softmax(row, t)
    r = p.clone()
    if q is not None and draft is not None:
        d = softmax(draft[q], t)
        r = torch.where(p - d > 0, p - d, torch.zeros_like(p))
    elif refused:
        for tok in refused:
            if 0 <= tok < p.numel():
                r[tok] = 0.0
    if not float(r.sum()) > 0:
        r = p
    c = r.cumsum(0)
    return len(path), path, int((c <= float(u[-1]) * float(c[-1])).sum())


def check(logits, tokens, u, draft=None, parents=None, lengths=None, t=1.0):
    accepted, path, nxt = ops.verify_drafts(logits, tokens, u, draft, parents, lengths, t)
    assert accepted.dtype == torch.int32 and path.dtype == nxt.dtype == torch.int64
    one = logits.dim() == 2
    x, tok, uu = (y[None] if one else y for y in (logits, tokens, u))
    d = draft[None] if one and draft is not None else draft
    accepted, path, nxt = (y[None] if one else y for y in (accepted, path, nxt))
    assert accepted.shape == nxt.shape == (x.shape[0],) and path.shape == tok.shape
    for b in range(x.shape[0]):
        par = None if parents is None else (parents if parents.dim() == 1 else parents[b]).cpu()
        want = rule(x[b].cpu(), tok[b].cpu(), uu[b].cpu(), None if d is None else d[b].cpu(), par,
                    None if lengths is None else lengths[b].item(), t)
        got = int(accepted[b]), path[b].tolist(), int(nxt[b])
        assert got == (want[0], want[1] + [-1] * (tok.shape[1] - want[0]), want[2]), (b, got, want)
    return accepted


def make(g, b, n, v, dtype, t=1.0, spread=3.0, near=0.5):
    x = (torch.randn(b, n + 1, v, generator=g, device=DEV) * spread).to(dtype)
    d = (x[:, :n].float() + near * torch.randn(b, n, v, generator=g, device=DEV)).to(dtype)
    gumbel = -torch.log(-torch.log(torch.rand(b, n, v, generator=g, device=DEV).clamp(min=1e-20)))
    tok = (d.float() / t + gumbel).argmax(-1)
    return x, d, tok, torch.rand(b, n + 1, generator=g, device=DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("b,n,v", [(1, 1, 1), (1, 0, 300), (2, 3, 2), (1, 4, 100), (3, 5, 8185), (2, 2, 8192), (1, 3, 8193), (1, 2, 50257),
                                   (4, 8, 1001), (1, 16, 32000), (2, 1, 262144)])
def test_chain(b, n, v, dtype):
    g = torch.Generator(device=DEV).manual_seed(b * 1000 + n * 100 + v)
    for t in (1.0, 0.7):
        x, d, tok, u = make(g, b, n, v, dtype, t)
        check(x, tok, u, d, t=t)
        check(x, tok, u, t=t)
        lengths = torch.randint(-1, n + 2, (b,), generator=g, device=DEV, dtype=torch.int32)
        check(x, tok, u, d, lengths=lengths, t=t)
    check(x[0], tok[0], u[0], d[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("b,n,v", [(1, 1, 50), (1, 48, 32000), (2, 128, 1000), (1, 70, 8), (3, 9, 20011)])
def test_tree(b, n, v, dtype):
    g = torch.Generator(device=DEV).manual_seed(b * 1000 + n * 100 + v)
    for spread in (1.0, 4.0):
        x, _, _, u = make(g, b, n, v, dtype, spread=spread)
        back = torch.randint(0, 6, (b, n), generator=g, device=DEV)
        parents = (torch.arange(n, device=DEV)[None] - 1 - back).clamp(min=-1).int()
        parents[:, n // 3] = 200  # unused, and what hangs on it
        src = torch.where(parents == 200, torch.zeros_like(parents), parents).long() + 1
        top = torch.gather(x, 1, src[:, :, None].expand(b, n, v)).float()
        tok = (top + torch.randn(top.shape, generator=g, device=DEV)).argmax(-1)
        check(x, tok, u, parents=parents)
        check(x, tok, u, parents=parents[0].contiguous())
        check(x, tok, u, parents=parents, lengths=torch.full((b,), n // 2, dtype=torch.int32, device=DEV))
    star = torch.full((n,), -1, dtype=torch.int32, device=DEV)  # every node hangs on the context, tokens twice
    check(x, tok % min(v, 5), u, parents=star)
    check(x, tok, u * 0 + 0.999, parents=star)
    check(x, tok, u * 0, parents=torch.arange(-1, n - 1, dtype=torch.int32, device=DEV))


def test_all_accepted_and_none():
    g = torch.Generator(device=DEV).manual_seed(5)
    x, d, tok, u = make(g, 2, 6, 900, torch.float32)
    u[:, :6] = 0.0
    assert check(x, tok, u, d).tolist() == [6, 6]
    u[:, :6] = 1.0 - 2.0 ** -24
    check(x, tok, u, x[:, :6].contiguous())  # the same distribution: q = p, u < 1 accepts
    tok[0, 0] = 900  # outside the vocabulary
    tok[1, 0] = -1
    assert check(x, tok, u, d).tolist() == [0, 0]
    assert check(x, tok, u).tolist() == [0, 0]


@pytest.mark.parametrize("u_last", [0.0, 1e-30, 0.5, 1.0 - 2.0 ** -24])
def test_draw_ends(u_last):
    """The draw's first and last token, with tokens that cannot follow around them."""
    g = torch.Generator(device=DEV).manual_seed(7)
    for v in (5, 8192, 20000):
        x, d, tok, u = make(g, 1, 2, v, torch.float32)
        x[:, :, 0] = -math.inf
        x[:, :, -1] = torch.finfo(torch.float32).min
        u[:, -1] = u_last
        check(x, tok, u, d)
        check(x, tok, u)
        x[:, :, : v // 2] = -math.inf
        check(x, tok, u, d)


def test_no_distribution():
    """Rows with NaN or +inf, or of -inf alone, accept nothing; the draw from one gives -1."""
    g = torch.Generator(device=DEV).manual_seed(9)
    for value in (math.nan, math.inf, None):
        for row in range(4):
            x, d, tok, u = make(g, 2, 3, 9000, torch.float32)
            if value is None:
                x[0, row] = -math.inf
            else:
                x[0, row, 8500] = value
            u[:, :3] = 0.0
            got = check(x, tok, u, d)
            assert got.tolist() == [row, 3]
            check(x, tok, u)
            check(x, tok, u, parents=torch.tensor([-1, 0, 1], dtype=torch.int32, device=DEV))
    d[0, 0] = math.nan  # what a token was drafted from is no distribution: refused, drawn from what is left: p
    a, _, nxt = ops.verify_drafts(x, tok, u, d)
    p = torch.softmax(x[0, 0].double(), -1).cumsum(0)
    assert int(a[0]) == 0 and int(nxt[0]) == int((p <= u[0, 3].double() * p[-1]).sum())


def test_far_logits():
    """Logits far apart or far out, bf16 minima as masks: shares of one token only, and of two."""
    x = torch.full((1, 3, 4000), torch.finfo(torch.bfloat16).min, device=DEV, dtype=torch.bfloat16)
    x[0, 0, 17] = 3.0
    x[0, 1, 18] = x[0, 1, 3999] = -30000.0
    x[0, 2, 5] = 30000.0
    tok = torch.tensor([[17, 3999]], device=DEV)
    for u1 in (0.3, 0.7):
        for last in (0.1, 0.9):
            u = torch.tensor([[0.99, u1, last]], device=DEV)
            check(x, tok, u)
            check(x, tok, u, parents=torch.tensor([-1, 0], dtype=torch.int32, device=DEV))


def test_strides_and_views():
    g = torch.Generator(device=DEV).manual_seed(11)
    x, d, tok, u = make(g, 3, 4, 777, torch.bfloat16)
    wide = torch.randn(3, 6, 800, generator=g, device=DEV).bfloat16()
    wide[:, 1:6, 5:782] = x
    far = torch.randn(3, 7, 791, generator=g, device=DEV).bfloat16()
    far[:, 2:6, 3:780] = d
    got = ops.verify_drafts(wide[:, 1:6, 5:782], torch.stack([tok, tok], 1)[:, 1], torch.cat([u, u], 1)[:, 5:], far[:, 2:6, 3:780])
    for a, b in zip(got, ops.verify_drafts(x, tok, u, d)):
        assert torch.equal(a, b)
    check(x, tok, u, d)


def test_frequencies():
    """Accepted and drawn tokens are distributed as the target's: the first token over 40000 requests, each count within five
    standard deviations of its expectation (that misses once in a million calls; the seed is fixed)."""
    g = torch.Generator(device=DEV).manual_seed(13)
    n, v = 40000, 12
    x = torch.randn(1, 2, v, generator=g, device=DEV)
    d = x[:, :1] + torch.randn(1, 1, v, generator=g, device=DEV)
    tok = torch.multinomial(torch.softmax(d[0, 0], -1).expand(n, v), 1, generator=g)
    u = torch.rand(n, 2, generator=g, device=DEV)
    acc, _, nxt = ops.verify_drafts(x.expand(n, 2, v).contiguous(), tok, u, d.expand(n, 1, v).contiguous())
    first = torch.where(acc == 1, tok[:, 0], nxt)
    p = torch.softmax(x[0, 0].double(), -1)
    seen = torch.bincount(first, minlength=v).double()
    assert ((seen - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt()).all()


def test_graph_and_streams():
    """A captured call replayed with new inputs, and calls on another stream, give what the eager call gives."""
    g = torch.Generator(device=DEV).manual_seed(17)
    x, d, tok, u = make(g, 2, 5, 30000, torch.bfloat16)
    for _ in range(2):
        ops.verify_drafts(x, tok, u, d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.verify_drafts(x, tok, u, d)
    side = torch.cuda.Stream()
    for i in range(6):
        x2, d2, tok2, u2 = make(g, 2, 5, 30000, torch.bfloat16)
        for a, b in zip((x, d, tok, u), (x2, d2, tok2, u2)):
            a.copy_(b)
        graph.replay()
        want = [r.clone() for r in ops.verify_drafts(x2, tok2, u2, d2)]
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            other = ops.verify_drafts(x2, tok2, u2, d2)
        torch.cuda.synchronize()
        for a, b, c in zip(out, want, other):
            assert torch.equal(a, b) and torch.equal(b, c)
