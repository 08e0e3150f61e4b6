"""Verification, sinks and the 8-bit cache as they are used together, and their native launch path."""
import threading

import pytest
import torch

from w8a8 import _lib, attention, cache, ops

DEV = "cuda"
pytestmark = pytest.mark.gpu


@pytest.fixture
def both(monkeypatch):
    """Runs f through the native path, which must take it, and through the wrappers' own code."""
    native = _lib.launch_module()

    def run(name, f):
        taken = []

        class Spy:
            def __getattr__(self, x):
                def call(*a):
                    r = getattr(native, x)(*a)
                    taken.append((x, r is not None))
                    return r
                return call
        out = []
        for way in (Spy(), None):
            for m in (attention, cache, ops):
                monkeypatch.setattr(m, "_native", way)
            out.append(f())
        assert (name, True) in taken, taken
        flat = lambda r: [r] if isinstance(r, torch.Tensor) else list(r)
        for x, y in zip(flat(out[0]), flat(out[1])):
            assert x.dtype == y.dtype and x.shape == y.shape and torch.equal(x, y)
    return run


def test_native_path(both):
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(3, 6, 3000, generator=g, device=DEV)
    d = (x[:, :5] + torch.randn(3, 5, 3000, generator=g, device=DEV))
    tok, u = torch.randint(0, 3000, (3, 5), generator=g, device=DEV), torch.rand(3, 6, generator=g, device=DEV)
    parents = torch.tensor([-1, 0, 0, 1, 2], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([5, 0, 3], dtype=torch.int32, device=DEV)
    for dt in (torch.float32, torch.bfloat16):
        both("verify_drafts", lambda: ops.verify_drafts(x.to(dt), tok, u, d.to(dt), None, lengths, 0.8))
        both("verify_drafts", lambda: ops.verify_drafts(x.to(dt), tok, u, None, parents))
        both("verify_drafts", lambda: ops.verify_drafts(x[0].to(dt), tok[0], u[0], None, parents))
        both("verify_drafts", lambda: ops.verify_drafts(x[0].to(dt), tok[0], u[0], d[0].to(dt), temperature=2))
        both("verify_drafts", lambda: ops.verify_drafts(x[:, :1].to(dt), tok[:, :0], u[:, :1]))
    q = torch.randn(8, 6, 256, generator=g, device=DEV).bfloat16()
    kv = torch.randn(2, 3, 400, 256, generator=g, device=DEV).bfloat16()
    k, v = kv[0, 1:], kv[1, :2]
    pos = torch.tensor([300], dtype=torch.int32, device=DEV)
    for start in (0, 300, pos):
        both("sink_attention", lambda: attention.sink_attention(q, k, v, start, 64, 4))
        both("sink_attention", lambda: attention.sink_attention(q[:, 0], k, v, start, 64, 4, 0.5))
    c = cache.BlockCache(2, 400, 256)
    cache.append(c, k, v, 0)
    both("block_read", lambda: cache.read(c, 17, 390))
    held = torch.tensor([330], dtype=torch.int32, device=DEV)
    for n in (64, 390, held):  # (whole blocks, or within the newest two)
        both("block_attention", lambda: attention.block_attention(q, c, n, 64, 4))
        both("block_attention", lambda: attention.block_attention(q[:, 0], c, n))

    def put(n):
        fresh = cache.BlockCache(2, 400, 256)
        fresh.data.zero_()
        cache.append(fresh, k[:, :100], v[:, :100], 0)
        cache.append(fresh, k[:, 100:], v[:, 100:], n)
        return fresh.data
    both("block_append", lambda: put(100))
    both("block_append", lambda: put(torch.tensor([100], dtype=torch.int32, device=DEV)))


def layer(g, H, KV, D, V):
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    return {"emb": r(V, D), "wq": r(H, D, D) * D ** -0.5, "wk": r(KV, D, D) * D ** -0.5, "wv": r(KV, D, D) * D ** -0.5, "out": r(H * D, V) * 0.02}


def project(m, tokens):
    x = m["emb"][tokens]
    return [(x @ w).bfloat16() for w in (m["wq"] * 0.25, m["wk"], m["wv"])]  # [heads, tokens, D]


def logits_of(m, o):
    return o.transpose(0, 1).flatten(1).float() @ m["out"]


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
def test_speculative_chat(codes):
    """A conversation in an 8-bit cache with a window and sinks: a prompt, then drafted runs that are verified, the refused
    tokens taken back, the next turn's tokens appended.  Every step against the same step over the cache's rows read
    back in bf16, and at the end the cache holds what one append of the accepted tokens gives."""
    g = torch.Generator(device=DEV).manual_seed(3)
    H, KV, D, V, W, S, draft = 4, 2, 128, 500, 90, 4, 5
    m = layer(g, H, KV, D, V)
    cap = 700
    c = cache.BlockCache(KV, cap, D, codes)
    tokens = torch.randint(0, V, (150,), generator=g, device=DEV)
    q, k, v = project(m, tokens)
    cache.append(c, k, v, 0)
    o = attention.block_attention(q, c, 150, W, S)
    step = lambda n: attention.sink_attention(q, *cache.read(c, 0, n), n - q.shape[1], W, S)
    near = lambda a, b, t=0.03: ((a.double() - b.double()).abs() <= t * b.double().abs().amax().clamp(min=1.0)).all()
    assert near(o, step(150))
    n, taken = 150, 0
    last = int(torch.randint(0, V, (1,), generator=g, device=DEV))
    for turn in range(40):
        if turn % 13 == 12:  # the user's next words
            more = torch.randint(0, V, (60,), generator=g, device=DEV)
            tokens = torch.cat([tokens, more])
            q, k, v = project(m, more)
            cache.append(c, k, v, n)
            n += 60
            assert near(attention.block_attention(q, c, n, W, S), step(n))
        drafted = torch.randint(0, V, (draft,), generator=g, device=DEV)
        run = torch.cat([torch.tensor([last], device=DEV), drafted])
        q, k, v = project(m, run)
        cache.append(c, k, v, n)
        o = attention.block_attention(q, c, n + draft + 1, W, S)
        assert near(o, step(n + draft + 1))
        x = logits_of(m, o)
        u = torch.rand(draft + 1, generator=g, device=DEV)
        u[:turn % 4] *= 1e-4  # some are accepted
        accepted, path, nxt = ops.verify_drafts(x, drafted, u)
        a = int(accepted)
        p = torch.softmax(x.double(), -1)
        for i in range(draft):
            ok = float(u[i]) < float(p[i, drafted[i]])
            assert ok == (i < a) or i > a
        assert path.tolist() == list(range(a)) + [-1] * (draft - a)
        r = p[a].clone()
        if a < draft:
            r[drafted[a]] = 0.0
        s = r.cumsum(0)
        assert int(nxt) == int((s <= u[draft].double() * s[-1]).sum())
        taken += a
        tokens = torch.cat([tokens, run[:a + 1]])
        n += a + 1  # the refused ones are written over next time
        last = int(nxt)
    assert taken > 5
    _, k, v = project(m, tokens)
    whole = cache.BlockCache(KV, cap, D, codes)
    cache.append(whole, k, v, 0)
    for a, b in zip(cache.read(c, 0, n), cache.read(whole, 0, n)):
        # (a product of other shapes may round a row's key differently, and its code: the largest e4m3 step is 32 of 448)
        assert near(a, b, 0.08)


def test_tree_step():
    """A tree of drafted tokens: attended to, verified, its accepted path moved up in the cache by the returned index."""
    g = torch.Generator(device=DEV).manual_seed(5)
    H, KV, D, V, past = 8, 1, 256, 300, 200
    m = layer(g, H, KV, D, V)
    prompt = torch.randint(0, V, (past,), generator=g, device=DEV)
    parents = torch.tensor([-1, 0, 0, 1, 2, 2, 4, -1, 7], dtype=torch.int32, device=DEV)
    M = parents.numel()
    nodes = torch.randint(0, V, (M,), generator=g, device=DEV)
    _, pk, pv = project(m, prompt)
    q, k, v = project(m, nodes)
    ck, cv = (torch.zeros(KV, past + M, D, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    ck[:, :past], cv[:, :past], ck[:, past:], cv[:, past:] = pk, pv, k, v
    o = attention.decode_tree(q, ck, cv, parents, past)
    root = torch.randn(1, V, generator=g, device=DEV)
    x = torch.cat([root, logits_of(m, o)])
    u = torch.rand(M + 1, generator=g, device=DEV)
    u[torch.tensor([0, 2, 5], device=DEV)] = 0.0  # this path
    u[1] = 1.0 - 2.0 ** -24
    accepted, path, nxt = ops.verify_drafts(x, nodes, u, parents=parents)
    assert path[:3].tolist() == [0, 2, 5] and int(accepted) == 3 and 0 <= int(nxt) < V
    rows = [t.clone() for t in (ck, cv)]
    cache.reorder([ck[:, past:], cv[:, past:]], path, dim=1)
    for t, old in zip((ck, cv), rows):
        assert torch.equal(t[:, past:past + 3], old[:, past:][:, [0, 2, 5]]) and torch.equal(t[:, :past], old[:, :past])


def test_two_at_once():
    """Two threads on two streams, each with its own cache: the results of each alone."""
    def work(seed, out):
        g = torch.Generator(device=DEV).manual_seed(seed)
        stream = torch.cuda.Stream()
        got = []
        with torch.cuda.stream(stream):
            c = cache.BlockCache(2, 900, 128)
            for _ in range(20):
                k, v = (torch.randn(2, 800, 128, generator=g, device=DEV).bfloat16() for _ in range(2))
                q = torch.randn(16, 3, 128, generator=g, device=DEV).bfloat16()
                x = torch.randn(4, 9000, generator=g, device=DEV)
                cache.append(c, k, v, 0)
                got.append(attention.block_attention(q, c, 800))
                got.append(attention.sink_attention(q, k, v, 797, 100, 4))
                got += list(ops.verify_drafts(x, torch.randint(0, 9000, (3,), generator=g, device=DEV), torch.rand(4, generator=g, device=DEV)))
            stream.synchronize()
        out[seed] = [t.clone() for t in got]
    alone, together = {}, {}
    for s in (1, 2):
        work(s, alone)
    threads = [threading.Thread(target=work, args=(s, together)) for s in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for s in (1, 2):
        assert all(torch.equal(a, b) for a, b in zip(alone[s], together[s]))
