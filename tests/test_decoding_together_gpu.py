"""Decoding over a cache as a user has it: drafted tokens attended to as a tree and the accepted path moved up, and
the calls of two requests at once on streams of their own, eager and replayed from graphs."""
import pytest
import torch

from w8a8 import attention, cache, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def seen_rows(window, position, rows):
    """The rows of a chain's cache that its newest position sees."""
    return [j for j in range(rows) if j <= position and (window <= 0 or position - j < window)]


def bound(p, v, ref):
    # the weights and the output rounded to bf16, fp32 sums
    return (2.0 ** -8 + 2.0 ** -10) * (p @ v.abs()) + 2.0 ** -8 * ref.abs()


@pytest.mark.parametrize("H,KV,D,window,graph", [(8, 1, 256, 40, False), (8, 1, 512, 0, False), (4, 2, 128, 64, True)])
def test_drafting_and_accepting(H, KV, D, window, graph):
    """Rounds of a drafted tree: its rows written behind the context, one call for all nodes, a path accepted, its rows
    moved up, the context longer by the path.  Every node's output equals attention over the sequence that it
    ends, made of the accepted tokens and its own chain, and so does a decode step over the cache that is left."""
    M, cap, rounds = 13, 200, 7
    scale = 0.5
    g = torch.Generator().manual_seed(H * D + window)
    V = 300                                                            # tokens: a query, key and value of each
    tq = (torch.randn(V, H, D, generator=g) * (4.0 / D ** 0.5)).bfloat16()
    tk, tv = torch.randn(V, KV, D, generator=g).bfloat16(), torch.randn(V, KV, D, generator=g).bfloat16()
    seq = torch.randint(0, V, (50,), generator=g).tolist()
    k = torch.full((KV, cap, D), 9.0, dtype=torch.bfloat16, device=DEV)            # rows not yet written
    v = k.clone()
    k[:, :50], v[:, :50] = tk[seq].transpose(0, 1).to(DEV), tv[seq].transpose(0, 1).to(DEV)
    n_past = torch.zeros(1, dtype=torch.int32, device=DEV)
    parents = torch.full((M,), -1, dtype=torch.int32, device=DEV)
    q = torch.zeros(H, M, D, dtype=torch.bfloat16, device=DEV)

    def attend():
        return attention.decode_tree(q, k, v, parents, n_past, window, scale)

    if graph:
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            attend()
        torch.cuda.synchronize()
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured, stream=stream):
            o = attend()

    def expected(tokens):
        at = seen_rows(window, len(tokens) - 1, len(tokens))
        ids = [tokens[j] for j in at]
        out, tol = [], []
        for h in range(H):
            kk, vv = tk[ids, h // (H // KV)].double(), tv[ids, h // (H // KV)].double()
            p = torch.softmax(scale * (kk @ tq[tokens[-1], h].double()), 0)
            out.append(p @ vv)
            tol.append(bound(p, vv, out[-1]))
        return torch.stack(out), torch.stack(tol)

    for r in range(rounds):
        n = len(seq)
        par = [int(torch.randint(-1, m, (1,), generator=g)) if m else -1 for m in range(M)]
        drafted = torch.randint(0, V, (M,), generator=g).tolist()
        k[:, n:n + M], v[:, n:n + M] = tk[drafted].transpose(0, 1).to(DEV), tv[drafted].transpose(0, 1).to(DEV)
        q.copy_(tq[drafted].transpose(0, 1).to(DEV))
        n_past.fill_(n)
        parents.copy_(torch.tensor(par, dtype=torch.int32))
        if graph:
            captured.replay()
        else:
            o = attend()
        got = o.double().cpu()
        chains = []
        for m in range(M):
            chains.append((chains[par[m]] if par[m] >= 0 else []) + [m])
            want, tol = expected(seq + [drafted[i] for i in chains[m]])
            assert ((got[:, m] - want).abs() <= tol).all(), (r, m)
        path = max(chains, key=len)
        cache.reorder([k[:, n:n + M], v[:, n:n + M]], torch.tensor(path, device=DEV), dim=1)
        seq = seq + [drafted[i] for i in path]
        n = len(seq)
        assert torch.equal(k[:, :n].cpu(), tk[seq].transpose(0, 1)) and torch.equal(v[:, :n].cpu(), tv[seq].transpose(0, 1))
        token = int(torch.randint(0, V, (1,), generator=g))            # and a step of one token
        seq.append(token)
        k[:, n], v[:, n] = tk[token].to(DEV), tv[token].to(DEV)
        step = attention.decode(tq[token].to(DEV), k, v, n, window, scale).double().cpu()
        want, tol = expected(seq)
        assert ((step - want).abs() <= tol).all(), r


def calls(seed):
    """Every operator's call of one request, with the sizes that take workspaces; returns a function that runs them
    all on fresh copies and gives their results."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV)
    q, k, v = rn(8, 20, 256).bfloat16() * 0.1, rn(1, 3000, 256).bfloat16(), rn(1, 3000, 256).bfloat16()
    parents = torch.tensor([m - 1 - m % 3 if m else -1 for m in range(20)], dtype=torch.int32, device=DEV)
    qp, kp = rn(8, 700, 256).bfloat16() * 0.1, rn(1, 700, 256).bfloat16()
    lse = rn(8, 700) + 9.0
    ke, ve, we = rn(2, 20000, 64).bfloat16(), rn(2, 20000, 64).bfloat16(), torch.rand(2, 20000, generator=g, device=DEV)
    pe = torch.arange(20000, dtype=torch.int32, device=DEV).repeat(2, 1)
    x, s = rn(3, 4, 20000) * 3, rn(3, 4)
    t = rn(4, 3, 500, 64).bfloat16()

    def run():
        o = attention.decode_tree(q, k, v, parents, 2900, 0, 1.0)
        w = torch.zeros(1, 700, device=DEV)
        attention.add_key_weights(qp, kp, lse, w, 0)
        a, b = ke * 1, ve * 1                                             # (kernels: the calls are captured too)
        kept = cache.evict(a, b, we, pe, 20000, 9000, 100)
        beams = ops.beam_select(x, s, 5)
        c = t * 1
        cache.reorder([c], beams[1][0, :4])
        return [o, w, a, b, *kept, *beams, c]
    return run


def test_two_requests_at_once():
    assert attention.decode_tree_workspace_bytes(8, 1, 20, 20, 3000, 256, 2900) > 0
    runs = [calls(1), calls(2)]
    want = [r() for r in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        got = [None, None]
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = runs[i]()
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_two_graphs_replayed_at_once():
    """Two captured requests, each with workspaces of its own, replayed on two streams with eager calls between."""
    runs = [calls(3), calls(4)]
    want = [r() for r in runs]
    torch.cuda.synchronize()
    streams, graphs, got = [torch.cuda.Stream(), torch.cuda.Stream()], [], []
    for s, run in zip(streams, runs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got.append(run())
        graphs.append(graph)
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = runs[0]()
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
        assert all(torch.equal(x, y) for x, y in zip(want[0], eager))
        for b in got:
            for x in b:
                x.zero_()
        torch.cuda.synchronize()
