"""Rows of the key / value cache put elsewhere (cache.reorder, cache.evict), bit for bit against plain Python."""
import math

import pytest
import torch

from w8a8 import W8A8Error, attention, cache, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rand(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    if dtype in (torch.int8, torch.int32, torch.int64, torch.uint8):
        return torch.randint(0, 100, shape, generator=g).to(dtype)
    return torch.randn(shape, generator=g).to(dtype)


# ---- reorder -----------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.int8, torch.float64])
@pytest.mark.parametrize("shape,n", [((4, 1, 30, 256), 4), ((2, 3, 7, 128), 2), ((1, 5, 8), 1), ((8, 2, 100, 64), 8), ((16, 1, 33, 128), 16),
                                     ((17, 2, 5, 16), 17), ((33, 300), 33), ((64, 3, 50), 64), ((64, 7), 5), ((100, 40), 64),
                                     ((5,), 5), ((9, 3), 9), ((6, 1, 1, 5), 6)], ids=str)
def test_reorder_the_first_dimension(shape, n, dtype):
    t = rand(shape, dtype, seed=n)
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        index = torch.randint(0, shape[0], (n,), generator=g)
        if seed == 1:
            index = torch.randperm(shape[0], generator=g)[:n]
        if seed == 2:
            index = torch.arange(n)                     # nothing moves
        if seed == 3:
            index = torch.full((n,), shape[0] - 1)      # all take the last
        d = t.to(DEV)
        cache.reorder(d, index.to(DEV))
        want = t.clone()
        want[:n] = t[index]
        assert torch.equal(d.cpu(), want), seed


def test_reorder_views_lists_and_dimensions():
    """Beams' live rows in several layers at once, rows of a cache, an index per request."""
    k = [rand((4, 2, 50, 64 * (i + 1)), torch.bfloat16, i) for i in range(5)]
    index = torch.tensor([2, 0, 0, 3])
    d = [t.to(DEV) for t in k]
    cache.reorder([t[:, :, : 10 + i] for i, t in enumerate(d)], index.to(DEV))
    for i, (t, got) in enumerate(zip(k, d)):
        want = t.clone()
        want[:, :, : 10 + i] = t[index, :, : 10 + i]
        assert torch.equal(got.cpu(), want)
    t = rand((3, 40, 128), torch.bfloat16, 9)
    d = t.to(DEV)
    cache.reorder([d[:, 20:33]], torch.tensor([0, 2, 3, 7, 12], device=DEV), dim=1)   # an accepted path moved up
    want = t.clone()
    want[:, 20:25] = t[:, [20, 22, 23, 27, 32]]
    assert torch.equal(d.cpu(), want)
    d = t.to(DEV)
    per = torch.tensor([[1, 0, 1], [39, 1, 2], [5, 5, 5]])
    cache.reorder(d, per.to(DEV), dim=-2)
    want = t.clone()
    for b in range(3):
        want[b, :3] = t[b, per[b]]
    assert torch.equal(d.cpu(), want)
    many = [rand((3, 5 + i), torch.float32, i) for i in range(120)]                   # more than one launch's tensors
    d = [x.to(DEV) for x in many]
    cache.reorder(d, torch.tensor([1, 2, 0], device=DEV))
    assert all(torch.equal(got.cpu(), x[[1, 2, 0]]) for got, x in zip(d, many))
    odd = rand((4, 1001), torch.int8, 3)
    d = torch.zeros(4, 1003, dtype=torch.int8, device=DEV)
    d[:, 1:1002] = odd.to(DEV)
    cache.reorder(d[:, 1:1002], torch.tensor([3, 3, 0, 1], device=DEV))               # bytes at odd addresses
    assert torch.equal(d[:, 1:1002].cpu(), odd[[3, 3, 0, 1]]) and (d[:, 0] == 0).all() and (d[:, 1002] == 0).all()


def test_reorder_leaves_rows_of_an_impossible_index():
    t = rand((5, 100), torch.float32, 1)
    d = t.to(DEV)
    cache.reorder(d, torch.tensor([-1, 5, 1, 1 << 40, 0], device=DEV))
    want = t.clone()
    want[2], want[4] = t[1], t[0]
    assert torch.equal(d.cpu(), want)


def test_reorder_past_32_bit_offsets():
    t = torch.zeros(5, 1 << 30, dtype=torch.bfloat16, device=DEV)                     # 2 GiB a row
    for i in range(5):
        t[i, -1000:] = i + 1.0
        t[i, 12345] = i + 10.0
    cache.reorder(t, torch.tensor([4, 0, 3, 3, 2], device=DEV))
    assert t[:, -1].tolist() == [5.0, 1.0, 4.0, 4.0, 3.0] and t[:, 12345].tolist() == [14.0, 10.0, 13.0, 13.0, 12.0]


def test_reorder_in_a_graph():
    t = rand((4, 2, 64, 128), torch.bfloat16, 1)
    d, index = t.to(DEV), torch.arange(4, device=DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        cache.reorder([d], index)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        cache.reorder([d], index)
    want = t
    for x in ([1, 0, 3, 2], [0, 0, 1, 1], [3, 2, 1, 0]):
        index.copy_(torch.tensor(x))
        graph.replay()
        torch.cuda.synchronize()
        want = want[x]
        assert torch.equal(d.cpu(), want)


def test_reorder_refusals():
    t = torch.zeros(4, 3, 8, device=DEV)
    i = torch.zeros(4, dtype=torch.int64, device=DEV)
    for args, error in [
        ((t, i.int()), TypeError), ((t, i.cpu()), ValueError), ((t.cpu(), i), ValueError), ((t, i[None, None]), TypeError),
        ((t, torch.zeros(5, dtype=torch.int64, device=DEV)), ValueError), ((t, i, 3), ValueError),
        ((torch.zeros(100, 2, device=DEV), torch.zeros(65, dtype=torch.int64, device=DEV)), ValueError),
        (([t, t[:3]], i[:2]), ValueError), ((t, torch.zeros(3, 2, dtype=torch.int64, device=DEV), 1), ValueError),
        ((t[:1].expand(4, 3, 8), i), ValueError), ((t[:, :1].expand(4, 3, 8), i), ValueError),
        ((torch.zeros(4, 3, 8, 5, device=DEV)[:, :2, :3, :2], i), ValueError),       # runs that are not evenly spaced
    ]:
        with pytest.raises(error):
            cache.reorder(*args)
    for args in (([t, t + 1, t], i), ([t, t[:, :2]], i)):                           # the same memory twice
        with pytest.raises(W8A8Error, match="same memory"):
            cache.reorder(*args)
    cache.reorder([], i)
    cache.reorder(t, i[:0])
    cache.reorder(torch.zeros(4, 0, device=DEV), i)


# ---- evict -------------------------------------------------------------------------------------


def evicted(w, pos, n, budget, recent):
    """The kept rows of one KV head, by the definition."""
    w, pos = w[:n].tolist(), pos[:n].tolist()
    newest = max(pos)

    def rank(r):
        if pos[r] > newest - recent:
            return (0, 0, r)
        return (1, -math.inf if math.isnan(w[r]) else 0, r) if math.isnan(w[r]) else (2, -w[r], r)

    keep = set(sorted(range(n), key=rank)[:budget])
    spare = iter(sorted(r for r in keep if r >= budget))
    return [r if r in keep else next(spare) for r in range(budget)]


def run_evict(k, v, w, pos, n, budget, recent, **kw):
    kd, vd, wd, pd = (t.to(DEV) for t in (k, v, w, pos))
    kept, wo, po = cache.evict(kd, vd, wd, pd, n, budget, recent, **kw)
    for g in range(k.shape[0]):
        want = evicted(w[g], pos[g], n, budget, recent)
        assert kept[g].tolist() == want
        assert torch.equal(po[g].cpu(), pos[g, want])
        assert torch.equal(wo[g].cpu().view(torch.int32), w[g, want].view(torch.int32))
        for t, d in ((k, kd), (v, vd)):
            whole = t[g].clone()
            whole[:budget] = t[g, want]
            assert torch.equal(d[g].cpu(), whole)  # the rows from the budget on as they were
    return kd, vd, wd, pd, kept, wo, po


@pytest.mark.parametrize("case", [
    # KV, rows, n, D, budget, recent
    (1, 1, 1, 128, 1, 0), (1, 2, 2, 128, 1, 1), (1, 2, 2, 128, 1, 0), (3, 10, 7, 64, 4, 2), (1, 64, 64, 256, 64, 5),
    (2, 65, 65, 128, 64, 64), (1, 1025, 1024, 512, 100, 10), (1, 4097, 4097, 512, 4096, 1024), (2, 5000, 4096, 128, 17, 0),
    (1, 16384, 16384, 64, 9000, 3000), (2, 16385, 16385, 64, 16384, 100), (1, 40000, 33333, 128, 1, 1), (4, 3001, 3001, 128, 1500, 1500),
    # few rows go
    (1, 3, 3, 128, 1, 1), (2, 9, 9, 64, 1, 0), (1, 10, 10, 64, 1, 1), (1, 16, 12, 64, 7, 3), (3, 1000, 1000, 128, 995, 64), (1, 4096, 4096, 64, 4095, 0),
    (2, 4100, 4097, 512, 4089, 1024), (1, 8192, 8192, 128, 8190, 8190), (2, 8193, 8193, 64, 8186, 100), (1, 16384, 16384, 128, 16383, 17),
    (1, 500, 500, 4096, 497, 5), (1, 500, 500, 4096, 493, 5), (1, 20480, 20480, 64, 20474, 7), (2, 33333, 33333, 64, 33332, 33332),
    (3, 40000, 36870, 64, 36865, 0), (1, 20000, 20000, 4096, 19998, 5), (1, 17000, 17000, 4096, 16994, 5),
], ids=lambda c: "x".join(map(str, c)))
def test_evict_matches_the_definition(case):
    KV, rows, n, D, budget, recent = case
    g = torch.Generator().manual_seed(sum(case))
    k, v = rand((KV, rows, D), torch.bfloat16, 1), rand((KV, rows, D), torch.bfloat16, 2)
    w = torch.exp(2 * torch.randn(KV, rows, generator=g))
    pos = torch.arange(rows, dtype=torch.int32).repeat(KV, 1)
    run_evict(k, v, w, pos, n, budget, recent)
    # rows in any order (a cache that was cut before), many equal weights
    pos = torch.stack([torch.randperm(rows, generator=g) for _ in range(KV)]).int() * 3 - 1000
    w = torch.randint(0, 3, (KV, rows), generator=g).float()
    run_evict(k, v, w, pos, n, budget, recent)


def test_evict_special_weights():
    n, budget = 200, 50
    k, v = rand((2, n, 64), torch.bfloat16, 1), rand((2, n, 64), torch.bfloat16, 2)
    pos = torch.arange(n, dtype=torch.int32).repeat(2, 1)
    w = torch.randn(2, n)
    w[0, 3::7], w[0, 4::9], w[0, 5::11], w[1, ::2], w[1, 1::4] = math.nan, math.inf, -math.inf, 0.0, -0.0
    run_evict(k, v, w, pos, n, budget, 20)
    run_evict(k, v, torch.full((2, n), math.nan), pos, n, budget, 0)
    for few in (n - 1, n - 6):
        run_evict(k, v, w, pos, n, few, 20)
        run_evict(k, v, torch.full((2, n), math.nan), pos, n, few, few)
        run_evict(k, v, w, pos[:, :1].expand(2, n).contiguous(), n, few, 1)          # every row is the newest
    run_evict(k, v, torch.full((2, n), 1e-42), pos, n, budget, 5)      # subnormal, all equal
    extreme = pos.clone()
    extreme[:, 0], extreme[:, 1] = -2 ** 31, 2 ** 31 - 1
    run_evict(k, v, w, extreme, n, budget, 50)


def test_evict_strided_in_place_and_other_types():
    KV, cap, n, D, budget = 2, 300, 250, 128, 100
    g = torch.Generator().manual_seed(1)
    w, pos = torch.rand(KV, cap, generator=g), torch.arange(cap, dtype=torch.int32).repeat(KV, 1)
    want = [evicted(w[i], pos[i], n, budget, 30) for i in range(KV)]
    # [T, KV, D] storage; weights and positions written over themselves
    k = rand((cap, KV, D), torch.bfloat16, 3)
    kd, vd = k.to(DEV), (k * 2).to(DEV)
    wd, pd = w.to(DEV), pos.to(DEV)
    kept = torch.empty(KV, budget, dtype=torch.int32, device=DEV)
    ws = torch.empty(cache.evict_workspace_bytes(KV, n, budget), dtype=torch.uint8, device=DEV)
    out = cache.evict(kd.transpose(0, 1), vd.transpose(0, 1), wd, pd, n, budget, 30, out=(kept, wd[:, :budget], pd[:, :budget]),
                      workspace=ws)
    assert out[1].data_ptr() == wd.data_ptr()
    for i in range(KV):
        assert kept[i].tolist() == want[i]
        assert torch.equal(kd[:budget, i].cpu(), k[want[i], i]) and torch.equal(vd[:budget, i].cpu(), (k * 2)[want[i], i])
        assert torch.equal(wd[i, :budget].cpu(), w[i, want[i]]) and torch.equal(wd[i, budget:].cpu(), w[i, budget:])
        assert torch.equal(pd[i, :budget].cpu(), pos[i, want[i]]) and torch.equal(pd[i, budget:].cpu(), pos[i, budget:])
    run_evict(rand((1, 90, 16), torch.int8, 1), rand((1, 90, 16), torch.int8, 2), torch.rand(1, 90), pos[:1, :90].clone(), 90, 33, 7)
    run_evict(rand((1, 90, 36), torch.float32, 1), rand((1, 90, 36), torch.float32, 2), torch.rand(1, 90), pos[:1, :90].clone(), 90, 33, 7)


@pytest.mark.parametrize("n,few", [(70, 1), (5000, 5), (20000, 6), (20000, 9000)])
def test_evict_step_by_step_in_place(n, few):
    """A full cache cut at every step, its weights and positions in place, with the caller's scratch, eager and replayed
    from a graph."""
    KV, D, recent, budget = 2, 64, 9, n - few
    g = torch.Generator().manual_seed(n + few)
    k, v = rand((KV, n, D), torch.bfloat16, 1), rand((KV, n, D), torch.bfloat16, 2)
    w = torch.randint(0, 50, (KV, n), generator=g).float()
    pos = torch.stack([torch.randperm(n, generator=g) for _ in range(KV)]).int()
    kd, vd, wd, pd = (t.to(DEV) for t in (k, v, w, pos))
    kept = torch.empty(KV, budget, dtype=torch.int32, device=DEV)
    ws = torch.empty(cache.evict_workspace_bytes(KV, n, budget), dtype=torch.uint8, device=DEV)

    def step():
        cache.evict(kd, vd, wd, pd, n, budget, recent, out=(kept, wd[:, :budget], pd[:, :budget]), workspace=ws)

    stream = torch.cuda.Stream()
    graph = None
    for i in range(4):
        want = [evicted(w[h], pos[h], n, budget, recent) for h in range(KV)]
        for t, d in ((k, kd), (v, vd), (w, wd), (pos, pd)):
            for h in range(KV):
                t[h, :budget] = t[h, want[h]]
        if i == 1:
            stream.wait_stream(torch.cuda.current_stream())
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                step()
        step() if graph is None else graph.replay()
        torch.cuda.synchronize()
        assert kept.tolist() == want, i
        for t, d in ((k, kd), (v, vd), (w, wd), (pos, pd)):
            assert torch.equal(d.cpu(), t), i
        # new rows behind the budget
        w[:, budget:] = torch.randint(0, 50, (KV, few), generator=g).float()
        pos[:, budget:] = n + i * few + torch.arange(few, dtype=torch.int32)
        wd.copy_(w)
        pd.copy_(pos)


def test_evict_past_32_bit_offsets():
    """One head's rows span more than 4 GiB."""
    n, step = 70_000, 65536
    store = torch.empty(n * step, dtype=torch.bfloat16, device=DEV)
    rows = store.view(n, step)
    k, v = rows[None, :, :64], rows[None, :, 64:128]
    k.copy_(torch.arange(n, device=DEV)[None, :, None] % 251)
    v.copy_(torch.arange(n, device=DEV)[None, :, None] // 251)
    w = torch.rand(1, n, generator=torch.Generator().manual_seed(2))
    pos = torch.arange(n, dtype=torch.int32)[None]
    kept, _, _ = cache.evict(k, v, w.to(DEV), pos.to(DEV), n, 30_000, 1000)
    want = evicted(w[0], pos[0], n, 30_000, 1000)
    assert kept[0].tolist() == want
    at = torch.tensor(want)
    assert torch.equal(k[0, :30_000, 5].float().cpu(), (at % 251).float())
    assert torch.equal(v[0, :30_000, 63].float().cpu(), (at // 251).float().bfloat16().float())


def test_evict_in_a_graph():
    n, budget = 600, 200
    k, v, w = rand((2, n, 128), torch.bfloat16, 1), rand((2, n, 128), torch.bfloat16, 2), torch.rand(2, n)
    pos = torch.arange(n, dtype=torch.int32).repeat(2, 1)
    kd, vd, wd, pd = (t.to(DEV) for t in (k, v, w, pos))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        cache.evict(kd.clone(), vd.clone(), wd, pd, n, budget, 50)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        kept, _, _ = cache.evict(kd, vd, wd, pd, n, budget, 50)
    for seed in range(3):
        kd.copy_(k)
        vd.copy_(v)
        w2 = torch.rand(2, n, generator=torch.Generator().manual_seed(seed))
        wd.copy_(w2)
        graph.replay()
        torch.cuda.synchronize()
        for g in range(2):
            want = evicted(w2[g], pos[g], n, budget, 50)
            assert kept[g].tolist() == want
            assert torch.equal(kd[g, :budget].cpu(), k[g, want]) and torch.equal(vd[g, budget:].cpu(), v[g, budget:])


def test_evict_refusals():
    k = torch.zeros(2, 50, 64, dtype=torch.bfloat16, device=DEV)
    w, p = torch.zeros(2, 50, device=DEV), torch.zeros(2, 50, dtype=torch.int32, device=DEV)
    ok = dict(k=k, v=k.clone(), weights=w, positions=p, n=50, budget=20, recent=5)
    cache.evict(**ok)
    for change, error in [
        (dict(k=k.cpu()), ValueError), (dict(k=k[0]), ValueError), (dict(v=k[:, :40]), ValueError), (dict(v=k.float()), ValueError),
        (dict(weights=w[:, :49]), ValueError), (dict(weights=w.double()), ValueError), (dict(weights=w.cpu()), ValueError),
        (dict(positions=p.long()), ValueError), (dict(positions=p[:1]), ValueError), (dict(n=51), ValueError),
        (dict(budget=0), ValueError), (dict(budget=51), ValueError), (dict(recent=21), ValueError), (dict(recent=-1), ValueError),
        (dict(k=k[:, :, ::2], v=k[:, :, ::2]), ValueError), (dict(workspace=torch.empty(8, dtype=torch.uint8, device=DEV)), W8A8Error),
        (dict(out=(p[:, :20], w[:, :20], w[:, :20])), ValueError),
        (dict(k=k[:, :, :60], v=k[:, :, :60]), W8A8Error),                           # rows of 120 bytes
    ]:
        with pytest.raises(error):
            cache.evict(**{**ok, **change})


# ---- together ----------------------------------------------------------------------------------


def test_a_bounded_cache_decodes_over_its_kept_rows():
    """Prompt attention, its weights, a cut, and decoding over the kept rows with further weights and cuts: each
    step equals attention over exactly the rows that the definition keeps."""
    H, T, D, cap, budget, recent = 8, 300, 256, 340, 120, 16
    g = torch.Generator().manual_seed(7)
    q = (torch.randn(H, T + 30, D, generator=g) * 0.15).bfloat16().to(DEV)
    k = torch.randn(1, T + 30, D, generator=g).bfloat16().to(DEV)
    v = torch.randn(1, T + 30, D, generator=g).bfloat16().to(DEV)
    kc, vc = torch.zeros(1, cap, D, dtype=torch.bfloat16, device=DEV), torch.zeros(1, cap, D, dtype=torch.bfloat16, device=DEV)
    w, pos = torch.zeros(1, cap, device=DEV), torch.zeros(1, cap, dtype=torch.int32, device=DEV)
    kc[:, :T], vc[:, :T], pos[:, :T] = k[:, :T], v[:, :T], torch.arange(T, device=DEV, dtype=torch.int32)
    _, lse = attention.attention(q[:, :T], kc[:, :T], vc[:, :T], 0, return_lse=True)
    attention.add_key_weights(q[:, :T], kc[:, :T], lse, w[:, :T], 0)
    kept = torch.empty(1, budget, dtype=torch.int32, device=DEV)
    rows = T
    for t in range(T, T + 30):
        if rows > budget + 9 or t == T:
            want = evicted(w[0].cpu(), pos[0].cpu(), rows, budget, recent)
            old = pos[0].cpu()
            cache.evict(kc, vc, w, pos, rows, budget, recent, out=(kept, w[:, :budget], pos[:, :budget]))
            assert kept[0].tolist() == want and pos[0, :budget].tolist() == old[want].tolist()
            rows = budget
        kc[:, rows], vc[:, rows], pos[:, rows], w[:, rows] = k[:, t], v[:, t], t, 0.0
        rows += 1
        o, lse = attention.decode(q[:, t], kc, vc, rows - 1, return_lse=True)
        attention.add_key_weights(q[:, t], kc, lse, w, rows - 1)
        at = pos[0, :rows].long()
        s = q[:, t].double().cpu() @ k[0, at].double().cpu().T
        p = torch.softmax(s, 1)
        ref, mag = p @ v[0, at].double().cpu(), p @ v[0, at].double().abs().cpu()
        assert ((o.double().cpu() - ref).abs() <= (2.0 ** -8 + 2.0 ** -10) * mag + 2.0 ** -8 * ref.abs()).all()
    assert pos[0, :rows].unique().numel() == rows


def test_a_beam_search_keeps_each_beam_with_its_own_cache():
    """Steps of choice, reordering and new rows: every beam's cache holds the rows of its own tokens."""
    nb, V, D, steps = 4, 1000, 64, 12
    g = torch.Generator().manual_seed(3)
    table = torch.randn(V, D, generator=g).bfloat16().to(DEV)          # a token's key, whatever the beam
    k = torch.zeros(nb, 1, steps, D, dtype=torch.bfloat16, device=DEV)
    tokens = torch.zeros(nb, steps, dtype=torch.int64, device=DEV)
    scores = torch.tensor([0.0] + [-math.inf] * (nb - 1), device=DEV)
    paths = [(0.0, [])] + [(-math.inf, [])] * (nb - 1)
    for t in range(steps):
        x = (torch.randn(nb, V, generator=g) * 3).to(DEV)
        scores, beams, toks = ops.beam_select(x, scores, nb)
        cache.reorder([k[:, :, :t], tokens[:, :t]], beams)
        k[:, 0, t] = table[toks]
        tokens[:, t] = toks
        lp = torch.log_softmax(x.double(), -1).cpu()
        cand = sorted(((-(paths[i][0] + float(lp[i, v])), i * V + v) for i in range(nb) if paths[i][0] > -math.inf
                       for v in torch.topk(lp[i], nb).indices.tolist()))[:nb]
        paths = [(-s, paths[a // V][1] + [a % V]) for s, a in cand]
        assert tokens[:, : t + 1].tolist() == [p for _, p in paths]
        assert torch.equal(k[:, 0, : t + 1], table[tokens[:, : t + 1]])
