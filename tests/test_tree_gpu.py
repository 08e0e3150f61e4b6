"""GPU parity of the attention of drafted tokens (attention.decode_tree) against its definition in 64 bits.

The reference walks each node's chain and takes the softmax over exactly the rows it sees.  Tolerance per
element: the softmax weights are rounded to bf16 for the second product (half a step, 2^-9 relative to the
weight's power of two, at most 2^-8 of its value) and the output once (half a step):

    |o - ref| <= 2^-8 sum_j p_j |v_j| + 2^-8 |ref| + small

with fp32 scores: an error e of a score moves every weight by e relative, e <= 2^-24 (D / 2 + 2) sum_d |q_d k_d|
for an fp32 sum of D products in any order (2^-24 per addition, D / 2 of them at the mean), which stays far
below 2^-8 for the inputs here and is covered by `small` = 2^-10 sum_j p_j |v_j|.
"""
import math

import pytest
import torch

from w8a8 import W8A8Error
from w8a8 import attention as attn

pytestmark = pytest.mark.gpu
DEV = "cuda"


def chain_of(parents, m):
    """Node m's chain from the root down, or None where it is unused."""
    chain = []
    while m >= 0:
        if not -1 <= parents[m] < m:
            return None
        chain.append(m)
        m = parents[m]
    return chain[::-1]


def reference(q, k, v, parents, past, window, scale):
    H, N, D = q.shape
    G = H // k.shape[0]
    M = len(parents)
    o = torch.zeros(H, N, D, dtype=torch.float64)
    mag = torch.zeros(H, N, D, dtype=torch.float64)
    lse = torch.full((H, N), -math.inf, dtype=torch.float64)
    for i in range(N):
        chain = chain_of(parents, M - N + i)
        if chain is None:
            continue
        rows = list(range(past)) + [past + c for c in chain]  # in order of position
        if window:
            rows = rows[-window:]
        rows = torch.tensor(rows)
        for h in range(H):
            s = scale * (k[h // G, rows].double() @ q[h, i].double())
            p = torch.softmax(s, 0)
            o[h, i] = p @ v[h // G, rows].double()
            mag[h, i] = p @ v[h // G, rows].double().abs()
            lse[h, i] = torch.logsumexp(s, 0)
    return o, mag, lse


def make(H, KV, N, Tk, D, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(H, N, D, generator=g) * (spread / math.sqrt(D))).bfloat16()
    k = torch.randn(KV, Tk, D, generator=g).bfloat16()
    v = torch.randn(KV, Tk, D, generator=g).bfloat16()
    return q, k, v


def random_tree(M, seed, back=4):
    g = torch.Generator().manual_seed(seed)
    return [int(m - 1 - torch.randint(0, min(m + 1, back), (1,), generator=g)) for m in range(M)]


def check(o, lse, ref, what):
    ro, mag, rl = ref
    got = o.double().cpu()
    assert torch.isfinite(got).all(), what
    tol = (2.0 ** -8 + 2.0 ** -10) * mag + 2.0 ** -8 * ro.abs()
    bad = (got - ro).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float(((got - ro).abs() / tol.clamp(min=1e-30)).max()):.3f}"
    if lse is not None:
        gl = lse.double().cpu()
        assert torch.equal(torch.isinf(gl), torch.isinf(rl)), what
        ok = ~torch.isinf(rl)
        # fp32 scores and sums: a few ulp of the largest score and of log's argument
        assert ((gl - rl).abs()[ok] <= 2e-5 * (1 + rl.abs()[ok])).all(), what


CASES = [
    # H, KV, N, M, past, D, window, spare rows behind the last node
    (8, 1, 8, 8, 700, 256, 512, 0),      # a sliding layer, a small tree
    (8, 1, 16, 16, 411, 512, 0, 5),      # a full layer
    (8, 1, 1, 1, 1, 512, 0, 0),          # one node, one context row
    (8, 1, 1, 1, 0, 512, 0, 3),          # no context at all
    (1, 1, 1, 1, 37, 128, 0, 0),
    (4, 4, 5, 5, 64, 128, 0, 1),         # one head per KV head
    (32, 8, 33, 50, 130, 128, 0, 0),     # the newest 33 of 50 nodes, 132 rows per KV head
    (12, 4, 7, 9, 95, 256, 0, 0),        # three heads per KV head
    (16, 1, 64, 64, 300, 128, 0, 0),     # 1024 rows
    (8, 1, 64, 64, 257, 512, 0, 0),
    (8, 2, 3, 128, 63, 256, 0, 2),       # few queries of the largest tree
    (2, 1, 128, 128, 31, 256, 0, 0),
    (8, 1, 9, 9, 100, 256, 4, 0),        # a window inside the tree
    (8, 1, 40, 40, 33, 128, 1, 0),       # a window of the node alone
    (8, 1, 12, 12, 500, 256, 64, 7),     # the window's edge inside a key block
    (8, 1, 6, 6, 40, 256, 512, 0),       # a window longer than the cache
    (5, 5, 2, 2, 1000, 512, 129, 0),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c)))
def test_matches_the_definition(case):
    H, KV, N, M, past, D, window, spare = case
    q, k, v = make(H, KV, N, past + M + spare, D, seed=sum(case))
    parents = random_tree(M, seed=past + M)
    scale = 1.0 if N % 2 else 0.7
    o, lse = attn.decode_tree(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor(parents, dtype=torch.int32, device=DEV), past,
                              window, scale, return_lse=True)
    check(o, lse, reference(q, k, v, parents, past, window, scale), str(case))


@pytest.mark.parametrize("D", [128, 256, 512])
@pytest.mark.parametrize("rows", [(1, 1), (8, 1), (8, 3), (8, 7), (8, 16), (4, 37)])
@pytest.mark.parametrize("past", [3, 1700])
def test_row_tiles_and_parts(D, rows, past):
    """Every row tile (16 to 128 rows, and several of them), in one part of the keys and in many."""
    H, N = rows
    q, k, v = make(H, 1, N, past + N, D, seed=D + N + past, spread=6.0)
    parents = random_tree(N, seed=N)
    args = [t.to(DEV) for t in (q, k, v)] + [torch.tensor(parents, dtype=torch.int32, device=DEV)]
    o, lse = attn.decode_tree(*args, past, return_lse=True)
    check(o, lse, reference(q, k, v, parents, past, 0, 1.0), f"{D} {rows} {past}")
    again = attn.decode_tree(*args, past)
    assert torch.equal(o, again)


def test_a_chain_is_causal_attention():
    """A tree without branches is the prefill attention of the tokens after the context."""
    q, k, v = (t.to(DEV) for t in make(8, 1, 24, 324, 256, seed=3))
    parents = torch.arange(-1, 23, dtype=torch.int32, device=DEV)
    for window in (0, 100):
        o = attn.decode_tree(q, k, v, parents, 300, window)
        ref = reference(q.cpu(), k.cpu(), v.cpu(), list(range(-1, 23)), 300, window, 1.0)
        check(o, None, ref, "chain")
        check(attn.attention(q, k, v, 300, window), None, ref, "prefill attention")


def test_unused_nodes_see_nothing():
    """Nodes with an impossible parent, and what hangs on them: zero rows, lse -inf; the others as ever."""
    parents = [-1, 0, 2, 1, -2, 4, 5, 3, 99, -1, 8, -7]   # 2 (its own parent), 4, 8, 11 unused; 5, 6 and 10 hang on them
    M, past = len(parents), 77
    q, k, v = make(8, 1, M, past + M, 128, seed=11)
    for window in (0, 20):
        for n_past in (past, 5):
            o, lse = attn.decode_tree(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor(parents, dtype=torch.int32, device=DEV),
                                      n_past, window, return_lse=True)
            ref = reference(q, k, v, parents, n_past, window, 1.0)
            check(o, lse, ref, f"{window} {n_past}")
            for m in (2, 4, 5, 6, 8, 10, 11):
                assert (o[:, m] == 0).all() and torch.isneginf(lse[:, m]).all()


@pytest.mark.parametrize("D", [128, 256, 512])
@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan])
def test_what_is_not_seen_does_not_reach_a_row(D, what):
    """Infinities and NaN in the keys and values of other branches, before the window and behind the last
    node leave a row alone, and reach the rows that see them."""
    past, M, window = 200, 9, 50
    parents = [-1, 0, 1, 0, 3, 3, -1, 6, 7]
    q, k, v = make(8, 1, M, past + M + 8, D, seed=D)
    clean = reference(q, k, v, parents, past, window, 1.0)
    bad_k, bad_v = k.clone(), v.clone()
    hit = {past + 3, past + 8}                       # nodes 3 and 8: seen by 3, 4, 5 and by 8
    for r in [*range(past - window), *range(past + M, past + M + 8)]:
        bad_k[:, r], bad_v[:, r] = math.nan, what    # seen by no node (node 0 sees past - 49 on)
    for r in hit:
        bad_v[0, r, 5::7] = what
    o = attn.decode_tree(q.to(DEV), bad_k.to(DEV), bad_v.to(DEV), torch.tensor(parents, dtype=torch.int32, device=DEV), past,
                         window)
    seeing = [m for m in range(M) if hit & {past + c for c in chain_of(parents, m)}]
    assert seeing == [3, 4, 5, 8]
    rest = [m for m in range(M) if m not in seeing]
    check(o[:, rest], None, tuple(t[:, rest] for t in clean), "unseen")
    got = o[:, seeing].cpu().float()
    assert not torch.isfinite(got[..., 5::7]).any()
    assert (torch.isnan(got[..., 5::7]).all() if math.isnan(what) else (got[..., 5::7] == what).all())
    keep = [d for d in range(D) if d % 7 != 5]
    check(o[:, seeing][..., keep], None, tuple(t[:, seeing][..., keep] if t.dim() == 3 else t for t in clean), "their other columns")


def test_the_window_edge_of_deeper_nodes():
    """A NaN in a context row that the root sees and a deeper node no longer does."""
    past, window = 130, 40
    parents = [-1, 0, 1, 2, 3, 4]
    q, k, v = make(4, 1, 6, past + 6, 256, seed=5)
    clean = reference(q, k, v, parents, past, window, 1.0)
    row = past + 2 - (window - 1)     # the oldest that node 2 sees
    k[0, row], v[0, row] = math.nan, math.nan
    o = attn.decode_tree(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor(parents, dtype=torch.int32, device=DEV), past, window)
    assert torch.isnan(o[:, :3].float()).all()
    check(o[:, 3:], None, tuple(t[:, 3:] for t in clean), "deeper nodes")


def test_strided_operands_and_output():
    """[T, H, D] storage, a cache with spare rows and heads, an output into a strided view."""
    H, KV, N, D, past, cap = 8, 2, 6, 256, 90, 160
    q, k, v = make(H, KV, N, cap, D, seed=9)
    parents = random_tree(N, seed=2)
    qd = q.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)             # [N, H, D] storage
    kd = torch.full((cap, KV + 1, D + 8), math.nan, dtype=torch.bfloat16, device=DEV)
    vd = kd.clone()
    kd[:, :KV, :D], vd[:, :KV, :D] = k.to(DEV).transpose(0, 1), v.to(DEV).transpose(0, 1)
    store = torch.full((N, H, D + 16), 7.0, dtype=torch.bfloat16, device=DEV)
    o = attn.decode_tree(qd, kd[:, :KV, :D].transpose(0, 1), vd[:, :KV, :D].transpose(0, 1),
                         torch.tensor(parents, dtype=torch.int32, device=DEV), past, out=store[:, :, :D].transpose(0, 1))
    check(o, None, reference(q, k, v, parents, past, 0, 1.0), "strided")
    assert o.data_ptr() == store.data_ptr() and (store[:, :, D:] == 7.0).all()


def test_length_in_device_memory_and_graph_replay():
    """One captured launch replayed at several context lengths, with eager work between the replays."""
    H, KV, N, D, cap = 8, 1, 7, 256, 700
    q, k, v = (t.to(DEV) for t in make(H, KV, N, cap, D, seed=21))
    parents = torch.tensor(random_tree(N, seed=4), dtype=torch.int32, device=DEV)
    n_past = torch.tensor([0], dtype=torch.int32, device=DEV)
    for window in (0, 64):
        out = torch.empty(H, N, D, dtype=torch.bfloat16, device=DEV)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            attn.decode_tree(q, k, v, parents, n_past, window, out=out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            attn.decode_tree(q, k, v, parents, n_past, window, out=out)
        for past in (0, 1, 31, 333, 693, 64):
            n_past.fill_(past)
            graph.replay()
            torch.cuda.synchronize()
            ref = reference(q.cpu(), k.cpu(), v.cpu(), parents.tolist(), past, window, 1.0)
            check(out, None, ref, f"replayed at {past}")
            check(attn.decode_tree(q, k, v, parents, past, window), None, ref, f"eager at {past}")
        for past in (-5, 694, 1 << 30):  # the caller's error: no access outside the cache
            n_past.fill_(past)
            graph.replay()
            torch.cuda.synchronize()
            clamped = max(0, min(past, cap - N))
            check(out, None, reference(q.cpu(), k.cpu(), v.cpu(), parents.tolist(), clamped, window, 1.0), f"clamped {past}")


def test_a_cache_whose_offsets_pass_32_bits():
    """Rows 40 KiB apart: the last key lies more than 4 GiB behind the first."""
    past, D, step = 110_000, 128, 20480
    M = 5
    store = torch.empty((past + M) * step, dtype=torch.bfloat16, device=DEV)
    rows = store.view(past + M, step)[:, :2 * D]
    g = torch.Generator(device=DEV).manual_seed(1)
    rows.copy_(torch.randn(past + M, 2 * D, generator=g, device=DEV))
    k, v = rows[None, :, :D], rows[None, :, D:]
    q = (torch.randn(4, M, D, generator=g, device=DEV) * 0.4).bfloat16()
    parents = [-1, 0, 0, -1, 3]
    o = attn.decode_tree(q, k, v, torch.tensor(parents, dtype=torch.int32, device=DEV), past)
    check(o, None, reference(q.cpu(), k.cpu(), v.cpu(), parents, past, 0, 1.0), "far rows")


def test_on_another_stream():
    q, k, v = (t.to(DEV) for t in make(8, 1, 5, 905, 128, seed=2))
    parents = torch.tensor([-1, 0, 0, 1, 1], dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        o = attn.decode_tree(q, k, v, parents, 900)
    stream.synchronize()
    check(o, None, reference(q.cpu(), k.cpu(), v.cpu(), parents.tolist(), 900, 0, 1.0), "stream")


def test_refusals():
    q, k, v = (t.to(DEV) for t in make(8, 1, 4, 104, 128, seed=1))
    parents = torch.tensor([-1, 0, 0, 1], dtype=torch.int32, device=DEV)
    ok = dict(q=q, k=k, v=v, parents=parents, n_past=100)
    attn.decode_tree(**ok)
    for change, error in [
        (dict(q=q.cpu()), ValueError), (dict(q=q.float()), TypeError), (dict(q=q[0]), ValueError),
        (dict(k=k[:, :50]), ValueError), (dict(v=v[:, :, :64]), ValueError),
        (dict(parents=parents.long()), ValueError), (dict(parents=parents.cpu()), ValueError),
        (dict(parents=parents[:3]), ValueError), (dict(parents=parents[:0]), ValueError),
        (dict(n_past=101), ValueError), (dict(n_past=-1), ValueError),
        (dict(n_past=torch.tensor([100], device=DEV)), ValueError),
        (dict(window=-1), ValueError), (dict(scale=0.0), W8A8Error), (dict(scale=math.inf), W8A8Error),
        (dict(out=torch.empty(8, 4, 64, dtype=torch.bfloat16, device=DEV)), ValueError),
        (dict(workspace=torch.empty(16, dtype=torch.uint8, device=DEV)), W8A8Error),
        (dict(q=q[:7, :, :], k=torch.cat([k, k]), v=torch.cat([v, v])), ValueError),   # 7 heads on 2
        (dict(q=q[:, :, :64].contiguous(), k=k[:, :, :64].contiguous(), v=v[:, :, :64].contiguous()), (ValueError, W8A8Error)),
        (dict(q=q.new_empty(8, 4, 132)[:, :, 1:129]), W8A8Error),                      # not 16-byte aligned
    ]:
        with pytest.raises(error):
            attn.decode_tree(**{**ok, **change})
    many = torch.full((129,), -1, dtype=torch.int32, device=DEV)
    with pytest.raises((ValueError, W8A8Error)):
        attn.decode_tree(q, torch.cat([k, k], 1), torch.cat([v, v], 1), many, 10)


PLANS = [
    # H, KV, N, past, D, rows per workgroup, several parts
    (16, 1, 33, 0, 128, 32, False), (1024, 64, 10, 0, 128, 64, False), (1024, 64, 20, 0, 128, 80, False), (384, 64, 64, 0, 128, 96, False),
    (512, 32, 64, 0, 128, 128, False), (16, 1, 128, 0, 128, 64, True), (16, 1, 33, 2000, 128, 80, True), (10, 2, 33, 8000, 128, 96, True),
    (256, 16, 33, 500, 128, 128, True), (32, 2, 33, 100, 256, 32, True), (16, 16, 33, 2000, 256, 64, True), (16, 1, 33, 2000, 256, 80, True),
    (10, 2, 33, 8000, 256, 96, True), (24, 8, 33, 8000, 256, 128, True), (512, 32, 64, 0, 256, 128, False), (16, 1, 33, 0, 512, 32, True),
    (1024, 64, 10, 0, 512, 64, False), (16, 1, 128, 0, 512, 64, True), (16, 4, 33, 8000, 512, 80, True), (64, 8, 12, 8000, 512, 96, True),
    (96, 16, 64, 2000, 512, 128, True), (256, 16, 128, 0, 512, 128, False),
]


def plan(H, KV, N, M, Tk, D, past, window=0):
    import ctypes

    from w8a8 import _lib
    tile, parts = ctypes.c_int(), ctypes.c_int()
    assert _lib.lib().w8a8_attention_tree_plan(H, KV, N, M, Tk, D, past, window, ctypes.byref(tile), ctypes.byref(parts)) == 0
    return tile.value, parts.value


@pytest.mark.parametrize("case", PLANS, ids=lambda c: "x".join(map(str, c)))
def test_every_row_tile(case):
    """Each row tile of the plan, with one part of the keys and with several; a branch's V holds an infinity."""
    H, KV, N, past, D, tile, several = case
    got = plan(H, KV, N, N, past + N, D, past)
    assert got[0] == tile and (got[1] > 1) == several, got
    q, k, v = (t.to(DEV) for t in make(H, KV, N, past + N, D, seed=tile))
    parents = random_tree(N, seed=N)
    parents[-1] = -1
    v[:, past + N - 1, 3] = math.inf    # the last node: a branch of its own
    o, lse = attn.decode_tree(q, k, v, torch.tensor(parents, dtype=torch.int32, device=DEV), past, return_lse=True)
    seen = torch.ones(N, past + N, dtype=torch.bool, device=DEV)
    seen[:, past:] = False
    for i in range(N):
        seen[i, [past + c for c in chain_of(parents, i)]] = True
    s = torch.matmul(q.double().view(KV, -1, D), k.double().transpose(1, 2).contiguous()).view(H, N, -1)
    s = s.masked_fill(~seen, -math.inf)
    rl = torch.logsumexp(s, -1)
    p = torch.softmax(s, -1).view(KV, -1, past + N)
    clean = v.double().clone()
    clean[:, past + N - 1, 3] = 0.0
    ro, mag = torch.matmul(p, clean).view(H, N, D), torch.matmul(p, clean.abs()).view(H, N, D)
    assert torch.isinf(o[:, -1, 3]).all()
    o[:, -1, 3] = ro[:, -1, 3].bfloat16()
    check(o, lse, (ro.cpu(), mag.cpu(), rl.cpu()), str(case))
