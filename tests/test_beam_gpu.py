"""A beam search step's choice (ops.beam_select) against its definition in 64 bits.

Beams and tokens must be equal: the scores are ranked in 64 bits, and the inputs' scores are either equal as
numbers (ties, which go to the lowest index) or further apart than the sums of exponentials are exact (fp32
terms and sums of a chunk: a few 2^-24 of the sum, below 2e-6 in its logarithm; the tests check the gaps of the
candidates around the choice).  Scores: that error and one rounding."""
import math

import pytest
import torch

from w8a8 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
LSE_ERR = 2e-6


def reference(logits, scores, k):
    """(values, beams, tokens) [B, k] in 64 bits."""
    B, nb, V = logits.shape
    x = logits.double()
    m = x.amax(-1, keepdim=True)
    none = (m[..., 0] == -math.inf) & ~torch.isnan(x).any(-1)
    lse = torch.where(torch.isinf(m) & (m < 0), 0.0, m) + torch.log(torch.exp(x - torch.where(m == -math.inf, 0.0, m)).sum(-1, keepdim=True))
    base = torch.where(none, torch.where(torch.isnan(scores), scores, -math.inf).double(), scores.double() - lse[..., 0])
    val = torch.where(torch.isfinite(base)[..., None], x + base[..., None], base[..., None].expand_as(x))
    flat = val.reshape(B, nb * V)
    v, at = torch.sort(flat, dim=1, descending=True, stable=True)
    return v[:, :k], at[:, :k] // V, at[:, :k] % V, v


def check(logits, scores, k, what, gaps=True):
    B, nb, V = logits.shape
    value, beam, token = ops.beam_select(logits.to(DEV), scores.to(DEV), k)
    rv, rb, rt, allv = reference(logits, scores, k)
    if gaps:  # neighbours around the choice are equal or well apart
        near = allv[:, : k + 1]
        d = (near[:, :-1] - near[:, 1:])
        d = d[torch.isfinite(d)]
        assert ((d == 0) | (d > 2 * LSE_ERR)).all(), f"{what}: the inputs' scores are too close to rank"
    assert torch.equal(beam.cpu(), rb), f"{what}: beams"
    assert torch.equal(token.cpu(), rt), f"{what}: tokens"
    got, ref = value.double().cpu(), rv
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), what
    assert torch.equal(torch.isinf(got), torch.isinf(ref)), what
    ok = torch.isfinite(ref)
    assert ((got - ref).abs()[ok] <= LSE_ERR + 2.0 ** -24 * ref.abs()[ok]).all(), what
    assert token.dtype == beam.dtype == torch.int64 and value.dtype == torch.float32


def make(B, nb, V, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, nb, V, generator=g) * spread
    return (x.bfloat16() if dtype == "bf16" else x), -20 * torch.rand(B, nb, generator=g)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("shape", [
    # B, nb, V, k
    (1, 1, 1, 1), (1, 1, 7, 7), (1, 2, 5, 10), (1, 4, 1000, 8), (3, 5, 8192, 16), (2, 3, 8193, 64), (1, 16, 20001, 64),
    (1, 4, 262144, 8), (2, 8, 32003, 16), (5, 1, 4096, 5), (1, 64, 3001, 32), (1, 200, 100, 64), (1, 3, 65537, 1),
    (1, 64, 32000, 64), (2, 256, 2000, 64), (1, 8, 262144, 64), (1, 100, 12345, 40),
], ids=lambda s: "x".join(map(str, s)))
def test_matches_the_definition(shape, dtype):
    B, nb, V, k = shape
    x, s = make(B, nb, V, dtype, seed=V + k)
    check(x, s, k, f"{shape} {dtype}")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("V", [50, 8192, 30000])
def test_ties_go_to_the_lowest_index(V, dtype):
    """Equal logits, equal beams and a few values only."""
    g = torch.Generator().manual_seed(V)
    for k in (1, 5, 33, 64):
        x = torch.zeros(1, 4, V)
        check(x.bfloat16() if dtype == "bf16" else x, torch.zeros(1, 4), k, "all equal")
        x = torch.randint(0, 3, (1, 4, V), generator=g).float()
        x[0, 2] = x[0, 0]
        x = x.bfloat16() if dtype == "bf16" else x
        s = torch.tensor([[-1.0, -9.0, -1.0, -20.0]])
        check(x, s, k, "few values, two equal beams")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("V", [40, 9000, 40000])
def test_masked_tokens_and_beams(V, dtype):
    cast = (lambda x: x.bfloat16()) if dtype == "bf16" else (lambda x: x)
    x, s = make(2, 4, V, "fp32", seed=V)
    # the first step: one beam, the others out
    check(cast(x), torch.tensor([[0.0, -math.inf, -math.inf, -math.inf]] * 2), 8, "first step")
    # a grammar that allows few tokens, more candidates asked for than there are
    y = torch.full_like(x, -math.inf)
    y[:, :, 3::max(1, V // 5)] = x[:, :, 3::max(1, V // 5)]
    check(cast(y), s, 16, "few tokens")
    check(cast(y), s, 33, "more than there are")
    # a beam that nothing can follow
    y = x.clone()
    y[0, 1] = -math.inf
    check(cast(y), s, 8, "no token")
    check(cast(torch.full_like(x, -math.inf)), s, 5, "nothing at all")
    # masks of the type's lowest value
    y = x.clone()
    y[:, :, ::2] = torch.finfo(torch.bfloat16 if dtype == "bf16" else torch.float32).min
    check(cast(y), s, 12, "lowest value")


@pytest.mark.parametrize("V,allowed", [(8192, 1), (8192, 7), (262144, 40), (70, 3)])
def test_a_grammar_with_few_tokens(V, allowed):
    """Less tokens than are asked for in each chunk, the allowed ones among the first or the last."""
    for seed in range(3):
        x, s = make(1, 3, V, "fp32", seed=V + seed)
        at = torch.randperm(V, generator=torch.Generator().manual_seed(seed))[:allowed]
        at = at if seed == 0 else at % 64 if seed == 1 else V - 1 - at % 64
        y = torch.full_like(x, -math.inf)
        y[:, :, at] = x[:, :, at]
        for k in (1, 8, 64):
            check(y, s, k, f"{V} {allowed} {seed} {k}")


def test_nan_and_infinite_logits():
    x, s = make(1, 3, 5000, "fp32", seed=1)
    y = x.clone()
    y[0, 1, 77] = math.nan
    check(y, s, 6, "a NaN logit")
    y[0, 1, 77] = math.inf
    check(y, s, 6, "an infinite logit")
    s2 = s.clone()
    s2[0, 2] = math.nan
    check(x, s2, 6, "a NaN score")


def test_strided_logits_one_request_and_workspace():
    x, s = make(2, 3, 1001, "fp32", seed=2)
    big = torch.full((2, 4, 1009), 50.0)
    big[:, :3, 4:1005] = x
    dev = big.to(DEV)[:, :3, 4:1005]
    for t in (dev, dev.bfloat16()):
        v, b, tok = ops.beam_select(t, s.to(DEV), 9)
        rv, rb, rt, _ = reference(t.cpu(), s, 9)
        assert torch.equal(b.cpu(), rb) and torch.equal(tok.cpu(), rt)
    ws = torch.empty(ops.beam_select_workspace_bytes(1, 3, 1001, 9), dtype=torch.uint8, device=DEV)
    v1, b1, t1 = ops.beam_select(dev[1], s[1].to(DEV), 9, workspace=ws)
    v, b, tok = ops.beam_select(dev, s.to(DEV), 9)
    assert v1.shape == (9,) and torch.equal(v1, v[1]) and torch.equal(b1, b[1]) and torch.equal(t1, tok[1])


def test_graph_replay():
    x, s = make(1, 4, 20000, "bf16", seed=3)
    xd, sd = x.to(DEV), s.to(DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.beam_select(xd, sd, 8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = ops.beam_select(xd, sd, 8)
    for seed in (4, 5, 6):
        y, s2 = make(1, 4, 20000, "bf16", seed=seed)
        xd.copy_(y)
        sd.copy_(s2)
        graph.replay()
        torch.cuda.synchronize()
        _, rb, rt, _ = reference(y, s2, 8)
        assert torch.equal(out[1].cpu(), rb) and torch.equal(out[2].cpu(), rt)


def test_refusals():
    x, s = make(2, 3, 100, "fp32", seed=1)
    x, s = x.to(DEV), s.to(DEV)
    for args, error in [
        ((x.cpu(), s.cpu(), 2), ValueError), ((x, s.cpu(), 2), ValueError), ((x.half(), s, 2), TypeError),
        ((x, s.double(), 2), TypeError), ((x, s[:, :2], 2), ValueError), ((x, s, 0), ValueError), ((x, s, 65), ValueError),
        ((x[:, :, :10], s, 31), ValueError), ((x.transpose(1, 2), s, 2), ValueError), ((x[..., ::2], s, 2), ValueError),
        ((torch.zeros(1, 257, 4, device=DEV), torch.zeros(1, 257, device=DEV), 2), ValueError),
    ]:
        with pytest.raises(error):
            ops.beam_select(*args)
