"""A beam search step's choice (ops.beam_select) where the join lists more candidates than it ranks at once and where
logits are finite but far out, against its definition in 64 bits.

Tolerance of a score: `err` for the beam's logsumexp, and the rounding to fp32 (half a step, 2^-24 of the value).  Where the
order of near ties is not what a test is about its inputs are more than `gap` apart and `err` is 2e-6, what sums in 32 bits
would be off by."""
import math

import pytest
import torch

from w8a8 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def reference(logits, scores, k):
    """(values, beams, tokens) [B, k] and the ranked values of all, in 64 bits."""
    B, nb, V = logits.shape
    x = logits.double()
    x = x - x.amax(-1, keepdim=True)
    x = x - torch.log(torch.exp(x).sum(-1, keepdim=True)) + scores.double()[..., None]
    v, at = torch.sort(x.reshape(B, nb * V), dim=1, descending=True, stable=True)
    return v[:, :k], at[:, :k] // V, at[:, :k] % V, v


def check(logits, scores, k, what, gap=4e-6, err=2e-6):
    """Compares with the reference; the inputs' scores around the choice are equal or more than `gap` apart."""
    value, beam, token = ops.beam_select(logits.to(DEV), scores.to(DEV), k)
    rv, rb, rt, allv = reference(logits, scores, k)
    near = allv[:, : k + 1]
    d = near[:, :-1] - near[:, 1:]
    assert ((d == 0) | (d > gap)).all(), f"{what}: the inputs' scores are too close to rank"
    assert torch.equal(beam.cpu(), rb), f"{what}: beams"
    assert torch.equal(token.cpu(), rt), f"{what}: tokens"
    assert ((value.double().cpu() - rv).abs() <= err + 2.0 ** -24 * rv.abs()).all(), what


@pytest.mark.parametrize("scores", ["equal", "near", "far", "farther", "one", "class"])
def test_the_join_tightens_its_bound_more_than_once(scores):
    """64 of 256 beams: thousands of candidates pass the first bound, more than a thousand the next."""
    nb, V, k = 256, 600, 64
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        x = torch.randn(1, nb, V, generator=g) * 3
        at = torch.randperm(nb, generator=g).float()[None]
        s = {"equal": 0 * at, "near": -0.01 * at, "far": -0.5 * at, "farther": -10 * at, "one": torch.where(at == 7, 0.0, -900.0),
             "class": torch.where(torch.arange(nb)[None] % 16 == 0, 0.0, -900.0)}[scores]
        check(x, s, k, f"{scores} {seed}")


LOWEST = {"fp32": torch.finfo(torch.float32).min, "bf16": torch.finfo(torch.bfloat16).min}


def cast(x, dtype):
    return x.bfloat16() if dtype == "bf16" else x


# B, nb, V: chunks of 4096 logits with a short last one, chunks of 8192, one chunk
SHAPES = [(1, 3, 12293), (9, 8, 60001), (2, 4, 900)]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("mask", ["lowest", -1e30, -1e10])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_whole_chunks_under_a_finite_mask(shape, mask, dtype):
    """A grammar's mask in finite numbers that leaves a few tokens, all in one chunk: the first, one between, the last."""
    B, nb, V = shape
    mask = LOWEST[dtype] if mask == "lowest" else mask
    for seed, first in enumerate((0, V // 2, V - 30)):
        g = torch.Generator().manual_seed(V + seed)
        x = torch.full((B, nb, V), mask)
        x[:, :, first:first + 30] = torch.randn(B, nb, 30, generator=g) * 3
        s = -20 * torch.rand(B, nb, generator=g)
        check(cast(x, dtype), s, 8, f"tokens from {first} on")
        if mask != -1e10:  # more than there are: the masked tokens' scores are the mask's, the lowest token first
            check(cast(x[:1, :2], dtype), s[:1, :2], 64, f"60 tokens from {first} on")
    if V < 4096:
        return
    # the short last chunk only
    g = torch.Generator().manual_seed(V)
    x = torch.randn(B, nb, V, generator=g) * 3
    x[:, :, V - V % 4096:] = mask
    s = -20 * torch.rand(B, nb, generator=g)
    check(cast(x, dtype), s, 8, "the last chunk masked")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("size", [1e9, 1e10, 1e20, 3e38])
def test_large_finite_logits(size, dtype):
    for V in (700, 9000):
        g = torch.Generator().manual_seed(V)
        x = torch.randn(1, 3, V, generator=g) * 3
        x[0, 0, V - 5:] = size * (1 - 0.1 * torch.arange(5))      # one token takes all
        x[0, 1] = -size * torch.rand(V, generator=g)
        x[0, 2, ::7] = size
        check(cast(x, dtype), torch.tensor([[-3.0, -4.0, -2.5]]), 5, f"{V}")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("level", ["lowest", -1e30, -1e10, 1e10, 3e38])
def test_beams_whose_every_logit_is_far_out(level, dtype):
    """log_softmax does not depend on the logits' level: equal logits of any size give -log V, and beams at different levels
    are weighed by their scores."""
    level = LOWEST[dtype] if level == "lowest" else level
    for V in (700, 9000):
        g = torch.Generator().manual_seed(V)
        x = torch.randn(1, 4, V, generator=g) * 0.01
        x[0, 1], x[0, 3] = level, level
        x[0, 3, 5::V // 4] = -level if level < 0 else level * 0.5
        check(cast(x, dtype), torch.tensor([[-9.0, -1.25, -9.5, -30.0]]), 8, f"{V} one level")
        check(torch.full((1, 3, V), level).to(cast(x, dtype).dtype), torch.tensor([[-3.0, -1.0, -2.0]]), 9, f"{V} all")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("V,nb", [(500, 8), (9000, 8), (40000, 5), (12293, 64)])
def test_beams_that_differ_by_less_than_32_bits_resolve(V, nb, dtype):
    """The same logits in every beam but for one token that cannot follow, another one each and none of them likely: the
    beams' scores differ by those tokens' probabilities, 1e-10 to 1e-6.

    In 64 bits a term is off by a few 2^-53 times log2 of its share, a beam's sum by as much, its logarithm and score by a
    few 2^-53 of themselves: below 1e-13 in all.  The inputs' scores are at least 1e-12 apart."""
    g = torch.Generator().manual_seed(V + nb)
    row = cast(torch.randn(V, generator=g) * 3, dtype)
    x = row[None, None].repeat(1, nb, 1)
    p = torch.softmax(row.double(), 0)
    unlikely = torch.nonzero((p > 1e-10) & (p < 1e-6))[:, 0]
    unlikely = unlikely[torch.randperm(len(unlikely), generator=g)]
    _, first = torch.unique(p[unlikely], return_inverse=True)         # of different probabilities
    seen, out = set(), []
    for t, f in zip(unlikely.tolist(), first.tolist()):
        if f not in seen:
            seen.add(f)
            out.append(t)
    for i in range(nb):
        x[0, i, out[i]] = -math.inf
    for score in (-3.0, -17.375):
        check(x, torch.full((1, nb), score), 40, f"score {score}", gap=1e-12, err=1e-12)
