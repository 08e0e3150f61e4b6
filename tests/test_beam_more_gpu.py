"""A beam search step's choice (ops.beam_select) where the join lists more candidates than it ranks at once, against its
definition in 64 bits.

Tolerance of a score: `err` for the beam's logsumexp (fp32 terms and sums of a chunk: a few 2^-24 of the sum, below 2e-6 in its
logarithm) and the rounding to fp32 (half a step, 2^-24 of the value)."""
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
