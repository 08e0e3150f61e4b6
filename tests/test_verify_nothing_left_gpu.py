"""ops.verify_drafts where a token is refused although the draft's distribution is the target's: nothing is left of p - q, and
the next token is p's, wherever the two rows lie in memory."""
import math

import pytest
import torch

from test_verify_gpu import DEV, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("b,n,v", [(3, 2, 4099), (2, 3, 20011), (1, 2, 262144), (2, 2, 524289), (1, 1, 1100003)])
def test_draft_is_target(b, n, v, dtype):
    g = torch.Generator(device=DEV).manual_seed(v)
    x, _, tok, u = make(g, b, n, v, dtype)
    wide = torch.zeros(b, n, v + 16, device=DEV, dtype=dtype)
    for lead in (0, 1, 3, 6):  # the draft's rows begin elsewhere in their 16-byte words
        d = wide[:, :, lead:v + lead]
        d.copy_(x[:, :n])
        for last in (0.0, 0.3, 0.9, 1.0 - 2.0 ** -24):
            u[:, n] = last
            for t in (1.0, 0.7):
                assert (check(x, torch.full_like(tok, v), u, d, t=t) == 0).all()  # a token outside the vocabulary
    x[:, 0, 7] = -math.inf  # one that neither may follow
    d = x[:, :n].clone()
    tok[:, 0] = 7
    assert (check(x, tok, u, d) == 0).all()
