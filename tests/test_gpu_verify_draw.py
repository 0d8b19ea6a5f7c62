"""The drawn token of a verification (tree.verify_tree) at the ends of the random numbers and of the
rows."""

import pytest
import torch

from test_gpu_verify import _case, _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", ["chain", "drawn", "best"])
@pytest.mark.parametrize("V,used", [(131072, 9000), (131072, 50001), (20011, 12289), (9001, 4096)])
def test_rows_that_end_in_tokens_without_probability(mode, V, used):
    """A vocabulary padded with tokens of probability 0, and sizes from 1e-30 to 1 before them: a
    number of 1 (one in 64 bits that rounds to it) draws the last token that has any, as just below 1
    and every other number draw one that has."""
    for seed in range(3):
        p, tokens, par, u, draft, nodes = _case([1] * 6 + [5, 12], V, mode, torch.float32, seed)
        size = torch.rand(V, generator=torch.Generator().manual_seed(seed)) * 30 * (seed > 0)
        tokens = [t % used for t in tokens]
        for x in (p,) if draft is None else (p, draft):
            x *= 10.0 ** -size
            x[:, used:] = 0
            x /= x.sum(-1, keepdim=True)
        for value in (1.0, 1.0 - 2.0 ** -24, 0.5, 0.0):
            _check(p, tokens, par, torch.full_like(u, value), draft, nodes)
