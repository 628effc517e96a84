"""The chunked 64-bit form of the long-prompt tests against the oracle's recurrence."""
import pytest
import torch

import oracle
from decay_parity import chunked


@pytest.mark.parametrize("n", [0, 1, 255, 256, 700])
@pytest.mark.parametrize("carried", [False, True])
def test_chunked_form_equals_the_recurrence(n, carried):
    g = torch.Generator().manual_seed(n)
    q, k, v = (torch.randn(n, h, d, generator=g) for h, d in ((4, 8), (2, 8), (2, 16)))
    s0 = torch.randn(2, 8, 16, generator=g) if carried else None
    for ld in ([-0.01, -1.0], [0.0, float("-inf")]):
        ld = torch.tensor(ld)
        for got, want in zip(chunked(q, k, v, ld, 0.3, s0), oracle.decay_attention(q, k, v, ld, 0.3, s0)):
            assert got.shape == want.shape
            assert torch.allclose(got, want, rtol=1e-11, atol=1e-11)
