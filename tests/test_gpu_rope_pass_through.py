"""Channels beyond the rotated ones pass through, whatever their neighbours hold."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("pairing", ["half", "adjacent"])
@pytest.mark.parametrize("dims", [(64, 32), (80, 60), (128, 64), (24, 8), (250, 130), (10, 6), (64, 0)])
def test_non_finite_channels_stay_alone(dev, dtype, pairing, dims):
    from catfuse_b200 import ops
    d, rot = dims
    g = torch.Generator().manual_seed(d)
    q, k = [torch.randn(20, h, d, generator=g).to(dtype).to(dev) for h in (5, 2)]
    pos = torch.arange(20, device=dev, dtype=torch.int32)
    freq = 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float32, device=dev) / max(rot // 2, 1))
    clean = ops.qk_norm_rope(q, k, pos, freq, norm=False, pairing=pairing)
    assert torch.equal(clean[0][..., rot:], q[..., rot:]) and torch.equal(clean[1][..., rot:], k[..., rot:])
    for c in {rot, (rot + d) // 2, d - 1}:
        for bad in (float("inf"), float("-inf"), float("nan")):
            q2, k2 = q.clone(), k.clone()
            q2[3, 1, c] = k2[7, 0, c] = bad
            got = ops.qk_norm_rope(q2, k2, pos, freq, norm=False, pairing=pairing)
            for a, b, at in ((got[0], clean[0], (3, 1, c)), (got[1], clean[1], (7, 0, c))):
                assert torch.equal(a[at], torch.tensor(bad, dtype=dtype, device=dev)) or bad != bad and a[at].isnan()
                keep = torch.ones_like(b, dtype=torch.bool)
                keep[at] = False
                assert torch.equal(a[keep], b[keep])
