"""DecayAttentionLIF: the norm and rotation, the attention, and the LIF together,
against the same steps in 64 bits, and against itself in pieces."""
import pytest
import torch

import oracle
from lif_parity import lif_trace

pytestmark = pytest.mark.gpu


def _block(dev, **kw):
    from catfuse_b200.decay_block import DecayAttentionLIF
    from catfuse_b200.ops import LIFConfig
    torch.manual_seed(1)
    m = DecayAttentionLIF(96, heads=6, kv_heads=3, head_dim=32, lif=LIFConfig(v_threshold=0.3),
                          dtype=torch.float16, **kw).to(dev)
    with torch.no_grad():
        m.q_weight.uniform_(0.8, 1.2)
        m.k_weight.uniform_(0.8, 1.2)
    return m


def test_block_follows_its_definition(dev):
    m = _block(dev, sections=(4, 6, 6))
    B, L = 2, 100
    x = torch.randn(B, L, 96, device=dev)
    t = torch.arange(L, device=dev)
    pos = torch.stack([t // 25, t // 5 % 5, t % 5])[:, None].expand(3, B, L).contiguous()
    spikes = m(x, pos)
    # every stage fed the block's own input of that stage (fp16), in 64 bits
    qkv = m.qkv(x.half())
    q, k, v = (z.unflatten(-1, (-1, 32)) for z in qkv.split((192, 96, 96), -1))
    from catfuse_b200 import ops
    qr, kr = ops.qk_norm_rope(q, k, pos, m.inv_freq, q_weight=m.q_weight, k_weight=m.k_weight, sections=(4, 6, 6))
    flat = pos.reshape(3, -1)
    for got, src, w in ((qr, q, m.q_weight), (kr, k, m.k_weight)):
        want, bound = oracle.qk_norm_rope(src.flatten(0, 1), flat, m.inv_freq, weight=w, sections=(4, 6, 6))
        err = (got.flatten(0, 1).cpu().double() - want).abs()
        assert (err <= 2.0 ** -11 * want.abs() + 2.0 ** -20 * bound + 2.0 ** -25).all()
    y = []
    for b in range(B):
        o, _, a, _ = oracle.decay_attention(qr[b], kr[b], v[b], m.log_decay)
        y.append(o.flatten(1))
    z = (torch.stack(y, 1).half().to(dev) @ m.proj.weight.detach().T).float().cpu().numpy()
    s, _, h = lif_trace(z, vth=0.3)
    got = spikes.transpose(0, 1).cpu().numpy()
    flips = got != s
    assert 0.01 < s.mean() < 0.99
    # attention and projection are rounded to fp16: only spikes near the threshold may differ
    assert flips.mean() <= 2e-2 and (abs(h[flips] - 0.3) < 2e-2).mean() >= 0.5


def test_block_in_pieces(dev):
    m = _block(dev)
    B, L = 3, 150
    x = torch.randn(B, L, 96, device=dev)
    pos = torch.arange(L, device=dev, dtype=torch.int32).repeat(B, 1)
    whole = m(x, pos)
    m.reset()
    parts = [m(x[:, :70], pos[:, :70].contiguous()), m(x[:, 70:131], pos[:, 70:131].contiguous())]
    for t in range(131, L):
        parts.append(m.step(x[:, t], pos[:, t].contiguous())[:, None])
    # a state rounded to fp16 for its product or not: a spike at the threshold may tip
    assert (torch.cat(parts, 1) != whole).float().mean() <= 2e-2
    m.reset()
    assert torch.equal(m(x, pos), whole)
