"""Packed calls of very many sequences, few of which are long enough to be cut."""
import pytest
import torch

from decay_parity import HALF, check_out, check_state, chunked

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("carried", [False, True])
def test_long_sequences_among_many_short_ones(dev, dtype, carried):
    from catfuse_b200 import ops
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 40, (5000,), generator=g)
    lens[torch.tensor([0, 17, 2500, 4998, 4999])] = torch.tensor([3000, 5000, 9000, 1409, 2816])
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)]).to(torch.int32)
    b, n = cu.tolist(), int(cu[-1])
    hq, hk, d = 4, 2, 64
    gd = torch.Generator(device=dev).manual_seed(2)
    q, k, v = [torch.randn(n, h, d, generator=gd, device=dev).to(dtype) for h in (hq, hk, hk)]
    ld = torch.tensor([-0.001, -0.4], device=dev)
    s0 = torch.randn(5000, hk, d, d, generator=gd, device=dev)
    s1 = s0.clone()
    out = ops.decay_attention(q, k, v, ld, s_in=s1 if carried else None, s_out=s1, cu_seqlens=cu.to(dev))
    pick = [0, 1, 16, 17, 18, 2499, 2500, 2501, 4997, 4998, 4999] + torch.randint(5000, (60,), generator=g).tolist()
    for i in pick:
        part = slice(b[i], b[i + 1])
        o, S, ao, aS = chunked(q[part], k[part], v[part], ld, s_in=s0[i] if carried else None)
        check_out(out[part], o, ao, f"sequence {i}")
        check_state(s1[i], S, aS, f"state {i}")


def test_short_sequences_need_no_states(dev):
    """65536 sequences of 16 tokens: a state for each would be 34 GB of workspace."""
    from catfuse_b200 import ops
    n_seq, length, h, d = 65536, 16, 8, 128
    g = torch.Generator(device=dev).manual_seed(3)
    q, k, v = [torch.randn(n_seq * length, h, d, generator=g, device=dev).bfloat16() for _ in range(3)]
    ld = -torch.exp2(torch.linspace(0.0, -9.0, h, device=dev))
    cu = torch.arange(0, n_seq * length + 1, length, device=dev, dtype=torch.int32)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = ops.decay_attention(q, k, v, ld, cu_seqlens=cu)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < 4 * out.numel() * 2
    for i in (0, 1, 777, 65535):
        part = slice(i * length, (i + 1) * length)
        o, _, ao, _ = chunked(q[part], k[part], v[part], ld)
        check_out(out[part], o, ao, f"sequence {i}")
