"""fp16 prompts hand a power of two per row from the warps that scale it to
those that undo it: every chunk has to meet its own."""
import pytest
import torch

from decay_parity import check_out, check_state, chunked

pytestmark = pytest.mark.gpu

DIMS = [(64, 64), (64, 128), (128, 64), (128, 128)]


def _inputs(n, hq, hk, dk, dv, seed, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [torch.randn(n, h, d, generator=g, device=dev) for h, d in ((hq, dk), (hk, dk), (hk, dv))]


def _steps(lens, dev):
    """2^(chunk mod 5) of every token, chunks of 64 counted from its sequence's start."""
    return torch.cat([2.0 ** (torch.arange(n, device=dev) // 64 % 5) for n in lens])[:, None, None]


def _decays(hk, dev):
    some = [-1e-3, 0.0, -0.02, -0.3, -2.0]
    return torch.tensor([some[i % len(some)] for i in range(hk)], device=dev)


@pytest.mark.parametrize("dims", DIMS)
def test_segment_sums_of_many_chunks_and_units(dev, dims):
    """Packed sequences cut into segments of 24 to 34 chunks, several of them summed by
    each CTA, in which no two neighbouring chunks have the same scale."""
    from catfuse_b200 import ops
    dk, dv = dims
    lens, h = [8000, 7423, 8100, 9001, 6400, 8192, 7777, 8107], 16
    q, k, v = _inputs(sum(lens), h, h, dk, dv, 1, dev)
    v = v * _steps(lens, dev)
    q, k, v = q.half(), k.half(), v.half()
    ld = _decays(h, dev)
    s0 = torch.randn(len(lens), h, dk, dv, device=dev, generator=torch.Generator(device=dev).manual_seed(2))
    s1 = torch.empty_like(s0)
    cu = torch.tensor([0] + lens, device=dev).cumsum(0).to(torch.int32)
    out = ops.decay_attention(q, k, v, ld, s_in=s0, s_out=s1, cu_seqlens=cu)
    b = cu.tolist()
    for i in range(len(lens)):
        part = slice(b[i], b[i + 1])
        o, S, ao, aS = chunked(q[part], k[part], v[part], ld, s_in=s0[i])
        check_out(out[part], o, ao, f"sequence {i}")
        check_state(s1[i], S, aS, f"state {i}")


@pytest.mark.parametrize("dims", DIMS)
def test_segment_sums_of_one_long_prompt(dev, dims):
    from catfuse_b200 import ops
    dk, dv = dims
    n, h = 40000, 16
    q, k, v = _inputs(n, h, h, dk, dv, 3, dev)
    v = v * _steps([n], dev)
    q, k, v = q.half(), k.half(), v.half()
    ld = _decays(h, dev)
    s0 = torch.randn(1, h, dk, dv, device=dev, generator=torch.Generator(device=dev).manual_seed(4))
    s1 = torch.empty_like(s0)
    out = ops.decay_attention(q[None], k[None], v[None], ld, s_in=s0, s_out=s1)
    o, S, ao, aS = chunked(q, k, v, ld, s_in=s0[0])
    check_out(out[0], o, ao)
    check_state(s1[0], S, aS)


@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("states", ["none", "some", "all"])
def test_units_that_start_from_zeros(dev, dims, aligned, states):
    """More (sequence, head) pairs than CTAs, long and short, where all, some or none
    begin with a state; neighbours differ in size by up to 2^6."""
    from catfuse_b200 import ops
    dk, dv = dims
    h, n_seq = 8, 64
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(60, 400, (n_seq,), generator=g).tolist()
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    b = cu.tolist()
    q, k, v = _inputs(b[-1], h, h, dk, dv, 6, dev)
    for i in range(n_seq):
        v[b[i]:b[i + 1]] *= 2.0 ** (i * 3 % 7)
    q, k, v = q.half(), k.half(), v.half()
    ld = _decays(h, dev)
    pool = 30.0 * torch.randn(n_seq, h, dk, dv, generator=g).to(dev)
    slots = torch.arange(n_seq, dtype=torch.int32)
    if states == "some":
        slots[torch.rand(n_seq, generator=g) < 0.6] = -1
    s_in = None if states == "none" else pool
    s_out = torch.zeros_like(pool)
    wide = torch.zeros(b[-1], h, dv + (0 if aligned else 3), dtype=torch.float16, device=dev)
    ops.decay_attention(q, k, v, ld, s_in=s_in, s_out=s_out, slots=slots.to(dev), cu_seqlens=cu.to(dev),
                        out=wide[..., :dv])
    for i in range(n_seq):
        part = slice(b[i], b[i + 1])
        held = s_in is not None and slots[i] >= 0
        o, S, ao, aS = chunked(q[part], k[part], v[part], ld, s_in=pool[i] if held else None)
        check_out(wide[part, :, :dv], o, ao, f"sequence {i}")
        if slots[i] >= 0:
            check_state(s_out[i], S, aS, f"state {i}")
        else:
            assert (s_out[i] == 0).all()
    assert (wide[..., dv:] == 0).all()
