"""Decayed linear attention (cf_decay_attention, cf_decay_attention_step) against
the token-by-token recurrence in 64 bits.

Tolerances, per element.  With u the unit roundoff of the 16-bit type and A the
sum of the absolute values of an output's terms:

* outputs: rounded once on the way out (u |o|), and each term may have one
  factor rounded to 16 bits on its way through a matrix product (u A);
* states: fp32 throughout; products of 16-bit values are exact, a decay's power
  and the sums of up to a few thousand terms stay within 2^-18 A.
"""
import pytest
import torch

import oracle

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}
HALF = [torch.float16, torch.bfloat16]


def _log_decay(hk, kind="mixed"):
    if kind == "mixed":  # a state that keeps all, long and short memories, one that keeps nothing
        some = [0.0, -0.002, -0.05, -0.7, -4.0, float("-inf"), -40.0, -1e-6]
        return torch.tensor([some[i % len(some)] for i in range(hk)])
    return torch.full((hk,), float(kind))


def _make(lead, hq, hk, dk, dv, dtype, seed, values="normal"):
    g = torch.Generator().manual_seed(seed)
    if values == "spikes":
        return [(torch.rand(*lead, h, d, generator=g) < 0.3).to(dtype).cuda()
                for h, d in ((hq, dk), (hk, dk), (hk, dv))]
    return [torch.randn(*lead, h, d, generator=g).to(dtype).cuda()
            for h, d in ((hq, dk), (hk, dk), (hk, dv))]


def _check_out(got, want, terms, what=""):
    u = U[got.dtype]
    err = (got.cpu().double() - want).abs()
    tol = u * (want.abs() + terms) + TINY[got.dtype]
    assert torch.isfinite(err).all(), what
    assert (err <= tol).all(), f"{what}: {float((err / tol).max())} of the tolerance"


def _check_state(got, want, terms, what=""):
    err = (got.cpu().double() - want).abs()
    tol = 2.0 ** -18 * terms + 1e-37
    assert torch.isfinite(err).all(), what
    assert (err <= tol).all(), f"{what}: {float((err / tol).max())} of the tolerance"


def _check_sequences(q, k, v, ld, bounds, out, s_in, s_out, rows=None, scale=None):
    """Every sequence [a, b) of packed tokens against the oracle."""
    for i, (a, b) in enumerate(bounds):
        r = i if rows is None else rows[i]
        s0 = None if s_in is None else s_in[r]
        o, S, ao, aS = oracle.decay_attention(q[a:b], k[a:b], v[a:b], ld, scale, s0)
        _check_out(out[a:b], o, ao, f"sequence {i}")
        if s_out is not None:
            _check_state(s_out[r], S, aS, f"state {i}")


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("length", [1, 2, 15, 63, 64, 65, 127, 128, 129, 300])
def test_lengths(dev, dtype, length):
    from catfuse_b200 import ops
    q, k, v = _make((2, length), 8, 8, 128, 128, dtype, length)
    ld = _log_decay(8).to(dev)
    s0 = torch.randn(2, 8, 128, 128, generator=torch.Generator().manual_seed(1)).to(dev)
    s1 = torch.empty_like(s0)
    out = ops.decay_attention(q, k, v, ld, s_in=s0, s_out=s1)
    flat = [t.flatten(0, 1) for t in (q, k, v, out)]
    _check_sequences(*flat[:3], ld, [(0, length), (length, 2 * length)], flat[3], s0, s1)
    # without a state: from zeros, and nothing stored
    fresh = ops.decay_attention(q, k, v, ld).flatten(0, 1)
    _check_sequences(*flat[:3], ld, [(0, length), (length, 2 * length)], fresh, None, None)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("dims", [(8, 8), (16, 128), (24, 40), (32, 32), (48, 96), (64, 64), (64, 128),
                                  (72, 80), (128, 8), (128, 64), (120, 104)])
@pytest.mark.parametrize("heads", [(3, 3), (6, 2), (5, 1)])
def test_head_layouts(dev, dtype, dims, heads):
    from catfuse_b200 import ops
    (dk, dv), (hq, hk) = dims, heads
    q, k, v = _make((1, 150), hq, hk, dk, dv, dtype, dk + dv)
    ld = _log_decay(hk, "-0.03").to(dev)
    s = torch.randn(1, hk, dk, dv, generator=torch.Generator().manual_seed(2)).to(dev)
    s0 = s.clone()
    out = ops.decay_attention(q, k, v, ld, s_in=s, s_out=s, scale=0.25)  # in place
    _check_sequences(q[0], k[0], v[0], ld, [(0, 150)], out[0], s0, s, scale=0.25)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("heads", [(4, 4), (8, 2)])
def test_packed_sequences(dev, dtype, heads):
    from catfuse_b200 import ops
    hq, hk = heads
    lens = [0, 1, 64, 0, 0, 63, 200, 2, 129, 65, 0, 31]
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    n, S = int(cu[-1]), len(lens)
    q, k, v = _make((n,), hq, hk, 64, 128, dtype, 5)
    ld = _log_decay(hk).to(dev)
    g = torch.Generator().manual_seed(3)
    pool = torch.randn(S + 5, hk, 64, 128, generator=g).to(dev)
    before = pool.clone()
    slots = torch.randperm(S + 5, generator=g)[:S].to(torch.int32)
    slots[4], slots[7] = -1, S + 5  # no row: start from zeros, store nothing
    out = ops.decay_attention(q, k, v, ld, s_in=pool, s_out=pool, slots=slots.to(dev), cu_seqlens=cu.to(dev))
    touched = set()
    for i, s in enumerate(slots.tolist()):
        a, b = int(cu[i]), int(cu[i + 1])
        inside = 0 <= s < S + 5
        o, st, ao, ast = oracle.decay_attention(q[a:b], k[a:b], v[a:b], ld, s_in=before[s] if inside else None)
        _check_out(out[a:b], o, ao, f"sequence {i}")
        if inside:
            touched.add(s)
            if b > a:
                _check_state(pool[s], st, ast, f"state {i}")
            else:
                assert torch.equal(pool[s], before[s])  # no tokens: the state as it was
    for s in set(range(S + 5)) - touched:
        assert torch.equal(pool[s], before[s])


def test_tokens_outside_every_sequence_are_not_written(dev):
    from catfuse_b200 import ops
    q, k, v = _make((300,), 2, 2, 64, 64, torch.bfloat16, 6)
    ld = _log_decay(2, "-0.1").to(dev)
    cu = torch.tensor([10, 75, 75, 233], dtype=torch.int32)
    out = torch.full_like(v, 7.0)
    ops.decay_attention(q, k, v, ld, cu_seqlens=cu.to(dev), out=out)
    assert (out[:10] == 7).all() and (out[233:] == 7).all()
    _check_sequences(q, k, v, ld, [(10, 75), (75, 75), (75, 233)], out, None, None)
    # boundaries beyond the tokens are clamped to them
    out2 = torch.full_like(v, 7.0)
    ops.decay_attention(q, k, v, ld, cu_seqlens=torch.tensor([-5, 100, 4000], dtype=torch.int32, device=dev), out=out2)
    _check_sequences(q, k, v, ld, [(0, 100), (100, 300)], out2, None, None)


@pytest.mark.parametrize("dtype", HALF)
def test_non_finite_tokens_stay_in_their_sequence(dev, dtype):
    """Infinities and NaN in the tokens around a sequence (another sequence's, or
    padding) change none of its bits."""
    from catfuse_b200 import ops
    q, k, v = _make((300,), 2, 2, 64, 64, dtype, 7)
    ld = _log_decay(2, "-0.1").to(dev)
    cu = torch.tensor([40, 141], dtype=torch.int32, device=dev)
    s_a, s_b = (torch.empty(1, 2, 64, 64, device=dev) for _ in range(2))
    a = ops.decay_attention(q, k, v, ld, cu_seqlens=cu, s_out=s_a)
    for bad in (float("nan"), float("inf"), float("-inf"), torch.finfo(dtype).min):
        q2, k2, v2 = q.clone(), k.clone(), v.clone()
        for t in (q2, k2, v2):
            t[:40] = bad
            t[141:] = bad
        b = ops.decay_attention(q2, k2, v2, ld, cu_seqlens=cu, s_out=s_b)
        assert torch.equal(a[40:141], b[40:141]) and torch.equal(s_a, s_b)


@pytest.mark.parametrize("dtype", HALF)
def test_a_non_finite_value_does_not_reach_earlier_tokens(dev, dtype):
    from catfuse_b200 import ops
    q, k, v = _make((1, 200), 2, 2, 64, 64, dtype, 8)
    ld = _log_decay(2, "-0.1").to(dev)
    a = ops.decay_attention(q, k, v, ld)
    for at in (0, 30, 100, 199):
        for which in range(3):
            for bad in (float("nan"), float("inf")):
                t = [x.clone() for x in (q, k, v)]
                t[which][0, at] = bad
                b = ops.decay_attention(*t, ld)
                assert torch.equal(a[:, :at], b[:, :at])
                assert not torch.isfinite(b[0, at]).all()
                if which:  # what enters the state stays in it
                    assert not torch.isfinite(b[0, -1]).all()


def test_spikes_fill_a_state_beyond_fp16(dev):
    """Spike counts pile up without a leak: the state passes fp16's largest value."""
    from catfuse_b200 import ops
    n = 3000
    q, k, v = _make((1, n), 2, 2, 32, 32, torch.float16, 9, "spikes")
    k, v = torch.ones_like(k) * 8, torch.ones_like(v) * 8
    q = q / 1024
    ld = torch.zeros(2, device=dev)
    s = torch.empty(1, 2, 32, 32, device=dev)
    out = ops.decay_attention(q, k, v, ld, s_out=s)
    assert float(s.max()) == 64.0 * n
    _check_sequences(q[0], k[0], v[0], ld, [(0, n)], out[0], None, s)


@pytest.mark.parametrize("size", [1e-4, 200.0])
def test_fp16_small_and_large_values(dev, size):
    """Values near fp16's ends: products of them leave its range on both sides."""
    from catfuse_b200 import ops
    q, k, v = _make((1, 300), 2, 2, 64, 64, torch.float16, 10)
    q, k = (q * size).half(), (k * size).half()
    v = (v * 1e-3 if size > 1 else v * 30).half()
    ld = torch.tensor([-0.01, -0.5], device=dev)
    s = torch.empty(1, 2, 64, 64, device=dev)
    scale = 1.0 / size ** 2 / 64
    out = ops.decay_attention(q, k, v, ld, s_out=s, scale=scale)
    _check_sequences(q[0], k[0], v[0], ld, [(0, 300)], out[0], None, s, scale=scale)


@pytest.mark.parametrize("dtype", HALF)
def test_strides(dev, dtype):
    """Slices of one fused projection, heads outside tokens, and a strided output."""
    from catfuse_b200 import ops
    g = torch.Generator().manual_seed(11)
    B, L, hq, hk, d = 2, 90, 4, 2, 64
    qkv = torch.randn(B, L, (hq + 2 * hk) * d + 24, generator=g).to(dtype).to(dev)
    q = qkv[..., :hq * d].unflatten(-1, (hq, d))
    k = qkv[..., hq * d:(hq + hk) * d].unflatten(-1, (hk, d))
    v = qkv[..., (hq + hk) * d:(hq + 2 * hk) * d].unflatten(-1, (hk, d))
    ld = _log_decay(hk, "-0.02").to(dev)
    want = ops.decay_attention(q.contiguous(), k.contiguous(), v.contiguous(), ld)
    wide = torch.zeros(B, L, hq, 2 * d, dtype=dtype, device=dev)
    got = ops.decay_attention(q, k, v, ld, out=wide[..., :d])
    assert torch.equal(got, want) and (wide[..., d:] == 0).all()
    # heads outside tokens (one sequence, so that the token axis has one stride)
    qh, kh, vh = (t[:1].transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))
    assert torch.equal(ops.decay_attention(qh, kh, vh, ld), want[:1])
    # a head starts on an odd element: rows are only aligned to their type
    odd = torch.zeros(B, L, hq + 2 * hk, d + 1, dtype=dtype, device=dev)
    odd[..., 1:] = torch.cat([q, k, v], 2)
    got = ops.decay_attention(odd[:, :, :hq, 1:], odd[:, :, hq:hq + hk, 1:], odd[:, :, hq + hk:, 1:], ld)
    assert _close_16(got, want)
    step = ops.decay_attention_step(odd[:, 0, :hq, 1:], odd[:, 0, hq:hq + hk, 1:], odd[:, 0, hq + hk:, 1:],
                                    ld, torch.zeros(B, hk, d, d, device=dev))
    assert _close_16(step, want[:, 0])


def _close_16(a, b):
    u = U[a.dtype]
    return bool(((a.double() - b.double()).norm() <= 2 * u * b.double().norm()))


@pytest.mark.parametrize("dtype", HALF)
def test_prompt_in_pieces_and_single_tokens(dev, dtype):
    from catfuse_b200 import ops
    q, k, v = _make((2, 150), 4, 2, 128, 64, dtype, 12)
    ld = _log_decay(2, "-0.05").to(dev)
    s = torch.zeros(2, 2, 128, 64, device=dev)
    parts = []
    for a, b in ((0, 1), (1, 66), (66, 140)):
        parts.append(ops.decay_attention(q[:, a:b].contiguous(), k[:, a:b].contiguous(),
                                         v[:, a:b].contiguous(), ld, s_in=s, s_out=s))
    for t in range(140, 150):
        parts.append(ops.decay_attention_step(q[:, t], k[:, t], v[:, t], ld, s)[:, None])
    got = torch.cat(parts, 1)
    for b in range(2):
        o, S, ao, aS = oracle.decay_attention(q[b], k[b], v[b], ld)
        _check_out(got[b], o, ao)
        _check_state(s[b], S, aS)


@pytest.mark.parametrize("case", [dict(S=1, L=5000, hq=2, hk=2, dk=128, dv=128),
                                  dict(S=3, L=2500, hq=4, hk=1, dk=64, dv=64),
                                  dict(S=1, L=9000, hq=1, hk=1, dk=64, dv=128)])
@pytest.mark.parametrize("dtype", HALF)
def test_long_prompts(dev, dtype, case):
    """Few heads and many tokens: the token axis is split over the GPU."""
    from catfuse_b200 import ops
    c = case
    q, k, v = _make((c["S"], c["L"]), c["hq"], c["hk"], c["dk"], c["dv"], dtype, 13)
    ld = _log_decay(c["hk"], "-0.001").to(dev)
    s = torch.randn(c["S"], c["hk"], c["dk"], c["dv"], generator=torch.Generator().manual_seed(4)).to(dev)
    s0 = s.clone()
    out = ops.decay_attention(q, k, v, ld, s_in=s, s_out=s)
    L = c["L"]
    _check_sequences(*(t.flatten(0, 1) for t in (q, k, v)), ld, [(i * L, i * L + L) for i in range(c["S"])],
                     out.flatten(0, 1), s0, s)
    s2 = s0.clone()
    assert torch.equal(out, ops.decay_attention(q, k, v, ld, s_in=s2, s_out=s2)) and torch.equal(s, s2)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("dims", [(64, 64), (128, 128), (128, 64), (64, 128)])
@pytest.mark.parametrize("heads", [(8, 8), (16, 8)])
def test_more_sequences_and_heads_than_fit_at_once(dev, dtype, dims, heads):
    """Every CTA walks several (sequence, head) pairs, long and short by turns."""
    from catfuse_b200 import ops
    (dk, dv), (hq, hk) = dims, heads
    g = torch.Generator().manual_seed(20)
    lens = torch.randint(0, 400, (60,), generator=g)
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)]).to(torch.int32)
    q, k, v = _make((int(cu[-1]),), hq, hk, dk, dv, dtype, 21)
    ld = _log_decay(hk).to(dev)
    s = torch.randn(60, hk, dk, dv, generator=g).to(dev)
    s0 = s.clone()
    out = ops.decay_attention(q, k, v, ld, s_in=s, s_out=s, cu_seqlens=cu.to(dev))
    b = cu.tolist()
    pick = [0, 1, 17, 36, 58, 59]  # the oracle is slow: every CTA's first and last pairs are among these
    _check_sequences(q, k, v, ld, [(b[i], b[i + 1]) for i in pick], out, s0[pick], s[pick])
    alone = torch.empty_like(s0)
    for i in range(60):  # all of them against calls of their own
        o = ops.decay_attention(q[b[i]:b[i + 1]][None], k[b[i]:b[i + 1]][None], v[b[i]:b[i + 1]][None], ld,
                                s_in=s0[i:i + 1], s_out=alone[i:i + 1])
        assert _close_16(out[b[i]:b[i + 1]], o[0])
    assert (s - alone).norm() <= 2.0 ** -18 * alone.norm()


def test_overlapping_boundaries_stay_in_bounds(dev):
    """Boundaries that do not ascend are the caller's error: outputs of the
    sequences concerned mean nothing, but nothing outside them is touched."""
    from catfuse_b200 import ops
    n = 3000
    q, k, v = _make((n + 64,), 1, 1, 64, 64, torch.float16, 23)
    ld = _log_decay(1, "-0.1").to(dev)
    cu = torch.tensor([0, n] * 20 + [0], dtype=torch.int32, device=dev)
    out = torch.full_like(v, 7.0)
    s = torch.full((41, 1, 64, 64), 5.0, device=dev)
    ops.decay_attention(q, k, v, ld, s_out=s[:40], cu_seqlens=cu, out=out)
    torch.cuda.synchronize()
    assert (out[n:] == 7).all() and (s[40] == 5).all()


def test_long_packed_prompts(dev):
    from catfuse_b200 import ops
    lens = [3000, 1, 0, 700, 64, 2111]
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    q, k, v = _make((int(cu[-1]),), 2, 1, 128, 128, torch.bfloat16, 14)
    ld = _log_decay(1, "-0.003").to(dev)
    s = torch.randn(6, 1, 128, 128, generator=torch.Generator().manual_seed(5)).to(dev)
    s0 = s.clone()
    out = ops.decay_attention(q, k, v, ld, s_in=s, s_out=s, cu_seqlens=cu.to(dev))
    b = cu.tolist()
    _check_sequences(q, k, v, ld, list(zip(b, b[1:])), out, s0, s)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("shape", [(1, 1, 1, 8, 8), (3, 6, 2, 32, 32), (5, 4, 4, 128, 128), (2, 7, 7, 40, 72),
                                   (70, 8, 1, 64, 128), (9, 12, 12, 128, 24)])
def test_step(dev, dtype, shape):
    from catfuse_b200 import ops
    B, hq, hk, dk, dv = shape
    q, k, v = _make((B,), hq, hk, dk, dv, dtype, sum(shape))
    ld = _log_decay(hk).to(dev)
    g = torch.Generator().manual_seed(6)
    pool = torch.randn(B + 3, hk, dk, dv, generator=g).to(dev)
    slots = torch.randperm(B + 3, generator=g)[:B].to(torch.int32)
    before = pool.clone()
    other = torch.full_like(pool, 3.0)
    out = ops.decay_attention_step(q, k, v, ld, pool, s_out=other, slots=slots.to(dev))
    assert torch.equal(pool, before)
    same = ops.decay_attention_step(q, k, v, ld, pool, slots=slots.to(dev))  # in place
    assert torch.equal(out, same)
    for i, r in enumerate(slots.tolist()):
        o, S, ao, aS = oracle.decay_attention(q[i:i + 1], k[i:i + 1], v[i:i + 1], ld, s_in=before[r])
        _check_out(out[i:i + 1], o, ao, f"row {i}")
        _check_state(pool[r], S, aS, f"state {i}")
        assert torch.equal(pool[r], other[r])
    for r in set(range(B + 3)) - set(slots.tolist()):
        assert torch.equal(pool[r], before[r]) and (other[r] == 3).all()


def test_step_padding_rows(dev):
    from catfuse_b200 import ops
    q, k, v = _make((4,), 4, 2, 64, 64, torch.float16, 15)
    ld = _log_decay(2, "-0.1").to(dev)
    pool = torch.randn(3, 2, 64, 64, device=dev)
    before = pool.clone()
    out = ops.decay_attention_step(q, k, v, ld, pool, slots=torch.tensor([-1, 2, 3, 2 ** 31 - 1],
                                                                         dtype=torch.int32, device=dev))
    assert (out[[0, 2, 3]] == 0).all() and not (out[1] == 0).all()
    assert torch.equal(pool[:2], before[:2]) and not torch.equal(pool[2], before[2])


def test_other_stream_and_graph(dev):
    from catfuse_b200 import ops
    q, k, v = _make((1, 700), 2, 2, 128, 128, torch.bfloat16, 16)
    ld = _log_decay(2, "-0.01").to(dev)
    s = torch.zeros(1, 2, 128, 128, device=dev)
    want = ops.decay_attention(q, k, v, ld, s_out=s)
    want_step = ops.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s.clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    s2 = torch.zeros_like(s)
    with torch.cuda.stream(side):
        got = ops.decay_attention(q, k, v, ld, s_out=s2)
        got_step = ops.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s2.clone())
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(s2, s) and torch.equal(got_step, want_step)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = ops.decay_attention(q, k, v, ld, s_out=s2)
    s2.zero_()
    held.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, want) and torch.equal(s2, s)


def test_offsets_beyond_32_bits(dev):
    from catfuse_b200 import ops
    n, row = 70, 2 ** 25  # tokens 2^25 elements apart: the last lies beyond 2^31
    buf = torch.zeros(n * row, dtype=torch.float16, device=dev).view(n, row)
    q, k, v = _make((n,), 1, 1, 64, 64, torch.float16, 17)
    views = []
    for i, t in enumerate((q, k, v)):
        buf[:, 64 * i:64 * i + 64] = t[:, 0]
        views.append(buf[:, 64 * i:64 * i + 64].unsqueeze(1))
    ld = _log_decay(1, "-0.05").to(dev)
    s = torch.zeros(1, 1, 64, 64, device=dev)
    out = ops.decay_attention(*views, ld, s_out=s, cu_seqlens=torch.tensor([0, n], dtype=torch.int32, device=dev))
    _check_sequences(q, k, v, ld, [(0, n)], out, None, s)
    del buf, views
    rows = 2 ** 31 // (128 * 128) + 5  # a pool of states beyond 2^31 elements
    pool = torch.empty(rows, 1, 128, 128, device=dev)
    pool[rows - 1].zero_()
    q, k, v = _make((1,), 1, 1, 128, 128, torch.float16, 18)
    slots = torch.tensor([rows - 1], dtype=torch.int32, device=dev)
    out = ops.decay_attention_step(q, k, v, ld, pool, slots=slots)
    cu = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    out2 = ops.decay_attention(q, k, v, ld, s_in=pool, s_out=pool, slots=slots, cu_seqlens=cu)
    o, S, ao, aS = oracle.decay_attention(*(torch.cat([t, t]) for t in (q, k, v)), ld)
    _check_out(out, o[:1], ao[:1])
    _check_out(out2, o[1:], ao[1:])
    _check_state(pool[rows - 1], S, aS)


def test_a_wait_that_runs_out_is_reported(dev):
    """One CTA's first load is left out: its waits give up within their limit, the
    host learns of it, and the next call is as ever."""
    from catfuse_b200 import _lib, ops
    q, k, v = _make((1, 200), 2, 2, 64, 64, torch.float16, 22)
    ld = _log_decay(2, "-0.1").to(dev)
    want = ops.decay_attention(q, k, v, ld)
    ops.check_device_error()
    ops.set_wait_limit(2000)
    try:
        _lib.call("cf_test_arm_stalled_load", 1)
        ops.decay_attention(q, k, v, ld)
        with pytest.raises(_lib.CatfuseNativeError) as e:
            ops.check_device_error()
        assert e.value.code == _lib.CF_ERR_DEVICE_TIMEOUT
    finally:
        _lib.call("cf_test_arm_stalled_load", 0)
        ops.set_wait_limit(0)
    assert torch.equal(ops.decay_attention(q, k, v, ld), want)
    ops.check_device_error()


def test_nothing_to_do(dev):
    from catfuse_b200 import ops
    z = torch.empty(0, 5, 2, 64, dtype=torch.float16, device=dev)
    ld = torch.zeros(2, device=dev)
    assert ops.decay_attention(z, z, z, ld).shape == z.shape
    e = torch.empty(3, 0, 2, 64, dtype=torch.float16, device=dev)
    s0, s1 = torch.randn(3, 2, 64, 64, device=dev), torch.empty(3, 2, 64, 64, device=dev)
    assert ops.decay_attention(e, e, e, ld, s_in=s0, s_out=s1).shape == e.shape
    assert torch.equal(s0, s1)
    ops.decay_attention(e, e, e, ld, s_out=s1)
    assert (s1 == 0).all()
    assert ops.decay_attention_step(z[:, 0], z[:, 0], z[:, 0], ld, s0).shape == (0, 2, 64)


def test_refusals(dev):
    from catfuse_b200 import ops
    from catfuse_b200._lib import CatfuseNativeError
    q, k, v = _make((2, 10), 4, 2, 64, 64, torch.float16, 19)
    ld = torch.zeros(2, device=dev)
    s = torch.zeros(2, 2, 64, 64, device=dev)
    ok = dict(s_in=s, s_out=s)
    with pytest.raises(TypeError):
        ops.decay_attention(q.float(), k.float(), v.float(), ld)
    with pytest.raises(TypeError):
        ops.decay_attention(q, k.bfloat16(), v, ld)
    with pytest.raises(ValueError):
        ops.decay_attention(q, k[:, :9], v, ld)
    with pytest.raises(ValueError):
        ops.decay_attention(q, k, v, torch.zeros(4, device=dev))
    with pytest.raises(CatfuseNativeError):  # 3 query heads on 2 states
        ops.decay_attention(q[:, :, :3].contiguous(), k, v, ld)
    with pytest.raises(CatfuseNativeError):
        ops.decay_attention(q[..., :60].contiguous(), k[..., :60].contiguous(), v, ld)
    big = torch.zeros(1, 1, 1, 136, dtype=torch.float16, device=dev)
    with pytest.raises(CatfuseNativeError):
        ops.decay_attention(big, big, big, ld[:1])
    with pytest.raises(ValueError):
        ops.decay_attention(q, k, v, ld, s_in=s[:, :1], s_out=s)
    with pytest.raises(TypeError):
        ops.decay_attention(q, k, v, ld, s_in=s.half())
    with pytest.raises(CatfuseNativeError):  # one state row for two sequences
        ops.decay_attention(q, k, v, ld, s_out=s[:1])
    with pytest.raises(ValueError):
        ops.decay_attention(q, k, v, ld, slots=torch.zeros(3, dtype=torch.int32, device=dev), **ok)
    with pytest.raises(TypeError):
        ops.decay_attention(q, k, v, ld, slots=torch.zeros(2, dtype=torch.int64, device=dev), **ok)
    with pytest.raises(TypeError):
        ops.decay_attention(q[0], k[0], v[0], ld, cu_seqlens=torch.zeros(2, dtype=torch.int64, device=dev))
    with pytest.raises(ValueError):  # two sequences whose tokens have no common stride
        ops.decay_attention(*(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)), ld)
    with pytest.raises(ValueError):
        ops.decay_attention(q[..., ::2], k[..., ::2], v, ld)
    with pytest.raises(CatfuseNativeError):
        ops.decay_attention(q.cpu(), k.cpu(), v.cpu(), ld)
    with pytest.raises(ValueError):
        ops.decay_attention_step(q, k, v, ld, s)
    with pytest.raises(CatfuseNativeError):
        ops.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s[:1])
    with pytest.raises(ValueError):
        ops.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s, s_out=torch.zeros(3, 2, 64, 64, device=dev))
