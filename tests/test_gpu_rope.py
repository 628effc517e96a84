"""Query/key norm with position rotation (cf_qk_norm_rope) against 64 bits.

Tolerance, per element: u |y| for the one rounding on the way out, and 2^-20 of
|a| + |b| of the element's pair for the fp32 norm, sine and cosine (each a few
units of 2^-24)."""
import pytest
import torch

import oracle

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
HALF = [torch.float16, torch.bfloat16]


def _check(got, x, pos, freq, **kw):
    y, bound = oracle.qk_norm_rope(x.flatten(0, -3), pos.reshape(-1, x.shape[:-2].numel()), freq, **kw)
    err = (got.flatten(0, -3).cpu().double() - y).abs()
    tol = U[got.dtype] * y.abs() + 2.0 ** -20 * bound + 2.0 ** -25
    assert torch.isfinite(err).all()
    assert (err <= tol).all(), float((err / tol).max())


def _inputs(lead, hq, hk, d, dtype, seed, dev):
    g = torch.Generator().manual_seed(seed)
    return [(2 * torch.randn(*lead, h, d, generator=g)).to(dtype).to(dev) for h in (hq, hk)]


def _freq(pairs, dev):
    return 10000.0 ** (-torch.arange(pairs, dtype=torch.float32, device=dev) / max(pairs, 1))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("pairing", ["half", "adjacent"])
@pytest.mark.parametrize("dims", [(2, 2), (8, 8), (8, 4), (10, 6), (24, 24), (32, 16), (64, 64), (80, 60),
                                  (96, 96), (128, 128), (128, 64), (160, 160), (256, 256), (250, 130), (64, 0)])
def test_dims(dev, dtype, pairing, dims):
    from catfuse_b200 import ops
    d, rot = dims
    q, k = _inputs((37,), 5, 2, d, dtype, d + rot, dev)
    pos = torch.randint(0, 4096, (37,), generator=torch.Generator().manual_seed(1)).to(dev, torch.int32)
    w = [1 + 0.2 * torch.randn(d, generator=torch.Generator().manual_seed(2 + i)).to(dev) for i in range(2)]
    freq = _freq(rot // 2, dev)
    for norm in (True, False):
        qo, ko = ops.qk_norm_rope(q, k, pos, freq, q_weight=w[0] if norm else None,
                                  k_weight=w[1] if norm else None, norm=norm, pairing=pairing)
        _check(qo, q, pos, freq, weight=w[0] if norm else None, norm=norm, pairing=pairing)
        _check(ko, k, pos, freq, weight=w[1] if norm else None, norm=norm, pairing=pairing)


@pytest.mark.parametrize("order", ["blocks", "cyclic"])
@pytest.mark.parametrize("sections", [(32,), (16, 16), (16, 8, 8), (2, 15, 15), (0, 30, 2), (8, 8, 8, 8)])
def test_axes(dev, order, sections):
    from catfuse_b200 import ops
    q, k = _inputs((3, 50), 4, 4, 64, torch.bfloat16, len(sections), dev)
    pos = torch.randint(-100, 1000, (len(sections), 3, 50), generator=torch.Generator().manual_seed(3)).to(dev)
    freq = _freq(32, dev)
    qo, ko = ops.qk_norm_rope(q, k, pos, freq, sections=sections, axis_order=order, eps=1e-5)
    for got, x in ((qo, q), (ko, k)):
        _check(got, x, pos, freq, sections=sections, axis_order=order, eps=1e-5)


@pytest.mark.parametrize("tokens", [0, 1, 2, 3, 7, 64, 1001])
@pytest.mark.parametrize("heads", [(1, 1), (12, 12), (40, 8), (7, 1), (200, 100)])
def test_tokens_and_heads(dev, tokens, heads):
    from catfuse_b200 import ops
    q, k = _inputs((tokens,), *heads, 32, torch.float16, tokens, dev)
    pos = torch.arange(tokens, device=dev, dtype=torch.int32)
    freq = _freq(16, dev)
    qo, ko = ops.qk_norm_rope(q, k, pos, freq)
    assert qo.shape == q.shape and ko.shape == k.shape
    if tokens:
        _check(qo, q, pos, freq)
        _check(ko, k, pos, freq)


def test_far_positions(dev):
    """Angles are reduced before they are rounded: positions up to a day of video
    frames, and beyond 32 bits."""
    from catfuse_b200 import ops
    q, k = _inputs((6,), 2, 2, 128, torch.float16, 4, dev)
    pos = torch.tensor([0, -1, 131071, 2 ** 24 + 1, 2 ** 31 - 1, 2 ** 33 + 5], device=dev)
    freq = _freq(64, dev)
    qo, ko = ops.qk_norm_rope(q, k, pos, freq)
    _check(qo, q, pos, freq)
    _check(ko, k, pos, freq)


def test_zero_and_non_finite_rows(dev):
    from catfuse_b200 import ops
    q, k = _inputs((8,), 2, 2, 64, torch.float16, 5, dev)
    q[3] = 0
    pos = torch.arange(8, device=dev, dtype=torch.int32)
    freq = _freq(32, dev)
    clean, _ = ops.qk_norm_rope(q, k, pos, freq)
    assert (clean[3] == 0).all()
    q2 = q.clone()
    q2[5, 1, 7] = float("inf")
    q2[6, 0, 0] = float("nan")
    got, _ = ops.qk_norm_rope(q2, k, pos, freq)
    assert torch.isnan(got[6, 0]).all() and not torch.isfinite(got[5, 1]).all()
    keep = torch.ones(8, 2, dtype=torch.bool)
    keep[5, 1] = keep[6, 0] = False
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("dtype", HALF)
def test_strides_and_in_place(dev, dtype):
    from catfuse_b200 import ops
    g = torch.Generator().manual_seed(6)
    B, L, hq, hk, d = 2, 33, 4, 2, 64
    qkv = torch.randn(B, L, (hq + 2 * hk) * d, generator=g).to(dtype).to(dev)
    q = qkv[..., :hq * d].unflatten(-1, (hq, d))
    k = qkv[..., hq * d:(hq + hk) * d].unflatten(-1, (hk, d))
    pos = torch.arange(L, device=dev).repeat(B, 1)
    freq = _freq(32, dev)
    qo, ko = ops.qk_norm_rope(q, k, pos, freq)
    _check(qo, q, pos, freq)
    _check(ko, k, pos, freq)
    # rows on odd elements
    odd = torch.zeros(B, L, hq + hk, d + 1, dtype=dtype, device=dev)
    odd[..., 1:] = torch.cat([q, k], 2)
    q1, k1 = ops.qk_norm_rope(odd[:, :, :hq, 1:], odd[:, :, hq:, 1:], pos, freq)
    _check(q1, q, pos, freq)
    _check(k1, k, pos, freq)
    v = qkv[..., (hq + hk) * d:].clone()
    ops.qk_norm_rope(q, k, pos, freq, q_out=q, k_out=k)
    assert torch.equal(q, qo) and torch.equal(k, ko) and torch.equal(qkv[..., (hq + hk) * d:], v)


def test_other_stream_and_graph(dev):
    from catfuse_b200 import ops
    q, k = _inputs((100,), 4, 4, 64, torch.float16, 7, dev)
    pos = torch.arange(100, device=dev, dtype=torch.int32)
    freq = _freq(32, dev)
    want = ops.qk_norm_rope(q, k, pos, freq)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = ops.qk_norm_rope(q, k, pos, freq)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals(dev):
    from catfuse_b200 import ops
    from catfuse_b200._lib import CatfuseNativeError
    q, k = _inputs((9,), 4, 2, 64, torch.float16, 8, dev)
    pos = torch.arange(9, device=dev)
    freq = _freq(32, dev)
    with pytest.raises(TypeError):
        ops.qk_norm_rope(q.float(), k.float(), pos, freq)
    with pytest.raises(TypeError):
        ops.qk_norm_rope(q, k.bfloat16(), pos, freq)
    with pytest.raises(TypeError):
        ops.qk_norm_rope(q, k, pos.float(), freq)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, k, pos[:8], freq)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, k, pos, freq, sections=(16, 16))
    with pytest.raises(CatfuseNativeError):
        ops.qk_norm_rope(q, k, pos, freq, sections=(16,))
    with pytest.raises(CatfuseNativeError):
        ops.qk_norm_rope(q, k, torch.stack([pos] * 5), freq, sections=(8, 8, 8, 4, 4))
    with pytest.raises(CatfuseNativeError):
        ops.qk_norm_rope(q, k, pos, _freq(33, dev))
    with pytest.raises(CatfuseNativeError):
        ops.qk_norm_rope(q[..., :63], k[..., :63], pos, _freq(16, dev))
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, k, pos, freq, pairing="thirds")
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, k, pos, freq, axis_order="random")
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, k, pos, freq, q_weight=torch.ones(32, device=dev))
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, k, pos, freq, q_out=torch.empty_like(k))
    with pytest.raises(CatfuseNativeError):
        ops.qk_norm_rope(q.cpu(), k.cpu(), pos, freq)
