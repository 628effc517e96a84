"""Decayed linear attention on the host: the oracle's recurrence against the
closed form, and the C entry points' refusals (no device is touched)."""
import ctypes

import pytest
import torch

import oracle


def test_recurrence_equals_closed_form():
    g = torch.Generator().manual_seed(0)
    n, hq, hk, dk, dv = 40, 4, 2, 8, 16
    q, k, v = (torch.randn(n, h, d, generator=g) for h, d in ((hq, dk), (hk, dk), (hk, dv)))
    s0 = torch.randn(hk, dk, dv, generator=g)
    ld = torch.tensor([-0.1, -1.5])
    o, S, a, A = oracle.decay_attention(q, k, v, ld, 0.5, s0)
    i = torch.arange(n, dtype=torch.float64)
    for h in range(hq):
        x = h // 2
        l = ld[x].double()
        w = torch.where(i[:, None] >= i, torch.exp(l * (i[:, None] - i)), 0.0)
        want = ((q[:, h].double() @ k[:, x].double().T) * w) @ v[:, x].double()
        want += torch.exp(l * (i + 1))[:, None] * (q[:, h].double() @ s0[x].double())
        assert torch.allclose(o[:, h], 0.5 * want, rtol=1e-12, atol=1e-12)
    assert (a >= o.abs() - 1e-12).all() and (A >= S.abs() - 1e-12).all()


def test_rotation_keeps_products_of_equal_distance():
    """q_m . k_n of rotated rows depends on m - n alone."""
    g = torch.Generator().manual_seed(1)
    q, k = torch.randn(1, 1, 16, generator=g), torch.randn(1, 1, 16, generator=g)
    freq = 10000.0 ** (-torch.arange(8) / 8.0)
    for pairing in ("half", "adjacent"):
        def dot(m, n):
            a, _ = oracle.qk_norm_rope(q, torch.tensor([[m]]), freq, norm=False, pairing=pairing)
            b, _ = oracle.qk_norm_rope(k, torch.tensor([[n]]), freq, norm=False, pairing=pairing)
            return float((a * b).sum())
        assert abs(dot(7, 3) - dot(104, 100)) < 1e-9


def test_axis_orders():
    assert oracle.axis_of_pair((2, 1, 1), "blocks") == [0, 0, 1, 2]
    assert oracle.axis_of_pair((3, 1, 2), "cyclic") == [0, 1, 2, 0, 2, 0]


def _strides(*s):
    return [x for pair in s for x in pair]


def test_entry_points_refuse_before_any_device():
    from catfuse_b200 import _lib
    lib = _lib.load()
    I = _lib.CF_ERR_INVALID_ARG
    st = _strides((64, 64)) * 4

    def step(fmt=1, hq=2, hk=2, dk=64, dv=64, q=16, s=16, rows=1, B=1):
        return lib.cf_decay_attention_step(q, 16, 16, 16, fmt, 16, s, s, None, rows, B, hq, hk, dk, dv,
                                           *st, 1.0, None)
    assert step(q=None) == I and step(fmt=0) == I and step(hq=3) == I and step(rows=0) == I
    assert step(dk=60) == _lib.CF_ERR_UNSUPPORTED and step(dv=136) == _lib.CF_ERR_UNSUPPORTED
    assert step(s=8) == _lib.CF_ERR_UNSUPPORTED and step(B=0) == _lib.CF_OK
    assert "" != _lib.last_error()

    def prompt(fmt=1, S=1, L=4, N=4, hq=2, hk=2, dk=64, q=16, rows=1, s=16):
        return lib.cf_decay_attention(q, 16, 16, 16, fmt, 16, s, s, None, rows, None, S, L, N, hq, hk, dk, 64,
                                      *st, 1.0, None, 0, None)
    assert prompt(q=None) == I and prompt(fmt=2) == I and prompt(hq=3) == I and prompt(N=5) == I
    assert prompt(rows=0) == I and prompt(dk=12) == _lib.CF_ERR_UNSUPPORTED and prompt(S=0, N=0) == _lib.CF_OK
    assert lib.cf_decay_attention_workspace(-1, 1, 1, 1, 64, 64, 0) < 0
    assert lib.cf_decay_attention_workspace(1, 64, 1, 1, 64, 64, 0) == 0

    def rope(D=64, rot=64, sec=(32,), pos=32, order=0, pairing=0, q=16, fmt=1, N=1):
        return lib.cf_qk_norm_rope(q, 16, 16, 16, fmt, N, 2, 2, D, *st, 16, pos, N, 16, rot,
                                   (ctypes.c_int32 * len(sec))(*sec), len(sec), order, pairing, None, None,
                                   1, 1e-6, None)
    assert rope(q=None) == I and rope(rot=66, sec=(33,)) == I and rope(sec=(31,)) == I
    assert rope(sec=(40, -8)) == I and rope(pos=16) == I and rope(order=2) == I and rope(pairing=5) == I
    assert rope(fmt=0) == I and rope(D=63, rot=62, sec=(31,)) == _lib.CF_ERR_UNSUPPORTED
    assert rope(D=258, rot=64) == _lib.CF_ERR_UNSUPPORTED
    assert rope(sec=(8, 8, 8, 4, 4)) == _lib.CF_ERR_UNSUPPORTED and rope(N=0) == _lib.CF_OK


def test_wrappers_need_cuda_tensors():
    from catfuse_b200 import ops
    from catfuse_b200._lib import CatfuseNativeError
    x = torch.zeros(1, 2, 1, 64, dtype=torch.float16)
    with pytest.raises(CatfuseNativeError):
        ops.decay_attention(x, x, x, torch.zeros(1))
    with pytest.raises(CatfuseNativeError):
        ops.decay_attention_step(x[0], x[0], x[0], torch.zeros(1), torch.zeros(2, 1, 64, 64))
    with pytest.raises(CatfuseNativeError):
        ops.qk_norm_rope(x, x, torch.zeros(1, 2, dtype=torch.int32), torch.ones(32))
