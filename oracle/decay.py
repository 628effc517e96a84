"""Decayed linear attention and the query/key norm with position rotation, in 64
bits from their definitions — test infrastructure only (checker for the CUDA
path, never shipped or measured)."""
from __future__ import annotations

import torch


def decay_attention(q, k, v, log_decay, scale=None, s_in=None):
    """One sequence q [n, Hq, Dk], k [n, Hk, Dk], v [n, Hk, Dv], token by token:
    ``S = l S + k^T v``, ``o = scale q S`` -> (o [n, Hq, Dv], S [Hk, Dk, Dv], and
    the same two with every term's absolute value, which bound rounding errors)."""
    f = torch.float64
    q, k, v = (t.detach().cpu().to(f) for t in (q, k, v))
    n, Hq, Dk = q.shape
    Hk, Dv = v.shape[1:]
    scale = Dk ** -0.5 if scale is None else scale
    lam = torch.exp(log_decay.detach().cpu().to(f)).view(Hk, 1, 1)
    S = torch.zeros(Hk, Dk, Dv, dtype=f) if s_in is None else s_in.detach().cpu().to(f).clone()
    A = S.abs()
    o = torch.empty(n, Hq, Dv, dtype=f)
    a = torch.empty(n, Hq, Dv, dtype=f)
    for t in range(n):
        kv = k[t, :, :, None] * v[t, :, None, :]
        S = torch.where(lam == 0, kv, lam * S + kv)  # 0 forgets, whatever the state holds
        A = torch.where(lam == 0, kv.abs(), lam * A + kv.abs())
        qt = q[t].view(Hk, Hq // Hk, Dk)
        o[t] = (qt @ S).reshape(Hq, Dv) * scale
        a[t] = (qt.abs() @ A).reshape(Hq, Dv) * abs(scale)
    return o, S, a, A


def axis_of_pair(sections, order):
    """Position axis of each rotated pair."""
    if order == "blocks":
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, got, a = list(sections), [], 0
    while len(got) < sum(sections):
        if left[a]:
            left[a] -= 1
            got.append(a)
        a = (a + 1) % len(left)
    return got


def qk_norm_rope(x, positions, inv_freq, weight=None, norm=True, eps=1e-6, sections=None,
                 axis_order="blocks", pairing="half"):
    """x [N, H, D], positions [axes, N] -> (y [N, H, D], bound [N, H, D]): bound is
    |a| + |b| of the pair behind each element (|x| where nothing turns)."""
    f = torch.float64
    y = x.detach().cpu().to(f)
    D = y.shape[-1]
    if norm:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
        if weight is not None:
            y = y * weight.detach().cpu().to(f)
    freq = inv_freq.detach().cpu().to(f)
    pairs = freq.numel()
    axis = axis_of_pair(sections or (pairs,), axis_order)
    pos = positions.detach().cpu().to(f)
    out, bound = y.clone(), y.abs()
    for p in range(pairs):
        i, j = (p, p + pairs) if pairing == "half" else (2 * p, 2 * p + 1)
        t = (pos[axis[p]] * freq[p])[:, None]
        a, b = y[..., i], y[..., j]
        out[..., i] = a * torch.cos(t) - b * torch.sin(t)
        out[..., j] = b * torch.cos(t) + a * torch.sin(t)
        bound[..., i] = bound[..., j] = a.abs() + b.abs()
    assert 2 * pairs <= D
    return out, bound
