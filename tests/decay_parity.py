"""Decayed linear attention in 64 bits by chunks (the oracle's token-by-token
recurrence is too slow for long prompts), and the tolerances of its tests.

Per element, with u the unit roundoff of the 16-bit type and A the sum of the
absolute values of an element's terms: outputs u (|o| + A), since they are
rounded once on the way out and each term may have one factor rounded to 16 bits;
states 2^-18 A, since they are fp32 throughout."""
import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}
HALF = [torch.float16, torch.bfloat16]
CHUNK = 256


def chunked(q, k, v, log_decay, scale=None, s_in=None):
    """One sequence q [n, Hq, Dk], k [n, Hk, Dk], v [n, Hk, Dv] on any device ->
    (o [n, Hq, Dv], S [Hk, Dk, Dv], and the sums of absolute terms of both)."""
    f = torch.float64
    q, k, v = (t.detach().to(f).transpose(0, 1) for t in (q, k, v))  # [H, n, D]
    (hq, n, dk), (hk, _, dv) = q.shape, v.shape
    scale = dk ** -0.5 if scale is None else scale
    ld = log_decay.detach().to(f).view(hk, 1)
    S = q.new_zeros(hk, dk, dv) if s_in is None else s_in.detach().to(f)
    A = S.abs()

    def power(d):  # l^d, d >= 0; 0^0 = 1
        return torch.where(d == 0, torch.ones_like(ld * 1.0), torch.exp(ld * d))

    o, a = q.new_empty(hq, n, dv), q.new_empty(hq, n, dv)
    for t in range(0, n, CHUNK):
        qc, kc, vc = q[:, t:t + CHUNK].unflatten(0, (hk, -1)), k[:, t:t + CHUNK], v[:, t:t + CHUNK]
        m = kc.shape[1]
        i = torch.arange(m, device=q.device, dtype=f)
        gap = i[:, None] - i
        within = power(gap.clamp(min=0).flatten()).view(hk, m, m) * (gap >= 0)
        grow, keep = power(i + 1)[:, None, :, None], power(m - 1 - i)[..., None]
        for dst, x, y, z, s in ((o, qc, kc, vc, S), (a, qc.abs(), kc.abs(), vc.abs(), A)):
            w = (x @ y.transpose(1, 2)[:, None]) * within[:, None]
            dst[:, t:t + m] = ((w @ z[:, None] + grow * (x @ s[:, None])) * abs(scale)).flatten(0, 1)
        whole = power(torch.tensor([float(m)], device=q.device, dtype=f))[..., None]
        S = whole * S + (kc * keep).transpose(1, 2) @ vc
        A = whole * A + (kc * keep).abs().transpose(1, 2) @ vc.abs()
    if scale < 0:
        o = -o
    return o.transpose(0, 1), S, a.transpose(0, 1), A


def check_out(got, want, terms, what=""):
    err = (got.double() - want).abs()
    tol = U[got.dtype] * (want.abs() + terms) + TINY[got.dtype]
    assert torch.isfinite(err).all(), what
    assert (err <= tol).all(), f"{what}: {float((err / tol).max())} of the tolerance"


def check_state(got, want, terms, what=""):
    err = (got.double() - want).abs()
    tol = 2.0 ** -18 * terms + 1e-37
    assert torch.isfinite(err).all(), what
    assert (err <= tol).all(), f"{what}: {float((err / tol).max())} of the tolerance"
