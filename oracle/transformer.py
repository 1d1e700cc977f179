"""64-bit torch restatements of the operators around attention (pyasc_b200/attention.py): rotary positions, per-head RMS
norm, attention to another sequence, and their gradients written out from the formulas."""
import math

import torch


def turns(positions, frequencies, scale):
    """cos and sin of [B or 1, S, 1, r / 2], in 64 bits, times ``scale``.  The angle is the exact product: what its
    rounding to 64 bits leaves out (Dekker's product of split factors) turns the rounded angle a little further."""
    p = (positions if positions.dim() == 2 else positions[None]).double()[:, :, None, None]
    f = frequencies.double()
    angle = p * f

    def split(x):
        t = x * 134217729.0
        high = t - (t - x)
        return high, x - high

    (ph, pl), (fh, fl) = split(p), split(f)
    rest = ((ph * fh - angle) + ph * fl + pl * fh) + pl * fl
    c, s = angle.cos(), angle.sin()
    return (c - s * rest) * scale, (s + c * rest) * scale


def rotate(x, cos, sin, interleaved):
    r = 2 * cos.shape[-1]
    y = x.clone()
    lo, hi = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    y[..., lo] = x[..., lo] * cos - x[..., hi] * sin
    y[..., hi] = x[..., hi] * cos + x[..., lo] * sin
    return y


def partner_sum(x, r, interleaved):
    """|lo| + |hi| of the pair every element belongs to, |x| of the others: what an element's rounding errors scale with."""
    one = torch.ones(r // 2, dtype=x.dtype, device=x.device)
    return rotate(x.abs(), one, -one, interleaved).abs().maximum(rotate(x.abs(), one, one, interleaved).abs())


def norm(x, gamma, eps):
    x = x.double()
    n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return n if gamma is None else n * gamma.double()


def norm_rotary(x, gamma, positions, frequencies, eps, scale, interleaved, normed=True):
    cos, sin = turns(positions, frequencies, scale)
    return rotate(norm(x, gamma, eps) if normed else x.double(), cos, sin, interleaved)


def norm_rotary_backward(dy, x, gamma, positions, frequencies, eps, scale, interleaved):
    """dx, dgamma, and the sums of magnitudes that bound the rounding errors of both."""
    x, dy = x.double(), dy.double()
    cos, sin = turns(positions, frequencies, scale)
    dn = rotate(dy, cos, -sin, interleaved)
    rstd = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    g = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if gamma is None else gamma.double()
    t = dn * g
    dx = rstd * t - x * rstd**3 * (x * t).mean(-1, keepdim=True)
    dn_size = partner_sum(dy, 2 * cos.shape[-1], interleaved) * scale
    dx_size = rstd * dn_size * g.abs() + x.abs() * rstd**3 * (x.abs() * dn_size * g.abs()).mean(-1, keepdim=True)
    return dx, (x * rstd * dn).sum((0, 1, 2)), dx_size, (x * rstd * dn_size).abs().sum((0, 1, 2))


def _scores(q, k, lengths, scale):
    """[B, H, S, T] scores of grouped heads, -inf where a key is not there."""
    group = q.shape[2] // k.shape[2]
    s = torch.einsum("bshd,bthd->bhst", q.double(), k.double().repeat_interleave(group, 2)) * scale
    if lengths is None:
        return s
    here = torch.arange(k.shape[1], device=s.device)[None] < lengths.to(s.device)[:, None]
    return torch.where(here[:, None, None, :], s, -math.inf)


def _clean(x, lengths):
    """x with zeros in the places of keys that are not there (which may hold anything)."""
    x = x.double()
    if lengths is None:
        return x
    here = torch.arange(x.shape[1], device=x.device)[None] < lengths.to(x.device)[:, None]
    return torch.where(here[:, :, None, None], x, 0.0)


def cross_attention(q, k, v, lengths=None, scale=None):
    """out [B, S, H, D], lse [B, H, S]; a query without keys: 0 and -inf."""
    scale = q.shape[-1]**-0.5 if scale is None else scale
    s = _scores(q, _clean(k, lengths), lengths, scale)
    lse = torch.logsumexp(s, -1) if s.shape[-1] else torch.full(s.shape[:3], -math.inf, dtype=s.dtype, device=s.device)
    p = torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[..., None])
    group = q.shape[2] // k.shape[2]
    return torch.einsum("bhst,bthd->bshd", p, _clean(v, lengths).repeat_interleave(group, 2)), lse


def cross_attention_backward(do, q, k, v, lengths=None, scale=None):
    """dq, dk, dv of :func:`cross_attention`'s out, in 64 bits."""
    scale = q.shape[-1]**-0.5 if scale is None else scale
    group = q.shape[2] // k.shape[2]
    kc, vc = _clean(k, lengths), _clean(v, lengths)
    out, lse = cross_attention(q, k, v, lengths, scale)
    s = _scores(q, kc, lengths, scale)
    p = torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[..., None])
    do = do.double()
    dp = torch.einsum("bshd,bthd->bhst", do, vc.repeat_interleave(group, 2))
    ds = p * (dp - (do * out).sum(-1).transpose(1, 2)[..., None]) * scale

    def grouped(x):
        return x.unflatten(2, (k.shape[2], group)).sum(3)

    return (torch.einsum("bhst,bthd->bshd", ds, kc.repeat_interleave(group, 2)),
            grouped(torch.einsum("bhst,bshd->bthd", ds, q.double())),
            grouped(torch.einsum("bhst,bshd->bthd", p, do)))


def cross_attention_backward_bounds(do, q, k, v, lengths, scale, step, least):
    """How far dq, dk, dv may be off when P, dS, out and the results are rounded to a type with half a step of ``step``
    (and ``least`` below its smallest normal), and scores, exponentials and sums are off by 2^-12 of their magnitudes:
    dS is off by step |dS| + p (2^-12 (|dO| |V| + |dO| |P||V|) + 2 step |dO| |P||V|) + least, and dq, dk, dv by the sums
    of that (of step p + 2^-12 p for dv) against |k|, |q|, |dO|, plus their own rounding."""
    group = q.shape[2] // k.shape[2]
    kc, vc = _clean(k, lengths), _clean(v, lengths)
    ka, va, da = kc.abs().repeat_interleave(group, 2), vc.abs().repeat_interleave(group, 2), do.double().abs()
    out, lse = cross_attention(q, k, v, lengths, scale)
    p = torch.exp(_scores(q, kc, lengths, scale) - torch.where(lse == -math.inf, 0.0, lse)[..., None])
    size = torch.einsum("bhst,bthd->bshd", p, va)
    along = (da * size).sum(-1).transpose(1, 2)[..., None]
    dp = torch.einsum("bshd,bthd->bhst", do.double(), vc.repeat_interleave(group, 2))
    ds = p * (dp - (do.double() * out).sum(-1).transpose(1, 2)[..., None])
    off = step * ds.abs() + p * (2.0**-12 * (torch.einsum("bshd,bthd->bhst", da, va) + along) + 2 * step * along) + least

    def grouped(x):
        return x.unflatten(2, (k.shape[2], group)).sum(3)

    dq, dk, dv = cross_attention_backward(do, q, k, v, lengths, scale)
    return (torch.einsum("bhst,bthd->bshd", off, ka) * scale + step * dq.abs() + least,
            grouped(torch.einsum("bhst,bshd->bthd", off, q.double().abs())) * scale + step * dk.abs() + least,
            grouped(torch.einsum("bhst,bshd->bthd", (step + 2.0**-12) * p + least, da)) + step * dv.abs() + least)
