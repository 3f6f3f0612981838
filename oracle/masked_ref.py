"""Float64 definitions of the rotary positions, the query / key norms and the masked
attention, on the CPU, with the magnitudes that error bounds are made of."""
import math

import torch

F64 = torch.float64


def _pairs(Dh, P, interleaved):
    i = torch.arange(P)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + P)


def rotary(x, positions, freqs, sections, interleaved):
    """(y, size) of x [..., token, head, Dh]: size is |x1| + |x2| of an element's pair."""
    y = x.to(F64).clone()
    size = y.abs()
    P = sum(sections)
    if P:
        axis = torch.cat([torch.full((n,), a, dtype=torch.long) for a, n in enumerate(sections)])
        angle = (positions.to(F64)[..., axis] * freqs.to(F64))[..., None, :]
        a, b = _pairs(x.shape[-1], P, interleaved)
        x1, x2 = y[..., a].clone(), y[..., b].clone()
        y[..., a] = x1 * torch.cos(angle) - x2 * torch.sin(angle)
        y[..., b] = x2 * torch.cos(angle) + x1 * torch.sin(angle)
        size[..., a] = size[..., b] = x1.abs() + x2.abs()
    return y, size


def norm(x, gamma, eps):
    x = x.to(F64)
    n = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    return n if gamma is None else n * gamma.to(F64)


def visible(B, Sq, Sk, key_range=None, q_pos=None, causal=False):
    """(mask [B, Sq, Sk], p [B, Sq])"""
    p = torch.arange(Sk - Sq, Sk).expand(B, Sq) if q_pos is None else q_pos.long().expand(B, Sq)
    j = torch.arange(Sk)
    m = torch.ones(B, Sq, Sk, dtype=torch.bool)
    if key_range is not None:
        r = key_range.long().expand(B, Sq, 2)
        m &= (j >= r[..., :1]) & (j < r[..., 1:])
    if causal:
        m &= j <= p[..., None]
    return m, p


def attention(q, k, v, key_range=None, q_pos=None, causal=False, scale=None, cap=0.0, slopes=None, rel_bias=None):
    """dict of o [B, Sq, H, Dh], A = sum w |v| per element, err: the largest error of a
    visible key's score in fp32 arithmetic per row, in units of 2^-24 [B, Sq, H, 1]."""
    B, Sq, H, Dh = q.shape
    Sk, Hkv = k.shape[1:3]
    scale = Dh ** -0.5 if scale is None else scale
    m, p = visible(B, Sq, Sk, key_range, q_pos, causal)
    kk = k.to(F64).repeat_interleave(H // Hkv, 2).permute(0, 2, 3, 1)
    vv = v.to(F64).repeat_interleave(H // Hkv, 2).transpose(1, 2)
    qq = q.to(F64).transpose(1, 2)
    s = qq @ kk * scale
    # a product's sum of Dh terms in fp32, two units a term
    err = 2 * (Dh + 4) * (qq.abs() @ kk.abs()) * scale
    if cap:
        s = cap * torch.tanh(s / cap)
        err = err + 16 * cap
    d = torch.arange(Sk)[None, None] - p[:, :, None]
    if slopes is not None:
        b = -slopes.to(F64)[None, :, None, None] * d.abs()[:, None]
        s, err = s + b, err + 4 * b.abs()
    if rel_bias is not None:
        R = rel_bias.shape[1] // 2
        b = rel_bias.to(F64)[:, d.clamp(-R, R) + R].transpose(0, 1)
        s = s + b
        err = err + torch.where(torch.isinf(b), 0.0, b.abs())
    m = m[:, None] & (s != -math.inf)
    s = torch.where(m, s, torch.full((), -math.inf, dtype=F64))
    top = s.amax(-1, keepdim=True) if Sk else torch.zeros(B, H, Sq, 1, dtype=F64)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    w = torch.exp(s - top)
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total > 0, total, torch.ones_like(total))
    # 8 units of the largest score of the row: its scaling, the difference to the base, 2^x
    err = torch.where(m, err + 8 * s.abs(), 0.0).amax(-1, keepdim=True) + 8 * top.abs() if Sk else top
    return {"o": (w @ vv).transpose(1, 2), "A": (w @ vv.abs()).transpose(1, 2), "err": err.transpose(1, 2)}
