"""8-bit rows, the norms that end in them and the 8-bit linear, in float64 on
the CPU (tests only; the reference has no 8-bit path).

``rows`` returns the quotients before their rounding too, so that a test can
tell a wrong integer from one whose quotient lies within a rounding error of a
half.
"""
import torch


def rows(v):
    """Quotients 127 v / max|v| (unrounded), their nearest integers (halves to
    even) and max|v| / 127 of each row of float64 v."""
    top = v.abs().amax(1, keepdim=True)
    t = torch.where(top > 0, v * 127.0 / torch.where(top > 0, top, torch.ones_like(top)), torch.zeros_like(v))
    return t, torch.round(t), top[:, 0] / 127.0


def rms_norm(h, gamma, eps):
    n = h / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    return n if gamma is None else n * gamma


def layer_norm(h, gamma, beta, eps):
    d = h - h.mean(1, keepdim=True)
    n = d / torch.sqrt((d * d).mean(1, keepdim=True) + eps)
    n = n if gamma is None else n * gamma
    return n if beta is None else n + beta


def linear(xq, sx, wq, sw, bias=None, residual=None, act="none", beta=1.0):
    """float64 result and, per output, the magnitude that fp32 rounding errors
    scale with."""
    z = (xq.double() @ wq.double().t()) * sx.double()[:, None] * sw.double()
    mag = z.abs()
    if bias is not None:
        z = z + bias.double()
        mag = mag + bias.double().abs()
    if act == "silu":
        y = z * torch.sigmoid(z)
    elif act == "gelu":
        y = z * torch.special.ndtr(z)
    elif act == "geglu":
        v, g = z.view(z.shape[0], -1, 2, 4).unbind(2)
        mv, mg = mag.view(z.shape[0], -1, 2, 4).unbind(2)
        phi = g * torch.special.ndtr(g)
        y = (v * phi).reshape(z.shape[0], -1)
        mag = (mv * phi.abs() + 2.0 * v.abs() * mg).reshape(z.shape[0], -1)
    else:
        y = z
    if residual is not None:
        y = y + beta * residual.double()
        mag = mag + (beta * residual.double()).abs()
    return y, mag
