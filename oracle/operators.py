"""The attention operators and the distillation loss from their formulas in float64 (test infrastructure;
see oracle/__init__.py). Gradients are written out by hand, so that a test can hold them to differences.
"""
from __future__ import annotations

import torch

EPS32 = torch.finfo(torch.float32).eps


def rotation(rope: torch.Tensor, positions: torch.Tensor):
    """cos, sin [..., 1, D / 2] of the table's rows at positions [..., T]."""
    rows = rope.double()[positions.long()].unsqueeze(-2)
    return rows.chunk(2, -1)


def rotate(x, c, s):
    a, b = x.chunk(2, -1)
    return torch.cat([a * c + b * s, -a * s + b * c], -1)


def rotate_back(x, c, s):
    return rotate(x, c, -s)


def norm_rope(x, c, s, weight=None, order='rotate_norm', eps=EPS32):
    """x [B, T, H, D] -> y (float64)."""
    x = x.double()
    z = rotate(x, c, s) if order == 'rotate_norm' else x
    n = z / (z.square().mean(-1, keepdim=True) + eps).sqrt()
    y = n if weight is None else n * weight.double()
    return y if order == 'rotate_norm' else rotate(y, c, s)


def norm_rope_backward(dy, x, c, s, weight=None, order='rotate_norm', eps=EPS32):
    """(dx, dw, |dw|): the last sums the terms' absolute values, the scale of the sum's rounding."""
    x, dy = x.double(), dy.double()
    z = rotate(x, c, s) if order == 'rotate_norm' else x
    r = (z.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = z * r
    g = dy if order == 'rotate_norm' else rotate_back(dy, c, s)
    terms = (g * n).reshape(-1, x.shape[-1])
    h = g if weight is None else g * weight.double()
    dz = r * (h - n * (n * h).mean(-1, keepdim=True))
    dx = rotate_back(dz, c, s) if order == 'rotate_norm' else dz
    return dx, terms.sum(0), terms.abs().sum(0)


def visible(Tq, Tk, offset, window, sinks, length):
    """[Tq, Tk] bool: query row i (position offset + i) sees key j."""
    p, j = torch.arange(Tq)[:, None] + offset, torch.arange(Tk)[None]
    return (j <= p) & ((p - j <= window) | (j < sinks)) & (p < length)


def window_attention(q, k, v, window, sinks=0, lengths=None, offset=None, scale=None):
    """q [B, Tq, H, D], k, v [B, Tk, Hk, D] on the CPU -> out, lse [B, H, Tq], and sum p |v| (all float64)."""
    B, Tq, H, D = q.shape
    Tk, group = k.shape[1], H // k.shape[2]
    offset = Tk - Tq if offset is None else offset
    scale = D ** -0.5 if scale is None else scale
    out, mag = torch.zeros(B, Tq, H, D, dtype=torch.float64), torch.zeros(B, Tq, H, D, dtype=torch.float64)
    lse = torch.full((B, H, Tq), -torch.inf, dtype=torch.float64)
    for b in range(B):
        length = Tk if lengths is None else int(lengths[b])
        seen = visible(Tq, Tk, offset, window, sinks, length)
        rows = seen.any(1)
        for h in range(H):
            kk, vv = k[b, :, h // group].double(), v[b, :, h // group].double()
            kk, vv = kk.clone(), vv.clone()
            kk[length:], vv[length:] = 0, 0  # padding may hold anything
            s = (q[b, :, h].double() @ kk.T * scale).masked_fill(~seen, -torch.inf)[rows]
            pr = torch.softmax(s, 1)
            out[b, rows, h], mag[b, rows, h] = pr @ vv, pr @ vv.abs()
            lse[b, h, rows] = torch.logsumexp(s, 1)
    return out, lse, mag


def window_attention_backward(do, q, k, v, window, sinks=0, lengths=None, offset=None, scale=None):
    """dq, dk, dv, and for each the sum of its terms' absolute values as the kernel forms them (P, and dS with
    its two parts apart): the scale of the roundings of P and dS to 16 bits."""
    B, Tq, H, D = q.shape
    Tk, group = k.shape[1], H // k.shape[2]
    offset = Tk - Tq if offset is None else offset
    scale = D ** -0.5 if scale is None else scale
    grads = [torch.zeros(t.shape, dtype=torch.float64) for t in (q, k, v)]
    mags = [torch.zeros(t.shape, dtype=torch.float64) for t in (q, k, v)]
    for b in range(B):
        length = Tk if lengths is None else int(lengths[b])
        seen = visible(Tq, Tk, offset, window, sinks, length)
        rows = seen.any(1)
        if not rows.any():
            continue
        for h in range(H):
            kv = h // group
            qq, dd = q[b, rows, h].double(), do[b, rows, h].double()
            kk, vv = k[b, :, kv].double().clone(), v[b, :, kv].double().clone()
            kk[length:], vv[length:] = 0, 0
            p = torch.softmax((qq @ kk.T * scale).masked_fill(~seen[rows], -torch.inf), 1)
            dp = dd @ vv.T
            delta = (p * dp).sum(1, keepdim=True)
            ds = p * (dp - delta) * scale
            size = p * (dd.abs() @ vv.abs().T + (dd.abs() * (p @ vv.abs())).sum(1, keepdim=True)) * scale
            grads[0][b, rows, h] = ds @ kk
            mags[0][b, rows, h] = size @ kk.abs()
            grads[1][b, :, kv] += ds.T @ qq
            mags[1][b, :, kv] += size.T @ qq.abs()
            grads[2][b, :, kv] += p.T @ dd
            mags[2][b, :, kv] += p.T @ dd.abs()
    return (*grads, *mags)


def distill(logits, ids, teacher, temperature=1.0, softcap=0.0):
    """(loss [N], q, p, th'): q = softmax(s), p the teacher's mass of each column (float64), th' = ds/dz * temperature.
    The gradient of loss n is temperature (q - p) th'."""
    z, V = logits.double(), logits.shape[1]
    th = torch.tanh(z / softcap) if softcap else None
    s = (softcap * th if softcap else z) / temperature
    logq = torch.log_softmax(s, 1)
    ids = ids.long()
    have = (ids >= 0) & (ids < V)
    t = (teacher.double() / temperature).masked_fill(~have, -torch.inf)
    empty = (t == -torch.inf).all(1)
    logp = torch.log_softmax(torch.where(empty[:, None], torch.zeros_like(t), t), 1)
    p = torch.where(empty[:, None], 0.0, logp.exp())
    at = ids.clamp(0, V - 1)
    terms = torch.where(p > 0, p * (logp - logq.gather(1, at)), 0.0)
    mass = torch.zeros_like(z).scatter_add_(1, at, torch.where(have, p, 0.0))
    q = torch.where(empty[:, None], 0.0, logq.exp())
    slope = 1 - th.square() if softcap else torch.ones_like(z)
    return temperature ** 2 * terms.sum(1), q, mass, slope
