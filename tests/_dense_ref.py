"""Plain 64-bit forms of the orthogonalised updates and of the 8-bit products,
on the CPU or the GPU, for the tests."""
from __future__ import annotations

import torch

COEF = (3.4445, -4.7750, 2.0315)


def orthogonalise(u, steps=5, coef=COEF, eps=1e-7):
    """newton_schulz in 64 bits; `coef` one triple or one a step."""
    x = u.double()
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    flip = x.shape[-2] > x.shape[-1]
    x = x.mT if flip else x
    for i in range(steps):
        a, b, c = coef[i] if isinstance(coef[0], (tuple, list)) else coef
        s = x @ x.mT
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.mT if flip else x


def muon(p, g, m, lr, momentum=0.95, nesterov=True, weight_decay=0.0, groups=1, match_rms=False):
    """(parameter, momentum) after a step, in 64 bits."""
    p, g, m = p.double(), g.double(), m.double()
    m = momentum * m + (1 - momentum) * g
    u = (1 - momentum) * g + momentum * m if nesterov else m
    rows, cols = p.shape[0] // groups, p.numel() // p.shape[0]
    o = orthogonalise(u.reshape(groups, rows, cols)).reshape(p.shape)
    s = 0.2 * max(rows, cols) ** 0.5 if match_rms else max(1.0, rows / cols) ** 0.5
    return (1 - lr * weight_decay) * p - lr * s * o, m


def codes(x):
    """(codes, scale) of the rows, in 64 bits."""
    x = x.double()
    scale = x.abs().amax(-1) / 127
    q = torch.round(x / scale.clamp(min=1e-300)[..., None])
    return torch.where(scale[..., None] > 0, q, torch.zeros_like(q)), scale


def columns(x, off, mask, kh, kw, stride, pad, dil):
    """Sampled columns (N, C, kh * kw, Ho * Wo) in 64 bits: corners outside the
    image count zero."""
    n, c, h, w = x.shape
    ho, wo = off.shape[2:]
    dg = off.shape[1] // (2 * kh * kw)
    o = off.double().reshape(n, dg, kh * kw, 2, ho * wo)
    out = torch.zeros(n, dg, c // dg, kh * kw, ho * wo, dtype=torch.float64, device=x.device)
    img = x.double().reshape(n, dg, c // dg, h * w)
    p = torch.arange(ho * wo, device=x.device)
    for t in range(kh * kw):
        ys = (p // wo) * stride[0] - pad[0] + (t // kw) * dil[0] + o[:, :, t, 0]
        xs = (p % wo) * stride[1] - pad[1] + (t % kw) * dil[1] + o[:, :, t, 1]
        y0, x0 = ys.floor(), xs.floor()
        for dy in (0, 1):
            for dx in (0, 1):
                i, j = y0 + dy, x0 + dx
                wt = (1 - (ys - i).abs()) * (1 - (xs - j).abs())
                inside = (i >= 0) & (i < h) & (j >= 0) & (j < w)
                at = (i.clamp(0, h - 1) * w + j.clamp(0, w - 1)).long()
                v = torch.gather(img, 3, at[:, :, None].expand(-1, -1, c // dg, -1))
                out[:, :, :, t] += torch.where(inside, wt, torch.zeros_like(wt))[:, :, None] * v
        if mask is not None:
            out[:, :, :, t] *= mask.double().reshape(n, dg, 1, kh * kw, ho * wo)[:, :, :, t]
    return out.reshape(n, c, kh * kw, ho * wo)


def deform_int8(x, off, wq, ws, bias, mask, stride, pad, dil):
    """deform_conv2d_int8 in 64 bits."""
    o, cg, kh, kw = wq.shape
    n, groups = x.shape[0], x.shape[1] // cg
    col = columns(x, off, mask, kh, kw, stride, pad, dil)
    col = col.reshape(n, groups, cg * kh * kw, -1).mT
    q, scale = codes(col)
    w = wq.contiguous().double().reshape(1, groups, o // groups, -1)
    y = (w @ q.mT) * scale[:, :, None] * ws.double().reshape(1, groups, -1, 1)
    y = y.reshape(n, o, *off.shape[2:])
    return y if bias is None else y + bias.double()[:, None, None]


def rel(got, want):
    """|got - want| / |want| in the 2-norm."""
    got, want = got.double(), want.double()
    n = want.norm()
    return float((got - want).norm() / (n if n > 0 else 1.0))
