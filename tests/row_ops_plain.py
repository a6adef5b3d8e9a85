"""The row operators of flyhigh_engine_b200.kernels from their definitions in 64 bits, with how far a kernel that rounds
where the header says may be from them.

A rounding to the element type is off by at most half a step, `e` = finfo.eps / 2 relative (f16 below its normal range:
2^-25 absolute); sums in 32 bits of n terms by at most n 2^-23 of the terms' magnitudes (a tensor core may truncate)."""
import math

import torch

SUBNORMAL = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def act64(kind, g):
    """act(g), act'(g) in 64 bits."""
    if kind in ("silu", "sigmoid"):
        s = 1 / (1 + torch.exp(-g))
        return (g * s, s * (1 + g * (1 - s))) if kind == "silu" else (s, s * (1 - s))
    if kind == "relu":
        return torch.clamp(g, min=0), (g > 0).double()
    if kind == "gelu":
        cdf = torch.erfc(-g / math.sqrt(2)) / 2
        return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (g + 0.044715 * g ** 3))
    return g * (1 + t) / 2, (1 + t) / 2 + g / 2 * (1 - t * t) * k * (1 + 3 * 0.044715 * g * g)


def _mm(a, b, ea, eb, n):
    """a @ b and its bound, for operands known to ea and eb (elementwise, or 0)."""
    v, mag = a @ b, a.abs() @ b.abs()
    e = mag * (n * 2.0 ** -23)
    if not isinstance(ea, float):
        e = e + ea @ b.abs()
    if not isinstance(eb, float):
        e = e + a.abs() @ eb
    return v, e


def ffn(x, wg, wu, wd, bg=None, bu=None, bd=None, act="silu", dy=None):
    """{name: (value, bound)} of the block, and with dy of its gradients; tensors as the kernel gets them."""
    t = x.dtype
    e, sub = half_step(t), SUBNORMAL[t]
    rnd = lambda v, err: (v, err + e * (v.abs() + err) + sub)
    has = (bg is not None, bu is not None, bd is not None)
    x, wg, wu, wd = (v.double() for v in (x, wg, wu, wd))
    f, c, o, m = wg.shape[0], x.shape[1], wd.shape[0], x.shape[0]
    bg, bu, bd = (torch.zeros(n, dtype=torch.float64, device=x.device) if b is None else b.double()
                  for b, n in ((bg, f), (bu, f), (bd, o)))
    g, eg = _mm(x, wg.t(), 0.0, 0.0, c + 1)
    u, eu = _mm(x, wu.t(), 0.0, 0.0, c + 1)
    g, u = g + bg, u + bu
    v, dv = act64(act, g)
    # |act'| <= 1.13 and |act''| <= 1 for all of them; the functions themselves to 2^-20 of 1 + |g|
    fn = 2.0 ** -20 * (1 + g.abs())
    ev = 1.13 * eg + fn
    a, ea = rnd(v * u, ev * u.abs() + v.abs() * eu + 1e-7 * (v * u).abs())
    y, ey = _mm(a, wd.t(), ea, 0.0, f + 1)
    r = {"y": rnd(y + bd, ey + 1e-7 * bd.abs())}
    if dy is None:
        return r
    dy = dy.double()
    da, eda = _mm(dy, wd, 0.0, 0.0, o)
    _, egr = rnd(g, eg)  # g and u as they were kept
    _, eur = rnd(u, eu)
    edv = egr + fn
    if act == "relu":  # its derivative steps at 0
        edv = fn + (g.abs() <= egr).double()
    dg, edg = rnd(da * u * dv, eda * (u * dv).abs() + (da * dv).abs() * eur + (da * u).abs() * edv + eda * eur + 1e-6 * (da * u * dv).abs())
    du, edu = rnd(da * v, eda * v.abs() + da.abs() * (1.13 * egr + fn) + 1e-6 * (da * v).abs())
    dx1, e1 = _mm(dg, wg, edg, 0.0, 2 * f)
    dx2, e2 = _mm(du, wu, edu, 0.0, 2 * f)
    r["x"] = rnd(dx1 + dx2, e1 + e2)
    r["w_gate"] = rnd(*_mm(dg.t(), x, edg.t(), 0.0, m))
    r["w_up"] = rnd(*_mm(du.t(), x, edu.t(), 0.0, m))
    r["w_down"] = rnd(*_mm(dy.t(), a, 0.0, ea, m))
    colsum = lambda d, ed: rnd(d.sum(0), ed.sum(0) + d.abs().sum(0) * (m * 2.0 ** -23))
    if has[0]:
        r["b_gate"] = colsum(dg, edg)
    if has[1]:
        r["b_up"] = colsum(du, edu)
    if has[2]:
        r["b_down"] = colsum(dy, torch.zeros_like(dy))
    return r


def ffn64(x, wg, wu, wd, bg, bu, bd, act):
    g, u = x @ wg.t(), x @ wu.t()
    if bg is not None:
        g, u = g + bg, u + bu
    y = (act64(act, g)[0] * u) @ wd.t()
    return y if bd is None else y + bd


def normed64(kind, v, eps):
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    return v if kind == "none" else v / torch.sqrt(v.square().mean(1, keepdim=True) + eps)


def affine64(n, w, b):
    n = n if w is None else n * w.double()
    return n if b is None else n + b.double()


def residual_norm64(x, f, gate, pre, post, eps, w_pre=None, b_pre=None, w_post=None, b_post=None, scale=None):
    """(y, h) in 64 bits; differentiable."""
    y = x
    if f is not None:
        p = affine64(normed64(post, f, eps), w_post, b_post)
        p = p if scale is None else p * scale.double()
        if gate is not None:
            p = p * gate.double().repeat_interleave(x.shape[0] // gate.shape[0], 0)
        y = x + p
    return y, None if pre == "none" else affine64(normed64(pre, y, eps), w_pre, b_pre)


def assert_within(name, got, value, bound):
    assert got.shape == value.shape, (name, got.shape, value.shape)
    off = (got.double() - value).abs()
    assert not torch.isnan(off).any(), name
    worst = (off - bound).max().item() if off.numel() else 0.0
    if worst > 0:
        i = int((off - bound).argmax())
        raise AssertionError(f"{name}: element {i} is {off.flatten()[i].item():.3g} off, its bound {bound.flatten()[i].item():.3g}")
