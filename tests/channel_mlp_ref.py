"""Plain 64-bit forms of the channel-MLP operators and the error bounds their kernels are held to.

u(t) = torch.finfo(t).eps / 2 is the largest relative error of one rounding to type t; U = u(float32).  A sum of n terms in fp32, in any
order, is off by at most n U sum|term| (to first order); every bound below counts the roundings a kernel makes on the way, with the
number of terms of its longest chain, and is doubled once for what first-order counting leaves out."""
import math

import torch

U = torch.finfo(torch.float32).eps / 2


def u(t):
    return torch.finfo(t).eps / 2


def rows_of(t):
    """[rows, C] of a tensor whose channels are dim 1 (4-D) or the last dim."""
    return t.permute(0, 2, 3, 1).reshape(-1, t.shape[1]) if t.dim() == 4 else t.reshape(-1, t.shape[-1])


# -- channel_norm ------------------------------------------------------------------------------
def norm_ref(x, w, b, eps, dy):
    """{name: (value, bound)} in fp64 for rows x, dy; the caller adds the output rounding."""
    x, w, dy = x.double(), w.double(), dy.double()
    C, R = x.shape[1], x.shape[0]
    m = x.mean(1, keepdim=True)
    xc = x - m
    rs = 1 / torch.sqrt((xc * xc).mean(1, keepdim=True) + eps)
    xh = xc * rs
    y = xh * w + (b.double() if b is not None else 0)
    g = dy * w
    dx = rs * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    # chains: a thread adds at most ceil(C / 64) + 16 terms, a wave 6 more steps, a block 16 more
    n = C / 64 + 48
    # the mean is off by n U mean|x|; x - m inherits that, a rounding of its own, and rs a relative n U (squares) / 2 + the shift
    dm = n * U * x.abs().mean(1, keepdim=True) + U * m.abs()
    dxh = rs * dm + (n + 8) * U * xh.abs() + xh.abs() * (rs * dm) ** 2
    gm, gx = g.abs().mean(1, keepdim=True), (g * xh).abs().mean(1, keepdim=True)
    ddx = rs * ((n + 16) * U * (g.abs() + gm + xh.abs() * gx) + dxh * gx + xh.abs() * (g.abs() * dxh).mean(1, keepdim=True)) + \
        (n + 8) * U * dx.abs()
    # weight gradients: rows in strips, the strips in turn
    k = R / 64 + 1100
    dw, db = (dy * xh).sum(0), dy.sum(0)
    out = {"y": (y, 2 * (dxh * w.abs() + 4 * U * (y.abs() + (xh * w).abs()))), "dx": (dx, 2 * ddx),
           "dw": (dw, 2 * ((dy.abs() * dxh).sum(0) + min(k, R + 8) * U * (dy * xh).abs().sum(0))),
           "db": (db, 2 * min(k, R + 8) * U * dy.abs().sum(0))}
    return out


# -- dropout -----------------------------------------------------------------------------------
def keep_mask(n, p, seed, step, first=0):
    """numpy restatement of the draw: Philox4x32-10 (Salmon et al., 2011), 16 bits an element; n elements from `first` (a multiple of 8)."""
    import numpy as np
    b = np.arange((n + 7) // 8, dtype=np.uint64) + np.uint64(first // 8)
    m32 = np.uint64(0xffffffff)
    seed, step = np.uint64(seed & (2 ** 64 - 1)), np.uint64(step & (2 ** 64 - 1))
    c = [b & m32, b >> np.uint64(32), np.full_like(b, step & m32), np.full_like(b, step >> np.uint64(32))]
    k0, k1 = int(seed & m32), int(seed >> np.uint64(32))
    for r in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        a0, a1 = np.uint64((k0 + r * 0x9E3779B9) & 0xffffffff), np.uint64((k1 + r * 0xBB67AE85) & 0xffffffff)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ a0, p1 & m32, (p0 >> np.uint64(32)) ^ c[3] ^ a1, p0 & m32]
    w = np.stack([h for v in c for h in (v & np.uint64(0xffff), v >> np.uint64(16))], 1).reshape(-1)[:n]
    return torch.from_numpy((w >= np.uint64(int(round(p * 65536)))))


def scale_of(p):
    return 65536.0 / (65536 - int(round(p * 65536)))


# -- gated_feed_forward ---------------------------------------------------------------------------
def gate(a, act):
    if act == "gelu":
        cdf = 0.5 * torch.special.erfc(-a / math.sqrt(2))
        return a * cdf, cdf + a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(a)
    return (a * s, s * (1 + a * (1 - s))) if act == "silu" else (s, s * (1 - s))


def gated_ref(x, wg, wv, wo, bg, bv, bo, act, dy):
    """{name: (value, bound without the output's own rounding)}: rows x [M, D], all inputs as the kernel reads them.

    The kernel holds h, da and dv in x's type (one rounding ut each; da and dv of few rows in fp32), u = act(a) and p = v act'(a) in the upper 24 bits of their fp32
    values (16-bit types; cut off: below 2^-15 of the value) and adds in fp32; a product of K terms is off by at most
    (K + 8) U sum|terms|, 4 more roundings an fp32 product that is put together from parts (its parts below 2^-23 are left out, less than 4 U)."""
    t = x.dtype
    ut, eta = u(t), torch.finfo(t).smallest_normal * u(t)       # one rounding: relative, and half a step of the smallest numbers
    x, wg, wv, dy = x.double(), wg.double(), wv.double(), dy.double()
    ab = torch.Tensor.abs
    M, D = x.shape
    F = wg.shape[0]

    def lin(p, q, dp=None, dq=None):
        """(p q^T, its error bound) for operands off by at most dp, dq"""
        v = p @ q.t().contiguous()
        e = (p.shape[1] + 12) * U * (ab(p) @ ab(q).t().contiguous())
        if dp is not None:
            e = e + dp @ ab(q).t().contiguous()
        if dq is not None:
            e = e + ab(p) @ dq.t().contiguous()
        return v, e

    a, ea = lin(x, wg)
    v, ev = lin(x, wv)
    if bg is not None:
        a = a + bg.double()
    if bv is not None:
        v = v + bv.double()
    ea, ev = ea + U * ab(a), ev + U * ab(v)
    g, dg = gate(a, act)
    # |act''| <= 1.2 for the three gates; a few roundings of exp / erf (4 U relative each)
    eg, edg = ab(dg) * ea + 1.2 * ea * ea + 16 * U * ab(g), 1.2 * ea + 16 * U * (ab(dg) + 1)
    h = g * v
    eh = ab(g) * ev + ab(v) * eg + eg * ev + (ut + 2 * U) * ab(h) + eta
    out = {}
    if wo is not None:
        wo = wo.double()
        y, ey = lin(h, wo, dp=eh)
        if bo is not None:
            y = y + bo.double()
            out["dbo"] = (dy.sum(0), (M + 8) * U * ab(dy).sum(0))
        out["y"] = (y, ey + U * ab(y))
        dh, edh = lin(dy, wo.t().contiguous())
        out["dwo"] = lin(dy.t().contiguous(), h.t().contiguous(), dq=eh.t().contiguous())
    else:
        out["y"] = (h, eh)
        dh, edh = dy, torch.zeros_like(dy)
    da, dv = dh * v * dg, dh * g
    # u and p as they are kept, then da = dh p and dv = dh u
    kt = 0 if t == torch.float32 else 2.0 ** -15
    ekp = ev * ab(dg) + ab(v) * edg + ev * edg + (kt + 2 * U) * ab(v * dg)
    eku = eg + kt * ab(g)
    eda = edh * ab(v * dg) + ab(dh) * ekp + edh * ekp + (ut + 2 * U) * ab(da) + eta
    edv = edh * ab(g) + ab(dh) * eku + edh * eku + (ut + 2 * U) * ab(dv) + eta
    p, ep = lin(da, wg.t().contiguous(), dp=eda)
    q, eq = lin(dv, wv.t().contiguous(), dp=edv)
    out["dx"] = (p + q, ep + eq + (F + 12) * U * (ab(p) + ab(q)))
    out["dwg"] = lin(da.t().contiguous(), x.t().contiguous(), dp=eda.t().contiguous())
    out["dwv"] = lin(dv.t().contiguous(), x.t().contiguous(), dp=edv.t().contiguous())
    out["dbg"] = (da.sum(0), eda.sum(0) + (M + 8) * U * ab(da).sum(0))
    out["dbv"] = (dv.sum(0), edv.sum(0) + (M + 8) * U * ab(dv).sum(0))
    return {k: (val, 2 * bound) for k, (val, bound) in out.items()}


def check(name, got, ref, bound):
    """|got - ref| <= bound + one rounding of the output (relative, or half a step of its smallest numbers)"""
    t = got.dtype
    got = got.double()
    ok = (got - ref).abs() <= bound + u(t) * (ref.abs() + bound) + torch.finfo(t).smallest_normal * u(t)
    if not bool(ok.all()):
        i = int(((got - ref).abs() - bound - u(t) * ref.abs()).argmax())
        raise AssertionError("%s: %d of %d values out of bounds; worst %r, expected %r, bound %.3g" % (
            name, int((~ok).sum()), ok.numel(), float(got.flatten()[i]), float(ref.flatten()[i]), float(bound.expand_as(ref).flatten()[i])))
