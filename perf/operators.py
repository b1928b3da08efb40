"""Workloads of the channel-MLP operators: channel_norm, dropout and gated_feed_forward, alone, forward and training.

`run` computes one pass through an operator on what `prepare` made: with `own` False in its plain form (elementary torch
operations in 32 bits, rounded once at the end), with `own` True by the calls a user makes of council_gan_amd.  `exact` computes
the same from the definitions in 64 bits.  A case is a dict of plain values; `listed` gives the fixed ones, `draw` more of the
same ranges.

    channel_norm         y = (x - mean) / sqrt(var + eps) * weight + bias over the channels of every row (biased variance)
    dropout              y = residual + x * keep / (1 - t / 65536); keep = (16-bit draw >= t), t = round(65536 p); the draws of the
                         8 values of block b are the 16-bit halves (low first) of Philox4x32-10 with counter (b, step) and key seed
    gated_feed_forward   y = (act(x Wg^T + bg) * (x Wv^T + bv)) Wo^T + bo
"""
import math

import torch

own = False

_DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}


# ------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------
def _norm(rows, c, dtype, wdtype=None, bias=True, train=True, image=0, eps=1e-5, **kw):
    return dict(op="norm", rows=rows, c=c, dtype=dtype, wdtype=wdtype or dtype, bias=bias, train=train, image=image, eps=eps, **kw)


def _drop(rows, c, dtype, p, residual, train=True, **kw):
    return dict(op="dropout", rows=rows, c=c, dtype=dtype, p=p, residual=residual, train=train, **kw)


def _gated(m, d, f, dtype, act="silu", bias=False, train=True, **kw):
    return dict(op="gated", m=m, d=d, f=f, dtype=dtype, act=act, bias=bias, train=train, **kw)


def listed():
    return [
        # the hidden vectors of the style MLP (mlp_dim 256) of a council of 4 at batch 4, in training: a call of pure latency
        _norm(16, 256, "fp32", name="norm_style"),
        # the 64 x 64 x 256 content codes of a council of 4 at batch 4, every pixel's channels normalised
        _norm(65536, 256, "fp32", image=64, name="norm_pixels"),
        # token rows of a wide transformer block in 16 bits: the largest rows
        _norm(16384, 4096, "bf16", name="norm_tokens"),
        # a ragged batch with an odd width (rows start at any alignment), norm weights kept in 32 bits
        _norm(5003, 1255, "fp16", wdtype="fp32", name="norm_ragged"),
        # dropout on the hidden vectors of the style MLP
        _drop(16, 256, "fp32", 0.1, False, name="dropout_style"),
        # dropout joined with the residual sum of a transformer block, the largest activations
        _drop(16384, 4096, "bf16", 0.1, True, name="dropout_residual"),
        # an odd number of values in 32 bits, strong dropout
        _drop(4099, 1001, "fp32", 0.5, False, name="dropout_ragged"),
        # serving one token: bound by reading the weights
        _gated(1, 1024, 2816, "bf16", train=False, name="gated_one_token"),
        # the style MLP's hidden vectors through a gated block, in training
        _gated(16, 256, 1024, "fp32", bias=True, name="gated_style"),
        # every pixel of the content codes through a gated block, in training, in the 32 bits this package trains in
        _gated(65536, 256, 1024, "fp32", bias=True, name="gated_pixels"),
        # a training step on a large batch of tokens in 16 bits
        _gated(16384, 2048, 5632, "bf16", name="gated_tokens"),
        # a ragged batch and odd widths, the gelu gate, biases
        _gated(777, 1001, 2730, "fp16", act="gelu", bias=True, name="gated_ragged"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("norm", "dropout", "gated"))
    dtype = rng.choice(("fp32", "fp16", "bf16"))
    if op == "norm":
        c = _log_int(rng, 16, 8192)
        image = rng.choice((0, 0, 0, 5, 16))
        rows = _log_int(rng, 1, min(65536, (1 << 26) // c))
        if image:
            rows = max(1, rows // (image * image)) * image * image
            rows = min(rows, max(1, (1 << 26) // (c * image * image)) * image * image)
        return _norm(rows, c, dtype, wdtype=rng.choice((dtype, "fp32")), bias=rng.random() < 0.7, train=rng.random() < 0.7,
                     image=image, eps=rng.choice((1e-5, 1e-6)))
    if op == "dropout":
        c = _log_int(rng, 1, 8192)
        rows = _log_int(rng, 1, min(65536, (1 << 26) // c))
        return _drop(rows, c, dtype, round(rng.uniform(0.01, 0.9), 3), rng.random() < 0.5, train=rng.random() < 0.7)
    d, f = _log_int(rng, 8, 2048), _log_int(rng, 8, 5632)
    return _gated(_log_int(rng, 1, 16384), d, f, dtype, act=rng.choice(("silu", "gelu", "sigmoid")), bias=rng.random() < 0.5,
                  train=rng.random() < 0.6)


def work(case):
    """What a pass cannot do without: every input read once, every output written once, the products and sums."""
    e = _SIZE[case["dtype"]]
    if case["op"] == "norm":
        n, we = case["rows"] * case["c"], _SIZE[case["wdtype"]] * case["c"] * (2 if case["bias"] else 1)
        return {"bytes": n * e * (4 if case["train"] else 2) + we * (2 if case["train"] else 1),
                "flops": n * (19 if case["train"] else 8)}
    if case["op"] == "dropout":
        n = case["rows"] * case["c"]
        return {"bytes": n * e * (2 + (1 if case["residual"] else 0) + (2 if case["train"] else 0)) + 16,
                "flops": n * (2 if case["train"] else 1) + (n if case["residual"] else 0)}
    m, d, f = case["m"], case["d"], case["f"]
    par = 3 * d * f + ((2 * f + d) if case["bias"] else 0)
    return {"bytes": e * (m * d * (4 if case["train"] else 2) + par * (2 if case["train"] else 1)),
            "flops": 6 * m * d * f * (3 if case["train"] else 1)}


# ------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------
def _make(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7fffffffffffffff)
    dt = _DT[case["dtype"]]

    def rnd(*shape, scale=1.0, shift=0.0, dtype=dt):
        return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(dtype)

    if case["op"] == "norm":
        rows, c, im = case["rows"], case["c"], case["image"]
        # activations with a mean of their own in every row, as they leave a residual stream
        x = (torch.randn((rows, c), generator=g, device="cuda") * 1.5 + torch.randn((rows, 1), generator=g, device="cuda")).to(dt)
        dy = rnd(rows, c)
        if im:      # logical NCHW, channels_last: every pixel's channels lie next to each other
            x, dy = (t.view(rows // (im * im), im, im, c).permute(0, 3, 1, 2) for t in (x, dy))
        wt = _DT[case["wdtype"]]
        return {"x": x, "dy": dy, "w": rnd(c, scale=0.2, shift=1.0, dtype=wt), "b": rnd(c, scale=0.2, dtype=wt) if case["bias"] else None}
    if case["op"] == "dropout":
        shape = (case["rows"], case["c"])
        key = torch.randint(0, 2 ** 62, (2,), generator=g, device="cuda", dtype=torch.int64)
        return {"x": rnd(*shape), "dy": rnd(*shape), "key": key, "res": rnd(*shape) if case["residual"] else None}
    m, d, f, b = case["m"], case["d"], case["f"], case["bias"]
    return {"x": rnd(m, d), "dy": rnd(m, d),
            "wg": rnd(f, d, scale=d ** -0.5), "wv": rnd(f, d, scale=d ** -0.5), "wo": rnd(d, f, scale=f ** -0.5),
            "bg": rnd(f, scale=0.1) if b else None, "bv": rnd(f, scale=0.1) if b else None, "bo": rnd(d, scale=0.1) if b else None}


_LEAVES = {"norm": ("x", "w", "b"), "dropout": ("x",), "gated": ("x", "wg", "wv", "wo", "bg", "bv", "bo")}


def prepare(case, seed):
    state = _make(case, seed)
    state["case"] = case
    if own:
        import council_gan_amd
        state["ops"] = council_gan_amd.ops
        if case["train"]:
            for k in _LEAVES[case["op"]]:
                if state[k] is not None:
                    state[k].requires_grad_(True)
    return state


# ------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------
def _forward_own(s):
    c, ops = s["case"], s["ops"]
    if c["op"] == "norm":
        return ops.channel_norm(s["x"], s["w"], s["b"], c["eps"])
    if c["op"] == "dropout":
        return ops.dropout(s["x"], c["p"], s["key"], residual=s["res"])
    return ops.gated_feed_forward(s["x"], s["wg"], s["wv"], s["wo"], s["bg"], s["bv"], s["bo"], act=c["act"])


def _run_own(s):
    c = s["case"]
    if not c["train"]:
        with torch.no_grad():
            return [_forward_own(s)]
    y = _forward_own(s)
    leaves = [s[k] for k in _LEAVES[c["op"]] if s[k] is not None]
    return [y.detach()] + list(torch.autograd.grad(y, leaves, s["dy"]))


def _rows(t, c):
    return t.permute(0, 2, 3, 1).reshape(-1, c) if t.dim() == 4 else t


def _image(t, like):
    if like.dim() != 4:
        return t
    n, c, h, w = like.shape
    return t.view(n, h, w, c).permute(0, 3, 1, 2)


def _plain_norm(s):
    c = s["case"]
    x, w = _rows(s["x"], c["c"]).float(), s["w"].float()
    mean = x.mean(1, keepdim=True)
    xc = x - mean
    rstd = 1.0 / torch.sqrt((xc * xc).mean(1, keepdim=True) + c["eps"])
    xh = xc * rstd
    y = xh * w
    if s["b"] is not None:
        y = y + s["b"].float()
    out = [_image(y.to(s["x"].dtype), s["x"])]
    if c["train"]:
        dy = _rows(s["dy"], c["c"]).float()
        g = dy * w
        dx = (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True)) * rstd
        out += [_image(dx.to(s["x"].dtype), s["x"]), (dy * xh).sum(0).to(s["w"].dtype)]
        if s["b"] is not None:
            out.append(dy.sum(0).to(s["b"].dtype))
    return out


_MASK = 0xffffffff


def _philox_words(blocks, key):
    """The four 32-bit words of Philox4x32-10 (Salmon et al., 2011) for `blocks` consecutive counters; 64-bit products wrap, their
    halves do not care."""
    c0 = torch.arange(blocks, device=key.device, dtype=torch.int64)
    c1 = c0 >> 32
    c0 = c0 & _MASK
    c2, c3 = (key[1] & _MASK).expand_as(c0), ((key[1] >> 32) & _MASK).expand_as(c0)
    k0, k1 = key[0] & _MASK, (key[0] >> 32) & _MASK
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & _MASK) ^ c1 ^ k0, p1 & _MASK, ((p0 >> 32) & _MASK) ^ c3 ^ k1, p0 & _MASK
        k0, k1 = (k0 + 0x9E3779B9) & _MASK, (k1 + 0xBB67AE85) & _MASK
    return c0, c1, c2, c3


def _plain_dropout(s):
    c = s["case"]
    x = s["x"]
    n, t = x.numel(), int(round(c["p"] * 65536))
    words = torch.stack(_philox_words((n + 7) // 8, s["key"]), 1)
    draws = torch.stack((words & 0xffff, words >> 16), 2).reshape(-1)[:n].view(x.shape)
    keep = (draws >= t).float() * (65536.0 / (65536 - t))
    y = x.float() * keep
    if s["res"] is not None:
        y = s["res"].float() + y
    out = [y.to(x.dtype)]
    if c["train"]:
        out.append((s["dy"].float() * keep).to(x.dtype))
    return out


def _gate(a, act):
    """act(a) and its derivative."""
    if act == "gelu":
        phi = 0.5 * (1.0 + torch.erf(a * (0.5 ** 0.5)))
        return a * phi, phi + a * torch.exp(-0.5 * a * a) * (1.0 / math.sqrt(2.0 * math.pi))
    sg = 1.0 / (1.0 + torch.exp(-a))
    if act == "silu":
        return a * sg, sg * (1.0 + a * (1.0 - sg))
    return sg, sg * (1.0 - sg)


def _plain_gated(s):
    c = s["case"]
    x, wg, wv, wo = (s[k].float() for k in ("x", "wg", "wv", "wo"))
    a, v = x @ wg.t(), x @ wv.t()
    if c["bias"]:
        a, v = a + s["bg"].float(), v + s["bv"].float()
    u, du = _gate(a, c["act"])
    h = u * v
    y = h @ wo.t()
    if c["bias"]:
        y = y + s["bo"].float()
    out = [y]
    if c["train"]:
        dy = s["dy"].float()
        dh = dy @ wo
        da, dv = dh * v * du, dh * u
        out += [da @ wg + dv @ wv, da.t() @ x, dv.t() @ x, dy.t() @ h]
        if c["bias"]:
            out += [da.sum(0), dv.sum(0), dy.sum(0)]
    return [t.to(s["x"].dtype) for t in out]


def run(state):
    if own:
        return _run_own(state)
    return {"norm": _plain_norm, "dropout": _plain_dropout, "gated": _plain_gated}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------
def _exact_norm(case, s):
    dim = s["x"].dim()
    axis = 1 if dim == 4 else dim - 1
    others = [i for i in range(dim) if i != axis]
    shape = [1] * dim
    shape[axis] = case["c"]
    x, w = s["x"].double(), s["w"].double().view(shape)
    var, mean = torch.var_mean(x, dim=axis, keepdim=True, correction=0)
    sd = torch.sqrt(var + case["eps"])
    z = (x - mean) / sd
    y = z * w
    if case["bias"]:
        y = y + s["b"].double().view(shape)
    out = [y]
    if case["train"]:
        dy = s["dy"].double()
        dz = dy * w
        out.append((dz - dz.mean(axis, keepdim=True) - z * (dz * z).mean(axis, keepdim=True)) / sd)
        out.append((dy * z).sum(others))
        if case["bias"]:
            out.append(dy.sum(others))
    return out


def _mulhilo(a, m):
    """(high, low) 32 bits of a * m for int64 arrays of 32-bit values, by 16-bit halves (nothing wraps)."""
    ah, al, mh, ml = a >> 16, a & 0xffff, m >> 16, m & 0xffff
    low = al * ml
    mid = ah * ml + (low >> 16)
    mid2 = al * mh + (mid & 0xffff)
    return ah * mh + (mid >> 16) + (mid2 >> 16), ((mid2 & 0xffff) << 16) | (low & 0xffff)


def _exact_dropout(case, s):
    n = s["x"].numel()
    seed, step = (int(v) for v in s["key"].tolist())
    blk = torch.arange((n + 7) // 8, device="cuda", dtype=torch.int64)
    ctr = [blk % (1 << 32), blk // (1 << 32), torch.full_like(blk, step % (1 << 32)), torch.full_like(blk, (step // (1 << 32)) % (1 << 32))]
    for r in range(10):
        k0 = (seed % (1 << 32) + r * 0x9E3779B9) % (1 << 32)
        k1 = (seed // (1 << 32) + r * 0xBB67AE85) % (1 << 32)
        h0, l0 = _mulhilo(ctr[0], 0xD2511F53)
        h1, l1 = _mulhilo(ctr[2], 0xCD9E8D57)
        ctr = [h1 ^ ctr[1] ^ k0, l1, h0 ^ ctr[3] ^ k1, l0]
    t = int(round(case["p"] * 65536))
    keep = torch.empty((blk.numel(), 8), dtype=torch.bool, device="cuda")
    for i, wd in enumerate(ctr):
        keep[:, 2 * i] = wd % 65536 >= t
        keep[:, 2 * i + 1] = wd // 65536 >= t
    keep = keep.view(-1)[:n].view(s["x"].shape)
    scale = 65536.0 / (65536 - t)
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    y = torch.where(keep, s["x"].double() * scale, zero)
    if s["res"] is not None:
        y = y + s["res"].double()
    return [y] + ([torch.where(keep, s["dy"].double() * scale, zero)] if case["train"] else [])


def _exact_gated(case, s):
    def lin(t, w, b):
        y = torch.mm(t, w.t().contiguous())
        return y if b is None else y.add_(b.double())

    x, wg, wv, wo = (s[k].double() for k in ("x", "wg", "wv", "wo"))
    a, v = lin(x, wg, s["bg"]), lin(x, wv, s["bv"])
    if case["act"] == "gelu":
        cdf = 0.5 * torch.special.erfc(-a / math.sqrt(2.0))
        u = a * cdf
    else:
        cdf = torch.sigmoid(a)
        u = a * cdf if case["act"] == "silu" else cdf
    h = u * v
    out = [lin(h, wo, s["bo"])]
    if case["train"]:
        if case["act"] == "gelu":
            du = cdf + a * torch.exp(a.square() * -0.5) / math.sqrt(2.0 * math.pi)
        elif case["act"] == "silu":
            du = cdf + u * (1.0 - cdf)
        else:
            du = cdf * (1.0 - cdf)
        dy = s["dy"].double()
        dh = torch.mm(dy, wo)
        dv = dh * u
        da = dh.mul_(v).mul_(du)
        del v, du, u
        out += [torch.mm(da, wg).add_(torch.mm(dv, wv)), torch.mm(da.t().contiguous(), x), torch.mm(dv.t().contiguous(), x),
                torch.mm(dy.t().contiguous(), h)]
        if case["bias"]:
            out += [da.sum(0), dv.sum(0), dy.sum(0)]
    return out


def exact(case, seed):
    s = _make(case, seed)
    return {"norm": _exact_norm, "dropout": _exact_dropout, "gated": _exact_gated}[case["op"]](case, s)
