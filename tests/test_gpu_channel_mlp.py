"""channel_norm, dropout and gated_feed_forward on the GPU against plain 64-bit forms (channel_mlp_ref.py), forward and backward:
every type, odd sizes and strides, one row to long ones, no rows, streams, captured graphs, member-batched parameters."""
import contextlib
import gc

import numpy as np
import pytest
import torch

import channel_mlp_ref as R

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DTYPES = [F32, F16, BF16]
ID = {F32: "fp32", F16: "fp16", BF16: "bf16"}


@pytest.fixture(scope="module")
def cga():
    import council_gan_amd
    council_gan_amd.hip.load()
    return council_gan_amd


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rnd(g, *shape, scale=1.0, shift=0.0, dtype=F32):
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * scale + shift).to(dtype).cuda()


# ------------------------------------------------------------------------------------------
# channel_norm
# ------------------------------------------------------------------------------------------
NORM_SIZES = [(1, 1), (3, 2), (1, 256), (16, 256), (5, 7), (33, 64), (17, 100), (130, 255), (64, 512), (9, 1000), (11, 1255), (6, 2048),
              (5, 4099), (3, 8192), (2, 20001), (1111, 48), (2500, 320)]


def norm_case(cga, x, w, b, dy, eps=1e-5):
    xl, wl = x.detach().requires_grad_(True), w.detach().clone().requires_grad_(True)
    bl = b.detach().clone().requires_grad_(True) if b is not None else None
    y = cga.ops.channel_norm(xl, wl, bl, eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    grads = torch.autograd.grad(y, [t for t in (xl, wl, bl) if t is not None], dy)
    with torch.no_grad():
        assert torch.equal(cga.ops.channel_norm(x, w, b, eps), y)
    ref = R.norm_ref(R.rows_of(x), w, b, eps, R.rows_of(dy))
    R.check("y", R.rows_of(y), *ref["y"])
    R.check("dx", R.rows_of(grads[0]), *ref["dx"])
    R.check("dw", grads[1], *ref["dw"])
    if b is not None:
        R.check("db", grads[2], *ref["db"])
    return y, grads


@pytest.mark.parametrize("dtype", DTYPES, ids=ID.get)
@pytest.mark.parametrize("size", NORM_SIZES, ids=str)
def test_channel_norm(cga, size, dtype):
    rows, C = size
    g = gen(rows * 10007 + C)
    x = rnd(g, rows, C, scale=1.5) + rnd(g, rows, 1, dtype=F32)
    bias = (rows + C) % 3 != 0
    wt = F32 if rows % 2 else dtype
    norm_case(cga, x.to(dtype), rnd(g, C, scale=0.3, shift=1.0, dtype=wt), rnd(g, C, scale=0.3, dtype=wt) if bias else None,
              rnd(g, rows, C, dtype=dtype))


@pytest.mark.parametrize("dtype", DTYPES, ids=ID.get)
def test_channel_norm_normalises_the_pixels_of_an_image(cga, dtype):
    g = gen(5)
    x = rnd(g, 2, 96, 5, 3, dtype=dtype)
    dy = rnd(g, 2, 96, 5, 3, dtype=dtype)
    w, b = rnd(g, 96, dtype=dtype), rnd(g, 96, dtype=dtype)
    y, _ = norm_case(cga, x, w, b, dy)
    assert y.is_contiguous(memory_format=torch.channels_last)
    y2, _ = norm_case(cga, x.contiguous(memory_format=torch.channels_last), w, b, dy)
    assert torch.equal(y, y2)


@pytest.mark.parametrize("dtype", DTYPES, ids=ID.get)
def test_channel_norm_of_strided_shifted_and_expanded_inputs(cga, dtype):
    g = gen(6)
    flat = rnd(g, 1 + 7 * 130, dtype=dtype)
    w, b, dy = rnd(g, 129, dtype=dtype), rnd(g, 129, dtype=dtype), rnd(g, 7, 129, dtype=dtype)
    norm_case(cga, flat[1:].view(7, 130)[:, 1:], w, b, dy)                       # gaps between rows, odd start
    norm_case(cga, flat[1:1 + 7 * 129].view(7, 129), w, b, dy)                   # dense, but starts off 16 bytes
    norm_case(cga, flat[:129 * 7].view(129, 7).t(), w, b, dy)                    # transposed
    norm_case(cga, flat[:129].expand(7, 129), w, b, dy[:1].expand(7, 129))       # one row for all


@pytest.mark.parametrize("dtype", DTYPES, ids=ID.get)
def test_channel_norm_far_from_zero_and_constant_rows(cga, dtype):
    g = gen(7)
    x = rnd(g, 8, 384, scale=0.25, shift=40.0, dtype=dtype)
    x[3] = 2.0                      # no variance: y = bias, finite gradients
    w, b, dy = rnd(g, 384, dtype=dtype), rnd(g, 384, dtype=dtype), rnd(g, 8, 384, dtype=dtype)
    y, grads = norm_case(cga, x, w, b, dy)
    assert torch.equal(y[3], b) and all(bool(torch.isfinite(t).all()) for t in grads)


def test_channel_norm_keeps_a_bad_row_to_itself(cga):
    g = gen(8)
    x, w = rnd(g, 6, 300), rnd(g, 300)
    y = cga.ops.channel_norm(x, w)
    x2 = x.clone()
    x2[2, 5], x2[4, 7] = float("inf"), float("nan")
    y2 = cga.ops.channel_norm(x2, w)
    for r in (0, 1, 3, 5):
        assert torch.equal(y[r], y2[r])
    assert bool(torch.isnan(y2[2]).any()) and bool(torch.isnan(y2[4]).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=ID.get)
def test_channel_norm_of_no_rows(cga, dtype):
    x = torch.empty(0, 64, dtype=dtype, device="cuda", requires_grad=True)
    w = torch.ones(64, dtype=dtype, device="cuda", requires_grad=True)
    b = torch.zeros(64, dtype=dtype, device="cuda", requires_grad=True)
    y = cga.ops.channel_norm(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == gx.shape == (0, 64) and not gw.any() and not gb.any()


def test_channel_norm_gradient_against_differences(cga):
    g = gen(9)
    x, w, b, dy = rnd(g, 4, 40), rnd(g, 40), rnd(g, 40), rnd(g, 4, 40)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(cga.ops.channel_norm(x, w, b), leaves, dy)
    for k, (t, gr) in enumerate(zip(leaves, grads)):
        d = rnd(g, *t.shape)
        e = 1e-3
        hi, lo = [cga.ops.channel_norm(*(s.detach() + (sg * e * d if j == k else 0) for j, s in enumerate(leaves)))
                  for sg in (1, -1)]
        got, want = float((gr * d).double().sum()), float(((hi - lo).double() * dy).sum() / (2 * e))
        # curvature: e^2 times third derivatives of order 10; rounding: 160 values with errors of some U over 2 e
        assert abs(got - want) < 160 * (e * e * 10 + 8 * R.U / e), (k, got, want)


# ------------------------------------------------------------------------------------------
# dropout
# ------------------------------------------------------------------------------------------
def key_of(seed, step):
    return torch.tensor([seed, step], dtype=torch.int64, device="cuda")


def drop_ref(x, p, seed, step, res=None):
    keep = R.keep_mask(x.numel(), p, seed, step).view(x.shape).cuda()
    v = torch.where(keep, x.double() * R.scale_of(p), torch.zeros((), dtype=torch.float64, device="cuda"))
    # one fp32 product, with a residual one fp32 sum
    return (v + res.double(), 2 * R.U * v.abs() + R.U * res.double().abs()) if res is not None else (v, 2 * R.U * v.abs())


@pytest.mark.parametrize("dtype", DTYPES, ids=ID.get)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (3, 5), (16, 256), (1025, 33), (4099, 101)], ids=str)
def test_dropout(cga, shape, dtype):
    g = gen(sum(shape))
    x, res, dy = (rnd(g, *shape, dtype=dtype) for _ in range(3))
    for p, seed, step in ((0.0, 1, 0), (0.1, 2 ** 61 + 12345, 3), (0.5, -7, 2 ** 40 + 1), (0.999, 99, -1)):
        xl, rl = x.detach().requires_grad_(True), res.detach().requires_grad_(True)
        for r in (None, rl):
            y = cga.ops.dropout(xl, p, key_of(seed, step), residual=r)
            grads = torch.autograd.grad(y, [xl] if r is None else [xl, rl], dy)
            R.check("y", y, *drop_ref(x, p, seed, step, None if r is None else res))
            R.check("dx", grads[0], *drop_ref(dy, p, seed, step))
            if r is not None:
                assert torch.equal(grads[1], dy)
            with torch.no_grad():
                assert torch.equal(cga.ops.dropout(x, p, key_of(seed, step), residual=None if r is None else res), y)


def test_dropout_takes_any_layout_and_alignment(cga):
    g = gen(1)
    x = rnd(g, 2, 6, 5, 4, dtype=BF16)
    y = cga.ops.dropout(x, 0.4, key_of(5, 6))
    assert y.is_contiguous(memory_format=torch.channels_last)
    flat = x.permute(0, 2, 3, 1).reshape(-1)                       # positions run over the channels_last form
    assert torch.equal(y.permute(0, 2, 3, 1).reshape(-1), cga.ops.dropout(flat, 0.4, key_of(5, 6)))
    odd = torch.cat((flat[:1], flat))[1:]
    assert odd.data_ptr() % 16 and torch.equal(cga.ops.dropout(odd, 0.4, key_of(5, 6)), cga.ops.dropout(flat, 0.4, key_of(5, 6)))
    t = rnd(g, 9, 8)
    assert torch.equal(cga.ops.dropout(t.t(), 0.4, key_of(5, 6)), cga.ops.dropout(t.t().contiguous(), 0.4, key_of(5, 6)))


def test_dropout_drops_infinities_and_nan_and_covers_no_values(cga):
    x = torch.full((4096,), float("nan"), device="cuda")
    x[::2] = float("inf")
    keep = R.keep_mask(4096, 0.5, 3, 4).cuda()
    y = cga.ops.dropout(x, 0.5, key_of(3, 4))
    assert not y[~keep].any() and not torch.isfinite(y[keep]).any()
    assert cga.ops.dropout(torch.empty(0, 5, device="cuda"), 0.5, key_of(3, 4)).shape == (0, 5)


def test_dropout_rate_and_independence_of_keys(cga):
    n = 1 << 20
    x = torch.ones(n, device="cuda")
    masks = [cga.ops.dropout(x, 0.3, key_of(s, t)) != 0 for s, t in ((1, 0), (1, 1), (2, 0))]
    for m in masks:      # 6 standard deviations of the binomial mean
        assert abs(float(m.double().mean()) - 0.7) < 6 * (0.21 / n) ** 0.5
    for i in range(3):
        for j in range(i):
            both = float((masks[i] & masks[j]).double().mean())
            assert abs(both - 0.49) < 6 * (0.25 / n) ** 0.5


def test_dropout_keys_advance_on_the_device(cga):
    st = cga.ops.dropout_state(2 ** 64 - 3)
    k0, k1 = cga.ops.dropout_key(st), cga.ops.dropout_key(st)
    assert k0.tolist() == [-3, 0] and k1.tolist() == [-3, 1] and st.tolist() == [-3, 2]


def test_dropout_refuses_a_key_that_changed_before_the_backward_pass(cga):
    st = cga.ops.dropout_state(1)
    x = torch.ones(64, device="cuda", requires_grad=True)
    y = cga.ops.dropout(x, 0.5, st)
    cga.ops.dropout_key(st)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# ------------------------------------------------------------------------------------------
# gated_feed_forward
# ------------------------------------------------------------------------------------------
# rows, D, F, O (0: no output projection), biases
GATED_SIZES = [(1, 1, 1, 1, True), (1, 8, 32, 8, False), (1, 256, 704, 256, False), (2, 64, 96, 32, True), (3, 5, 7, 9, True), (16, 256, 1024, 256, True),
               (17, 33, 65, 31, True), (48, 128, 200, 128, False), (64, 64, 64, 64, True), (65, 100, 130, 70, False),
               (127, 257, 129, 255, True), (130, 96, 352, 0, True), (200, 72, 40, 0, False), (300, 512, 384, 512, True),
               (1000, 40, 24, 16, True), (90, 3, 200, 5, True), (90, 200, 3, 70, True), (70, 65, 70, 2, False), (300, 1, 2, 0, True),
               (517, 320, 264, 328, False), (2300, 128, 256, 128, True)]


def gated_inputs(g, rows, D, F, O, bias, dtype):
    x = rnd(g, rows, D, dtype=dtype)
    ps = [rnd(g, F, D, scale=D ** -0.5, dtype=dtype), rnd(g, F, D, scale=D ** -0.5, dtype=dtype),
          rnd(g, O, F, scale=F ** -0.5, dtype=dtype) if O else None,
          rnd(g, F, scale=0.2, dtype=dtype) if bias else None, rnd(g, F, scale=0.2, dtype=dtype) if bias else None,
          rnd(g, O, scale=0.2, dtype=dtype) if bias and O else None]
    return x, ps, rnd(g, rows, O or F, dtype=dtype)


NAMES = ("dwg", "dwv", "dwo", "dbg", "dbv", "dbo")


def gated_case(cga, x, ps, dy, act, need=None):
    leaves = [x.detach().requires_grad_(True)] + [None if p is None else p.detach().clone().requires_grad_(True) for p in ps]
    y = cga.ops.gated_feed_forward(*leaves, act=act)
    assert y.dtype == x.dtype
    have = [(n, t) for n, t in zip(("dx",) + NAMES, leaves) if t is not None and (need is None or n in need)]
    grads = torch.autograd.grad(y, [t for _, t in have], dy)
    with torch.no_grad():
        y0 = cga.ops.gated_feed_forward(x, *ps, act=act)
    ref = R.gated_ref(R.rows_of(x), *ps[:3], *ps[3:], act, R.rows_of(dy))
    R.check("y", R.rows_of(y), *ref["y"])
    R.check("y (serving)", R.rows_of(y0), *ref["y"])
    for (n, t), gr in zip(have, grads):
        assert gr.shape == t.shape and gr.dtype == t.dtype
        R.check(n, R.rows_of(gr) if n == "dx" else gr, *ref[n])
    return y, dict(zip([n for n, _ in have], grads))


@pytest.mark.parametrize("dtype", DTYPES, ids=ID.get)
@pytest.mark.parametrize("size", GATED_SIZES, ids=str)
def test_gated_feed_forward(cga, size, dtype):
    x, ps, dy = gated_inputs(gen(sum(size)), *size, dtype)
    gated_case(cga, x, ps, dy, ("silu", "gelu", "sigmoid")[sum(size) % 3])


@pytest.mark.parametrize("dtype", DTYPES, ids=ID.get)
@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
def test_gated_feed_forward_gates(cga, act, dtype):
    x, ps, dy = gated_inputs(gen(3), 70, 64, 96, 48, True, dtype)
    gated_case(cga, x * 8, ps, dy, act)             # far into the gates' tails


@pytest.mark.parametrize("dtype", DTYPES, ids=ID.get)
@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("rows,D", [(3, 24), (70, 2), (70, 40), (40, 1600), (700, 64)], ids=str)
def test_gated_feed_forward_over_the_whole_range_of_the_gates(cga, rows, D, act, dtype):
    """few rows, narrow rows, tiles, sums split over a long axis and several tiles.  The gate's weights are zero, so its arguments are the
    biases exactly: from -200 to 200, and densely where exp(-a) leaves the range of fp32 (88.72) and where its last bit goes (104)."""
    edges = torch.cat([torch.linspace(-200, 200, 301), -torch.linspace(88.5, 104.5, 401), torch.linspace(88.5, 104.5, 60)])
    x, ps, dy = gated_inputs(gen(rows + D), rows, D, edges.numel(), 24, True, dtype)
    ps[0], ps[3] = torch.zeros_like(ps[0]), edges.to(dtype).cuda()
    gated_case(cga, x, ps, dy, act)


@pytest.mark.parametrize("dtype", DTYPES, ids=ID.get)
def test_gated_feed_forward_large(cga, dtype):
    """several tiles in every direction, sums split over a long axis"""
    x, ps, dy = gated_inputs(gen(4), 5000, 520, 776, 392, True, dtype)
    gated_case(cga, x, ps, dy, "silu")


@pytest.mark.parametrize("dtype", DTYPES, ids=ID.get)
def test_gated_feed_forward_of_images_and_strided_inputs(cga, dtype):
    g = gen(5)
    x = rnd(g, 2, 24, 3, 5, dtype=dtype)
    _, ps, _ = gated_inputs(g, 1, 24, 40, 16, True, dtype)
    y, _ = gated_case(cga, x, ps, rnd(g, 2, 16, 3, 5, dtype=dtype), "silu")
    assert y.shape == (2, 16, 3, 5) and y.is_contiguous(memory_format=torch.channels_last)
    big = rnd(g, 31, 26, dtype=dtype)
    gated_case(cga, big[:, 1:25], ps, rnd(g, 16, 31, dtype=dtype).t(), "gelu")
    gated_case(cga, rnd(g, 3, 4, 24, dtype=dtype).transpose(0, 1), ps, rnd(g, 4, 3, 16, dtype=dtype), "gelu")
    wt = [rnd(g, 24, 40, dtype=dtype).t(), rnd(g, 41 * 24 + 1, dtype=dtype)[1:41 * 24 + 1].view(41, 24)[1:]] + ps[2:]     # transposed / shifted weights
    gated_case(cga, big[:, 1:25], wt, rnd(g, 31, 16, dtype=dtype), "silu")


@pytest.mark.parametrize("need", [("dx",), ("dwo",), ("dwg", "dbv"), ("dbo",)], ids=str)
def test_gated_feed_forward_gradients_one_by_one(cga, need):
    x, ps, dy = gated_inputs(gen(6), 90, 48, 56, 40, True, BF16)
    gated_case(cga, x, ps, dy, "silu", need=need)


@pytest.mark.parametrize("dtype", DTYPES, ids=ID.get)
def test_gated_feed_forward_of_no_rows(cga, dtype):
    x, ps, dy = gated_inputs(gen(7), 0, 16, 24, 8, True, dtype)
    leaves = [t.requires_grad_(True) for t in [x] + ps]
    y = cga.ops.gated_feed_forward(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    assert y.shape == (0, 8) and grads[0].shape == (0, 16) and not any(bool(t.any()) for t in grads[1:])


def test_gated_feed_forward_keeps_a_bad_row_to_itself(cga):
    for dtype in DTYPES:
        for rows in (3, 40, 300):
            x, ps, _ = gated_inputs(gen(8), rows, 128, 160, 96, True, dtype)
            y = cga.ops.gated_feed_forward(x, *ps)
            x2 = x.clone()
            x2[1, 3] = float("nan")
            y2 = cga.ops.gated_feed_forward(x2, *ps)
            ok = torch.arange(rows, device="cuda") != 1
            assert torch.equal(y[ok], y2[ok]) and bool(torch.isnan(y2[1]).all())


def test_gated_feed_forward_gradient_against_differences(cga):
    g = gen(9)
    x, ps, dy = gated_inputs(g, 6, 24, 40, 16, True, F32)
    leaves = [t.requires_grad_(True) for t in [x] + ps]
    grads = torch.autograd.grad(cga.ops.gated_feed_forward(*leaves), leaves, dy)
    for k, (t, gr) in enumerate(zip(leaves, grads)):
        d, e = rnd(g, *t.shape), 1e-3
        hi, lo = [cga.ops.gated_feed_forward(*(s.detach() + (sg * e * d if j == k else 0) for j, s in enumerate(leaves))) for sg in (1, -1)]
        got, want = float((gr * d).double().sum()), float(((hi - lo).double() * dy).sum() / (2 * e))
        # 96 outputs: curvature e^2 times third derivatives (up to order 100 along d), rounding of some 40 U over 2 e each
        assert abs(got - want) < 96 * (e * e * 100 + 40 * R.U / (2 * e)), (k, got, want)


def test_gated_feed_forward_errors_have_no_common_sign(cga):
    """Errors that share a sign grow with the rows in a bias gradient: the mean error over many rows is far below one rounding."""
    g = gen(41)
    M, D, F = 8192, 512, 96
    x, ps, dy = gated_inputs(g, M, D, F, 64, True, F32)
    h = cga.ops.gated_feed_forward(x, ps[0], ps[1], None, ps[3], ps[4])
    x64, wg, wv, bg, bv = (t.double() for t in (x, ps[0], ps[1], ps[3], ps[4]))
    v = x64 @ wv.t().contiguous() + bv
    h64 = R.gate(x64 @ wg.t().contiguous() + bg, "silu")[0] * v
    err = (h.double() - h64).mean(0) / h64.square().mean(0).sqrt()
    # A product of K = 512 is 6 * 512 / 16 = 192 additions to a running sum that grows to the result (0.7 of its size on average), each off
    # by up to half a step, 2^-24 of what it rounds, evenly: 192^0.5 / 3^0.5 * 0.7 * 2^-24 = 3.3e-7 of the result.  Gate and value together
    # 2^0.5 of that, their mean over 8192 rows 1 / 90.5 of it: 5.2e-9, and the largest of 96 columns stays below 5 times that, 2.6e-8.
    assert float(err.abs().max()) < 2.0 ** -25
    # over all columns the mean's spread is 5.2e-9 / 96^0.5 = 5.3e-10; 2^-28 is 7 times that
    assert float(err.mean().abs()) < 2.0 ** -28


@pytest.mark.parametrize("dtype", DTYPES, ids=ID.get)
@pytest.mark.parametrize("rows", [31, 32, 33, 34])
def test_gated_feed_forward_where_few_rows_end(cga, rows, dtype):
    x, ps, dy = gated_inputs(gen(rows), rows, 72, 136, 40, True, dtype)
    gated_case(cga, x, ps, dy, "silu")


# ------------------------------------------------------------------------------------------
# more than 2^32 elements: the rows at the end are those of a small call, or what the formula gives
# ------------------------------------------------------------------------------------------
def huge(rows, C, seed):
    """bf16 rows; the last 64 of their own"""
    x = torch.empty(rows, C, dtype=BF16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(seed))
    assert x.numel() > 2 ** 32
    return x


def test_channel_norm_past_32_bits(cga):
    C = 2056
    x, dy = huge(2 ** 21 + 7, C, 1).requires_grad_(True), huge(2 ** 21 + 7, C, 2)
    g = gen(1)
    w, b = rnd(g, C, shift=1.0, scale=0.3, dtype=BF16), rnd(g, C, scale=0.3, dtype=BF16)
    y = cga.ops.channel_norm(x, w, b)
    dx, = torch.autograd.grad(y, x, dy)
    ref = R.norm_ref(x[-64:].detach(), w, b, 1e-5, dy[-64:])
    R.check("y", y[-64:], *ref["y"])
    R.check("dx", dx[-64:], *ref["dx"])


def test_dropout_past_32_bits(cga):
    x = huge(2 ** 21 + 7, 2056, 3)
    y = cga.ops.dropout(x, 0.25, key_of(5, 6))
    n, tail = x.numel(), 4096
    keep = R.keep_mask(tail, 0.25, 5, 6, first=n - tail).cuda()
    v = torch.where(keep, x.view(-1)[-tail:].double() * R.scale_of(0.25), torch.zeros((), dtype=torch.float64, device="cuda"))
    R.check("y", y.view(-1)[-tail:], v, 2 * R.U * v.abs())


def test_gated_feed_forward_past_32_bits(cga):
    rows, D, F = 2 ** 22 + 5, 8, 1032          # the hidden units pass 2^32 elements
    g = gen(4)
    x, ps, _ = gated_inputs(g, 1, D, F, D, True, BF16)
    x = torch.empty(rows, D, dtype=BF16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(4)).requires_grad_(True)
    dy = torch.empty(rows, D, dtype=BF16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(5))
    y = cga.ops.gated_feed_forward(x, *ps)
    dx, = torch.autograd.grad(y, x, dy)
    ref = R.gated_ref(x[-64:].detach(), *ps, "silu", dy[-64:])
    R.check("y", y[-64:], *ref["y"])
    R.check("dx", dx[-64:], *ref["dx"])


def test_results_do_not_change_from_call_to_call(cga):
    for dtype in DTYPES:
        x, ps, dy = gated_inputs(gen(10), 2100, 200, 300, 100, True, dtype)
        w, b = rnd(gen(11), 200, dtype=dtype), rnd(gen(12), 200, dtype=dtype)
        runs = []
        for _ in range(3):
            leaves = [t.detach().clone().requires_grad_(True) for t in [x, w, b] + ps]
            y = cga.ops.gated_feed_forward(cga.ops.channel_norm(*leaves[:3]), *leaves[3:])
            runs.append([y] + list(torch.autograd.grad(y, leaves, dy)))
        for r in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(runs[0], r))


# ------------------------------------------------------------------------------------------
# together
# ------------------------------------------------------------------------------------------
def block(cga, x, w, b, ps, key, p=0.25):
    return cga.ops.dropout(cga.ops.gated_feed_forward(cga.ops.channel_norm(x, w, b), *ps), p, key, residual=x)


@pytest.mark.parametrize("dtype", DTYPES, ids=ID.get)
def test_block_of_all_three(cga, dtype):
    """x + dropout(gated_feed_forward(channel_norm(x))): values and gradients against the same block in 64 bits.  Each stage's own
    bound is tested above; here a stage's rounded output feeds the next, so errors are held to a multiple of one rounding of the
    type, relative to the largest value: 8 stored intermediates on the way, gains of at most 8 between them."""
    g = gen(20)
    rows, D, F = 150, 64, 96
    x, ps, dy = gated_inputs(g, rows, D, F, D, True, dtype)
    w, b = rnd(g, D, scale=0.2, shift=1, dtype=dtype), rnd(g, D, scale=0.2, dtype=dtype)
    leaves = [t.requires_grad_(True) for t in [x, w, b] + ps]
    y = block(cga, *leaves[:3], leaves[3:], key_of(4, 5))
    grads = torch.autograd.grad(y, leaves, dy)
    ref = [t.detach().double().requires_grad_(True) for t in leaves]
    xr, wr, br, wg, wv, wo, bg, bv, bo = ref
    n = torch.nn.functional.layer_norm(xr, (D,), wr, br, 1e-5)
    h = torch.nn.functional.silu(n @ wg.t() + bg) * (n @ wv.t() + bv)
    keep = R.keep_mask(x.numel(), 0.25, 4, 5).view(x.shape).cuda()
    yr = xr + torch.where(keep, (h @ wo.t() + bo) / 0.75, torch.zeros((), dtype=torch.float64, device="cuda"))
    gr = torch.autograd.grad(yr, ref, dy.double())
    tol = 8 * 8 * max(R.u(dtype), 16 * R.U)
    for k, (a, r) in enumerate(zip([y] + list(grads), [yr] + list(gr))):
        err = float((a.double() - r).abs().max() / r.abs().max())
        assert err < tol, (k, err, tol)


def test_on_a_stream_of_its_own(cga):
    g = gen(21)
    x, ps, dy = gated_inputs(g, 700, 128, 192, 128, True, BF16)
    w, b = rnd(g, 128, dtype=BF16), rnd(g, 128, dtype=BF16)

    def step():
        leaves = [t.detach().clone().requires_grad_(True) for t in [x, w, b] + ps]
        y = block(cga, *leaves[:3], leaves[3:], key_of(1, 2))
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))
    want = step()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:                              # several at once
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(step())
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for o in outs:
        assert all(torch.equal(a, c) for a, c in zip(want, o))


def test_captured_and_replayed(cga):
    """two graphs of the block's training step, replayed in turn between eager steps: new inputs every time, a new mask on every replay"""
    g = gen(22)
    D, F = 96, 128
    graphs = []
    for i, rows in enumerate((40, 600)):
        x, ps, dy = gated_inputs(g, rows, D, F, D, True, (F32, F16)[i])
        w, b = rnd(g, D, dtype=x.dtype), rnd(g, D, dtype=x.dtype)
        st = cga.ops.dropout_state(77 + i)
        leaves = [t.requires_grad_(True) for t in [x, w, b] + ps]

        def step(leaves=leaves, st=st, dy=dy, key=None):
            k = cga.ops.dropout_key(st) if key is None else key
            y = block(cga, *leaves[:3], leaves[3:], k)
            return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step()
        graphs.append((gr, out, step, x, st))
    for it in range(4):
        for i, (gr, out, step, x, st) in enumerate(graphs):
            with torch.no_grad():
                x.copy_(rnd(g, *x.shape, dtype=x.dtype))
            seed, at = st.tolist()
            gr.replay()
            torch.cuda.synchronize()
            assert st.tolist() == [seed, at + 1]
            want = step(key=key_of(seed, at))
            assert all(torch.equal(a, c) for a, c in zip(out, want)), (it, i)


# ------------------------------------------------------------------------------------------
# parameters of an optimizer and of several members
# ------------------------------------------------------------------------------------------
def member_params(n, D, F, g):
    out = []
    for _ in range(n):
        out.append([torch.nn.Parameter(t) for t in (
            torch.randn(D, generator=g) * 0.2 + 1, torch.randn(D, generator=g) * 0.2, torch.randn(F, D, generator=g) / D ** 0.5,
            torch.randn(F, D, generator=g) / D ** 0.5, torch.randn(D, F, generator=g) / F ** 0.5, torch.randn(F, generator=g) * 0.1,
            torch.randn(F, generator=g) * 0.1, torch.randn(D, generator=g) * 0.1)])
    return out


def pooled(cga, n, D, F, g):
    from council_gan_amd.optim import FlatAdam, ParamPool
    ps = member_params(n, D, F, g)
    pool = ParamPool([FlatAdam(p, lr=1e-3) for p in ps])
    pool.materialize("cuda")
    pool.zero_grad()
    return ps, pool


@pytest.mark.parametrize("n,rows,D,F", [(2, 5, 48, 40), (3, 150, 64, 96)])
def test_member_batched_matches_single_members(cga, n, rows, D, F):
    g = gen(30)
    ps, pool = pooled(cga, n, D, F, g)
    x, dy = rnd(g, n * rows, D), rnd(g, n * rows, D)
    xl = x.detach().requires_grad_(True)
    with cga.ops.members(n):
        p = ps[0]
        y = cga.ops.gated_feed_forward(cga.ops.channel_norm(xl, p[0], p[1]), *p[2:])
        y.backward(dy)
    got = [[t._cg_grad.clone() for t in p] for p in ps]
    assert all(t._cg_grad._cg_touched for t in ps[0])
    for k, p in enumerate(ps):
        sl = slice(k * rows, (k + 1) * rows)
        leaves = [t.detach().clone().requires_grad_(True) for t in [x[sl]] + p]
        yk = cga.ops.gated_feed_forward(cga.ops.channel_norm(*leaves[:3]), *leaves[3:])
        assert torch.equal(yk, y[sl])
        grads = torch.autograd.grad(yk, leaves, dy[sl])
        assert torch.equal(grads[0], xl.grad[sl])
        for a, b in zip(got[k], grads[1:]):
            assert torch.equal(a, b)


def test_gradients_add_to_the_optimizer_buffers(cga):
    g = gen(31)
    (p,), pool = pooled(cga, 1, 32, 40, g)
    x, dy = rnd(g, 20, 32), rnd(g, 20, 32)

    def step():
        cga.ops.gated_feed_forward(cga.ops.channel_norm(x, p[0], p[1]), *p[2:]).backward(dy)
    step()
    once = [t.grad.clone() for t in p]
    step()
    for a, t in zip(once, p):
        # the second pass adds the same value again: 2 a exactly
        assert torch.equal(t.grad, 2 * a)


def test_a_gradient_buffer_that_does_not_fit_is_refused(cga):
    """on the host, as after optimizer.materialize("cpu") and module.cuda(), or of another size: nothing is written"""
    g = gen(36)
    x, dy = rnd(g, 20, 32), rnd(g, 20, 32)
    for bad in (lambda t: torch.zeros(t.shape), lambda t: torch.zeros(t.numel() // 2, device="cuda")):
        for i in range(8):
            p = [t.detach().cuda().requires_grad_(True) for t in member_params(1, 32, 40, g)[0]]
            p[i]._cg_grad = bad(p[i])
            y = cga.ops.gated_feed_forward(cga.ops.channel_norm(x, p[0], p[1]), *p[2:])
            with pytest.raises(RuntimeError, match="gradient buffer"):
                y.backward(dy)
            assert not p[i]._cg_grad.any()


def test_one_buffer_for_two_parameters(cga):
    """A tensor that serves as two parameters gets the sum of both gradients in its one buffer."""
    g = gen(32)
    D = 48
    (p,), pool = pooled(cga, 1, D, D, g)
    w, wg, b = p[0], p[2], p[5]
    x, dy = rnd(g, 70, D), rnd(g, 70, D)

    def run(leaf_w, leaf_g, leaf_b):
        return cga.ops.gated_feed_forward(cga.ops.channel_norm(x, leaf_w[0], leaf_w[1]), *leaf_g, *leaf_b)
    run((w, w), (wg, wg, wg), (b, b, b)).backward(dy)
    apart = [[t.detach().clone().requires_grad_(True) for _ in range(k)] for t, k in ((w, 2), (wg, 3), (b, 3))]
    grads = torch.autograd.grad(run(*apart), [t for ts in apart for t in ts], dy)
    for t, gs in ((w, grads[:2]), (wg, grads[2:5]), (b, grads[5:])):
        want = sum(v.double() for v in gs)
        # the same gradients, added in fp32: two more roundings of partial sums
        tol = 3 * R.U * sum(v.double().abs() for v in gs)
        assert bool(((t._cg_grad.double() - want).abs() <= tol).all())


def test_negated_views(cga):
    """views that carry their sign as a bit (the imaginary part of a conjugate), as inputs, parameters and gradients"""
    g = gen(35)
    x, ps, dy = gated_inputs(g, 40, 24, 32, 24, True, F32)
    w, b = rnd(g, 24), rnd(g, 24)
    key = key_of(1, 2)
    one = torch.complex(rnd(g, 1, 1), rnd(g, 1, 1)).conj().imag
    assert one.is_neg() and one.is_contiguous()
    n = torch._neg_view
    for f, ts in ((lambda *t: cga.ops.channel_norm(*t), [x, w, b]), (lambda t, r: cga.ops.dropout(t, 0.25, key, r), [x, dy]),
                  (lambda *t: cga.ops.gated_feed_forward(*t), [x] + ps)):
        for i in range(len(ts)):
            a = [n(t) if k == i else t for k, t in enumerate(ts)]
            assert torch.equal(f(*a), f(*[t.resolve_neg().clone() for t in a]))
        leaves = [t.detach().clone().requires_grad_(True) for t in ts]
        for p, q in zip(torch.autograd.grad(f(*leaves), leaves, n(dy)), torch.autograd.grad(f(*leaves), leaves, -dy)):
            assert torch.equal(p, q)
    assert torch.equal(cga.ops.dropout(one, 0.0, key), one.resolve_neg())


def test_an_operand_that_moved_is_refused(cga):
    x, ps, dy = gated_inputs(gen(33), 40, 33, 47, 31, False, F16)
    leaves = [t.requires_grad_(True) for t in ps[:3]]
    y = cga.ops.gated_feed_forward(x, *leaves)
    leaves[1].data = leaves[1].detach().clone()
    with pytest.raises(RuntimeError, match="moved since"):
        y.backward(dy)


# rows, dims, shift: elements by which every operand starts off 16 bytes
HOOKED = [(F32, 20, 64, 96, 0), (F32, 70, 33, 47, 1), (F16, 20, 64, 96, 1), (F16, 70, 64, 96, 1), (BF16, 90, 64, 96, 0), (BF16, 150, 33, 47, 0)]


def shifted(t, k):
    out = torch.empty(t.numel() + 16, dtype=t.dtype, device=t.device)[k:k + t.numel()].view(t.shape)
    return out.copy_(t.detach())


def train(cga, tensors, dy, hooks):
    """a step of norm and gated block under saved-tensor hooks: y and all gradients"""
    leaves = [t.detach().requires_grad_(True) for t in tensors]
    with hooks:
        y = cga.ops.gated_feed_forward(cga.ops.channel_norm(*leaves[:3]), *leaves[3:])
    return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))


@pytest.mark.parametrize("dtype,rows,D,F,shift", HOOKED, ids=str)
def test_saved_tensors_may_come_back_elsewhere(cga, dtype, rows, D, F, shift):
    """on the host and back, and as copies on 16 bytes or off them, of any operand and of what the calls keep"""
    g = gen(50)
    x, ps, dy = gated_inputs(g, rows, D, F, 40, True, dtype)
    ts = [shifted(t, shift) for t in (x, rnd(g, D, dtype=dtype), rnd(g, D, dtype=dtype), *ps)]
    plain = torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t)
    want = train(cga, ts, dy, plain)
    for a, b in zip(want, train(cga, ts, dy, contextlib.nullcontext())):
        assert torch.equal(a, b)
    for hooks in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.save_on_cpu(pin_memory=True),
                  torch.autograd.graph.saved_tensors_hooks(lambda t: shifted(t, 1), lambda t: t),
                  torch.autograd.graph.saved_tensors_hooks(lambda t: shifted(t, 0), lambda t: t)):
        got = train(cga, ts, dy, hooks)
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_saved_images_may_come_back_in_another_layout(cga):
    g = gen(51)
    x, dy = rnd(g, 2, 24, 3, 5, dtype=F16).contiguous(memory_format=torch.channels_last), rnd(g, 2, 40, 3, 5, dtype=F16)
    ts = [x, rnd(g, 24, dtype=F16), rnd(g, 24, dtype=F16), rnd(g, 40, 24, dtype=F16), rnd(g, 40, 24, dtype=F16)]
    want = train(cga, ts, dy, torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t))
    got = train(cga, ts, dy, torch.autograd.graph.saved_tensors_hooks(lambda t: t.contiguous(), lambda t: t))
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_a_saved_tensor_that_comes_back_as_another_is_refused(cga):
    g = gen(52)
    x, ps, dy = gated_inputs(g, 40, 24, 32, 16, False, F32)
    w = rnd(g, 24)
    half = lambda t: t.half() if t.is_floating_point() else t.int()
    for f in (lambda: cga.ops.gated_feed_forward(x.requires_grad_(True), *ps), lambda: cga.ops.channel_norm(x.requires_grad_(True), w),
              lambda: cga.ops.dropout(x.requires_grad_(True), 0.5, key_of(1, 2))):
        for change in (half, lambda t: t[..., :-1]):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
                y = f()
            with pytest.raises(RuntimeError, match="came back"):
                y.sum().backward()


@pytest.mark.parametrize("dtype,rows", [(F32, 24), (F32, 500), (BF16, 500)], ids=str)
def test_checkpointed(cga, dtype, rows):
    """the same bits as without, and nothing kept but the input"""
    from torch.utils.checkpoint import checkpoint
    g = gen(53)
    D, F = 256, 1024
    x, ps, dy = gated_inputs(g, rows, D, F, D, True, dtype)
    w, b = rnd(g, D, dtype=dtype), rnd(g, D, dtype=dtype)

    def step(run):
        leaves = [t.detach().clone().requires_grad_(True) for t in [x, w, b] + ps]

        def f(t):
            return t + cga.ops.gated_feed_forward(cga.ops.channel_norm(t, *leaves[1:3]), *leaves[3:])
        gc.collect()                                    # what earlier tests left in cycles is not freed in between
        before = torch.cuda.memory_allocated()
        y = run(f, run(f, leaves[0]))
        kept = torch.cuda.memory_allocated() - before
        y.backward(dy)                                  # a reentrant checkpoint takes no autograd.grad
        return kept, [y.detach()] + [t.grad for t in leaves]
    kept0, want = step(lambda f, t: f(t))
    kept1, got = step(lambda f, t: checkpoint(f, t, use_reentrant=False))
    _, again = step(lambda f, t: checkpoint(f, t, use_reentrant=True))
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and all(torch.equal(a, b) for a, b in zip(want, again))
    hidden = rows * F * x.element_size()
    assert kept0 > 6 * hidden and kept1 <= 2 * rows * D * x.element_size() + 4096


def test_capture_beside_a_living_eager_graph_is_refused(cga):
    x, ps, dy = gated_inputs(gen(34), 40, 32, 48, 32, False, F32)
    w = torch.ones(32, device="cuda", requires_grad=True)
    leaves = [t.requires_grad_(True) for t in ps[:3]]
    ops = [lambda: cga.ops.gated_feed_forward(x, *leaves), lambda: cga.ops.channel_norm(x, w),
           lambda: cga.ops.dropout(w, 0.5, key)]
    key = key_of(1, 2)
    alive = [f() for f in ops]
    gr = torch.cuda.CUDAGraph()
    refused = []
    with torch.cuda.graph(gr):
        for f in ops:
            try:
                f()
            except RuntimeError as e:
                refused.append("eager graph of the same leaves" in str(e))
        with torch.no_grad():
            y = cga.ops.channel_norm(x, w)          # no gradient, no objection
    assert refused == [True] * 3
    gr.replay()
    assert torch.equal(y, alive[1])


def test_member_batched_refusals(cga):
    x = torch.zeros(5, 32, device="cuda")
    w = torch.ones(32, device="cuda")
    with cga.ops.members(2):
        with pytest.raises(cga.hip.HipError, match="ParamPool"):
            cga.ops.channel_norm(x, w)
        ps, _ = pooled(cga, 2, 32, 40, gen(1))
        with pytest.raises(cga.hip.HipError, match="equal blocks"):
            cga.ops.channel_norm(x, ps[0][0])
        with pytest.raises(cga.hip.HipError, match="equal blocks"):
            cga.ops.gated_feed_forward(x, *ps[0][2:])


def test_backward_passes_are_not_differentiated_again(cga):
    x, ps, dy = gated_inputs(gen(40), 6, 16, 24, 16, False, F32)
    w = torch.ones(16, device="cuda")
    for f in (lambda t: cga.ops.channel_norm(t, w), lambda t: cga.ops.dropout(t, 0.5, key_of(1, 2)),
              lambda t: cga.ops.gated_feed_forward(t, *ps)):
        xl = x.detach().requires_grad_(True)
        with pytest.raises(RuntimeError, match="cannot be differentiated again"):
            torch.autograd.grad(f(xl), xl, dy, create_graph=True)
