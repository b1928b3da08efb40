"""The channel-MLP operators without a GPU: their refusals, and the references of their GPU tests against autograd in 64 bits."""
import ctypes

import pytest
import torch

import channel_mlp_ref as R
import council_gan_amd as cga
from council_gan_amd import hip, ops


def t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


KEY = torch.zeros(2, dtype=torch.int64)
NO_DEVICE = -2              # CG_ERR_LAUNCH: what the check behind a backward pass says where there is no GPU
WIDE = (1 << 29) + 1        # twice as many columns of sums no longer fit 31 bits with a step past their end
REFUSED = [
    ("norm_int", lambda: ops.channel_norm(t(2, 4, dtype=torch.int32), t(4)), "float32, float16 or bfloat16"),
    ("norm_double", lambda: ops.channel_norm(t(2, 4, dtype=torch.float64), t(4)), "float32, float16 or bfloat16"),
    ("norm_scalar", lambda: ops.channel_norm(torch.tensor(1.0), t(1)), "channel dimension"),
    ("norm_no_channels", lambda: ops.channel_norm(t(2, 0), t(0)), "at least one channel"),
    ("norm_width", lambda: ops.channel_norm(t(2, 4), t(5)), "weight must be"),
    ("norm_image_width", lambda: ops.channel_norm(t(2, 4, 3, 5), t(5)), "weight must be"),
    ("norm_weight_type", lambda: ops.channel_norm(t(2, 4), t(4, dtype=torch.float16)), "weight is"),
    ("norm_bias_width", lambda: ops.channel_norm(t(2, 4), t(4), t(3)), "bias must be"),
    ("norm_bias_type", lambda: ops.channel_norm(t(2, 4, dtype=torch.float16), t(4), t(4, dtype=torch.float16)), "bias is"),
    ("norm_eps", lambda: ops.channel_norm(t(2, 4), t(4), None, -1.0), "eps"),
    ("norm_eps_nan", lambda: ops.channel_norm(t(2, 4), t(4), None, float("nan")), "eps"),
    ("norm_wide", lambda: ops.channel_norm(t(0, WIDE), t(1).expand(WIDE)), "at most 2\\^29"),
    ("drop_p_one", lambda: ops.dropout(t(4), 1.0, KEY), "p must be"),
    ("drop_p_negative", lambda: ops.dropout(t(4), -0.1, KEY), "p must be"),
    ("drop_p_nan", lambda: ops.dropout(t(4), float("nan"), KEY), "p must be"),
    ("drop_p_tiny", lambda: ops.dropout(t(4), 1e-7, KEY), "closer to 0"),
    ("drop_p_near_one", lambda: ops.dropout(t(4), 1 - 1e-7, KEY), "closer to 1"),
    ("drop_type", lambda: ops.dropout(t(4, dtype=torch.int64), 0.5, KEY), "float32, float16 or bfloat16"),
    ("drop_residual_shape", lambda: ops.dropout(t(4, 2), 0.5, KEY, residual=t(2)), "residual"),
    ("drop_residual_type", lambda: ops.dropout(t(4), 0.5, KEY, residual=t(4, dtype=torch.float16)), "residual"),
    ("key_type", lambda: ops.dropout_key(t(2)), "two contiguous int64"),
    ("key_size", lambda: ops.dropout_key(torch.zeros(3, dtype=torch.int64)), "two contiguous int64"),
    ("gated_act", lambda: ops.gated_feed_forward(t(2, 4), t(6, 4), t(6, 4), act="relu"), "act must be"),
    ("gated_dim", lambda: ops.gated_feed_forward(t(2, 4), t(6), t(6, 4)), "w_gate must be"),
    ("gated_width", lambda: ops.gated_feed_forward(t(2, 4), t(6, 5), t(6, 5)), "w_gate must be"),
    ("gated_value", lambda: ops.gated_feed_forward(t(2, 4), t(6, 4), t(5, 4)), "w_value must be"),
    ("gated_no_value", lambda: ops.gated_feed_forward(t(2, 4), t(6, 4), None), "w_value must be"),
    ("gated_out", lambda: ops.gated_feed_forward(t(2, 4), t(6, 4), t(6, 4), t(4, 5)), "w_out must be"),
    ("gated_bias", lambda: ops.gated_feed_forward(t(2, 4), t(6, 4), t(6, 4), b_gate=t(4)), "b_gate must be"),
    ("gated_bias_out", lambda: ops.gated_feed_forward(t(2, 4), t(6, 4), t(6, 4), b_out=t(4)), "b_out without w_out"),
    ("gated_mixed", lambda: ops.gated_feed_forward(t(2, 4, dtype=torch.bfloat16), t(6, 4), t(6, 4)), "w_gate is"),
    ("gated_wide", lambda: ops.gated_feed_forward(t(0, (1 << 21) + 1), t(1, (1 << 21) + 1), t(1, (1 << 21) + 1)), "at most 2"),
    ("gated_empty", lambda: ops.gated_feed_forward(t(2, 4), t(0, 4), t(0, 4)), "at least 1"),
]


@pytest.mark.parametrize("case", REFUSED, ids=[c[0] for c in REFUSED])
def test_refused(case):
    with pytest.raises(ValueError, match=case[2]):
        case[1]()


def test_no_cpu_fallback():
    for call in (lambda: ops.channel_norm(t(2, 4), t(4)), lambda: ops.dropout(t(4), 0.5, KEY), lambda: ops.dropout_key(KEY),
                 lambda: ops.gated_feed_forward(t(2, 4), t(6, 4), t(6, 4))):
        with pytest.raises(hip.HipError, match="no CPU fallback"):
            call()


@pytest.mark.parametrize("call", [
    lambda d: ops.channel_norm(d(2, 4), t(4)), lambda d: ops.channel_norm(t(2, 4), d(4)), lambda d: ops.channel_norm(t(2, 4), t(4), d(4)),
    lambda d: ops.dropout(d(2, 4), 0.5, KEY), lambda d: ops.dropout(t(2, 4), 0.5, KEY, residual=d(2, 4)),
    lambda d: ops.gated_feed_forward(d(2, 4), t(6, 4), t(6, 4)), lambda d: ops.gated_feed_forward(t(2, 4), t(6, 4), d(6, 4)),
    lambda d: ops.gated_feed_forward(t(2, 4), t(6, 4), t(6, 4), d(3, 6)),
    lambda d: ops.gated_feed_forward(t(2, 4), t(6, 4), t(6, 4), t(3, 6), b_out=d(3))],
    ids=["norm_x", "norm_w", "norm_b", "drop_x", "drop_residual", "gated_x", "gated_value", "gated_out", "gated_bias"])
def test_forward_mode_tangents_are_refused(call):
    """none is lost in silence; the refusal comes before the one of the device"""
    import torch.autograd.forward_ad as fw
    with fw.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(lambda *s: fw.make_dual(torch.zeros(*s), torch.ones(*s)))


def test_members_past_the_end_of_the_pool_are_refused():
    """a batched call reads and writes n members' parameters from its own on: all of them must be there"""
    from council_gan_amd.optim import FlatAdam, ParamPool
    ps = [[torch.nn.Parameter(torch.zeros(s)) for s in ((4,), (4,), (6, 4), (6, 4), (3, 6))] for _ in range(2)]
    ParamPool([FlatAdam(p) for p in ps]).materialize("cpu")
    a, b = ps
    calls = [lambda p, q: ops.channel_norm(t(6, 4), p[0], q[1]), lambda p, q: ops.gated_feed_forward(t(6, 4), p[2], p[3], q[4])]
    for f in calls:
        with ops.members(3), pytest.raises(hip.HipError, match="pool of 2"):
            f(a, a)
        with ops.members(2), pytest.raises(hip.HipError, match="pool of 2"):
            f(b, b)
        with ops.members(2), pytest.raises(hip.HipError, match="one member"):
            f(a, b)
        with ops.members(2), pytest.raises(hip.HipError, match="no CPU fallback"):
            f(a, a)


def test_library_refuses_bad_arguments_before_any_launch():
    lib = hip.load()
    p = ctypes.c_void_p(256)
    assert lib.cg_channel_norm_fwd(None, None, p, None, p, None, None, 4, 8, 0, 0, 1e-5, None) == -1
    assert lib.cg_channel_norm_fwd(None, p, p, None, p, None, None, 4, 0, 0, 0, 1e-5, None) == -1
    assert lib.cg_channel_norm_fwd(None, p, p, None, p, None, None, 4, 8, 0, 1, 1e-5, None) == -1       # fp16 weight of an fp32 row
    assert lib.cg_channel_norm_fwd(None, p, p, None, p, p, None, 4, 8, 0, 0, 1e-5, None) == -1          # mean without rstd
    assert lib.cg_channel_norm_bwd(None, p, p, p, p, p, p, p, p, 0, 4096, 8, 0, 0, p, 8, None) == -3       # workspace
    assert lib.cg_channel_norm_bwd(ctypes.byref(hip.Group(3, 0, 32)), p, p, p, p, p, p, p, p, 0, 4, 8, 0, 0, p, 1 << 20, None) == -1
    assert lib.cg_dropout(p, None, p, 4, 65536, p, 0, None) == -1
    assert lib.cg_dropout(p, None, p, 4, 1, p, 3, None) == -1
    assert lib.cg_dropout_key(p, p, None) == -1
    d = hip.GatedDims(4, 8, 16, 8, 1, 0, 0)
    args = [p] * 12
    assert lib.cg_gated_ff_fwd(ctypes.byref(hip.GatedDims(4, 8, 16, 8, 1, 3, 0)), None, *args, 0, None) == -1
    assert lib.cg_gated_ff_fwd(ctypes.byref(d), ctypes.byref(hip.Group(2, 0, 32)), *args, 0, None) == -1   # members hold fp32
    assert lib.cg_gated_ff_fwd(ctypes.byref(d), None, p, p, p, None, None, None, None, p, p, p, None, None, 0, None) == -1
    assert lib.cg_gated_ff_bwd(ctypes.byref(d), None, *([p] * 14), 0, p, p, 0, None) == -3
    assert b"workspace" in lib.cg_last_error()
    off = ctypes.c_void_p(264)                      # h, kept, pack and the workspace are on 16 bytes
    for i in (7, 8, 10, 11):
        assert lib.cg_gated_ff_fwd(ctypes.byref(d), None, *(off if k == i else p for k in range(12)), 1 << 30, None) == -1
    for i in (5, 6, 14, 15):
        a = [off if k == i else p for k in range(16)]
        assert lib.cg_gated_ff_bwd(ctypes.byref(d), None, *a[:14], 0, *a[14:], 1 << 30, None) == -1
    odd = hip.GatedDims(64, 9, 16, 8, 1, 0, 0)      # rows of 9 halves do not start on 16 bytes: the copies need memory
    assert lib.cg_gated_ff_pack_bytes(ctypes.byref(odd), None, p, p, p, p) >= (64 + 2 * 16) * 16 * 2
    assert lib.cg_gated_ff_fwd(ctypes.byref(odd), None, p, p, p, p, None, None, None, p, p, p, None, p, 1 << 30, None) == -3
    assert lib.cg_gated_ff_pack_bytes(ctypes.byref(hip.GatedDims(64, 8, 16, 8, 1, 0, 0)), None, p, p, p, p) == 0
    assert lib.cg_gated_ff_pack_bytes(ctypes.byref(hip.GatedDims(64, 8, 16, 8, 1, 0, 0)), None, ctypes.c_void_p(258), p, p, p) > 0


def test_library_refuses_rows_past_31_bits():
    """no rows and no gradients: nothing is launched, whatever the answer"""
    lib = hip.load()
    p = ctypes.c_void_p(256)
    for C, rc in ((WIDE - 1, 0), (WIDE, -1), ((1 << 31) - 1, -1)):
        assert lib.cg_channel_norm_fwd(None, p, p, None, p, None, None, 0, C, 0, 0, 1e-5, None) == rc
        assert lib.cg_channel_norm_bwd(None, p, p, p, p, p, None, None, None, 0, 0, C, 0, 0, p, 1 << 40, None) in (rc, rc or NO_DEVICE)
        assert (lib.cg_channel_norm_bwd_workspace(None, 1, C, 0) == 0) == (rc != 0)


def test_workspaces_of_any_size_are_finite():
    lib = hip.load()
    for rows in (0, 1, 7, 4096, 10 ** 7):
        for dt in (0, 1, 2):
            for n in (1, 3) if dt == 0 else (1,):
                if rows % n:
                    continue
                d, grp = ctypes.byref(hip.GatedDims(rows, 264, 520, 72, dt, 0, 0)), ctypes.byref(hip.Group(n, 0, 1 << 20))
                assert lib.cg_gated_ff_fwd_workspace(d, grp) < 1 << 33
                hidden = rows * 520 * (4 if dt == 0 else 2)
                assert 2 * hidden <= lib.cg_gated_ff_bwd_workspace(d, grp) < 2 * hidden + rows * 144 + (1 << 33)
        assert lib.cg_channel_norm_bwd_workspace(None, rows, 264, 0) < 1 << 33


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
def test_reference_of_the_gated_block_against_autograd(act):
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    x, wg, wv, wo, bg, bv, bo, dy = r(5, 4), r(6, 4), r(6, 4), r(3, 6), r(6), r(6), r(3), r(5, 3)
    ls = [v.requires_grad_(True) for v in (x, wg, wv, wo, bg, bv, bo)]
    f = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "sigmoid": torch.sigmoid}[act]
    y = (f(x @ wg.t() + bg) * (x @ wv.t() + bv)) @ wo.t() + bo
    want = dict(zip(("dx", "dwg", "dwv", "dwo", "dbg", "dbv", "dbo"), torch.autograd.grad(y, ls, dy)), y=y)
    got = R.gated_ref(*[v.detach() for v in ls], act, dy)
    for k, v in want.items():
        torch.testing.assert_close(got[k][0], v.detach(), rtol=1e-12, atol=1e-12)


def test_reference_of_the_norm_against_autograd():
    g = torch.Generator().manual_seed(2)
    x, w, b, dy = (torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_(True) for s in ((5, 7), (7,), (7,), (5, 7)))
    y = torch.nn.functional.layer_norm(x, (7,), w, b, 1e-5)
    want = dict(zip(("dx", "dw", "db"), torch.autograd.grad(y, (x, w, b), dy.detach())), y=y)
    got = R.norm_ref(x.detach(), w.detach(), b.detach(), 1e-5, dy.detach())
    for k, v in want.items():
        torch.testing.assert_close(got[k][0], v.detach(), rtol=1e-12, atol=1e-12)


def test_reference_draw_against_the_published_vectors():
    """Philox4x32-10 of counter 0 under key 0: 6627e8d5 e169c58d bc57ac4c 9b00dbd8 (the known-answer vectors of Salmon et al.)"""
    words = (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)
    draws = [h for w in words for h in (w & 0xffff, w >> 16)]
    for d in sorted(draws):
        p = d / 65536
        assert R.keep_mask(8, p, 0, 0).tolist() == [v >= d for v in draws]
