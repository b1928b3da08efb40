"""The modules over the channel-MLP operators on the GPU: blocks against 64 bits, dropout states, trainers with a gated style MLP."""

import pytest
import torch

import channel_mlp_ref as R
import test_gpu_graph as G

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cga():
    import council_gan_amd
    council_gan_amd.hip.load()
    return council_gan_amd


def block64(b, x):
    """GatedBlock without dropout from its parameters, in 64 bits"""
    p = {k: v.detach().double().cpu().requires_grad_(True) for k, v in b.named_parameters()}
    d = x - x.mean(-1, keepdim=True)
    n = d / (d.square().mean(-1, keepdim=True) + b.norm.eps).sqrt() * p["norm.weight"] + p["norm.bias"]
    a, v = n @ p["gate.weight"].t() + p["gate.bias"], n @ p["value.weight"].t() + p["value.bias"]
    return x + (R.gate(a, b.activation)[0] * v) @ p["out.weight"].t() + p["out.bias"], p


@pytest.mark.parametrize("rows,dim,hidden,act", [(1, 8, None, "silu"), (16, 256, None, "silu"), (33, 52, 70, "gelu"), (300, 64, 96, "sigmoid")])
def test_gated_block(cga, rows, dim, hidden, act):
    torch.manual_seed(5)
    b = cga.GatedBlock(dim, hidden, act).cuda()
    x = torch.randn(rows, dim)
    dy = torch.randn(rows, dim)
    xl = x.cuda().requires_grad_(True)
    y = b(xl)
    y.backward(dy.cuda())
    x64 = x.double().requires_grad_(True)
    y64, p64 = block64(b, x64)
    y64.backward(dy.double())
    # Three stages of the forward and six of the backward pass, each off by at most (K + 12) 2^-24 of the sum of its terms' sizes, which is
    # below sqrt(K) times the result's own size (random signs) times 4 (the largest of a few thousand results): relative to the largest value
    K = max(rows, dim, b.gate.out_features)
    tol = 9 * (K + 12) * 2.0 ** -24 * 4 * K ** 0.5
    for name, got, want in [("y", y, y64), ("dx", xl.grad, x64.grad)] + [(k, v.grad, p64[k].grad) for k, v in b.named_parameters()]:
        err = float((got.double().cpu() - want).abs().max() / want.abs().max())
        assert err <= tol, (name, err, tol)


def test_block_takes_pixels(cga):
    torch.manual_seed(6)
    b = cga.GatedBlock(16, dropout=0.3).cuda().eval()
    x = torch.randn(2, 16, 5, 7).cuda()
    rows = x.permute(0, 2, 3, 1).reshape(-1, 16)
    assert torch.equal(b(x).permute(0, 2, 3, 1).reshape(-1, 16), b(rows.contiguous()))


def test_dropout_module(cga):
    d = cga.Dropout(0.25, seed=11).cuda()
    x = torch.ones(64, 96, device="cuda")
    a, b = d(x), d(x, x)
    assert d.state.tolist() == [11, 2]
    kept = torch.tensor(65536 / (65536 - 16384))
    for y in (a, b - x):
        assert bool(((y == 0) | (y - kept.cuda()).abs().lt(1e-6)).all())
    assert not torch.equal(a, b - x)
    # a restored state draws the same masks again
    e = cga.Dropout(0.25, seed=1).cuda()
    saved = {k: v.clone() for k, v in d.state_dict().items()}
    c = d(x)
    e.load_state_dict(saved)
    assert torch.equal(e(x), c) and torch.equal(e.state, d.state)
    assert d.eval()(x) is x and d.state.tolist() == [11, 3]


def test_block_with_dropout_drops_what_it_adds(cga):
    torch.manual_seed(7)
    b = cga.GatedBlock(32, 64, dropout=0.5).cuda()
    with torch.no_grad():
        b.norm.bias.normal_()
    x = torch.randn(40, 32, device="cuda", requires_grad=True)
    dy = torch.randn_like(x)
    full = b.eval()(x) - x
    key = b.drop.state.clone()
    y = b.train()(x)
    keep = cga.ops.dropout(torch.ones_like(x), 0.5, key)
    # x + 2 (y - x): a rounding of the sum, and what the difference lost on the way
    assert bool(((y - (x + keep * full)).abs() <= 4 * 2.0 ** -24 * (y.abs() + x.abs() + 2 * full.abs())).all())
    g = torch.autograd.grad(y, x, dy)[0]
    z = b.eval()(x)
    want = torch.autograd.grad(z, x, dy * keep)[0] + dy - dy * keep
    # the same kernels on the same gradient; the residual's part joins in another order
    assert bool(((g - want).abs() <= 8 * 2.0 ** -24 * (g.abs() + dy.abs() * 4 + (g - dy).abs())).all())


def test_block_checkpointed(cga):
    from torch.utils.checkpoint import checkpoint
    torch.manual_seed(8)
    b = cga.GatedBlock(32, 64).cuda()
    x, dy = torch.randn(70, 32, device="cuda", requires_grad=True), torch.randn(70, 32, device="cuda")
    leaves = [x] + list(b.parameters())
    want = torch.autograd.grad(b(x), leaves, dy)
    got = torch.autograd.grad(checkpoint(b, x, use_reentrant=False), leaves, dy)
    assert all(torch.equal(a, c) for a, c in zip(want, got))


@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpointed_dropout_draws_no_other_mask(cga, reentrant):
    """A checkpoint runs its function again inside the backward pass: a key drawn there would be another mask than the forward pass's."""
    from torch.utils.checkpoint import checkpoint
    torch.manual_seed(9)
    b = cga.GatedBlock(32, 64, dropout=0.5).cuda()
    x, dy = torch.randn(70, 32, device="cuda", requires_grad=True), torch.randn(70, 32, device="cuda")
    with pytest.raises(cga.hip.HipError, match="another mask"):
        checkpoint(b, x, use_reentrant=reentrant).backward(dy)
    leaves = [x] + list(b.parameters())

    def step(run):
        for t in leaves:
            t.grad = None
        y = run(cga.ops.dropout_key(b.drop.state))
        y.backward(dy)
        return [y.detach()] + [t.grad for t in leaves]
    saved = b.drop.state.clone()
    want = step(lambda key: b(x, key))
    assert b.drop.state.tolist() == [int(saved[0]), int(saved[1]) + 1]
    b.drop.state.copy_(saved)
    got = step(lambda key: checkpoint(b, x, key, use_reentrant=reentrant))
    b.drop.state.copy_(saved)
    drawn = step(lambda key: b(x, key))
    assert all(torch.equal(a, c) and torch.equal(a, d) for a, c, d in zip(want, got, drawn))
    b.drop.state.copy_(saved)
    assert torch.equal(b(x), want[0])           # the key that the block draws by itself


@pytest.mark.parametrize("council,group,drop", [(2, None, 0.0), (2, None, 0.25), (2, 1, 0.25)])
def test_trainer_with_a_gated_style_mlp(cga, council, group, drop):
    """Training runs, moves the block's weights, and a captured iteration repeats the eager one's bits, masks included."""
    cfg = G._tiny("male2female_council_folder.yaml", council, 2)
    cfg["gen"].update(mlp_block="gated", mlp_dropout=drop)
    try:
        e_rows, e_w, _, _, e_cap = G._run(cga, cfg, False, 5, 64, group)
        g_rows, g_w, _, _, g_cap = G._run(cga, cfg, True, 5, 64, group)
    finally:
        cga.ops.X3_FORWARD = cga.ops.X3_BACKWARD = cga.ops.X3_DYNAMIC_INPUT = True
    assert e_cap == 0 and g_cap >= 4
    assert e_rows == g_rows
    for k in e_w:
        assert torch.equal(e_w[k], g_w[k]) and bool(torch.isfinite(e_w[k].double()).all()), k
    O = G.O
    O.seed_all(11)
    c = dict(cfg, cg_graph="0")
    first = {k: v for k, v in cga.Council_Trainer(c, "cuda:0").gen_a2b_s[0].state_dict().items()}
    block = [k for k in first if k.startswith("mlp.model.1.")]
    assert len(block) == (9 if drop else 8)
    for k in block:
        assert not torch.equal(first[k], e_w[("a2b", "gen", 0, k)]), k


def test_trainer_with_dropout_keeps_one_stream(cga, monkeypatch):
    cfg = G._tiny("male2female_council_folder.yaml", 2, 1)
    cfg["gen"].update(mlp_block="gated", mlp_dropout=0.1)
    cfg["cg_graph"] = "0"
    tr = cga.Council_Trainer(cfg, "cuda:0")
    tr.cuda("cuda:0")
    assert not tr._overlap and not tr._side
    monkeypatch.setenv("CG_OVERLAP_UPDATES", "1")
    with pytest.raises(cga.hip.HipError, match="mlp_dropout"):
        cga.Council_Trainer(cfg, "cuda:0").cuda("cuda:0")
    cga.ops.X3_FORWARD = cga.ops.X3_BACKWARD = cga.ops.X3_DYNAMIC_INPUT = True
