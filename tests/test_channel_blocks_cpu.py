"""The modules over the channel-MLP operators (ChannelNorm, Dropout, GatedBlock, the gated MLP) without a GPU."""
import copy
import os

import pytest
import torch
import yaml

import council_gan_amd as cga

CONFIGS = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "configs")


def config(**gen):
    cfg = yaml.safe_load(open(os.path.join(CONFIGS, "male2female_council_folder.yaml")))
    cfg["gen"].update(dim=16, mlp_dim=32, n_res=2)
    cfg["gen"].update(gen)
    cfg["dis"].update(dim=16)
    cfg["council"]["council_size"] = 2
    return cfg


def test_the_linear_mlp_is_the_default():
    torch.manual_seed(3)
    a = cga.AdaINGen(3, config()["gen"], cuda_device="cpu")
    torch.manual_seed(3)
    b = cga.AdaINGen(3, config(mlp_block="linear", mlp_dropout=0.0)["gen"], cuda_device="cpu")
    sa, sb = a.state_dict(), b.state_dict()
    assert list(sa) == list(sb) and all(torch.equal(sa[k], sb[k]) for k in sa)
    assert [k for k in sa if k.startswith("mlp.")] == ["mlp.model.%d.fc.%s" % (i, n) for i in range(3) for n in ("weight", "bias")]


def test_gated_mlp_layout():
    m = cga.MLP(8, 20, 32, 4, block="gated", dropout=0.1)
    shapes = {k: tuple(v.shape) for k, v in m.state_dict().items()}
    for i in (1, 2):
        pre = "model.%d." % i
        assert shapes[pre + "norm.weight"] == shapes[pre + "norm.bias"] == shapes[pre + "out.bias"] == (32,)
        assert shapes[pre + "gate.weight"] == shapes[pre + "value.weight"] == (128, 32) and shapes[pre + "out.weight"] == (32, 128)
        assert shapes[pre + "gate.bias"] == shapes[pre + "value.bias"] == (128,) and shapes[pre + "drop.state"] == (2,)
    assert shapes["model.3.fc.weight"] == (20, 32)
    assert not any("state" in k for k in cga.MLP(8, 20, 32, 4, block="gated").state_dict())      # no dropout, no state


@pytest.mark.parametrize("call,words", [
    (lambda: cga.MLP(8, 20, 32, 3, block="dense"), "MLP block"),
    (lambda: cga.MLP(8, 20, 32, 3, dropout=0.5), "without gated"),
    (lambda: cga.GatedBlock(8, activation="relu"), "activation"),
], ids=["block", "dropout_linear", "activation"])
def test_unsupported(call, words):
    with pytest.raises(NotImplementedError, match=words):
        call()


@pytest.mark.parametrize("p", [1.0, -0.1, float("nan")])
def test_dropout_refuses(p):
    with pytest.raises(ValueError, match="p must be"):
        cga.Dropout(p)


def test_dropout_off_and_its_state():
    x = torch.randn(3, 8)
    assert cga.Dropout()(x) is x and torch.equal(cga.Dropout()(x, x), x + x)
    d = cga.Dropout(0.5, seed=7).eval()
    assert d(x) is x and d.state.tolist() == [7, 0]
    torch.manual_seed(1)
    a, b = cga.Dropout(0.5), cga.Dropout(0.5)
    torch.manual_seed(1)
    assert torch.equal(a.state, cga.Dropout(0.5).state) and not torch.equal(a.state, b.state)
    with pytest.raises(cga.hip.HipError):           # training is a kernel's work
        d.train()(x)


def test_trainer_takes_the_gated_mlp():
    cfg = config(mlp_block="gated", mlp_dropout=0.25)
    tr = cga.Council_Trainer(copy.deepcopy(cfg), "cuda:0")
    gen = tr.gen_a2b_s[0]
    assert isinstance(gen.mlp.model[1], cga.GatedBlock) and gen.mlp.model[1].drop.p == 0.25
    assert any(p is gen.mlp.model[1].gate.weight for g in tr.gen_opt_s[0].param_groups for p in g["params"])
    # replicas of a member draw different masks, the first one those of the checkpoint
    state = gen.mlp.model[1].drop.state
    first = state.clone()
    tr._replica_masks(gen)
    assert torch.equal(state, first)
    tr.shard.slice_idx = 3
    tr._replica_masks(gen)
    assert state.tolist() == [int(first[0]) + 3, 0]
