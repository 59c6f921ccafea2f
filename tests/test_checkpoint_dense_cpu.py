"""Checkpoints of models that hold the dense modules beside the packed ones: saved, restored into the dense skeleton, saved again."""
import json

import pytest
import torch
import torch.nn as nn

import dartmoq_b200 as D
from dartmoq_b200 import checkpoint as ckpt
from dartmoq_b200 import synth

H, I = 256, 384


class Mlp(nn.Module):
    def __init__(self, act=None):
        super().__init__()
        self.gate_proj, self.up_proj = nn.Linear(H, I, bias=False), nn.Linear(H, I, bias=False)
        self.down_proj = nn.Linear(I, H, bias=False)
        self.act_fn = act if act is not None else nn.SiLU()


def skeleton(act=None):
    mlp = nn.Module()
    mlp.gate = synth.SyntheticRouter(H, 4, 2, 6, torch.bfloat16, None)
    mlp.shared_expert = Mlp(act)
    mlp.shared_expert_gate = nn.Linear(H, 1, bias=False)
    layer = nn.Module()
    layer.mlp, layer.dense_mlp = mlp, Mlp(act)
    layer.attn = nn.Module()
    layer.attn.q_proj, layer.attn.o_proj = nn.Linear(H, 33, bias=True), nn.Linear(64, H, bias=False)
    model = nn.Module()
    model.layers = nn.ModuleList([layer])
    return model


def w8(n, k, bias=None):
    g = torch.Generator().manual_seed(n + k)
    return D.W8A8Linear(torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8), torch.rand(n, generator=g),
                        None if bias is None else torch.rand(n, generator=g).to(bias))


def model_with_dense_modules():
    model = skeleton()
    layer = model.layers[0]
    moe = synth.build_layer(hidden=H, n_experts=4, top_k=2, inter=128, bit_mix={2: 0.5, 4: 0.5}, seed=5)
    moe.shared_expert = D.W8A8GatedFeedForward(w8(I, H), w8(I, H), w8(H, I))
    moe.shared_expert_gate = nn.Linear(H, 1, bias=False, dtype=torch.bfloat16)
    layer.mlp = moe
    layer.dense_mlp = D.GatedFeedForward(H, I)
    layer.attn.q_proj, layer.attn.o_proj = w8(33, H, torch.float16), w8(H, 64)
    return model


@pytest.mark.parametrize("prefix", (None, ("layers", "inner.layers")))
def test_dense_modules_are_saved_and_restored(tmp_path, prefix):
    model = model_with_dense_modules()
    ckpt.save_quantized_model(model, str(tmp_path / "a"))
    meta = json.load(open(tmp_path / "a" / "meta.json"))
    kinds = {p: m["type"] for p, m in meta["modules"].items()}
    assert kinds["layers.0.mlp.shared_expert"] == "w8a8_gated_ffn" and kinds["layers.0.dense_mlp"] == "gated_ffn"
    assert kinds["layers.0.attn.q_proj"] == kinds["layers.0.mlp.shared_expert.up_proj"] == "w8a8_linear"
    again = skeleton()
    root = again
    if prefix:
        root = nn.Module()
        root.inner = again
    ckpt.load_quantized_layers(root, str(tmp_path / "a"), prefix)
    layer = again.layers[0]
    assert type(layer.mlp) is D.WxA16BitPartitionedGroupMoE and type(layer.mlp.shared_expert) is D.W8A8GatedFeedForward
    assert type(layer.dense_mlp) is D.GatedFeedForward and (layer.dense_mlp.hidden_size, layer.dense_mlp.intermediate_size) == (H, I)
    assert type(layer.attn.q_proj) is D.W8A8Linear and layer.attn.q_proj.bias.dtype == torch.float16
    assert layer.attn.o_proj.bias is None
    want, got = model.state_dict(), again.state_dict()
    assert set(want) == set(got)
    for k, v in want.items():
        assert got[k].dtype == v.dtype and torch.equal(got[k], v), k
    ckpt.save_quantized_model(again, str(tmp_path / "b"))
    twice = json.load(open(tmp_path / "b" / "meta.json"))
    assert twice["modules"] == meta["modules"] and twice["layers"] == meta["layers"]


@pytest.mark.parametrize("eight_bit", (False, True))
def test_a_block_is_not_restored_into_one_that_computes_something_else(tmp_path, eight_bit):
    model = model_with_dense_modules()
    if eight_bit:
        model.layers[0].dense_mlp = Mlp()
    else:
        model.layers[0].mlp.shared_expert = Mlp()
    ckpt.save_quantized_model(model, str(tmp_path))
    with pytest.raises(ValueError, match="act_fn"):
        ckpt.load_quantized_layers(skeleton(nn.GELU()), str(tmp_path))
