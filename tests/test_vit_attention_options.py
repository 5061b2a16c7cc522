"""The ViT's attention options and the matrices' optimizer on the CPU: configuration, parameters,
which optimizer takes what, and what is refused."""

import pytest
import torch

import rational_kat_cu_b200 as kat
from rational_kat_cu_b200 import grkan_vit as gv


def tiny_cfg(**kw):
    base = dict(image_size=32, patch_size=16, num_classes=10, embed_dim=64, depth=2,
                num_heads=2, num_groups=4)
    base.update(kw)
    return gv.ViTConfig(**base)


def test_options_are_off_by_default():
    plain = gv.GRKANViT(tiny_cfg(), kat_device="cpu")
    names = {n for n, _ in plain.named_parameters()}
    full = gv.GRKANViT(tiny_cfg(qk_norm=True, rope=True, rel_pos_bias=True), kat_device="cpu")
    more = {n for n, _ in full.named_parameters()} - names
    assert names < {n for n, _ in full.named_parameters()}
    assert {n.split(".", 2)[2] for n in more} == {"attn.norm_rope.q_weight",
                                                  "attn.norm_rope.k_weight",
                                                  "attn.pos_bias.table"}
    attn = full.blocks[0].attn
    assert attn.norm_rope.cos.shape == (5, 16) and torch.equal(attn.norm_rope.cos[0],
                                                               torch.ones(16))
    assert attn.pos_bias.table.shape == (3 * 3 + 3, 2)
    # the state of a model without them loads as before, and tables are no part of any state
    plain.load_state_dict(gv.GRKANViT(tiny_cfg(), kat_device="cpu").state_dict())
    assert not any(n.endswith((".cos", ".sin")) for n in full.state_dict())


def test_rope_needs_the_norm():
    with pytest.raises(ValueError, match="qk_norm"):
        gv.GRKANViT(tiny_cfg(rope=True), kat_device="cpu")
    model = gv.GRKANViT(tiny_cfg(qk_norm=True), kat_device="cpu")
    assert model.blocks[0].attn.norm_rope.cos is None
    with pytest.raises(RuntimeError, match="CUDA"):
        model(torch.zeros(1, 3, 32, 32))


def test_optimizers_share_the_parameters():
    model = gv.GRKANViT(tiny_cfg(qk_norm=True, rel_pos_bias=True), kat_device="cpu")
    assert isinstance(gv.make_optimizer(model), torch.optim.AdamW)
    opt = gv.make_optimizer(model, lr=0.01, matrices="muon")
    muon, adamw = opt.optimizers
    assert isinstance(muon, kat.Muon) and isinstance(adamw, torch.optim.AdamW)
    mine = [p for g in muon.param_groups for p in g["params"]]
    assert len(mine) == 4 * 2
    assert {id(p) for p in mine} == {id(m.weight) for b in model.blocks for m in
                                     (b.attn.qkv, b.attn.proj, b.mlp.fc1, b.mlp.fc2)}
    both = [id(p) for g in opt.param_groups for p in g["params"]]
    assert len(both) == len(set(both)) == len(list(model.parameters()))
    with pytest.raises(ValueError, match="matrices"):
        gv.make_optimizer(model, matrices="sgd")
    state = opt.state_dict()
    opt.load_state_dict(state)
    with pytest.raises(ValueError, match="optimizers"):
        opt.load_state_dict({"optimizers": state["optimizers"][:1]})
    for p in model.parameters():
        p.grad = torch.ones_like(p)
    opt.zero_grad()
    assert all(p.grad is None for p in model.parameters())


def test_tables_survive_a_start_on_the_meta_device():
    cfg = tiny_cfg(qk_norm=True, rope=True, rel_pos_bias=True)
    want = gv.GRKANViT(cfg, kat_device="cpu").blocks[1].attn
    with torch.device("meta"):
        model = gv.GRKANViT(cfg, kat_device="cpu")
        buckets = kat.DistanceBuckets(8, 20)
    attn = model.to_empty(device="cpu").blocks[1].attn
    assert torch.equal(attn.norm_rope.cos, want.norm_rope.cos)
    assert torch.equal(attn.norm_rope.sin, want.norm_rope.sin)
    for a, b in zip(attn.pos_bias.buckets.on(torch.device("cpu")),
                    want.pos_bias.buckets.on(torch.device("cpu"))):
        assert torch.equal(a, b)
    assert torch.equal(buckets._of, kat.DistanceBuckets(8, 20)._of)
