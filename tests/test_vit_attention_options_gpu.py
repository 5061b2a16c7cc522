"""The three operators together, as the ViT uses them: heads normalised and rotated, the learned bias
in the scores, and the blocks' matrices updated by orthogonalised momentum; forward, gradients and
update against a plain model in 64 bits."""

import copy
import math

import pytest
import torch
import torch.nn.functional as F

from oracle import kat_torch_oracle
from rational_kat_cu_b200 import grkan_vit as gv
from rational_kat_cu_b200 import muon

pytestmark = pytest.mark.gpu
A, B, C = 3.4445, -4.7750, 2.0315


def small_cfg(**kw):
    base = dict(image_size=64, patch_size=16, num_classes=10, embed_dim=128, depth=2,
                num_heads=4, num_groups=8, qk_norm=True, rope=True, rel_pos_bias=True)
    base.update(kw)
    return gv.ViTConfig(**base)


def make(cfg, dtype=torch.float32, seed=0):
    torch.manual_seed(seed)
    model = gv.GRKANViT(cfg)
    with torch.no_grad():   # away from the starting point, where biases and angles could hide
        for n, p in model.named_parameters():
            if n.endswith("table"):
                p.normal_(0, 0.5)
            elif "norm_rope" in n:
                p.add_(0.2 * torch.randn_like(p))
    return model.to("cuda", dtype)


def plain_attention(attn, cos, sin, index):
    """The same attention from elementary operations, in its weights' type."""
    def forward(x):
        b, n, c = x.shape
        h, d = attn.num_heads, c // attn.num_heads
        q, k, v = attn.qkv(x).view(b, n, 3, h, d).unbind(2)
        turned = []
        for t, w in ((q, attn.norm_rope.q_weight), (k, attn.norm_rope.k_weight)):
            t = t / (t.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w
            if cos is not None:
                first, second = t[..., : d // 2], t[..., d // 2:]
                cc, ss = cos[:, None].to(t), sin[:, None].to(t)
                t = torch.cat([first * cc - second * ss, first * ss + second * cc], -1)
            turned.append(t.transpose(1, 2))
        scores = turned[0] @ turned[1].transpose(-1, -2) / math.sqrt(d)
        if index is not None:
            scores = scores + attn.pos_bias.table.t()[:, index]
        out = scores.softmax(-1) @ v.transpose(1, 2)
        return attn.proj(out.transpose(1, 2).reshape(b, n, c))
    return forward


def plain_model(model, dtype):
    ref = copy.deepcopy(model)
    tables = [(b.attn.norm_rope.cos, b.attn.norm_rope.sin) for b in model.blocks]
    ref = ref.to(dtype)
    for m in ref.kat_modules():
        m.rational = kat_torch_oracle.rational_1dgroup
    for block, (cos, sin) in zip(ref.blocks, tables):
        a = block.attn
        index = None
        if a.pos_bias is not None:
            n = ref.cfg.num_tokens
            index = a.pos_bias.buckets.on(torch.device("cuda", 0))[0][:, :n].long()
        a.forward = plain_attention(a, cos, sin, index)
    return ref


def step(model, images, labels):
    logits = model(images)
    F.cross_entropy(logits, labels).backward()
    return {"logits": logits.detach(), **{n: p.grad for n, p in model.named_parameters()}}


@pytest.fixture
def strict_fp32():
    old = (torch.backends.cuda.matmul.allow_tf32, torch.backends.cudnn.allow_tf32)
    torch.backends.cuda.matmul.allow_tf32 = torch.backends.cudnn.allow_tf32 = False
    yield
    torch.backends.cuda.matmul.allow_tf32, torch.backends.cudnn.allow_tf32 = old


@pytest.mark.parametrize("rope", [True, False])
@pytest.mark.parametrize("rel_pos_bias", [True, False])
def test_step_against_64_bits(cuda_device, strict_fp32, rope, rel_pos_bias):
    """Logits and all gradients: the model's error against 64 bits is of the size of the plain model's
    in 32 bits, whose roundings are as many (a factor of 8 between two orders of them)."""
    cfg = small_cfg(rope=rope, rel_pos_bias=rel_pos_bias)
    model = make(cfg)
    images, labels = gv.synthetic_batch(3, cfg, dtype=torch.float32, seed=1)
    images, labels = images.cuda(), labels.cuda()
    exact = step(plain_model(model, torch.float64), images.double(), labels)
    plain = step(plain_model(model, torch.float32), images, labels)
    got = step(model, images, labels)
    assert set(got) == set(exact)
    for n, want in exact.items():
        size = float(want.norm())
        floor = 2.0 ** -20 * size + 1e-9
        assert float((got[n].double() - want).norm()) <= 8 * float(
            (plain[n].double() - want).norm()) + floor, n


def test_muon_updates_the_matrices(cuda_device, strict_fp32):
    cfg = small_cfg()
    model = make(cfg)
    opt = gv.make_optimizer(model, lr=0.01, weight_decay=0.1, matrices="muon")
    images, labels = gv.synthetic_batch(4, cfg, dtype=torch.float32, seed=2)
    images, labels = images.cuda(), labels.cuda()
    mats = gv.block_matrices(model)
    before = [p.detach().clone() for p in mats]
    gv.train_step(model, opt, images, labels)
    for p, old in zip(mats, before):
        g = p.grad.double()
        u = g + 0.95 * g            # nesterov, the momentum begins at zero
        x = u if u.shape[0] <= u.shape[1] else u.t()
        x = x / x.norm()
        for _ in range(5):
            a = x @ x.t()
            x = A * x + (B * a + C * (a @ a)) @ x
        o = x if u.shape[0] <= u.shape[1] else x.t()
        want = old.double() * (1 - 0.01 * 0.1) - 0.01 * 0.2 * max(old.shape) ** 0.5 * o
        # the update's relative error is below 1e-4 (see the orthogonalisation's own tests), the
        # weight's rounding 2^-24, thrice
        moved = float((want - old.double()).norm())
        assert moved > 0
        assert float((p.detach().double() - want).norm()) <= 1e-4 * moved + 2.0 ** -22 * float(want.norm())
    assert muon.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_graphed_steps_equal_eager_ones(cuda_device, dtype):
    """Five steps replayed from a graph leave the weights five eager ones leave, bit for bit."""
    cfg = small_cfg(embed_dim=256, fused_gemm=dtype == torch.bfloat16)
    images, labels = gv.synthetic_batch(8, cfg, dtype=dtype, seed=3)
    images, labels = images.cuda(), labels.cuda()
    models = [make(cfg, dtype, seed=4) for _ in range(2)]
    opts = [gv.make_optimizer(m, lr=1e-3, capturable=True, matrices="muon") for m in models]
    graphed = gv.GraphedTrainStep(models[0], opts[0], images, labels, warmup=3)
    for _ in range(5):
        loss = graphed()
    torch.cuda.synchronize()
    for _ in range(8):
        eager = gv.train_step(models[1], opts[1], images, labels)
    assert torch.isfinite(loss) and torch.isfinite(eager)
    for (n, a), (_, b) in zip(models[0].named_parameters(), models[1].named_parameters()):
        # attention's and the convolution's library kernels may add in another order from run to run
        a, b = a.detach().double(), b.detach().double()
        assert float((a - b).norm()) <= 1e-2 * float(b.norm()) + 1e-6, n


def test_optimizer_state_round_trip(cuda_device):
    cfg = small_cfg()
    images, labels = gv.synthetic_batch(2, cfg, dtype=torch.float32, seed=5)
    images, labels = images.cuda(), labels.cuda()
    a, b = make(cfg, seed=6), make(cfg, seed=6)
    oa = gv.make_optimizer(a, lr=1e-3, matrices="muon")
    ob = gv.make_optimizer(b, lr=1e-3, matrices="muon")
    gv.train_step(a, oa, images, labels)
    b.load_state_dict(a.state_dict())
    ob.load_state_dict(oa.state_dict())
    ma, mb = oa.optimizers[0], ob.optimizers[0]
    for p, q in zip(gv.block_matrices(a), gv.block_matrices(b)):
        q.grad = p.grad.clone()
        assert torch.equal(ma.state[p]["momentum_buffer"], mb.state[q]["momentum_buffer"])
    ma.step()
    mb.step()
    for p, q in zip(gv.block_matrices(a), gv.block_matrices(b)):
        assert torch.equal(p, q)
