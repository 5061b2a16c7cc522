"""Training steps with all three operators, replayed from a graph: the change of the weights, not the
weights, is what eager steps leave."""

import pytest
import torch

import rational_kat_cu_b200 as kat
from rational_kat_cu_b200 import grkan_vit as gv
from rational_kat_cu_b200 import muon
from test_vit_attention_options_gpu import make, small_cfg, strict_fp32  # noqa: F401

pytestmark = pytest.mark.gpu


def test_graphed_steps_change_what_eager_ones_change(cuda_device, strict_fp32):  # noqa: F811
    """Library kernels may add in another order: gradients differ by about 2^-22 of their norm, which
    the iteration raises by at most 3.4445^5 = 485 in an update, 1.2e-4; in eight steps that follow
    one another 1e-3.  A step that read stale momenta or gradients would change half of it or more;
    1e-2 is asserted."""
    cfg = small_cfg(embed_dim=256)
    images, labels = gv.synthetic_batch(8, cfg, dtype=torch.float32, seed=3)
    images, labels = images.cuda(), labels.cuda()
    models = [make(cfg, seed=4) for _ in range(2)]
    start = [p.detach().clone() for p in gv.block_matrices(models[0])]
    opts = [gv.make_optimizer(m, lr=1e-3, capturable=True, matrices="muon") for m in models]
    graphed = gv.GraphedTrainStep(models[0], opts[0], images, labels, warmup=3)
    for _ in range(5):
        graphed()
    torch.cuda.synchronize()
    for _ in range(8):
        gv.train_step(models[1], opts[1], images, labels)
    for a, b, old in zip(*(gv.block_matrices(m) for m in models), start):
        a, b = a.detach().double() - old, b.detach().double() - old
        assert float(b.norm()) > 0
        assert float((a - b).norm()) <= 1e-2 * float(b.norm())
    assert muon.device_status() == 0


def test_schedulers_of_the_set_s_optimizers(cuda_device):
    """torch's schedulers take each optimizer of the set; the step size reaches the next step."""
    model = make(small_cfg(), seed=1)
    opt = gv.make_optimizer(model, lr=1e-3, matrices="muon")
    schedulers = [torch.optim.lr_scheduler.LambdaLR(o, lambda step: 0.5 ** step)
                  for o in opt.optimizers]
    images, labels = gv.synthetic_batch(2, small_cfg(), dtype=torch.float32, seed=2)
    images, labels = images.cuda(), labels.cuda()
    mats, state = gv.block_matrices(model), opt.optimizers[0].state
    for k in range(3):
        assert all(abs(g["lr"] - 1e-3 * 0.5 ** k) < 1e-12 for g in opt.param_groups)
        weights = [p.detach().clone() for p in mats]
        momenta = [state[p]["momentum_buffer"].clone() if k else torch.zeros_like(p) for p in mats]
        gv.train_step(model, opt, images, labels)
        kat.muon_step(weights, [p.grad for p in mats], momenta, lr=1e-3 * 0.5 ** k, weight_decay=0.05)
        assert all(torch.equal(w, p) for w, p in zip(weights, mats))
        for s in schedulers:
            s.step()
