"""Calls of the attention-input operators around their values: forward-mode tangents, in-place use of
their results, plans made ahead and copied, tracing, and tensors with a pending negation."""

import copy
import io

import pytest
import torch
import torch.autograd.forward_ad as fwd

import rational_kat_cu_b200 as kat
from rational_kat_cu_b200 import grkan_vit as gv

pytestmark = pytest.mark.gpu


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def grid_plan():
    return kat.IndexBuckets(*kat.grid_index(3, 4, prefix=1))


@pytest.mark.parametrize("no_grad", [False, True])
@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("which", ["q", "k", "weight", "qkv", "packed weight", "distance", "index"])
def test_forward_mode_raises(cuda_device, which, requires_grad, no_grad):
    """No tangent is dropped without a word."""
    shape = {"q": (2, 3, 4, 16), "k": (2, 3, 2, 16), "weight": (16,), "packed weight": (16,),
             "qkv": (2, 3, 64), "distance": (32, 2), "index": (38, 2)}[which]
    x = normal(*shape).requires_grad_(requires_grad)
    q, k, qkv, w = (normal(2, 3, 4, 16), normal(2, 3, 2, 16), normal(2, 3, 64), normal(16))
    with fwd.dual_level(), torch.set_grad_enabled(not no_grad):
        d = fwd.make_dual(x, normal(*shape, seed=1))
        call = {"q": lambda: kat.qk_norm_rope(d, k, w, w),
                "k": lambda: kat.qk_norm_rope(q, d, w, w),
                "weight": lambda: kat.qk_norm_rope(q, k, None, d),
                "qkv": lambda: kat.qkv_norm_rope(d, 2, 1, w, w),
                "packed weight": lambda: kat.qkv_norm_rope(qkv, 2, 1, d, w),
                "distance": lambda: kat.distance_bias(d, kat.DistanceBuckets(), 5, 6),
                "index": lambda: kat.index_bias(d, grid_plan())}[which]
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


def test_forward_mode_of_gradients_raises(cuda_device):
    table, x = normal(32, 2).requires_grad_(), normal(2, 3, 64).requires_grad_()
    outs = (kat.distance_bias(table, kat.DistanceBuckets(), 5, 6), kat.qkv_norm_rope(x, 2, 1)[0])
    with fwd.dual_level():
        for out, leaf in zip(outs, (table, x)):
            up = fwd.make_dual(normal(*out.shape, seed=2), normal(*out.shape, seed=3))
            with pytest.raises((RuntimeError, NotImplementedError)):
                torch.autograd.grad(out, leaf, up)


@pytest.mark.parametrize("lk", [197, 200, 1, 8])
@pytest.mark.parametrize("kind", ["distance", "index"])
def test_results_change_in_place(cuda_device, kind, lk):
    """A mask added to or written into a bias that needs a gradient, at any length."""
    lq = 5
    if kind == "distance":
        b = kat.DistanceBuckets(8, 20)
        make = lambda t: kat.distance_bias(t, b, lq, lk)  # noqa: E731
    else:
        b = kat.IndexBuckets((torch.arange(lq)[:, None] + torch.arange(lk)) % 8, 8)
        make = lambda t: kat.index_bias(t, b)  # noqa: E731
    table = normal(8, 3).requires_grad_()
    mask = torch.rand(lq, lk, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) < 0.5
    grad = normal(3, lq, lk, seed=2)
    plain = make(table)
    want = torch.where(mask, -1.0, 2 * (plain + 1))
    want_grad, = torch.autograd.grad(want, table, grad)
    bias = make(table)
    bias += 1
    bias.mul_(2).masked_fill_(mask, -1.0)
    assert torch.equal(bias, want)
    assert torch.equal(torch.autograd.grad(bias, table, grad)[0], want_grad)
    with torch.no_grad():
        bias = make(table)
        bias[:, 0] = 3.0
    assert bias.stride(1) % 8 == 0 and (bias[:, 0] == 3).all()


def test_plans_made_for_cuda_are_ready(cuda_device):
    """device="cuda" is the current device: the first use copies nothing and may be captured."""
    b = kat.DistanceBuckets(32, 128, device="cuda")
    assert all(t.device == torch.device("cuda", 0) for t in b.on(torch.device("cuda")))
    assert b.on(torch.device("cuda"))[0] is b.on(torch.device("cuda", 0))[0]
    plan = grid_plan()
    plan.on(torch.device("cuda"))
    table, cells = normal(32, 2), normal(38, 2)
    kat.distance_bias(table, kat.DistanceBuckets(), 3, 3)      # the library is loaded
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kat.distance_bias(table, b, 40, 50), kat.index_bias(cells, plan)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], kat.distance_bias(table, b, 40, 50))
    assert torch.equal(got[1], kat.index_bias(cells, plan))


@pytest.mark.parametrize("kind", ["distance", "index"])
def test_stored_plans_hold_no_device_copies(cuda_device, kind):
    """torch.load may put a stored tensor on another device than the one it was kept for."""
    b = kat.DistanceBuckets() if kind == "distance" else grid_plan()
    dev = torch.device("cuda", 0)
    want = b.on(dev)
    buffer = io.BytesIO()
    torch.save(b, buffer)
    for where in ("cpu", None):
        buffer.seek(0)
        back = torch.load(buffer, map_location=where, weights_only=False)
        got = back.on(dev)
        assert all(t.device == dev for t in got)
        assert all(torch.equal(s, t) for s, t in zip(got, want))
    # a copied model's plans are as ready as the model's
    assert copy.deepcopy(b).on(dev)[0] is want[0]


def test_compiled_callers_go_on(cuda_device):
    """torch.compile leaves the operators out of its graphs, as it does rat_cuda."""
    torch._dynamo.reset()
    b, plan = kat.DistanceBuckets(device="cuda"), grid_plan()
    cos, sin = kat.rope_table(7, 16, device="cuda")

    def attention(x, w, table, cells):
        q, k, v = kat.qkv_norm_rope(x * 2, 2, 1, w, w, cos, sin)
        q, k = kat.qk_norm_rope(q + 1, k, w, None)
        return (q.sum() + k.sum() * v.sum() + kat.distance_bias(table, b, 7, 5).square().sum()
                + kat.index_bias(cells, plan).square().sum())

    args = [t.requires_grad_() for t in (normal(2, 7, 64), normal(16), normal(32, 2), normal(38, 2))]
    want = attention(*args)
    got = torch.compile(attention, backend="eager")(*args)
    assert torch.equal(got, want)
    for g, w in zip(torch.autograd.grad(got, args), torch.autograd.grad(want, args)):
        assert torch.equal(g, w)


def test_compiled_updates_go_on(cuda_device):
    torch._dynamo.reset()
    w, g = normal(24, 40), normal(24, 40, seed=1)
    other = w.clone()
    m, n = torch.zeros(2, 24, 40, device="cuda")

    def update(w, g, m):
        kat.muon_step([w], [g * 2], [m], lr=0.1)
        return kat.orthogonalize(g + 1) + 1

    want = update(w, g, m)
    assert torch.equal(torch.compile(update, backend="eager")(other, g, n), want)
    assert torch.equal(w, other) and torch.equal(m, n)


def test_compiled_attention_options(cuda_device):
    """The options of the attention blocks (KAT_Group itself cannot be traced: plain MLPs)."""
    torch._dynamo.reset()
    cfg = gv.ViTConfig(image_size=32, patch_size=16, num_classes=5, embed_dim=64, depth=1,
                       num_heads=2, act="gelu", qk_norm=True, rope=True, rel_pos_bias=True)
    torch.manual_seed(0)
    model = gv.GRKANViT(cfg).cuda()
    images, labels = gv.synthetic_batch(2, cfg, dtype=torch.float32, seed=1)
    images, labels = images.cuda(), labels.cuda()
    want = model(images)
    got = torch.compile(model, backend="eager")(images)
    assert torch.equal(got, want)


def test_pending_negations(cuda_device):
    """The imaginary part of a conjugate is a view whose values are still to be negated."""
    def negated(*shape, seed=0):
        z = torch.complex(normal(*shape, seed=seed), normal(*shape, seed=seed + 1))
        return z.conj().imag

    q, k, w = negated(2, 3, 4, 16), negated(2, 3, 2, 16, seed=2), negated(16, seed=4)
    assert q.is_neg()
    for got, want in zip(kat.qk_norm_rope(q, k, w.clone(), w.clone()),
                         kat.qk_norm_rope(q.resolve_neg(), k.resolve_neg(), w.resolve_neg().clone(),
                                          w.resolve_neg().clone())):
        assert torch.equal(got, want)
    x = torch._neg_view(normal(2, 3, 64))
    wn = torch._neg_view(normal(16))
    tables = [torch._neg_view(t) for t in kat.rope_table(3, 16, device="cuda")]
    for got, want in zip(kat.qkv_norm_rope(x, 2, 1, wn, wn, *tables),
                         kat.qkv_norm_rope(x.resolve_neg(), 2, 1, wn.resolve_neg(), wn.resolve_neg(),
                                           *[t.resolve_neg() for t in tables])):
        assert torch.equal(got, want)
    table, b, plan = torch._neg_view(normal(32, 2)), kat.DistanceBuckets(), grid_plan()
    assert torch.equal(kat.distance_bias(table, b, 5, 6),
                       kat.distance_bias(table.resolve_neg(), b, 5, 6))
    cells = torch._neg_view(normal(38, 2))
    assert torch.equal(kat.index_bias(cells, plan), kat.index_bias(cells.resolve_neg(), plan))
    # gradients
    leaves = [normal(32, 2).requires_grad_(), normal(38, 2).requires_grad_(),
              normal(2, 3, 64).requires_grad_()]
    outs = [kat.distance_bias(leaves[0], b, 5, 8), kat.index_bias(leaves[1], plan),
            *kat.qkv_norm_rope(leaves[2], 2, 1)]
    ups = [torch._neg_view(normal(*o.shape, seed=i)) for i, o in enumerate(outs)]
    got = torch.autograd.grad(outs, leaves, ups, retain_graph=True)
    want = torch.autograd.grad(outs, leaves, [u.resolve_neg() for u in ups])
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    # updates
    u = torch._neg_view(normal(24, 40))
    assert torch.equal(kat.orthogonalize(u), kat.orthogonalize(u.resolve_neg()))
    ws, ms = normal(2, 24, 40), torch.zeros(2, 24, 40, device="cuda")
    ws[1] = ws[0]
    kat.muon_step([ws[0]], [u], [ms[0]], lr=0.1)
    kat.muon_step([ws[1]], [u.resolve_neg()], [ms[1]], lr=0.1)
    assert torch.equal(ws[0], ws[1]) and torch.equal(ms[0], ms[1])
    for a, c in ((torch._neg_view(ws[0]), ms[0]), (ws[0], torch._neg_view(ms[0]))):
        with pytest.raises(ValueError, match="negat"):
            kat.muon_step([a], [u], [c], lr=0.1)
    with pytest.raises(ValueError, match="lr"):
        kat.muon_step([ws[0]], [u], [ms[0]], lr=torch._neg_view(torch.ones(1, device="cuda")))
