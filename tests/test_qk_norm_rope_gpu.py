"""The norm of queries and keys with the rotation, on the GPU against its formula in 64 bits.

Tolerances.  The kernels work in fp32 and round once: a value may be off by half a step of its type
(eps / 2 of it) and by the fp32 errors before.  The sum of D squares adds at most 32 + 5 terms one
after the other (2^-24 each, halved by the root: 2^-19.8), rsqrt is good to 2 steps (2^-22), and a
handful of products follow: below 2^-18 of the terms' magnitudes |n_a cos| + |n_b sin|.  In the
backward the mean over D is a second such sum times two more factors: 2^-16 of
r (|dn w| + |x r| mean|dn w x r|).  The weights' gradients add each thread's terms one after the
other (at most 200 here: 2^-16.3) after those errors: 2^-15 of the sum of magnitudes."""

import pytest
import torch
import torch.utils.checkpoint

import rational_kat_cu_b200 as kat

pytestmark = pytest.mark.gpu
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}
TYPES = list(HALF)


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).to("cuda")


def halves(n, rot, interleaved):
    if interleaved:
        return n[..., 0:rot:2], n[..., 1:rot:2]
    return n[..., : rot // 2], n[..., rot // 2: rot]


def joined(a, b, rest, interleaved):
    ab = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([ab, rest], -1)


def formula(x, w, cos, sin, pos, eps, interleaved):
    """(y, magnitudes of its terms) in 64 bits; differentiable."""
    x = x.double()
    n = x * (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    if w is not None:
        n = n * w.double()
    if cos is None:
        return n, n.abs()
    rot = 2 * cos.shape[1]
    c, s = cos.double()[pos].unsqueeze(2), sin.double()[pos].unsqueeze(2)
    a, b = halves(n, rot, interleaved)
    y = joined(a * c - b * s, a * s + b * c, n[..., rot:], interleaved)
    m = joined((a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs(), n[..., rot:].abs(),
               interleaved)
    return y, m.detach()


def turned_back(dy, cos, sin, pos, interleaved):
    """Magnitudes of the terms of R^T dy."""
    dy = dy.double().abs()
    if cos is None:
        return dy
    rot = 2 * cos.shape[1]
    c, s = cos.double()[pos].unsqueeze(2).abs(), sin.double()[pos].unsqueeze(2).abs()
    a, b = halves(dy, rot, interleaved)
    return joined(a * c + b * s, a * s + b * c, dy[..., rot:], interleaved)


def within(got, want, size, share):
    off = (got.double() - want).abs()
    # below the smallest normal number the steps no longer shrink with the value: half of the last
    # one is smallest_normal eps / 2 (fp16: 2^-14 2^-11 = 2^-25)
    least = torch.finfo(got.dtype).smallest_normal
    allowed = HALF[got.dtype] * want.abs().clamp(min=least) + share * size + 1e-30
    worst = (off / allowed).max().item() if off.numel() else 0.0
    assert worst <= 1.0, worst


def check(q, k, wq, wk, table, positions=None, eps=1e-6, interleaved=False, packed=False):
    """Forward and backward of one call against the formula."""
    cos, sin = table if table is not None else (None, None)
    B, L, Hq, D = q.shape
    pos = torch.arange(L, device="cuda").expand(B, L) if positions is None else \
        positions.long().expand(B, L)
    leaves = [t.detach().clone().requires_grad_() if t is not None else None for t in (wq, wk)]
    if packed:
        v = normal(B, L, k.shape[2], D, seed=77, dtype=q.dtype)
        qkv = torch.cat([q, k, v], 2).flatten(2).requires_grad_()
        outs = kat.qkv_norm_rope(qkv, Hq, k.shape[2], *leaves, cos, sin, positions, eps,
                                 interleaved)
        assert torch.equal(outs[2], v)
        src = [qkv]
    else:
        src = [t.detach().requires_grad_() for t in (q, k)]
        outs = kat.qk_norm_rope(*src, *leaves, cos, sin, positions, eps, interleaved)
    ups = [normal(*o.shape, seed=50 + i, dtype=o.dtype) for i, o in enumerate(outs)]
    named = [t for t in src + leaves if t is not None]
    grads = dict(zip(map(id, named), torch.autograd.grad(outs, named, ups)))
    if packed:
        full = grads[id(qkv)].view(B, L, -1, D)
        dxs = full.split((Hq, k.shape[2], k.shape[2]), 2)
        assert torch.equal(dxs[2], ups[2])
    else:
        dxs = [grads[id(t)] for t in src]
    for x, w, leaf, out, up, dx in zip((q, k), (wq, wk), leaves, outs, ups, dxs):
        x64 = x.detach().double().requires_grad_()
        w64 = None if w is None else w.detach().double().requires_grad_()
        y, size = formula(x64, w64, cos, sin, pos, eps, interleaved)
        within(out, y.detach(), size, 2.0 ** -18)
        want = torch.autograd.grad(y, [x64] + ([w64] if w is not None else []), up.double())
        r = (x64.detach().pow(2).mean(-1, keepdim=True) + eps).rsqrt()
        hat = (x64.detach() * r).abs()
        dn = turned_back(up, cos, sin, pos, interleaved)
        g = dn if w is None else dn * w.double().abs()
        within(dx, want[0], r * (g + hat * (g * hat).mean(-1, keepdim=True)), 2.0 ** -16)
        if w is not None:
            within(grads[id(leaf)], want[1], (dn * hat).sum((0, 1, 2)), 2.0 ** -15)
    return outs


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(16, 16), (32, 32), (64, 64), (64, 32), (96, 96), (80, 48),
                                     (128, 128), (128, 0), (192, 64), (256, 256), (256, 16),
                                     # the general kernels
                                     (2, 2), (1, 0), (7, 4), (40, 40), (64, 6), (320, 320),
                                     (1024, 1024)])
def test_head_sizes(cuda_device, dim, rot, interleaved, dtype):
    table = kat.rope_table(9, rot, device="cuda") if rot else None
    q, k = normal(2, 5, 3, dim, dtype=dtype), normal(2, 5, 2, dim, seed=1, dtype=dtype)
    check(q, k, 1 + 0.1 * normal(dim, seed=2), 1 + 0.1 * normal(dim, seed=3), table,
          interleaved=interleaved)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("B,L,Hq,Hk", [(1, 1, 1, 1), (5, 1, 8, 2), (1, 1025, 4, 4),
                                       (2, 333, 12, 12), (33, 7, 5, 1)])
def test_lengths_and_heads(cuda_device, B, L, Hq, Hk, packed):
    for dtype, dim in ((torch.bfloat16, 64), (torch.float32, 48)):
        q = normal(B, L, Hq, dim, dtype=dtype)
        k = normal(B, L, Hk, dim, seed=1, dtype=dtype)
        check(q, k, 1 + 0.1 * normal(dim, seed=2), 1 + 0.1 * normal(dim, seed=3),
              kat.rope_table(L, dim, device="cuda"), packed=packed)


@pytest.mark.parametrize("wdtype", [None] + TYPES)
def test_weight_types(cuda_device, wdtype):
    q, k = (normal(2, 6, 2, 64, seed=i, dtype=torch.float16) for i in range(2))
    w = None if wdtype is None else (1 + 0.1 * normal(64, seed=3)).to(wdtype)
    check(q, k, w, None, kat.rope_table(6, 64, device="cuda"))
    check(q, k, None, w, None)


@pytest.mark.parametrize("offset,dim", [(0, 64), (1, 64), (8, 64), (3, 20)])
def test_strides_and_alignment(cuda_device, offset, dim):
    """Heads inside larger rows, odd starts, transposed tokens and heads, spread batches, strided
    values."""
    dtype = torch.bfloat16
    big = normal(2, 6, 4, dim + 16, dtype=dtype)[..., offset:offset + dim]
    k = normal(2, 2, 6, dim, seed=1, dtype=dtype).transpose(1, 2)
    table = kat.rope_table(6, dim, device="cuda")
    w = 1 + 0.1 * normal(dim, seed=2)
    outs = check(big, k, w, w, table)
    plain = kat.qk_norm_rope(big.contiguous(), k.contiguous(), w, w, *table)
    for a, b in zip(outs, plain):
        within(a, b.double(), b.double().abs() + 1, 2.0 ** -17)
    spread = normal(1, 6, 3, dim, seed=4, dtype=dtype).expand(2, 6, 3, dim)
    check(spread, k, w, w, table)
    apart = normal(2, 6, 3, 2 * dim, seed=5, dtype=dtype)[..., ::2]
    check(apart, k, w, w, table)


def test_upstream_gradients_in_any_layout(cuda_device):
    q, k = (normal(2, 5, 3, 64, seed=i).requires_grad_() for i in range(2))
    table = kat.rope_table(5, 64, device="cuda")
    outs = kat.qk_norm_rope(q, k, None, None, *table)
    up = normal(2, 3, 5, 64, seed=3).transpose(1, 2)
    want = torch.autograd.grad(outs, (q, k), (up.contiguous(), up.contiguous()), retain_graph=True)
    got = torch.autograd.grad(outs, (q, k), (up, up), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # a sum's gradient is one value spread over all of them
    got = torch.autograd.grad(outs[0].sum(), q, retain_graph=True)[0]
    assert torch.equal(got, torch.autograd.grad(outs[0], q, torch.ones_like(q),
                                                retain_graph=True)[0])
    # an output that is not used has a zero gradient
    assert not torch.autograd.grad(outs[0].sum(), k)[0].any()


def test_positions(cuda_device):
    table = kat.rope_table(40000, 64, device="cuda")
    q, k = normal(3, 4, 2, 64, dtype=torch.bfloat16), normal(3, 4, 1, 64, seed=1,
                                                             dtype=torch.bfloat16)
    w = 1 + 0.1 * normal(64, seed=2)
    start = torch.tensor([[39996], [0], [777]], device="cuda")
    each = start + torch.arange(4, device="cuda")
    a = check(q, k, w, w, table, each)
    check(q, k, w, w, table, each.flip(1).int(), interleaved=True)
    check(q, k, w, w, table, torch.tensor([5, 5, 5, 0], device="cuda"))   # repeated, broadcast
    # a token on its own is what it is among others
    for t in range(4):
        one = kat.qk_norm_rope(q[:, t:t + 1], k[:, t:t + 1], w, w, *table,
                               positions=each[:, t:t + 1])
        assert torch.equal(one[0], a[0][:, t:t + 1]) and torch.equal(one[1], a[1][:, t:t + 1])


@pytest.mark.parametrize("dim", [64, 40])
def test_positions_outside_the_table_are_nan(cuda_device, dim):
    table = kat.rope_table(10, dim, device="cuda")
    q, k = (normal(1, 4, 2, dim, seed=i).requires_grad_() for i in range(2))
    pos = torch.tensor([[3, 10, -1, 9]], device="cuda")
    outs = kat.qk_norm_rope(q, k, None, None, *table, positions=pos)
    grads = torch.autograd.grad(outs, (q, k), [torch.ones_like(o) for o in outs])
    for t in outs + grads:
        assert t[:, 1:3].isnan().all() and t[:, [0, 3]].isfinite().all()


def test_values_that_end_a_formula(cuda_device):
    """Zero heads, an infinity, a NaN: theirs alone."""
    for dim in (64, 40):
        x = normal(1, 4, 2, dim)
        x[0, 0, 0] = 0
        x[0, 1, 1, 5] = float("nan")
        x[0, 2, 0, 3] = float("inf")
        out = kat.qk_norm_rope(x, x, None, None, *kat.rope_table(4, dim, device="cuda"))[0]
        assert not out[0, 0, 0].any()
        assert out[0, 1, 1].isnan().all() and out[0, 2, 0].isnan().any()
        rest = torch.ones(1, 4, 2, dtype=torch.bool)
        rest[0, 1, 1] = rest[0, 2, 0] = False
        assert out[rest.cuda()].isfinite().all()


def test_empty(cuda_device):
    w = torch.ones(64, device="cuda", requires_grad=True)
    q = torch.empty(2, 0, 3, 64, device="cuda", requires_grad=True)
    outs = kat.qk_norm_rope(q, q, w, None, *kat.rope_table(0, 64, device="cuda"))
    assert outs[0].shape == q.shape
    grads = torch.autograd.grad(outs, (q, w), outs)
    assert grads[0].shape == q.shape and not grads[1].any()
    # heads on one side only, and lengths that mean nothing without them
    full, none = normal(2, 3, 4, 64).requires_grad_(), torch.empty(2, 3, 0, 64, device="cuda")
    v = torch.full((64,), 2.0, device="cuda", requires_grad=True)
    for q, k in ((full, none), (none, full)):
        torch.empty(1 << 12, device="cuda").fill_(7.0)      # what a fresh tensor may find
        out = kat.qk_norm_rope(q, k, w, v)
        got = torch.autograd.grad(out, (full, w, v), out)
        assert got[0].any() and bool(got[1].any()) != bool(got[2].any())
    endless = torch.empty(1, 1 << 32, 0, 64, device="cuda")
    assert kat.qk_norm_rope(endless, endless)[0].shape == endless.shape


def test_differences(cuda_device):
    """Gradients against differences of the formula in 64 bits along random directions."""
    dim, h = 64, 1e-5
    q, k = normal(2, 3, 2, dim), normal(2, 3, 1, dim, seed=1)
    w = 1 + 0.1 * normal(dim, seed=2)
    table = kat.rope_table(3, 48, device="cuda")
    pos = torch.arange(3, device="cuda").expand(2, 3)
    ql, wl = q.clone().requires_grad_(), w.clone().requires_grad_()
    out = kat.qk_norm_rope(ql, k, wl, None, *table)[0]
    up = normal(*out.shape, seed=4)
    dq, dw = torch.autograd.grad(out, (ql, wl), up)

    def f(x, w):
        return (formula(x, w, *table, pos, 1e-6, False)[0] * up.double()).sum()

    for seed in range(3):
        d = normal(*q.shape, seed=10 + seed).double()
        slope = (f(q.double() + h * d, w) - f(q.double() - h * d, w)) / (2 * h)
        # fp32 errors of 768 terms (2^-16 each) against the differences' h^2 and 2^-52 / h
        assert abs(float((dq.double() * d).sum() - slope)) <= 2.0 ** -16 * float(
            (dq.double() * d).abs().sum()) + 1e-6
        e = normal(dim, seed=20 + seed).double()
        slope = (f(q, w.double() + h * e) - f(q, w.double() - h * e)) / (2 * h)
        assert abs(float((dw.double() * e).sum() - slope)) <= 2.0 ** -15 * float(
            (dw.double() * e).abs().sum()) + 1e-6


def test_streams_graphs_and_repeats(cuda_device):
    """The same bits on a side stream, from run to run, and from a captured forward and backward
    replayed while an eager graph of the same leaves lives."""
    q = normal(3, 50, 4, 64, dtype=torch.bfloat16).requires_grad_()
    k = normal(3, 50, 2, 64, seed=1, dtype=torch.bfloat16).requires_grad_()
    w = (1 + 0.1 * normal(64, seed=2)).requires_grad_()
    table = kat.rope_table(50, 64, device="cuda")
    ups = [normal(3, 50, h, 64, seed=h, dtype=torch.bfloat16) for h in (4, 2)]

    def work():
        outs = kat.qk_norm_rope(q, k, w, w, *table)
        return outs + torch.autograd.grad(outs, (q, k, w), ups)

    first = [t.detach().clone() for t in work()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = work()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    alive = kat.qk_norm_rope(q.detach(), k.detach(), w.detach(), None, *table)
    graph = torch.cuda.CUDAGraph()
    ql, kl, wl = (t.detach().clone().requires_grad_() for t in (q, k, w))
    with torch.cuda.stream(side):
        outs = kat.qk_norm_rope(ql, kl, wl, wl, *table)
        torch.autograd.grad(outs, (ql, kl, wl), ups)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        outs = kat.qk_norm_rope(ql, kl, wl, wl, *table)
        captured = outs + torch.autograd.grad(outs, (ql, kl, wl), ups)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, captured))
    assert torch.equal(alive[0], first[0])


def test_gradients_are_differentiated_once(cuda_device):
    qkv = normal(2, 3, 4 * 16).requires_grad_()
    w = torch.ones(16, device="cuda", requires_grad=True)
    for outs in (kat.qkv_norm_rope(qkv, 2, 1, w, None),
                 kat.qk_norm_rope(qkv.view(2, 3, 4, 16), qkv.view(2, 3, 4, 16), None, w)):
        ups = [normal(*o.shape, seed=i) for i, o in enumerate(outs)]
        plain = torch.autograd.grad(outs, (qkv, w), ups, retain_graph=True)
        grads = torch.autograd.grad(outs, (qkv, w), ups, create_graph=True)
        for a, b in zip(grads, plain):
            assert torch.equal(a, b) and a.requires_grad
            with pytest.raises(RuntimeError, match="differentiated again"):
                torch.autograd.grad(a.sum(), qkv, retain_graph=True)


def test_views_and_frozen_inputs(cuda_device):
    """Values are a view of the projection's output; weights alone, or inputs alone, may train."""
    qkv = normal(2, 3, 3 * 32)
    w = torch.ones(32, device="cuda", requires_grad=True)
    q, k, v = kat.qkv_norm_rope(qkv, 1, 1, w, w)
    assert v.data_ptr() == qkv.data_ptr() + 2 * 32 * 4 and not kat.qkv_norm_rope(qkv, 1, 1)[0].requires_grad
    both = torch.autograd.grad((q, k), w, (q.detach(), k.detach()))[0]
    assert both.isfinite().all()
    with torch.no_grad():
        assert not kat.qkv_norm_rope(qkv, 1, 1, w, w)[0].requires_grad
    x = qkv.clone().requires_grad_()
    q, k, v = kat.qkv_norm_rope(x, 1, 1, w.detach(), None)
    dv = torch.autograd.grad(v, x, torch.ones_like(v))[0]       # of the values alone
    assert not dv[..., :64].any() and (dv[..., 64:] == 1).all()


def test_recomputed_moved_and_overwritten_inputs(cuda_device):
    """Saved tensors may be recomputed or kept elsewhere; one that was written over is refused."""
    x = normal(2, 5, 3 * 64).requires_grad_()
    w = torch.ones(64, device="cuda", requires_grad=True)

    def f(x):
        return kat.qkv_norm_rope(x, 1, 1, w, w)[0]

    want = torch.autograd.grad(f(x).square().sum(), (x, w))
    again = torch.utils.checkpoint.checkpoint(f, x, use_reentrant=False)
    with torch.autograd.graph.save_on_cpu():
        moved = f(x)
    for out in (again, moved):
        got = torch.autograd.grad(out.square().sum(), (x, w))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    y = x.clone()
    out = f(y)
    y.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    with pytest.raises(RuntimeError, match="view"):
        kat.qkv_norm_rope(x.clone(), 1, 1, w, w)[2].mul_(2.0)


def test_refusals(cuda_device):
    q = normal(1, 2, 3, 64)
    for k, error in ((q.half(), TypeError), (q[..., :32], ValueError), (q[:, :1], ValueError),
                     (q.cpu(), RuntimeError), (q[0], ValueError)):
        with pytest.raises(error):
            kat.qk_norm_rope(q, k)
    with pytest.raises(TypeError):
        kat.qk_norm_rope(q.double(), q.double())
    with pytest.raises(ValueError):
        kat.qk_norm_rope(q, q, None, None, *kat.rope_table(1, 64, device="cuda"))
    with pytest.raises(ValueError):
        kat.qk_norm_rope(q, q, None, None, *kat.rope_table(2, 64))
    for args in ((0, 1), (1, 0), (1, 3)):
        with pytest.raises(ValueError):
            kat.qkv_norm_rope(normal(1, 2, 64 * 3), *args)
