"""Orthogonalised updates on the GPU against the iteration in 64 bits.

Tolerance.  One step maps singular values by p(s) = a s + b s^3 + c s^5, and the change of its
result by a change of its input is at most L = max(|p'|, |p(s)/s|) = 3.9 on [0, 1.21].  A step's own
error is at most (|a| + 2 |b| s^2 + 3 |c| s^4) u |X|_F < 30 u |X|_F (s <= 1.21), u being the
error of one product relative to its operands' Frobenius norms: 2^-22 from the two planes of each
operand and sqrt(K) 2^-23 from adding K terms in fp32 (rounding or cutting).  So the result is within
30 u sum_j L^j |X_(steps - j)|_F of the exact one, plus half a step of the output's type.  Wide and
small matrices (2 n >= 3 m, or m <= 128) take blocks of steps on their Gram matrix, with at most three
times the products a step, each with the same error: 90 instead of 30.  The last step of a bf16 result
and the last two of a 16-bit weight take single planes: u = 2^-11 from two operands of 11 bits."""

import math

import pytest
import torch

import rational_kat_cu_b200 as kat
from rational_kat_cu_b200 import muon

pytestmark = pytest.mark.gpu

A, B, C = 3.4445, -4.7750, 2.0315
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}


def reference(u, steps=5, late=0):
    """(result, error allowed for it before rounding) of a matrix in 64 bits."""
    x = u.double()
    flip = x.shape[0] > x.shape[1]
    x = x.t() if flip else x
    norm = x.norm()
    x = x / norm if norm > 0 else x
    sums = math.sqrt(x.shape[1]) * 2.0 ** -23
    share = 90 if 2 * x.shape[1] >= 3 * x.shape[0] or x.shape[0] <= 128 else 30
    allowed = 0.0
    for step in range(steps):
        a = x @ x.t()
        unit = sums + 2.0 ** (-11 if steps - step <= late else -22)
        allowed = 3.9 * allowed + share * unit * float(x.norm())
        x = A * x + (B * a + C * (a @ a)) @ x
    return (x.t() if flip else x), allowed


LATE = {torch.float32: 0, torch.float16: 0, torch.bfloat16: 1}


def assert_close(got, want, allowed, dtype):
    assert got.dtype == dtype
    off = float((got.double() - want).norm())
    assert off <= allowed + HALF[dtype] * float(want.norm()) + 1e-30, (off, allowed)


def normal(*shape, seed=0, dtype=torch.float32, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).to(device)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1), (1, 9), (7, 1), (8, 8), (33, 65), (128, 128),
                                   (129, 127), (64, 520), (520, 64), (200, 333), (384, 1000)])
def test_sizes(cuda_device, shape, dtype):
    x = normal(*shape, dtype=dtype, seed=shape[0])
    before = x.clone()
    want, allowed = reference(x, late=LATE[dtype])
    assert_close(kat.orthogonalize(x), want, allowed, dtype)
    assert torch.equal(x, before) and muon.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(3, 1024, 1280), (3, 1000, 2600), (2, 2600, 1000),
                                   (9, 700, 777)])
def test_tiles_beyond_one_wave(cuda_device, shape, dtype):
    """More tiles than SMs: blocks take several tiles and both accumulators, CTA pairs the large
    tiles, square and wide, with edges inside a pair's tile."""
    x = normal(*shape, seed=5, dtype=dtype)
    out = kat.orthogonalize(x)
    for i in range(shape[0]):
        want, allowed = reference(x[i], late=LATE[dtype])
        assert_close(out[i], want, allowed, dtype)
    assert muon.device_status() == 0


def test_spread_singular_values(cuda_device):
    """Singular values 1 / k, where steps on the Gram matrix lose digits first."""
    for shape in ((160, 200), (160, 480)):
        u, _, v = torch.linalg.svd(normal(*shape).double(), full_matrices=False)
        x = ((u / torch.arange(1, 161, device="cuda")) @ v).float()
        want, allowed = reference(x)
        assert_close(kat.orthogonalize(x), want, allowed, torch.float32)


@pytest.mark.parametrize("shape", [(96, 130), (96, 160), (300, 1100)])
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps(cuda_device, steps, shape, dtype):
    x = normal(*shape, dtype=dtype)
    want, allowed = reference(x, steps, LATE[dtype])
    assert_close(kat.orthogonalize(x, steps=steps), want, allowed, dtype)


@pytest.mark.parametrize("count,m,n", [(1, 130, 140), (1, 250, 900), (2, 300, 310), (5, 128, 256),
                                       (9, 200, 70), (30, 64, 64), (1, 768, 768)])
def test_few_tiles(cuda_device, count, m, n):
    """Fewer tiles than SMs; a block of steps in one CTA, and products of their own."""
    x = normal(count, m, n, seed=m)
    out = kat.orthogonalize(x)
    for i in range(count):
        want, allowed = reference(x[i])
        assert_close(out[i], want, allowed, torch.float32)
    assert muon.device_status() == 0


def test_error_is_small(cuda_device):
    """Far below the bounds above: 1e-4 of fp32 results, 3e-3 of bf16 ones with their rounding."""
    for shape in ((300, 400), (256, 1000)):
        x = normal(*shape)
        want, _ = reference(x)
        assert float((kat.orthogonalize(x).double() - want).norm() / want.norm()) < 1e-4
        x = x.bfloat16()
        want, _ = reference(x)
        assert float((kat.orthogonalize(x).double() - want).norm() / want.norm()) < 3e-3


def test_batches_and_strides(cuda_device):
    x = normal(2, 3, 40, 72, seed=1)
    out = kat.orthogonalize(x)
    assert out.shape == x.shape
    for i in range(2):
        for j in range(3):
            assert torch.equal(out[i, j], kat.orthogonalize(x[i, j]))
    # transposed and strided inputs are the same matrices
    assert torch.equal(kat.orthogonalize(x.transpose(-1, -2).contiguous().transpose(-1, -2)), out)
    wide = normal(40, 144, seed=2)
    assert torch.equal(kat.orthogonalize(wide[:, ::2]),
                       kat.orthogonalize(wide[:, ::2].contiguous()))
    assert kat.orthogonalize(x[:0]).shape == (0, 3, 40, 72)
    assert kat.orthogonalize(torch.empty(3, 0, 5, device="cuda")).shape == (3, 0, 5)
    # more matrices than a call takes
    many = normal(70, 16, 24, seed=3)
    out = kat.orthogonalize(many)
    assert torch.equal(out[69], kat.orthogonalize(many[69]))


def test_zero_tiny_huge_and_bad_values(cuda_device):
    assert not kat.orthogonalize(torch.zeros(2, 20, 30, device="cuda")).any()
    x = normal(50, 70)
    base = kat.orthogonalize(x)
    # a power of two does not change the normalised update: same bits
    for e in (-100, 100):
        assert torch.equal(kat.orthogonalize(x * 2.0 ** e), base)
    for bad in (float("nan"), float("inf"), -float("inf")):
        y = torch.stack([x, x])
        y[1, 3, 5] = bad
        out = kat.orthogonalize(y)
        assert torch.equal(out[0], base) and out[1].isnan().all()


def test_low_rank(cuda_device):
    x = normal(100, 4) @ normal(4, 200, seed=1)
    want, allowed = reference(x)
    assert_close(kat.orthogonalize(x), want, allowed, torch.float32)
    one = torch.zeros(64, 64, device="cuda")
    one[3, 60] = -2.0
    want, allowed = reference(one)
    assert_close(kat.orthogonalize(one), want, allowed, torch.float32)


def step_reference(w, g, m, lr, mu, nesterov, wd, steps=5):
    m = mu * m.double() + g.double()
    u = g.double() + mu * m if nesterov else m
    o, allowed = reference(u, steps, late=0 if w.dtype == torch.float32 else 2)
    s = 0.2 * math.sqrt(max(w.shape))
    return w.double() * (1 - lr * wd) - lr * s * o, m, lr * s * allowed


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("nesterov", [True, False])
def test_step(cuda_device, dtype, nesterov):
    shapes = [(40, 72), (72, 40), (40, 72), (13, 9), (128, 256)]
    ws = [normal(*s, seed=i, dtype=dtype) for i, s in enumerate(shapes)]
    gs = [normal(*s, seed=10 + i, dtype=dtype) for i, s in enumerate(shapes)]
    gs[2] = gs[2].t().contiguous().t()           # not contiguous
    ms = [normal(*s, seed=20 + i) for i, s in enumerate(shapes)]
    lr, mu, wd = 0.02, 0.9, 0.1
    want = [step_reference(w, g, m, lr, mu, nesterov, wd) for w, g, m in zip(ws, gs, ms)]
    kat.muon_step(ws, gs, ms, lr=lr, momentum=mu, nesterov=nesterov, weight_decay=wd)
    for w, m, (rw, rm, allowed) in zip(ws, ms, want):
        # m: one product and one sum of fp32; w: the same twice over before its rounding
        assert (m.double() - rm).abs().max() <= 2.0 ** -23 * (rm.abs().max() + 5)
        assert_close(w, rw, allowed + 2.0 ** -22 * float(rw.norm()), dtype)


def test_step_refusals_leave_everything(cuda_device):
    w, g, m = normal(8, 8), normal(8, 8, seed=1), normal(8, 8, seed=2)
    before = w.clone(), m.clone()
    half = torch.zeros(8, 8, device="cuda", dtype=torch.float16)
    for ws, gs, ms in (([w, w], [g, g], [m, m.clone()]), ([w], [g], [w]), ([w], [half], [m]),
                       ([w], [g], [half]), ([w.t()[:, :7]], [g[:, :7]], [m[:, :7]]),
                       ([w], [g[:4]], [m]), ([w], [g.to_sparse()], [m]), ([w], [m], [m]),
                       ([w], [w], [m])):
        with pytest.raises((ValueError, TypeError)):
            kat.muon_step(ws, gs, ms, lr=0.1)
    for lr in (torch.zeros(2, device="cuda"), torch.zeros(1, device="cuda").half()):
        with pytest.raises(ValueError, match="lr"):
            kat.muon_step([w], [g], [m], lr=lr)
    assert torch.equal(w, before[0]) and torch.equal(m, before[1])


def test_version_counter(cuda_device):
    w = normal(8, 8).requires_grad_()
    y = (w * w).sum()
    kat.muon_step([w.detach()], [normal(8, 8)], [torch.zeros(8, 8, device="cuda")], lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_optimizer_streams_and_graph(cuda_device):
    """A captured step with the step size on the device, replayed next to an eager one and beside
    a second captured graph; a step on a side stream."""
    def fresh():
        p = torch.nn.Parameter(normal(96, 64, seed=4))
        p.grad = normal(96, 64, seed=5)
        return p

    a, b, c, d = (fresh() for _ in range(4))
    lr = torch.tensor(0.05, device="cuda")
    opts = [kat.Muon([p], lr=lr, weight_decay=0.01) for p in (a, b, c)]
    opts.append(kat.Muon([d], lr=0.05, weight_decay=0.01))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for o in opts:
            o.step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for p in (b, c, d):
        assert torch.equal(a, p)
    graphs = []
    for o in opts[1:3]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o.step()
        graphs.append(graph)
    assert torch.equal(a, b)        # capturing ran nothing
    for value in (0.05, 0.01):
        lr.fill_(value)
        opts[3].param_groups[0]["lr"] = value
        opts[0].step()
        graphs[0].replay()
        graphs[1].replay()
        opts[3].step()
        torch.cuda.synchronize()
        for p in (b, c, d):
            assert torch.equal(a, p)


def test_first_step_is_not_captured(cuda_device):
    """A captured first step would set the momentum to zero on every replay."""
    p = torch.nn.Parameter(normal(16, 16))
    p.grad = normal(16, 16, seed=1)
    opt = kat.Muon([p], lr=0.1)
    kat.muon_step([], [], [], lr=0.1)
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    torch.cuda.synchronize()
    before = p.detach().clone()
    opt.step()
    assert not torch.equal(p, before)


def test_alone_and_in_a_batch(cuda_device):
    """Together the matrices take the large tiles, alone the small ones.  A diagonal tile holds both
    halves of a symmetric product, p_i q_j + p_i q_j' + p_i' q_j added in that order; beyond the
    diagonal tiles the upper half is read from the lower, where the last two come in the other
    order.  So the bits differ; each result is within its bound, and the two within their sum."""
    for shape, dtype in (((12, 768, 768), torch.float32), ((9, 500, 1700), torch.bfloat16)):
        x = normal(*shape, seed=3, dtype=dtype)
        out = kat.orthogonalize(x)
        for i in (0, shape[0] - 1):
            want, allowed = reference(x[i], late=LATE[dtype])
            alone = kat.orthogonalize(x[i])
            assert_close(alone, want, allowed, dtype)
            assert_close(out[i], want, allowed, dtype)
            most = 2 * (allowed + HALF[dtype] * float(want.norm()))
            assert float((alone.double() - out[i].double()).norm()) <= most


def test_repeatable(cuda_device):
    x = normal(4, 300, 700, seed=9)
    first = kat.orthogonalize(x)
    for _ in range(5):
        assert torch.equal(kat.orthogonalize(x), first)
