"""The relative position bias on the GPU.  Forward: the table's values, rounded to the output's
type, bit for bit.  Backward against sums in 64 bits: a thread adds at most 256 terms in fp32 one
after the other (256 x 2^-24 = 2^-16 of their magnitudes), all else is fp64, and the result is
rounded once (eps / 2)."""

import math

import pytest
import torch
import torch.nn.functional as F

import rational_kat_cu_b200 as kat

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).to("cuda")


def sums(grad, bucket, nb, seen=None):
    """(sums, sums of magnitudes) [nb, heads] in 64 bits."""
    g = grad.double().cpu().flatten(1)
    keep = bucket.cpu().flatten() >= 0
    if seen is not None:
        keep &= seen.cpu().flatten()
    at = bucket.cpu().flatten()[keep]
    out = torch.zeros(2, nb, grad.shape[0], dtype=torch.float64)
    out[0].index_add_(0, at, g[:, keep].t())
    out[1].index_add_(0, at, g[:, keep].t().abs())
    return out.to("cuda")


def close(got, want):
    allowed = 2.0 ** -16 * want[1] + torch.finfo(got.dtype).eps / 2 * want[0].abs() + 1e-30
    assert ((got.double() - want[0]).abs() <= allowed).all()


def check_distance(buckets, heads, lq, lk, offset=0, causal=False, dtype=torch.float32,
                   tdtype=torch.float32, grad=None):
    table = normal(buckets.num_buckets, heads, seed=3, dtype=tdtype).requires_grad_()
    out = kat.distance_bias(table, buckets, lq, lk, offset, causal, dtype)
    d = (torch.arange(lk)[None] - torch.arange(lq)[:, None] - offset).cuda()
    bucket, seen = buckets.bucket(d), d <= 0
    want = table.detach().t()[:, bucket].to(dtype)
    if causal:
        want = want.masked_fill(~seen, -math.inf)
    assert out.shape == (heads, lq, lk) and out.dtype == dtype and torch.equal(out, want)
    assert out.stride() == ((lq * out.stride(1)), (lk + 7) // 8 * 8, 1)
    # the columns that fill the rows up are zeros
    whole = out.detach().as_strided((heads, lq, out.stride(1)), out.stride())
    assert not whole[:, :, lk:].any()
    if grad is None:
        grad = normal(heads, lq, lk, seed=4, dtype=dtype)
    got = torch.autograd.grad(out, table, grad)[0]
    assert got.dtype == tdtype
    close(got, sums(grad, bucket, buckets.num_buckets, seen if causal else None))
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lq,lk,offset", [(1, 1, 0), (1, 4097, 4096), (1, 7, 3), (8, 8, 0),
                                          (9, 17, 0), (17, 9, 0), (64, 200, 136), (197, 197, 0),
                                          (333, 40, -300), (5, 1000, 2000), (300, 2, 7),
                                          (1025, 1030, -5), (3, 5, -100)])
def test_distance(cuda_device, lq, lk, offset, causal, dtype):
    check_distance(kat.DistanceBuckets(32, 128, not causal), 3, lq, lk, offset, causal, dtype)


@pytest.mark.parametrize("args", [(2, 5, False), (4, 3, True), (32, 1000, True), (64, 100, False),
                                  (8, 500, False)])
def test_distance_bucket_kinds(cuda_device, args):
    b = kat.DistanceBuckets(*args)
    for causal in (False, True):
        check_distance(b, 2, 150, 170, 10, causal, torch.bfloat16, torch.float16)


def test_long_distances_and_many_heads(cuda_device):
    b = kat.DistanceBuckets(32, 128)
    check_distance(b, 1, 2100, 2300, 0, False, torch.bfloat16)
    check_distance(b, 70, 40, 24, 0, False, torch.float16, torch.bfloat16)
    # an offset far behind every key: all in one bucket
    check_distance(b, 2, 16, 16, 2 ** 31 - 100, False)
    check_distance(b, 2, 16, 16, -(2 ** 31 - 100), True)


def test_gradients_in_any_layout(cuda_device):
    b = kat.DistanceBuckets(32, 128)
    index = kat.IndexBuckets(torch.randint(0, 9, (50, 61)), 9)
    base = normal(2, 50, 64, seed=8)
    for grad in (base[:, :, :61], base[:, :, 1:62], base.transpose(1, 2).contiguous()
                 .transpose(1, 2)[:, :, :61], base[:1, :, :61].expand(2, 50, 61),
                 normal(1, 1, 1).expand(2, 50, 61), base.bfloat16()[:, :, :61].float()):
        check_distance(b, 2, 50, 61, grad=grad)
        check_index(index, 2, grad=grad)


def test_masked_gradients_do_not_count(cuda_device):
    """NaN and infinities where a causal mask leaves nothing change no sum."""
    b = kat.DistanceBuckets(32, 128, False)
    for dtype in TYPES:
        grad = normal(2, 70, 90, seed=1, dtype=dtype)
        d = (torch.arange(90)[None] - torch.arange(70)[:, None] - 3).cuda()
        clean = check_distance(b, 2, 70, 90, 3, True, dtype, grad=grad)
        for bad in (math.nan, math.inf):
            dirty = grad.masked_fill(d > 0, bad)
            table = torch.zeros(32, 2, device="cuda", requires_grad=True)
            out = kat.distance_bias(table, b, 70, 90, 3, True, dtype)
            assert torch.equal(torch.autograd.grad(out, table, dirty)[0], clean)
    # every key of the first rows is masked: rows of -infinity
    out = kat.distance_bias(normal(32, 1), b, 4, 6, -10, True)
    assert (out == -math.inf).all()


def check_index(buckets, heads, dtype=torch.float32, tdtype=torch.float32, grad=None):
    lq, lk = buckets.shape
    nb = buckets.num_buckets
    table = normal(nb, heads, seed=3, dtype=tdtype).requires_grad_()
    out = kat.index_bias(table, buckets, dtype)
    index = buckets.on(torch.device("cuda", 0))[0][:, :lk].long()
    want = torch.cat([table.detach().to(dtype), table.new_zeros(1, heads, dtype=dtype)]).t()[
        :, index]
    assert out.shape == (heads, lq, lk) and torch.equal(out, want)
    whole = out.detach().as_strided((heads, lq, (lk + 7) // 8 * 8),
                                    (lq * ((lk + 7) // 8 * 8), (lk + 7) // 8 * 8, 1))
    assert not whole[:, :, lk:].any()
    if grad is None:
        grad = normal(heads, lq, lk, seed=4, dtype=dtype)
    got = torch.autograd.grad(out, table, grad)[0]
    assert got.dtype == tdtype
    close(got, sums(grad, torch.where(index == nb, -1, index), nb))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lq,lk,nb,heads", [(1, 1, 1, 1), (5, 9, 3, 2), (197, 197, 732, 12),
                                            (40, 33, 7, 70), (300, 70, 2, 3), (3, 16384, 5, 1),
                                            (130, 127, 40000, 2), (30, 31, 120000, 1)])
def test_index(cuda_device, lq, lk, nb, heads, dtype):
    g = torch.Generator().manual_seed(lq)
    b = kat.IndexBuckets(torch.randint(-1, nb, (lq, lk), generator=g).cuda(), nb)
    check_index(b, heads, dtype)


@pytest.mark.parametrize("rows,cols,prefix", [(1, 1, 0), (1, 9, 1), (14, 14, 1), (20, 7, 0),
                                              (32, 32, 5)])
def test_grid(cuda_device, rows, cols, prefix):
    b = kat.IndexBuckets(*kat.grid_index(rows, cols, prefix))     # made on the CPU
    check_index(b, 4, torch.bfloat16, torch.bfloat16)


def test_empty(cuda_device):
    b = kat.DistanceBuckets(8, 20)
    table = normal(8, 2).requires_grad_()
    for lq, lk in ((0, 5), (5, 0)):
        out = kat.distance_bias(table, b, lq, lk)
        assert out.shape == (2, lq, lk)
        assert not torch.autograd.grad(out.sum(), table)[0].any()
    for index in (torch.zeros(0, 4, dtype=torch.int64), torch.zeros(4, 0, dtype=torch.int64),
                  torch.full((3, 4), -1)):
        out = kat.index_bias(table, kat.IndexBuckets(index, 8))
        assert out.shape == (2, *index.shape) and not out.any()
        assert not torch.autograd.grad(out.sum(), table)[0].any()
    none = torch.zeros(8, 0, device="cuda")
    assert kat.distance_bias(none, b, 3, 4).shape == (0, 3, 4)


def test_bias_inside_attention(cuda_device):
    """The bias as the mask of scores: the table's gradient against the formula's in 64 bits and
    against differences."""
    b = kat.DistanceBuckets(16, 40)
    # leaves, as in training: torch keeps the softmax statistics for the mask's gradient only if
    # queries, keys or values have one
    q, k, v = (normal(2, 3, 37, 16, seed=i).requires_grad_() for i in range(3))
    up = normal(2, 3, 37, 16, seed=5)
    table = normal(16, 3, seed=6).requires_grad_()
    bias = kat.distance_bias(table, b, 37, 37)
    out = F.scaled_dot_product_attention(q, k, v, attn_mask=bias)
    got = torch.autograd.grad(out, table, up)[0]
    d = (torch.arange(37)[None] - torch.arange(37)[:, None]).cuda()

    def f(t):
        q64, k64, v64 = (x.detach().double() for x in (q, k, v))
        s = (q64 @ k64.transpose(-1, -2)) / 4 + t.t()[:, b.bucket(d)]
        return ((s.softmax(-1) @ v64) * up.double()).sum()

    t64 = table.detach().double().requires_grad_()
    want = torch.autograd.grad(f(t64), t64)[0]
    # scores, softmax and products in fp32 by the library: 37 x 16 terms and their sums, 2^-24 each
    size = (up.abs().sum() / up.numel() * 2 * 37 * 4).item()
    assert (got.double() - want).abs().max() <= 2.0 ** -14 * size
    e, h = normal(16, 3, seed=9).double(), 1e-5
    slope = (f(t64.detach() + h * e) - f(t64.detach() - h * e)) / (2 * h)
    assert abs(float((want * e).sum() - slope)) <= 1e-6 * float((want * e).abs().sum()) + 1e-6


def test_streams_graphs_and_repeats(cuda_device):
    d = kat.DistanceBuckets(32, 128)
    g = kat.IndexBuckets(*kat.grid_index(14, 14, 1))
    td, ti = normal(32, 4).requires_grad_(), normal(g.num_buckets, 4, seed=1).requires_grad_()
    up = normal(4, 197, 197, seed=2, dtype=torch.bfloat16)

    def work(td, ti):
        a = kat.distance_bias(td, d, 197, 197, dtype=torch.bfloat16)
        b = kat.index_bias(ti, g, dtype=torch.bfloat16)
        return (a, b, torch.autograd.grad(a, td, up)[0], torch.autograd.grad(b, ti, up)[0])

    first = [t.detach().clone() for t in work(td, ti)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = work(td, ti)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    graphs, captured = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        t1, t2 = (t.detach().clone().requires_grad_() for t in (td, ti))
        with torch.cuda.graph(graph):
            captured.append(work(t1, t2))
        graphs.append(graph)
    for _ in range(2):
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for c in captured:
            assert all(torch.equal(a, b) for a, b in zip(first, c))


def test_gradients_are_differentiated_once(cuda_device):
    table = normal(8, 2).requires_grad_()
    up = normal(2, 3, 3, seed=1).requires_grad_()
    index = torch.arange(9).view(3, 3) % 8
    for out in (kat.distance_bias(table, kat.DistanceBuckets(8, 20), 3, 3),
                kat.index_bias(table, kat.IndexBuckets(index, 8))):
        plain = torch.autograd.grad(out, table, up, retain_graph=True)[0]
        grad = torch.autograd.grad(out, table, up, create_graph=True)[0]
        assert torch.equal(grad, plain) and grad.requires_grad
        with pytest.raises(RuntimeError, match="differentiated again"):
            torch.autograd.grad(grad.sum(), up)


def test_refusals(cuda_device):
    b = kat.DistanceBuckets(8, 20)
    for table, error in ((normal(7, 2), ValueError), (normal(8, 2)[0], ValueError),
                         (normal(8, 2).double(), TypeError)):
        with pytest.raises(error):
            kat.distance_bias(table, b, 3, 3)
    for args in ((-1, 3), (3, -1), (3, 3, 1 << 31), (1 << 31, 3)):
        with pytest.raises(ValueError):
            kat.distance_bias(normal(8, 2), b, *args)
    with pytest.raises(TypeError):
        kat.distance_bias(normal(8, 2), b, 3, 3, dtype=torch.float64)
