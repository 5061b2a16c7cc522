"""The main loops of the q/k norm's and the distance bias's kernels over many turns: more heads than
a launch has groups of lanes (runs of heads, the ring's reuse, angles carried from head to head,
weight sums over several heads a thread), and more rows than a thread takes in one step (the ring
over several steps, the flush of its sums).  Tolerances are those of the operators' own tests
(test_qk_norm_rope_gpu.py: a thread adds fewer than 200 heads here; test_position_bias_gpu.py)."""

import pytest
import torch

import rational_kat_cu_b200 as kat
from test_qk_norm_rope_gpu import check

pytestmark = pytest.mark.gpu


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("B,L,Hq,Hk,dim,rot,interleaved,packed,dtype", [
    # D = 64: 28416 groups forward, 18944 backward; runs of four and, of the fewer keys, of one or two
    (7, 1999, 12, 12, 64, 64, False, True, torch.bfloat16),
    (5, 2003, 16, 3, 64, 32, True, False, torch.float16),
    (3, 3001, 13, 13, 32, 32, False, True, torch.float32),
    # D = 256 (7104 and 4736 groups), 80 (14208 and 9472, one in five idle lanes)
    (3, 1251, 9, 2, 256, 256, False, False, torch.float32),
    (2, 1777, 8, 8, 256, 64, True, True, torch.bfloat16),
    (3, 2777, 6, 5, 80, 48, False, True, torch.float16),
    # the general kernels: 3552 and 2368 warps
    (2, 1501, 5, 3, 40, 24, False, True, torch.bfloat16),
    (3, 901, 4, 4, 72, 72, True, False, torch.float32),
])
def test_heads_beyond_one_turn(cuda_device, B, L, Hq, Hk, dim, rot, interleaved, packed, dtype):
    q, k = normal(B, L, Hq, dim, dtype=dtype), normal(B, L, Hk, dim, seed=1, dtype=dtype)
    positions = torch.randint(0, 4000, (B, L), generator=torch.Generator().manual_seed(2)).cuda()
    for pos in (None, positions):
        check(q, k, 1 + 0.1 * normal(dim, seed=2), 1 + 0.1 * normal(dim, seed=3),
              kat.rope_table(4000, rot, device="cuda"), positions=pos, interleaved=interleaved,
              packed=packed)


def table_sums(grad, buckets, offset, causal):
    """(sums, sums of magnitudes) [buckets, heads] in 64 bits, diagonals first."""
    heads, lq, lk = grad.shape
    d = torch.arange(lq + lk - 1, device="cuda") - (lq - 1) - offset
    keep = d <= 0 if causal else torch.ones_like(d, dtype=torch.bool)
    out = torch.zeros(2, buckets.num_buckets, heads, device="cuda", dtype=torch.float64)
    bucket = buckets.bucket(d)
    for h in range(heads):
        # rows, the last one first, each shifted by one more place, put equal distances in a column
        g = torch.zeros(lq, lk + lq, device="cuda", dtype=torch.float64)
        g[:, :lk] = grad[h].flip(0)
        g = g.flatten()[: lq * (lk + lq - 1)].view(lq, lk + lq - 1)
        for i, rows in enumerate((g, g.abs())):
            out[i, :, h].index_add_(0, bucket[keep], rows.sum(0)[keep])
    return out


@pytest.mark.parametrize("heads,lq,lk,pad,dtype", [
    (16, 2051, 2045, 2048, torch.bfloat16),   # 16-byte rows, 8 steps a thread
    (24, 2051, 2045, 2048, torch.float32),
    (64, 8323, 521, 528, torch.bfloat16),     # 64: the flush after 32, and more steps behind it
    (64, 8323, 521, 524, torch.float32),
    (64, 2101, 521, 521, torch.float32),      # rows at any start, 512 rows a thread
    (64, 2101, 521, 523, torch.float16),
])
@pytest.mark.parametrize("causal", [False, True])
def test_rows_beyond_one_step(cuda_device, heads, lq, lk, pad, dtype, causal):
    b = kat.DistanceBuckets(32, 128, not causal)
    grad = normal(heads, lq, pad, seed=5, dtype=dtype)[:, :, :lk]
    table = torch.zeros(32, heads, device="cuda", requires_grad=True)
    offset = lk - lq if causal else -3
    out = kat.distance_bias(table, b, lq, lk, offset, causal, dtype)
    got, = torch.autograd.grad(out, table, grad)
    del out
    want = table_sums(grad, b, offset, causal)
    allowed = 2.0 ** -16 * want[1] + 2.0 ** -24 * want[0].abs() + 1e-30
    assert ((got.double() - want[0]).abs() <= allowed).all()
