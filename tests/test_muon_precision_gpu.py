"""How exact the orthogonalised updates are, on every way a product takes: a block of steps in one
CTA, half tiles, whole tiles, CTA pairs, blocks on the Gram matrix, and sums of any length.

Tolerances.  Operands of 22 bits leave 2^-22 of a product's operands.  The tensor cores cut their
sums: adding 16 terms at a time of three products, a sum of at most 1024 terms is cut 192 times, each
time by at most 2^-23 of what it has grown to, on average half of that of half of the sum: 192 / 4
x 2^-23 = 6e-6 of |P| |Q| (longer sums are added up from such parts with rounding).  Five steps pass
this on about eightfold: 5e-5, and 1e-4 is asserted.  Operands that lose their second plane leave
1e-3, a sum cut 12288 times (65536 terms) 7e-4.

A 16-bit result is the fp32 one, rounded once.  Of an element off by d before the rounding, the
neighbour of the right one is taken with probability d / step, and is a step off then; the steps
are below eps of the values, so that with errors of 5e-5 of the result's norm the results are
sqrt(eps 5e-5) of it apart (6.2e-4 for bf16, 2.2e-4 for fp16), where errors of 7e-4 leave 4 times
that."""

import math

import pytest
import torch

import rational_kat_cu_b200 as kat
from rational_kat_cu_b200 import muon

pytestmark = pytest.mark.gpu
A, B, C = 3.4445, -4.7750, 2.0315


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def polar(u, steps=5):
    """The steps in 64 bits, on the m x m side."""
    x = u.double()
    if x.shape[0] > x.shape[1]:
        return polar(u.t(), steps).t()
    x = x / x.norm()
    gram, total = x @ x.t(), torch.eye(x.shape[0], device=x.device, dtype=x.dtype)
    for _ in range(steps):
        p = B * gram + C * (gram @ gram)
        p.diagonal().add_(A)
        total, gram = p @ total, p @ gram @ p
    return total @ x


def apart(got, want):
    return float((got.double() - want.double()).norm() / want.double().norm())


# a block of steps in one CTA; half tiles; whole tiles; CTA pairs; both ways of taking the steps; tall
SHAPES = [(1, 96, 160), (3, 128, 512), (1, 300, 310), (2, 300, 1100), (1, 768, 768), (3, 197, 1000),
          (3, 1024, 1280), (9, 700, 777), (12, 768, 768), (3, 1000, 2600), (2, 2600, 1000)]


@pytest.mark.parametrize("shape", SHAPES)
def test_fp32(cuda_device, shape):
    x = normal(*shape, seed=shape[1])
    out = kat.orthogonalize(x)
    for i in {0, shape[0] - 1}:
        assert apart(out[i], polar(x[i])) <= 1e-4
    assert muon.device_status() == 0


@pytest.mark.parametrize("shape", [(1, 100, 65536), (2, 128, 16384), (1, 256, 16400), (2, 256, 65536),
                                   (1, 20000, 300), (6, 700, 5000), (1, 2048, 2100),
                                   (1, 1100, 65536)])
@pytest.mark.parametrize("steps", [3, 5])
def test_long_sums(cuda_device, shape, steps):
    """Sums of more than 1024 terms, in single CTAs and pairs, several tiles to a block."""
    x = normal(*shape, seed=shape[2])
    out = kat.orthogonalize(x, steps=steps)
    for i in {0, shape[0] - 1}:
        assert apart(out[i], polar(x[i], steps)) <= 1e-4
    assert muon.device_status() == 0
    assert torch.equal(out, kat.orthogonalize(x, steps=steps))


@pytest.mark.parametrize("shape", [(12, 768, 2304), (3, 1500, 4000), (1, 4000, 4100), (2, 3000, 2050)])
def test_long_sums_in_pairs(cuda_device, shape):
    """CTA pairs: parts of the Gram matrix alone, of every product, several tiles to a pair."""
    x = normal(*shape, seed=shape[2])
    out = kat.orthogonalize(x)
    for i in {0, shape[0] - 1}:
        assert apart(out[i], polar(x[i])) <= 1e-4
    assert muon.device_status() == 0
    assert torch.equal(out, kat.orthogonalize(x))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1100, 1100), (2, 2600, 2700), (1, 3000, 1300)])
def test_long_sums_of_16_bit_weights(cuda_device, shape, dtype):
    gs = [normal(*shape[1:], seed=i, dtype=dtype) for i in range(shape[0])]
    ws = [torch.zeros_like(g) for g in gs]
    ms = [torch.zeros_like(g, dtype=torch.float32) for g in gs]
    kat.muon_step(ws, gs, ms, lr=0.5, momentum=0.5, nesterov=False)
    scale = 0.5 * 0.2 * math.sqrt(max(shape[1:]))
    for w, g in zip(ws, gs):
        assert apart(w, (-scale * polar(g)).to(dtype)) <= math.sqrt(torch.finfo(dtype).eps * 5e-5)


def test_long_sums_of_one_direction(cuda_device):
    """Rows that agree: every term of a sum has one sign."""
    x = 1 + 0.1 * normal(64, 40000)
    assert apart(kat.orthogonalize(x), polar(x)) <= 1e-4


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_16_bit_results_are_rounded_once(cuda_device, shape, dtype):
    x = normal(*shape, seed=shape[1], dtype=dtype)
    out = kat.orthogonalize(x)
    most = math.sqrt(torch.finfo(dtype).eps * 5e-5)
    for i in {0, shape[0] - 1}:
        assert apart(out[i], polar(x[i]).to(dtype)) <= most


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("steps", [1, 2, 3, 5])
def test_16_bit_weights_are_rounded_once(cuda_device, shape, dtype, steps):
    """Weights that start at zero are the update itself (lr: entries of about 0.1, normal numbers)."""
    n = shape[0]
    gs = [normal(*shape[1:], seed=i, dtype=dtype) for i in range(n)]
    ws = [torch.zeros_like(g) for g in gs]
    ms = [torch.zeros_like(g, dtype=torch.float32) for g in gs]
    kat.muon_step(ws, gs, ms, lr=0.5, momentum=0.5, nesterov=False, steps=steps)
    most = math.sqrt(torch.finfo(dtype).eps * 5e-5)
    scale = 0.5 * 0.2 * math.sqrt(max(shape[1:]))
    for i in {0, n - 1}:
        want = -scale * polar(gs[i], steps)
        assert apart(ws[i], want.to(dtype)) <= most


def test_16_bit_weights_of_a_step(cuda_device):
    """Weights of the update's own size, decayed."""
    for dtype in (torch.float16, torch.bfloat16):
        w, g = normal(256, 384, dtype=dtype) * 0.02, normal(256, 384, seed=1, dtype=dtype)
        m = normal(256, 384, seed=2)
        u = g.double() + 0.9 * (0.9 * m.double() + g.double())
        want = w.double() * (1 - 0.02 * 0.1) - 0.02 * 0.2 * math.sqrt(384) * polar(u)
        kat.muon_step([w], [g], [m], lr=0.02, momentum=0.9, weight_decay=0.1)
        assert apart(w, want.to(dtype)) <= math.sqrt(torch.finfo(dtype).eps * 5e-5)
