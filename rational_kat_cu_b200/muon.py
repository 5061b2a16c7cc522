"""Orthogonalised matrix updates: `orthogonalize`, `muon_step` and the `Muon` optimizer.

A momentum update of a weight matrix is replaced by its Newton-Schulz polar factor, which has
the update's singular vectors and singular values near one, so that every direction of the
matrix moves by about the same amount.  With X = u / |u|_F, `steps` times

    A = X X^T,   X <- a X + (b A + c A^2) X,   (a, b, c) = (3.4445, -4.7750, 2.0315)

on the tcgen05 kernels of libkat_rational.so (include/kat_muon.h).  Matrices of one shape and
type share their launches.  Operands are pairs of fp16 planes (22 bits) with fp32 accumulation, whatever the
matrices' type and size: after five steps the result's relative error is about 1e-5 and at most
1e-4, below any 16-bit rounding.  There is no CPU implementation: CPU tensors raise, and a missing
library raises on first use.
"""

from __future__ import annotations

import bisect
import ctypes
import math
from typing import Iterable, List, Sequence, Union

import torch
from torch import Tensor

from . import _native

DTYPES = {torch.float32: _native.KAT_DTYPE_F32, torch.float16: _native.KAT_DTYPE_F16,
          torch.bfloat16: _native.KAT_DTYPE_BF16}
MAX_MATRICES = 64
MAX_DIM = 65536
MAX_STEPS = 32
# A call's matrices are taken in runs whose workspace stays below this (or one at a time).
WORKSPACE_LIMIT = 2 << 30


def _stream(device: torch.device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _pointers(tensors: Sequence[Tensor]):
    return (ctypes.c_void_p * len(tensors))(*[t.data_ptr() for t in tensors])


def _check_steps(name: str, steps: int) -> None:
    if not isinstance(steps, int) or not 1 <= steps <= MAX_STEPS:
        raise ValueError(f"{name}: steps must be an integer in 1..{MAX_STEPS}, got {steps!r}")


def _check_matrix(name: str, what: str, t: Tensor) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name}: {what} must be a CUDA tensor; there is no CPU implementation")
    if t.dtype not in DTYPES:
        raise TypeError(f"{name}: {what} must be float32, float16 or bfloat16, got {t.dtype}")
    if t.shape[-2] > MAX_DIM or t.shape[-1] > MAX_DIM:
        raise ValueError(f"{name}: {what} must have at most {MAX_DIM} rows and columns, got "
                         f"{tuple(t.shape)}")


def _runs(count: int, rows: int, cols: int):
    """(start, length, workspace bytes) of the runs `count` matrices are taken in."""
    lib = _native.lib()
    one = lib.kat_muon_workspace_bytes(1, rows, cols)
    most = max(1, min(MAX_MATRICES, WORKSPACE_LIMIT // one))
    for start in range(0, count, most):
        n = min(most, count - start)
        yield start, n, lib.kat_muon_workspace_bytes(n, rows, cols)


@_native.untraced
@torch.no_grad()
def orthogonalize(x: Tensor, steps: int = 5) -> Tensor:
    """The Newton-Schulz polar factor of each matrix of x [..., rows, cols], in x's type.  Zero
    matrices stay zero; a matrix with a NaN or an infinity becomes NaN.  Not differentiable.
    The same call gives the same bits; a matrix alone and the same matrix among others may take
    tiles of different sizes and then differ within the error above."""
    if x.dim() < 2:
        raise ValueError(f"orthogonalize: expected [..., rows, cols], got {tuple(x.shape)}")
    _check_steps("orthogonalize", steps)
    _check_matrix("orthogonalize", "x", x)
    rows, cols = x.shape[-2:]
    out = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    if x.numel() == 0:
        return out
    src = x.detach().resolve_neg().contiguous().view(-1, rows, cols)
    dst = out.view(-1, rows, cols)
    size = rows * cols * x.element_size()
    with torch.cuda.device(x.device):
        for start, n, ws_bytes in _runs(src.shape[0], rows, cols):
            ws = torch.empty(ws_bytes, device=x.device, dtype=torch.uint8)
            xs = (ctypes.c_void_p * n)(*[src.data_ptr() + (start + i) * size for i in range(n)])
            os = (ctypes.c_void_p * n)(*[dst.data_ptr() + (start + i) * size for i in range(n)])
            st = _native.lib().kat_orthogonalize(xs, os, n, rows, cols, DTYPES[x.dtype], steps,
                                                 ws.data_ptr(), ws_bytes, _stream(x.device))
            _native.check("kat_orthogonalize", st)
    return out


def _check_step_lists(weights, grads, momenta) -> None:
    if not len(weights) == len(grads) == len(momenta):
        raise ValueError(f"muon_step: {len(weights)} weights, {len(grads)} gradients and "
                         f"{len(momenta)} momenta")
    written = []
    for w, g, m in zip(weights, grads, momenta):
        if w.dim() != 2:
            raise ValueError(f"muon_step: weights must be matrices, got shape {tuple(w.shape)}")
        _check_matrix("muon_step", "weights", w)
        if g.is_sparse or g.shape != w.shape or g.dtype != w.dtype or g.device != w.device:
            raise ValueError(f"muon_step: a gradient must be dense and have its weight's shape, "
                             f"type and device; got {tuple(g.shape)} {g.dtype} on {g.device} for "
                             f"{tuple(w.shape)} {w.dtype} on {w.device}")
        if m.shape != w.shape or m.dtype != torch.float32 or m.device != w.device:
            raise ValueError(f"muon_step: momenta must be float32 and have the weights' shapes "
                             f"and devices, got {tuple(m.shape)} {m.dtype} on {m.device}")
        if not (w.is_contiguous() and m.is_contiguous()) or w.is_neg() or m.is_neg():
            raise ValueError("muon_step: weights and momenta are updated in place and must be "
                             "contiguous, without a pending negation")
        if w.numel():
            written.append((w.data_ptr(), w.numel() * w.element_size()))
            written.append((m.data_ptr(), m.numel() * 4))
    written.sort()
    for (a, size), (b, _) in zip(written, written[1:]):
        if a + size > b:
            raise ValueError("muon_step: two of the weights and momenta share memory")
    for g in grads:
        if g.numel():
            a = g.data_ptr()
            size = (1 + sum((n - 1) * s for n, s in zip(g.shape, g.stride()))) * g.element_size()
            i = bisect.bisect_left(written, (a + size, 0))
            if i and written[i - 1][0] + written[i - 1][1] > a:
                raise ValueError("muon_step: a gradient shares memory with a weight or momentum")


@_native.untraced
@torch.no_grad()
def muon_step(weights: Sequence[Tensor], grads: Sequence[Tensor], momenta: Sequence[Tensor],
              lr: Union[float, Tensor], momentum: float = 0.95, nesterov: bool = True,
              weight_decay: float = 0.0, steps: int = 5) -> None:
    """One optimizer step of weight matrices [rows, cols], in place:

        m <- momentum m + g
        u  = g + momentum m  (nesterov)  or  m
        w <- (1 - lr weight_decay) w - lr 0.2 sqrt(max(rows, cols)) orthogonalize(u)

    Weights and gradients are float32, float16 or bfloat16, momenta float32; all arithmetic is
    fp32 or wider and a 16-bit weight is rounded once.  The factor 0.2 sqrt(max(rows, cols))
    gives the update the root mean square an AdamW step has, so one step size serves both.
    `lr` may be a float32 CUDA tensor of one element: it is then read on the device when the step
    runs, also in a replayed graph."""
    _check_steps("muon_step", steps)
    weights, grads, momenta = list(weights), list(grads), list(momenta)
    _check_step_lists(weights, grads, momenta)
    if not weights:
        return
    lr_ptr, lr_value = None, 0.0
    if isinstance(lr, Tensor):
        if lr.is_cuda:
            if lr.numel() != 1 or lr.dtype != torch.float32 or lr.is_neg():
                raise ValueError(f"muon_step: a CUDA lr must be one float32, got "
                                 f"{tuple(lr.shape)} {lr.dtype}")
            if any(w.device != lr.device for w in weights):
                raise ValueError("muon_step: a CUDA lr must be on the weights' device")
            lr_ptr = lr.data_ptr()
        else:
            lr_value = float(lr)
    else:
        lr_value = float(lr)

    groups = {}
    for i, w in enumerate(weights):
        if w.numel():
            groups.setdefault((w.device, w.dtype, tuple(w.shape)), []).append(i)
    for (device, dtype, (rows, cols)), members in groups.items():
        scale = 0.2 * math.sqrt(max(rows, cols))
        with torch.cuda.device(device):
            for start, n, ws_bytes in _runs(len(members), rows, cols):
                at = members[start:start + n]
                ws = torch.empty(ws_bytes, device=device, dtype=torch.uint8)
                gs = [grads[i].resolve_neg().contiguous() for i in at]
                st = _native.lib().kat_muon_step(
                    _pointers([weights[i] for i in at]), _pointers(gs),
                    _pointers([momenta[i] for i in at]), n, rows, cols, DTYPES[dtype], lr_value,
                    lr_ptr, momentum, int(nesterov), weight_decay, scale, steps, ws.data_ptr(),
                    ws_bytes, _stream(device))
                _native.check("kat_muon_step", st)
    torch.autograd.graph.increment_version(weights + momenta)


def device_status(device: int = 0, reset: bool = False) -> int:
    """Sticky status word of the orthogonalisation kernels (0 = no pipeline wait ran out)."""
    out = ctypes.c_int(0)
    _native.check("kat_muon_device_status",
                  _native.lib().kat_muon_device_status(device, 1 if reset else 0,
                                                       ctypes.byref(out)))
    return out.value


class Muon(torch.optim.Optimizer):
    """Optimizer of weight matrices by orthogonalised momentum (`muon_step`).  Every parameter
    is a CUDA matrix; embeddings, biases, norms and activation coefficients belong to another
    optimizer (`grkan_vit.make_optimizer(matrices="muon")` makes both)."""

    def __init__(self, params: Iterable, lr: Union[float, Tensor] = 1e-3, momentum: float = 0.95,
                 nesterov: bool = True, weight_decay: float = 0.0, steps: int = 5):
        if not isinstance(lr, Tensor) and not lr >= 0.0:
            raise ValueError(f"Muon: lr must not be negative, got {lr}")
        if not 0.0 <= momentum < 1.0:
            raise ValueError(f"Muon: momentum must be in [0, 1), got {momentum}")
        if not weight_decay >= 0.0:
            raise ValueError(f"Muon: weight_decay must not be negative, got {weight_decay}")
        _check_steps("Muon", steps)
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov,
                                      weight_decay=weight_decay, steps=steps))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() != 2:
                    raise ValueError(f"Muon: parameters must be matrices, got shape "
                                     f"{tuple(p.shape)}")

    def load_state_dict(self, state_dict) -> None:
        """As torch's, but momenta stay float32 whatever the parameters' type."""
        kept = {i: s["momentum_buffer"] for i, s in state_dict["state"].items()
                if "momentum_buffer" in s}
        super().load_state_dict(state_dict)
        order = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(order, params):
            if i in kept:
                self.state[p]["momentum_buffer"] = kept[i].to(
                    device=p.device, dtype=torch.float32).clone(
                        memory_format=torch.contiguous_format)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            params: List[Tensor] = [p for p in group["params"] if p.grad is not None]
            for p in params:
                if "momentum_buffer" not in self.state[p]:
                    if torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("Muon: the first step of a parameter cannot be captured "
                                           "(every replay would begin its momentum anew): take one "
                                           "step before")
                    self.state[p]["momentum_buffer"] = torch.zeros(
                        p.shape, device=p.device, dtype=torch.float32)
            muon_step(params, [p.grad for p in params],
                      [self.state[p]["momentum_buffer"] for p in params], lr=group["lr"],
                      momentum=group["momentum"], nesterov=group["nesterov"],
                      weight_decay=group["weight_decay"], steps=group["steps"])
        return loss
