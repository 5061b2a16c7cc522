"""Norm of queries and keys for each head with the position rotation, in one pass.

Every head's vector x [D] of a token becomes n = x w / sqrt(mean(x^2) + eps), and the pairs of
its first `rot_dim` values are turned by their angles:
(y_a, y_b) = (n_a cos - n_b sin, n_a sin + n_b cos).  Pairs are (i, i + rot_dim / 2), or
(2i, 2i + 1) with `interleaved`.  Forward and backward run on the sm_100a kernels of
libkat_rational.so (include/kat_qk_norm_rope.h), called by the torch operators of libkat_torch.so
(csrc/kat_torch.cpp): a head is read once and written once, and queries and keys share a launch.  Arithmetic is fp32; outputs are rounded once.

  qk_norm_rope    queries [B, L, Hq, D] and keys [B, L, Hk, D], any strides
  qkv_norm_rope   one projection's output [B, L, (Hq + 2 Hk) D]; its gradient is written whole,
                  the values' part included, by the same kernel
  rope_table, rope_grid_table   cos and sin of the angles, computed in 64 bits

A gradient cannot be differentiated again (it raises).  There is no CPU implementation: CPU tensors
raise, and a missing library raises on first use.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn as nn
from torch import Tensor

from . import _native

DTYPES = {torch.float32: _native.KAT_DTYPE_F32, torch.float16: _native.KAT_DTYPE_F16,
          torch.bfloat16: _native.KAT_DTYPE_BF16}
MAX_HEAD_DIM = 1024


def rope_table(length: int, rot_dim: int, base: float = 10000.0,
               device=None) -> Tuple[Tensor, Tensor]:
    """cos and sin [length, rot_dim / 2] (fp32) of position p and pair i: the angle is
    p base^(-2 i / rot_dim), taken in 64 bits, so far positions keep theirs."""
    if length < 0 or rot_dim < 0 or rot_dim % 2:
        raise ValueError(f"rope_table: need length >= 0 and an even rot_dim >= 0, got {length} "
                         f"and {rot_dim}")
    return _turns(torch.arange(length, dtype=torch.float64, device=device), rot_dim // 2, base)


def _turns(position: Tensor, pairs: int, base: float) -> Tuple[Tensor, Tensor]:
    step = torch.arange(pairs, dtype=torch.float64, device=position.device) / max(pairs, 1)
    angle = position[:, None] * base ** -step
    return angle.cos().float(), angle.sin().float()


def rope_grid_table(rows: int, cols: int, rot_dim: int, prefix: int = 0, base: float = 100.0,
                    device=None) -> Tuple[Tensor, Tensor]:
    """cos and sin [prefix + rows * cols, rot_dim / 2] for tokens that are a grid's patches, row
    by row, behind `prefix` tokens without a place (angle zero): the first half of the pairs turns
    by the patch's row, the second half by its column."""
    if rows < 0 or cols < 0 or prefix < 0 or rot_dim < 0 or rot_dim % 4:
        raise ValueError(f"rope_grid_table: need rows, cols, prefix >= 0 and rot_dim a multiple "
                         f"of 4, got {rows}, {cols}, {prefix} and {rot_dim}")
    y = torch.arange(rows, dtype=torch.float64, device=device).repeat_interleave(cols)
    x = torch.arange(cols, dtype=torch.float64, device=device).repeat(rows)
    place = torch.zeros(prefix, dtype=torch.float64, device=device)
    tables = [_turns(torch.cat([place, p]), rot_dim // 4, base) for p in (y, x)]
    return (torch.cat([tables[0][0], tables[1][0]], 1),
            torch.cat([tables[0][1], tables[1][1]], 1))


# The torch operators check their arguments.  What they refuse, or positions that are to be spread
# first, comes here for an error that says what is wrong.

def _check_rest(name: str, x: Tensor, head_dim: int, q_weight, k_weight, cos, sin, positions):
    """Checks what both functions share; returns positions as the kernels read them."""
    if x.dtype not in DTYPES:
        raise TypeError(f"{name}: queries and keys must be float32, float16 or bfloat16, got "
                        f"{x.dtype}")
    if not 1 <= head_dim <= MAX_HEAD_DIM:
        raise ValueError(f"{name}: head size must be 1..{MAX_HEAD_DIM}, got {head_dim}")
    for what, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None:
            continue
        if w.dtype not in DTYPES:
            raise TypeError(f"{name}: {what} must be float32, float16 or bfloat16, got {w.dtype}")
        if tuple(w.shape) != (head_dim,) or w.device != x.device or not w.is_contiguous():
            raise ValueError(f"{name}: {what} must be a contiguous [{head_dim}] on {x.device}, "
                             f"got {tuple(w.shape)} on {w.device}")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise TypeError(f"{name}: q_weight and k_weight have types {q_weight.dtype} and "
                        f"{k_weight.dtype}")
    if (cos is None) != (sin is None):
        raise ValueError(f"{name}: cos and sin come together")
    if cos is None:
        if positions is not None:
            raise ValueError(f"{name}: positions without a table")
        return None
    for what, t in (("cos", cos), ("sin", sin)):
        if t.dtype != torch.float32:
            raise TypeError(f"{name}: {what} must be float32, got {t.dtype}")
        if t.requires_grad:
            raise ValueError(f"{name}: {what} gets no gradient and must not require one")
        if t.dim() != 2 or t.device != x.device or not t.is_contiguous():
            raise ValueError(f"{name}: {what} must be a contiguous [rows, rot_dim / 2] on "
                             f"{x.device}, got {tuple(t.shape)} on {t.device}")
    if cos.shape != sin.shape:
        raise ValueError(f"{name}: cos {tuple(cos.shape)} and sin {tuple(sin.shape)} differ")
    if 2 * cos.shape[1] > head_dim:
        raise ValueError(f"{name}: a table of {cos.shape[1]} angles turns {2 * cos.shape[1]} "
                         f"values, a head has {head_dim}")
    B, L = x.shape[:2]
    if positions is None:
        if cos.shape[0] < L:
            raise ValueError(f"{name}: {L} tokens, and a table of {cos.shape[0]} rows")
        return None
    if positions.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{name}: positions must be int64 or int32, got {positions.dtype}")
    if positions.device != x.device:
        raise ValueError(f"{name}: positions must be on {x.device}, got {positions.device}")
    if positions.shape == (B, L) and positions.dtype == torch.int64:
        return positions
    try:
        return positions.long().expand(B, L)
    except RuntimeError:
        raise ValueError(f"{name}: positions {tuple(positions.shape)} do not spread over "
                         f"[{B}, {L}]") from None


def _need_cuda(name: str, t: Tensor) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name}: queries and keys must be CUDA tensors; there is no CPU "
                           f"implementation")


@_native.untraced
def qk_norm_rope(q: Tensor, k: Tensor, q_weight: Optional[Tensor] = None,
                 k_weight: Optional[Tensor] = None, cos: Optional[Tensor] = None,
                 sin: Optional[Tensor] = None, positions: Optional[Tensor] = None,
                 eps: float = 1e-6, interleaved: bool = False) -> Tuple[Tensor, Tensor]:
    """Normalised and rotated queries [B, L, Hq, D] and keys [B, L, Hk, D] (contiguous).

    q_weight, k_weight: [D] or None (no scaling).  cos, sin: [rows, rot_dim / 2] fp32, or None
    (no rotation); token t takes row t, or positions [B, L] (broadcast) says which.  A position
    outside the table makes that token's heads NaN."""
    if positions is None or (positions.dtype == torch.int64 and positions.shape == q.shape[:2]):
        try:
            return _native.ops().qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps,
                                              interleaved)
        except RuntimeError:
            _check_qk(q, k, q_weight, k_weight, cos, sin, positions)
            raise
    positions = _check_qk(q, k, q_weight, k_weight, cos, sin, positions)
    return _native.ops().qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps,
                                      interleaved)


def _check_qk(q, k, q_weight, k_weight, cos, sin, positions):
    _need_cuda("qk_norm_rope", q)
    _need_cuda("qk_norm_rope", k)
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError(f"qk_norm_rope: expected q [B, L, Hq, D] and k [B, L, Hk, D], got "
                         f"{tuple(q.shape)} and {tuple(k.shape)}")
    if q.dtype != k.dtype or q.device != k.device:
        raise TypeError(f"qk_norm_rope: q is {q.dtype} on {q.device}, k {k.dtype} on {k.device}")
    return _check_rest("qk_norm_rope", q, q.shape[3], q_weight, k_weight, cos, sin, positions)


@_native.untraced
def qkv_norm_rope(qkv: Tensor, q_heads: int, k_heads: int, q_weight: Optional[Tensor] = None,
                  k_weight: Optional[Tensor] = None, cos: Optional[Tensor] = None,
                  sin: Optional[Tensor] = None, positions: Optional[Tensor] = None,
                  eps: float = 1e-6,
                  interleaved: bool = False) -> Tuple[Tensor, Tensor, Tensor]:
    """`qk_norm_rope` of a projection's output qkv [B, L, (q_heads + 2 k_heads) D], the queries'
    heads first, then the keys', then the values'.  Returns (q, k, v) as [B, L, heads, D]; v is a
    view of qkv."""
    if positions is None or (positions.dtype == torch.int64 and positions.shape == qkv.shape[:2]):
        try:
            return _native.ops().qkv_norm_rope(qkv, q_heads, k_heads, q_weight, k_weight, cos, sin,
                                               positions, eps, interleaved)
        except RuntimeError:
            _check_qkv(qkv, q_heads, k_heads, q_weight, k_weight, cos, sin, positions)
            raise
    positions = _check_qkv(qkv, q_heads, k_heads, q_weight, k_weight, cos, sin, positions)
    return _native.ops().qkv_norm_rope(qkv, q_heads, k_heads, q_weight, k_weight, cos, sin,
                                       positions, eps, interleaved)


def _check_qkv(qkv, q_heads, k_heads, q_weight, k_weight, cos, sin, positions):
    _need_cuda("qkv_norm_rope", qkv)
    if q_heads < 1 or k_heads < 1:
        raise ValueError(f"qkv_norm_rope: need at least one head of each, got {q_heads} and "
                         f"{k_heads}")
    if qkv.dim() != 3 or qkv.shape[2] == 0 or qkv.shape[2] % (q_heads + 2 * k_heads):
        raise ValueError(f"qkv_norm_rope: expected [B, L, (Hq + 2 Hk) D] for {q_heads} and "
                         f"{k_heads} heads, got {tuple(qkv.shape)}")
    return _check_rest("qkv_norm_rope", qkv, qkv.shape[2] // (q_heads + 2 * k_heads),
                       q_weight, k_weight, cos, sin, positions)


class QKNormRope(nn.Module):
    """Learned norm weights of queries and keys and the rotation table of an attention block.
    forward(qkv) is `qkv_norm_rope`."""

    def __init__(self, head_dim: int, q_heads: int, k_heads: Optional[int] = None,
                 table: Optional[Tuple[Tensor, Tensor]] = None, eps: float = 1e-6,
                 interleaved: bool = False):
        super().__init__()
        self.q_heads = q_heads
        self.k_heads = k_heads or q_heads
        self.eps = eps
        self.interleaved = interleaved
        self.q_weight = nn.Parameter(torch.ones(head_dim))
        self.k_weight = nn.Parameter(torch.ones(head_dim))
        cos, sin = table if table is not None else (None, None)
        if any(t is not None and t.is_meta for t in (cos, sin)):
            raise ValueError("QKNormRope: the table has no values (made on the meta device)")
        self.register_buffer("cos", cos, persistent=False)
        self.register_buffer("sin", sin, persistent=False)

    def _apply(self, fn, recurse=True):
        # the table moves, but keeps its values and stays fp32: where the module goes to another
        # floating type, and where its storage is made anew (to_empty)
        tables = (self.cos, self.sin)
        super()._apply(fn, recurse)
        for name, t in zip(("cos", "sin"), tables):
            if t is None:
                continue
            if t.is_meta and not getattr(self, name).is_meta:
                raise RuntimeError("QKNormRope: the table's values were left on the meta device; "
                                   "make the module again")
            setattr(self, name, t.to(getattr(self, name).device))
        return self

    def forward(self, qkv: Tensor,
                positions: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor]:
        return qkv_norm_rope(qkv, self.q_heads, self.k_heads, self.q_weight, self.k_weight,
                             self.cos, self.sin, positions, self.eps, self.interleaved)

    def extra_repr(self) -> str:
        rot = 0 if self.cos is None else 2 * self.cos.shape[1]
        return (f"head_dim={self.q_weight.shape[0]}, q_heads={self.q_heads}, "
                f"k_heads={self.k_heads}, rot_dim={rot}, interleaved={self.interleaved}")
