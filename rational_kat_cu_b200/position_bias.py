"""Learned relative position bias by buckets, with its gradient.

A bias [heads, Lq, Lk] for attention scores, looked up in a learned table [buckets, heads] by a
bucket of each (query, key).  Two kinds of bucket:

  DistanceBuckets   of the distance key - query: one bucket for each short distance, then buckets
                    that widen with the logarithm of the distance, up to `max_distance`
  IndexBuckets      of an index matrix [Lq, Lk], as `grid_index` makes one for a grid of patches

`distance_bias` and `index_bias` evaluate them on the sm_100a kernels of libkat_rational.so
(include/kat_position_bias.h), forward and backward, called by the torch operators of libkat_torch.so
(csrc/kat_torch.cpp); RelativePositionBias and GridPositionBias hold the table.  A bias is returned as a view whose rows start at multiples of 16 bytes (its row
stride is Lk rounded up to 8), ready to be an attention kernel's mask.  There is no CPU
implementation: CPU tables raise, and a missing library raises on first use.
"""

from __future__ import annotations

from typing import Dict, List, Optional, Tuple

import torch
import torch.nn as nn
from torch import Tensor

from . import _native

DTYPES = {torch.float32: _native.KAT_DTYPE_F32, torch.float16: _native.KAT_DTYPE_F16,
          torch.bfloat16: _native.KAT_DTYPE_BF16}
SLAB_CELLS = 16384    # KAT_BIAS_SLAB_CELLS
SEGMENT = 32          # KAT_BIAS_SEGMENT
MAX_BUCKETS = 1 << 24
MAX_DISTANCE_BUCKETS = 1024   # their borders are exact, in integers of that many digits
MAX_LENGTH = (1 << 31) - 64
MAX_REACH = 1 << 24
INT32_MIN, INT32_MAX = -(1 << 31), (1 << 31) - 1


def _round8(n: int) -> int:
    return (n + 7) // 8 * 8


def _kept_on(kept: Dict[torch.device, Tuple[Tensor, ...]], tensors: Tuple[Tensor, ...],
             device: torch.device) -> Tuple[Tensor, ...]:
    """The copies of `tensors` that `kept` holds for `device` ("cuda" is the current device), made
    if it has none."""
    if device not in kept:
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        if device not in kept:
            kept[device] = _copied(tensors, device)
    return kept[device]


def _copied(tensors: Tuple[Tensor, ...], device: torch.device) -> Tuple[Tensor, ...]:
    """Copies on `device` that any stream may use."""
    copies = tuple(t.to(device) for t in tensors)
    if device.type == "cuda":
        torch.cuda.current_stream(device).synchronize()
    return copies


class _Plan:
    """What bucket plans share.  A plan does not change once made: copies of a module share it.  Its copies
    on devices are not stored with it, since torch.load may put those on any device."""

    def __getstate__(self) -> dict:
        return {**self.__dict__, "_on": {}}

    def __setstate__(self, state: dict) -> None:
        self.__dict__.update(state, _on={})

    def __deepcopy__(self, memo) -> "_Plan":
        return self


class DistanceBuckets(_Plan):
    """Buckets of a distance d = key - query.

    bidirectional: half of the buckets for d <= 0, half for d > 0, by |d|; otherwise all of them
    by max(0, -d) (keys behind the query share bucket 0 with the query itself).  Of a side's n
    buckets the first n / 2 hold one distance each; bucket n / 2 + k begins at the least distance
    x with (x / (n/2)) ^ (n - n/2) >= (max_distance / (n/2)) ^ k, compared as integers, and the
    last one has no end."""

    def __init__(self, num_buckets: int = 32, max_distance: int = 128,
                 bidirectional: bool = True, device=None):
        if num_buckets < 2 or num_buckets > MAX_DISTANCE_BUCKETS:
            raise ValueError(f"DistanceBuckets: num_buckets must be 2..{MAX_DISTANCE_BUCKETS}, got "
                             f"{num_buckets}")
        if bidirectional and (num_buckets % 2 or num_buckets < 4):
            raise ValueError(f"DistanceBuckets: two directions need an even number of buckets, "
                             f"at least 4, got {num_buckets}")
        side = num_buckets // 2 if bidirectional else num_buckets
        half = side // 2
        if not half < max_distance <= MAX_REACH:
            raise ValueError(f"DistanceBuckets: max_distance must be {half + 1}..{MAX_REACH} for "
                             f"{num_buckets} buckets, got {max_distance}")
        self.num_buckets, self.max_distance = num_buckets, max_distance
        self.bidirectional = bidirectional
        # starts[b]: the least distance of bucket b of a side
        self.starts = list(range(half)) + self._borders(side, half, max_distance)
        reach = max(self.starts[-1], 1)
        by_size = torch.bucketize(torch.arange(reach + 1, device="cpu"),
                                  torch.tensor(self.starts, device="cpu"), right=True) - 1
        behind = by_size.flip(0)[:-1]                   # d = -reach .. -1
        ahead = by_size + side if bidirectional else torch.zeros_like(by_size)
        self.reach = reach
        self._of = torch.cat([behind, by_size[:1], ahead[1:]]).to(torch.int32)
        self._begin, self._end = self._runs()
        self._on: Dict[torch.device, Tuple[Tensor, Tensor, Tensor]] = {}
        if device is not None:
            self.on(torch.device(device))

    @staticmethod
    def _borders(side: int, half: int, max_distance: int) -> List[int]:
        rest, found, low = side - half, [], half
        for k in range(rest):
            goal = max_distance ** k * half ** rest
            scale = half ** k
            high = max_distance            # satisfies every k < rest
            while low < high:
                mid = (low + high) // 2
                if mid ** rest * scale >= goal:
                    high = mid
                else:
                    low = mid + 1
            found.append(low)
        return found

    def _runs(self) -> Tuple[Tensor, Tensor]:
        """First and last distance of each bucket (the outermost without an end; empty buckets
        end before they begin)."""
        d = torch.arange(-self.reach, self.reach + 1, device="cpu")
        of = self._of.long()
        begin = torch.zeros(self.num_buckets, dtype=torch.int64, device="cpu")
        end = torch.full((self.num_buckets,), -1, dtype=torch.int64, device="cpu")
        first = torch.ones_like(of, dtype=torch.bool)
        first[1:] = of[1:] != of[:-1]
        last = torch.ones_like(first)
        last[:-1] = first[1:]
        begin[of[first]] = d[first]
        end[of[last]] = d[last]
        begin[of[0]] = INT32_MIN
        end[of[-1]] = INT32_MAX
        return begin.to(torch.int32), end.to(torch.int32)

    def bucket(self, distance: Tensor) -> Tensor:
        """Buckets of integer distances (key - query), on their device."""
        of = self._of.to(distance.device)
        return of[distance.long().clamp(-self.reach, self.reach) + self.reach].long()

    def on(self, device: torch.device) -> Tuple[Tensor, Tensor, Tensor]:
        """(bucket_of, run_begin, run_end) on `device`, kept there (the first use on a device
        copies them: not inside a graph capture)."""
        return _kept_on(self._on, (self._of, self._begin, self._end), device)

    def __repr__(self) -> str:
        return (f"DistanceBuckets(num_buckets={self.num_buckets}, "
                f"max_distance={self.max_distance}, bidirectional={self.bidirectional})")


class IndexBuckets(_Plan):
    """Buckets of an index matrix [Lq, Lk] with values in [0, num_buckets); -1 marks cells without
    a bias (0, and no gradient).  Keeps the cells sorted by bucket, for the gradient: make it
    once.  Lk is at most 16384 (long sequences go by distance)."""

    def __init__(self, index: Tensor, num_buckets: int):
        if index.dim() != 2 or index.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"IndexBuckets: expected an int32 or int64 matrix, got "
                             f"{tuple(index.shape)} {index.dtype}")
        lq, lk = index.shape
        if not 1 <= num_buckets <= MAX_BUCKETS:
            raise ValueError(f"IndexBuckets: num_buckets must be 1..{MAX_BUCKETS}, got "
                             f"{num_buckets}")
        if lk > SLAB_CELLS or lq * _round8(lk) > INT32_MAX:
            raise ValueError(f"IndexBuckets: at most {SLAB_CELLS} keys and 2^31 cells, got "
                             f"[{lq}, {lk}]")
        if index.numel() and not (-1 <= int(index.min()) and int(index.max()) < num_buckets):
            raise ValueError(f"IndexBuckets: values must be -1..{num_buckets - 1}, got "
                             f"{int(index.min())}..{int(index.max())}")
        self.num_buckets = num_buckets
        self.shape = (lq, lk)
        ld = _round8(lk)
        dev = index.device
        padded = torch.full((lq, ld), num_buckets, dtype=torch.int32, device=dev)
        padded[:, :lk] = torch.where(index < 0, num_buckets, index)
        # rows of a slab: at most what its shared memory holds, and at least 16 slabs' worth of
        # blocks for each head
        self.slab_rows = max(1, min(SLAB_CELLS // max(ld, 1), -(-lq // 16)))
        self.slabs = -(-lq // self.slab_rows)

        flat = padded.flatten()
        at = (flat < num_buckets).nonzero().flatten()
        row, col = at // max(ld, 1), at % max(ld, 1)
        key = row // self.slab_rows * num_buckets + flat[at]
        key, order = key.sort(stable=True)
        in_slab = row % self.slab_rows
        cells, padded_cells = ((in_slab * pitch + col)[order].to(torch.uint16)
                               for pitch in (lk, ld))
        n = key.numel()
        place = torch.arange(n, device=dev)
        new = torch.ones(n, dtype=torch.bool, device=dev)
        new[1:] = key[1:] != key[:-1]
        start = torch.where(new, place, 0).cummax(0).values if n else place
        begin = ((place - start) % SEGMENT == 0).nonzero().flatten()
        self.segments = begin.numel()
        seg_slab, seg_bucket = key[begin] // num_buckets, key[begin] % num_buckets
        sorted_bucket, by_bucket = seg_bucket.sort(stable=True)
        seg_place = torch.empty_like(by_bucket)
        seg_place[by_bucket] = torch.arange(self.segments, device=dev)
        self._tensors = (
            padded,
            cells,
            padded_cells if ld != lk else cells,
            torch.cat([begin, torch.tensor([n], device=dev)]).to(torch.int32),
            torch.searchsorted(seg_slab, torch.arange(self.slabs + 1, device=dev)).to(torch.int32),
            seg_place.to(torch.int32),
            torch.searchsorted(sorted_bucket,
                               torch.arange(num_buckets + 1, device=dev)).to(torch.int32))
        if dev.type == "cuda":      # any stream may use them
            torch.cuda.current_stream(dev).synchronize()
        self._on: Dict[torch.device, Tuple[Tensor, ...]] = {dev: self._tensors}

    def on(self, device: torch.device) -> Tuple[Tensor, ...]:
        """(index, cells, padded_cells, seg_begin, slab_begin, seg_place, bucket_begin) on `device`,
        kept there (the first use on a device copies them: not inside a graph capture)."""
        return _kept_on(self._on, self._tensors, device)

    def __repr__(self) -> str:
        return f"IndexBuckets(shape={self.shape}, num_buckets={self.num_buckets})"


def grid_index(rows: int, cols: int, prefix: int = 0) -> Tuple[Tensor, int]:
    """(index [n, n], num_buckets) of n = prefix + rows * cols tokens, the patches of a grid row
    by row behind `prefix` others: one bucket for each displacement of two patches (query minus
    key), and behind those one each for prefix to patch, patch to prefix and prefix to prefix."""
    if rows < 1 or cols < 1 or prefix < 0:
        raise ValueError(f"grid_index: need rows, cols >= 1 and prefix >= 0, got {rows}, {cols} "
                         f"and {prefix}")
    y = torch.arange(rows, device="cpu").repeat_interleave(cols)
    x = torch.arange(cols, device="cpu").repeat(rows)
    pairs = (2 * rows - 1) * (2 * cols - 1)
    n = prefix + rows * cols
    index = torch.empty(n, n, dtype=torch.int64, device="cpu")
    index[prefix:, prefix:] = ((y[:, None] - y + rows - 1) * (2 * cols - 1)
                               + x[:, None] - x + cols - 1)
    index[:prefix, prefix:] = pairs
    index[prefix:, :prefix] = pairs + 1
    index[:prefix, :prefix] = pairs + 2
    return index, pairs + (3 if prefix else 0)


# The torch operators check their arguments; what they refuse comes here for an error that says what
# is wrong.

def _check_table(name: str, table: Tensor, num_buckets: int, dtype: torch.dtype) -> None:
    if not table.is_cuda:
        raise RuntimeError(f"{name}: the table must be a CUDA tensor; there is no CPU "
                           f"implementation")
    if table.dtype not in DTYPES or dtype not in DTYPES:
        raise TypeError(f"{name}: table and bias must be float32, float16 or bfloat16, got "
                        f"{table.dtype} and {dtype}")
    if table.dim() != 2 or table.shape[0] != num_buckets or table.shape[1] > 65535:
        raise ValueError(f"{name}: expected a table [{num_buckets}, heads], got "
                         f"{tuple(table.shape)}")


@_native.untraced
def distance_bias(table: Tensor, buckets: DistanceBuckets, lq: int, lk: int, offset: int = 0,
                  causal: bool = False, dtype: Optional[torch.dtype] = None) -> Tensor:
    """bias[h, i, j] = table[bucket(j - i - offset), h], [heads, lq, lk] of type `dtype` (default:
    the table's).  `offset` is the place of the first query behind the first key (lk - lq for the
    last queries of a sequence, the cache's length for new tokens).  With `causal`, keys ahead of
    their query get -infinity and take no part in the gradient."""
    dtype = dtype or table.dtype
    try:
        return _native.ops().distance_bias(table, buckets.on(table.device), buckets.num_buckets,
                                           buckets.reach, lq, lk, offset, bool(causal),
                                           DTYPES.get(dtype, -1))
    except RuntimeError:
        _check_distance(table, buckets, lq, lk, offset, dtype)
        raise


def _check_distance(table, buckets, lq, lk, offset, dtype) -> None:
    _check_table("distance_bias", table, buckets.num_buckets, dtype)
    if not (0 <= lq <= MAX_LENGTH and 0 <= lk <= MAX_LENGTH and abs(offset) <= MAX_LENGTH):
        raise ValueError(f"distance_bias: lq, lk and |offset| must be 0..{MAX_LENGTH}, got "
                         f"{lq}, {lk} and {offset}")


@_native.untraced
def index_bias(table: Tensor, buckets: IndexBuckets,
               dtype: Optional[torch.dtype] = None) -> Tensor:
    """bias[h, i, j] = table[index[i, j], h], [heads, Lq, Lk] of type `dtype` (default: the
    table's)."""
    dtype = dtype or table.dtype
    try:
        return _native.ops().index_bias(table, buckets.on(table.device), buckets.num_buckets,
                                        *buckets.shape, buckets.slab_rows, buckets.slabs,
                                        buckets.segments, DTYPES.get(dtype, -1))
    except RuntimeError:
        _check_table("index_bias", table, buckets.num_buckets, dtype)
        raise


class RelativePositionBias(nn.Module):
    """A learned bias by distance: forward(lq, lk, offset=0, causal=False) -> [heads, lq, lk]."""

    def __init__(self, heads: int, num_buckets: int = 32, max_distance: int = 128,
                 bidirectional: bool = True):
        super().__init__()
        self.buckets = DistanceBuckets(num_buckets, max_distance, bidirectional)
        self.table = nn.Parameter(torch.zeros(num_buckets, heads))

    def forward(self, lq: int, lk: int, offset: int = 0, causal: bool = False,
                dtype: Optional[torch.dtype] = None) -> Tensor:
        return distance_bias(self.table, self.buckets, lq, lk, offset, causal, dtype)

    def extra_repr(self) -> str:
        return f"heads={self.table.shape[1]}, {self.buckets!r}"


class GridPositionBias(nn.Module):
    """A learned bias by displacement on a grid of patches behind `prefix` other tokens:
    forward() -> [heads, n, n]."""

    def __init__(self, heads: int, rows: int, cols: int, prefix: int = 0):
        super().__init__()
        self.grid = (rows, cols, prefix)
        self.buckets = IndexBuckets(*grid_index(rows, cols, prefix))
        self.table = nn.Parameter(torch.zeros(self.buckets.num_buckets, heads))

    def forward(self, dtype: Optional[torch.dtype] = None) -> Tensor:
        return index_bias(self.table, self.buckets, dtype)

    def extra_repr(self) -> str:
        rows, cols, prefix = self.grid
        return f"heads={self.table.shape[1]}, rows={rows}, cols={cols}, prefix={prefix}"
