"""The relative position bias on the CPU: buckets against their definition in integers, the sorted
cells of an index, and what the entry points and functions refuse."""

import ctypes

import pytest
import torch

import rational_kat_cu_b200 as kat
from rational_kat_cu_b200 import _native, position_bias


def by_definition(d, num_buckets, max_distance, bidirectional):
    """The bucket of one distance, counting up from the definition."""
    side = num_buckets // 2 if bidirectional else num_buckets
    half = side // 2
    rest = side - half
    x = abs(d) if bidirectional else max(0, -d)
    if x < half:
        b = x
    else:
        k = 0
        while k + 1 < rest and x ** rest * half ** (k + 1) >= max_distance ** (k + 1) * half ** rest:
            k += 1
        b = half + k
    return b + (side if bidirectional and d > 0 else 0)


@pytest.mark.parametrize("args", [(32, 128, True), (32, 128, False), (8, 500, True), (2, 5, False),
                                  (4, 2, True), (64, 100, False), (7, 20, False)])
def test_distance_buckets(args):
    b = kat.DistanceBuckets(*args)
    far = 3 * args[1]
    d = torch.arange(-far, far + 1)
    got = b.bucket(d)
    assert got.tolist() == [by_definition(x, *args) for x in d.tolist()]
    # each bucket is one run of distances
    for k in range(args[0]):
        inside = d[got == k]
        low, high = max(int(b._begin[k]), -far), min(int(b._end[k]), far)
        assert inside.tolist() == list(range(low, high + 1))
    assert b.bucket(torch.tensor([-10 ** 9, 10 ** 9])).tolist() == \
        [by_definition(-10 ** 9, *args), by_definition(10 ** 9, *args)]


def test_distance_buckets_refuse():
    for bad in ((1, 128, False), (2, 128, True), (5, 128, True), (32, 8, True), (32, 16, False),
                (32, 1 << 25, True), (1026, 4096, True)):
        with pytest.raises(ValueError, match="DistanceBuckets"):
            kat.DistanceBuckets(*bad)


@pytest.mark.parametrize("lq,lk,nb", [(1, 1, 1), (5, 9, 3), (40, 33, 7), (300, 70, 2),
                                      (3, 16384, 5), (130, 127, 1000)])
def test_index_buckets_list_every_cell_once(lq, lk, nb):
    g = torch.Generator().manual_seed(lq)
    index = torch.randint(-1, nb, (lq, lk), generator=g)
    b = kat.IndexBuckets(index, nb)
    padded, plain, cells, seg_begin, slab_begin, seg_place, bucket_begin = b.on(index.device)
    ld = (lk + 7) // 8 * 8
    assert padded.shape == (lq, ld) and (padded[:, lk:] == nb).all()
    assert b.slab_rows * ld <= position_bias.SLAB_CELLS or b.slab_rows == 1
    assert b.slabs * b.slab_rows >= lq > (b.slabs - 1) * b.slab_rows
    seen = torch.zeros(lq, ld, dtype=torch.int64)
    bucket_of_segment = {}
    for s in range(b.slabs):
        for seg in range(int(slab_begin[s]), int(slab_begin[s + 1])):
            begin, end = int(seg_begin[seg]), int(seg_begin[seg + 1])
            assert 0 < end - begin <= position_bias.SEGMENT
            at = cells[begin:end].long()
            row, col = s * b.slab_rows + at // ld, at % ld
            assert torch.equal(plain[begin:end].long(), at // ld * lk + col)
            assert (row < lq).all() and (col < lk).all()
            seen[row, col] += 1
            values = index[row, col]
            assert (values == values[0]).all()
            bucket_of_segment[seg] = int(values[0])
    assert torch.equal(seen[:, :lk], (index >= 0).long()) and not seen[:, lk:].any()
    assert sorted(seg_place.tolist()) == list(range(b.segments)) == sorted(bucket_of_segment)
    by_bucket = seg_place.long().argsort()
    for k in range(nb):
        for g in by_bucket[int(bucket_begin[k]):int(bucket_begin[k + 1])].tolist():
            assert bucket_of_segment[g] == k
    assert int(bucket_begin[0]) == 0 and int(bucket_begin[nb]) == b.segments


def test_index_buckets_refuse():
    ok = torch.zeros(2, 3, dtype=torch.int64)
    for bad, nb in ((ok[0], 1), (ok.float(), 1), (ok, 0), (ok - 2, 1), (ok + 1, 1),
                    (torch.zeros(1, 16385, dtype=torch.int32), 1)):
        with pytest.raises(ValueError, match="IndexBuckets"):
            kat.IndexBuckets(bad, nb)
    # empty matrices and matrices without a bias hold no cells
    assert kat.IndexBuckets(ok[:0], 1).segments == kat.IndexBuckets(ok - 1, 1).segments == 0


def test_grid_index():
    index, n = kat.grid_index(2, 3, prefix=1)
    assert n == 3 * 5 + 3 and index.shape == (7, 7)
    assert index[0, 0] == n - 1 and (index[0, 1:] == n - 3).all() and (index[1:, 0] == n - 2).all()
    for a in range(6):
        for b in range(6):
            dy, dx = a // 3 - b // 3, a % 3 - b % 3
            assert index[1 + a, 1 + b] == (dy + 1) * 5 + dx + 2
    assert kat.grid_index(2, 3)[1] == 15
    for bad in ((0, 1, 0), (1, 0, 0), (1, 1, -1)):
        with pytest.raises(ValueError):
            kat.grid_index(*bad)


def test_entry_points_refuse():
    lib, E = _native.lib(), _native
    stride = (ctypes.c_int64 * 3)(8, 8, 1)
    P = 256

    def dfwd(table=P, tdt=0, nb=4, heads=2, of=P, reach=3, lq=5, lk=6, off=0, out=P, odt=0):
        return lib.kat_distance_bias_fwd(table, tdt, nb, heads, of, reach, lq, lk, off, 0, out,
                                         odt, None)

    def dbwd(dout=P, ddt=0, st=stride, nb=4, heads=2, rb=P, re=P, lq=5, lk=6, off=0, dt=P, tdt=0,
             ws=P, size=1 << 20):
        return lib.kat_distance_bias_bwd(dout, ddt, st, nb, heads, rb, re, lq, lk, off, 0, dt, tdt,
                                         ws, size, None)

    def ifwd(table=P, tdt=0, nb=4, heads=2, index=P, lq=5, lk=6, out=P, odt=0):
        return lib.kat_index_bias_fwd(table, tdt, nb, heads, index, lq, lk, out, odt, None)

    def ibwd(dout=P, ddt=0, st=stride, nb=4, heads=2, lq=5, lk=6, cells=P, pc=P, sb=P, segs=9, slb=P,
             slabs=1, rows=5, bb=P, bkb=P, dt=P, tdt=0, ws=P, size=1 << 20):
        return lib.kat_index_bias_bwd(dout, ddt, st, nb, heads, lq, lk, cells, pc, sb, segs, slb,
                                      slabs, rows, bb, bkb, dt, tdt, ws, size, None)

    for f in (dfwd, dbwd, ifwd, ibwd):
        assert f(tdt=3) == E.KAT_ERR_BAD_DTYPE
        for bad in (dict(nb=0), dict(heads=-1), dict(heads=65536), dict(lq=-1), dict(lk=-1),
                    dict(lk=1 << 31)):
            assert f(**bad) == E.KAT_ERR_BAD_SHAPE
        assert f(heads=0) == E.KAT_OK
    for f, names in ((dfwd, ("table", "of", "out")), (dbwd, ("dout", "st", "rb", "re", "dt")),
                     (ifwd, ("table", "index", "out")),
                     (ibwd, ("dout", "st", "cells", "pc", "sb", "slb", "bb", "bkb", "dt"))):
        for name in names:
            assert f(**{name: None}) == E.KAT_ERR_NULL_POINTER
    for f in (dfwd, ifwd):
        assert f(odt=7) == E.KAT_ERR_BAD_DTYPE and f(out=264) == E.KAT_ERR_BAD_SHAPE
        assert f(lq=0, out=None) == f(lk=0, table=None) == E.KAT_OK
    for f in (dbwd, ibwd):
        assert f(ddt=7) == E.KAT_ERR_BAD_DTYPE
        assert f(ws=None) == f(size=8) == f(ws=264) == E.KAT_ERR_WORKSPACE
    assert dfwd(reach=-1) == dfwd(off=1 << 40) == dbwd(off=-(1 << 40)) == E.KAT_ERR_BAD_SHAPE
    assert ifwd(index=264) == E.KAT_ERR_BAD_SHAPE
    for bad in (dict(segs=-1), dict(rows=0), dict(rows=4), dict(lk=16385), dict(slabs=2)):
        assert ibwd(**bad) == E.KAT_ERR_BAD_SHAPE
    assert lib.kat_distance_bias_bwd_workspace_bytes(2, 0, 5) == 0
    assert lib.kat_distance_bias_bwd_workspace_bytes(-1, 5, 5) == 0
    assert lib.kat_index_bias_bwd_workspace_bytes(2, 100) == 800


def test_distance_plan_bytes_stay_small():
    """Partial sums: at most 64 bytes for 8 x 8 cells (or 4 for 8 of a diagonal), plus the diagonals."""
    lib = _native.lib()
    for h, lq, lk in ((1, 1, 1), (16, 1, 4097), (16, 4096, 4096), (12, 197, 197), (1, 100000, 3),
                      (2, 3, 100000)):
        cells8 = ((lq + 7) // 8) * ((lk + 7) // 8 + 31)
        size = lib.kat_distance_bias_bwd_workspace_bytes(h, lq, lk)
        cells1 = ((lq + 7) // 8) * (lq + lk)
        assert 0 < size <= h * (max(cells8 * 64, cells1 * 4) + (lq + lk) * 8 + 16)


def test_functions_refuse():
    b = kat.DistanceBuckets(8, 20)
    with pytest.raises(RuntimeError, match="CUDA"):
        kat.distance_bias(torch.zeros(8, 2), b, 3, 3)
    with pytest.raises(RuntimeError, match="CUDA"):
        kat.GridPositionBias(2, 3, 3)()
    with pytest.raises(RuntimeError, match="CUDA"):
        kat.RelativePositionBias(2)(4, 4)
    assert list(kat.RelativePositionBias(2).state_dict()) == ["table"]
    assert "rows=3" in repr(kat.GridPositionBias(2, 3, 4, 1))
