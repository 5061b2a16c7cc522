"""The norm of queries and keys with the rotation, on the CPU: what the C entry points and the
Python functions refuse, and the angle tables."""

import ctypes
import math

import pytest
import torch

import rational_kat_cu_b200 as kat
from rational_kat_cu_b200 import _native, head_norm


class Stream(ctypes.Structure):
    """`kat_head_stream`."""

    _fields_ = [("x", ctypes.c_void_p), ("dy", ctypes.c_void_p), ("out", ctypes.c_void_p),
                ("weight", ctypes.c_void_p), ("dweight", ctypes.c_void_p),
                ("x_stride", ctypes.c_int64 * 3), ("dy_stride", ctypes.c_int64 * 3),
                ("out_stride", ctypes.c_int64 * 3), ("heads", ctypes.c_int32)]


class Problem(ctypes.Structure):
    """`kat_head_problem`."""

    _fields_ = [("batch", ctypes.c_int64), ("tokens", ctypes.c_int64),
                ("head_dim", ctypes.c_int32), ("rot_dim", ctypes.c_int32),
                ("interleaved", ctypes.c_int32), ("dtype", ctypes.c_int32),
                ("weight_dtype", ctypes.c_int32), ("eps", ctypes.c_float),
                ("cos_table", ctypes.c_void_p), ("sin_table", ctypes.c_void_p),
                ("table_rows", ctypes.c_int64), ("positions", ctypes.c_void_p),
                ("position_stride", ctypes.c_int64 * 2)]


def problem(**kw):
    base = dict(batch=2, tokens=3, head_dim=64, rot_dim=64, interleaved=0, dtype=0, weight_dtype=0,
                eps=1e-6, cos_table=256, sin_table=256, table_rows=3, positions=None,
                position_stride=(0, 0))
    base.update(kw)
    return Problem(*base.values())


def stream(**kw):
    base = dict(x=256, dy=256, out=256, weight=None, dweight=None, x_stride=(0, 0, 0),
                dy_stride=(0, 0, 0), out_stride=(0, 0, 0), heads=2)
    base.update(kw)
    return Stream(*base.values())


def fwd(p, *streams, count=None):
    return _native.lib().kat_qk_norm_rope_fwd(
        ctypes.byref(p), (Stream * len(streams))(*streams),
        len(streams) if count is None else count, None)


def bwd(p, *streams, ws=None, size=0):
    return _native.lib().kat_qk_norm_rope_bwd(
        ctypes.byref(p), (Stream * len(streams))(*streams), len(streams), ws, size,
        None)


def test_entry_points_refuse():
    E, lib = _native, _native.lib()
    assert lib.kat_qk_norm_rope_fwd(None, None, 1, None) == E.KAT_ERR_NULL_POINTER
    for f in (fwd, bwd):
        for bad in (dict(dtype=3), dict(weight_dtype=-1)):
            assert f(problem(**bad), stream()) == E.KAT_ERR_BAD_DTYPE
        for bad in (dict(head_dim=0), dict(head_dim=1025), dict(rot_dim=66), dict(rot_dim=31),
                    dict(rot_dim=-2), dict(batch=-1), dict(tokens=-1), dict(table_rows=2),
                    dict(batch=1 << 30)):
            assert f(problem(**bad), stream()) == E.KAT_ERR_BAD_SHAPE
        assert f(problem(), stream(heads=-1)) == E.KAT_ERR_BAD_SHAPE
        assert f(problem(cos_table=None), stream()) == E.KAT_ERR_NULL_POINTER
        assert f(problem(sin_table=None), stream()) == E.KAT_ERR_NULL_POINTER
        assert f(problem(), stream(out=None)) == E.KAT_ERR_NULL_POINTER
        # no tokens, no heads: nothing to do, nothing asked of the pointers
        assert f(problem(tokens=0), stream(x=None, dy=None, out=None)) == E.KAT_OK
        assert f(problem(), stream(heads=0, x=None, dy=None, out=None)) == E.KAT_OK
    assert fwd(problem(), stream(x=None)) == E.KAT_ERR_NULL_POINTER
    assert bwd(problem(), stream(dy=None)) == E.KAT_ERR_NULL_POINTER
    assert bwd(problem(), stream(x=None, dweight=256)) == E.KAT_ERR_NULL_POINTER
    for f in (fwd, bwd):
        assert f(problem(tokens=1 << 32), stream(heads=0)) == E.KAT_OK
    assert fwd(problem(), stream(), count=0) == E.KAT_ERR_BAD_SHAPE
    assert fwd(problem(), *[stream()] * 4) == E.KAT_ERR_BAD_SHAPE
    assert lib.kat_qk_norm_rope_bwd_workspace_bytes(0, 1, 0) == 0
    assert lib.kat_qk_norm_rope_bwd_workspace_bytes(64, 4, 0) == 0


def test_functions_need_cuda():
    q = torch.zeros(1, 2, 3, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        kat.qk_norm_rope(q, q)
    with pytest.raises(RuntimeError, match="CUDA"):
        kat.qkv_norm_rope(torch.zeros(1, 2, 24), 1, 1)


def test_rest_is_checked():
    x = torch.zeros(2, 3, 4, 16)
    cos = torch.zeros(5, 8)
    ok = dict(q_weight=torch.ones(16), k_weight=None, cos=cos, sin=cos, positions=None)

    def check(x=x, head_dim=16, **kw):
        return head_norm._check_rest("f", x, head_dim, **{**ok, **kw})

    assert check() is None
    assert check(positions=torch.tensor([[4], [1]], dtype=torch.int32)).shape == (2, 3)
    for bad in (dict(x=x.double()), dict(q_weight=torch.ones(16).double()),
                dict(k_weight=torch.ones(16).half()), dict(cos=cos.half(), sin=cos.half()),
                dict(positions=torch.zeros(2, 3))):
        with pytest.raises(TypeError):
            check(**bad)
    for bad in (dict(head_dim=2048, q_weight=None), dict(q_weight=torch.ones(8)),
                dict(q_weight=torch.ones(16, 2)[:, 0]), dict(sin=None), dict(cos=cos.t()),
                dict(cos=cos[:2], sin=cos[:2]), dict(sin=cos[:4]),
                dict(cos=torch.zeros(5, 9), sin=torch.zeros(5, 9)),
                dict(cos=None, sin=None, positions=torch.zeros(2, 3, dtype=torch.int64)),
                dict(cos=cos.clone().requires_grad_()),
                dict(positions=torch.zeros(3, 3, dtype=torch.int64))):
        with pytest.raises(ValueError):
            check(**bad)


def test_tables():
    cos, sin = kat.rope_table(100001, 6, base=10000.0)
    assert cos.shape == sin.shape == (100001, 3) and cos.dtype == torch.float32
    for p in (0, 1, 99999, 100000):
        for i in range(3):
            angle = p * 10000.0 ** (-2 * i / 6)
            # 2^-24: one rounding; 1e-9: the angle's 64-bit rounding at this size
            assert abs(float(cos[p, i]) - math.cos(angle)) <= 2.0 ** -24 + 1e-9
            assert abs(float(sin[p, i]) - math.sin(angle)) <= 2.0 ** -24 + 1e-9
    cos, sin = kat.rope_grid_table(2, 3, 8, prefix=1)
    assert cos.shape == (7, 4)
    assert torch.equal(cos[0], torch.ones(4)) and not sin[0].any()
    y, x = 1, 2
    row = 1 + y * 3 + x
    want = [math.sin(y), math.sin(y * 100 ** -0.5), math.sin(x), math.sin(x * 100 ** -0.5)]
    assert torch.allclose(sin[row], torch.tensor(want), atol=1e-7)
    for bad in (lambda: kat.rope_table(-1, 4), lambda: kat.rope_table(3, 5),
                lambda: kat.rope_grid_table(2, 2, 6), lambda: kat.rope_grid_table(-1, 2, 8)):
        with pytest.raises(ValueError):
            bad()
    assert kat.rope_table(4, 0)[0].shape == (4, 0)


def test_module_keeps_its_table_in_fp32():
    m = kat.QKNormRope(16, 4, 2, table=kat.rope_table(7, 16))
    assert list(m.state_dict()) == ["q_weight", "k_weight"]
    before = m.cos.clone()
    m = m.to(torch.bfloat16)
    assert m.q_weight.dtype == torch.bfloat16
    assert m.cos.dtype == m.sin.dtype == torch.float32 and torch.equal(m.cos, before)
    assert "rot_dim=16" in repr(m)
