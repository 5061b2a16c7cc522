"""Arguments the orthogonalised updates refuse, on the CPU: the C entry points before anything is
enqueued, the Python functions and the optimizer before the library is asked."""

import ctypes

import pytest
import torch

import rational_kat_cu_b200 as kat
from rational_kat_cu_b200 import _native, muon


def test_workspace_bytes():
    lib = _native.lib()
    one = lib.kat_muon_workspace_bytes(1, 768, 768)
    # X twice and A, B: two fp16 planes each
    assert one >= 4 * 2 * 768 * 768 * 2
    assert lib.kat_muon_workspace_bytes(12, 768, 768) >= 12 * 4 * 2 * 768 * 768 * 2
    assert lib.kat_muon_workspace_bytes(1, 2304, 768) == lib.kat_muon_workspace_bytes(1, 768, 2304)
    for count, r, c in ((0, 8, 8), (-1, 8, 8), (65, 8, 8), (1, 0, 8), (1, 8, 65537)):
        assert lib.kat_muon_workspace_bytes(count, r, c) == 0


def test_entry_points_refuse():
    lib, E = _native.lib(), _native
    one = (ctypes.c_void_p * 1)(256)
    none = (ctypes.c_void_p * 1)(None)

    def ortho(x=one, out=one, count=1, r=8, c=8, dtype=0, steps=5, ws=256, size=1 << 20):
        return lib.kat_orthogonalize(x, out, count, r, c, dtype, steps, ws, size, None)

    def step(w=one, g=one, m=one, count=1, r=8, c=8, dtype=0, steps=5, ws=256, size=1 << 20):
        return lib.kat_muon_step(w, g, m, count, r, c, dtype, 0.1, None, 0.9, 1, 0.0, 1.0, steps,
                                 ws, size, None)

    for f in (ortho, step):
        assert f(count=0) == E.KAT_OK
        assert f(count=65) == f(count=-1) == f(r=0) == f(c=0) == E.KAT_ERR_BAD_SHAPE
        assert f(r=65537) == f(steps=0) == f(steps=33) == E.KAT_ERR_BAD_SHAPE
        assert f(dtype=3) == f(dtype=-1) == E.KAT_ERR_BAD_DTYPE
        assert f(ws=None) == f(size=16) == f(ws=264) == E.KAT_ERR_WORKSPACE
    assert ortho(x=None) == ortho(out=None) == ortho(x=none) == E.KAT_ERR_NULL_POINTER
    assert step(w=None) == step(g=None) == step(m=None) == E.KAT_ERR_NULL_POINTER
    assert step(w=none) == step(g=none) == step(m=none) == E.KAT_ERR_NULL_POINTER
    assert lib.kat_muon_device_status(0, 0, None) == E.KAT_ERR_NULL_POINTER


def test_functions_refuse():
    x = torch.zeros(4, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        kat.orthogonalize(x)
    with pytest.raises(ValueError, match="rows, cols"):
        kat.orthogonalize(torch.zeros(4))
    for steps in (0, 33, 2.0):
        with pytest.raises(ValueError, match="steps"):
            kat.orthogonalize(x, steps=steps)
    with pytest.raises(RuntimeError, match="CUDA"):
        kat.muon_step([x], [x], [x], lr=0.1)
    with pytest.raises(ValueError, match="1 weights, 0 gradients"):
        kat.muon_step([x], [], [x], lr=0.1)
    with pytest.raises(ValueError, match="matrices"):
        kat.muon_step([x[0]], [x[0]], [x[0]], lr=0.1)


def test_optimizer_refuses():
    p = torch.nn.Parameter(torch.zeros(4, 4))
    for bad in (dict(lr=-1.0), dict(momentum=1.0), dict(momentum=-0.1), dict(weight_decay=-1.0),
                dict(steps=0)):
        with pytest.raises(ValueError, match="Muon"):
            kat.Muon([p], **bad)
    with pytest.raises(ValueError, match="matrices"):
        kat.Muon([torch.nn.Parameter(torch.zeros(4))])


def test_momenta_stay_float32_through_state_dict():
    p = torch.nn.Parameter(torch.zeros(3, 5, dtype=torch.bfloat16))
    a, b = kat.Muon([p], lr=0.1), kat.Muon([p], lr=0.2)
    a.state[p]["momentum_buffer"] = torch.full((3, 5), 1 + 2.0 ** -20)
    b.load_state_dict(a.state_dict())
    m = b.state[p]["momentum_buffer"]
    assert m.dtype == torch.float32 and torch.equal(m, a.state[p]["momentum_buffer"])
    assert m.data_ptr() != a.state[p]["momentum_buffer"].data_ptr()
    assert b.param_groups[0]["lr"] == 0.1


def test_runs_cover_every_matrix(monkeypatch):
    for limit in (1, 1 << 20, 2 << 30):
        monkeypatch.setattr(muon, "WORKSPACE_LIMIT", limit)
        runs = list(muon._runs(150, 100, 30))
        assert [r[0] for r in runs] == [sum(x[1] for x in runs[:i]) for i in range(len(runs))]
        assert sum(r[1] for r in runs) == 150 and max(r[1] for r in runs) <= muon.MAX_MATRICES
