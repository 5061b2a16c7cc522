"""Calls of the attention-input operators that need no GPU: stored and copied plans, and the torch
operators' own checks."""

import copy
import io

import pytest
import torch

import rational_kat_cu_b200 as kat
from rational_kat_cu_b200 import _native


@pytest.mark.parametrize("make", [kat.DistanceBuckets, lambda: kat.IndexBuckets(*kat.grid_index(3, 4))])
def test_stored_plans_hold_no_device_copies(make):
    """torch.load may move a stored tensor; a plan's copy for a device must not move with it."""
    plan = make()
    want = plan.on(torch.device("cpu"))
    elsewhere = plan.on(torch.device("meta"))
    buffer = io.BytesIO()
    torch.save(plan, buffer)
    buffer.seek(0)
    back = torch.load(buffer, weights_only=False)
    assert not back._on
    assert all(torch.equal(a, b) for a, b in zip(back.on(torch.device("cpu")), want))
    assert all(t.device.type == "meta" for t in elsewhere)
    assert copy.deepcopy(plan) is plan and copy.deepcopy([plan])[0] is plan
    module = copy.deepcopy(kat.GridPositionBias(2, 3, 4))
    assert module.buckets.num_buckets == 35


def test_tables_without_values_are_refused():
    """A table is not stored: one that the meta device lost would come back as whatever memory held."""
    with torch.device("meta"):
        with pytest.raises(ValueError, match="no values"):
            kat.QKNormRope(16, 2, table=kat.rope_table(4, 16))
        plain = kat.QKNormRope(16, 2)
        kept = kat.QKNormRope(16, 2, table=kat.rope_table(4, 16, device="cpu"))
    plain.to_empty(device="cpu")
    table = kat.rope_table(4, 16)
    kept.to_empty(device="cpu").half()
    assert torch.equal(kept.cos, table[0]) and torch.equal(kept.sin, table[1])
    kept.to("meta")
    with pytest.raises(RuntimeError, match="left on the meta device"):
        kept.to_empty(device="cpu")


def operators():
    return _native.ops()


def qk_args(**changed):
    args = dict(q=torch.zeros(2, 3, 4, 16), k=torch.zeros(2, 3, 2, 16), q_weight=torch.ones(16),
                k_weight=torch.ones(16), cos=torch.ones(5, 8), sin=torch.ones(5, 8),
                positions=torch.zeros(2, 3, dtype=torch.int64), eps=1e-6, interleaved=False)
    return {**args, **changed}


LONG = dict(dtype=torch.int64)


@pytest.mark.parametrize("changed", [
    dict(q=torch.zeros(2, 3, 4)), dict(k=torch.zeros(2, 4, 2, 16)), dict(k=torch.zeros(1, 3, 2, 16)),
    dict(k=torch.zeros(2, 3, 2, 8)), dict(k=torch.zeros(2, 3, 2, 16).half()),
    dict(k=torch.zeros(2, 3, 2, 16, device="meta")),
    dict(q=torch.zeros(2, 3, 4, 16).double(), k=torch.zeros(2, 3, 2, 16).double()),
    dict(q=torch.zeros(2, 3, 4, 16).to_sparse()), dict(k=torch.zeros(2, 3, 2, 16).to_sparse()),
    dict(q=torch.zeros(2, 3, 4, 0), k=torch.zeros(2, 3, 4, 0), q_weight=None, k_weight=None),
])
def test_norm_operator_checks_its_heads(changed):
    """Whoever calls the operators past the Python functions: no size is taken on trust."""
    with pytest.raises(RuntimeError, match="^qk_norm_rope: (?!expected CUDA)"):
        operators().qk_norm_rope(**qk_args(**changed))


@pytest.mark.parametrize("changed", [
    dict(q_weight=torch.ones(8)), dict(k_weight=torch.ones(32)[::2]), dict(q_weight=torch.ones(1, 16)),
    dict(q_weight=torch.ones(16).half()), dict(k_weight=torch.ones(16).double()),
    dict(q_weight=torch.ones(16, device="meta")),
    dict(sin=None), dict(cos=None), dict(cos=None, sin=None), dict(sin=torch.ones(5, 4)),
    dict(sin=torch.ones(4, 8)), dict(cos=torch.ones(5, 9), sin=torch.ones(5, 9)),
    dict(cos=torch.ones(5, 8).double()), dict(sin=torch.ones(8, 5).t()), dict(sin=torch.ones(40)),
    dict(cos=torch.ones(2, 8), sin=torch.ones(2, 8), positions=None),
    dict(positions=torch.zeros(2, 3, dtype=torch.int32)), dict(positions=torch.zeros(2, 4, **LONG)),
    dict(positions=torch.zeros(1, 3, **LONG)), dict(positions=torch.zeros(6, **LONG)),
    dict(positions=torch.zeros(2, 3, device="meta", **LONG)),
])
def test_norm_operators_check_the_rest(changed):
    args = qk_args(**changed)
    with pytest.raises(RuntimeError, match="^qk_norm_rope: (?!expected CUDA)"):
        operators().qk_norm_rope(**args)
    del args["q"], args["k"]
    with pytest.raises(RuntimeError, match="^qkv_norm_rope: (?!expected CUDA)"):
        operators().qkv_norm_rope(torch.zeros(2, 3, 64), 2, 1, **args)


@pytest.mark.parametrize("qkv", [torch.zeros(2, 64), torch.zeros(2, 3, 65), torch.zeros(2, 3, 0),
                                 torch.zeros(2, 3, 64).double(), torch.zeros(2, 3, 64).to_sparse(),
                                 torch.zeros(2, 3, 4 * 1025)])
def test_packed_operator_checks_its_input(qkv):
    with pytest.raises(RuntimeError, match="^qkv_norm_rope: (?!expected CUDA)"):
        operators().qkv_norm_rope(qkv, 2, 1, None, None, None, None, None, 1e-6, False)


@pytest.mark.parametrize("q_heads,k_heads", [(0, 1), (2, 0), (-1, 1), (2, 2), (1 << 62, 1 << 62)])
def test_packed_operator_checks_its_heads(q_heads, k_heads):
    args = qk_args()
    with pytest.raises(RuntimeError, match=r"^qkv_norm_rope: expected \[B"):
        operators().qkv_norm_rope(torch.zeros(2, 3, 64), q_heads, k_heads, None, None, args["cos"],
                                  args["sin"], None, 1e-6, False)


def test_good_arguments_get_to_the_device_check():
    for name in ("qk_norm_rope", "qkv_norm_rope", "distance_bias", "index_bias"):
        call = {"qk_norm_rope": lambda: operators().qk_norm_rope(**qk_args()),
                "qkv_norm_rope": lambda: operators().qkv_norm_rope(
                    torch.zeros(2, 3, 64), 2, 1, None, None, None, None, None, 1e-6, False),
                "distance_bias": lambda: operators().distance_bias(**distance_args()),
                "index_bias": lambda: operators().index_bias(**index_args())}[name]
        with pytest.raises(RuntimeError, match=f"^{name}: expected CUDA"):
            call()


def distance_args(**changed):
    b = kat.DistanceBuckets(8, 20)
    args = dict(table=torch.zeros(8, 2), plan=b.on(torch.device("cpu")), buckets=8, reach=b.reach,
                lq=4, lk=5, offset=0, causal=False, type=_native.KAT_DTYPE_F32)
    return {**args, **changed}


def index_args(**changed):
    b = kat.IndexBuckets(*kat.grid_index(3, 4))
    args = dict(table=torch.zeros(35, 2), plan=b.on(torch.device("cpu")), buckets=35, lq=12, lk=12,
                slab_rows=b.slab_rows, slabs=b.slabs, segments=b.segments, type=_native.KAT_DTYPE_F32)
    return {**args, **changed}


def other_plans(plan):
    """The same plan with one tensor longer, of another type or on another device, or left out."""
    for i, t in enumerate(plan):
        for u in (torch.cat([t.flatten().int(), t.flatten().int()[:1]]).to(t.dtype), t.to(torch.int64),
                  t.to("meta")):
            yield (*plan[:i], u, *plan[i + 1:])
        yield (*plan[:i], *plan[i + 1:])


COMMON = [dict(table=torch.zeros(7, 2)), dict(table=torch.zeros(8)), dict(buckets=0), dict(buckets=9),
          dict(lq=-1), dict(lk=1 << 40), dict(type=7)]


@pytest.mark.parametrize("changed", COMMON + [dict(reach=3), dict(reach=-1), dict(reach=1 << 61),
                                              dict(offset=1 << 40), dict(offset=-(1 << 40)),
                                              dict(table=torch.zeros(8, 2).double())])
def test_distance_operator_checks_its_arguments(changed):
    with pytest.raises(RuntimeError, match="^distance_bias: (?!expected CUDA)"):
        operators().distance_bias(**distance_args(**changed))


@pytest.mark.parametrize("changed", COMMON + [dict(lq=13), dict(lk=8), dict(lk=17), dict(slabs=1),
                                              dict(slab_rows=0), dict(segments=3), dict(segments=-1),
                                              dict(lk=1 << 20),
                                              dict(table=torch.zeros(35, 2).double())])
def test_index_operator_checks_its_arguments(changed):
    with pytest.raises(RuntimeError, match="^index_bias: (?!expected CUDA)"):
        operators().index_bias(**index_args(**changed))


def test_operators_check_their_plans():
    for plan in other_plans(distance_args()["plan"]):
        with pytest.raises(RuntimeError, match="^distance_bias: the plan"):
            operators().distance_bias(**distance_args(plan=plan))
    for plan in other_plans(index_args()["plan"]):
        with pytest.raises(RuntimeError, match="^index_bias: the plan"):
            operators().index_bias(**index_args(plan=plan))


class Wrapped(torch.Tensor):
    """A tensor whose values lie in another one, as distributed tensors' do."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype,
                                                   device=inner.device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError(str(func))


@pytest.mark.parametrize("which", ["q", "k", "q_weight", "k_weight", "cos", "sin", "positions"])
def test_wrapped_tensors_are_refused(which):
    """They have no values of their own: a weight without an address would count as none."""
    args = qk_args()
    args[which] = Wrapped(args[which])
    with pytest.raises(RuntimeError, match="^qk_norm_rope: (?!expected CUDA)"):
        operators().qk_norm_rope(**args)
    if which in ("q", "k"):
        return
    del args["q"], args["k"]
    with pytest.raises(RuntimeError, match="^qkv_norm_rope: (?!expected CUDA)"):
        operators().qkv_norm_rope(torch.zeros(2, 3, 64), 2, 1, **args)


def test_wrapped_tables_are_refused():
    with pytest.raises(RuntimeError, match="^distance_bias: (?!expected CUDA)"):
        operators().distance_bias(**distance_args(table=Wrapped(torch.zeros(8, 2))))
    with pytest.raises(RuntimeError, match="^index_bias: (?!expected CUDA)"):
        operators().index_bias(**index_args(table=Wrapped(torch.zeros(35, 2))))
