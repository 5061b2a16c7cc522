"""Calls of the attention-input operators that need no GPU: stored and copied plans."""

import copy
import io

import pytest
import torch

import rational_kat_cu_b200 as kat


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
