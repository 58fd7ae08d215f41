"""Pools without slots and calls without sequences (flowedge_b200.ops)."""

import pytest
import torch

from flowedge_b200 import ops

pytestmark = pytest.mark.gpu


def _call(name, rows, window, state, **kw):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(rows, 32, generator=g).cuda()
    if name == "conv":
        return ops.conv(x, torch.ones(32, 4, device="cuda"), torch.zeros(32, device="cuda"), window=window, **kw)
    proj = torch.randn(rows, 24, generator=g).cuda()
    weights = [-torch.ones(8, 32, device="cuda"), torch.ones(32, device="cuda"), torch.ones(8, 32, device="cuda"),
               torch.zeros(32, device="cuda")]
    return ops.scan(x, proj, *weights, state=state, **kw)


@pytest.mark.parametrize("name", ["conv", "scan"])
@pytest.mark.parametrize("form", ["tokens", "prompts"])
def test_a_pool_without_slots_is_refused(name, form):
    """It ran without states, whatever the slots."""
    offsets = None if form == "tokens" else torch.tensor([0, 3, 4], dtype=torch.int32, device="cuda")
    n = 4 if form == "tokens" else 2
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    empty = torch.empty(0, 32, 4, device="cuda"), torch.empty(0, 8, 32, device="cuda")
    with pytest.raises(ops.FlowEdgeError, match="no slots"):
        _call(name, 4, *empty, slots=slots, offsets=offsets)
    assert _call(name, 4, None, None, slots=slots, offsets=offsets).shape == (4, 32)  # without states
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert _call(name, 0, *empty, offsets=none if form == "prompts" else None).shape == (0, 32)


def test_prompts_that_are_all_empty():
    """No rows at all: a fresh sequence's slot becomes zero, another's stays."""
    offsets = torch.zeros(4, dtype=torch.int32, device="cuda")
    slots = torch.tensor([2, 0, -1], dtype=torch.int32, device="cuda")
    fresh = torch.tensor([1, 0, 1], dtype=torch.uint8, device="cuda")
    for name, pool in (("conv", torch.ones(3, 32, 4, device="cuda")), ("scan", torch.ones(3, 8, 32, device="cuda"))):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = _call(name, 0, pool, pool, offsets=offsets, slots=slots, fresh=fresh, status=status)
        assert out.shape == (0, 32) and int(status) == 0
        assert (pool[:2] == 1).all() and (pool[2] == 0).all()
