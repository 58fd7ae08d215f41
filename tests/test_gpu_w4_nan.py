"""NaN in a float32 x of the 4-bit products, whatever its payload."""

import pytest
import torch

from flowedge_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k", [128, 127])
@pytest.mark.parametrize("layout", ["blocks", "rows"])
def test_a_nan_of_every_payload_stays_one(k, layout):
    """x is split into terms of its leading bits: a NaN whose payload sits in the low bits alone must not read as an infinity."""
    packed, scales = ops.w4_quantize(torch.eye(128, device="cuda")[:, :k].contiguous() * 7, 32, layout=layout)
    bits = [0x7F800001, 0x7F80FFFF, -0x7FFFFF, 0x7FC00000, 0x7F810000]
    x = torch.zeros(len(bits), k, device="cuda")
    x[:, 5] = torch.tensor(bits, dtype=torch.int32, device="cuda").view(torch.float32)
    assert torch.isnan(x[:, 5]).all()
    assert torch.isnan(ops.w4_matvec(x, packed, scales, group=32)[:, 5]).all()
