"""Infinities, NaN and padded states in the slot-state convolution and scan (flowedge_b200.ops), against the definitions
in 64 bits: a value that the definition does not use spoils nothing."""

import pytest
import torch

import ops_reference as ref
from flowedge_b200 import ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
INF, NAN = float("inf"), float("nan")


def _offsets(lengths):
    return torch.tensor([0] + lengths, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()


def _same(got, want, bound, what):
    """NaN and infinities where the definition has them, finite values within the bound (where it is finite itself)."""
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]) and not torch.isinf(got[~inf]).any(), what
    fine = torch.isfinite(want)
    off = (got - want).abs()[fine] - torch.nan_to_num(bound[fine], nan=INF, posinf=INF)
    assert (off <= 0).all(), f"{what}: {off.max().item():.3g} over its bound"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dc", range(1, 9))
@pytest.mark.parametrize("di", [8, 7])
@pytest.mark.parametrize("form", ["prompts", "tokens"])
def test_conv_uses_its_own_taps_alone(dtype, dc, di, form):
    """An infinite or NaN input reaches the rows that read it and no others; the window's oldest input is never read."""
    g = torch.Generator().manual_seed(dc)
    lengths = [40, 3, 25, 0] if form == "prompts" else [1] * 12
    rows, n = sum(lengths), len(lengths)
    x = torch.randn(rows, di, generator=g).to(dtype)
    for i, v in enumerate([INF, -INF, NAN]):
        x[4 * i + 1 if form == "tokens" else 9 * i + 4, i] = v
    x[rows - 2, 4] = INF
    w = (torch.rand(di, dc, generator=g) + 0.1).cuda()
    b = torch.randn(di, generator=g).cuda()
    window = torch.randn(n, di, dc, generator=g)
    window[:, :, 0] = torch.tensor([INF, -INF, NAN])[torch.arange(di) % 3]
    if dc > 1:
        window[0, 6 % di, dc - 1] = INF  # the newest input of the past: read dc - 1 times
    args = (x.cuda(), w, b, window.cuda(), _offsets(lengths) if form == "prompts" else None, None, None)
    out = torch.full((rows, di), 7.0, dtype=dtype, device="cuda")
    want, win, bound = ref.conv(*args, out)
    ops.conv(args[0], w, b, window=args[3], offsets=args[4], out=out)
    _same(out, want, bound, "u")
    _same(args[3], win, torch.zeros_like(win), "window")
