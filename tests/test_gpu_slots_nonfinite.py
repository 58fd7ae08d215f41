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


def _scan_case(seed, rows, di, ds, dr, dtype, pool):
    g = torch.Generator().manual_seed(seed)
    return {"u": torch.randn(rows, di, generator=g).to(dtype).cuda(), "proj": torch.randn(rows, dr + 2 * ds, generator=g).to(dtype).cuda(),
            "a": -(torch.rand(ds, di, generator=g) * ds + 0.5).cuda(), "d": torch.randn(di, generator=g).cuda(),
            "dt_w": (torch.randn(dr, di, generator=g) * 0.5 * dr ** -0.5).cuda(),
            "dt_b": (torch.rand(di, generator=g) * 4 - 5).cuda(), "z": torch.randn(rows, di, generator=g).to(dtype).cuda(),
            "state": torch.randn(pool, ds, di, generator=g).cuda()}


def _check_scan(case, offsets):
    out = torch.full_like(case["u"], 7.0)
    keys = ("u", "proj", "a", "d", "dt_w", "dt_b", "z", "state")
    y, pool, bound, pool_bound = ref.scan(*(case[k] for k in keys), offsets, None, None, out)
    ops.scan(*(case[k] for k in keys[:1] + keys[1:6]), z=case["z"], state=case["state"], offsets=offsets, out=out)
    _same(out, y, bound, "y")
    _same(case["state"], pool, pool_bound, "state")


# sequences, channels: dt of tokens made in the scan, beforehand (from 16 sequences that fill the GPU), and of prompts
FORMS = [("tokens", 6, 130), ("tokens", 40, 2050), ("prompts", 5, 130), ("prompts", 5, 131)]


def _shape(form, n):
    lengths = [1] * n if form == "tokens" else [3, 1, 12, 9, 16][:n]
    return sum(lengths), None if form == "tokens" else _offsets(lengths)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form,n,di", FORMS)
@pytest.mark.parametrize("value", [INF, -INF, NAN])
def test_scan_with_an_infinite_step_input(dtype, form, n, di, value):
    """dt = softplus(dt_in dt_w + dt_b) of a row with an infinite dt_in: infinite, or zero where the weight's sign makes
    it minus infinity, and NaN where the weight is zero."""
    rows, offsets = _shape(form, n)
    case = _scan_case(1, rows, di, 16, 8, dtype, n)
    case["dt_w"][3, ::7] = 0.0
    case["proj"][2, 3] = value
    case["proj"][5, 7] = value
    _check_scan(case, offsets)


@pytest.mark.parametrize("form,n,di", FORMS)
@pytest.mark.parametrize("value", [INF, -INF, NAN])
def test_scan_with_an_infinite_step_weight(form, n, di, value):
    rows, offsets = _shape(form, n)
    case = _scan_case(2, rows, di, 8, 20, torch.float32, n)
    case["dt_w"][11, 5] = value
    case["dt_w"][0, 64] = value
    case["dt_b"][1] = value
    case["proj"][1, 11] = 0.0
    _check_scan(case, offsets)


@pytest.mark.parametrize("form,n,di", FORMS)
def test_scan_with_a_step_input_at_the_end_of_float32(form, n, di):
    """A dt_in that bf16 rounds to infinity is finite all the same."""
    rows, offsets = _shape(form, n)
    case = _scan_case(3, rows, di, 16, 8, torch.float32, n)
    case["dt_w"] *= 1e-30
    case["proj"][2, 3], case["proj"][4, 0] = 3.4e38, -3.4e38
    _check_scan(case, offsets)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form,n,di", FORMS)
@pytest.mark.parametrize("ds", [1, 5, 8, 12, 15, 16, 20, 31, 32])
@pytest.mark.parametrize("value", [INF, NAN])
def test_scan_with_an_infinite_input_and_few_states(dtype, form, n, di, ds, value):
    """States that the call does not have add nothing, whatever u and dt hold."""
    rows, offsets = _shape(form, n)
    case = _scan_case(4, rows, di, ds, 4, dtype, n)
    case["proj"][:, 4:] = case["proj"][:, 4:].abs() + 0.25  # B and C of one sign: sums of infinities of one sign
    case["d"] = case["d"].abs() + 0.1
    case["state"] = case["state"].abs()
    case["u"][1, ::3] = value
    case["u"][5, 1] = value
    case["dt_b"][4] = INF
    _check_scan(case, offsets)


@pytest.mark.parametrize("form,n,di", FORMS)
@pytest.mark.parametrize("ds", [4, 16, 24])
def test_scan_with_a_missing_decay(form, n, di, ds):
    """A NaN in a spoils its channel, in every form alike; the others keep their values."""
    rows, offsets = _shape(form, n)
    case = _scan_case(5, rows, di, ds, 4, torch.float32, n)
    case["a"][0, 3] = NAN
    case["a"][1, 9] = NAN
    case["a"][ds - 1, 20] = NAN
    _check_scan(case, offsets)


@pytest.mark.parametrize("form,n,di", FORMS)
def test_scan_decays_to_nothing(form, n, di):
    """exp(dt a) far below float32's range takes the old state away, an infinite one too where it is zero in 64 bits."""
    rows, offsets = _shape(form, n)
    case = _scan_case(6, rows, di, 16, 4, torch.float32, n)
    case["a"][:, 5] = -1e30
    case["state"][:, :, 5] = 3e38
    _check_scan(case, offsets)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ds", [8, 16])
def test_an_infinite_state_stays_infinite_over_tiles(dtype, ds):
    """Tiles of 16 rows whose decay is below float32's range, while every row's is above it: the state behind an infinite
    input is infinite in prompts as it is in single tokens."""
    lengths, di = [75, 16, 40], 130
    case = _scan_case(7, sum(lengths), di, ds, 4, dtype, 3)
    case["a"] = -(torch.rand(ds, di, generator=torch.Generator().manual_seed(1)) * 6 + 2).cuda()
    case["dt_w"] *= 0.1
    case["dt_b"] = torch.full((di,), 5.0, device="cuda")  # sums of 16 steps near 80, decays e^-160 to e^-640
    case["proj"][:, 4:] = case["proj"][:, 4:].abs() + 0.25
    case["u"], case["d"], case["state"] = case["u"].abs(), case["d"].abs() + 0.1, case["state"].abs()
    case["u"][3, ::3] = INF
    case["u"][95, 1] = INF
    case["state"][1, 0, 5] = INF
    _check_scan(case, _offsets(lengths))
