"""Prompts whose tiles have many rows (the form of every large call): the convolution and the scan of flowedge_b200.ops
against their definitions in 64 bits, with lengths that end before, at and behind every multiple that a kernel counts in."""

import ctypes as C

import pytest
import torch

from flowedge_b200 import engine as fe
from flowedge_b200 import ops
from ops_reference import U, out_step

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _offsets(lengths):
    return torch.tensor([0] + lengths, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()


def _normal(*shape):
    return torch.randn(*shape, device="cuda")


def _wide(rows, width, dtype, extra):
    return _normal(rows, width + extra).to(dtype)[:, extra // 2:extra // 2 + width]


def _sub(dtype):
    return 1e-37 + (6e-8 if dtype == F16 else 0.0)  # half's subnormal step


def _close(got, want, bound, what):
    off = (got.double() - want).abs() - bound
    assert torch.isfinite(got).all(), what
    assert (off <= 0).all(), f"{what}: {off.max().item():.3g} over its bound"


def _lengths(chunk, rows, step):
    """Ragged lengths around multiples of `step` (what a kernel takes at a time) and of the tile; the last fills up."""
    some = [0, chunk - 1, chunk, chunk + 1, 1, 2 * chunk - 1, 2 * chunk, 2 * chunk + 2, 0, step, step + 1, 2 * step - 1,
            2 * step + 3, chunk + step, 3 * chunk + 3, chunk - step + 2, 3]
    return some + [rows - sum(some) - 5, 5]


@pytest.mark.parametrize("chunk,rows,di,dc,dtype,vec,extra", [
    (16, 12300, 512, 4, BF16, 4, 0), (24, 15000, 512, 4, F32, 4, 8), (40, 13001, 1024, 4, BF16, 4, 1024),
    (64, 47000, 512, 4, F16, 4, 0), (40, 9000, 640, 8, F32, 2, 4), (32, 5000, 511, 3, BF16, 1, 1), (64, 11000, 515, 5, F32, 1, 0),
    (56, 18001, 1024, 2, F16, 4, 0), (48, 17000, 1024, 1, F32, 4, 0), (64, 13000, 1026, 6, BF16, 2, 4)])
def test_conv(chunk, rows, di, dc, dtype, vec, extra):
    torch.manual_seed(chunk + di)
    hook = fe.load_library().febtest_conv_chunk
    hook.argtypes = [C.c_size_t] * 3
    lengths = _lengths(chunk, rows, 8)
    n = len(lengths)
    threads = di // vec
    block = min(128, (threads + 31) // 32 * 32)
    assert hook(rows + 4, n, -(-threads // block)) == chunk
    x, w, b = _wide(rows + 4, di, dtype, extra), (torch.rand(di, dc, device="cuda") - 0.5) * 2 * dc ** -0.5, _normal(di)
    window, slots = _normal(n + 2, di, dc), torch.randperm(n + 2, device="cuda")[:n].to(torch.int32)
    slots[6] = -1
    fresh = torch.arange(n, device="cuda") % 3 == 1
    offsets = _offsets(lengths)
    out = torch.full((rows + 4, di), 7.0, dtype=dtype, device="cuda")
    # every sequence behind its window: [window | rows], so that the taps of row t start at t + 1 there
    want, bound, new = out.double(), torch.zeros(rows + 4, di, dtype=torch.float64, device="cuda"), window.double()
    for s, (lo, hi) in enumerate(zip(offsets[:-1].tolist(), offsets[1:].tolist())):
        slot = int(slots[s])
        if slot < 0:
            continue
        past = torch.zeros(dc, di, device="cuda", dtype=torch.float64) if fresh[s] else window[slot].double().t()
        line = torch.cat([past, x[lo:hi].double()])
        taps = line.unfold(0, dc, 1)[1:]  # [rows][di][dc]
        products = taps * w.double()
        v = b.double() + products.sum(2)
        u = v * torch.sigmoid(v)
        want[lo:hi] = u
        bound[lo:hi] = (1.1 * (dc + 1) * U * (b.double().abs() + products.abs().sum(2)) + 8 * U * u.abs() +
                        out_step(dtype) * u.abs() * 1.01 + _sub(dtype))
        new[slot] = line[line.shape[0] - dc:].t()
    ops.conv(x, w, b, window=window, offsets=offsets, slots=slots, fresh=fresh, out=out)
    _close(out, want, bound, "u")
    assert torch.equal(window.double(), new)


def _scan_chunk(rows, n, di, ds, dr):
    """The tile's rows, from the size of the workspace: dt of all rows, then 1 + ds rows of channels for every tile."""
    size = fe.load_library().fe_selective_scan_workspace(ops._SCAN.pack(
        ops._SCAN.size, 0, 0, ds, rows, di, dr, n, n, di, dr + 2 * ds, di, di, ds * di, 0, 0, 0, 0, 0, 0, 0, 0, 0, 64, 0, 0, 0,
        0, 0))
    tiles = (size - (rows * di * 4 + 255) // 256 * 256) // ((1 + ds) * di * 4) - n
    chunk = 16
    while rows // chunk > tiles:
        chunk *= 2
    assert rows // chunk == tiles
    return chunk


def _scan_reference(c, offsets, slots, fresh, out, chunk):
    """All sequences side by side, longest first, one row after the other: (y, state, bound on y, bound on state).

    The bound goes by the roundings of the kernel: those of dt (its projection, and 10 steps of its own), of the decay's
    exponent and exponential, of each sum; and where tiles join, those of the sum of the tile's steps (four at a time,
    then one addition for each four), which stand in the decay of what entered the tile."""
    dtype = out.dtype
    u, proj, a, d, dt_w, dt_b = (c[k].double() for k in ("u", "proj", "a", "d", "dt_w", "dt_b"))
    ds, dr = a.shape[0], dt_w.shape[0]
    o, slot = offsets.tolist(), slots.tolist()
    order = sorted((s for s in range(len(slot)) if slot[s] >= 0), key=lambda s: o[s] - o[s + 1])
    begin = torch.tensor([o[s] for s in order], device="cuda")
    length = [o[s + 1] - o[s] for s in order]
    pool = torch.tensor([slot[s] for s in order], device="cuda")
    h = c["state"].double()[pool]
    if fresh is not None:
        h[fresh[torch.tensor(order, device="cuda")] != 0] = 0.0
    y, state = out.double(), c["state"].double()
    y_bound, e = torch.zeros_like(y), torch.zeros_like(h)
    entered, total = h.clone(), torch.zeros_like(h[:, 0])
    for t in range(max(length)):
        k = sum(v > t for v in length)
        at = begin[:k] + t
        p, ut = proj[at], u[at]
        if t and t % chunk == 0:  # the tile behind these rows joined: what entered it, decayed by the sum of its steps
            x = (total[:k, None] * a).abs()
            e[:k] += torch.exp(-x) * entered[:k].abs() * x * (chunk / 4 + 8) * U
            entered[:k], total[:k] = h[:k], 0.0
        pre = p[:, :dr] @ dt_w + dt_b
        dt_rel = (dr + 1) * U * (p[:, :dr].abs() @ dt_w.abs() + dt_b.abs()) + 10 * U
        dt = torch.logaddexp(pre, torch.zeros_like(pre))
        total[:k] += dt
        x = dt[:, None] * a
        decay = torch.exp(x)
        decay_rel = x.abs() * (dt_rel[:, None] + 3 * U) + 5 * U
        add = (dt * ut)[:, None] * p[:, dr:dr + ds, None]
        e[:k] = decay * e[:k] * (1 + decay_rel) + (decay * h[:k]).abs() * decay_rel + add.abs() * (dt_rel[:, None] + 4 * U)
        h[:k] = decay * h[:k] + add
        e[:k] += U * h[:k].abs()
        cn = p[:, dr + ds:, None]
        v = d * ut + (h[:k] * cn).sum(1)
        err = (e[:k] * cn.abs()).sum(1) + (ds + 2) * U * ((d * ut).abs() + (h[:k] * cn).abs().sum(1))
        gate, gate_rel = torch.ones_like(v), 0.0
        if c["z"] is not None:
            z = c["z"][at].double()
            gate, gate_rel = z * torch.sigmoid(z), (8 + 2 * z.abs()) * U
        y[at] = v * gate
        y_bound[at] = 1.05 * (err * gate.abs() + y[at].abs() * (gate_rel + 2 * U) + out_step(dtype) * y[at].abs() * 1.01)
    bound = torch.zeros_like(state)
    state[pool], bound[pool] = h, e
    return y, state, y_bound + _sub(dtype), bound + 1e-37


@pytest.mark.parametrize("chunk,rows,di,ds,dr,dtype,gated,fresh,extra", [
    (32, 2000, 2050, 16, 20, F32, True, False, 0), (64, 3700, 2050, 16, 32, BF16, True, True, 4),
    (64, 3900, 2048, 8, 9, F32, False, True, 0), (64, 3800, 1999, 32, 16, F16, True, False, 1),
    (128, 7300, 2048, 16, 64, F32, True, False, 2048), (64, 3750, 2048, 12, 7, BF16, False, False, 0),
    (128, 4000, 4096, 5, 4, F32, True, True, 0), (256, 7200, 4100, 16, 16, BF16, True, False, 0),
    (64, 7400, 1024, 28, 300, F32, True, False, 0)])
def test_scan(chunk, rows, di, ds, dr, dtype, gated, fresh, extra):
    torch.manual_seed(chunk + di + ds)
    lengths = _lengths(chunk, rows, 16)
    n = len(lengths)
    assert _scan_chunk(rows + 4, n, di, ds, dr) == chunk
    case = {"u": _wide(rows + 4, di, dtype, extra), "proj": _wide(rows + 4, dr + 2 * ds, dtype, extra % 8),
            "a": -(torch.rand(ds, di, device="cuda") * ds + 0.5), "d": _normal(di), "dt_w": _normal(dr, di) * 0.5 * dr ** -0.5,
            "dt_b": torch.rand(di, device="cuda") * 4 - 7, "z": _wide(rows + 4, di, dtype, extra) if gated else None,
            "state": _normal(n + 2, ds, di)}
    slots = torch.randperm(n + 2, device="cuda")[:n].to(torch.int32)
    slots[6] = -1
    flags = torch.arange(n, device="cuda") % 3 == 1 if fresh else None
    offsets = _offsets(lengths)
    out = torch.full((rows + 4, di), 7.0, dtype=dtype, device="cuda")
    y, state, bound, state_bound = _scan_reference(case, offsets, slots, flags, out, chunk)
    ops.scan(*(case[k] for k in ("u", "proj", "a", "d", "dt_w", "dt_b")), z=case["z"], state=case["state"], offsets=offsets,
             slots=slots, fresh=flags, out=out)
    _close(out, y, bound, "y")
    _close(case["state"], state, state_bound, "state")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lengths", [None, [1, 3, 16, 9, 15, 0, 4]])
def test_scan_within_one_tile_is_held_to_its_own_roundings(dtype, lengths):
    """Single tokens and prompts of one tile join no sum of steps: their bound has none."""
    torch.manual_seed(3)
    rows, di, ds, dr = (sum(lengths) if lengths else 40), 2050, 16, 20
    n = len(lengths) if lengths else rows
    offsets = _offsets(lengths) if lengths else torch.arange(rows + 1, dtype=torch.int32, device="cuda")
    case = {"u": _normal(rows, di).to(dtype), "proj": _normal(rows, dr + 2 * ds).to(dtype),
            "a": -(torch.rand(ds, di, device="cuda") * ds + 0.5), "d": _normal(di), "dt_w": _normal(dr, di) * 0.5 * dr ** -0.5,
            "dt_b": torch.rand(di, device="cuda") * 4 - 5, "z": _normal(rows, di).to(dtype), "state": _normal(n, ds, di)}
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    out = torch.zeros(rows, di, dtype=dtype, device="cuda")
    y, state, bound, state_bound = _scan_reference(case, offsets, slots, None, out, 1 << 30)
    ops.scan(*(case[k] for k in ("u", "proj", "a", "d", "dt_w", "dt_b")), z=case["z"], state=case["state"],
             offsets=offsets if lengths else None, slots=slots, out=out)
    _close(out, y, bound, "y")
    _close(case["state"], state, state_bound, "state")
