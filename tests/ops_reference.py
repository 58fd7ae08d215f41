"""The operators of flowedge_b200.ops from their definitions in 64 bits, one sequence and one row after the other, with
a bound on what a 32-bit evaluation may be off (the kernels' roundings, propagated through the recurrence)."""

import torch

U = 2.0 ** -24  # half a step of float32


def out_step(dtype):
    """Relative error of one rounding to the output's type."""
    return torch.finfo(dtype).eps / 2


def silu(x):
    return x * torch.sigmoid(x)


def spans(rows, offsets):
    if offsets is None:
        return [(i, i + 1) for i in range(rows)]
    o = offsets.tolist()
    return list(zip(o[:-1], o[1:]))


def conv(x, weight, bias, window, offsets, slots, fresh, out):
    """(u, window, bound on u's error); `out` holds what skipped rows keep."""
    dtype = out.dtype
    x, w, b = x.double().cpu(), weight.double().cpu(), bias.double().cpu()
    u, win = out.double().cpu(), None if window is None else window.double().cpu()
    bound = torch.zeros_like(u)
    dc = w.shape[1]
    for s, (lo, hi) in enumerate(spans(x.shape[0], offsets)):
        slot = s if slots is None else int(slots[s])
        if slot < 0:
            continue
        held = torch.zeros(x.shape[1], dc, dtype=torch.float64)
        if win is not None and (fresh is None or not bool(fresh[s])):
            held = win[slot].clone()
        for t in range(lo, hi):
            held = torch.cat([held[:, 1:], x[t][:, None]], 1)
            v = b + (held * w).sum(1)
            u[t] = silu(v)
            # dc fused products and their sum, then SiLU (slope at most 1.1) with its own few roundings
            size = b.abs() + (held * w).abs().sum(1)
            bound[t] = 1.1 * (dc + 1) * U * size + 8 * U * u[t].abs() + out_step(dtype) * u[t].abs() * 1.01
        if win is not None:
            win[slot] = held
    return u, win, bound + 1e-37 + (6e-8 if dtype == torch.float16 else 0.0)  # half's subnormal step


def scan(u, proj, a, d, dt_w, dt_b, z, state, offsets, slots, fresh, out, longest_sum=64):
    """(y, state, bound on y, bound on state).  `longest_sum` is the number of roundings behind a sum of steps (a piece
    of a prompt is scanned from the sum of the steps before it)."""
    dtype = out.dtype
    u, proj = u.double().cpu(), proj.double().cpu()
    a, d, dt_w, dt_b = (t.double().cpu() for t in (a, d, dt_w, dt_b))
    z = None if z is None else z.double().cpu()
    y, pool = out.double().cpu(), None if state is None else state.double().cpu()
    y_bound, pool_bound = torch.zeros_like(y), None if pool is None else torch.zeros_like(pool)
    ds, dr = a.shape[0], dt_w.shape[0]
    for s, (lo, hi) in enumerate(spans(u.shape[0], offsets)):
        slot = s if slots is None else int(slots[s])
        if slot < 0:
            continue
        h = torch.zeros_like(a)
        if pool is not None and (fresh is None or not bool(fresh[s])):
            h = pool[slot].clone()
        e = torch.zeros_like(h)  # bound on h's error
        for t in range(lo, hi):
            p = proj[t]
            pre = p[:dr] @ dt_w + dt_b
            # the projection's roundings; softplus'(x) <= softplus(x), so they are dt's relative error, and its own
            dt_rel = (dr + 1) * U * (p[:dr].abs() @ dt_w.abs() + dt_b.abs()) + 10 * U
            dt = torch.logaddexp(pre, torch.zeros_like(pre))
            decay = torch.exp(dt * a)
            # the exponent's error, the exponential's (4 U), and the sum of steps where pieces are joined
            decay_rel = (dt * a).abs() * (dt_rel + (3 + longest_sum) * U) + 5 * U
            add = (dt * u[t])[None, :] * p[dr:dr + ds, None]
            e = decay * e * (1 + decay_rel) + (decay * h).abs() * decay_rel + add.abs() * (dt_rel + 4 * U)
            h = decay * h + add
            e = e + U * h.abs()
            c = p[dr + ds:, None]
            v = d * u[t] + (h * c).sum(0)
            size = (d * u[t]).abs() + (h * c).abs().sum(0)
            err = (e * c.abs()).sum(0) + (ds + 2) * U * size
            gate = torch.ones_like(v) if z is None else silu(z[t])
            y[t] = v * gate
            # __expf in the gate: a few steps, and one more for every unit of its argument
            gate_rel = 0.0 if z is None else (8 + 2 * z[t].abs()) * U
            y_bound[t] = err * gate.abs() + y[t].abs() * (gate_rel + 2 * U) + out_step(dtype) * y[t].abs() * 1.01
        if pool is not None:
            pool[slot], pool_bound[slot] = h, e
    return y, pool, y_bound * 1.05 + 1e-37 + (6e-8 if dtype == torch.float16 else 0.0), pool_bound
