"""Measured cases of the serving operators (flowedge_b200.ops): the short causal convolution and the selective scan
with their slot states, products with 4-bit weights, and the residual norm.

`own` false computes each operator in elementary torch operations; `own` true calls the framework.  `exact` evaluates
the definitions in 64 bits.
"""

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZES = {"fp32": 4, "bf16": 2, "fp16": 2}
# nibble i of a 32-bit word of 4-bit weights holds element NIBBLE[i] of the word's eight
NIBBLE = (0, 2, 4, 6, 1, 3, 5, 7)


def listed():
    return [
        # one streaming client of the 512-wide encoder (d_inner 1024): pure latency
        {"name": "conv_token_1", "op": "conv", "form": "tokens", "seqs": 1, "pad": 0, "di": 1024, "dc": 4,
         "dtype": "fp32"},
        # a batch of ragged prompts through the encoder's conv, empty and one-token prompts among them
        {"name": "conv_prompts_ragged", "op": "conv", "form": "prompts", "seqs": 96, "rows": 12289, "di": 1024, "dc": 4,
         "fresh": True, "dtype": "bf16"},
        # one streaming client
        {"name": "scan_token_1", "op": "scan", "form": "tokens", "seqs": 1, "pad": 0, "di": 1024, "ds": 16, "dr": 32,
         "dtype": "fp32"},
        # a padded decode batch over many slots, a wider encoder
        {"name": "scan_tokens_512", "op": "scan", "form": "tokens", "seqs": 512, "pad": 37, "di": 2048, "ds": 16,
         "dr": 64, "dtype": "bf16"},
        # the encoder's 128-token prompt, alone
        {"name": "scan_prompt_128", "op": "scan", "form": "prompts", "seqs": 1, "rows": 128, "di": 1024, "ds": 16,
         "dr": 32, "fresh": True, "dtype": "fp32"},
        # a batch of ragged prompts, continuing from states held in slots
        {"name": "scan_prompts_ragged", "op": "scan", "form": "prompts", "seqs": 96, "rows": 12289, "di": 1024,
         "ds": 16, "dr": 32, "fresh": False, "dtype": "fp32"},
        # one long history: the sequence has to be split to fill the GPU
        {"name": "scan_prompt_16k", "op": "scan", "form": "prompts", "seqs": 1, "rows": 16384, "di": 2048, "ds": 16,
         "dr": 64, "fresh": True, "dtype": "bf16"},
        # the encoder's in-projection for one token
        {"name": "w4_in_proj_1", "op": "w4", "rows": 1, "m": 2048, "k": 512, "group": 64, "dtype": "fp32"},
        # an odd-sized projection for a small decode batch
        {"name": "w4_odd_11", "op": "w4", "rows": 11, "m": 4100, "k": 2056, "group": 32, "dtype": "fp16"},
        # a large projection for one token: the weights' stream from memory
        {"name": "w4_large_1", "op": "w4", "rows": 1, "m": 16384, "k": 8192, "group": 128, "dtype": "bf16"},
        # the residual and the next layer's norm for one token
        {"name": "norm_1", "op": "norm", "rows": 1, "dim": 512, "dtype": "fp32", "post": False, "gate": "none",
         "rdtype": "fp32"},
        # a prompt batch with both norms and a gate per token
        {"name": "norm_gated_16k", "op": "norm", "rows": 16384, "dim": 2048, "dtype": "bf16", "post": True,
         "gate": "rows", "rdtype": "fp32"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv", "scan", "scan", "w4", "norm"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op in ("conv", "scan"):
        case = {"op": op, "form": rng.choice(["tokens", "prompts"]), "di": _log_int(rng, 64, 2048), "dtype": dtype}
        if rng.random() < 0.6:
            case["di"] = max(8, case["di"] // 8 * 8)
        if op == "conv":
            case["dc"] = rng.choice([2, 3, 4, 4, 5, 8])
        else:
            case["ds"] = rng.choice([4, 8, 12, 16, 16, 16, 32])
            case["dr"] = _log_int(rng, 4, 64)
        if case["form"] == "tokens":
            case["seqs"] = _log_int(rng, 1, 512)
            case["pad"] = rng.randrange(0, case["seqs"] // 4 + 1)
        else:
            case["seqs"] = _log_int(rng, 1, 128)
            case["rows"] = _log_int(rng, case["seqs"], 16384)
            case["fresh"] = rng.random() < 0.5
            if op == "scan":
                most = 16384 * 2048 * 16 // (case["di"] * case["ds"])
                case["rows"] = max(1, min(case["rows"], most))
        return case
    if op == "w4":
        group = rng.choice([32, 64, 128])
        return {"op": op, "rows": _log_int(rng, 1, 32), "m": _log_int(rng, 64, 16384), "k": _log_int(rng, 64, 8192),
                "group": group, "dtype": dtype}
    dim = _log_int(rng, 64, 8192)
    rows = min(_log_int(rng, 1, 16384), 16384 * 2048 // dim)
    return {"op": op, "rows": rows, "dim": dim, "dtype": dtype, "post": rng.random() < 0.5,
            "gate": rng.choice(["none", "rows", "one"]), "rdtype": rng.choice(["fp32", dtype])}


def _seqs(case, g):
    """Lengths (with empty and one-token prompts where there are several), offsets, slots and the pool's size."""
    n = case["seqs"]
    if case["form"] == "tokens":
        n_slots = n + 5
        slots = torch.randperm(n_slots, generator=g)[:n]
        if case["pad"]:
            slots[n - case["pad"]:] = -1
        return None, slots.to(torch.int32).cuda(), n_slots, n
    rows = case["rows"]
    cuts = torch.sort(torch.randint(0, rows + 1, (n - 1,), generator=g)).values
    if n > 4:
        cuts[1] = cuts[0]  # an empty prompt
        cuts[3] = min(int(cuts[2]) + 1, int(cuts[4]) if n > 5 else rows)  # at most one token
    offsets = torch.cat([torch.zeros(1, dtype=torch.long), cuts, torch.tensor([rows])])
    n_slots = n + 3
    slots = torch.randperm(n_slots, generator=g)[:n]
    return offsets.to(torch.int32).cuda(), slots.to(torch.int32).cuda(), n_slots, rows


def prepare(case, seed):
    g = torch.Generator().manual_seed(seed)
    cg = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=cg, device="cuda") * scale

    def uniform(*shape, lo=0.0, hi=1.0):
        return torch.rand(*shape, generator=cg, device="cuda") * (hi - lo) + lo

    s = {"case": case}
    if case["op"] in ("conv", "scan"):
        di = case["di"]
        s["offsets"], s["slots"], n_slots, rows = _seqs(case, g)
        s["fresh"] = None
        if case["form"] == "prompts" and case["fresh"]:
            s["fresh"] = torch.ones(case["seqs"], dtype=torch.uint8, device="cuda")
        s["out"] = torch.zeros(rows, di, dtype=dt, device="cuda")
        xz = normal(rows, 2 * di).to(dt)  # the in-projection's rows: x, then the gate z
    if case["op"] == "conv":
        dc = case["dc"]
        s["x"] = xz[:, :di]
        s["w"] = uniform(di, dc, lo=-dc ** -0.5, hi=dc ** -0.5)
        s["b"] = uniform(di, lo=-dc ** -0.5, hi=dc ** -0.5)
        s["window"] = normal(n_slots, di, dc)
    elif case["op"] == "scan":
        ds, dr = case["ds"], case["dr"]
        s["z"] = xz[:, di:]
        s["u"] = torch.nn.functional.silu(normal(rows, di)).to(dt)
        s["proj"] = normal(rows, dr + 2 * ds).to(dt)  # [dt_in | B | C]
        s["a"] = -(torch.arange(1, ds + 1, device="cuda", dtype=torch.float32)[:, None] * uniform(ds, di, lo=0.8, hi=1.2))
        s["d"] = 1.0 + normal(di, scale=0.1)
        s["dt_w"] = normal(dr, di, scale=0.3 * dr ** -0.5)  # laid out with the channels innermost
        step = torch.exp(uniform(di, lo=math.log(1e-3), hi=math.log(0.1)))
        s["dt_b"] = step + torch.log(-torch.expm1(-step))  # softplus(dt_b) = step
        s["state"] = normal(n_slots, ds, di, scale=0.5)
    elif case["op"] == "w4":
        m, k, group = case["m"], case["k"], case["group"]
        words = (k + 31) // 32 * 4
        q = torch.randint(0, 16, (m, words * 8), generator=cg, device="cuda", dtype=torch.int64)
        q[:, k:] = 8  # behind the last column: zero
        q = q.view(m, words, 8)[:, :, list(NIBBLE)]
        byte = q[:, :, 0::2] | (q[:, :, 1::2] << 4)
        s["packed"] = byte.to(torch.uint8).reshape(m, words * 4).contiguous()
        s["scales"] = uniform(m, (k + group - 1) // group, lo=0.5, hi=1.5).mul_(0.2 * k ** -0.5).half()
        s["x"] = normal(case["rows"], k).to(dt)
    else:
        rows, dim = case["rows"], case["dim"]
        s["x"] = normal(rows, dim).to(dt)
        s["residual"] = normal(rows, dim, scale=2.0).to(DTYPES[case["rdtype"]])
        s["weight"] = 1.0 + normal(dim, scale=0.2)
        s["post"] = 1.0 + normal(dim, scale=0.2) if case["post"] else None
        s["gate"] = None if case["gate"] == "none" else normal(rows if case["gate"] == "rows" else 1, dim).to(dt)
    return s


def _unpack(packed, k):
    """Whole numbers 0 .. 15 of packed 4-bit weights, [m][k]."""
    m = packed.shape[0]
    nib = torch.stack([packed & 15, packed >> 4], -1).view(m, -1, 8)
    place = torch.tensor(NIBBLE, device=packed.device).argsort()
    return nib[:, :, place].reshape(m, -1)[:, :k]


def _bounds(state, rows):
    """Start and end rows of every sequence, as 64-bit tensors."""
    if state["offsets"] is None:
        start = torch.arange(rows, device="cuda")
        return start, start + 1
    o = state["offsets"].long()
    return o[:-1], o[1:]


def _conv(state):
    x, w, window, out = state["x"], state["w"], state["window"], state["out"]
    rows, di = x.shape
    dc = w.shape[1]
    start, end = _bounds(state, rows)
    live = state["slots"] >= 0
    slot = state["slots"].long().clamp(min=0)
    old = window[slot]
    if state["fresh"] is not None:
        old = old * (state["fresh"] == 0)[:, None, None]
    pos = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(end, pos, right=True)  # the sequence of every row
    back = torch.arange(dc - 1, -1, -1, device="cuda")
    at = pos[:, None] - back  # [rows][dc] input rows
    inside = at >= start[seq][:, None]
    taps = x.float()[at.clamp(min=0)]  # [rows][dc][di]
    before = (dc + at - start[seq][:, None]).clamp(0, dc - 1)
    held = old.permute(0, 2, 1)[seq[:, None], before]
    taps = torch.where(inside[:, :, None], taps, held)
    acc = state["b"] + (taps * w.t()).sum(1)
    u = acc / (1 + torch.exp(-acc))
    rowlive = live[seq]
    out.copy_(torch.where(rowlive[:, None], u, out.float()).to(out.dtype))
    # the last dc inputs of every sequence, older ones from its window
    last = end[:, None] - dc + torch.arange(dc, device="cuda")
    new_in = x.float()[last.clamp(0, max(rows - 1, 0))]  # [seqs][dc][di]
    keep = (last - start[:, None] + dc).clamp(0, dc - 1)
    kept = torch.gather(old.permute(0, 2, 1), 1, keep[:, :, None].expand(-1, -1, di))
    new = torch.where((last >= start[:, None])[:, :, None], new_in, kept).permute(0, 2, 1)
    window[slot[live]] = new[live]
    return {"u": out, "window": window}


def _scan(state):
    u, z, proj, h0, out = state["u"].float(), state["z"].float(), state["proj"].float(), state["state"], state["out"]
    rows, di = u.shape
    ds = state["a"].shape[0]
    dr = proj.shape[1] - 2 * ds
    start, end = _bounds(state, rows)
    live = state["slots"] >= 0
    slot = state["slots"].long().clamp(min=0)
    old = h0[slot]
    if state["fresh"] is not None:
        old = old * (state["fresh"] == 0)[:, None, None]
    pre = proj[:, :dr] @ state["dt_w"] + state["dt_b"]
    step = torch.clamp(pre, min=0) + torch.log1p(torch.exp(-pre.abs()))
    b, c = proj[:, dr:dr + ds], proj[:, dr + ds:]
    # h_t = decay_t h_(t-1) + add_t: the sequences' first rows take their state in and pass no decay on, then
    # doubled prefixes: after the pass of distance k every row holds the sum over its last 2 k rows
    decay = torch.exp(step[:, None, :] * state["a"])
    add = (step * u)[:, None, :] * b[:, :, None]
    some = end > start
    first = start[some]
    add[first] += decay[first] * old[some]
    decay[first] = 0
    longest = int((end - start).max())
    k = 1
    while k < longest:
        more = decay[k:] * add[:-k]
        decay[k:] = decay[k:] * decay[:-k]
        add[k:] += more
        k *= 2
    y = state["d"] * u + (add * c[:, :, None]).sum(1)
    y = y * (z / (1 + torch.exp(-z)))
    seq = torch.searchsorted(end, torch.arange(rows, device="cuda"), right=True)
    out.copy_(torch.where(live[seq][:, None], y, out.float()).to(out.dtype))
    new = old.clone()
    new[some] = add[end[some] - 1]
    h0[slot[live]] = new[live]
    return {"y": out, "state": h0}


def _w4(state):
    case = state["case"]
    q = _unpack(state["packed"], case["k"]).float() - 8
    scale = state["scales"].float().repeat_interleave(case["group"], 1)[:, :case["k"]]
    return (state["x"].float() @ (q * scale).t()).to(state["x"].dtype)


def _norm(state):
    case = state["case"]
    x, r = state["x"].float(), state["residual"]
    if state["post"] is not None:
        x = x * torch.rsqrt(x.square().mean(1, keepdim=True) + 1e-5) * state["post"]
    if state["gate"] is not None:
        x = x * state["gate"].float()
    new = r.float() + 0.5 * x
    r.copy_(new.to(r.dtype))
    y = new * torch.rsqrt(new.square().mean(1, keepdim=True) + 1e-5) * state["weight"]
    return {"out": y.to(DTYPES[case["dtype"]]), "residual": r}


def run(state):
    op = state["case"]["op"]
    if own:
        from flowedge_b200 import ops

        if op == "conv":
            u = ops.conv(state["x"], state["w"], state["b"], window=state["window"], offsets=state["offsets"],
                         slots=state["slots"], fresh=state["fresh"], out=state["out"])
            return {"u": u, "window": state["window"]}
        if op == "scan":
            y = ops.scan(state["u"], state["proj"], state["a"], state["d"], state["dt_w"], state["dt_b"],
                         z=state["z"], state=state["state"], offsets=state["offsets"], slots=state["slots"],
                         fresh=state["fresh"], out=state["out"])
            return {"y": y, "state": state["state"]}
        if op == "w4":
            return ops.w4_matvec(state["x"], state["packed"], state["scales"], group=state["case"]["group"])
        y = ops.residual_norm(state["x"], state["residual"], state["weight"], post_weight=state["post"],
                              gate=state["gate"], scale=0.5)
        return {"out": y, "residual": state["residual"]}
    if op == "conv":
        return _conv(state)
    if op == "scan":
        return _scan(state)
    return _w4(state) if op == "w4" else _norm(state)


def work(case):
    e = SIZES[case["dtype"]]
    if case["op"] in ("conv", "scan"):
        live = case["seqs"] - case.get("pad", 0)
        rows = live if case["form"] == "tokens" else case["rows"]
        reads = 0 if case.get("fresh") else 1
        di = case["di"]
        if case["op"] == "conv":
            dc = case["dc"]
            return {"bytes": 2 * rows * di * e + (1 + reads) * live * di * dc * 4 + di * (dc + 1) * 4,
                    "flops": rows * di * (2 * dc + 4)}
        ds, dr = case["ds"], case["dr"]
        return {"bytes": rows * (3 * di + dr + 2 * ds) * e + (1 + reads) * live * di * ds * 4 + di * (dr + ds + 2) * 4,
                "flops": rows * di * (2 * dr + 7 * ds + 12)}
    if case["op"] == "w4":
        m, k, rows = case["m"], case["k"], case["rows"]
        return {"bytes": m * ((k + 1) // 2) + 2 * m * ((k + case["group"] - 1) // case["group"]) + rows * (k + m) * e,
                "flops": 2 * rows * m * k}
    rows, dim = case["rows"], case["dim"]
    gate = {"none": 0, "rows": rows, "one": 1}[case["gate"]]
    return {"bytes": 2 * rows * dim * (e + SIZES[case["rdtype"]]) + gate * dim * e + dim * 4 * (1 + case["post"]),
            "flops": rows * dim * (6 + 4 * case["post"])}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("conv", "scan"):
        return _exact_sequences(case, s)
    x = s["x"].double()
    if case["op"] == "w4":
        k, group = case["k"], case["group"]
        word = s["packed"].view(torch.int32).long()  # eight elements to a word
        m = word.shape[0]
        w = torch.zeros(m, word.shape[1] * 8, dtype=torch.float64, device="cuda")
        for i, place in enumerate(NIBBLE):
            w[:, place::8] = ((word >> (4 * i)) & 15).double() - 8.0
        for j in range(s["scales"].shape[1]):
            w[:, j * group:(j + 1) * group] *= s["scales"][:, j:j + 1].double()
        return torch.einsum("rk,mk->rm", x, w[:, :k])
    r = s["residual"].double()
    if s["post"] is not None:
        x = s["post"].double() * x / torch.sqrt((x * x).sum(1, keepdim=True) / case["dim"] + 1e-5)
    if s["gate"] is not None:
        x = s["gate"].double() * x
    r = r + x * 0.5
    return {"out": s["weight"].double() * r / torch.sqrt((r * r).sum(1, keepdim=True) / case["dim"] + 1e-5),
            "residual": r}


def _exact_sequences(case, s):
    """All sequences side by side, one position after the other."""
    n = case["seqs"]
    if s["offsets"] is None:
        begin, length = list(range(n)), [1] * n
    else:
        o = s["offsets"].tolist()
        begin, length = o[:-1], [q - p for p, q in zip(o[:-1], o[1:])]
    slots = s["slots"].tolist()
    # longest first, so that at each position the sequences still running are the first ones
    order = sorted((i for i in range(n) if slots[i] >= 0), key=lambda i: -length[i])
    lens = [length[i] for i in order]
    base = torch.tensor([begin[i] for i in order], device="cuda")
    pool = torch.tensor([slots[i] for i in order], device="cuda")
    longest = max(lens, default=0)
    running = [0] * (longest + 1)
    for v in lens:
        running[v] += 1
    for t in range(longest - 1, -1, -1):
        running[t] += running[t + 1]  # sequences of at least t rows
    out = s["out"].double()
    held = (s["window"] if case["op"] == "conv" else s["state"]).double()
    now = held[pool]
    if s["fresh"] is not None:
        now = torch.zeros_like(now)
    if case["op"] == "conv":
        w, b, x = s["w"].double(), s["b"].double(), s["x"].double()
        for t in range(longest):
            k = running[t + 1]
            at = base[:k] + t
            now[:k] = torch.cat([now[:k, :, 1:], x[at][:, :, None]], 2)
            v = b + torch.einsum("sck,ck->sc", now[:k], w)
            out[at] = v * torch.sigmoid(v)
        held[pool] = now
        return {"u": out, "window": held}
    ds, dr = case["ds"], case["dr"]
    a, d, dt_w, dt_b = (s[name].double() for name in ("a", "d", "dt_w", "dt_b"))
    for t in range(longest):
        k = running[t + 1]
        at = base[:k] + t
        p, u, z = s["proj"][at].double(), s["u"][at].double(), s["z"][at].double()
        step = torch.logaddexp(torch.einsum("sr,rc->sc", p[:, :dr], dt_w) + dt_b, torch.zeros((), device="cuda", dtype=torch.float64))
        now[:k] = torch.exp(torch.einsum("sc,nc->snc", step, a)) * now[:k] + torch.einsum("sc,sn->snc", step * u, p[:, dr:dr + ds])
        y = d * u + torch.einsum("snc,sn->sc", now[:k], p[:, dr + ds:])
        out[at] = y * z * torch.sigmoid(z)
    held[pool] = now
    return {"y": out, "state": held}
