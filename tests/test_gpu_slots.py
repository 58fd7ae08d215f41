"""The slot-state convolution and selective scan (flowedge_b200.ops) against their definitions in 64 bits."""

import pytest
import torch

import ops_reference as ref
from flowedge_b200 import ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _offsets(lengths):
    return torch.tensor([0] + lengths, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()


def _wide(rows, width, dtype, g, extra):
    """A matrix whose rows are `width + extra` apart, starting at an odd column."""
    return torch.randn(rows, width + extra, generator=g).to(dtype).cuda()[:, extra // 2:extra // 2 + width]


def _conv_case(seed, rows, di, dc, dtype, n_seq, pool, extra=0):
    g = torch.Generator().manual_seed(seed)
    x = _wide(rows, di, dtype, g, extra)
    w = ((torch.rand(di, dc, generator=g) - 0.5) * 2 * dc ** -0.5).cuda()
    b = torch.randn(di, generator=g).cuda()
    window = torch.randn(pool, di, dc, generator=g).cuda()
    slots = torch.randperm(pool, generator=g)[:n_seq].to(torch.int32).cuda()
    return x, w, b, window, slots


def _scan_case(seed, rows, di, ds, dr, dtype, n_seq, pool, extra=0):
    g = torch.Generator().manual_seed(seed)
    case = {"u": _wide(rows, di, dtype, g, extra), "proj": _wide(rows, dr + 2 * ds, dtype, g, extra),
            "a": -(torch.rand(ds, di, generator=g) * ds + 0.5).cuda(), "d": torch.randn(di, generator=g).cuda(),
            "dt_w": (torch.randn(dr, di, generator=g) * 0.5 * dr ** -0.5).cuda(),
            "dt_b": (torch.rand(di, generator=g) * 4 - 5).cuda(), "z": _wide(rows, di, dtype, g, extra),
            "state": torch.randn(pool, ds, di, generator=g).cuda()}
    return case, torch.randperm(pool, generator=g)[:n_seq].to(torch.int32).cuda()


def _close(got, want, bound, what):
    off = (got.double().cpu() - want).abs() - bound
    assert torch.isfinite(got).all(), what
    assert (off <= 0).all(), f"{what}: {off.max().item():.3g} over its bound"


def _run_conv(x, w, b, window, slots, offsets, fresh, out):
    want, wwin, bound = ref.conv(x, w, b, window, offsets, slots, fresh, out)
    got = ops.conv(x, w, b, window=window, offsets=offsets, slots=slots, fresh=fresh, out=out)
    assert got is out
    _close(got, want, bound, "u")
    if window is not None:
        assert torch.equal(window.double().cpu(), wwin)  # inputs as they are: nothing is rounded


def _run_scan(case, slots, offsets, fresh, out):
    rounds = 64 + max(b - a for a, b in ref.spans(out.shape[0], offsets)) // 8 if out.shape[0] else 64
    y, pool, bound, pool_bound = ref.scan(*(case[k] for k in ("u", "proj", "a", "d", "dt_w", "dt_b", "z", "state")),
                                          offsets, slots, fresh, out, rounds)
    got = ops.scan(case["u"], case["proj"], case["a"], case["d"], case["dt_w"], case["dt_b"], z=case["z"],
                   state=case["state"], offsets=offsets, slots=slots, fresh=fresh, out=out)
    _close(got, y, bound, "y")
    if case["state"] is not None:
        _close(case["state"], pool, pool_bound, "state")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,di,dc,extra", [(1, 64, 4, 0), (5, 1, 1, 3), (7, 129, 2, 5), (40, 300, 4, 4), (3, 31, 8, 1),
                                              (2, 260, 5, 0)])
def test_conv_tokens(dtype, rows, di, dc, extra):
    x, w, b, window, slots = _conv_case(rows + di, rows, di, dc, dtype, rows, rows + 3, extra)
    out = torch.full((rows, di), 7.0, dtype=dtype, device="cuda")
    if rows > 2:
        slots[1] = -1  # a padded row
    _run_conv(x, w, b, window, slots, None, None, out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,di,dc,extra", [([1], 64, 4, 0), ([0, 3, 0, 1, 70, 2, 33, 0], 136, 4, 8),
                                                 ([5, 64, 32, 31, 1], 33, 3, 3), ([2, 9, 100], 257, 8, 2),
                                                 ([200], 128, 1, 0), ([4, 3, 2, 1], 20, 7, 0)])
@pytest.mark.parametrize("fresh", [None, "some"])
def test_conv_prompts(dtype, lengths, di, dc, extra, fresh):
    n, rows = len(lengths), sum(lengths)
    x, w, b, window, slots = _conv_case(rows + di, rows + 4, di, dc, dtype, n, n + 2, extra)
    flags = None
    if fresh:
        flags = (torch.arange(n) % 2 == 0).to(torch.uint8).cuda()
        for s in range(0, n, 2):
            window[int(slots[s])] = float("nan")  # a fresh start reads nothing of its slot
    if n > 3:
        slots[2] = -1
        if fresh:
            window[torch.isnan(window)] = 0.5
    out = torch.full((rows + 4, di), 7.0, dtype=dtype, device="cuda")  # four rows behind the last sequence
    _run_conv(x, w, b, window, slots, _offsets(lengths), flags, out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,di,ds,dr,extra", [(1, 64, 16, 8, 0), (6, 1, 1, 1, 3), (9, 200, 4, 5, 1), (33, 129, 16, 32, 2),
                                                 (3, 40, 32, 64, 0), (70, 1200, 12, 17, 0), (5, 100, 20, 130, 4),
                                                 (19, 4099, 16, 300, 0), (300, 300, 8, 512, 0), (2, 30, 9, 512, 0)])
def test_scan_tokens(dtype, rows, di, ds, dr, extra):
    case, slots = _scan_case(rows + di, rows, di, ds, dr, dtype, rows, rows + 3, extra)
    if rows > 2:
        slots[1] = -1
    fresh = (torch.arange(rows) % 3 == 2).cuda()
    _run_scan(case, slots, None, fresh, torch.full((rows, di), 7.0, dtype=dtype, device="cuda"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,di,ds,dr,extra", [([1], 64, 16, 8, 0), ([0, 3, 0, 1, 70, 2, 33, 0], 136, 16, 32, 2),
                                                    ([15, 16, 17, 1, 32], 129, 8, 4, 1), ([130], 40, 32, 9, 0),
                                                    ([300, 7], 70, 5, 3, 5), ([9, 40], 24, 16, 130, 0),
                                                    ([50, 1, 20], 66, 17, 300, 1), ([700], 2050, 16, 7, 0)])
def test_scan_prompts(dtype, lengths, di, ds, dr, extra):
    n, rows = len(lengths), sum(lengths)
    case, slots = _scan_case(rows + di, rows + 4, di, ds, dr, dtype, n, n + 2, extra)
    fresh = (torch.arange(n) % 2 == 1).to(torch.uint8).cuda()
    if n > 3:
        slots[2] = -1
    for s in range(1, n, 2):
        if n <= 3:
            case["state"][int(slots[s])] = float("nan")
    _run_scan(case, slots, _offsets(lengths), fresh, torch.full((rows + 4, di), 7.0, dtype=dtype, device="cuda"))


@pytest.mark.parametrize("lengths", [[3, 50, 0, 20], None])
def test_without_states_or_gate(lengths):
    rows = sum(lengths) if lengths else 6
    offsets = _offsets(lengths) if lengths else None
    x, w, b, _, _ = _conv_case(1, rows, 70, 4, torch.float32, 1, 1)
    _run_conv(x, w, b, None, None, offsets, None, torch.zeros(rows, 70, device="cuda"))
    case, _ = _scan_case(2, rows, 70, 16, 8, torch.float32, 1, 1)
    case["state"] = case["z"] = None
    _run_scan(case, None, offsets, None, torch.zeros(rows, 70, device="cuda"))


def test_prompt_in_pieces_and_tokens_equals_one_prompt():
    """conv -> projection -> scan over a prompt, then token by token, against one longer prompt."""
    g = torch.Generator().manual_seed(5)
    di, ds, dr, total, cut = 96, 16, 8, 90, 61
    x = torch.randn(2 * total, 2 * di, generator=g).cuda()
    wx = (torch.randn(di, dr + 2 * ds, generator=g) * di ** -0.5).cuda()
    w, b = torch.randn(di, 4, generator=g).cuda() * 0.5, torch.randn(di, generator=g).cuda()
    case, _ = _scan_case(3, 1, di, ds, dr, torch.float32, 1, 4)
    weights = [case[k] for k in ("a", "d", "dt_w", "dt_b")]

    def mixer(rows, window, state, **kw):
        u = ops.conv(rows[:, :di], w, b, window=window, **kw)
        return ops.scan(u, u @ wx, *weights, z=rows[:, di:], state=state, **kw)

    pools = [(torch.zeros(4, di, 4, device="cuda"), torch.zeros(4, ds, di, device="cuda")) for _ in range(2)]
    slots = torch.tensor([3, 1], dtype=torch.int32, device="cuda")
    whole = mixer(x, *pools[0], offsets=_offsets([total, total]), slots=slots).view(2, total, di)
    seqs = x.view(2, total, 2 * di)
    parts = [mixer(seqs[:, :cut].reshape(-1, 2 * di), *pools[1], offsets=_offsets([cut, cut]), slots=slots,
                   fresh=torch.ones(2, dtype=torch.bool, device="cuda")).view(2, cut, di)]
    for t in range(cut, total):
        parts.append(mixer(seqs[:, t].contiguous(), *pools[1], slots=slots).view(2, 1, di))
    torch.testing.assert_close(torch.cat(parts, 1), whole, rtol=1e-4, atol=1e-4)
    for p, q in zip(*pools):
        torch.testing.assert_close(p, q, rtol=1e-4, atol=1e-4)


def test_faulty_sequences_are_skipped_and_reported():
    x, w, b, window, _ = _conv_case(1, 12, 32, 4, torch.float32, 1, 4)
    case, _ = _scan_case(2, 12, 32, 16, 8, torch.float32, 1, 4)
    weights = [case[k] for k in ("a", "d", "dt_w", "dt_b")]
    for offsets, slots, bits in [([0, 5, 3, 12], [0, 1, 2], ops.BAD_OFFSETS), ([0, 4, 8, 13], [0, 1, 2], ops.BAD_OFFSETS),
                                 ([-1, 4, 8, 12], [0, 1, 2], ops.BAD_OFFSETS), ([0, 4, 8, 12], [0, 4, 2], ops.BAD_SLOT),
                                 ([0, 4, 8, 12], [2, 1, 2], ops.DUPLICATE_SLOT),
                                 (None, [0, 1, 2, 3, 1, -1, -1, 9, -1, -1, -1, -1], ops.DUPLICATE_SLOT | ops.BAD_SLOT)]:
        o = None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device="cuda")
        s = torch.tensor(slots, dtype=torch.int32, device="cuda")
        first = 2 if offsets is None else None
        for call in ("conv", "scan"):
            status = torch.zeros(1, dtype=torch.int32, device="cuda")
            out = torch.full((12, 32), 7.0, device="cuda")
            if call == "conv":
                ops.conv(x, w, b, window=window.clone(), offsets=o, slots=s, status=status, out=out)
            else:
                ops.scan(case["u"], case["proj"], *weights, state=case["state"].clone(), offsets=o, slots=s,
                         status=status, out=out)
            assert int(status) == bits
            if first is not None:  # the first sequence of a slot ran, the later one did not
                assert (out[1] != 7).any() and (out[4] == 7).all() and (out[7] == 7).all()
            elif bits == ops.DUPLICATE_SLOT:
                assert (out[0] != 7).any() and (out[8:] == 7).all()


def test_slots_far_apart():
    """Slots whose distance passes 2^31 elements."""
    di, ds = 64, 16
    far = 2 ** 31 + 64
    try:
        big = torch.zeros(far + di * ds, device="cuda")
    except torch.cuda.OutOfMemoryError:
        pytest.skip("not enough memory")
    state = big.as_strided((2, ds, di), (far, di, 1))
    window = big.as_strided((2, di, 4), (far, 4, 1))
    case, _ = _scan_case(4, 2, di, ds, 8, torch.float32, 1, 1)
    case["state"] = torch.zeros(2, ds, di, device="cuda")
    want = ops.scan(case["u"], case["proj"], case["a"], case["d"], case["dt_w"], case["dt_b"], state=case["state"])
    got = ops.scan(case["u"], case["proj"], case["a"], case["d"], case["dt_w"], case["dt_b"], state=state)
    assert torch.equal(got, want) and torch.equal(state, case["state"])
    big.zero_()
    small = torch.zeros(2, di, 4, device="cuda")
    x, w, b, _, _ = _conv_case(5, 2, di, 4, torch.float32, 1, 1)
    assert torch.equal(ops.conv(x, w, b, window=window), ops.conv(x, w, b, window=small))
    assert torch.equal(window, small)


def test_streams_and_graphs():
    """A captured step replays over new inputs; calls on two streams do not disturb one another."""
    case, slots = _scan_case(6, 40, 128, 16, 8, torch.float32, 2, 2)
    weights = [case[k] for k in ("a", "d", "dt_w", "dt_b")]
    offsets = _offsets([25, 15])
    first = case["state"].clone()

    def call(state, out):
        return ops.scan(case["u"], case["proj"], *weights, z=case["z"], state=state, offsets=offsets, slots=slots, out=out)

    want_state = first.clone()
    want = [call(want_state, torch.empty(40, 128, device="cuda")) for _ in range(3)]
    out, state = torch.empty(40, 128, device="cuda"), first.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call(first.clone(), out)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(state, out)
    for w in want:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)
    assert torch.equal(state, want_state)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for s in streams:
        with torch.cuda.stream(s):
            st = first.clone()
            results.append([call(st, torch.empty(40, 128, device="cuda")) for _ in range(3)])
    torch.cuda.synchronize()
    for r in results:
        for got, w in zip(r, want):
            assert torch.equal(got, w)


def test_refusals():
    x, w, b, window, slots = _conv_case(1, 6, 32, 4, torch.float32, 6, 8)
    case, _ = _scan_case(2, 6, 32, 16, 8, torch.float32, 6, 8)
    weights = [case[k] for k in ("a", "d", "dt_w", "dt_b")]
    bad = [lambda: ops.conv(x.cpu(), w, b), lambda: ops.conv(x.double(), w, b), lambda: ops.conv(x, w.half(), b),
           lambda: ops.conv(x, torch.zeros(32, 9, device="cuda"), b), lambda: ops.conv(x, w, b[:31]),
           lambda: ops.conv(x, w, b, out=x), lambda: ops.conv(x, w, b, window=window[:4]),
           lambda: ops.conv(x, w, b, window=window, slots=slots.long()), lambda: ops.conv(x, w, b, slots=slots[:5]),
           lambda: ops.conv(x, w, b, window=window.transpose(1, 2)), lambda: ops.conv(x.requires_grad_(), w, b),
           lambda: ops.conv(x.detach()[:, ::2], w[::2].contiguous(), b[::2].contiguous()),
           lambda: ops.conv(x.detach()[:1].expand(6, 32), w, b),
           lambda: ops.scan(case["u"], case["proj"][:, 1:], *weights), lambda: ops.scan(case["u"], case["proj"].half(), *weights),
           lambda: ops.scan(case["u"], case["proj"], *weights, out=case["u"]),
           lambda: ops.scan(case["u"], case["proj"], *weights, z=case["z"], out=case["z"]),
           lambda: ops.scan(case["u"], case["proj"], *weights, offsets=torch.zeros(3, device="cuda")),
           lambda: ops.scan(case["u"], torch.zeros(6, 8 + 66, device="cuda"), torch.zeros(33, 32, device="cuda"),
                            *weights[1:])]
    for call in bad:
        with pytest.raises(ops.FlowEdgeError, match="status 1"):
            call()
    # columns beside one another of the same rows are no overlap
    xz = torch.randn(6, 64, device="cuda")
    out = ops.conv(xz[:, :32], w, b, out=xz[:, 32:])
    assert out.data_ptr() == xz[:, 32:].data_ptr()


def test_nothing_to_do():
    w, b = torch.ones(8, 4, device="cuda"), torch.zeros(8, device="cuda")
    assert ops.conv(torch.empty(0, 8, device="cuda"), w, b).shape == (0, 8)
    window = torch.ones(2, 8, 4, device="cuda")
    empty = _offsets([0, 0])
    ops.conv(torch.empty(0, 8, device="cuda"), w, b, window=window, offsets=empty,
             fresh=torch.tensor([0, 1], dtype=torch.uint8, device="cuda"))
    assert (window[0] == 1).all() and (window[1] == 0).all()
