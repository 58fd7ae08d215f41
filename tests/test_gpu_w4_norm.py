"""Products with 4-bit weights and the residual norm (flowedge_b200.ops) against their definitions in 64 bits."""

import pytest
import torch

from flowedge_b200 import ops
from ops_reference import U, out_step

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _close(got, want, bound, what):
    off = (got.double() - want).abs() - bound
    assert torch.isfinite(got).all(), what
    assert (off <= 0).all(), f"{what}: {off.max().item():.3g} over its bound"


def _sub(dtype):
    return 6e-8 if dtype == torch.float16 else 1e-37  # half's subnormal step


def _rule(weight, group):
    """(q - 8, scale) by the documented rule, [m][k] each, in 64 bits where nothing is rounded to 16."""
    m, k = weight.shape
    w = torch.zeros(m, (k + group - 1) // group * group, dtype=torch.float32, device=weight.device)
    w[:, :k] = weight.float()
    w = w.view(m, -1, group)
    scale = (w.abs().amax(2) / 7).clamp(max=65504).half().float()
    q = torch.where(scale[:, :, None] > 0, torch.round(w / scale[:, :, None]).clamp(-8, 7), torch.zeros_like(w))
    return q.view(m, -1)[:, :k].double(), scale.repeat_interleave(group, 1)[:, :k].double()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,group", [(1, 1, 32), (3, 31, 64), (17, 128, 128), (40, 200, 64), (130, 1000, 32), (5, 385, 128)])
def test_quantize_and_dequantize(dtype, m, k, group):
    g = torch.Generator().manual_seed(m + k)
    wide = torch.randn(m, k + 3, generator=g).to(dtype).cuda()
    weight = wide[:, 1:k + 1]
    if m > 2:
        weight[1] = 0  # a group of zeros has scale zero
    packed, scales = ops.w4_quantize(weight, group)
    assert packed.shape == (m, (k + 127) // 128 * 64) and scales.shape == (m, (k + group - 1) // group)
    q, s = _rule(weight, group)
    assert torch.equal(ops.w4_dequantize(packed, scales, k, group=group).double(), q * s)
    for t in (torch.bfloat16, torch.float16):
        assert torch.equal(ops.w4_dequantize(packed, scales, k, group=group, dtype=t), (q * s).float().to(t))
    # the layout as it is documented, and elements behind the last are zero
    words = packed.view(torch.int32).cpu().view(m, -1, 4, 4)  # [block][t][j]
    for c in range(words.shape[1] * 128):
        place = (0, 2, 4, 6, 1, 3, 5, 7).index(c % 8)
        got = (words[:, c // 128, c % 32 // 8, c % 128 // 32] >> (4 * place)) & 15
        want = q[:, c].cpu() + 8 if c < k else torch.full((m,), 8.0)
        assert torch.equal(got.double(), want.double())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,m,k,extra", [(1, 64, 128, 0), (1, 1, 1, 1), (2, 33, 40, 3), (8, 100, 513, 1), (9, 300, 1000, 0),
                                            (17, 48, 2048, 2), (32, 129, 300, 0), (33, 20, 700, 5), (70, 65, 129, 0),
                                            (5, 3000, 96, 0)])
def test_matvec(dtype, group, rows, m, k, extra):
    g = torch.Generator().manual_seed(rows + m + k)
    weight = torch.randn(m, k, generator=g).cuda() * k ** -0.5
    packed, scales = ops.w4_quantize(weight, group)
    x = torch.randn(rows, k + extra, generator=g).to(dtype).cuda()[:, extra // 2:extra // 2 + k]
    out = torch.full((rows, m + extra), 7.0, dtype=dtype, device="cuda")
    got = ops.w4_matvec(x, packed, scales, group=group, out=out[:, :m])
    w = ops.w4_dequantize(packed, scales, k, group=group).double()
    want = x.double() @ w.t()
    # products exact, k sums, the groups' scaled sums and the split's joins, each rounded once: (k + 2 k / 32 + 16) U
    size = x.double().abs() @ w.abs().t()
    _close(got, want, (k * 1.07 + 16) * U * size + out_step(dtype) * want.abs() * 1.01 + _sub(dtype), "y")
    assert (out[:, m:] == 7).all()
    assert torch.equal(ops.w4_matvec(x, packed, scales, group=group), got)  # the same every time
    for i in (0, rows - 1):  # a row's result does not depend on the rows beside it beyond the order of its sums
        alone = ops.w4_matvec(x[i:i + 1], packed, scales, group=group)
        _close(alone, want[i:i + 1], ((k * 1.07 + 16) * U * size + out_step(dtype) * want.abs() * 1.01 + _sub(dtype))[i:i + 1], "row")


def test_matvec_extremes():
    """float32 x from its largest to its smallest normal values, an infinity and a NaN."""
    weight = torch.eye(128, device="cuda") * 7
    packed, scales = ops.w4_quantize(weight, 32)
    x = torch.zeros(3, 128, device="cuda")
    x[0, :5] = torch.tensor([3.4e38 / 8, 1.2e-38, -1.0000001, 65536.0, 1e-30])
    x[1, 3], x[2, 4] = float("inf"), float("nan")
    y = ops.w4_matvec(x, packed, scales, group=32)
    want = ops.w4_dequantize(packed, scales, 128, group=32).double()
    _close(y[0], x[0].double() @ want.t(), (x[0].double() @ want.t()).abs() * 2 * U + 1e-37, "y")
    assert y[1, 3] == float("inf") and torch.isnan(y[2, 4])


def test_w4_refusals_and_nothing_to_do():
    x = torch.randn(4, 200, device="cuda")
    packed, scales = ops.w4_quantize(torch.randn(60, 200, device="cuda"), 64)
    bad = [lambda: ops.w4_matvec(x[:, :128], packed, scales), lambda: ops.w4_matvec(x, packed, scales, group=32),
           lambda: ops.w4_matvec(x, packed, scales, group=48), lambda: ops.w4_matvec(x, packed[:, 1:], scales),
           lambda: ops.w4_matvec(x, packed, scales.float()), lambda: ops.w4_matvec(x.cpu(), packed, scales),
           lambda: ops.w4_matvec(x, packed, scales, out=x[:, :60]), lambda: ops.w4_matvec(x.requires_grad_(), packed, scales),
           lambda: ops.w4_dequantize(packed.cpu(), scales.cpu(), 200), lambda: ops.w4_quantize(torch.randn(2, 8))]
    for call in bad:
        with pytest.raises(ops.FlowEdgeError, match="status 1"):
            call()
    assert ops.w4_matvec(x.detach()[:0], packed, scales).shape == (0, 60)


def _norm_reference(x, residual, weight, post, gate, scale, eps):
    x, r = x.double(), residual.double()
    dim = x.shape[1]
    t = x
    if post is not None:
        t = x * post.double() / torch.sqrt(x.square().mean(1, keepdim=True) + eps)
    if gate is not None:
        t = t * gate.double()
    t = scale * t
    new = r + t
    # per row: dim roundings of a sum of squares are half of them in its root, then a few products
    new_err = (dim / 2 + 8) * U * t.abs() + U * new.abs()
    root = torch.sqrt(new.square().mean(1, keepdim=True) + eps)
    out = new * weight.double() / root
    # the mean's error: 2 new new_err, and its own sum's
    root_rel = (new.abs() * new_err).mean(1, keepdim=True) / root.square() + (dim / 2 + 6) * U
    out_err = new_err * weight.double().abs() / root + out.abs() * root_rel
    return new, new_err, out, out_err


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("wide_residual", [True, False])
@pytest.mark.parametrize("rows,dim,extra", [(1, 512, 0), (1, 1, 0), (3, 7, 1), (300, 64, 0), (5, 1000, 0), (700, 129, 2),
                                            (2, 16384, 0), (4, 16383, 0), (2, 16384, 1), (400, 2048, 8), (310, 5000, 0), (300, 9001, 3)])
def test_residual_norm(dtype, wide_residual, rows, dim, extra):
    g = torch.Generator().manual_seed(rows + dim)
    r_dtype = torch.float32 if wide_residual else dtype
    wide = lambda n, t: torch.randn(n, dim + extra, generator=g).to(t).cuda()[:, extra // 2:extra // 2 + dim]  # noqa: E731
    weight, post = 1 + 0.3 * torch.randn(dim, generator=g).cuda(), 1 + 0.3 * torch.randn(dim, generator=g).cuda()
    for use_post, gate_rows, scale in [(False, 0, 1.0), (True, 0, 0.5), (False, 1, -1.5), (True, rows, 0.25)]:
        x, residual = wide(rows, dtype), wide(rows, r_dtype)
        if rows > 2:
            x[1] = 0  # a row without anything to add
            residual[1] = 0  # and one that stays zero: eps alone under the root
        gate = wide(gate_rows, dtype) if gate_rows else None
        if gate is not None and gate_rows != rows:
            gate = gate[:1]
        new, new_err, want, err = _norm_reference(x, residual, weight, post if use_post else None, gate, scale, 1e-5)
        out = torch.full((rows, dim), 7.0, dtype=dtype, device="cuda")
        got = ops.residual_norm(x, residual, weight, post_weight=post if use_post else None, gate=gate, scale=scale, out=out)
        _close(got, want, err + out_step(dtype) * want.abs() * 1.01 + _sub(dtype), "out")
        _close(residual, new, new_err + (out_step(r_dtype) * new.abs() * 1.01 if r_dtype != torch.float32 else 0) + _sub(r_dtype), "residual")


def test_norm_refusals_and_nothing_to_do():
    x, r, w = torch.randn(4, 64, device="cuda"), torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    bad = [lambda: ops.residual_norm(x, r.half(), w), lambda: ops.residual_norm(x, r[:3], w), lambda: ops.residual_norm(x, x, w),
           lambda: ops.residual_norm(x, r, w, out=r), lambda: ops.residual_norm(x, r, w, gate=x[:2]),
           lambda: ops.residual_norm(x, r, w, gate=r), lambda: ops.residual_norm(x, r, w, eps=-1.0),
           lambda: ops.residual_norm(x, r, w, post_weight=w[:63]), lambda: ops.residual_norm(x.cpu(), r, w),
           lambda: ops.residual_norm(x, r.requires_grad_(), w),
           lambda: ops.residual_norm(torch.zeros(1, 16385, device="cuda"), torch.zeros(1, 16385, device="cuda"),
                                     torch.ones(16385, device="cuda"))]
    for call in bad:
        with pytest.raises(ops.FlowEdgeError, match="status 1"):
            call()
    assert ops.residual_norm(x[:0], r.detach()[:0], w).shape == (0, 64)


@pytest.mark.parametrize("scale,eps", [(1e300, 1e-5), (1.0, 1e300), ("1", 1e-5), (1.0, float("nan"))])
def test_norm_refuses_what_is_no_float32(scale, eps):
    x, r, w = torch.randn(4, 64, device="cuda"), torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    before = r.clone()
    with pytest.raises(ops.FlowEdgeError, match="status 1"):
        ops.residual_norm(x, r, w, scale=scale, eps=eps)
    assert torch.equal(r, before)
