"""4-bit weights packed in the order of their elements (uint8), against the layout's and the product's definition."""

import pytest
import torch

from flowedge_b200 import ops
from ops_reference import U, out_step

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NIBBLE = (0, 2, 4, 6, 1, 3, 5, 7)  # the element of a word's eight that its nibble i holds


def _pack(q):
    """Whole numbers 0 .. 15 [m][k], elements of k behind the last 8 -> bytes."""
    m, k = q.shape
    full = torch.full((m, -(-k // 32) * 32), 8, dtype=torch.int64)
    full[:, :k] = q
    word = torch.zeros(m, full.shape[1] // 8, dtype=torch.int64)
    for i, e in enumerate(NIBBLE):
        word |= full[:, e::8] << (4 * i)
    return torch.stack([word >> (8 * b) & 255 for b in range(4)], -1).to(torch.uint8).view(m, -1)


def _bound(x, w, want, k, dtype):
    # as for the other layout: products exact, k sums, the groups' scaled sums and the split's joins, each rounded once
    sub = 6e-8 if dtype == torch.float16 else 1e-37
    return (k * 1.07 + 16) * U * (x.double().abs() @ w.abs().t()) + out_step(dtype) * want.abs() * 1.01 + sub


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,m,k,extra", [(1, 64, 128, 0), (1, 1, 1, 1), (2, 33, 40, 3), (8, 100, 513, 1), (9, 300, 1000, 0),
                                            (17, 48, 2048, 2), (32, 129, 300, 0), (33, 20, 704, 5), (70, 65, 129, 0),
                                            (5, 3000, 96, 0), (1, 17, 4128, 0), (11, 41, 2056, 0)])
def test_matvec(dtype, group, rows, m, k, extra):
    g = torch.Generator().manual_seed(rows + m + k)
    q = torch.randint(0, 16, (m, k), generator=g)
    scales = (torch.rand(m, -(-k // group), generator=g) + 0.5).mul_(0.2 * k ** -0.5).half()
    w = ((q - 8).double() * scales.double().repeat_interleave(group, 1)[:, :k]).cuda()
    packed, scales = _pack(q).cuda(), scales.cuda()
    x = torch.randn(rows, k + extra, generator=g).to(dtype).cuda()[:, extra // 2:extra // 2 + k]
    out = torch.full((rows, m + extra), 7.0, dtype=dtype, device="cuda")
    got = ops.w4_matvec(x, packed, scales, group=group, out=out[:, :m])
    want = x.double() @ w.t()
    off = (got.double() - want).abs() - _bound(x, w, want, k, dtype)
    assert torch.isfinite(got).all() and (off <= 0).all(), f"{off.max().item():.3g} over its bound"
    assert (out[:, m:] == 7).all()
    assert torch.equal(ops.w4_matvec(x, packed, scales, group=group), got)
    assert torch.equal(ops.w4_dequantize(packed, scales, k, group=group).double(), w.float().double())


@pytest.mark.parametrize("m,k,group", [(1, 1, 32), (3, 31, 64), (17, 128, 128), (40, 200, 64), (130, 1000, 32), (5, 385, 128)])
def test_quantize_gives_the_same_weights_in_both_layouts(m, k, group):
    weight = torch.randn(m, k, generator=torch.Generator().manual_seed(m + k)).cuda()
    blocks, scales = ops.w4_quantize(weight, group)
    packed, again = ops.w4_quantize(weight, group, layout="rows")
    assert packed.dtype == torch.uint8 and packed.shape == (m, (k + 31) // 32 * 16)
    assert blocks.dtype == torch.int8 and torch.equal(again, scales)
    values = ops.w4_dequantize(blocks, scales, k, group=group)
    assert torch.equal(ops.w4_dequantize(packed, scales, k, group=group), values)
    step = scales.float().repeat_interleave(group, 1)[:, :k]
    q = torch.where(step > 0, torch.round(values / step), torch.zeros_like(step)).long().cpu() + 8
    assert torch.equal(packed.cpu(), _pack(q))


def test_refusals():
    x, weight = torch.randn(4, 200, device="cuda"), torch.randn(60, 200, device="cuda")
    blocks, scales = ops.w4_quantize(weight, 64)
    packed, _ = ops.w4_quantize(weight, 64, layout="rows")
    bad = [lambda: ops.w4_quantize(weight, 64, layout="columns"), lambda: ops.w4_matvec(x, packed[:, :96], scales),
           lambda: ops.w4_matvec(x, packed.to(torch.int8), scales), lambda: ops.w4_matvec(x, blocks.view(torch.uint8), scales),
           lambda: ops.w4_matvec(x, packed.int(), scales), lambda: ops.w4_dequantize(packed, scales, 300)]
    for call in bad:
        with pytest.raises(ops.FlowEdgeError, match="status 1"):
            call()
