"""Matrices of more than 2^31 elements through the operators of flowedge_b200.ops: their last rows against small calls on
copies of those rows."""

import pytest
import torch

from flowedge_b200 import ops

pytestmark = pytest.mark.gpu

ROWS, DIM = 2 ** 21 + 9, 1024
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def room():
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("not enough memory")
    yield
    torch.cuda.empty_cache()


def _big(rows=ROWS, width=DIM):
    """Random rows at both ends, zeros between (a whole random matrix takes longer than the calls)."""
    x = torch.zeros(rows, width, dtype=BF16, device="cuda")
    x[:512], x[-512:] = torch.randn(512, width, device="cuda"), torch.randn(512, width, device="cuda")
    return x


def _offsets(*o):
    return torch.tensor(o, dtype=torch.int32, device="cuda")


def test_conv():
    torch.manual_seed(1)
    x, w, b = _big(), torch.randn(DIM, 4, device="cuda"), torch.randn(DIM, device="cuda")
    u = ops.conv(x, w, b, offsets=_offsets(0, 300, ROWS - 7, ROWS))
    assert torch.equal(u[:300], ops.conv(x[:300].clone(), w, b, offsets=_offsets(0, 300)))
    tail = ops.conv(x[-200:].clone(), w, b, offsets=_offsets(0, 193, 200))
    assert torch.equal(u[-197:], tail[3:])  # (three rows of a past that the copy does not have)
    tokens = ops.conv(x, w, b, out=u)
    assert torch.equal(tokens[-100:], ops.conv(x[-100:].clone(), w, b))


def test_scan():
    torch.manual_seed(2)
    x, ds, dr = _big(), 4, 4
    proj = _big(width=dr + 2 * ds)
    weights = [-torch.rand(ds, DIM, device="cuda") - 0.5, torch.randn(DIM, device="cuda"), torch.randn(dr, DIM, device="cuda") * 0.3,
               torch.rand(DIM, device="cuda") - 4]
    y = ops.scan(x, proj, *weights, z=x, offsets=_offsets(0, 9, ROWS - 11, ROWS))
    assert torch.equal(y[:9], ops.scan(x[:9].clone(), proj[:9].clone(), *weights, z=x[:9].clone(), offsets=_offsets(0, 9)))
    last = x[-11:].clone()
    want = ops.scan(last, proj[-11:].clone(), *weights, z=last, offsets=_offsets(0, 11))
    assert torch.equal(y[-11:], want)
    tokens = ops.scan(x, proj, *weights, z=x, out=y)
    many = x[-400:].clone()
    assert torch.equal(tokens[-400:], ops.scan(many, proj[-400:].clone(), *weights, z=many))


def test_residual_norm():
    torch.manual_seed(3)
    x, residual, weight = _big(), _big(), torch.randn(DIM, device="cuda")
    small, held = x[-400:].clone(), residual[-400:].clone()
    got = ops.residual_norm(x, residual, weight, post_weight=weight, gate=x)
    assert torch.equal(got[-400:], ops.residual_norm(small, held, weight, post_weight=weight, gate=small))
    assert torch.equal(residual[-400:], held)


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8])
@pytest.mark.parametrize("group", [32, 128])
def test_w4_matvec(dtype, group):
    torch.manual_seed(4)
    m, k = 2 ** 18, 2 ** 15
    packed = torch.zeros(m, k // 2, dtype=torch.uint8, device="cuda")
    packed[-64:] = torch.randint(0, 256, (64, k // 2), dtype=torch.uint8, device="cuda")
    packed = packed.view(dtype)
    scales = torch.rand(m, k // group, device="cuda").half()
    x = torch.randn(3, k, device="cuda")
    got = ops.w4_matvec(x, packed, scales, group=group)
    w = ops.w4_dequantize(packed[-64:].clone(), scales[-64:].clone(), k, group=group).double()
    want = x.double() @ w.t()
    size = x.double().abs() @ w.abs().t()
    assert ((got[:, -64:].double() - want).abs() <= (k * 1.07 + 16) * 2.0 ** -24 * size).all()
