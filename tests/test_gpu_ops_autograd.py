"""The operators of flowedge_b200.ops beside autograd: they have no gradients and say so."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from flowedge_b200 import ops

pytestmark = pytest.mark.gpu


def _calls():
    """(call over a dict of tensors, its tensors) of every operator."""
    g = torch.Generator().manual_seed(1)

    def r(*shape):
        return torch.randn(*shape, generator=g).cuda()

    yield (lambda t: ops.conv(t["x"], t["weight"], t["bias"], window=t["window"], out=t["out"]),
           {"x": r(6, 32), "weight": r(32, 4), "bias": r(32), "window": r(6, 32, 4), "out": r(6, 32)})
    yield (lambda t: ops.scan(t["u"], t["proj"], t["a"], t["d"], t["dt_w"], t["dt_b"], z=t["z"], state=t["state"], out=t["out"]),
           {"u": r(6, 32), "proj": r(6, 24), "a": -r(8, 32).abs(), "d": r(32), "dt_w": r(8, 32), "dt_b": r(32), "z": r(6, 32),
            "state": r(6, 8, 32), "out": r(6, 32)})
    yield (lambda t: ops.residual_norm(t["x"], t["residual"], t["weight"], post_weight=t["post"], gate=t["gate"], out=t["out"]),
           {"x": r(6, 64), "residual": r(6, 64), "weight": r(64), "post": r(64), "gate": r(6, 64), "out": r(6, 64)})
    packed, _ = ops.w4_quantize(r(50, 96))
    yield (lambda t: ops.w4_matvec(t["x"], packed, t["scales"], out=t["out"]),
           {"x": r(6, 96), "scales": r(50, 2).half(), "out": r(6, 50)})
    yield lambda t: ops.w4_dequantize(packed, t["scales"], 96), {"scales": r(50, 2).half()}
    yield lambda t: ops.w4_quantize(t["weight"]), {"weight": r(50, 96)}


def test_a_forward_mode_tangent_is_refused():
    for call, tensors in _calls():
        for name in tensors:
            with fwad.dual_level():
                call(tensors)  # plain tensors inside a level
                dual = fwad.make_dual(tensors[name].clone(), torch.ones_like(tensors[name]))
                with pytest.raises(ops.FlowEdgeError, match="tangent"):
                    call(tensors | {name: dual})
            call(tensors)


CHANGED = [("window", "out"), ("state", "out"), ("residual", "out"), ("out",), (), ()]


def test_tensors_changed_in_place_show_it():
    for (call, tensors), changed in zip(_calls(), CHANGED):
        before = {name: t._version for name, t in tensors.items()}
        call(tensors)
        assert {name for name, t in tensors.items() if t._version != before[name]} == set(changed)
        with torch.inference_mode():  # tensors made here have no counter
            call({name: t.clone() if i % 2 else t for i, (name, t) in enumerate(tensors.items())})


def test_a_saved_tensor_that_was_changed_is_found_out():
    call, tensors = next(c for c in _calls() if "residual" in c[1])
    scale = torch.ones(6, 64, device="cuda", requires_grad=True)
    product = scale * tensors["residual"]  # saves the residual
    call(tensors)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()
