"""Refusals of the operators on device buffers at the C entry points: nothing is launched, so no GPU is needed."""

import pytest
import torch

from flowedge_b200 import build, ops
from flowedge_b200 import engine as fe

BIG = 1 << 40  # addresses that nothing reads


@pytest.fixture(scope="module")
def lib():
    build.build()
    return fe.load_library()


def _conv(lib, **kw):
    v = {"size": ops._CONV.size, "device": -1, "dtype": 0, "dc": 4, "rows": 6, "di": 32, "n_seq": 6, "n_slots": 8,
         "x_ld": 32, "u_ld": 32, "stride": 128, "x": BIG, "w": 64, "b": 64, "u": 2 * BIG, "window": 64, "offsets": 0,
         "slots": 64, "fresh": 0, "status": 0} | kw
    return lib.fe_causal_conv_device(ops._CONV.pack(*v.values()), None)


def _scan(lib, **kw):
    v = {"size": ops._SCAN.size, "device": -1, "dtype": 0, "ds": 16, "rows": 6, "di": 32, "dr": 8, "n_seq": 6,
         "n_slots": 8, "u_ld": 32, "proj_ld": 40, "z_ld": 32, "y_ld": 32, "stride": 512, "u": BIG, "proj": 2 * BIG,
         "z": 3 * BIG, "a": 64, "d": 64, "dt_w": 64, "dt_b": 64, "y": 4 * BIG, "state": 64, "offsets": 0, "slots": 64,
         "fresh": 0, "status": 0, "workspace": 0, "bytes": 0} | kw
    return lib.fe_selective_scan_device(ops._SCAN.pack(*v.values()), None)


@pytest.mark.parametrize("change,said", [
    ({"size": 8}, "size"), ({"dtype": 3}, "dtype"), ({"dc": 0}, "d_conv"), ({"dc": 9}, "d_conv"), ({"di": 0}, "d_inner"),
    ({"n_seq": 5}, "n_seq equals rows"), ({"rows": 2 ** 31, "n_seq": 2 ** 31}, "2^30"), ({"x": 0}, "required"),
    ({"w": 0}, "required"), ({"u": BIG}, "overlaps"), ({"u": BIG + 6 * 128 - 4}, "overlaps"), ({"x_ld": 31}, "x_ld"),
    ({"x": BIG + 2}, "aligned"), ({"stride": 127}, "slot_stride"), ({"n_slots": 0}, "n_slots"),
    ({"slots": 0, "n_slots": 5}, "n_slots"), ({"device": -2}, "device"), ({"slots": 66}, "aligned")])
def test_conv_refusals(lib, change, said):
    assert _conv(lib, **change) == 1
    text = lib.fe_engine_last_error().decode()
    assert text.startswith("fe_causal_conv_device") and said in text


@pytest.mark.parametrize("change,said", [
    ({"size": 8}, "size"), ({"ds": 0}, "d_state"), ({"ds": 33}, "d_state"), ({"dr": 0}, "dt_rank"), ({"dr": 513}, "dt_rank"),
    ({"proj_ld": 39}, "proj_ld"), ({"z_ld": 31}, "z_ld"), ({"y": BIG}, "overlaps u"), ({"y": 3 * BIG}, "overlaps z"),
    ({"y": 2 * BIG}, "overlaps proj"), ({"dt_w": 0}, "required"), ({"state": 66}, "aligned"), ({"stride": 511}, "slot_stride"),
    ({"n_seq": 7}, "n_seq equals rows")])
def test_scan_refusals(lib, change, said):
    assert _scan(lib, **change) == 1
    text = lib.fe_engine_last_error().decode()
    assert text.startswith("fe_selective_scan_device") and said in text


def test_null_arguments(lib):
    assert lib.fe_causal_conv_device(None, None) == 1
    assert lib.fe_selective_scan_device(None, None) == 1
    assert lib.fe_selective_scan_workspace(None) == 0


def test_cpu_tensors_are_refused():
    with pytest.raises(fe.FlowEdgeError, match="not on a GPU"):
        ops.conv(torch.zeros(2, 8), torch.zeros(8, 4), torch.zeros(8))


def _w4(lib, call="fe_w4_matvec_device", **kw):
    v = {"size": ops._W4.size, "device": -1, "dtype": 0, "group": 64, "rows": 4, "m": 100, "k": 200, "x_ld": 200,
         "y_ld": 200, "x": BIG, "packed": 64, "scales": 64, "y": 2 * BIG} | kw
    return getattr(lib, call)(ops._W4.pack(*v.values()), None)


@pytest.mark.parametrize("call", ["fe_w4_matvec_device", "fe_w4_quantize_device", "fe_w4_dequantize_device"])
@pytest.mark.parametrize("change,said", [
    ({"size": 8}, "size"), ({"dtype": 7}, "dtype"), ({"group": 16}, "group"), ({"m": 0}, "m and k"),
    ({"k": 2 ** 21}, "m and k"), ({"m": 2 ** 20, "k": 2 ** 19}, "2^38"), ({"packed": 72}, "packed"), ({"scales": 0}, "scales"), ({"device": -3}, "device")])
def test_w4_refusals(lib, call, change, said):
    assert _w4(lib, call, **change) == 1
    text = lib.fe_engine_last_error().decode()
    assert text.startswith(call) and said in text


def test_w4_matrix_refusals(lib):
    for call, change, said in [("fe_w4_matvec_device", {"x_ld": 199}, "x_ld"), ("fe_w4_matvec_device", {"y_ld": 99}, "y_ld"),
                               ("fe_w4_matvec_device", {"y": BIG}, "overlaps"), ("fe_w4_matvec_device", {"x": 0}, "x is"),
                               ("fe_w4_quantize_device", {"x": BIG + 1}, "x is"), ("fe_w4_dequantize_device", {"y": 0}, "y is"),
                               ("fe_w4_dequantize_device", {"y_ld": 199}, "y_ld")]:
        assert _w4(lib, call, **change) == 1 and said in lib.fe_engine_last_error().decode()
    assert _w4(lib, rows=0, x=0, y=0) == 0  # nothing to do


@pytest.mark.parametrize("change,said", [
    ({"size": 8}, "size"), ({"dtype": 3}, "dtype"), ({"r_dtype": 2}, "residual_dtype"), ({"dim": 0}, "dim"),
    ({"dim": 16385}, "dim"), ({"x": 0}, "required"), ({"x_ld": 63}, "x_ld"), ({"gate_ld": 5}, "gate_ld"),
    ({"out": BIG}, "out overlaps"), ({"residual": BIG}, "residual overlaps"), ({"gate": 4 * BIG}, "out overlaps"),
    ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"), ({"weight": 0}, "weight")])
def test_norm_refusals(lib, change, said):
    v = {"size": ops._NORM.size, "device": -1, "dtype": 0, "r_dtype": 0, "rows": 4, "dim": 64, "x_ld": 64, "r_ld": 64,
         "gate_ld": 64, "out_ld": 64, "x": BIG, "post": 0, "gate": 2 * BIG, "residual": 3 * BIG, "weight": 64,
         "out": 4 * BIG, "scale": 1.0, "eps": 1e-5} | change
    assert lib.fe_residual_norm_device(ops._NORM.pack(*v.values()), None) == 1
    text = lib.fe_engine_last_error().decode()
    assert text.startswith("fe_residual_norm_device") and said in text
