"""The layout field of the 4-bit products' arguments at the C entry points (nothing is launched)."""

import struct

import pytest

from flowedge_b200 import build, ops
from flowedge_b200 import engine as fe


@pytest.fixture(scope="module")
def lib():
    build.build()
    return fe.load_library()


def _args(size, *behind):
    return ops._W4.pack(size, -1, 0, 64, 0, 100, 200, 200, 200, 0, 64, 64, 0) + struct.pack("@II", *behind)


@pytest.mark.parametrize("call", ["fe_w4_matvec_device", "fe_w4_quantize_device", "fe_w4_dequantize_device"])
def test_unknown_layouts_are_refused(lib, call):
    for behind in [(2, 0), (0, 1), (1, 7)]:
        assert getattr(lib, call)(_args(ops._W4.size + 8, *behind), None) == 1
        assert "layout" in lib.fe_engine_last_error().decode()


def test_a_structure_that_ends_before_the_layout_reads_as_blocks(lib):
    # (no rows: nothing to do; what lies behind the structure is not read)
    assert lib.fe_w4_matvec_device(_args(ops._W4.size, 99, 99), None) == 0
    assert lib.fe_w4_matvec_device(_args(ops._W4.size + 4, 99, 99), None) == 0
    assert lib.fe_w4_matvec_device(_args(ops._W4.size + 8, 1, 0), None) == 0
    assert lib.fe_w4_matvec_device(_args(ops._W4.size - 8, 0, 0), None) == 1
