"""Sizes of appended structures as the public header states them, and the reserved field of the engine's options."""

import ctypes as C
import re
from pathlib import Path

import pytest

from flowedge_b200 import build, ops
from flowedge_b200 import engine as fe

REPO = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def lib():
    build.build()
    return fe.load_library()


def test_the_header_names_the_sizes_of_the_earlier_structures():
    text = re.sub(r"\s*\n\s*\*\s*", " ", (REPO / "include" / "flowedge_b200.h").read_text())
    options = re.search(r"ends before this field \(struct_size (\d+)\)", text)
    w4 = re.search(r"ends before `layout` \(struct_size (\d+)\)", text)
    assert int(options.group(1)) == fe.EngineOptions.weights4_group.offset
    assert int(w4.group(1)) == ops._W4.size
    assert f"struct_size {C.sizeof(fe.EngineOptions)})" in text


@pytest.mark.parametrize("size,group,reserved,said", [(40, 0, 1, "reserved"), (40, 64, 7, "reserved"), (40, 16, 0, "weights4_group"),
                                                      (24, 0, 0, "Invalid engine options")])
def test_options_that_are_refused(lib, size, group, reserved, said):
    path = str(REPO / "tests" / "golden" / "mamba_flow_tiny.safetensors").encode()
    opts = fe.EngineOptions(size, 0, 0, 1, 1, 16, group, reserved)
    assert not lib.fe_engine_load_with_options(path, C.byref(opts))
    assert said in lib.fe_engine_last_error().decode()
