"""The number of sequences that a call with states in slots takes (refused at the C entries; nothing is launched)."""

import pytest

from flowedge_b200 import build, ops
from flowedge_b200 import engine as fe

BIG = 1 << 40  # addresses that nothing reads


@pytest.fixture(scope="module")
def lib():
    build.build()
    return fe.load_library()


@pytest.mark.parametrize("call", ["conv", "scan"])
@pytest.mark.parametrize("offsets", [0, 64])
def test_too_many_sequences_with_slots_are_refused(lib, call, offsets):
    n = 2 ** 16 + 1
    rows = n if not offsets else 7
    if call == "conv":
        args = ops._CONV.pack(ops._CONV.size, -1, 0, 4, rows, 32, n, n, 32, 32, 128, BIG, 64, 64, 2 * BIG, 64, offsets, 64, 0, 0)
        rc = lib.fe_causal_conv_device(args, None)
    else:
        args = ops._SCAN.pack(ops._SCAN.size, -1, 0, 16, rows, 32, 8, n, n, 32, 40, 32, 32, 512, BIG, 2 * BIG, 3 * BIG, 64, 64,
                              64, 64, 4 * BIG, 64, offsets, 64, 0, 0, 0, 0)
        rc = lib.fe_selective_scan_device(args, None)
    assert rc == 1 and "2^16 sequences" in lib.fe_engine_last_error().decode()
