"""Weights at the end of fp16's range in an engine with 4-bit projections."""

import numpy as np
import pytest

from flowedge_b200 import Engine
from flowedge_b200 import checkpoint as ck

pytestmark = pytest.mark.gpu

SPEC = ck.MambaSpec(vocab=17, d_model=64, n_layers=1, d_inner=64, d_state=4, d_conv=4, dt_rank=4)


@pytest.mark.parametrize("precision,largest,loads", [("fp32", 65504.0, False), ("fp32", 60000.0, True), ("bf16", 65280.0, True)])
def test_values_that_fp16_does_not_hold_are_refused(tmp_path, precision, largest, loads):
    """65504 / 7 rounds up to 9360 in fp16, and 7 times that is 65520, which fp16 rounds to infinity."""
    tensors = ck.mamba_tensors(SPEC, seed=1)
    tensors["backbone.layers.0.mixer.out_proj.weight"][3, 5] = largest
    path = tmp_path / "m.safetensors"
    ck.write_checkpoint(path, tensors)
    if loads:
        e = Engine(path, threads=0, device=0, precision=precision, weights4_group=32)
        assert np.isfinite(e.run(np.arange(140, dtype=np.int32) % 17)).all()
        e.close()
    else:
        with pytest.raises(RuntimeError, match="rounded to 4 bits"):
            Engine(path, threads=0, device=0, precision=precision, weights4_group=32)
