"""Growth of the engine's Mamba buffers where an allocation fails (refused on the host): the call reports it, and the
states, the slots and the calls of the size that there was room for stay."""

import ctypes as C

import numpy as np
import pytest

from flowedge_b200 import Engine, FlowEdgeError
from flowedge_b200 import checkpoint as ck
from flowedge_b200 import engine as fe
from oracle import restate

pytestmark = pytest.mark.gpu

SPEC = ck.MambaSpec(vocab=17, d_model=72, n_layers=2, d_inner=120, d_state=8, d_conv=3, dt_rank=4)


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    tensors = ck.mamba_tensors(SPEC, seed=3)
    path = tmp_path_factory.mktemp("growth") / "m.safetensors"
    ck.write_checkpoint(path, tensors)
    return path, restate.MambaModel(tensors)


@pytest.fixture
def refuse():
    """refuse(first, count): those allocations fail; refuse(0, 0): none."""
    hook = fe.load_library().febtest_fail_allocations
    hook.argtypes, hook.restype = [C.c_long, C.c_long], None
    yield hook
    hook(0, 0)


CALLS = {"reserve_batch": lambda e, t: e.reserve_batch(3), "prompt": lambda e, t: e.prompt_batch([t], [0]),
         "reserve_slots": lambda e, t: e.reserve_slots(6)}


@pytest.mark.parametrize("first", range(1, 6))
@pytest.mark.parametrize("count", [1, 2, 3, 4, 30])
@pytest.mark.parametrize("call", ["reserve_batch", "prompt", "reserve_slots"])
def test_a_refused_allocation_loses_nothing(model, refuse, call, first, count):
    path, oracle = model
    e = Engine(path, threads=0, device=0, precision="fp32", max_sequence=16)
    e.reserve_slots(2)
    tokens = np.random.default_rng(6).integers(0, 17, 40).astype(np.int32)
    for t in tokens[:5]:
        e.step(int(t))
    e.prompt_batch([tokens[:8], tokens[:3]], [1, 0])
    refuse(first, count)
    try:
        CALLS[call](e, tokens)
        failed = False
    except FlowEdgeError as error:
        assert "status 2" in str(error)
        failed = True
    refuse(0, 0)
    assert failed or count < 30 or first > 3
    zero = tokens if call == "prompt" and not failed else tokens[:3]  # slot 0's history

    def same(got, history):
        np.testing.assert_allclose(got, oracle.run(history)[-1], atol=1e-3)

    # the slots first: a small call takes what it needs
    same(e.step_batch(tokens[8:9], [1])[0], tokens[:9])
    same(e.step_batch(tokens[8:9], [0])[0], np.append(zero, tokens[8]))
    same(e.step(int(tokens[5])), tokens[:6])
    same(e.prompt_batch([tokens], [0])[0], tokens)  # and growth goes through when there is room again
    same(e.step(int(tokens[6])), tokens[:7])
    same(e.step_batch(tokens[9:10], [1])[0], tokens[:10])
    e.close()


def test_the_decode_state_outlives_a_workspace_that_cannot_be_put_back(model, refuse):
    path, oracle = model
    e = Engine(path, threads=0, device=0, precision="fp32", max_sequence=16)
    tokens = np.random.default_rng(7).integers(0, 17, 12).astype(np.int32)
    for t in tokens[:5]:
        e.step(int(t))
    refuse(2, 30)
    with pytest.raises(FlowEdgeError, match="status 2"):
        e.reserve_batch(3)
    with pytest.raises(FlowEdgeError, match="status 2"):
        e.step(int(tokens[5]))
    snapshot = e.decode_state()
    refuse(0, 0)
    e.reserve_batch(1)
    np.testing.assert_allclose(e.step(int(tokens[5])), oracle.run(tokens[:6])[-1], atol=1e-3)
    e.restore_decode_state(snapshot)
    np.testing.assert_allclose(e.step(int(tokens[5])), oracle.run(tokens[:6])[-1], atol=1e-3)
    e.close()
