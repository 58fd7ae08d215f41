"""Which rows and which calls a fault of the engine's slot calls is charged to."""

import ctypes as C

import numpy as np
import pytest
import torch

from flowedge_b200 import Engine, FlowEdgeError
from flowedge_b200 import checkpoint as ck
from flowedge_b200 import engine as fe
from oracle import restate

pytestmark = pytest.mark.gpu

SPEC = ck.MambaSpec(vocab=17, d_model=64, n_layers=2, d_inner=128, d_state=8, d_conv=4, dt_rank=4)


@pytest.fixture(scope="module")
def made(tmp_path_factory):
    tensors = ck.mamba_tensors(SPEC, seed=5)
    path = tmp_path_factory.mktemp("faults") / "m.safetensors"
    ck.write_checkpoint(path, tensors)
    e = Engine(path, threads=0, device=0, precision="fp32", max_sequence=64)
    e.reserve_slots(4)
    yield e, restate.MambaModel(tensors)
    e.close()


def _dev(a, dtype=torch.int32):
    return torch.as_tensor(a, dtype=dtype, device="cuda")


def _step(e, tokens, slots):
    t, s, out = _dev(tokens), _dev(slots), torch.full((len(tokens), 64), 7.0, device="cuda")
    torch.cuda.synchronize()
    e.step_device(t.data_ptr(), s.data_ptr(), len(tokens), out.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("pad", [-1, 17, 2 ** 31 - 1])
def test_tokens_of_rows_that_do_not_run_are_no_fault(made, pad):
    e, model = made
    e.prompt_batch([[1, 2, 3], [4]], [0, 2])
    out = _step(e, [5, pad, 6, pad, pad], [0, -1, 2, 9, 0])  # skipped, outside the pool, given twice
    e.synchronize()
    np.testing.assert_allclose(out[0].cpu(), model.run([1, 2, 3, 5])[-1], atol=1e-3)
    np.testing.assert_allclose(out[2].cpu(), model.run([4, 6])[-1], atol=1e-3)
    # a prompt between rows of no sequence, a skipped one and rows behind the last
    t, o, s = _dev([pad, 7, 8, pad, pad, 9, pad, pad]), _dev([1, 3, 5, 6]), _dev([1, -1, 3])
    fresh, last = _dev([1, 1, 1], torch.uint8), torch.full((3, 64), 7.0, device="cuda")
    torch.cuda.synchronize()
    e.prompt_device(t.data_ptr(), 8, o.data_ptr(), s.data_ptr(), 3, last.data_ptr(), fresh.data_ptr(),
                    stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    e.synchronize()
    np.testing.assert_allclose(last[0].cpu(), model.run([7, 8])[-1], atol=1e-3)
    np.testing.assert_allclose(last[2].cpu(), model.run([9])[-1], atol=1e-3)
    np.testing.assert_allclose(e.step_batch([10], [3])[0], model.run([9, 10])[-1], atol=1e-3)


def test_a_token_fault_is_reported_once_and_charged_to_no_later_call(made):
    e, model = made
    e.prompt_batch([[1, 2], [3]], [0, 1])
    _step(e, [17, 4], [0, 1])
    np.testing.assert_allclose(e.step_batch([5], [1])[0], model.run([3, 4, 5])[-1], atol=1e-3)
    np.testing.assert_allclose(e.prompt_batch([[6]], [1], resume=True)[0], model.run([3, 4, 5, 6])[-1], atol=1e-3)
    e.reset()
    np.testing.assert_allclose(e.step(2), model.run([2])[-1], atol=1e-3)
    with pytest.raises(FlowEdgeError, match="Device work failed"):
        e.synchronize()
    e.synchronize()


@pytest.mark.parametrize("call", ["step_batch", "prompt_batch", "step"])
def test_a_fault_of_an_earlier_call_is_known_before_a_state_advances(made, call):
    e, model = made
    post = fe.load_library().febtest_post_device_error
    post.argtypes = [C.c_void_p, C.c_int]
    e.prompt_batch([[1, 2]], [0])
    e.reset()
    e.step(1)
    run = {"step_batch": lambda: e.step_batch([3], [0])[0], "prompt_batch": lambda: e.prompt_batch([[3]], [0], resume=True)[0],
           "step": lambda: e.step(3)}[call]
    assert post(e.handle, 7) == 0  # a dependency wait that gave up
    with pytest.raises(FlowEdgeError, match="earlier call.*timed out"):
        run()
    np.testing.assert_allclose(run(), model.run([1, 3] if call == "step" else [1, 2, 3])[-1], atol=1e-3)
