"""Ragged prompts and batched single tokens over the engine's slots (through the C ABI), against the oracle.

Tolerances are the bars of the other Mamba parity tests: max-abs 1e-3 for fp32 engines, 2e-2 for bf16 engines (their
weights rounded to bf16 in the oracle's copy too); 4-bit engines compare with the oracle on the values that the packed
weights stand for."""

import ctypes as C

import numpy as np
import pytest
import torch

from flowedge_b200 import Engine, FlowEdgeError
from flowedge_b200 import checkpoint as ck
from flowedge_b200 import engine as fe
from oracle import restate

pytestmark = pytest.mark.gpu

SPECS = {"wide": ck.MambaSpec(vocab=40, d_model=128, n_layers=2, d_inner=256, d_state=16, d_conv=4, dt_rank=32),
         "odd": ck.MambaSpec(vocab=17, d_model=72, n_layers=3, d_inner=120, d_state=8, d_conv=3, dt_rank=4)}


def _w4(w, group):
    """The values of a weight rounded to 4 bits by the documented rule."""
    m, k = w.shape
    pad = np.zeros((m, -(-k // group) * group), np.float32)
    pad[:, :k] = w
    g = pad.reshape(m, -1, group)
    s = (np.abs(g).max(2) / np.float32(7)).astype(np.float16).astype(np.float32)[:, :, None]
    q = np.clip(np.rint(np.divide(g, s, out=np.zeros_like(g), where=s > 0)), -8, 7)
    return (q * s).reshape(m, -1)[:, :k].astype(np.float32)


def _model(tensors, precision, group):
    t = {}
    for name, v in tensors.items():
        if "_proj.weight" in name and "dt_proj" not in name and group:
            v = _w4(v, group)
        elif "_proj.weight" in name and precision == "bf16":
            v = ck.bf16_bits_to_f32(ck.to_bf16_bits(v))
        t[name] = v
    return restate.MambaModel(t)


@pytest.fixture(scope="module")
def engines(tmp_path_factory):
    made = {}

    def get(spec, precision="fp32", group=0, seed=3):
        key = (spec, precision, group)
        if key not in made:
            tensors = ck.mamba_tensors(SPECS[spec], seed=seed)
            path = tmp_path_factory.mktemp("slots") / "m.safetensors"
            ck.write_checkpoint(path, tensors)
            e = Engine(path, threads=0, device=0, precision=precision, max_sequence=400, weights4_group=group)
            e.reserve_slots(8)
            made[key] = (e, _model(tensors, precision, group), path)
        return made[key]

    yield get
    for e, _, _ in made.values():
        e.close()


def _bar(precision):
    return 1e-3 if precision == "fp32" else 2e-2


@pytest.mark.parametrize("precision,group", [("fp32", 0), ("bf16", 0), ("fp32", 64), ("bf16", 32), ("bf16", 128)])
@pytest.mark.parametrize("spec", ["wide", "odd"])
@pytest.mark.parametrize("lengths", [[1], [5, 1, 17], [40, 3, 90, 25, 1], [200]])
def test_prompts_then_tokens(engines, spec, precision, group, lengths):
    """Ragged prompts leave the states that batched tokens continue from (few rows, the GEMM's rows, 4-bit weights)."""
    e, model, _ = engines(spec, precision, group)
    rng = np.random.default_rng(sum(lengths))
    vocab = SPECS[spec].vocab
    prompts = [rng.integers(0, vocab, n).astype(np.int32) for n in lengths]
    slots = rng.permutation(8)[:len(lengths)]
    got = e.prompt_batch(prompts, slots)
    want = [model.run(p) for p in prompts]
    np.testing.assert_allclose(got, np.stack([w[-1] for w in want]), atol=_bar(precision))
    tails = rng.integers(0, vocab, (3, len(lengths))).astype(np.int32)
    for i in range(3):
        order = rng.permutation(len(lengths))  # the batch's order is free
        rows = e.step_batch(tails[i][order], slots[order])
        for r, s in zip(rows, order):
            full = np.concatenate([prompts[s], tails[:i + 1, s]])
            np.testing.assert_allclose(r, model.run(full)[-1], atol=_bar(precision))


def test_pieces_equal_the_whole_and_the_single_stream(engines):
    e, model, _ = engines("wide")
    tokens = np.random.default_rng(1).integers(0, 40, 30).astype(np.int32)
    whole = e.prompt_batch([tokens], [2])
    e.prompt_batch([tokens[:11], tokens[:4]], [5, 0])
    e.prompt_batch([tokens[11:20], tokens[4:20]], [5, 0], resume=True)
    last = e.prompt_batch([tokens[20:], tokens[20:]], [5, 0], resume=True)
    np.testing.assert_allclose(last, np.repeat(whole, 2, 0), atol=2e-5, rtol=1e-4)
    e.reset()
    e.reset_slots([6, 7])
    for t in tokens[:12]:
        one = e.step(t)
        two = e.step_batch([t, t], [7, 6])
        np.testing.assert_allclose(two, np.stack([one, one]), atol=2e-5, rtol=1e-4)


def test_existing_entry_points_see_the_4_bit_weights(engines):
    e, model, _ = engines("wide", "fp32", 64)
    tokens = np.random.default_rng(2).integers(0, 40, 140).astype(np.int32)
    np.testing.assert_allclose(e.run(tokens), model.run(tokens), atol=1e-3)
    np.testing.assert_allclose(e.run(tokens[:9]), model.run(tokens[:9]), atol=1e-3)
    e.reset()
    np.testing.assert_allclose(np.stack([e.step(t) for t in tokens[:6]]), model.run(tokens[:6]), atol=1e-3)


def _dev(a, dtype=torch.int32):
    return torch.as_tensor(a, dtype=dtype, device="cuda")


def test_device_buffers_padding_status_and_capture(engines):
    e, model, _ = engines("wide")
    rng = np.random.default_rng(4)
    tokens = rng.integers(0, 40, 60).astype(np.int32)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        toks, offs = _dev(tokens), _dev([0, 20, 20, 45, 60])
        slots, fresh = _dev([3, 1, -1, 4]), _dev([1, 1, 1, 1], torch.uint8)
        out, status = torch.full((4, 128), 7.0, device="cuda"), _dev([0])
        e.prompt_device(toks.data_ptr(), 60, offs.data_ptr(), slots.data_ptr(), 4, out.data_ptr(), fresh.data_ptr(),
                        status.data_ptr(), stream.cuda_stream)
        step_tokens, step_slots = _dev([1, 2, 3, 4]), _dev([4, -1, 3, 1])
        steps = torch.full((4, 128), 7.0, device="cuda")
        e.step_device(step_tokens.data_ptr(), step_slots.data_ptr(), 4, steps.data_ptr(), stream=stream.cuda_stream)
    stream.synchronize()
    e.synchronize()
    assert int(status) == 0
    np.testing.assert_allclose(out[0].cpu(), model.run(tokens[:20])[-1], atol=1e-3)
    np.testing.assert_allclose(out[3].cpu(), model.run(tokens[45:])[-1], atol=1e-3)
    assert (out[1:3] == 7).all() and (steps[1] == 7).all()  # an empty prompt and skipped ones
    np.testing.assert_allclose(steps[0].cpu(), model.run(np.append(tokens[45:], 1))[-1], atol=1e-3)
    np.testing.assert_allclose(steps[2].cpu(), model.run(np.append(tokens[:20], 3))[-1], atol=1e-3)
    np.testing.assert_allclose(steps[3].cpu(), model.run([4])[-1], atol=1e-3)
    # a caller's graph of one step replays over new tokens
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        e.step_device(step_tokens.data_ptr(), step_slots.data_ptr(), 4, steps.data_ptr(),
                      stream=torch.cuda.current_stream().cuda_stream)
    for t in (5, 6):
        step_tokens.fill_(t)
        graph.replay()
    torch.cuda.synchronize()
    np.testing.assert_allclose(steps[3].cpu(), model.run([4, 5, 6])[-1], atol=1e-3)
    # the same slot twice: the first one runs, the other is reported
    step_slots.copy_(_dev([2, 2, 9, -1]))
    steps.fill_(7.0)
    e.step_device(step_tokens.data_ptr(), step_slots.data_ptr(), 4, steps.data_ptr(), status.data_ptr(),
                  torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert int(status) == 4 | 2
    assert (steps[0] != 7).any() and (steps[1:] == 7).all()  # what did not run leaves its row
    # a token outside the vocabulary is reported, not read
    step_tokens.fill_(40)
    e.step_device(step_tokens.data_ptr(), step_slots[:1].data_ptr(), 1, steps.data_ptr(), stream=0)
    with pytest.raises(FlowEdgeError, match="Device work failed"):
        e.synchronize()
    e.synchronize()


def test_growth_keeps_states_and_warm_calls_do_not_allocate(engines):
    _, model, path = engines("odd")
    e = Engine(path, threads=0, device=0, precision="fp32", max_sequence=16)
    e.reserve_slots(2)
    tokens = np.random.default_rng(5).integers(0, 17, 50).astype(np.int32)
    e.prompt_batch([tokens[:8], tokens[:3]], [1, 0])
    e.reserve_slots(5)  # a larger pool
    np.testing.assert_allclose(e.step_batch(tokens[8:9], [1])[0], model.run(tokens[:9])[-1], atol=1e-3)
    np.testing.assert_allclose(e.prompt_batch([tokens], [4])[0], model.run(tokens)[-1], atol=1e-3)  # more rows than reserved
    np.testing.assert_allclose(e.step_batch(tokens[9:10], [1])[0], model.run(tokens[:10])[-1], atol=1e-3)
    np.testing.assert_allclose(e.step_batch(tokens[3:4], [0])[0], model.run(tokens[:4])[-1], atol=1e-3)
    before = fe.device_malloc_count(), fe.host_malloc_count()
    for n in (1, 3):
        e.prompt_batch([tokens[:16]] * n, list(range(n)))  # 48 rows at most, of the 50 there is room for
        e.step_batch(tokens[:n], list(range(n)))
    assert (fe.device_malloc_count(), fe.host_malloc_count()) == before
    e.reserve_batch(4)  # the batch's buffers move: the slots' follow
    history = np.concatenate([tokens[:16], tokens[:1], tokens[20:21]])
    np.testing.assert_allclose(e.step_batch(tokens[20:21], [0])[0], model.run(history)[-1], atol=1e-3)
    e.close()


def test_growth_beyond_the_device_leaves_everything_usable(engines):
    """No device holds the batch: the call says so, and the buffers, the single stream's state and the slots' stay."""
    _, model, path = engines("odd")
    e = Engine(path, threads=0, device=0, precision="fp32", max_sequence=16)
    e.reserve_slots(2)
    tokens = np.random.default_rng(6).integers(0, 17, 24).astype(np.int32)
    for t in tokens[:5]:
        e.step(int(t))
    e.prompt_batch([tokens[:8]], [1])
    for batch in (1 << 30, 1 << 62):
        with pytest.raises(FlowEdgeError, match="status 2"):
            e.reserve_batch(batch)
    np.testing.assert_allclose(e.step(int(tokens[5])), model.run(tokens[:6])[-1], atol=1e-3)
    np.testing.assert_allclose(e.step_batch(tokens[8:9], [1])[0], model.run(tokens[:9])[-1], atol=1e-3)
    np.testing.assert_allclose(e.prompt_batch([tokens], [0])[0], model.run(tokens)[-1], atol=1e-3)  # grows
    np.testing.assert_allclose(e.step(int(tokens[6])), model.run(tokens[:7])[-1], atol=1e-3)
    e.close()


def test_slot_refusals(engines, golden):
    e, _, path = engines("odd")
    fresh = Engine(path, threads=0, device=0, precision="fp32")
    for call, status in [(lambda: fresh.step_batch([1], [0]), 7), (lambda: fresh.prompt_batch([[1]], [0]), 7),
                         (lambda: e.step_batch([1], [8]), 1), (lambda: e.step_batch([1], [-1]), 1),
                         (lambda: e.step_batch([1, 2], [3, 3]), 1), (lambda: e.step_batch([17], [0]), 3),
                         (lambda: e.step_batch([1, 2], [0]), 1), (lambda: e.step_batch([], []), 1),
                         (lambda: e.prompt_batch([[1], []], [0, 1]), 1), (lambda: e.prompt_batch([[1], [2]], [4, 4]), 1),
                         (lambda: e.prompt_batch([[-1]], [0]), 3), (lambda: e.prompt_batch([], []), 1),
                         (lambda: e.reset_slots([9]), 1), (lambda: e.reserve_slots(0), 1)]:
        with pytest.raises(FlowEdgeError, match=f"status {status}"):
            call()
    fresh.close()
    unet = Engine("tests/golden/unet_tiny.safetensors", threads=0, device=0)
    with pytest.raises(FlowEdgeError, match="status 4"):
        unet.reserve_slots(2)
    unet.close()
    with pytest.raises(RuntimeError, match="weights4_group"):
        Engine(path, threads=0, device=0, weights4_group=16)


def test_options_of_the_earlier_size(engines):
    """A caller built before the 4-bit field passes a shorter structure."""
    _, _, path = engines("odd")
    lib = fe.load_library()
    size = fe.EngineOptions.weights4_group.offset
    opts = fe.EngineOptions(size, 0, 0, 1, 1, 16, 99, 99)  # what lies behind is not read
    h = lib.fe_engine_load_with_options(str(path).encode(), C.byref(opts))
    assert h
    lib.fe_engine_free(h)
    opts.struct_size = size - 8
    assert not lib.fe_engine_load_with_options(str(path).encode(), C.byref(opts))
