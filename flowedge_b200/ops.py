"""Operators on CUDA tensors over the C ABI (include/flowedge_b200.h, part 3).

The Mamba mixer's operators for many sequences whose states live in slots:
ragged prompts (`offsets`) or one token per row, each sequence with a slot of
a pool (`slots`; negative skips it) and, where `fresh` says so, a zero start;
products of a few rows with 4-bit weights; the residual and the norms around it.

Each call checks its arguments, enqueues its kernels on the current stream of
its tensors' device and returns; it keeps nothing.  A refused argument raises
FlowEdgeError (status 1) before anything is launched.  These are inference
operators: tensors that require a gradient are refused while gradients are
being recorded, and tensors with a forward-mode tangent.  Outputs share no
element with inputs; states, the residual and a given `out` are changed in
place, which their version counters show (a tensor that autograd saved for a
backward pass and that is changed is found out there).  With `out` given, rows
of skipped sequences and rows behind the last sequence keep what they held;
without it they are undefined.
"""

from __future__ import annotations

import struct

import torch
import torch.autograd.forward_ad as _forward
from torch._C import _cuda_getCurrentRawStream as _raw_stream

from .engine import FlowEdgeError, load_library

__all__ = ["conv", "scan", "w4_quantize", "w4_dequantize", "w4_matvec", "residual_norm", "BAD_OFFSETS", "BAD_SLOT",
           "DUPLICATE_SLOT"]

# bits that `status` collects
BAD_OFFSETS, BAD_SLOT, DUPLICATE_SLOT = 1, 2, 4

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_CONV = struct.Struct("@IiII4Q3q9P")
_SCAN = struct.Struct("@IiII5Q5q14PQ")
_W4 = struct.Struct("@IiII3Q2q4P")  # and behind it the layout
_W4_LAYOUT = {torch.int8: struct.pack("@II", 0, 0), torch.uint8: struct.pack("@II", 1, 0)}
_W4_SIZE = _W4.size + 8
_NORM = struct.Struct("@IiII2Q4q6Pff")


def _refuse(message: str):
    raise FlowEdgeError(1, message)


def _failed(rc: int):
    raise FlowEdgeError(rc, load_library().fe_engine_last_error().decode())


# The checks below take the plain case in a few attribute reads (a call of small
# sizes costs little more than its checks); _explain goes through the same
# conditions again and names the one that failed.  `device` is a CUDA index.


def _explain(t, name: str, shape, dtype, device: int):
    if not isinstance(t, torch.Tensor):
        _refuse(f"{name} is a tensor")
    if t.dtype != dtype:
        _refuse(f"{name} is {dtype}, not {t.dtype}")
    if not t.is_cuda or t.get_device() != device:
        _refuse(f"{name} is on {t.device}, not cuda:{device}")
    if t.requires_grad and torch.is_grad_enabled():
        _refuse(f"{name} requires a gradient: this operator has none")
    if t.layout != torch.strided or t.shape != shape:
        _refuse(f"{name} has shape {tuple(t.shape)}, not {tuple(shape)}")


def _no_tangents(**tensors):
    """Refuses dual tensors (called inside a dual level alone: there are none outside)."""
    for name, t in tensors.items():
        if isinstance(t, torch.Tensor) and _forward.unpack_dual(t).tangent is not None:
            _refuse(f"{name} has a forward-mode tangent: this operator has none")


def _matrix(t, name: str, shape: tuple, dtype, device: int) -> int:
    """Checks a matrix with contiguous rows and returns the distance of its rows."""
    try:
        plain = t.dtype is dtype and t.get_device() == device and t.shape == shape and not t.requires_grad
    except (AttributeError, RuntimeError):
        plain = False
    if not plain:
        _explain(t, name, shape, dtype, device)
    ld, inner = t.stride()
    rows, width = shape
    if inner != 1 and width > 1:
        _refuse(f"{name} has rows that are not contiguous")
    return ld if rows > 1 or ld > width else width


def _flat(t, name: str, shape: tuple, dtype, device: int):
    """Checks a contiguous tensor of the given shape."""
    try:
        if (t.dtype is dtype and t.get_device() == device and t.shape == shape and t.is_contiguous()
                and not t.requires_grad):
            return
    except (AttributeError, RuntimeError):
        pass
    _explain(t, name, shape, dtype, device)
    if not t.is_contiguous():
        _refuse(f"{name} is a contiguous tensor of shape {tuple(shape)}")


def _first(x, name: str):
    """Checks the matrix that the other arguments go by: (shape, dtype, device)."""
    if not isinstance(x, torch.Tensor) or x.dtype not in _DTYPES or x.dim() != 2:
        _refuse(f"{name} is a matrix of float32, bfloat16 or float16")
    device = x.get_device() if x.is_cuda else -1
    if device < 0:
        _refuse(f"{name} is on {x.device}, not on a GPU")
    return x.shape, x.dtype, device


def _sequences(rows: int, offsets, slots, fresh, status, device: int) -> int:
    """Checks the sequences' description and returns their number."""
    n_seq = rows
    if offsets is not None:
        if not isinstance(offsets, torch.Tensor) or offsets.dim() != 1 or offsets.shape[0] < 1:
            _refuse("offsets is a tensor of n_seq + 1 elements")
        n_seq = offsets.shape[0] - 1
        _flat(offsets, "offsets", (n_seq + 1,), torch.int32, device)
    if slots is not None:
        _flat(slots, "slots", (n_seq,), torch.int32, device)
    if fresh is not None:
        _flat(fresh, "fresh", (n_seq,), torch.bool if getattr(fresh, "dtype", None) is torch.bool else torch.uint8, device)
    if status is not None:
        _flat(status, "status", (1,), torch.int32, device)
    return n_seq


def _pool(state, name: str, inner: tuple, n_seq: int, device: int) -> tuple:
    """Checks a pool of slot states and returns (slots, distance of two slots)."""
    if not isinstance(state, torch.Tensor) or state.dim() != 3:
        _refuse(f"{name} is a tensor of shape {('slots',) + inner}")
    n_slots = state.shape[0]
    if (state.dtype is not torch.float32 or state.get_device() != device or state.shape != (n_slots, *inner)
            or state.requires_grad):
        _explain(state, name, (n_slots, *inner), torch.float32, device)
    outer, mid, last = state.stride()
    if (mid != inner[1] and inner[0] > 1) or (last != 1 and inner[1] > 1):
        _refuse(f"{name} has slots that are not contiguous")
    if n_slots == 0 and n_seq > 0:  # (an empty tensor has no address: the call would run without states)
        _refuse(f"{name} has no slots")
    per = inner[0] * inner[1]
    return n_slots, outer if n_slots > 1 or outer > per else per


def _changed(*tensors):
    """Raises the version counters of tensors that a call has written (inference tensors have none)."""
    try:
        torch._C._increment_version(tensors)
    except RuntimeError:
        for t in tensors:
            if not t.is_inference():
                torch._C._increment_version((t,))


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def conv(x, weight, bias, *, window=None, offsets=None, slots=None, fresh=None, status=None, out=None):
    """SiLU(short causal depthwise convolution): u[t, c] = SiLU(bias[c] + sum_k weight[c, k] x[t - (d_conv - 1) + k, c]).

    x [rows, d_inner] float32 / bfloat16 / float16 (rows may be apart); weight [d_inner, d_conv] and bias [d_inner]
    float32, d_conv 1 to 8.  `window` [slots, d_inner, d_conv] float32 holds each slot's last inputs, newest last; a
    sequence reads the inputs before its first row there and leaves its own last ones.  Returns u like x.
    """
    if _forward._current_level >= 0:
        _no_tangents(x=x, weight=weight, bias=bias, window=window, out=out)
    shape, dtype, device = _first(x, "x")
    rows, di = shape
    x_ld = _matrix(x, "x", shape, dtype, device)
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        _refuse("weight is a tensor of shape (d_inner, d_conv)")
    dc = weight.shape[1]
    _flat(weight, "weight", (di, dc), torch.float32, device)
    _flat(bias, "bias", (di,), torch.float32, device)
    n_seq = _sequences(rows, offsets, slots, fresh, status, device)
    n_slots, stride = (0, 0) if window is None else _pool(window, "window", (di, dc), n_seq, device)
    written = () if window is None else (window,)
    if out is None:
        out = torch.empty_like(x)
    else:
        written += (out,)
    u_ld = _matrix(out, "out", shape, dtype, device)
    args = _CONV.pack(_CONV.size, device, _DTYPES[dtype], dc, rows, di, n_seq, n_slots, x_ld, u_ld, stride,
                      x.data_ptr(), weight.data_ptr(), bias.data_ptr(), out.data_ptr(), _ptr(window), _ptr(offsets),
                      _ptr(slots), _ptr(fresh), _ptr(status))
    rc = load_library().fe_causal_conv_device(args, _raw_stream(device))
    if rc:
        _failed(rc)
    if written:
        _changed(*written)
    return out


def scan(u, proj, a, d, dt_w, dt_b, *, z=None, state=None, offsets=None, slots=None, fresh=None, status=None,
         out=None):
    """The selective scan with its step projection and gate.

    A row of proj is [dt_in (dt_rank) | B (d_state) | C (d_state)].  Per row and channel: dt = softplus(dt_in dt_w +
    dt_b), h = exp(dt a) h + dt B u, y = (d u + sum h C) SiLU(z); without z there is no gate.  u, z [rows, d_inner]
    and proj are float32, bfloat16 or float16 alike (rows may be apart); a [d_state, d_inner] (negative), d [d_inner],
    dt_w [dt_rank, d_inner] and dt_b [d_inner] float32, d_state 1 to 32, dt_rank 1 to 512.  `state` [slots, d_state,
    d_inner] float32.  Returns y like u.
    """
    if _forward._current_level >= 0:
        _no_tangents(u=u, proj=proj, a=a, d=d, dt_w=dt_w, dt_b=dt_b, z=z, state=state, out=out)
    shape, dtype, device = _first(u, "u")
    rows, di = shape
    u_ld = _matrix(u, "u", shape, dtype, device)
    if not isinstance(a, torch.Tensor) or a.dim() != 2 or not isinstance(dt_w, torch.Tensor) or dt_w.dim() != 2:
        _refuse("a is a tensor of shape (d_state, d_inner) and dt_w one of shape (dt_rank, d_inner)")
    ds, dr = a.shape[0], dt_w.shape[0]
    proj_ld = _matrix(proj, "proj", (rows, dr + 2 * ds), dtype, device)
    z_ld = 0 if z is None else _matrix(z, "z", shape, dtype, device)
    _flat(a, "a", (ds, di), torch.float32, device)
    _flat(d, "d", (di,), torch.float32, device)
    _flat(dt_w, "dt_w", (dr, di), torch.float32, device)
    _flat(dt_b, "dt_b", (di,), torch.float32, device)
    n_seq = _sequences(rows, offsets, slots, fresh, status, device)
    n_slots, stride = (0, 0) if state is None else _pool(state, "state", (ds, di), n_seq, device)
    written = () if state is None else (state,)
    if out is None:
        out = torch.empty_like(u)
    else:
        written += (out,)
    y_ld = _matrix(out, "out", shape, dtype, device)
    lib = load_library()
    workspace, size = 0, 0
    if offsets is not None or n_seq >= 16:  # fewer single tokens need none
        # the sizes alone decide; the tensor returns to torch's allocator in stream order
        size = lib.fe_selective_scan_workspace(_SCAN.pack(_SCAN.size, device, _DTYPES[dtype], ds, rows, di, dr, n_seq,
                                                          n_slots, u_ld, proj_ld, z_ld, y_ld, stride, 0, 0, 0, 0, 0, 0,
                                                          0, 0, 0, _ptr(offsets), 0, 0, 0, 0, 0))
        if size:
            held = u.new_empty(size, dtype=torch.uint8)
            workspace = held.data_ptr()
    args = _SCAN.pack(_SCAN.size, device, _DTYPES[dtype], ds, rows, di, dr, n_seq, n_slots, u_ld, proj_ld, z_ld, y_ld,
                      stride, u.data_ptr(), proj.data_ptr(), _ptr(z), a.data_ptr(), d.data_ptr(), dt_w.data_ptr(),
                      dt_b.data_ptr(), out.data_ptr(), _ptr(state), _ptr(offsets), _ptr(slots), _ptr(fresh),
                      _ptr(status), workspace, size)
    rc = lib.fe_selective_scan_device(args, _raw_stream(device))
    if rc:
        _failed(rc)
    if written:
        _changed(*written)
    return out


# Packed 4-bit weights come in two layouts, which their type tells apart: uint8 has a row's words in the order of their
# elements, int8 has them in blocks of 128 elements in the order in which the products read them.


def _w4_shapes(m: int, k: int, group: int, packed_dtype) -> tuple:
    if group not in (32, 64, 128):
        _refuse(f"group is 32, 64 or 128, not {group}")
    width = (k + 31) // 32 * 16 if packed_dtype is torch.uint8 else (k + 127) // 128 * 64
    return (m, width), (m, (k + group - 1) // group)


def w4_quantize(weight, group: int = 64, *, layout: str = "blocks") -> tuple:
    """(packed, scales) of a finite weight matrix [m, k]: 4 bits per element, one float16 scale per `group` of k.

    packed is int8 [m, ceil(k / 128) * 64] in blocks of 128 elements, or with `layout` "rows" uint8
    [m, ceil(k / 32) * 16] in the order of the elements (include/flowedge_b200.h, fe_w4_args, has both; products with
    groups of 32 and 64 read blocks faster); scales [m, ceil(k / group)].  Its type tells the other calls which layout a
    packed weight has.
    """
    if _forward._current_level >= 0:
        _no_tangents(weight=weight)
    shape, dtype, device = _first(weight, "weight")
    m, k = shape
    ld = _matrix(weight, "weight", shape, dtype, device)
    if layout not in ("blocks", "rows"):
        _refuse(f"layout is 'blocks' or 'rows', not {layout!r}")
    packed_dtype = torch.uint8 if layout == "rows" else torch.int8
    packed_shape, scales_shape = _w4_shapes(m, k, group, packed_dtype)
    packed = weight.new_empty(packed_shape, dtype=packed_dtype)
    scales = weight.new_empty(scales_shape, dtype=torch.float16)
    args = _W4.pack(_W4_SIZE, device, _DTYPES[dtype], group, 0, m, k, ld, 0, weight.data_ptr(), packed.data_ptr(),
                    scales.data_ptr(), 0) + _W4_LAYOUT[packed_dtype]
    rc = load_library().fe_w4_quantize_device(args, _raw_stream(device))
    if rc:
        _failed(rc)
    return packed, scales


def _w4_weight(packed, scales, k: int, group: int, device: int) -> int:
    """Checks a packed weight of k columns and returns its rows."""
    if not isinstance(packed, torch.Tensor) or packed.dim() != 2 or packed.dtype not in _W4_LAYOUT:
        _refuse("packed is an int8 tensor of shape (m, ceil(k / 128) * 64) or a uint8 one of shape (m, ceil(k / 32) * 16)")
    m = packed.shape[0]
    packed_shape, scales_shape = _w4_shapes(m, k, group, packed.dtype)
    _flat(packed, "packed", packed_shape, packed.dtype, device)
    _flat(scales, "scales", scales_shape, torch.float16, device)
    return m


def w4_dequantize(packed, scales, k: int, *, group: int = 64, dtype=torch.float32):
    """The matrix [m, k] that a packed weight of either layout stands for, rounded to `dtype`."""
    if _forward._current_level >= 0:
        _no_tangents(scales=scales)
    if dtype not in _DTYPES:
        _refuse("dtype is float32, bfloat16 or float16")
    if not isinstance(packed, torch.Tensor) or not packed.is_cuda:
        _refuse("packed is a tensor on a GPU")
    device = packed.get_device()
    m = _w4_weight(packed, scales, k, group, device)
    weight = packed.new_empty((m, k), dtype=dtype)
    args = _W4.pack(_W4_SIZE, device, _DTYPES[dtype], group, 0, m, k, 0, k, 0, packed.data_ptr(), scales.data_ptr(),
                    weight.data_ptr()) + _W4_LAYOUT[packed.dtype]
    rc = load_library().fe_w4_dequantize_device(args, _raw_stream(device))
    if rc:
        _failed(rc)
    return weight


def w4_matvec(x, packed, scales, *, group: int = 64, out=None):
    """x [rows, k] times the transpose of a packed weight [m, k], for a few rows (32 read the weight once).

    float32, bfloat16 or float16 x and result; sums in float32, the weight exact.  packed is uint8 with its words in the
    order of their elements, or int8 in blocks (w4_quantize).
    """
    if _forward._current_level >= 0:
        _no_tangents(x=x, scales=scales, out=out)
    shape, dtype, device = _first(x, "x")
    rows, k = shape
    x_ld = _matrix(x, "x", shape, dtype, device)
    m = _w4_weight(packed, scales, k, group, device)
    given = out is not None
    if given:
        y_ld = _matrix(out, "out", (rows, m), dtype, device)
    else:
        out, y_ld = x.new_empty((rows, m)), m
    args = _W4.pack(_W4_SIZE, device, _DTYPES[dtype], group, rows, m, k, x_ld, y_ld, x.data_ptr(), packed.data_ptr(),
                    scales.data_ptr(), out.data_ptr()) + _W4_LAYOUT[packed.dtype]
    rc = load_library().fe_w4_matvec_device(args, _raw_stream(device))
    if rc:
        _failed(rc)
    if given:
        _changed(out)
    return out


def residual_norm(x, residual, weight, *, post_weight=None, gate=None, scale: float = 1.0, eps: float = 1e-5, out=None):
    """residual += scale * gate * RMSNorm(x; post_weight), in place; returns RMSNorm(residual; weight).

    x, gate ([rows, dim], or [1, dim] for all rows) and the result are float32, bfloat16 or float16 alike; residual
    float32 or the same; weights [dim] float32, dim 1 to 16384.  Without post_weight x is added as it is.  The returned
    norm is taken before the residual is rounded to its type.
    """
    if _forward._current_level >= 0:
        _no_tangents(x=x, residual=residual, weight=weight, post_weight=post_weight, gate=gate, out=out)
    shape, dtype, device = _first(x, "x")
    rows, dim = shape
    x_ld = _matrix(x, "x", shape, dtype, device)
    r_dtype = dtype if getattr(residual, "dtype", None) is dtype else torch.float32
    r_ld = _matrix(residual, "residual", shape, r_dtype, device)
    _flat(weight, "weight", (dim,), torch.float32, device)
    if post_weight is not None:
        _flat(post_weight, "post_weight", (dim,), torch.float32, device)
    gate_ld = 0
    if gate is not None:
        one = isinstance(gate, torch.Tensor) and gate.dim() == 2 and gate.shape[0] == 1
        gate_ld = _matrix(gate, "gate", (1, dim) if one else shape, dtype, device)
        gate_ld = 0 if one else gate_ld
    written = (residual,)
    if out is None:
        out = torch.empty_like(x)
    else:
        written += (out,)
    y_ld = _matrix(out, "out", shape, dtype, device)
    try:
        args = _NORM.pack(_NORM.size, device, _DTYPES[dtype], _DTYPES[r_dtype], rows, dim, x_ld, r_ld, gate_ld, y_ld,
                          x.data_ptr(), _ptr(post_weight), _ptr(gate), residual.data_ptr(), weight.data_ptr(),
                          out.data_ptr(), scale, eps)
    except struct.error:
        _refuse("scale and eps are numbers")
    rc = load_library().fe_residual_norm_device(args, _raw_stream(device))
    if rc:
        _failed(rc)
    _changed(*written)
    return out
