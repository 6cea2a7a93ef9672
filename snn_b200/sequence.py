"""The sequence operators over CUDA tensors (Part 4 of include/snn_b200.h).

Thin mirrors of the C entry points for callers whose arrays are torch tensors:
outputs and workspaces come from torch's allocator, the work goes to the
tensors' device and to its current stream, and a refused call raises SnnError.
A tensor of uint8 or bool is a spike raster (non-zero = one spike).

    w = mx4_quantize(weights)                  # [post, pre], packed once
    current = mx4_linear(raster, w)            # [rows, pre] -> [rows, post]
    y, h_last = leaky_scan(current, decays)    # [batch, steps, channels]
"""
from __future__ import annotations

import ctypes as C
import math

from . import SNN_ERR_INVALID_ARGUMENT, SnnError, _check, lib

F32, F16, BF16, SPIKES = 0, 1, 2, 3
LEAKY_BLOCK = 8  # SNN_B200_LEAKY_BLOCK


class _Torch:
    """torch, the element types and the library, looked up at the first call
    (importing snn_b200 needs neither)."""

    def __init__(self):
        import torch
        self.torch = torch
        self.codes = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16, torch.uint8: SPIKES,
                      torch.bool: SPIKES}
        self.float32, self.uint8, self.empty = torch.float32, torch.uint8, torch.empty
        # torch's own short way to the current stream's handle, where it has one.
        self.stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                              lambda device: torch.cuda.current_stream(device).cuda_stream)
        self.lib = lib()


_T = None


def _t() -> _Torch:
    global _T
    if _T is None:
        _T = _Torch()
    return _T


def _refuse(what: str):
    raise SnnError(SNN_ERR_INVALID_ARGUMENT, what)


def _code(T, t, what: str) -> int:
    code = T.codes.get(t.dtype)
    if code is None:
        _refuse(f"{what}: element type {t.dtype} is not one of float32, float16, bfloat16, uint8, bool")
    return code


def _device(first, *others) -> int:
    """The CUDA device that all the tensors are on."""
    d = first.get_device()
    if d < 0:
        _refuse("tensors must be on a CUDA device")
    for t in others:
        if t is not None and t.get_device() != d:
            _refuse("tensors must be on one CUDA device")
    return d


def _state(T, t, shape, what: str):
    """A float32 tensor of `shape`, contiguous."""
    if t is None:
        return None
    if t.dtype != T.float32 or t.shape != shape:
        _refuse(f"{what}: float32 of shape {shape} expected")
    return t.contiguous()


def _p(t):
    return None if t is None else t.data_ptr()


# ---------------------------------------------------------------------------
# MXFP4
# ---------------------------------------------------------------------------
class Mx4:
    """A packed matrix: `codes` and `scales` (uint8 tensors laid out as the
    header says) of `rows` x `cols` elements."""
    __slots__ = ("codes", "scales", "rows", "cols")

    def __init__(self, codes, scales, rows: int, cols: int):
        self.codes, self.scales, self.rows, self.cols = codes, scales, rows, cols

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()


def mx4_sizes(rows: int, cols: int) -> tuple[int, int]:
    """Bytes of a packed matrix's codes and scales (snn_b200_mx4_sizes)."""
    a, b = C.c_uint64(), C.c_uint64()
    _check(lib().snn_b200_mx4_sizes(rows, cols, C.byref(a), C.byref(b)), "snn_b200_mx4_sizes")
    return a.value, b.value


def mx4_quantize(x, out: Mx4 | None = None) -> Mx4:
    """Packs the rows of a 2-D tensor (any strides; `w.t()` packs a layer
    stored one row per presynaptic neuron), into `out` where given."""
    T = _t()
    dev = _device(x)
    if x.dim() != 2:
        _refuse("mx4_quantize: a 2-D tensor expected")
    rows, cols = x.shape
    code = _code(T, x, "mx4_quantize")
    if out is None:
        blocks = (cols + 31) // 32  # as snn_b200_mx4_sizes
        ns = (rows + 127) // 128 * ((blocks + 3) // 4) * 512 if cols else 0
        out = Mx4(T.empty(rows * blocks * 16, dtype=T.uint8, device=x.device),
                  T.empty(ns, dtype=T.uint8, device=x.device), rows, cols)
    elif (out.rows, out.cols) != (rows, cols) or out.codes.get_device() != dev:
        _refuse("mx4_quantize: `out` is of another shape or device")
    rs, cs = x.stride()
    st = T.lib.snn_b200_mx4_quantize_async(dev, T.stream(dev), x.data_ptr(), code, rows, cols, rs, cs,
                                           out.codes.data_ptr(), out.scales.data_ptr())
    if st:
        _check(st, "snn_b200_mx4_quantize_async")
    return out


def mx4_dequantize(q: Mx4, dtype=None):
    """The values that a packed matrix stands for (float32 by default)."""
    T = _t()
    dev = _device(q.codes, q.scales)
    y = T.empty((q.rows, q.cols), dtype=dtype or T.float32, device=q.codes.device)
    st = T.lib.snn_b200_mx4_dequantize_async(dev, T.stream(dev), q.codes.data_ptr(), q.scales.data_ptr(), q.rows,
                                             q.cols, y.data_ptr(), _code(T, y, "mx4_dequantize"), q.cols)
    if st:
        _check(st, "snn_b200_mx4_dequantize_async")
    return y


def _bias(T, bias, n: int):
    if bias is None:
        return None
    if bias.dtype != T.float32 or bias.shape != (n,) or not bias.is_contiguous():
        _refuse(f"bias: {n} contiguous float32 expected")
    return bias.data_ptr()


def mx4_matmul(x: Mx4, w: Mx4, bias=None, dtype=None):
    """x [m, k] times the transpose of w [n, k], plus bias [n]."""
    T = _t()
    dev = _device(x.codes, x.scales, w.codes, w.scales, bias)
    if x.cols != w.cols:
        _refuse(f"mx4_matmul: {x.cols} columns against {w.cols}")
    y = T.empty((x.rows, w.rows), dtype=dtype or T.float32, device=x.codes.device)
    st = T.lib.snn_b200_mx4_matmul_async(dev, T.stream(dev), x.codes.data_ptr(), x.scales.data_ptr(), x.rows,
                                         w.codes.data_ptr(), w.scales.data_ptr(), w.rows, w.cols,
                                         _bias(T, bias, w.rows), y.data_ptr(), _code(T, y, "mx4_matmul"), w.rows)
    if st:
        _check(st, "snn_b200_mx4_matmul_async")
    return y


def mx4_linear(x, w: Mx4, bias=None, dtype=None):
    """x [..., k] packed on the way, times the transpose of w [n, k], plus
    bias [n]: the currents that a raster (or activations) sends through a
    packed layer. The result's type is x's, float32 for spikes, or `dtype`."""
    T = _t()
    dev = _device(x, w.codes, w.scales, bias)
    k, n = w.cols, w.rows
    shape = x.shape
    if not shape or shape[-1] != k:
        _refuse(f"mx4_linear: rows of {k} elements expected, not {tuple(shape)}")
    code = _code(T, x, "mx4_linear")
    flat = x if len(shape) == 2 else x.reshape(math.prod(shape[:-1]), k)
    m = flat.shape[0]
    out = dtype or (T.float32 if code == SPIKES else x.dtype)
    y = T.empty((m, n), dtype=out, device=x.device)
    need = T.lib.snn_b200_mx4_linear_workspace(m, k)
    ws = T.empty(need, dtype=T.uint8, device=x.device)
    rs, cs = flat.stride()
    st = T.lib.snn_b200_mx4_linear_async(dev, T.stream(dev), flat.data_ptr(), code, m, k, rs, cs, w.codes.data_ptr(),
                                         w.scales.data_ptr(), n, _bias(T, bias, n), y.data_ptr(),
                                         T.codes.get(out, -1), n, ws.data_ptr(), need)
    if st:
        _check(st, "snn_b200_mx4_linear_async")
    return y if len(shape) == 2 else y.view(*shape[:-1], n)


# ---------------------------------------------------------------------------
# Leaky recurrence
# ---------------------------------------------------------------------------
class Leaky(C.Structure):
    """snn_b200_leaky_t (include/snn_b200.h)."""
    _fields_ = [("batch", C.c_uint64), ("steps", C.c_uint64), ("channels", C.c_uint64),
                ("x_dtype", C.c_int), ("gate_dtype", C.c_int), ("y_dtype", C.c_int),
                ("logit", C.c_int), ("complement", C.c_int), ("decay", C.c_float), ("input_scale", C.c_float),
                ("x_batch_stride", C.c_int64), ("x_step_stride", C.c_int64),
                ("gate_batch_stride", C.c_int64), ("gate_step_stride", C.c_int64),
                ("y_batch_stride", C.c_int64), ("y_step_stride", C.c_int64),
                ("dy_batch_stride", C.c_int64), ("dy_step_stride", C.c_int64),
                ("dx_batch_stride", C.c_int64), ("dx_step_stride", C.c_int64),
                ("dgate_batch_stride", C.c_int64), ("dgate_step_stride", C.c_int64)]


def _sequences(t, what: str):
    """[batch, steps, channels] with neighbouring channels, and its strides."""
    if t.dim() != 3:
        _refuse(f"{what}: [batch, steps, channels] expected")
    strides = t.stride()
    if strides[2] != 1 and t.shape[2] > 1:
        t = t.contiguous()
        strides = t.stride()
    return t, strides


def _gate(T, gate, decay, shape):
    """The gate array, its type and its strides over the sequences and the
    steps: [channels], [batch, channels] or [batch, steps, channels]."""
    if (gate is None) == (decay is None):
        _refuse("leaky: either a gate array or a decay is needed")
    if gate is None:
        return None, F32, 0, 0
    own = gate.shape
    if own != shape and own != shape[2:] and own != (shape[0], shape[2]):
        _refuse(f"leaky: a gate of shape [channels], [batch, channels] or [batch, steps, channels] expected, not "
                f"{tuple(own)}")
    strides = gate.stride()
    if strides[-1] != 1 and own[-1] > 1:
        gate = gate.contiguous()
        strides = gate.stride()
    dims = len(own)
    return gate, _code(T, gate, "gate"), strides[0] if dims > 1 else 0, strides[1] if dims == 3 else 0


def _lengths(T, lengths, batch: int):
    if lengths is None:
        return None
    if lengths.dtype not in (T.torch.int32, T.torch.uint32) or lengths.shape != (batch,) \
            or not lengths.is_contiguous():
        _refuse(f"lengths: {batch} contiguous int32 expected")
    return lengths.data_ptr()


def _like(T, x, strides, dtype):
    """An empty [batch, steps, channels] tensor whose steps come first in
    memory where x's do, and its strides."""
    b, t, c = x.shape
    if b > 1 and t > 1 and strides[0] < strides[1]:
        return T.empty((t, b, c), dtype=dtype, device=x.device).transpose(0, 1), c, b * c
    return T.empty((b, t, c), dtype=dtype, device=x.device), t * c, c


def leaky_scan(x, gate=None, *, decay: float | None = None, h0=None, lengths=None, logit: bool = False,
               complement: bool = False, input_scale: float = 1.0, dtype=None, save: bool = False):
    """h[t] = a[t] h[t-1] + input_scale x[t] (times 1 - a[t] with
    `complement`) over x [batch, steps, channels]: returns (h, h_last), and
    with `save` also what leaky_scan_backward needs. The gate ([channels],
    [batch, channels] or [batch, steps, channels]) holds a, or its logits with
    `logit`; `decay` is one a for all. h is of x's type (float32 for spikes)
    or of `dtype`; rows at or behind lengths[b] are zero there."""
    T = _t()
    dev = _device(x, gate, h0, lengths)
    x, xs = _sequences(x, "leaky_scan")
    shape = x.shape
    b, t, c = shape
    gate, gcode, gb, gt = _gate(T, gate, decay, shape)
    code = _code(T, x, "leaky_scan")
    out = dtype or (T.float32 if code == SPIKES else x.dtype)
    y, yb, yt = _like(T, x, xs, out)
    h0 = _state(T, h0, (b, c), "h0")
    h_last = T.empty((b, c), dtype=T.float32, device=x.device)
    saved = T.empty((b, -(-t // LEAKY_BLOCK), c), dtype=T.float32, device=x.device) if save else None
    q = Leaky(b, t, c, code, gcode, T.codes.get(out, -1), logit, complement, decay or 0.0, input_scale, xs[0], xs[1],
              gb, gt, yb, yt)
    at = C.byref(q)
    need = T.lib.snn_b200_leaky_workspace(at)
    ws = T.empty(need, dtype=T.uint8, device=x.device)
    st = T.lib.snn_b200_leaky_scan_async(dev, T.stream(dev), at, x.data_ptr(), _p(gate), _p(h0),
                                         _lengths(T, lengths, b), y.data_ptr(), h_last.data_ptr(), _p(saved),
                                         ws.data_ptr(), need)
    if st:
        _check(st, "snn_b200_leaky_scan_async")
    return (y, h_last, saved) if save else (y, h_last)


def leaky_scan_backward(dy, x, gate=None, saved=None, *, dh_last=None, decay: float | None = None, lengths=None,
                        logit: bool = False, complement: bool = False, input_scale: float = 1.0):
    """The gradients (dx, dgate, dh0) of leaky_scan from those of its outputs:
    dy (h's type) and dh_last (None: zero); `saved` is what leaky_scan(...,
    save=True) returned for the same inputs. dgate is shaped like the gate,
    float32 where the gate is shared over the steps, None without a gate."""
    T = _t()
    dev = _device(x, gate, saved, dy, dh_last, lengths)
    x, xs = _sequences(x, "leaky_scan_backward")
    dy, ys = _sequences(dy, "leaky_scan_backward")
    shape = x.shape
    b, t, c = shape
    if dy.shape != shape:
        _refuse("leaky_scan_backward: dy of x's shape expected")
    gate, gcode, gb, gt = _gate(T, gate, decay, shape)
    if saved is None or saved.shape != (b, -(-t // LEAKY_BLOCK), c) or saved.dtype != T.float32 \
            or not saved.is_contiguous():
        _refuse("leaky_scan_backward: `saved` of leaky_scan(..., save=True) expected")
    code = _code(T, x, "leaky_scan_backward")
    dx, xb, xt = _like(T, x, xs, T.float32 if code == SPIKES else x.dtype)
    dgate, db, dt = None, 0, 0
    if gt:
        dgate, db, dt = _like(T, gate, (gb, gt), gate.dtype)
    elif gate is not None:
        dgate = T.empty((b, c) if gate.dim() > 1 else (c,), dtype=T.float32, device=x.device)
        db = c if gb else 0
    dh_last = _state(T, dh_last, (b, c), "dh_last")
    dh0 = T.empty((b, c), dtype=T.float32, device=x.device)
    q = Leaky(b, t, c, code, gcode, _code(T, dy, "dy"), logit, complement, decay or 0.0, input_scale, xs[0], xs[1], gb,
              gt, 0, 0, ys[0], ys[1], xb, xt, db, dt)
    at = C.byref(q)
    need = T.lib.snn_b200_leaky_workspace(at)
    ws = T.empty(need, dtype=T.uint8, device=x.device)
    st = T.lib.snn_b200_leaky_scan_backward_async(dev, T.stream(dev), at, x.data_ptr(), _p(gate),
                                                  _lengths(T, lengths, b), saved.data_ptr(), dy.data_ptr(),
                                                  _p(dh_last), dx.data_ptr(), _p(dgate), dh0.data_ptr(),
                                                  ws.data_ptr(), need)
    if st:
        _check(st, "snn_b200_leaky_scan_backward_async")
    return dx, dgate, dh0


def leaky_step(x, gate=None, pool=None, *, slots=None, decay: float | None = None, logit: bool = False,
               complement: bool = False, input_scale: float = 1.0, dtype=None):
    """One step of x [batch, channels]: pool[slots[i]] (pool [slot_count,
    channels], float32, updated in place; without `slots` pool[i]) becomes
    a pool[slots[i]] + input_scale x[i] (times 1 - a with `complement`), which
    is returned. The gate is [channels] or [batch, channels]. Rows with a slot
    outside the pool are padding (zero)."""
    T = _t()
    shape = x.shape
    if pool is None or len(shape) != 2 or pool.dim() != 2 or pool.dtype != T.float32:
        _refuse("leaky_step: x [batch, channels] and a float32 pool [slot_count, channels] expected")
    b, c = shape
    dev = _device(x, gate, pool, slots)
    count, channels = pool.shape
    ps = pool.stride()
    if channels != c or (ps[1] != 1 and c > 1):
        _refuse("leaky_step: a pool [slot_count, channels] with neighbouring channels expected")
    xs = x.stride()
    if xs[1] != 1 and c > 1:
        x = x.contiguous()
        xs = x.stride()
    if (gate is None) == (decay is None):
        _refuse("leaky_step: either a gate array or a decay is needed")
    z, gcode, gs = None, F32, 0
    if gate is not None:
        own = gate.shape
        if own != shape and own != shape[1:]:
            _refuse("leaky_step: a gate of shape [channels] or [batch, channels] expected")
        strides = gate.stride()
        if strides[-1] != 1 and c > 1:
            gate = gate.contiguous()
            strides = gate.stride()
        z, gcode, gs = gate.data_ptr(), _code(T, gate, "gate"), strides[0] if len(own) == 2 else 0
    at = None
    if slots is not None:
        if slots.dtype != T.torch.int32 or slots.shape != shape[:1] or not slots.is_contiguous():
            _refuse(f"leaky_step: slots must be {b} contiguous int32")
        at = slots.data_ptr()
    code = _code(T, x, "leaky_step")
    out = dtype or (T.float32 if code == SPIKES else x.dtype)
    y = T.empty(shape, dtype=out, device=x.device)
    st = T.lib.snn_b200_leaky_step_async(dev, T.stream(dev), b, count, c, x.data_ptr(), code, xs[0], z, gcode, gs,
                                         logit, complement, decay or 0.0, input_scale, pool.data_ptr(), ps[0], at,
                                         y.data_ptr(), T.codes.get(out, -1), c)
    if st:
        _check(st, "snn_b200_leaky_step_async")
    return y
