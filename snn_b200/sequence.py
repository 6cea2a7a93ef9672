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

_DTYPES: dict = {}


def _torch():
    import torch
    if not _DTYPES:
        _DTYPES.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16, torch.uint8: SPIKES,
                        torch.bool: SPIKES})
    return torch


def _refuse(what: str):
    raise SnnError(SNN_ERR_INVALID_ARGUMENT, what)


def _code(t, what: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        _refuse(f"{what}: element type {t.dtype} is not one of float32, float16, bfloat16, uint8, bool")
    return code


def _same_device(first, *others):
    if not first.is_cuda:
        _refuse("tensors must be on a CUDA device")
    for t in others:
        if t is not None and t.device != first.device:
            _refuse("tensors must be on one device")
    return first.device


def _state(t, shape, what: str):
    """A float32 tensor of `shape`, contiguous."""
    torch = _torch()
    if t is None:
        return None
    if t.dtype != torch.float32 or tuple(t.shape) != tuple(shape):
        _refuse(f"{what}: float32 of shape {tuple(shape)} expected")
    return t.contiguous()


def _p(t):
    return None if t is None else t.data_ptr()


def _stream(torch, device):
    return torch.cuda.current_stream(device).cuda_stream


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
    torch = _torch()
    dev = _same_device(x)
    if x.dim() != 2:
        _refuse("mx4_quantize: a 2-D tensor expected")
    rows, cols = x.shape
    code = _code(x, "mx4_quantize")
    if out is None:
        nc, ns = mx4_sizes(rows, cols)
        out = Mx4(torch.empty(nc, dtype=torch.uint8, device=dev), torch.empty(ns, dtype=torch.uint8, device=dev),
                  rows, cols)
    elif (out.rows, out.cols) != (rows, cols) or out.codes.device != dev:
        _refuse("mx4_quantize: `out` is of another shape or device")
    st = lib().snn_b200_mx4_quantize_async(dev.index, _stream(torch, dev), x.data_ptr(), code, rows, cols,
                                           x.stride(0), x.stride(1), out.codes.data_ptr(), out.scales.data_ptr())
    _check(st, "snn_b200_mx4_quantize_async")
    return out


def mx4_dequantize(q: Mx4, dtype=None):
    """The values that a packed matrix stands for (float32 by default)."""
    torch = _torch()
    dev = _same_device(q.codes, q.scales)
    y = torch.empty(q.rows, q.cols, dtype=dtype or torch.float32, device=dev)
    st = lib().snn_b200_mx4_dequantize_async(dev.index, _stream(torch, dev), q.codes.data_ptr(), q.scales.data_ptr(),
                                             q.rows, q.cols, y.data_ptr(), _code(y, "mx4_dequantize"), q.cols)
    _check(st, "snn_b200_mx4_dequantize_async")
    return y


def _bias(bias, n: int):
    torch = _torch()
    if bias is not None and (bias.dtype != torch.float32 or tuple(bias.shape) != (n,) or not bias.is_contiguous()):
        _refuse(f"bias: {n} contiguous float32 expected")
    return bias


def mx4_matmul(x: Mx4, w: Mx4, bias=None, dtype=None):
    """x [m, k] times the transpose of w [n, k], plus bias [n]."""
    torch = _torch()
    dev = _same_device(x.codes, x.scales, w.codes, w.scales, bias)
    if x.cols != w.cols:
        _refuse(f"mx4_matmul: {x.cols} columns against {w.cols}")
    y = torch.empty(x.rows, w.rows, dtype=dtype or torch.float32, device=dev)
    st = lib().snn_b200_mx4_matmul_async(dev.index, _stream(torch, dev), x.codes.data_ptr(), x.scales.data_ptr(),
                                         x.rows, w.codes.data_ptr(), w.scales.data_ptr(), w.rows, w.cols,
                                         _p(_bias(bias, w.rows)), y.data_ptr(), _code(y, "mx4_matmul"), w.rows)
    _check(st, "snn_b200_mx4_matmul_async")
    return y


def mx4_linear(x, w: Mx4, bias=None, dtype=None):
    """x [..., k] packed on the way, times the transpose of w [n, k], plus
    bias [n]: the currents that a raster (or activations) sends through a
    packed layer. The result's type is x's, float32 for spikes, or `dtype`."""
    torch = _torch()
    dev = _same_device(x, w.codes, w.scales, bias)
    if x.dim() < 1 or x.shape[-1] != w.cols:
        _refuse(f"mx4_linear: rows of {w.cols} elements expected, not {tuple(x.shape)}")
    code = _code(x, "mx4_linear")
    m = math.prod(x.shape[:-1])
    flat = x if x.dim() == 2 else x.reshape(m, w.cols)
    y = torch.empty(m, w.rows, dtype=dtype or (torch.float32 if code == SPIKES else x.dtype), device=dev)
    need = lib().snn_b200_mx4_linear_workspace(m, w.cols)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    st = lib().snn_b200_mx4_linear_async(dev.index, _stream(torch, dev), flat.data_ptr(), code, m, w.cols,
                                         flat.stride(0), flat.stride(1), w.codes.data_ptr(), w.scales.data_ptr(),
                                         w.rows, _p(_bias(bias, w.rows)), y.data_ptr(), _code(y, "mx4_linear"),
                                         w.rows, ws.data_ptr(), need)
    _check(st, "snn_b200_mx4_linear_async")
    return y if x.dim() == 2 else y.view(*x.shape[:-1], w.rows)


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
    if t.dim() != 3:
        _refuse(f"{what}: [batch, steps, channels] expected")
    if t.stride(2) != 1 and t.shape[2] > 1:
        t = t.contiguous()
    return t


def _gate(gate, decay, shape):
    """The gate array with its strides over the sequences and the steps: [C], [B, C] or [B, T, C]."""
    b, t, c = shape
    if (gate is None) == (decay is None):
        _refuse("leaky: either a gate array or a decay is needed")
    if gate is None:
        return None, 0, 0
    if gate.dim() not in (1, 2, 3) or tuple(gate.shape) != ((c,), (b, c), (b, t, c))[gate.dim() - 1]:
        _refuse(f"leaky: a gate of shape [channels], [batch, channels] or [batch, steps, channels] expected, not "
                f"{tuple(gate.shape)}")
    if c > 1 and gate.stride(-1) != 1:
        gate = gate.contiguous()
    return gate, (gate.stride(0) if gate.dim() > 1 else 0), (gate.stride(1) if gate.dim() == 3 else 0)


def _lengths(lengths, batch: int):
    torch = _torch()
    if lengths is not None and (lengths.dtype not in (torch.int32, torch.uint32) or tuple(lengths.shape) != (batch,)
                                or not lengths.is_contiguous()):
        _refuse(f"lengths: {batch} contiguous int32 expected")
    return lengths


def _like(torch, x, dtype):
    """An empty [batch, steps, channels] tensor whose steps come first in memory where x's do."""
    b, t, c = x.shape
    if b > 1 and t > 1 and x.stride(0) < x.stride(1):
        return torch.empty(t, b, c, dtype=dtype, device=x.device).transpose(0, 1)
    return torch.empty(b, t, c, dtype=dtype, device=x.device)


def leaky_scan(x, gate=None, *, decay: float | None = None, h0=None, lengths=None, logit: bool = False,
               complement: bool = False, input_scale: float = 1.0, dtype=None, save: bool = False):
    """h[t] = a[t] h[t-1] + input_scale x[t] (times 1 - a[t] with
    `complement`) over x [batch, steps, channels]: returns (h, h_last), and
    with `save` also what leaky_scan_backward needs. The gate ([channels],
    [batch, channels] or [batch, steps, channels]) holds a, or its logits with
    `logit`; `decay` is one a for all. h is of x's type (float32 for spikes)
    or of `dtype`; rows at or behind lengths[b] are zero there."""
    torch = _torch()
    dev = _same_device(x, gate, h0, lengths)
    x = _sequences(x, "leaky_scan")
    b, t, c = x.shape
    gate, gb, gt = _gate(gate, decay, (b, t, c))
    code = _code(x, "leaky_scan")
    y = _like(torch, x, dtype or (torch.float32 if code == SPIKES else x.dtype))
    h0 = _state(h0, (b, c), "h0")
    h_last = torch.empty(b, c, dtype=torch.float32, device=dev)
    saved = torch.empty(b, -(-t // LEAKY_BLOCK), c, dtype=torch.float32, device=dev) if save else None
    q = Leaky(b, t, c, code, F32 if gate is None else _code(gate, "gate"), _code(y, "leaky_scan"), int(logit),
              int(complement), decay or 0.0, input_scale, x.stride(0), x.stride(1), gb, gt, y.stride(0), y.stride(1))
    L = lib()
    need = L.snn_b200_leaky_workspace(C.byref(q))
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    st = L.snn_b200_leaky_scan_async(dev.index, _stream(torch, dev), C.byref(q), x.data_ptr(), _p(gate), _p(h0),
                                     _p(_lengths(lengths, b)), y.data_ptr(), h_last.data_ptr(), _p(saved),
                                     ws.data_ptr(), need)
    _check(st, "snn_b200_leaky_scan_async")
    return (y, h_last, saved) if save else (y, h_last)


def leaky_scan_backward(dy, x, gate=None, saved=None, *, dh_last=None, decay: float | None = None, lengths=None,
                        logit: bool = False, complement: bool = False, input_scale: float = 1.0):
    """The gradients (dx, dgate, dh0) of leaky_scan from those of its outputs:
    dy (h's type) and dh_last (None: zero); `saved` is what leaky_scan(...,
    save=True) returned for the same inputs. dgate is shaped like the gate,
    float32 where the gate is shared over the steps, None without a gate."""
    torch = _torch()
    dev = _same_device(x, gate, saved, dy, dh_last, lengths)
    x, dy = _sequences(x, "leaky_scan_backward"), _sequences(dy, "leaky_scan_backward")
    b, t, c = x.shape
    if tuple(dy.shape) != (b, t, c):
        _refuse("leaky_scan_backward: dy of x's shape expected")
    gate, gb, gt = _gate(gate, decay, (b, t, c))
    if saved is None or tuple(saved.shape) != (b, -(-t // LEAKY_BLOCK), c) or saved.dtype != torch.float32 \
            or not saved.is_contiguous():
        _refuse("leaky_scan_backward: `saved` of leaky_scan(..., save=True) expected")
    code = _code(x, "leaky_scan_backward")
    dx = _like(torch, x, torch.float32 if code == SPIKES else x.dtype)
    dgate, db, dt = None, 0, 0
    if gate is not None:
        if gt:
            dgate = _like(torch, gate, gate.dtype)
            db, dt = dgate.stride(0), dgate.stride(1)
        else:
            dgate = torch.empty((b, c) if gb else (c,), dtype=torch.float32, device=dev)
            db = c if gb else 0
    dh_last = _state(dh_last, (b, c), "dh_last")
    dh0 = torch.empty(b, c, dtype=torch.float32, device=dev)
    q = Leaky(b, t, c, code, F32 if gate is None else _code(gate, "gate"), _code(dy, "dy"), int(logit),
              int(complement), decay or 0.0, input_scale, x.stride(0), x.stride(1), gb, gt, 0, 0, dy.stride(0),
              dy.stride(1), dx.stride(0), dx.stride(1), db, dt)
    L = lib()
    need = L.snn_b200_leaky_workspace(C.byref(q))
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    st = L.snn_b200_leaky_scan_backward_async(dev.index, _stream(torch, dev), C.byref(q), x.data_ptr(), _p(gate),
                                              _p(_lengths(lengths, b)), saved.data_ptr(), dy.data_ptr(), _p(dh_last),
                                              dx.data_ptr(), _p(dgate), dh0.data_ptr(), ws.data_ptr(), need)
    _check(st, "snn_b200_leaky_scan_backward_async")
    return dx, dgate, dh0


def leaky_step(x, gate=None, pool=None, *, slots=None, decay: float | None = None, logit: bool = False,
               complement: bool = False, input_scale: float = 1.0, dtype=None):
    """One step of x [batch, channels]: pool[slots[i]] (pool [slot_count,
    channels], float32, updated in place; without `slots` pool[i]) becomes
    a pool[slots[i]] + input_scale x[i] (times 1 - a with `complement`), which
    is returned. Rows with a slot outside the pool are padding (zero)."""
    torch = _torch()
    if pool is None or x.dim() != 2 or pool.dim() != 2 or pool.dtype != torch.float32 \
            or pool.shape[1] != x.shape[1] or (pool.stride(1) != 1 and pool.shape[1] > 1):
        _refuse("leaky_step: x [batch, channels] and a float32 pool [slot_count, channels] expected")
    dev = _same_device(x, gate, pool, slots)
    b, c = x.shape
    if c > 1 and x.stride(1) != 1:
        x = x.contiguous()
    if (gate is None) == (decay is None):
        _refuse("leaky_step: either a gate array or a decay is needed")
    if gate is not None:
        if tuple(gate.shape) not in ((c,), (b, c)) or gate.dim() not in (1, 2):
            _refuse("leaky_step: a gate of shape [channels] or [batch, channels] expected")
        if c > 1 and gate.stride(-1) != 1:
            gate = gate.contiguous()
    if slots is not None and (slots.dtype != torch.int32 or tuple(slots.shape) != (b,) or not slots.is_contiguous()):
        _refuse(f"leaky_step: slots must be {b} contiguous int32")
    code = _code(x, "leaky_step")
    y = torch.empty(b, c, dtype=dtype or (torch.float32 if code == SPIKES else x.dtype), device=dev)
    st = lib().snn_b200_leaky_step_async(
        dev.index, _stream(torch, dev), b, pool.shape[0], c, x.data_ptr(), code, x.stride(0), _p(gate),
        F32 if gate is None else _code(gate, "gate"), gate.stride(0) if gate is not None and gate.dim() == 2 else 0,
        int(logit), int(complement), decay or 0.0, input_scale, pool.data_ptr(), pool.stride(0), _p(slots),
        y.data_ptr(), _code(y, "leaky_step"), c)
    _check(st, "snn_b200_leaky_step_async")
    return y
