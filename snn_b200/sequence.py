"""The sequence operators over CUDA tensors (Part 4 of include/snn_b200.h).

Thin mirrors of the C entry points for callers whose arrays are torch tensors:
outputs and workspaces come from torch's allocator, the work goes to the
tensors' device and to its current stream, and a refused call raises SnnError.
A tensor of uint8 or bool is a spike raster (non-zero = one spike).

    w = mx4_quantize(weights)                  # [post, pre], packed once
    current = mx4_linear(raster, w)            # [rows, pre] -> [rows, post]
    y, h_last = leaky_scan(current, decays)    # [batch, steps, channels]

None of them has an autograd formula. A result of tensors that require a
gradient carries that on, and going back through it raises NotImplementedError:
gradients come from leaky_scan_backward (in a torch.autograd.Function, say).
leaky_scan_backward's own results are plain, unless dy or dh_last require a
gradient. What is updated in place (a pool, `out`) counts as a new version.

The checks and the calls are compiled (csrc/torch/sequence_ops.cpp, built to
_lib/sequence_ops.so); torch is imported when an operator is first called.
"""
from __future__ import annotations

import ctypes as C
import os

from . import HERE, SNN_ERR_CUDA, SnnError, _check, last_error, lib

OPS_PATH = os.path.join(HERE, "_lib", "sequence_ops.so")

_OPS = None


def _raise(status: int, what: str):
    detail = last_error() if status == SNN_ERR_CUDA else ""
    raise SnnError(status, f"{what} [{detail}]" if detail else what)


def _ops():
    """The compiled operators; raises if they have not been built."""
    global _OPS
    if _OPS is None:
        import importlib.machinery
        import importlib.util

        import torch  # noqa: F401  (its libraries are loaded before ours)
        lib()
        if not os.path.exists(OPS_PATH):
            raise RuntimeError(f"{OPS_PATH} is missing: build it with `python -m snn_b200.build`")
        loader = importlib.machinery.ExtensionFileLoader("sequence_ops", OPS_PATH)
        ops = importlib.util.module_from_spec(importlib.util.spec_from_loader("sequence_ops", loader))
        loader.exec_module(ops)
        ops.setup(_raise)
        _OPS = ops
    return _OPS


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
    ops = _OPS or _ops()
    if out is None:
        codes, scales = ops.quantize(x, None, None)
        return Mx4(codes, scales, *x.shape)
    if (out.rows, out.cols) != tuple(x.shape):
        _raise(-1, "mx4_quantize: `out` is of another shape")
    ops.quantize(x, out.codes, out.scales)
    return out


def mx4_dequantize(q: Mx4, dtype=None):
    """The values that a packed matrix stands for (float32 by default)."""
    return (_OPS or _ops()).dequantize(q.codes, q.scales, q.rows, q.cols, dtype)


def mx4_matmul(x: Mx4, w: Mx4, bias=None, dtype=None):
    """x [m, k] times the transpose of w [n, k], plus bias [n] (float32);
    float32 by default."""
    return (_OPS or _ops()).matmul(x.codes, x.scales, x.rows, x.cols, w.codes, w.scales, w.rows, w.cols, bias, dtype)


def mx4_linear(x, w: Mx4, bias=None, dtype=None):
    """x [..., k] packed on the way, times the transpose of w [n, k], plus
    bias [n]: the currents that a raster (or activations) sends through a
    packed layer. The result's type is x's, float32 for spikes, or `dtype`."""
    return (_OPS or _ops()).linear(x, w.codes, w.scales, w.rows, w.cols, bias, dtype)


# ---------------------------------------------------------------------------
# Leaky recurrence
# ---------------------------------------------------------------------------
def leaky_scan(x, gate=None, *, decay: float | None = None, h0=None, lengths=None, logit: bool = False,
               complement: bool = False, input_scale: float = 1.0, dtype=None, save: bool = False):
    """h[t] = a[t] h[t-1] + input_scale x[t] (times 1 - a[t] with
    `complement`) over x [batch, steps, channels]: returns (h, h_last), and
    with `save` also what leaky_scan_backward needs. The gate ([channels] or
    [batch, channels] in float32, or [batch, steps, channels], which may be of
    x's 16-bit type too) holds a, or its logits with `logit`; `decay` is one a
    for all. h is of x's type (float32 for spikes)
    or of `dtype`; rows at or behind lengths[b] are zero there."""
    return (_OPS or _ops()).scan(x, gate, decay, lengths, logit, complement, input_scale, h0, dtype, save)


def leaky_scan_backward(dy, x, gate=None, saved=None, *, dh_last=None, decay: float | None = None, lengths=None,
                        logit: bool = False, complement: bool = False, input_scale: float = 1.0):
    """The gradients (dx, dgate, dh0) of leaky_scan from those of its outputs:
    dy (h's type) and dh_last (None: zero); `saved` is what leaky_scan(...,
    save=True) returned for the same inputs. dgate is shaped like the gate (an
    expanded gate's has an element for each of its own), float32 for a gate of
    [channels] or [batch, channels], None without a gate."""
    return (_OPS or _ops()).scan_backward(x, gate, decay, lengths, logit, complement, input_scale, dy, saved, dh_last)


def leaky_step(x, gate=None, pool=None, *, slots=None, decay: float | None = None, logit: bool = False,
               complement: bool = False, input_scale: float = 1.0, dtype=None):
    """One step of x [batch, channels]: pool[slots[i]] (pool [slot_count,
    channels], float32, updated in place; without `slots` pool[i]) becomes
    a pool[slots[i]] + input_scale x[i] (times 1 - a with `complement`), which
    is returned. The gate is [channels] in float32, or [batch, channels], which
    may be of x's 16-bit type too. Rows with a slot outside the pool are padding
    (zero)."""
    return (_OPS or _ops()).step(x, gate, pool, slots, decay, logit, complement, input_scale, dtype)
