"""What the sequence operators refuse, before any device is touched, and
their size helpers. Pointers are made-up numbers: a refused call reads none."""
import ctypes as C

import numpy as np
import pytest

import snn_b200 as sb
from tests._sequence_ref import LeakyRef, mx4_values, scale_offsets

BAD, OVER, UNSUP, OK = (sb.SNN_ERR_INVALID_ARGUMENT, sb.SNN_ERR_OVERFLOW, sb.SNN_ERR_UNSUPPORTED, sb.SNN_OK)
P = 1 << 20  # an aligned address
BIG = 1 << 31
F32, F16, BF16, SPIKES = 0, 1, 2, 3


def test_sizes():
    assert sb.mx4_sizes(1000, 784) == (1000 * 25 * 16, 8 * 7 * 512)
    assert sb.mx4_sizes(1, 1) == (16, 512)
    assert sb.mx4_sizes(0, 5) == (0, 0) and sb.mx4_sizes(5, 0) == (0, 0)
    for rows, cols in ((1, 1), (129, 33), (300, 4100)):
        assert scale_offsets(rows, cols).max() < sb.mx4_sizes(rows, cols)[1]
    with pytest.raises(sb.SnnError) as e:
        sb.mx4_sizes(BIG, 1)
    assert e.value.status == OVER
    L = sb.lib()
    assert L.snn_b200_mx4_sizes(1, 1, None, None) == BAD
    assert L.snn_b200_mx4_linear_workspace(P, F32, 17, 784, 784, 1) == sum(sb.mx4_sizes(17, 784))
    assert L.snn_b200_mx4_linear_workspace(P, F32, 16, 784, 784, 1) == 0  # packed by the product's kernel
    assert L.snn_b200_mx4_linear_workspace(P + 4, F32, 16, 784, 784, 1) == sum(sb.mx4_sizes(16, 784))
    assert L.snn_b200_mx4_linear_workspace(P, F32, 16, 783, 783, 1) == sum(sb.mx4_sizes(16, 783))
    assert L.snn_b200_leaky_saved_floats(3, 33, 5) == 3 * 5 * 5
    assert L.snn_b200_leaky_workspace(None, 0) == L.snn_b200_leaky_workspace(None, 1) == 0


QUANT = dict(device=0, stream=None, src=P, dtype=F32, rows=4, cols=64, rs=64, cs=1, codes=P, scales=P)


@pytest.mark.parametrize("change,status", [
    (dict(device=-1), BAD), (dict(src=None), BAD), (dict(src=P + 2), BAD), (dict(dtype=4), BAD), (dict(dtype=-1), BAD),
    (dict(rows=BIG), OVER), (dict(cols=BIG), OVER), (dict(rs=-64), BAD), (dict(cs=-1), BAD), (dict(rs=1 << 60), BAD),
    (dict(codes=None), BAD), (dict(codes=P + 8), BAD), (dict(scales=P + 4), BAD), (dict(scales=None), BAD),
    (dict(rows=0), OK), (dict(cols=0, codes=None, scales=None), OK)])
def test_quantize_refusals(change, status):
    assert sb.lib().snn_b200_mx4_quantize_async(*{**QUANT, **change}.values()) == status


DEQ = dict(device=0, stream=None, codes=P, scales=P, rows=4, cols=64, dst=P, dtype=F32, rs=64)


@pytest.mark.parametrize("change,status", [
    (dict(device=-1), BAD), (dict(dst=None), BAD), (dict(dst=P + 2), BAD), (dict(dtype=SPIKES), BAD),
    (dict(rs=63), BAD), (dict(rs=-64), BAD), (dict(codes=P + 1), BAD), (dict(scales=None), BAD),
    (dict(rows=BIG), OVER), (dict(rows=0), OK)])
def test_dequantize_refusals(change, status):
    assert sb.lib().snn_b200_mx4_dequantize_async(*{**DEQ, **change}.values()) == status


MATMUL = dict(device=0, stream=None, xc=P, xs=P, m=4, wc=P, ws=P, n=8, k=64, bias=None, out=P, dtype=F32, rs=8)


@pytest.mark.parametrize("change,status", [
    (dict(device=-1), BAD), (dict(xc=None), BAD), (dict(xs=P + 8), BAD), (dict(wc=P + 8), BAD), (dict(ws=None), BAD),
    (dict(bias=P + 2), BAD), (dict(out=None), BAD), (dict(out=P + 1), BAD), (dict(dtype=SPIKES), BAD),
    (dict(rs=7), BAD), (dict(m=BIG), OVER), (dict(n=BIG), OVER), (dict(k=BIG), OVER), (dict(m=0), OK), (dict(n=0), OK)])
def test_matmul_refusals(change, status):
    assert sb.lib().snn_b200_mx4_matmul_async(*{**MATMUL, **change}.values()) == status


LINEAR = dict(device=0, stream=None, x=P, x_dtype=BF16, m=20, k=64, xrs=64, xcs=1, wc=P, ws=P, n=8, bias=None, out=P,
              dtype=F32, rs=8, work=P, work_bytes=1 << 20)


@pytest.mark.parametrize("change,status", [
    (dict(device=-1), BAD), (dict(x=None), BAD), (dict(x=P + 1), BAD), (dict(x_dtype=9), BAD), (dict(xrs=-1), BAD),
    (dict(wc=None), BAD), (dict(out=None), BAD), (dict(rs=7), BAD), (dict(work=None), BAD), (dict(work=P + 8), BAD),
    (dict(work_bytes=sum(sb.mx4_sizes(20, 64)) - 1), BAD), (dict(m=BIG), OVER), (dict(k=BIG), OVER), (dict(m=0), OK)])
def test_linear_refusals(change, status):
    assert sb.lib().snn_b200_mx4_linear_async(*{**LINEAR, **change}.values()) == status


SHAPE = dict(batch=2, steps=400, channels=8, x_dtype=BF16, gate_dtype=BF16, y_dtype=BF16, logit=0, complement=0,
             decay=0.5, input_scale=1.0, x_batch_stride=3200, x_step_stride=8, gate_batch_stride=3200,
             gate_step_stride=8, y_batch_stride=3200, y_step_stride=8, dy_batch_stride=3200, dy_step_stride=8,
             dx_batch_stride=3200, dx_step_stride=8, dgate_batch_stride=3200, dgate_step_stride=8)
SCAN = dict(x=P, gate=P, h0=P, lengths=P, y=P, h_last=P, saved=P, work=P, work_bytes=1 << 30)
BACK = dict(x=P, gate=P, lengths=P, saved=P, dy=P, dh_last=P, dx=P, dgate=P, dh0=P, work=P, work_bytes=1 << 30)


def call(name, shape, args, change, device=0):
    s = {k: change.get(k, v) for k, v in shape.items()}
    q = sb.Leaky(*s.values())
    a = {k: change.get(k, v) for k, v in args.items()}
    return getattr(sb.lib(), name)(device, None, C.byref(q), *a.values())


COMMON = [
    (dict(x=None), BAD), (dict(x=P + 1), BAD), (dict(gate=P + 1), BAD), (dict(lengths=P + 2), BAD),
    (dict(batch=BIG), OVER), (dict(steps=BIG), OVER), (dict(channels=BIG), OVER), (dict(x_dtype=7), BAD),
    (dict(gate_dtype=SPIKES), BAD), (dict(y_dtype=SPIKES), BAD), (dict(x_batch_stride=-8), BAD),
    (dict(gate_step_stride=-8), BAD), (dict(x_dtype=F32), UNSUP), (dict(x_dtype=F16), UNSUP),
    (dict(y_dtype=F16), UNSUP), (dict(gate_step_stride=0), UNSUP), (dict(x_dtype=SPIKES, y_dtype=F32), UNSUP),
    (dict(work=None), BAD), (dict(work=P + 8), BAD), (dict(work_bytes=0), BAD), (dict(channels=0), OK),
    (dict(batch=0), OK)]


@pytest.mark.parametrize("change,status", COMMON + [
    (dict(y=None), BAD), (dict(y=P + 1), BAD), (dict(h0=P + 2), BAD), (dict(h_last=P + 1), BAD), (dict(saved=P + 2), BAD),
    (dict(y_step_stride=7), BAD), (dict(y_batch_stride=3199), BAD), (dict(y_batch_stride=8, y_step_stride=8), BAD),
    (dict(y_step_stride=0), BAD)])
def test_scan_refusals(change, status):
    assert call("snn_b200_leaky_scan_async", SHAPE, SCAN, change) == status


@pytest.mark.parametrize("change,status", COMMON + [
    (dict(saved=None), BAD), (dict(saved=P + 2), BAD), (dict(dy=None), BAD), (dict(dy=P + 1), BAD),
    (dict(dh_last=P + 2), BAD), (dict(dh0=P + 1), BAD), (dict(dx=P + 1), BAD), (dict(dgate=P + 1), BAD),
    (dict(dx_step_stride=7), BAD), (dict(dgate_batch_stride=3199), BAD), (dict(gate=None), BAD),
    (dict(gate_batch_stride=0), UNSUP), (dict(gate_dtype=F32, gate_step_stride=0, dgate_batch_stride=7), BAD)])
def test_backward_refusals(change, status):
    assert call("snn_b200_leaky_scan_backward_async", SHAPE, BACK, change) == status


def test_scan_refuses_no_shape_and_no_device():
    L = sb.lib()
    assert L.snn_b200_leaky_scan_async(0, None, None, *SCAN.values()) == BAD
    assert L.snn_b200_leaky_scan_backward_async(0, None, None, *BACK.values()) == BAD
    assert call("snn_b200_leaky_scan_async", SHAPE, SCAN, {}, device=-1) == BAD
    assert call("snn_b200_leaky_scan_backward_async", SHAPE, BACK, {}, device=-1) == BAD


STEP = dict(device=0, stream=None, batch=4, slot_count=6, channels=8, x=P, x_dtype=BF16, xs=8, gate=P, gate_dtype=BF16,
            gs=8, logit=0, complement=0, decay=0.5, scale=1.0, pool=P, ps=8, slots=P, y=P, y_dtype=BF16, ys=8)


@pytest.mark.parametrize("change,status", [
    (dict(device=-1), BAD), (dict(x=None), BAD), (dict(y=None), BAD), (dict(pool=None), BAD), (dict(pool=P + 2), BAD),
    (dict(slots=P + 1), BAD), (dict(slots=None, batch=7), BAD), (dict(gate=P + 1), BAD), (dict(xs=-8), BAD),
    (dict(ys=7), BAD), (dict(ps=7), BAD), (dict(ps=-8), BAD), (dict(x_dtype=F32), UNSUP), (dict(gs=0), UNSUP),
    (dict(x_dtype=5), BAD), (dict(batch=BIG), OVER), (dict(channels=BIG), OVER), (dict(slot_count=BIG), OVER),
    (dict(batch=0), OK), (dict(channels=0), OK)])
def test_step_refusals(change, status):
    assert sb.lib().snn_b200_leaky_step_async(*{**STEP, **change}.values()) == status


def test_wrappers_refuse_host_tensors():
    torch = pytest.importorskip("torch")
    x = torch.ones(2, 64)
    for f in (lambda: sb.mx4_quantize(x), lambda: sb.leaky_scan(x[None], decay=0.5),
              lambda: sb.leaky_step(x, None, torch.zeros(2, 64), decay=0.5)):
        with pytest.raises(sb.SnnError) as e:
            f()
        assert e.value.status == BAD


def test_valid_calls_need_a_device(gpu_count):
    if gpu_count:
        pytest.skip("a device is present")
    L = sb.lib()
    assert L.snn_b200_mx4_quantize_async(*QUANT.values()) == sb.SNN_ERR_CUDA
    assert L.snn_b200_mx4_dequantize_async(*DEQ.values()) == sb.SNN_ERR_CUDA
    assert L.snn_b200_mx4_matmul_async(*MATMUL.values()) == sb.SNN_ERR_CUDA
    assert L.snn_b200_mx4_linear_async(*LINEAR.values()) == sb.SNN_ERR_CUDA
    assert call("snn_b200_leaky_scan_async", SHAPE, SCAN, {}) == sb.SNN_ERR_CUDA
    assert call("snn_b200_leaky_scan_backward_async", SHAPE, BACK, {}) == sb.SNN_ERR_CUDA
    assert L.snn_b200_leaky_step_async(*STEP.values()) == sb.SNN_ERR_CUDA
    assert sb.last_error()


def test_reference_packing_keeps_representable_values():
    grid = np.array([[0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.5, -6] + [0] * 22], np.float64)
    for e in (-120, -3, 0, 90):
        assert np.array_equal(mx4_values(grid * 2.0 ** e), grid * 2.0 ** e)


def test_reference_gradient_against_differences():
    rng = np.random.default_rng(0)
    x, z, h0 = rng.standard_normal((2, 9, 3)), rng.standard_normal((2, 3)), rng.standard_normal((2, 3))
    dy, dh = rng.standard_normal((2, 9, 3)), rng.standard_normal((2, 3))
    lengths = np.array([9, 4])

    def loss(x, z, h0):
        r = LeakyRef(x, z, None, h0, lengths, True, True, 0.7)
        return (r.y * dy).sum() + (r.h_last * dh).sum()

    ref = LeakyRef(x, z, None, h0, lengths, True, True, 0.7)
    ref.backward(dy, dh)
    eps = 1e-5  # third-order term 1e-10, rounding 1e-11
    for k, got in enumerate((ref.dx, ref.dgate, ref.dh0)):
        for at in np.ndindex(got.shape):
            args = [x.copy(), z.copy(), h0.copy()]
            args[k][at] += eps
            hi = loss(*args)
            args[k][at] -= 2 * eps
            assert abs((hi - loss(*args)) / (2 * eps) - got[at]) < 1e-8
