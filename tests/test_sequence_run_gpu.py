"""The sequence operators together, as a program uses them: the raster of a
simulated layer goes through packed weights, a leaky readout integrates the
currents, and its gradient comes back."""
import numpy as np
import pytest

import snn_b200 as sb
from oracle.oracle import Oracle, baseline_lif
from tests._sequence_ref import LeakyRef, check, mx4_values

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_raster_through_packed_layer_into_leaky_readout():
    n, steps, out = 512, 40, 10
    net = Oracle("port").random_pool(n, 32, 0.0, 0.6, 5, lif=baseline_lif())
    raster = np.zeros((steps, n), np.uint8)
    rng = np.random.default_rng(0)
    with sb.CudaContext.create(net, None, sb.default_options(device=0)) as ctx:
        for t in range(steps):
            idx = np.sort(rng.choice(n, 100, replace=False))
            ctx.inject_current(idx, np.full(100, 20.0, np.float32))
            ctx.step(out=raster[t])
    assert raster.sum() > 100
    weights = (rng.standard_normal((n, out)) / n ** 0.5).astype(np.float32)  # a row per presynaptic neuron
    leak = np.linspace(0.5, 3.0, out).astype(np.float32)  # logits
    spikes = torch.from_numpy(raster).cuda()
    gate = torch.from_numpy(leak).cuda()
    packed = sb.mx4_quantize(torch.from_numpy(weights).cuda().t())
    current = sb.mx4_linear(spikes, packed)
    kept = mx4_values(weights.T)
    want = raster.astype(np.float64) @ kept.T
    check(current.cpu().numpy(), want, 2.0 ** -20 * (raster.astype(np.float64) @ np.abs(kept).T), "f32", "current")

    # Training: the whole sequence and its gradient.
    x = current[None]
    y, last, saved = sb.leaky_scan(x, gate, logit=True, complement=True, save=True)
    ref = LeakyRef(x.double().cpu().numpy(), leak, logit=True, complement=True)
    check(y.cpu().numpy(), ref.y, ref.y_err, "f32", "readout")
    dy = torch.zeros_like(y)
    dy[0, -1] = 1.0
    dx, dgate, _ = sb.leaky_scan_backward(dy, x, gate, saved, logit=True, complement=True)
    ref.backward(dy.double().cpu().numpy())
    check(dx.cpu().numpy(), ref.dx, ref.dx_err, "f32", "dx")
    check(dgate.cpu().numpy(), ref.dgate, ref.dgate_err, "f32", "dgate")

    # Serving: step by step, the same readout.
    pool = torch.zeros(1, out, device="cuda")
    for t in range(steps):
        now = sb.mx4_linear(spikes[t:t + 1], packed)
        step = sb.leaky_step(now, gate, pool, logit=True, complement=True)
    room = 2.0 ** -20 * (raster.astype(np.float64) @ np.abs(kept).T).max() / (1 - 1 / (1 + np.exp(-leak[-1])))
    check(step.cpu().numpy(), ref.y[:, -1], ref.y_err[:, -1] + room, "f32", "last step")
    assert torch.equal(step, pool)
