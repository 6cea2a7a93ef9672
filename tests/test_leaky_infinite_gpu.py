"""Infinite states of the leaky recurrence, forward and backward: how a call's
steps are split over the GPU does not show in what becomes of them."""
import numpy as np
import pytest

import snn_b200 as sb
from tests._sequence_ref import LeakyRef, check

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
INF = float("inf")
# Walked whole, by crews of 16 and of 8 warps, in segments; odd and even channels.
SIZES = [(2, 12, 8), (1, 400, 8), (1, 403, 7), (10, 41, 1000), (7, 41, 701), (1, 5000, 8), (1, 5003, 7), (40, 30, 1300),
         (1, 40001, 6)]


def same(got, want, err, what):
    """Finite values within their bound, the others equal."""
    got = got.double().cpu().numpy()
    ok = np.isfinite(want)
    assert np.array_equal(got[~ok], want[~ok], equal_nan=True), what
    check(got[ok], want[ok], np.nan_to_num(err[ok], nan=0.0, posinf=0.0), "f32", what)


@pytest.mark.parametrize("kind", ["step", "channel", "logits"])
@pytest.mark.parametrize("b,t,c", SIZES)
def test_infinite_states_stay_infinite(b, t, c, kind):
    """Gates so small that their products over a part of the steps are zero in 32
    bits, of either sign; one channel has a gate of zero, which makes NaN of an infinity."""
    g = torch.Generator().manual_seed(b + t + c)
    x, dy = torch.randn(b, t, c, generator=g), torch.randn(b, t, c, generator=g)
    h0, dh = torch.randn(b, c, generator=g), torch.randn(b, c, generator=g)
    small = torch.tensor([0.1, -0.1, 1e-7, -1e-7, 0.1, 0.1, 0.9])
    if kind == "channel":
        gate = small[torch.arange(c) % 7].clone()
        gate[4] = 0.0
    else:
        gate = small[torch.arange(c) % 7].expand(b, t, c).clone()
        if kind == "logits":
            gate = torch.log(gate.abs() / (1 - gate.abs()))
            gate[:, t // 2, 4] = -INF
        else:
            gate[:, t // 2, 4] = 0.0
    h0[:, :6] = torch.tensor([INF, INF, -INF, INF, INF, 1.0])
    dh[:, :6] = torch.tensor([INF, -INF, INF, INF, INF, 1.0])
    x[0, 3, 5] = -INF
    logit = kind == "logits"
    with np.errstate(invalid="ignore", over="ignore"):
        ref = LeakyRef(x.numpy(), gate.numpy(), None, h0.numpy(), None, logit)
        ref.backward(dy.numpy(), dh.numpy())
    y, h_last, saved = sb.leaky_scan(x.cuda(), gate.cuda(), h0=h0.cuda(), logit=logit, save=True)
    same(y, ref.y, ref.y_err, "y")
    same(h_last, ref.h_last, ref.h_last_err, "h_last")
    dx, _, dh0 = sb.leaky_scan_backward(dy.cuda(), x.cuda(), gate.cuda(), saved, dh_last=dh.cuda(), logit=logit)
    same(dx, ref.dx, ref.dx_err, "dx")
    same(dh0, ref.dh0, ref.dh0_err, "dh0")
    assert np.isinf(ref.y[:, -1, :4]).all() and np.isinf(ref.dh0[:, :4]).all()
