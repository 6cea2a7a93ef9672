"""How near the leaky recurrence comes to its definition in 64 bits, with limits
below what rougher arithmetic would give."""
import numpy as np
import pytest

import snn_b200 as sb

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
def test_gates_of_large_16_bit_logits(kind):
    """Every logit of the type up to 87, alone: with complement and no state y is 1 - a, without it and with
    no input a. The product with log2(e) is off by half a unit and by the constant's share of 2^-26.2, the
    hardware exponential by 2^-22 at most; the sum, quotient and products behind it by less than 2^-22 together."""
    bits = torch.arange(1, 0x7c00 if kind == torch.float16 else 0x7f80, dtype=torch.int32).to(torch.int16)
    z = bits.view(kind)
    z = z[(z >= 2.0 ** -14) & (z <= 87)]
    z = torch.cat([z, -z])
    c = z.numel()
    z64 = z.double().numpy()
    m = np.abs(z64) * np.log2(np.e)
    half = np.spacing(m.astype(np.float32)).astype(np.float64) / 2
    off = np.log(2) * (half + m * 2.0 ** -26.2) + 2.0 ** -21
    assert off[np.abs(z64) <= 22].max() < 2.0 ** -19 and off.max() < 2.0 ** -17  # what the header says
    one, none = torch.ones(1, 1, c), torch.zeros(1, 1, c)
    gate = z.view(1, 1, c).cuda()
    y, _ = sb.leaky_scan(one.to(kind).cuda(), gate, logit=True, complement=True, dtype=torch.float32)
    want = 1 / (1 + np.exp(z64))
    assert (np.abs(y.double().cpu().numpy().ravel() - want) <= off * want).all()
    y, _ = sb.leaky_scan(none.to(kind).cuda(), gate, h0=one[0].cuda(), logit=True, dtype=torch.float32)
    want = 1 / (1 + np.exp(-z64))
    assert (np.abs(y.double().cpu().numpy().ravel() - want) <= off * want).all()


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


def off(got, want):
    """How far all of it is off, as a share of all of it."""
    return ((got.double() - want).norm() / want.norm()).item()


# Channels in segments; in crews of 16 and of 8 warps, where 104 and 149 columns of a thread each are walked.
FORMS = [400, 3401, 4801]


@pytest.mark.parametrize("c", FORMS)
def test_shared_gate_over_a_long_memory(c):
    """The gradient of a leak a channel over 5280 steps. A block's product of gates is the same in every map: one
    rounding of it leaves the sum 4.9e-7 off in an emulation of the crews in 32 bits (steps one by one 3.3e-7),
    seven roundings 1.3e-6."""
    t = 5280
    x, dy, dh, h0 = normal(1, 1, t, c), normal(2, 1, t, c), normal(3, 1, c), normal(4, 1, c)
    a = torch.exp(-1 / torch.exp(np.log(5.0) + np.log(40.0) * torch.rand(c, generator=torch.Generator().manual_seed(5)))).cuda()
    y, h_last, saved = sb.leaky_scan(x, a, h0=h0, save=True)
    dx, dgate, dh0 = sb.leaky_scan_backward(dy, x, a, saved, dh_last=dh)
    a64, h, before = a.double(), h0[0].double(), torch.empty(t, c, dtype=torch.float64, device="cuda")
    for i in range(t):
        before[i] = h
        h = a64 * h + x[0, i]
    assert off(h_last[0], h) < 8e-7 and off(y[0, :-1], before[1:]) < 8e-7
    e, want, delta = dh[0].double(), torch.zeros(c, dtype=torch.float64, device="cuda"), torch.empty_like(before)
    for i in range(t - 1, -1, -1):
        delta[i] = dy[0, i] + e
        want += delta[i] * before[i]
        e = a64 * delta[i]
    assert off(dgate, want) < 8e-7
    assert off(dx[0], delta) < 8e-7 and off(dh0[0], e) < 8e-7


@pytest.mark.parametrize("complement", [False, True])
@pytest.mark.parametrize("c", FORMS)
def test_states_of_long_memories_from_logits(c, complement):
    """Logits around 6, memories of 400 steps: a gate's error grows by 1 / (1 - a) on its way into a state. With gates
    within half a unit (of a sum 1 + exp that is rounded itself) 4000 steps one by one in 32 bits leave the states
    5.9e-7 off, with a half more at the reciprocal 7.4e-7, with reciprocals a unit off 1.1e-6 at least."""
    t = 4000
    x, z = normal(6, 1, t, c), 6 + normal(7, 1, t, c) / 2
    y, _ = sb.leaky_scan(x, z, logit=True, complement=complement)
    z64 = z[0].double()
    a, u = torch.sigmoid(z64), x[0].double() * (torch.sigmoid(-z64) if complement else 1.0)
    h, want = torch.zeros(c, dtype=torch.float64, device="cuda"), torch.empty(t, c, dtype=torch.float64, device="cuda")
    for i in range(t):
        h = a[i] * h + u[i]
        want[i] = h
    assert off(y[0], want) < 9e-7


@pytest.mark.parametrize("src,gate", [("u8", "channel"), ("bf16", "step"), ("f32", "channel")])
def test_a_few_rows_of_many_take_the_same_values(src, gate):
    """Rows of a large batch, walked whole, beside the same rows by themselves, in crews: each step's state has one
    rounding of its own, which a map's has too, so they part by a few units of 2^-24 of the largest that decay."""
    from tests.test_leaky_gpu import Problem
    p = Problem(1300, 60, 130, src, gate, "bf16" if src == "bf16" else "f32", "f32", seed=8)
    y, h_last = p.forward()
    few = Problem(2, 60, 130, src, gate, "bf16" if src == "bf16" else "f32", "f32", seed=8)
    few.x, few.h0 = p.x[:2].contiguous(), p.h0[:2].contiguous()
    few.gate = p.gate if gate == "channel" else p.gate[:2].contiguous()
    y2, h2 = few.forward()
    assert off(y[:2], y2.double()) < 4 * 2.0 ** -24 and off(h_last[:2], h2.double()) < 4 * 2.0 ** -24
