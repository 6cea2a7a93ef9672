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
