"""Tensors as a program has them: expanded, with lazy signs, under autograd."""
import numpy as np
import pytest

import snn_b200 as sb
from tests._sequence_ref import LeakyRef, check
from tests.test_leaky_gpu import Problem, host

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("t", [1, 2, 40, 1500])
def test_16_bit_gates_expanded_over_the_steps(kind, t):
    """A gate [batch, steps, channels] is what its elements say, however it is stored."""
    for shape in ((3, 1, 50), (1, 1, 50), (3, 1, 51)):
        for logit in (False, True):
            p = Problem(3, t, shape[2], kind, "none", None, None, logit, True, seed=31)
            p.how.pop("decay")
            p.gate = p.leak(logit, *shape).to(TYPES[kind]).cuda().expand(3, t, shape[2])
            p.verify()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("b", [1, 5, 700])
def test_16_bit_gates_expanded_over_the_rows_of_a_step(kind, b):
    p = Problem(b, 1, 66, kind, "none", seed=32)
    z = p.leak(True, 1, 66).to(TYPES[kind]).cuda().expand(b, 66)
    pool = torch.randn(b, 66, generator=p.g).cuda()
    ref = LeakyRef(host(p.x), host(z)[:, None], None, host(pool), None, True, True)
    y = sb.leaky_step(p.x[:, 0], z, pool, logit=True, complement=True)
    check(host(y), ref.y[:, 0], ref.y_err[:, 0], kind, "y")
    check(host(pool), ref.h_last, ref.h_last_err, "f32", "pool")


def test_signs_that_are_only_noted():
    """The imaginary part of a conjugate is a view whose sign torch keeps as a flag."""
    g = torch.Generator().manual_seed(33)
    lazy = lambda *shape: torch.randn(*shape, dtype=torch.complex64, generator=g).cuda().conj().imag  # noqa: E731
    x, z, h0, dy = lazy(2, 40, 12), lazy(2, 40, 12), lazy(2, 12), lazy(2, 40, 12)
    assert x.is_neg() and z.is_neg()
    plain = [t.clone().resolve_neg() for t in (x, z, h0, dy)]
    y, h, saved = sb.leaky_scan(x, z, h0=h0, logit=True, save=True)
    want = sb.leaky_scan(plain[0], plain[1], h0=plain[2], logit=True, save=True)
    assert all(torch.equal(a, b) for a, b in zip((y, h, saved), want))
    for a, b in zip(sb.leaky_scan_backward(dy, x, z, saved, dh_last=h0, logit=True),
                    sb.leaky_scan_backward(plain[3], plain[0], plain[1], saved, dh_last=plain[2], logit=True)):
        assert torch.equal(a, b)
    w, b = lazy(7, 12), lazy(7)
    assert torch.equal(sb.mx4_linear(x, sb.mx4_quantize(w), bias=b.resolve_neg()),
                       sb.mx4_linear(plain[0], sb.mx4_quantize(w.resolve_neg()), bias=b.resolve_neg()))
    pools = torch.zeros(2, 12, device="cuda"), torch.zeros(2, 12, device="cuda")
    assert torch.equal(sb.leaky_step(x[:, 0], z[:, 0], pools[0], logit=True),
                       sb.leaky_step(plain[0][:, 0], plain[1][:, 0], pools[1], logit=True))
    assert torch.equal(*pools)
    with pytest.raises(sb.SnnError) as e:
        sb.leaky_step(plain[0][:, 0], plain[1][:, 0], torch._neg_view(pools[0]), logit=True)
    assert e.value.status == sb.SNN_ERR_INVALID_ARGUMENT
    assert torch.equal(*pools)
