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
