"""The forms in which a call of the leaky recurrence is walked, each against the
definition in 64 bits: rasters of four and of two channels a thread, crews of 8
and of 16 warps, whole walks with their gradient."""
import numpy as np
import pytest

from tests.test_leaky_gpu import Problem

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("gate,logit", [("channel", True), ("sequence", False), ("step", True), ("none", False)])
@pytest.mark.parametrize("time_major", [False, True])
@pytest.mark.parametrize("b,t,c,ragged", [
    (51, 33, 1000, False), (64, 70, 1000, True), (49, 40, 1024, False), (80, 261, 1008, True), (95, 30, 804, False),
    (60, 20, 1602, True), (3, 1100, 1000, False), (2, 1200, 1040, True)])
def test_rasters_of_many_and_of_few_channels(b, t, c, ragged, time_major, gate, logit):
    """Rows in pieces of 16 bytes (1024, 1040, 1008 channels), of 4 (1000, 804), of 2 (1602); walked whole from
    740 columns of 64 channels on (1184 above 256 steps), few long ones in segments."""
    lengths = np.random.default_rng(t).integers(0, t + 1, b).tolist() if ragged else None
    Problem(b, t, c, "u8", gate, "f32", None, logit, True, 0.5, lengths, time_major, seed=21).verify(gradient=False)
