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


KINDS = [("f32", "channel", "f32", "f32", True, True), ("f32", "step", "f32", "f32", False, True),
         ("bf16", "step", "bf16", "bf16", True, True), ("bf16", "step", "f32", "f32", True, False),
         ("f16", "step", "f16", "f16", True, True), ("f16", "sequence", "f32", "f16", True, False),
         ("u8", "step", "f32", "f32", True, True), ("u8", "channel", "f32", "f32", True, False)]


@pytest.mark.parametrize("src,gate,gate_type,out,logit,complement", KINDS)
@pytest.mark.parametrize("b,t,c,ragged,time_major", [
    (10, 41, 1000, False, False), (12, 133, 1024, True, True), (7, 70, 1401, True, False), (46, 17, 1002, False, True),
    (3, 1030, 3400, False, False)])
def test_crews_of_8_warps(b, t, c, ragged, time_major, src, gate, gate_type, out, logit, complement):
    """149 to 739 columns of 64 (odd rows: 32) channels: two crews an SM, full and ragged rounds of 8 blocks."""
    lengths = np.random.default_rng(t).integers(0, t + 1, b).tolist() if ragged else None
    Problem(b, t, c, src, gate, gate_type, out, logit, complement, 0.75, lengths, time_major, seed=22).verify()


@pytest.mark.parametrize("src,gate,gate_type,out,logit,complement", KINDS[1:3])
def test_crews_of_8_warps_up_to_1183_columns(src, gate, gate_type, out, logit, complement):
    Problem(30, 261, 1602, src, gate, gate_type, out, logit, complement, seed=23).verify()


@pytest.mark.parametrize("src,gate,gate_type,out,logit,complement", KINDS)
@pytest.mark.parametrize("b,t,c,ragged,time_major", [
    (50, 100, 1000, False, True), (52, 41, 1024, True, False), (40, 33, 701, True, True), (1200, 65, 64, True, False)])
def test_whole_walks_and_their_gradients(b, t, c, ragged, time_major, src, gate, gate_type, out, logit, complement):
    """740 columns and more of 17 to 256 steps: one warp walks each from end to end."""
    lengths = np.random.default_rng(t).integers(0, t + 1, b).tolist() if ragged else None
    Problem(b, t, c, src, gate, gate_type, out, logit, complement, 0.75, lengths, time_major, seed=24).verify()
