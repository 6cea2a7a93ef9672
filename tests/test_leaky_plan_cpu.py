"""How calls of the leaky recurrence are cut, seen in the workspaces they ask
for: a call whose channels are enough is walked whole and asks for none."""
import ctypes as C

import pytest

import snn_b200 as sb

F32, F16, BF16, SPIKES = 0, 1, 2, 3


def workspace(b, t, c, x, step_gate, backward):
    y = F32 if x == SPIKES else x
    q = sb.Leaky(b, t, c, x, F32, y, 0, 0, 0.5, 1.0, t * c, c, 0, c if step_gate else 0, t * c, c, t * c, c, t * c, c,
                 t * c, c)
    return sb.lib().snn_b200_leaky_workspace(C.byref(q), backward)


@pytest.mark.parametrize("x", [F32, F16, BF16])
@pytest.mark.parametrize("step_gate", [False, True])
@pytest.mark.parametrize("b,t,c", [(100, 2000, 1000), (100, 20000, 1000), (80, 1500, 1000), (128, 400, 1024), (64, 200, 1000)])
def test_whole_walks_ask_for_sums_only(b, t, c, x, step_gate):
    assert workspace(b, t, c, x, step_gate, 0) == 0
    sums = 0 if step_gate else (b * c * 4 + 255) // 256 * 256  # a shared gate's gradient, one a channel
    assert workspace(b, t, c, x, step_gate, 1) == sums


@pytest.mark.parametrize("b,t,c,crew", [(4, 8192, 2048, 16), (8, 2048, 1500, 8), (2, 400, 8, 16)])
def test_crews_ask_for_no_segments(b, t, c, crew):
    for x in (F32, BF16):
        assert workspace(b, t, c, x, True, 0) == workspace(b, t, c, x, True, 1) == 256
        assert workspace(b, t, c, x, False, 1) == max(256, (crew * b * c * 4 + 255) // 256 * 256)


def test_short_sequences_in_crews_ask_for_none():
    for b, t, c in ((2, 30, 64), (100, 127, 300)):
        assert workspace(b, t, c, F32, False, 0) == workspace(b, t, c, SPIKES, True, 0) == 0
        assert workspace(b, t, c, F32, True, 1) == 0


def test_segments_ask_for_their_maps_and_states():
    # 64 steps a segment; a map of 8 bytes and a state of 4 a channel and segment.
    assert workspace(1, 6400, 800, F32, True, 0) == 100 * 800 * 12


@pytest.mark.parametrize("step_gate", [False, True])
@pytest.mark.parametrize("b,t,c", [(64, 200, 1000), (128, 400, 1024), (100, 2000, 1000), (46, 200, 1040), (151, 257, 1000)])
def test_rasters_are_cut_like_other_sequences(b, t, c, step_gate):
    """Four channels a thread are half the columns, not a reason for segments."""
    assert workspace(b, t, c, SPIKES, step_gate, 0) == workspace(b, t, c, F32, step_gate, 0) == 0


def test_rows_of_a_step_that_name_slots():
    """As many as are looked through in seconds; rows without slots may be more."""
    call = lambda batch, slots: sb.lib().snn_b200_leaky_step_async(  # noqa: E731
        0, None, batch, 1 << 23, 0, 1 << 20, F32, 0, None, F32, 0, 0, 0, 0.5, 1.0, 1 << 20, 0, slots, 1 << 20, F32, 0)
    assert call(1 << 22, 1 << 20) == call((1 << 22) + 1, None) == sb.SNN_OK  # no channels: nothing is launched
    assert call((1 << 22) + 1, 1 << 20) == sb.SNN_ERR_OVERFLOW
