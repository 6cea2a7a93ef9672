"""Packed 4-bit matrices on the GPU: packing, reading back and the product,
against their definitions in 64 bits."""
import numpy as np
import pytest

import snn_b200 as sb
from tests._sequence_ref import check, mx4_parts, mx4_values, scale_offsets

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "u8": torch.uint8}


def host(t):
    return t.double().cpu().numpy() if t.dtype.is_floating_point else t.cpu().numpy()


def draw(shape, kind, seed, spread=0.0):
    """Normal values whose rows' magnitudes spread over powers of two, or spikes."""
    g = torch.Generator().manual_seed(seed)
    if kind == "u8":
        return (torch.rand(*shape, generator=g) < 0.2).to(torch.uint8).cuda()
    x = torch.randn(*shape, generator=g)
    if spread:
        x = x * torch.exp2(torch.randint(-int(spread), int(spread) + 1, (shape[0], 1), generator=g).float())
    return x.to(TYPES[kind]).cuda()


def unpacked(q):
    codes = q.codes.cpu().numpy().reshape(q.rows, -1)
    out = np.empty((q.rows, codes.shape[1] * 2), np.int64)
    out[:, 0::2], out[:, 1::2] = codes & 15, codes >> 4
    return out


SHAPES = [(1, 1), (1, 31), (3, 32), (5, 33), (127, 128), (128, 129), (129, 784), (1000, 784), (257, 1027), (33, 4100)]


@pytest.mark.parametrize("order", ["rows", "cols", "words", "wide"])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16", "u8"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_pack_matches_definition(rows, cols, kind, order):
    x = draw((rows, cols), kind, rows * 7 + cols, spread=8 if kind != "u8" else 0)
    if order == "cols":
        view = x.t().contiguous().t()
    elif order == "words":  # columns of a whole number of words
        big = torch.zeros(cols, (rows + 7) // 4 * 4, dtype=x.dtype, device="cuda")
        view = big[:, :rows].t()
        view.copy_(x)
    elif order == "wide":  # every third element of wider rows, at an odd offset
        big = torch.zeros(rows, cols * 3 + 5, dtype=x.dtype, device="cuda")
        view = big[:, 1:1 + cols * 3:3]
        view.copy_(x)
    else:
        view = x
    q = sb.mx4_quantize(view)
    codes, scales = mx4_parts(host(x) != 0 if kind == "u8" else host(x))
    assert np.array_equal(unpacked(q), codes)
    raw = q.scales.cpu().numpy()
    at = scale_offsets(rows, cols)
    assert np.array_equal(raw[at], scales)
    rest = np.ones(raw.size, bool)
    rest[at.ravel()] = False
    assert not raw[rest].any()  # bytes without a row or a block
    values = mx4_values(host(x) != 0 if kind == "u8" else host(x))
    assert np.array_equal(host(sb.mx4_dequantize(q)), values)
    assert np.array_equal(host(sb.mx4_dequantize(q, torch.bfloat16)), values)
    want16 = values.astype(np.float16)
    assert np.array_equal(host(sb.mx4_dequantize(q, torch.float16)), want16.astype(np.float64))


def test_pack_ties_extremes_and_not_finite():
    x = torch.zeros(12, 64)
    x[0, :8] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0])  # ties; amax 5 -> scale 1
    x[1, :8] = -x[0, :8]
    x[2, :4] = torch.tensor([7.99, 6.5, 6.0, 5.01])  # beyond 6
    x[3, 0] = 2.0 ** -149  # smallest subnormal
    x[3, 1] = 2.0 ** -127
    x[4, 0] = torch.finfo(torch.float32).max
    x[4, 1] = -2.0 ** 125
    x[5, 40] = float("inf")
    x[5, 0] = 1.0
    x[6, 3] = float("nan")
    x[7, 3] = -0.0
    x[8, :] = 2.0 ** -126
    x[9, 0], x[9, 1] = 2.0 ** -124, 2.0 ** -126
    x[10, 33] = float("-inf")
    q = sb.mx4_quantize(x.cuda())
    codes, scales = mx4_parts(x.numpy())
    assert np.array_equal(q.scales.cpu().numpy()[scale_offsets(12, 64)], scales)
    got, want = host(sb.mx4_dequantize(q)), mx4_values(x.numpy())
    assert np.array_equal(got, want, equal_nan=True)
    assert np.isnan(got[5, 32:]).all() and np.isfinite(got[5, :32]).all()
    assert np.isnan(got[6, :32]).all() and not got[6, 32:].any()


def test_pack_offsets_beyond_32_bits():
    """Rows that start more than 2^31 elements into their array."""
    big = torch.zeros((1 << 31) + 4096, dtype=torch.uint8, device="cuda")
    stride = (1 << 31) // 2
    view = torch.as_strided(big, (3, 300), (stride, 1))
    view[2, 7], view[1, 5], view[0, 299] = 1, 1, 1
    got = sb.mx4_dequantize(sb.mx4_quantize(view))
    assert torch.equal(got != 0, view != 0)


def product_bound(x, w):
    """What sums in 32 bits may lose: a unit of 2^-22 of all magnitudes for each 64 products joined."""
    k = x.shape[1]
    return (-(-k // 64) + 2) * 2.0 ** -22 * (np.abs(x) @ np.abs(w).T)


LINEAR = [(1, 1, 1), (1, 784, 1000), (2, 32, 8), (3, 33, 129), (4, 8192, 256), (7, 1000, 10), (16, 500, 300),
          (17, 256, 128), (31, 64, 1), (33, 1027, 200), (64, 2048, 136), (100, 128, 128), (128, 4100, 257),
          (129, 96, 130), (257, 640, 384), (300, 784, 1000), (1, 40000, 3), (1000, 1000, 10), (513, 31, 127),
          (3300, 200, 1300), (4097, 300, 1025), (20000, 64, 250), (130, 300, 19000), (300, 4100, 200), (70, 5000, 130)]


@pytest.mark.parametrize("m,k,n", LINEAR)
@pytest.mark.parametrize("src,out,bias", [("u8", "f32", False), ("bf16", "bf16", True), ("f32", "f32", True),
                                          ("f16", "f16", False), ("bf16", "f32", False)])
def test_linear_matches_definition(m, k, n, src, out, bias):
    x = draw((m, k), src, m + k, spread=3 if src != "u8" else 0)
    weights = draw((n, k), "f32", n + 3 * k, spread=2) / k ** 0.5
    b = torch.randn(n, generator=torch.Generator().manual_seed(n)).cuda() if bias else None
    w = sb.mx4_quantize(weights)
    y = sb.mx4_linear(x, w, bias=b, dtype=TYPES[out])
    xv = mx4_values(host(x) != 0 if src == "u8" else host(x))
    wv = mx4_values(host(weights))
    want = xv @ wv.T
    err = product_bound(xv, wv)
    if bias:
        want = want + host(b)
        err = err + 2.0 ** -24 * np.abs(want)
    check(host(y), want, err, out, "linear")
    # The same through a matrix packed before.
    z = sb.mx4_matmul(sb.mx4_quantize(x), w, bias=b, dtype=TYPES[out])
    assert torch.equal(y, z)
    # Results repeat.
    assert torch.equal(y, sb.mx4_linear(x, w, bias=b, dtype=TYPES[out]))


@pytest.mark.parametrize("m", [1, 5, 40, 130, 600])
def test_spikes_through_packed_weights_are_exact(m):
    """Spikes are exact in the packed form, and sums of a few hundred packed
    weights of one magnitude fit 24 bits: nothing is rounded but the weights."""
    x = draw((m, 784), "u8", m)
    weights = draw((1000, 784), "f32", 2)
    weights[:, ::32] = 4.0  # one scale for all blocks
    w = sb.mx4_quantize(weights.clamp_(-4, 4))
    want = (host(x) != 0) @ mx4_values(host(weights)).T
    assert np.array_equal(host(sb.mx4_linear(x, w)), want)


def test_linear_rows_do_not_depend_on_their_neighbours():
    """A NaN or an infinity in one row, or in one weight row, stays there."""
    x = draw((130, 300), "bf16", 1)
    w0 = draw((140, 300), "f32", 2)
    clean = sb.mx4_linear(x, sb.mx4_quantize(w0))
    x[7, 3], x[129, 299] = float("nan"), float("inf")
    w0[11, 40] = float("inf")
    y = sb.mx4_linear(x, sb.mx4_quantize(w0))
    bad = torch.zeros(130, 140, dtype=torch.bool, device="cuda")
    bad[7], bad[129], bad[:, 11] = True, True, True
    assert torch.isnan(y[bad]).all()
    assert torch.equal(y[~bad], clean[~bad])


def test_linear_strides_and_rows_behind():
    """Rows of x and of the result inside wider arrays: what lies beside them stays as it was."""
    m, k, n = 37, 200, 70
    wide = draw((m, 333), "f16", 5)
    x = wide[:, 11:11 + k]
    w = sb.mx4_quantize(draw((n, k), "f32", 6))
    want = sb.mx4_linear(x.contiguous(), w)
    assert torch.equal(sb.mx4_linear(x, w), want)
    assert torch.equal(sb.mx4_linear(x.t().contiguous().t(), w), want)
    out = torch.full((m + 2, n + 13), -7.0, dtype=torch.float16, device="cuda")
    need = sb.lib().snn_b200_mx4_linear_workspace(x.data_ptr(), 1, m, k, x.stride(0), 1)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    st = sb.lib().snn_b200_mx4_linear_async(0, torch.cuda.current_stream().cuda_stream, x.data_ptr(), 1, m, k,
                                            x.stride(0), 1, w.codes.data_ptr(), w.scales.data_ptr(), n, None,
                                            out.data_ptr(), 1, n + 13, ws.data_ptr(), need)
    assert st == sb.SNN_OK
    assert torch.equal(out[:m, :n], want)
    assert (out[m:] == -7).all() and (out[:, n:] == -7).all()


def test_empty_products():
    w = sb.mx4_quantize(torch.ones(5, 64, device="cuda"))
    assert sb.mx4_linear(torch.ones(0, 64, device="cuda"), w).shape == (0, 5)
    none = sb.mx4_quantize(torch.ones(0, 64, device="cuda"))
    assert sb.mx4_linear(torch.ones(3, 64, device="cuda"), none).shape == (3, 0)
    flat = sb.mx4_quantize(torch.ones(5, 0, device="cuda"))
    bias = torch.arange(5.0, device="cuda")
    assert torch.equal(sb.mx4_linear(torch.ones(3, 0, device="cuda"), flat, bias=bias), bias.expand(3, 5))
    assert torch.equal(sb.mx4_linear(torch.ones(200, 0, device="cuda"), flat), torch.zeros(200, 5, device="cuda"))
    assert sb.mx4_linear(torch.ones(2, 3, 64, device="cuda"), w).shape == (2, 3, 5)


@pytest.mark.parametrize("m", [1, 24, 400])
def test_linear_on_a_side_stream_and_replayed(m):
    x = draw((m, 784), "u8", 3)
    w = sb.mx4_quantize(draw((100, 784), "f32", 4))
    want = sb.mx4_linear(x, w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a = sb.mx4_linear(x, w)
    side.synchronize()
    assert torch.equal(a, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b = sb.mx4_linear(x, w)
    for seed in (8, 9):
        x.copy_(draw((m, 784), "u8", seed))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(b, sb.mx4_linear(x, w))


@pytest.mark.parametrize("m,k,n", [(1, 784, 1000), (700, 512, 640)])
def test_two_products_at_once(m, k, n):
    """Calls on two streams, each with its own workspace, do not disturb each other."""
    w = sb.mx4_quantize(draw((n, k), "f32", 4))
    xs = [draw((m, k), "bf16", s) for s in range(2)]
    want = [sb.mx4_linear(x, w) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for _ in range(10):
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                got.append(sb.mx4_linear(x, w))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 2])


def test_a_device_that_is_not_there_and_the_callers_own():
    """A device index beyond the last one is an error of the call alone; the caller's current device stays."""
    x = torch.ones(4, 64, device="cuda")
    q = sb.mx4_quantize(x)
    L = sb.lib()
    args = (None, x.data_ptr(), 0, 4, 64, 64, 1, q.codes.data_ptr(), q.scales.data_ptr())
    before = torch.cuda.current_device()
    assert L.snn_b200_mx4_quantize_async(torch.cuda.device_count() + 7, *args) == sb.SNN_ERR_CUDA
    assert sb.last_error()
    assert torch.cuda.current_device() == before
    assert L.snn_b200_mx4_quantize_async(before, *args) == sb.SNN_OK
    assert torch.equal(sb.mx4_dequantize(q), x)
    torch.cuda.synchronize()
