"""The packed product of rows whose blocks differ by many powers of two, where
sums that were aligned in fewer than 32 bits would show."""
import pytest

import snn_b200 as sb
from tests._sequence_ref import check
from tests.test_mx4_gpu import TYPES, host, product_bound

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def blocks(rows, cols, kind, spread, seed):
    """Normal values, each block of 32 scaled by a power of two of its own, within the type's range."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g)
    e = torch.randint(-spread, spread + 1, (rows, -(-cols // 32)), generator=g).float()
    return (x * torch.exp2(e).repeat_interleave(32, 1)[:, :cols]).to(TYPES[kind]).cuda()


# Rows of x packed on the way (up to 16), packed before, with k split over CTAs, by pairs of CTAs.
@pytest.mark.parametrize("m,k,n", [(1, 64, 130), (4, 8192, 136), (16, 500, 300), (24, 4100, 200), (100, 2048, 128),
                                   (130, 5000, 300), (300, 784, 1000), (700, 256, 640), (1, 40000, 3)])
@pytest.mark.parametrize("kind,spread", [("f32", 4), ("f32", 12), ("f32", 40), ("bf16", 12), ("f16", 8)])
def test_rows_of_uneven_blocks(m, k, n, kind, spread):
    x, w = blocks(m, k, kind, spread, m + k), blocks(n, k, "f32", spread, n + k)
    w[:, 32:64] *= -1  # sums that cancel
    q = sb.mx4_quantize(w)
    xv, wv = host(sb.mx4_dequantize(sb.mx4_quantize(x))), host(sb.mx4_dequantize(q))
    want, room = xv @ wv.T, product_bound(xv, wv)
    check(host(sb.mx4_linear(x, q, dtype=torch.float32)), want, room, "f32", "linear")
    check(host(sb.mx4_matmul(sb.mx4_quantize(x), q)), want, room, "f32", "matmul")


@pytest.mark.parametrize("m", [1, 40, 300])
def test_a_large_block_beside_small_ones(m):
    """One block 2^18 times the others, which cancels in itself. Every partial sum is a multiple of 1/2 below 2^22,
    so sums in 32 bits round nothing, in any order."""
    k, n = 256, 64
    x = torch.ones(m, k, device="cuda")
    w = torch.full((n, k), 0.5, device="cuda")
    w[:, :32] = 2.0 ** 17
    w[:, 16:32] = -2.0 ** 17
    y = sb.mx4_linear(x, sb.mx4_quantize(w))
    assert (y == 0.5 * (k - 32)).all()
