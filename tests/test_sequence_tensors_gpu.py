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


def test_results_of_inputs_that_require_a_gradient_say_so():
    """Going back through an operator without a formula is an error, not an empty gradient."""
    g = torch.Generator().manual_seed(34)
    x = torch.randn(2, 40, 12, generator=g).cuda()
    z, h0 = torch.randn(12, generator=g).cuda(), torch.randn(2, 12, generator=g).cuda()
    w, bias = sb.mx4_quantize(torch.randn(7, 12, generator=g).cuda()), torch.randn(7, generator=g).cuda()
    pool = torch.zeros(2, 12, device="cuda")
    takes = {"leaky_scan_backward": (0, 1, 2), "leaky_scan": (0, 1, 2), "leaky_step": (0, 1), "mx4_linear": (0, 3),
             "mx4_matmul": (3,)}
    calls = {
        "leaky_scan_backward": lambda x, z, h0, b: sb.leaky_scan(x, z, h0=h0, logit=True)[0],
        "leaky_scan": lambda x, z, h0, b: sb.leaky_scan(x.transpose(0, 1).contiguous().transpose(0, 1), z, h0=h0)[1],
        "leaky_step": lambda x, z, h0, b: sb.leaky_step(x[:, 0], z, pool),
        "mx4_linear": lambda x, z, h0, b: sb.mx4_linear(x, w, bias=b),
        "mx4_matmul": lambda x, z, h0, b: sb.mx4_matmul(w, w, bias=b),
    }
    for text, f in calls.items():
        plain = f(x, z, h0, bias)
        assert not plain.requires_grad
        for i, t in enumerate((x, z, h0, bias)):
            pool.zero_()
            leaf = t.clone().requires_grad_()
            args = [leaf if j == i else u for j, u in enumerate((x, z, h0, bias))]
            y = f(*args)
            assert torch.equal(y, plain)
            with torch.no_grad():
                assert not f(*args).requires_grad
            assert y.requires_grad == (i in takes[text])
            if not y.requires_grad:
                continue
            with pytest.raises(NotImplementedError, match=text):
                (y.sum() + leaf.sum()).backward()
            with pytest.raises(RuntimeError):
                torch.autograd.grad(f(*args).sum(), leaf)
            args[i] = leaf * 2
            with pytest.raises(NotImplementedError, match=text):
                torch.autograd.grad(f(*args).sum() + leaf.sum(), leaf)


def test_gradient_calls_under_autograd():
    """x and the gate may be leaves that are trained by hand, or inside a Function."""
    g = torch.Generator().manual_seed(35)
    x = torch.randn(3, 50, 10, generator=g).cuda().requires_grad_()
    z = torch.randn(10, generator=g).cuda().requires_grad_()
    dy = torch.randn(3, 50, 10, generator=g).cuda()
    y, _, saved = sb.leaky_scan(x, z, logit=True, save=True)
    assert y.requires_grad and not saved.requires_grad
    by_hand = sb.leaky_scan_backward(dy, x, z, saved, logit=True)
    assert not any(t.requires_grad for t in by_hand)
    twice = sb.leaky_scan_backward(dy.clone().requires_grad_(), x, z, saved, logit=True)
    with pytest.raises(NotImplementedError):
        twice[0].sum().backward()

    class Scan(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, z):
            y, _, saved = sb.leaky_scan(x, z, logit=True, save=True)
            ctx.save_for_backward(x, z, saved)
            return y

        @staticmethod
        def backward(ctx, dy):
            x, z, saved = ctx.saved_tensors
            return sb.leaky_scan_backward(dy, x, z, saved, logit=True)[:2]

    Scan.apply(x, z).backward(dy)
    assert torch.equal(x.grad, by_hand[0]) and torch.equal(z.grad, by_hand[1])

    # The results above live on: they do not tie the leaves to the stream that they were made on.
    assert y.requires_grad and not y.grad_fn.next_functions
    x.grad = z.grad = None
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        Scan.apply(x, z).backward(dy)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(x.grad, by_hand[0]) and torch.equal(z.grad, by_hand[1])


def test_updates_in_place_are_new_versions():
    pool, scale = torch.ones(2, 12, device="cuda"), torch.ones(2, 12, device="cuda", requires_grad=True)
    loss = (pool * scale).sum()  # keeps the pool for the gradient of scale
    sb.leaky_step(torch.ones(2, 12, device="cuda"), None, pool, decay=0.5)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    with pytest.raises(sb.SnnError) as e:
        sb.leaky_step(torch.ones(2, 12, device="cuda"), None, pool.clone().requires_grad_(), decay=0.5)
    assert e.value.status == sb.SNN_ERR_INVALID_ARGUMENT
    q = sb.mx4_quantize(torch.ones(4, 64, device="cuda"))
    before = q.codes._version, q.scales._version
    sb.mx4_quantize(torch.zeros(4, 64, device="cuda"), out=q)
    assert q.codes._version > before[0] and q.scales._version > before[1]
    with torch.inference_mode():
        still = torch.ones(2, 12, device="cuda")
        sb.leaky_step(still, None, still.clone(), decay=0.5)
    sb.leaky_step(torch.ones(2, 12, device="cuda"), None, still, decay=0.5)
    assert torch.equal(still, torch.full((2, 12), 1.5, device="cuda"))


def test_captured_with_leaves_that_require_a_gradient():
    x = torch.randn(2, 30, 8, device="cuda").requires_grad_()
    z = torch.randn(2, 30, 8, device="cuda").requires_grad_()
    eager, _, saved = sb.leaky_scan(x, z, logit=True, save=True)  # lives on beside the graph
    want = [eager, *sb.leaky_scan_backward(eager.detach(), x, z, saved, logit=True)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _, saved = sb.leaky_scan(x, z, logit=True, save=True)
        got = [y, *sb.leaky_scan_backward(y.detach(), x, z, saved, logit=True)]
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
