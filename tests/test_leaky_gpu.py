"""The leaky recurrence on the GPU: scan, gradient and single step, against
their definitions in 64 bits."""
import numpy as np
import pytest

import snn_b200 as sb
from tests._sequence_ref import LeakyRef, check

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "u8": torch.uint8}


def host(t):
    return t.double().cpu().numpy() if t.dtype.is_floating_point else t.cpu().numpy()


class Problem:
    """Inputs of one call, and the call, forward and backward."""

    def __init__(self, b, t, c, src="f32", gate="channel", gate_type="f32", out=None, logit=False, complement=False,
                 scale=1.0, lengths=None, time_major=False, seed=0, h0=True, decay=None):
        self.g = torch.Generator().manual_seed(seed * 1000 + b * 31 + t * 7 + c)
        self.b, self.t, self.c, self.src, self.time_major = b, t, c, src, time_major
        self.out = out or ("f32" if src == "u8" else src)
        self.x = self.sequence(src)
        shape = {"channel": (c,), "sequence": (b, c)}.get(gate)
        if gate == "none":
            self.gate = None
        elif shape:
            self.gate = self.leak(logit, *shape).cuda()
        elif gate == "step":
            self.gate = self.sequence(gate_type, lambda *s: self.leak(logit, *s))
        elif gate == "shared":  # every step its own, the same for all sequences
            self.gate = self.leak(logit, t, c).to(TYPES[gate_type]).cuda()[None].expand(b, t, c)
        self.h0 = torch.randn(b, c, generator=self.g).cuda() if h0 else None
        self.lengths = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
        self.dy, self.dh = self.sequence(self.out), torch.randn(b, c, generator=self.g).cuda()
        self.how = dict(logit=logit, complement=complement, input_scale=scale, lengths=self.lengths)
        if gate == "none":
            self.how["decay"] = 0.9 if decay is None else decay
        if lengths is not None:  # nothing behind a sequence may be looked at
            for i, n in enumerate(lengths):
                if src != "u8":
                    self.x[i, n:] = float("nan")
                self.dy[i, n:] = float("inf")
                if gate == "step":
                    self.gate[i, n:] = float("nan")

    def leak(self, logit, *shape):
        if logit:
            return torch.randn(*shape, generator=self.g) * 3 + 1
        return torch.exp(-1 / (2 + 50 * torch.rand(*shape, generator=self.g)))

    def sequence(self, kind, make=None):
        shape = (self.t, self.b, self.c) if self.time_major else (self.b, self.t, self.c)
        if make is not None:
            v = make(*shape)
        elif kind == "u8":
            v = torch.rand(*shape, generator=self.g) < 0.3
        else:
            v = torch.randn(*shape, generator=self.g)
        v = v.to(TYPES[kind]).cuda()
        return v.transpose(0, 1) if self.time_major else v

    def reference(self):
        gate = None if self.gate is None else host(self.gate)
        x = host(self.x) != 0 if self.src == "u8" else host(self.x)
        return LeakyRef(x, gate, self.how.get("decay"), None if self.h0 is None else host(self.h0),
                        None if self.lengths is None else self.lengths.cpu().numpy(), self.how["logit"],
                        self.how["complement"], np.float64(np.float32(self.how["input_scale"])))

    def forward(self, save=False):
        return sb.leaky_scan(self.x, self.gate, h0=self.h0, dtype=TYPES[self.out], save=save, **self.how)

    def backward(self, saved):
        return sb.leaky_scan_backward(self.dy, self.x, self.gate, saved, dh_last=self.dh, **self.how)

    def verify(self, gradient=True):
        with np.errstate(invalid="ignore"):
            ref = self.reference()
        y, h_last, saved = self.forward(save=True)
        assert (y.stride(0) < y.stride(1)) == (self.time_major and self.b > 1 and self.t > 1) or self.b == 1
        check(host(y), ref.y, ref.y_err, self.out, "y")
        check(host(h_last), ref.h_last, ref.h_last_err, "f32", "h_last")
        y2, h2 = self.forward()
        assert torch.equal(y, y2) and torch.equal(h_last, h2)
        if not gradient:
            return
        ref.backward(host(self.dy), host(self.dh))
        dx, dgate, dh0 = self.backward(saved)
        check(host(dx), ref.dx, ref.dx_err, "f32" if self.src == "u8" else self.src, "dx")
        check(host(dh0), ref.dh0, ref.dh0_err, "f32", "dh0")
        if self.gate is None:
            assert dgate is None
        else:
            kind = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}[dgate.dtype]
            check(host(dgate), ref.dgate, ref.dgate_err, kind, "dgate")
        for a, b in zip((dx, dgate, dh0), self.backward(saved)):  # results repeat
            assert a is b or torch.equal(a, b)


SIZES = [(1, 1, 1), (1, 2, 3), (2, 15, 64), (3, 16, 65), (2, 17, 33), (5, 25, 1000), (1, 127, 2), (2, 128, 128),
         (1, 129, 66), (3, 300, 40), (1, 2049, 64), (2, 4097, 34), (1, 5000, 7), (300, 3, 10), (1, 1000, 300)]


@pytest.mark.parametrize("b,t,c", SIZES)
@pytest.mark.parametrize("src,gate,gate_type,out,logit,complement", [
    ("f32", "channel", "f32", "f32", False, False),
    ("f32", "step", "f32", "f32", True, True),
    ("bf16", "step", "bf16", "bf16", True, True),
    ("bf16", "step", "f32", "f32", False, True),
    ("f16", "step", "f16", "f16", False, False),
    ("f16", "sequence", "f32", "f32", True, False),
    ("u8", "channel", "f32", "f32", True, True),
    ("u8", "step", "f32", "f32", False, False),
])
def test_scan_and_gradient_match_definition(b, t, c, src, gate, gate_type, out, logit, complement):
    Problem(b, t, c, src, gate, gate_type, out, logit, complement, scale=0.75, seed=1).verify()


@pytest.mark.parametrize("src,gate,gate_type,out", [
    ("bf16", "step", "f32", "bf16"), ("bf16", "step", "bf16", "f32"), ("bf16", "channel", "f32", "bf16"),
    ("bf16", "none", "f32", "f32"), ("f16", "step", "f32", "f16"), ("f16", "step", "f16", "f32"),
    ("f16", "step", "f32", "f32"), ("f16", "channel", "f32", "f16"), ("f32", "none", "f32", "f32"),
    ("u8", "none", "f32", "f32"), ("f32", "sequence", "f32", "f32"), ("u8", "sequence", "f32", "f32")])
@pytest.mark.parametrize("time_major", [False, True])
def test_every_listed_type(src, gate, gate_type, out, time_major):
    for b, t, c in ((3, 37, 70), (2, 290, 96), (2, 50, 51)):
        Problem(b, t, c, src, gate, gate_type, out, gate != "none", True, time_major=time_major, seed=2).verify()


@pytest.mark.parametrize("gate,logit", [("channel", True), ("sequence", False), ("step", True), ("none", False)])
@pytest.mark.parametrize("src", ["f32", "bf16", "u8"])
def test_uneven_lengths(src, gate, logit):
    """Lengths of zero, one, block borders and all steps; what lies behind them is NaN and not read."""
    lengths = [0, 1, 15, 16, 17, 127, 128, 129, 200, 300, 1000]
    Problem(len(lengths), 300, 40, src, gate, "f32", None, logit, True, lengths=lengths, seed=3).verify()
    Problem(3, 20, 66, src, gate, "f32", None, logit, False, lengths=[0, 20, 7], time_major=True, seed=4).verify()
    Problem(2, 5000, 34, src, gate, "f32", None, logit, False, lengths=[4000, 2048], seed=5).verify()


@pytest.mark.parametrize("src,gate,gate_type,out", [("bf16", "step", "bf16", "bf16"), ("f32", "step", "f32", "f32"),
                                                    ("bf16", "step", "f32", "f32"), ("f16", "channel", "f32", "f16"),
                                                    ("u8", "channel", "f32", "f32"), ("u8", "step", "f32", "f32")])
@pytest.mark.parametrize("b,t,c,lengths", [(3, 300, 1500, None), (4, 129, 1026, [129, 0, 128, 57]), (70, 135, 61, None)])
def test_columns_in_the_hundreds(b, t, c, lengths, src, gate, gate_type, out):
    """Enough channels for whole rows of CTAs, too few for a warp each."""
    Problem(b, t, c, src, gate, gate_type, out, True, True, 0.5, lengths, seed=18).verify()


def test_many_sequences_take_the_same_values():
    """How the work is split does not show: rows of a large batch against a small one."""
    p = Problem(2000, 25, 130, "u8", "channel", time_major=True, seed=6)
    y, _ = p.forward()
    ref = p.reference()
    check(host(y), ref.y, ref.y_err, "f32", "y")


@pytest.mark.parametrize("t", [1, 40, 1500])
def test_gates_expanded_over_sequences_or_steps(t):
    """An expanded gate is read where it is; its gradient has an element for each of its own."""
    Problem(3, t, 50, "bf16", "shared", "bf16", None, True, True, seed=7).verify()
    for shape in ((3, 1, 50), (1, 1, 50)):
        p = Problem(3, t, 50, "f32", "step", logit=True, seed=7)
        p.gate = p.leak(True, *shape).cuda().expand(3, t, 50)
        p.verify()
    p = Problem(3, t, 50, "f32", "sequence", logit=True, seed=7)
    p.gate = p.leak(True, 1, 50).cuda().expand(3, 50)
    p.verify()


def test_dependent_calls_without_a_wait():
    """Kernels that start while their predecessors end still wait for what those
    write: a chain of calls, each on the last one's results, against the same
    chain with a wait after every call."""
    g = torch.Generator().manual_seed(3)
    w = [sb.mx4_quantize(torch.randn(256, 256, generator=g).cuda() / 16) for _ in range(2)]
    z = torch.randn(2, 300, 256, generator=g).cuda()
    start = torch.randn(2, 300, 256, generator=g).cuda()

    def chain(wait):
        x, pool = start, torch.zeros(2, 256, device="cuda")
        for i in range(6):
            for f in (lambda: sb.mx4_linear(x, w[i % 2]), lambda: sb.leaky_scan(x, z, logit=True, complement=True)[0],
                      lambda: sb.mx4_dequantize(sb.mx4_quantize(x.view(-1, 256))).view(2, 300, 256),
                      lambda: sb.mx4_linear(x[:, :7], w[0])):
                out = f()
                if wait:
                    torch.cuda.synchronize()
                if out.shape == x.shape:
                    x = out
            y, last, saved = sb.leaky_scan(x, z, logit=True, save=True)
            x, dz, _ = sb.leaky_scan_backward(y, x, z, saved, logit=True)
            x = x / x.abs().amax()
            sb.leaky_step(out[:, 0], None, pool, decay=0.5)
            if wait:
                torch.cuda.synchronize()
        return x, dz, pool

    want = chain(True)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(chain(False), want))


def test_extreme_gates_and_inputs():
    """Gates of zero, one and minus one half, logits of the type's largest
    magnitude, infinite inputs: each stays in its channel and its later steps."""
    p = Problem(1, 400, 8, "f32", "step", seed=8)
    p.gate[0, :, 0], p.gate[0, :, 1], p.gate[0, :, 2] = 0.0, 1.0, -0.5
    p.verify()
    q = Problem(1, 400, 8, "f32", "step", "f32", None, True, True, seed=9)
    top = torch.finfo(torch.float32).max
    q.gate[0, :, 0], q.gate[0, :, 1], q.gate[0, ::2, 2] = top, -top, float("-inf")
    q.gate[0, ::3, 3] = float("inf")
    q.verify()
    clean, _ = q.forward()
    q.x[0, 137, 5] = float("inf")
    q.x[0, 200, 6] = float("nan")
    y, _ = q.forward()
    hit = torch.zeros_like(y, dtype=torch.bool)
    hit[0, 137:, 5], hit[0, 200:, 6] = True, True
    assert torch.equal(y[~hit], clean[~hit])
    assert not torch.isfinite(y[0, 137, 5]) and torch.isnan(y[0, 200:, 6]).all()


def test_long_sequences_keep_their_accuracy():
    p = Problem(1, 70001, 5, "f32", "channel", seed=10)
    p.verify()
    Problem(1, 33000, 3, "bf16", "step", "bf16", None, True, True, seed=11).verify()
    Problem(1, 40000, 64, "bf16", "step", "bf16", None, True, True, seed=15).verify()
    Problem(2, 17000, 48, "f32", "step", "f32", None, False, True, lengths=[17000, 9000], seed=16).verify()
    Problem(1, 35000, 80, "u8", "channel", "f32", None, False, False, seed=17).verify()


def test_gradient_against_differences():
    """Central differences of the definition in 64 bits, in every direction of a small problem."""
    p = Problem(2, 19, 3, "f32", "step", "f32", None, True, True, scale=0.5, seed=12)
    _, _, saved = p.forward(save=True)
    dx, dgate, dh0 = p.backward(saved)
    x, z, h0 = host(p.x), host(p.gate), host(p.h0)

    def loss(x, z, h0):
        r = LeakyRef(x, z, None, h0, None, True, True, 0.5)
        return (r.y * host(p.dy)).sum() + (r.h_last * host(p.dh)).sum()

    eps = 2.0 ** -12  # its third-order term is below 2^-24 of values that are of order one
    for array, got, put in ((x, dx, 0), (z, dgate, 1), (h0, dh0, 2)):
        got = host(got)
        for at in np.ndindex(array.shape):
            args = [x, z, h0]
            up, down = array.copy(), array.copy()
            up[at] += eps
            down[at] -= eps
            args[put] = up
            hi = loss(*args)
            args[put] = down
            lo = loss(*args)
            assert abs((hi - lo) / (2 * eps) - got[at]) < 1e-5 * (1 + abs(got[at])), (put, at)


def test_rows_inside_wider_arrays():
    """Channels cut out of wider rows, at an odd offset: nothing beside them is touched."""
    b, t, c, w = 2, 140, 33, 61
    g = torch.Generator().manual_seed(1)
    x = torch.randn(b, t, w, generator=g).to(torch.bfloat16).cuda()
    z = torch.randn(b, t, w, generator=g).cuda()
    y = torch.full((b, t, w), 9.0, dtype=torch.bfloat16, device="cuda")
    xs, zs, ys = x[..., 5:5 + c], z[..., 3:3 + c], y[..., 7:7 + c]
    want, last = sb.leaky_scan(xs.contiguous(), zs.contiguous(), logit=True)
    got, last2 = sb.leaky_scan(xs, zs, logit=True)
    assert torch.equal(got, want) and torch.equal(last, last2)
    q = sb.Leaky(b, t, c, 2, 0, 2, 1, 0, 0.0, 1.0, t * w, w, t * w, w, t * w, w)
    L = sb.lib()
    import ctypes as C
    need = L.snn_b200_leaky_workspace(C.byref(q), 0)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    st = L.snn_b200_leaky_scan_async(0, torch.cuda.current_stream().cuda_stream, C.byref(q), xs.data_ptr(),
                                     zs.data_ptr(), None, None, ys.data_ptr(), None, None, ws.data_ptr(), need)
    assert st == sb.SNN_OK
    assert torch.equal(ys, want)
    assert (y[..., :7] == 9).all() and (y[..., 7 + c:] == 9).all()


def test_empty_sequences():
    x = torch.empty(2, 0, 3, device="cuda")
    h0 = torch.arange(6.0, device="cuda").view(2, 3)
    y, last, saved = sb.leaky_scan(x, decay=0.5, h0=h0, save=True)
    assert y.shape == (2, 0, 3) and torch.equal(last, h0)
    _, last = sb.leaky_scan(x, decay=0.5)
    assert not last.any()
    gate = torch.full((3,), 0.5, device="cuda")
    dx, dgate, dh0 = sb.leaky_scan_backward(x, x, gate, saved, dh_last=h0)
    assert not dgate.any() and torch.equal(dh0, h0)
    none = torch.empty(0, 4, 3, device="cuda")
    y, last, saved = sb.leaky_scan(none, gate, save=True)
    assert y.shape == (0, 4, 3)
    _, dgate, _ = sb.leaky_scan_backward(none, none, gate, saved)
    assert not dgate.any()
    assert sb.leaky_scan(torch.empty(2, 4, 0, device="cuda"), decay=0.5)[0].shape == (2, 4, 0)


@pytest.mark.parametrize("b,t,c", [(4, 20, 100), (1, 3000, 64)])
def test_replayed_and_on_other_streams(b, t, c):
    p = Problem(b, t, c, "bf16", "step", "bf16", None, True, True, seed=13)
    y, last, saved = p.forward(save=True)
    want = [y, last, *p.backward(saved)]
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(6):
        for s in side:  # two calls at once, each with its own workspace
            with torch.cuda.stream(s):
                y, last, saved = p.forward(save=True)
                got.append([y, last, *p.backward(saved)])
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, last, saved = p.forward(save=True)
        outs = [y, last, *p.backward(saved)]
    for seed in (1, 2):
        p.x.copy_(torch.randn(p.x.shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        y, last, saved = p.forward(save=True)
        assert all(torch.equal(a, b) for a, b in zip(outs, [y, last, *p.backward(saved)]))


# ---------------------------------------------------------------------------
# Single step
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("src,gate_type,out", [("f32", "f32", "f32"), ("u8", "f32", "f32"), ("bf16", "bf16", "bf16"),
                                               ("bf16", "f32", "f32"), ("f16", "f16", "f32"), ("f16", "f32", "f16")])
@pytest.mark.parametrize("gate", ["channel", "row", "none"])
@pytest.mark.parametrize("b,c,slots", [(1, 1, 1), (1, 1000, 4), (7, 33, 7), (65, 130, 200), (300, 1000, 301)])
def test_step_matches_definition(b, c, slots, gate, src, gate_type, out):
    if gate == "channel" and gate_type != "f32":
        gate_type = "f32"
    p = Problem(b, 1, c, src, "none", seed=b)
    x = p.x[:, 0]
    z = None if gate == "none" else p.leak(True, *((c,) if gate == "channel" else (b, c))).to(TYPES[gate_type]).cuda()
    pool = torch.randn(slots, c, generator=p.g).cuda()
    at = torch.randperm(slots, generator=p.g)[:b].to(torch.int32).cuda()
    old = pool.clone()
    how = dict(decay=0.9) if z is None else dict(logit=True)
    y = sb.leaky_step(x, z, pool, slots=at, complement=True, input_scale=0.5, dtype=TYPES[out], **how)
    ref = LeakyRef((host(x) != 0 if src == "u8" else host(x))[:, None],
                   None if z is None else host(z) if gate == "channel" else host(z)[:, None], how.get("decay"),
                   host(old[at.long()]), None, z is not None, True, 0.5)
    check(host(y), ref.y[:, 0], ref.y_err[:, 0], out, "y")
    check(host(pool[at.long()]), ref.h_last, ref.h_last_err, "f32", "pool")
    rest = torch.ones(slots, dtype=torch.bool, device="cuda")
    rest[at.long()] = False
    assert torch.equal(pool[rest], old[rest])
    # Without slots, rows are the pool's first.
    pool.copy_(old)
    y2 = sb.leaky_step(x, z, pool, complement=True, input_scale=0.5, dtype=TYPES[out], **how)
    other = old.clone()
    idx = torch.arange(b, dtype=torch.int32, device="cuda")
    y3 = sb.leaky_step(x, z, other, slots=idx, complement=True, input_scale=0.5, dtype=TYPES[out], **how)
    assert torch.equal(y2, y3) and torch.equal(pool, other) and torch.equal(pool[b:], old[b:])


def test_step_padding_and_repeated_slots():
    """Slots outside the pool are padding; a slot named again takes its rows in order."""
    c = 70
    g = torch.Generator().manual_seed(2)
    pool = torch.randn(5, c, generator=g).cuda()
    slots = [3, -1, 0, 3, 5, 2, 3, -2 ** 31, 2 ** 31 - 1, 5, -1, 2 ** 31 - 1]
    x = torch.randn(len(slots), c, generator=g).cuda()
    want_pool, want = pool.clone(), torch.zeros(len(slots), c, device="cuda")
    torch.full((64, 1024), 7.0, device="cuda")  # what a row that is not written might show
    for i, s in enumerate(slots):
        if 0 <= s < 5:
            row = want_pool[s:s + 1].clone()
            want[i] = sb.leaky_step(x[i:i + 1], None, row, decay=0.75)[0]
            want_pool[s] = row[0]
    y = sb.leaky_step(x, None, pool, slots=torch.tensor(slots, dtype=torch.int32, device="cuda"), decay=0.75)
    assert torch.equal(y, want) and torch.equal(pool, want_pool)


@pytest.mark.parametrize("b", [700, 3000])
def test_step_of_many_rows_with_repeated_slots(b):
    """Enough rows for several to a CTA, some slots named many times, some rows padding."""
    c, count = 36, 500
    g = torch.Generator().manual_seed(b)
    pool = torch.randn(count, c, generator=g).cuda()
    x = torch.randn(b, c, generator=g).cuda()
    slots = torch.randint(-20, count + 20, (b,), generator=g).to(torch.int32)
    state, want = pool.cpu().clone(), torch.zeros(b, c)
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < count:  # 0.75 h is exact, so the sum is the fused one
            state[s] = 0.75 * state[s].double() + x[i].cpu().double()
            want[i] = state[s]
    y = sb.leaky_step(x, None, pool, slots=slots.cuda(), decay=0.75)
    assert torch.equal(y.cpu(), want) and torch.equal(pool.cpu(), state)


def test_steps_continue_a_scan():
    """A prompt through the scan, then single steps, against one scan of it all."""
    p = Problem(6, 50, 90, "f32", "step", "f32", None, True, True, seed=14)
    ref = p.reference()
    y, state = sb.leaky_scan(p.x[:, :40], p.gate[:, :40], h0=p.h0, logit=True, complement=True)
    check(host(y), ref.y[:, :40], ref.y_err[:, :40], "f32", "prompt")
    pool = torch.zeros(8, 90, device="cuda")
    slots = torch.tensor([7, 1, 3, 0, 2, 5], dtype=torch.int32, device="cuda")
    pool[slots.long()] = state
    for t in range(40, 50):
        y = sb.leaky_step(p.x[:, t], p.gate[:, t], pool, slots=slots, logit=True, complement=True)
        check(host(y), ref.y[:, t], ref.y_err[:, t], "f32", "step")
