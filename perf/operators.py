"""Cases that time the sequence operators of snn_b200: the microscaled 4-bit
weights with their product, and the leaky (gated linear) recurrence with its
gradient and its single step.

``run`` computes an operator in its plain form (elementary torch operations in
32 bits, rounded once at the end), or, where ``own`` is true, makes the calls a
user makes of the library. ``exact`` gives the same outputs from the operator's
definition in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"u8": torch.uint8, "f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"u8": 1, "f16": 2, "bf16": 2, "f32": 4}
BLOCK = 32        # elements that share one scale
MX_BYTES = 17 / 32  # a byte of scale for each block, half a byte for each element


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _pack(name, rows, cols, src, transposed):
    return {"name": name, "kind": "pack", "rows": rows, "cols": cols, "src": src, "transposed": transposed}


def _linear(name, m, k, n, src, out, bias):
    return {"name": name, "kind": "linear", "m": m, "k": k, "n": n, "src": src, "out": out, "bias": bias}


def _leaky(name, kind, batch, steps, channels, src, gate, gate_type, logit, complement, ragged, time_major):
    return {"name": name, "kind": kind, "batch": batch, "steps": steps, "channels": channels, "src": src,
            "gate": gate, "gate_type": gate_type, "logit": logit, "complement": complement, "ragged": ragged,
            "time_major": time_major}


def _step(name, batch, slots, channels, src, gate, gate_type, logit, complement):
    return {"name": name, "kind": "step", "batch": batch, "slots": slots, "channels": channels, "src": src,
            "gate": gate, "gate_type": gate_type, "logit": logit, "complement": complement}


def listed():
    return [
        # The first layer of the 784-1000-10 network, stored one row per presynaptic neuron, packed along them.
        _pack("pack_784x1000", 1000, 784, "f32", True),
        # A large layer's weights, packed once when they are loaded.
        _pack("pack_16384x8192", 16384, 8192, "bf16", False),
        # One sample's spikes of one step through the first layer.
        _linear("linear_1x784x1000", 1, 784, 1000, "u8", "f32", False),
        # A whole raster, 25 steps of 2,000 samples, through the first layer.
        _linear("linear_50000x784x1000", 50000, 784, 1000, "u8", "f32", False),
        # A few activations through a large layer: the weights' bytes count.
        _linear("linear_4x8192x8192", 4, 8192, 8192, "bf16", "bf16", True),
        # Many activations through the same layer: the matrix units count.
        _linear("linear_8192x8192x8192", 8192, 8192, 8192, "bf16", "bf16", True),
        # Leaky traces of the hidden layer's raster, one decay per neuron.
        _leaky("scan_2000x25x1000", "scan", 2000, 25, 1000, "u8", "channel", "f32", False, False, False, True),
        # One long sequence with a gate for every step.
        _leaky("scan_1x65536x1024", "scan", 1, 65536, 1024, "bf16", "step", "bf16", True, True, False, False),
        # Training learned leaks over short sequences of uneven lengths: forward and backward.
        _leaky("train_256x100x1000", "train", 256, 100, 1000, "f32", "channel", "f32", True, False, True, False),
        # Training a gated layer over long sequences: forward and backward.
        _leaky("train_4x8192x2048", "train", 4, 8192, 2048, "bf16", "step", "bf16", True, True, False, False),
        # One step of one sample.
        _step("step_1x1000", 1, 1, 1000, "f32", "channel", "f32", False, False),
        # One step of many samples whose states sit in a pool.
        _step("step_2000x1000", 2000, 4096, 1000, "bf16", "step", "bf16", True, True),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm, odd or even by chance."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["pack", "linear", "linear", "scan", "scan", "train", "train", "step"])
    if kind == "pack":
        rows, cols = _log(rng, 1, 16384), _log(rng, 1, 8192)
        return {k: v for k, v in _pack("", rows, cols, rng.choice(["u8", "f16", "bf16", "f32"]),
                                       rng.random() < 0.5).items() if k != "name"}
    if kind == "linear":
        k, n = _log(rng, 1, 8192), _log(rng, 1, 8192)
        m = _log(rng, 1, max(1, min(50000, 8192 ** 3 // (k * n))))
        m = min(m, (1 << 26) // n, (1 << 27) // k)  # outputs and inputs within the listed ones
        src = rng.choice(["u8", "f16", "bf16", "f32"])
        out = rng.choice(["f32", "bf16"] if src == "u8" else ["f32", src])
        return {k_: v for k_, v in _linear("", max(m, 1), k, n, src, out, rng.random() < 0.5).items()
                if k_ != "name"}
    src = rng.choice(["f16", "bf16", "f32"] if kind in ("train", "step") else ["u8", "f16", "bf16", "f32"])
    gate = rng.choice(["channel", "step"])
    gate_type = "f32" if gate == "channel" or src == "u8" else rng.choice(["f32", src])
    logit = rng.random() < 0.5
    complement = rng.random() < 0.5
    channels = _log(rng, 1, 4096)
    if kind == "step":
        batch = _log(rng, 1, 4096)
        slots = batch + rng.randrange(0, 2048)
        case = _step("", batch, slots, channels, src, gate, gate_type, logit, complement)
    else:
        steps = _log(rng, 1, 65536 if kind == "scan" else 8192)
        batch = _log(rng, 1, max(1, min(2048, (1 << 26) // (steps * channels))))
        case = _leaky("", kind, batch, steps, channels, src, gate, gate_type, logit, complement,
                      steps <= 8192 and rng.random() < 0.4, rng.random() < 0.4)
    return {k: v for k, v in case.items() if k != "name"}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _inputs(case, seed):
    """The tensors of a case, on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    def uniform(*shape):
        return torch.rand(*shape, device="cuda", generator=g)

    def signal(*shape):  # spikes that one neuron in eight fires, or activations
        if case["src"] == "u8":
            return (uniform(*shape) < 0.125).to(torch.uint8)
        return normal(*shape).to(DTYPES[case["src"]])

    kind = case["kind"]
    if kind == "pack":
        r, c = case["rows"], case["cols"]
        x = signal(*((c, r) if case["transposed"] else (r, c)))
        if case["src"] != "u8":
            x.mul_(1.0 / math.sqrt(c))
        return {"x": x.t() if case["transposed"] else x}
    if kind == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        s = {"x": signal(m, k), "weights": normal(n, k).mul_(1.0 / math.sqrt(k))}
        s["bias"] = normal(n).mul_(0.1) if case["bias"] else None
        return s
    c, b = case["channels"], case["batch"]

    def leak(*shape):  # decays of 5 to 200 steps, or their logits
        if case["logit"]:
            return normal(*shape).mul_(1.5).add_(2.0).to(DTYPES[case["gate_type"]])
        tau = torch.exp(math.log(5.0) + uniform(*shape) * math.log(40.0))
        return torch.exp(-1.0 / tau).to(DTYPES[case["gate_type"]])

    if kind == "step":
        return {"x": signal(b, c), "gate": leak(c) if case["gate"] == "channel" else leak(b, c),
                "pool": normal(case["slots"], c),
                "slots": torch.randperm(case["slots"], device="cuda", generator=g)[:b].to(torch.int32)}
    t = case["steps"]

    def sequence(make):  # [batch, steps, channels], stored with the steps first where time_major
        return make(t, b, c).transpose(0, 1) if case["time_major"] else make(b, t, c)

    s = {"x": sequence(signal), "gate": leak(c) if case["gate"] == "channel" else sequence(leak), "h0": normal(b, c)}
    s["lengths"] = None
    if case["ragged"]:
        n = (uniform(b) * (t + 1)).to(torch.int32).clamp_(max=t)
        n[0] = t
        s["lengths"] = n
    if kind == "train":
        s["dy"] = sequence(lambda *shape: normal(*shape).to(DTYPES[case["src"]]))
        s["dh_last"] = normal(b, c)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["kind"] == "linear":
        weights = s.pop("weights")  # a program keeps the packed weights only
        if own:
            import snn_b200 as sb
            s["packed"] = sb.mx4_quantize(weights)
        else:
            s["values"] = _quantized(weights)
    return s


# ---------------------------------------------------------------------------
# Plain forms, in 32 bits
# ---------------------------------------------------------------------------
def _power(e):
    """2^e, put together from its bits: torch.ldexp's power is off by a rounding on some devices, which moves ties."""
    return ((e.long() + 1023) << 52).view(torch.float64).float()


def _quantized(x):
    """The values that MXFP4 keeps of the rows of x: blocks of 32, each with the
    scale 2^(floor(log2(largest magnitude)) - 2), elements rounded to the nearest
    of 0, .5, 1, 1.5, 2, 3, 4, 6 (ties to the even code), larger ones to 6."""
    rows, cols = x.shape
    x = x.float()
    pad = -cols % BLOCK
    if pad:
        x = torch.cat([x, x.new_zeros(rows, pad)], 1)
    x = x.reshape(rows, -1, BLOCK)
    top = x.abs().amax(2, keepdim=True)
    e = torch.where(top > 0, torch.frexp(top)[1] - 3, -127).clamp(min=-127)
    q = x * _power(-e)
    m = q.abs()
    m = torch.where(m < 2, torch.round(m * 2) / 2, torch.where(m < 4, torch.round(m), torch.round(m / 2) * 2))
    q = torch.copysign(m.clamp(max=6), q)
    return (q * _power(e)).reshape(rows, -1)[:, :cols]


def _gates(z, logit):
    """The gate and its complement in 32 bits; each from its own exponential, as 1 - gate would lose its small values."""
    z = z.float()
    if not logit:
        return z, 1 - z
    return 1 / (1 + torch.exp(-z)), 1 / (1 + torch.exp(z))


def _steps_first(x):
    return x.transpose(0, 1).float() if x.dim() == 3 else x.float()


def _out_type(case):
    return torch.float32 if case["src"] == "u8" else DTYPES[case["src"]]


def _plain_scan(s):
    """h_t = a_t h_{t-1} + u_t over [steps, batch, channels], every h kept."""
    case = s["case"]
    a, rest = _gates(_steps_first(s["gate"]), case["logit"])
    u = _steps_first(s["x"])
    if case["complement"]:
        u = u * rest
    h, t = s["h0"], case["steps"]
    every = a.dim() == 3
    kept = torch.empty(t, case["batch"], case["channels"], device="cuda")
    for i in range(t):
        new = torch.addcmul(u[i], a[i] if every else a, h, out=kept[i])
        if s["lengths"] is not None:
            new.copy_(torch.where((s["lengths"] > i)[:, None], new, h))
        h = new
    return a, rest, kept


def _live(s):
    """[steps, batch, 1]: which rows lie within their sequence."""
    return (torch.arange(s["case"]["steps"], device="cuda")[:, None] < s["lengths"])[..., None]


def _plain_train(s):
    case = s["case"]
    a, rest, kept = _plain_scan(s)
    dy, t = _steps_first(s["dy"]), case["steps"]
    every = a.dim() == 3
    delta, e = torch.empty_like(kept), s["dh_last"]
    for i in range(t - 1, -1, -1):
        d = dy[i] + e
        back = (a[i] if every else a) * d
        if s["lengths"] is not None:
            live = (s["lengths"] > i)[:, None]
            d, back = torch.where(live, d, 0.0), torch.where(live, back, e)
        delta[i], e = d, back
    before = torch.cat([s["h0"][None], kept[:-1]])
    x = _steps_first(s["x"])
    dx = delta * rest if case["complement"] else delta
    dgate = delta * ((before - x) if case["complement"] else before)
    if not every:
        dgate = dgate.sum((0, 1), dtype=torch.float64)
    if case["logit"]:
        dgate = dgate * (a * rest)
    y = kept if s["lengths"] is None else torch.where(_live(s), kept, 0.0)
    kind = DTYPES[case["src"]]
    dgate = dgate.transpose(0, 1).to(DTYPES[case["gate_type"]]) if every else dgate.float()
    return {"y": y.transpose(0, 1).to(kind), "h_last": kept[-1].clone(), "dx": dx.transpose(0, 1).to(kind),
            "dgate": dgate, "dh0": e}


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "pack":
        x = s["x"] if case["src"] != "u8" else s["x"] != 0
        return _quantized(x).to(torch.bfloat16)
    if kind == "linear":
        y = _quantized(s["x"]) @ s["values"].t()
        return (y if s["bias"] is None else y + s["bias"]).to(DTYPES[case["out"]])
    if kind == "step":
        a, rest = _gates(s["gate"], case["logit"])
        u = s["x"].float()
        if case["complement"]:
            u = u * rest
        at = s["slots"].long()
        h = torch.addcmul(u, a, s["pool"][at])
        s["pool"][at] = h
        return {"y": h.to(_out_type(case)), "pool": s["pool"]}
    if kind == "scan":
        _, _, kept = _plain_scan(s)
        y = kept if s["lengths"] is None else torch.where(_live(s), kept, 0.0)
        return {"y": y.transpose(0, 1).to(_out_type(case)), "h_last": kept[-1].clone()}
    return _plain_train(s)


# ---------------------------------------------------------------------------
# The library's calls
# ---------------------------------------------------------------------------
def _own(s):
    import snn_b200 as sb
    case = s["case"]
    kind = case["kind"]
    if kind == "pack":
        return sb.mx4_dequantize(sb.mx4_quantize(s["x"]), dtype=torch.bfloat16)
    if kind == "linear":
        return sb.mx4_linear(s["x"], s["packed"], bias=s["bias"], dtype=DTYPES[case["out"]])
    how = {"logit": case["logit"], "complement": case["complement"]}
    if kind == "step":
        return {"y": sb.leaky_step(s["x"], s["gate"], s["pool"], slots=s["slots"], **how), "pool": s["pool"]}
    how.update(h0=s["h0"], lengths=s["lengths"])
    if kind == "scan":
        y, h_last = sb.leaky_scan(s["x"], s["gate"], **how)
        return {"y": y, "h_last": h_last}
    y, h_last, saved = sb.leaky_scan(s["x"], s["gate"], save=True, **how)
    dx, dgate, dh0 = sb.leaky_scan_backward(s["dy"], s["x"], s["gate"], saved, dh_last=s["dh_last"],
                                            logit=case["logit"], complement=case["complement"],
                                            lengths=s["lengths"])
    return {"y": y, "h_last": h_last, "dx": dx, "dgate": dgate, "dh0": dh0}


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# Work
# ---------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "pack":  # read, keep packed, read back, written as 16-bit values
        size = case["rows"] * case["cols"]
        return {"bytes": size * (BYTES[case["src"]] + 2 * MX_BYTES + 2), "flops": 4 * size}
    if kind == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": m * k * BYTES[case["src"]] + n * k * MX_BYTES + m * n * BYTES[case["out"]] +
                (4 * n if case["bias"] else 0), "flops": 2 * m * k * n}
    b, c = case["batch"], case["channels"]
    rows = b if kind == "step" else b * case["steps"]
    size = rows * c
    x, g = BYTES[case["src"]], BYTES[case["gate_type"]]
    y = 4 if case["src"] == "u8" else x
    gate = c * g if case["gate"] == "channel" else size * g
    ends = 2 * 4 * b * c  # the state before and after
    flops = (2 + 2 * case["complement"] + (4 * case["logit"] if case["gate"] == "step" else 0)) * size
    if kind != "train":
        return {"bytes": size * (x + y) + gate + ends, "flops": flops}
    # forward, then backward: x, gate and dy read, dx and the gate's gradient written
    return {"bytes": size * (x + y) + gate + ends + size * (2 * x + y) + 2 * gate + ends, "flops": 4 * flops}


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------
def _quantized64(x):
    rows, cols = x.shape
    x = torch.nn.functional.pad(x.double(), (0, -cols % BLOCK)).unflatten(1, (-1, BLOCK))
    bits = x.abs().amax(2, keepdim=True).view(torch.int64)
    e = ((bits >> 52) - 1023 - 2).clamp(min=-127)  # of normal numbers in 64 bits, or of zero
    powers = torch.tensor([math.ldexp(1.0, i) for i in range(-127, 128)], dtype=torch.float64, device=x.device)
    scale = powers[e + 127]
    m = x.abs() / scale
    code = torch.zeros_like(m, dtype=torch.int64)
    # Borders between neighbours; one that lies between an odd code and the even one above goes up.
    for border, up in ((0.25, 0), (0.75, 1), (1.25, 0), (1.75, 1), (2.5, 0), (3.5, 1), (5.0, 0)):
        code += (m >= border) if up else (m > border)
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    return (torch.where(x < 0, -grid[code], grid[code]) * scale).flatten(1)[:, :cols]


def _scan64(a, u):
    """All h_t = a_t h_{t-1} + u_t, from h_{-1} = 0, by doubling the span that each row covers."""
    span = 1
    while span < a.shape[0]:
        u = torch.cat([u[:span], u[span:] + a[span:] * u[:-span]])
        a = torch.cat([a[:span], a[span:] * a[:-span]])
        span *= 2
    return u


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "pack":
        return _quantized64(s["x"])
    if kind == "linear":
        y = _quantized64(s["x"]) @ _quantized64(s["weights"]).T
        return y if s["bias"] is None else y + s["bias"].double()
    z = s["gate"].double()
    a = torch.sigmoid(z) if case["logit"] else z
    rest = torch.sigmoid(-z) if case["logit"] else 1.0 - z
    x = s["x"].double()
    u = x * rest if case["complement"] else x
    if kind == "step":
        at = s["slots"].long()
        pool = s["pool"].double()
        h = a * pool[at] + u
        pool[at] = h
        return {"y": h, "pool": pool}
    b, t, c = u.shape
    live = torch.ones(b, t, 1, dtype=torch.bool, device="cuda")
    if s["lengths"] is not None:
        live = (torch.arange(t, device="cuda") < s["lengths"][:, None])[..., None]
    # A row behind its sequence keeps the state: gate one, input zero.
    aa = torch.where(live, a.expand(b, t, c), 1.0).transpose(0, 1)
    uu = torch.where(live, u, 0.0).transpose(0, 1).clone()
    uu[0] += aa[0] * s["h0"].double()
    h = _scan64(aa, uu)
    del uu
    mask = live.transpose(0, 1)
    if kind == "scan":
        return {"y": torch.where(mask, h, 0.0).transpose(0, 1), "h_last": h[-1].clone()}
    g = torch.where(mask, s["dy"].double().transpose(0, 1), 0.0)
    g[-1] += s["dh_last"].double()
    after = torch.cat([aa[1:], torch.ones_like(aa[:1])])
    delta = _scan64(after.flip(0), g.flip(0)).flip(0)
    del g, after
    dh0 = aa[0] * delta[0]
    delta = torch.where(mask, delta, 0.0)
    before = torch.cat([s["h0"].double()[None], h[:-1]])
    if case["complement"]:
        before = before - torch.where(mask, x.transpose(0, 1), 0.0)
    dgate = (delta * before).transpose(0, 1)
    del before
    dgate = dgate.sum((0, 1)) if case["gate"] == "channel" else dgate
    if case["logit"]:
        dgate = dgate * a * rest
    dx = delta.transpose(0, 1)
    if case["complement"]:
        dx = dx * rest
    return {"y": torch.where(mask, h, 0.0).transpose(0, 1), "h_last": h[-1].clone(), "dx": dx, "dgate": dgate,
            "dh0": dh0}
