"""The sequence operators from their definitions, in 64 bits with numpy, with
bounds on what 32-bit arithmetic may lose beside them."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
# Half a step of each output type, relative.
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
# Per step of the recurrence: the gate (exponential 2, sum and product 1/2
# each, quotient 2 units of 2^-23), the input's two products and the fused
# update together stay below 2^-20 of the magnitudes they combine.
STEP = 2.0 ** -20
# A rounding to 32 bits is off by half a unit of the result, that is by a share
# of 2^-24 of it, but never by less than half of the smallest subnormal, 2^-150,
# where the result is subnormal. A step has at most four roundings that reach its
# state (two of the input's products, one each of a product and a sum).
TINY = 4 * 2.0 ** -150


def mx4_parts(x):
    """(codes, scale bytes) of the rows of x, padded to whole blocks."""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    nb = -(-cols // 32)
    v = np.zeros((rows, nb * 32))
    v[:, :cols] = x
    v = v.reshape(rows, nb, 32)
    top = np.abs(v).max(2)
    bad = ~np.isfinite(v).all(2)
    e = np.full(top.shape, -127, np.int64)
    ok = (top > 0) & ~bad
    e[ok] = np.maximum(np.frexp(top[ok])[1] - 1 - 2, -127)
    with np.errstate(invalid="ignore"):
        m = np.abs(np.ldexp(np.where(bad[..., None], 0.0, v), -e[..., None]))
    # Nearest of the grid; of two equally near ones the even code.
    d = np.abs(m[..., None] - GRID)
    best = d.min(-1, keepdims=True)
    tied = d == best
    even = tied & (np.arange(8) % 2 == 0)
    codes = np.where(even.any(-1), even.argmax(-1), tied.argmax(-1))
    codes = np.where(m > 6, 7, codes) | (np.signbit(v) & ~bad[..., None]) * 8
    return codes.reshape(rows, nb * 32), np.where(bad, 255, e + 127)


def mx4_values(x):
    codes, s = mx4_parts(x)
    rows, cols = np.asarray(x).shape
    v = np.where(codes & 8, -1.0, 1.0) * GRID[codes & 7]
    v = v.reshape(rows, -1, 32) * np.ldexp(1.0, s - 127)[..., None]
    v[s == 255] = np.nan
    return v.reshape(rows, -1)[:, :cols]


def scale_offsets(rows, cols):
    """Byte of (row, block) in the scale array."""
    nb = -(-cols // 32)
    r, b = np.meshgrid(np.arange(rows), np.arange(nb), indexing="ij")
    return 512 * ((r // 128) * (-(-nb // 4)) + b // 4) + 16 * (r % 32) + 4 * (r % 128 // 32) + b % 4


def leaks(gate, logit):
    z = np.asarray(gate, np.float64)
    if not logit:
        return z, 1.0 - z
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-z)), 1.0 / (1.0 + np.exp(z))


def full_gate(gate, shape):
    """[C], [B, C] or [B, T, C] as [B, T, C]."""
    b, t, c = shape
    g = np.asarray(gate)
    if g.ndim == 1:
        g = g[None, None]
    elif g.ndim == 2:
        g = g[:, None]
    return np.broadcast_to(g, (b, t, c))


class LeakyRef:
    """Forward and backward of one problem; *_err bound the 32-bit errors."""

    def __init__(self, x, gate=None, decay=None, h0=None, lengths=None, logit=False, complement=False, scale=1.0):
        b, t, c = self.shape = np.asarray(x).shape
        self.live = np.arange(t)[None, :] < (np.full(b, t) if lengths is None else np.minimum(lengths, t))[:, None]
        live = self.live[..., None]
        x = np.where(live, np.asarray(x, np.float64), 0.0)
        g = np.full((b, t, c), np.float32(decay)) if gate is None else full_gate(gate, self.shape)
        self.a, self.rest = leaks(np.where(live, g, 0.0), logit and gate is not None)
        self.logit, self.complement, self.scale, self.gate = logit, complement, scale, gate
        self.sx = scale * x
        u = self.sx * self.rest if complement else self.sx
        h = np.zeros((b, c)) if h0 is None else np.asarray(h0, np.float64)
        big, err = np.abs(h), np.zeros((b, c))
        self.before = np.zeros((b, t, c))
        self.before_err = np.zeros((b, t, c))
        self.y, self.y_err = np.zeros((b, t, c)), np.zeros((b, t, c))
        for i in range(t):
            on = live[:, i]
            self.before[:, i], self.before_err[:, i] = h, err
            a = self.a[:, i]
            nbig = np.abs(a) * big + np.abs(u[:, i])
            big, err = np.where(on, nbig, big), np.where(on, np.abs(a) * err + STEP * nbig + TINY, err)
            h = np.where(on, a * h + u[:, i], h)
            self.y[:, i], self.y_err[:, i] = np.where(on, h, 0), np.where(on, err, 0)
        self.h_last, self.h_last_err = h, err

    def backward(self, dy, dh_last=None):
        b, t, c = self.shape
        live = self.live[..., None]
        dy = np.where(live, np.asarray(dy, np.float64), 0.0)
        e = np.zeros((b, c)) if dh_last is None else np.asarray(dh_last, np.float64)
        big, err = np.abs(e), np.zeros((b, c))
        d, derr = np.zeros(self.shape), np.zeros(self.shape)
        for i in range(t - 1, -1, -1):
            on = live[:, i]
            a = self.a[:, i]
            step, nbig = dy[:, i] + e, np.abs(dy[:, i]) + big
            serr = err + STEP * nbig + TINY
            d[:, i], derr[:, i] = np.where(on, step, 0), np.where(on, serr, 0)
            e, big = np.where(on, a * step, e), np.where(on, np.abs(a) * nbig, big)
            err = np.where(on, np.abs(a) * serr + STEP * big + TINY, err)
        self.dh0, self.dh0_err = e, err
        f = self.scale * (self.rest if self.complement else 1.0)
        self.dx = d * f
        self.dx_err = np.abs(f) * (derr + STEP * np.abs(d)) + TINY
        k = self.before - self.sx if self.complement else self.before
        kmag = np.abs(self.before) + (np.abs(self.sx) if self.complement else 0.0)
        s = self.a * self.rest if self.logit else 1.0
        dg = d * k * s
        derr = np.abs(s) * (derr * np.abs(k) + (np.abs(d) + derr) * (self.before_err + STEP * kmag)) + STEP * np.abs(dg) + TINY
        if self.gate is None:
            return
        g = np.asarray(self.gate)
        if g.ndim < 3:  # summed over what shares it: a rounding for each step, block and sequence on the way
            axes = (0, 1) if g.ndim == 1 else (1,)
            roundings = (16 + t / 16 + b) * 2.0 ** -24
            self.dgate = dg.sum(axes)
            self.dgate_err = derr.sum(axes) + roundings * np.abs(dg).sum(axes)
        else:
            self.dgate, self.dgate_err = dg, derr


def check(got, want, err, kind, what, tiny=0.0):
    """|got - want| within the 32-bit bound and half a step of the output's type."""
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    # Below a type's normal range half a step is absolute.
    floor = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}[kind]
    room = err * (1 + HALF[kind]) + np.maximum(HALF[kind] * np.abs(want), floor) + tiny
    off = np.abs(got - want)
    bad = ~(off <= room)
    if bad.any():
        at = np.unravel_index(np.argmax(np.where(bad, off / np.maximum(room, 1e-300), 0)), bad.shape)
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} off, worst at {at}: {got[at]} against {want[at]}, "
                             f"room {room[at]}")
