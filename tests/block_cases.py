"""64-bit definitions of the block operators with elementwise error bounds, shared by test_blocks_gpu.py and test_blocks_cpu.py.

A bound is built next to its value: u = 2^-24 is half a step of fp32, r half a step of the tensors' type (0 for fp32: a stored fp32 result adds
one u).  A sum of n products formed in fp32 is off by at most (n + c) u times the sum of the products' magnitudes; a rounding to the type
by r times the magnitude; what enters a function is passed on by the largest slope it has."""
import numpy as np
import torch

U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}      # half a step of the smallest numbers


def act64(g, kind):
    """act(g), act'(g) and the largest |act''|"""
    if kind == "relu":
        return torch.relu(g), (g > 0).double(), 0.0
    if kind == "sigmoid":
        s = torch.sigmoid(g)
        return s, s * (1 - s), 0.1
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s)), 0.51
    k, c = (2 / np.pi) ** 0.5, 0.044715
    t = torch.tanh(k * (g + c * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * c * g * g), 1.2


def mlp64(x, wg, wu, wd, kind, dy=None):
    """{name: (value, bound)} of the gated block in 64 bits for tensors of one type"""
    dt = x.dtype
    r, tiny = HALF_STEP[dt], TINY[dt]
    hid = 0.0 if dt == torch.float32 else r            # the hidden layer's own rounding
    # products a sum is made of: fp32 operands go as three bf16 terms, six products for one, and up to 2^-25 of one is left out
    n = lambda k: (6 * k + 16) * U if dt == torch.float32 else (k + 8) * U  # noqa: E731
    x, wg, wu, wd = (t.double() for t in (x, wg, wu, wd))
    g, u = x @ wg.t(), x @ wu.t()
    gb, ub = n(x.shape[1]) * (x.abs() @ wg.abs().t()), n(x.shape[1]) * (x.abs() @ wu.abs().t())
    a, s, bend = act64(g, kind)
    h = a * u
    ab = 1.2 * gb + 8 * U * a.abs()
    hb = u.abs() * ab + a.abs() * ub + ab * ub + 4 * U * h.abs()
    hs = hb + hid * h.abs() + tiny
    y = h @ wd.t()
    yb = hs @ wd.abs().t() + n(h.shape[1]) * ((h.abs() + hs) @ wd.abs().t())
    out = {"y": (y, yb + r * (y.abs() + yb) + tiny)}
    if dy is not None:
        dy = dy.double()
        d = dy @ wd
        db = n(dy.shape[1]) * (dy.abs() @ wd.abs())
        sb = bend * gb + 16 * U * (1 + g.abs()) if kind != "relu" else (g.abs() <= gb).double()      # next to relu's corner: either slope
        dg, du = d * u * s, d * a
        dgb = db * (u.abs() + ub) * (s.abs() + sb) + d.abs() * ub * (s.abs() + sb) + d.abs() * u.abs() * sb + 4 * U * dg.abs()
        dub = db * (a.abs() + ab) + d.abs() * ab + 4 * U * du.abs()
        dgs, dus = dgb + hid * (dg.abs() + dgb) + tiny, dub + hid * (du.abs() + dub) + tiny
        for name, terms in (("dx", [(dg, dgs, wg), (du, dus, wu)]), ("dw_gate", [(dg.t(), dgs.t(), x)]), ("dw_up", [(du.t(), dus.t(), x)]),
                            ("dw_down", [(dy.t(), None, h)])):
            k = sum(t[0].shape[1] for t in terms)
            v = sum(p @ q for p, _, q in terms)
            if name == "dw_down":
                b = dy.abs().t() @ hs + n(k) * (dy.abs().t() @ (h.abs() + hs))
            else:
                b = sum(pb @ q.abs() for _, pb, q in terms) + n(k) * sum((p.abs() + pb) @ q.abs() for p, pb, q in terms)
            out[name] = (v, b + r * (v.abs() + b) + tiny)
    return out


def scan64(gate, value, rays, state, blend, dt, dh=None, dlast=None):
    """{name: (value, bound)} of the recurrence, row by row in numpy; inputs numpy float64 of values the type holds"""
    T, C = gate.shape
    N = len(rays)
    r, tiny = HALF_STEP[dt], TINY[dt]
    e = 16 * U                       # what one step's arithmetic (the sigmoid above all) is off by, relative to the magnitudes it joins
    with np.errstate(over="ignore"):
        a, an = 1 / (1 + np.exp(-gate)), 1 / (1 + np.exp(gate))
    k = an if blend else np.ones_like(a)
    z = lambda *s: np.zeros(s)  # noqa: E731
    h, hb, prev, prevb = z(T, C), z(T, C), z(T, C), z(T, C)
    last, lastb = state.copy(), z(N, C)
    dgate, dgb, dval, dvb = z(T, C), z(T, C), z(T, C), z(T, C)
    dstate, dsb = (z(N, C) if dlast is None else dlast.copy()), z(N, C)
    for ident, off, cnt in rays:
        if cnt <= 0 or off < 0 or off + cnt > T:
            continue
        known = 0 <= ident < N
        c = state[ident].copy() if known else z(C)
        cb, mag = z(C), np.abs(c)
        for t in range(off, off + cnt):
            prev[t], prevb[t] = c, cb
            mag_in = a[t] * mag + k[t] * np.abs(value[t])
            cb = a[t] * cb + e * (a[t] * mag + k[t] * (np.abs(value[t]) + mag) + mag_in)
            c = a[t] * c + k[t] * value[t]
            mag = mag_in
            h[t], hb[t] = c, cb
        if known:
            last[ident], lastb[ident] = c, cb
        if dh is None:
            continue
        E = dlast[ident].copy() if known and dlast is not None else z(C)
        Eb, mag = z(C), np.abs(E)
        for t in range(off + cnt - 1, off - 1, -1):
            G, Gb, mag = dh[t] + E, Eb + e * (mag + np.abs(dh[t])), mag + np.abs(dh[t])
            src, srcb = (prev[t] - value[t], prevb[t] + e * (np.abs(prev[t]) + np.abs(value[t]))) if blend else (prev[t], prevb[t])
            w = a[t] * an[t]
            dgate[t], dgb[t] = G * src * w, w * (Gb * (np.abs(src) + srcb) + np.abs(G) * srcb) + e * w * mag * (np.abs(src) + srcb)
            dval[t], dvb[t] = G * k[t], k[t] * Gb + e * k[t] * mag
            E, Eb = a[t] * G, a[t] * Gb + e * a[t] * mag
            mag = a[t] * mag
        if known:
            dstate[ident], dsb[ident] = E, Eb
    stored = lambda v, b: (v, b + r * (np.abs(v) + b) + tiny)  # noqa: E731
    f32 = lambda v, b: (v, b + U * (np.abs(v) + b) + TINY[torch.float32])  # noqa: E731
    out = {"h": stored(h, hb), "last": f32(last, lastb)}
    if dh is not None:
        out |= {"dgate": stored(dgate, dgb), "dvalue": stored(dval, dvb), "dstate": f32(dstate, dsb)}
    return out


def philox_bits(key, call, n, first=0):
    """16 bits an element of the Philox4x32-10 stream (Salmon et al. 2011), from element `first` (a multiple of 8) on, in unsigned 64-bit words"""
    u = np.uint64
    low, half = u(0xFFFFFFFF), u(32)
    i = np.arange((n + 7) // 8, dtype=u) + u(first // 8)
    key, call = int(key) % 2 ** 64, int(call) % 2 ** 64
    c = [i & low, i >> half, np.full_like(i, call & 0xFFFFFFFF), np.full_like(i, call >> 32)]
    k0, k1 = key & 0xFFFFFFFF, key >> 32
    for _ in range(10):
        p, q = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(q >> half) ^ c[1] ^ u(k0), q & low, (p >> half) ^ c[3] ^ u(k1), p & low]
        k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
    return np.stack(c, 1).astype("<u4").view("<u2").reshape(-1)[:n]


def within(got, want, bound, what=""):
    got = got.detach().double().cpu().numpy() if isinstance(got, torch.Tensor) else got
    want, bound = (t.cpu().numpy() if isinstance(t, torch.Tensor) else t for t in (want, bound))
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = np.abs(got - want)
    bad = ~(off <= bound)
    if bad.any():
        at = np.unravel_index(np.argmax(np.where(bad, off / np.maximum(bound, 1e-300), 0)), off.shape)
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} values off; at {at}: got {got[at]!r}, want {want[at]!r}, bound {bound[at]:.3g}")
