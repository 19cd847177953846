"""The sequence operators in float64 NumPy from their definitions, with bounds on what single precision may round off.
Test helper, not part of the product.

Every bound counts roundings in units of U = 2^-24: the fp32 operations behind a value each add half a unit of their
result, the hardware's exp2, log2 and reciprocal a unit or two; what enters a recurrence is carried along with it."""
import numpy as np

from tests.philox import philox4x32_10

U = 2.0 ** -24
HALF_ULP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 1e-37, "bfloat16": 1e-37, "float16": 2.0 ** -25}


def rounding(dtype, value):
    """What rounding ``value`` to ``dtype`` may change."""
    name = str(dtype).replace("torch.", "")
    return HALF_ULP[name] * np.abs(value) + TINY[name]


# ------------------------------------------------------------------------------------------- recurrence
def softplus(g):
    return np.maximum(g, 0) + np.log1p(np.exp(-np.abs(g)))


def sigmoid(g):
    e = np.exp(-np.abs(g))
    return np.where(g >= 0, 1 / (1 + e), e / (1 + e))


def scan(x, g, start, dt=None, h0=None):
    """(y, last, E): states, last states and the states' rounding bound.  A step adds the roundings of a (4 units and 4
    per unit of its exponent, as exp2's argument is rounded relatively), of the token's weight and product (8) and of
    the sum (1), each relative to the sums' magnitudes M."""
    N, D = x.shape
    B = len(start) - 1
    z = softplus(g) * (1.0 if dt is None else dt[:, None])
    a, w = np.exp(-z), sigmoid(g)
    y, E = np.zeros((N, D)), np.zeros((N, D))
    last = np.zeros((B, D)) if h0 is None else h0.astype(np.float64).copy()
    for b in range(B):
        h = last[b].copy()
        m, e = np.abs(h), np.zeros(D)
        for i in range(start[b], start[b + 1]):
            u = w[i] * x[i]
            e = a[i] * (e + (4 + 4 * np.abs(z[i])) * m)
            m = a[i] * m + np.abs(u)
            e = e + 8 * np.abs(u) + m
            h = a[i] * h + u
            y[i], E[i] = h, e * U
        last[b] = h
    return y, last, E


def scan_bwd(x, g, start, gy, glast, dt=None, h0=None):
    """Gradients (gx, gg, gh0) and their bounds."""
    N, D = x.shape
    B = len(start) - 1
    y, _, Ey = scan(x, g, start, dt, h0)
    step = np.ones(N) if dt is None else dt
    z = softplus(g) * step[:, None]
    a, w = np.exp(-z), sigmoid(g)
    wc = sigmoid(-g)
    gx, gg = np.zeros((N, D)), np.zeros((N, D))
    Bx, Bg = np.zeros((N, D)), np.zeros((N, D))
    gh0, B0 = glast.astype(np.float64).copy(), np.zeros((B, D))
    for b in range(B):
        C = glast[b].astype(np.float64)
        mC, eC = np.abs(C), np.zeros(D)
        for i in range(start[b + 1] - 1, start[b] - 1, -1):
            first = i == start[b]
            hp = (np.zeros(D) if h0 is None else h0[b].astype(np.float64)) if first else y[i - 1]
            ep = np.zeros(D) if first else Ey[i - 1]
            mp = np.abs(hp) + ep
            H, mH = gy[i] + C, np.abs(gy[i]) + mC
            eH = eC + mH * U
            gx[i] = H * w[i]
            Bx[i] = (eH + 6 * U * mH) * w[i]
            da = step[i] * a[i]
            t = x[i] * wc[i] - da * hp
            mt = np.abs(x[i]) * wc[i] + np.abs(da) * mp
            gg[i] = H * w[i] * t
            Bg[i] = w[i] * (eH * mt + mH * (U * (16 + 4 * np.abs(z[i])) * mt + np.abs(da) * ep))
            C = a[i] * H
            eC = a[i] * (eH + (5 + 4 * np.abs(z[i])) * mH * U)
            mC = a[i] * mH
        gh0[b], B0[b] = C, eC
    return (gx, gg, gh0), (Bx, Bg, B0)


# ------------------------------------------------------------------------------------------- norm
def keeps(N, D, p, seed, offset):
    t = round(65536 * p)
    groups = (D + 7) // 8
    row = np.repeat(np.arange(N), groups)
    grp = np.tile(np.arange(groups), N)
    full = lambda v: np.full(row.shape, v, np.uint32)
    words = philox4x32_10(row.astype(np.uint32), (grp + 2 ** 31).astype(np.uint32), full(offset & 0xFFFFFFFF),
                          full(offset >> 32), seed & 0xFFFFFFFF, seed >> 32)
    bits = np.stack([h for v in words for h in (v & np.uint32(0xFFFF), v >> np.uint32(16))], 1)
    return bits.reshape(N, groups * 8)[:, :D] >= t


def norm(s, w, eps):
    r = 1 / np.sqrt((s * s).mean(1, keepdims=True) + eps)
    return s * r * w, r


def norm_bwd(s, w, eps, gy, gs):
    """(ds, gw) and their bounds.  A row's sums have at most 32 terms in sequence and 8 levels; 64 units cover them, the
    reciprocal root and the products.  gw adds N rows in any order: N units."""
    y, r = norm(s, w, eps)
    hat = s * r
    mean = (w * gy * hat).mean(1, keepdims=True)
    ds = gs + r * (w * gy - hat * mean)
    mag = np.abs(gs) + r * (np.abs(w * gy) + np.abs(hat) * np.abs(w * gy * hat).mean(1, keepdims=True))
    return (ds, (gy * hat).sum(0)), (64 * U * mag, (64 + s.shape[0]) * U * np.abs(gy * hat).sum(0))


# ------------------------------------------------------------------------------------------- embedding
def embed_bwd(ids, V, scale, g):
    """gtable and its bound: a row of n terms is off by at most n units of the sum of their magnitudes."""
    D = g.shape[1]
    out, mag, n = np.zeros((V, D)), np.zeros((V, D)), np.zeros(V)
    ok = (ids >= 0) & (ids < V)
    np.add.at(out, ids[ok], g[ok])
    np.add.at(mag, ids[ok], np.abs(g[ok]))
    np.add.at(n, ids[ok], 1)
    return out * scale, (n[:, None] + 2) * U * mag * abs(scale)
