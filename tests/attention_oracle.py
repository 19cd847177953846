"""The attention operators in float64 NumPy from their definitions, with bounds on what the kernels may round off.  Test
helper, not part of the product.

Every bound counts roundings in units of U = 2^-24 of sums of magnitudes: each fp32 operation behind a value adds half a unit of
its result, the hardware's exponential a unit or two and its argument one per unit of the exponent.  Where operands go on as
two pieces of a 16-bit type (the pairs' weights and the states), what is left behind both is counted for them."""
import numpy as np

from tests.sequence_oracle import HALF_ULP, U

# What is left of a state behind its pieces, and of a value behind the smallest half precision number where its largest
# neighbour is brought to 2^14 first (2^-25 / 2^14, and as much again).
PIECES = {"float32": 0.0, "bfloat16": HALF_ULP["bfloat16"] ** 2, "float16": HALF_ULP["float16"] ** 2}
FLOOR = {"float32": 0.0, "bfloat16": 0.0, "float16": 2.0 ** -38}
PAIR = PIECES                                             # the weights of pairs too go on in two pieces
FORGOTTEN = 400.0 * np.log(2.0)


def _sweep(X, Y, W, z, given, ps, xs, us, dtype):
    """One window's recurrence over rows (n, H, D) with row i's decay z (n, H) applied before its product:
    out_i = ps sum_j e^{..} (X_i Y_j) W_j + xs e^{..} X_i given, end = e^{..} given + us sum e^{..} Y W^T; (out, end) and their
    bounds."""
    n, H, D = X.shape
    units = 3 * D + 300 + 3 * (n // 64 + 1)
    z = np.where(z > FORGOTTEN, FORGOTTEN, z)              # the kernels' own definition of an endless gap
    E = np.cumsum(z, 0)
    out, bound = np.zeros((n, H, D)), np.zeros((n, H, D))
    end, bend = np.zeros((H, D, D)), np.zeros((H, D, D))
    low = np.tril(np.ones((n, n), bool))
    near = low & (np.arange(n)[:, None] - np.arange(n)[None] < 64)
    for h in range(H):
        x, y, w = X[:, h], Y[:, h], W[:, h]
        d = np.where(low, E[:, h][:, None] - E[:, h][None], 0.0)
        L = np.where(low, np.exp(-d), 0.0)
        La = L * (1 + np.abs(d))
        e = np.exp(-E[:, h])[:, None]
        ea = e * (1 + np.abs(E[:, h])[:, None])
        P = L * (x @ y.T)
        Pa = La * (np.abs(x) @ np.abs(y).T)
        out[:, h] = ps * (P @ w) + xs * e * (x @ given[h])
        mag = abs(ps) * (Pa @ np.abs(w)) + abs(xs) * ea * (np.abs(x) @ np.abs(given[h]))
        bound[:, h] = (units * U + PIECES[dtype]) * mag + PAIR[dtype] * abs(ps) * (np.where(near, np.abs(P), 0) @ np.abs(w))
        if n:
            top = np.abs(w).max() * n * np.abs(P).max() * abs(ps) + abs(xs) * np.abs(x).sum(1).max() * np.abs(given[h]).max()
            bound[:, h] += FLOOR[dtype] * top
            f = np.exp(-(E[-1, h] - E[:, h]))[:, None]
            fa = f * (1 + np.abs(E[-1, h] - E[:, h])[:, None])
            g, ga = np.exp(-E[-1, h]), np.exp(-E[-1, h]) * (1 + abs(E[-1, h]))
            end[h] = g * given[h] + us * (f * y).T @ w
            bend[h] = units * U * (ga * np.abs(given[h]) + abs(us) * (fa * np.abs(y)).T @ np.abs(w))
            bend[h] += FLOOR[dtype] * n * np.abs(y).max() * np.abs(w).max() * abs(us)
        else:
            end[h] = given[h]
    return out, end, bound, bend


def _gaps(rate, dt, lo, hi):
    step = np.ones(hi - lo) if dt is None else dt[lo:hi]
    return step[:, None] * rate[None]


def attention(q, k, v, rate, start, dt, h0, scale, dtype):
    """(y, last), (by, blast) for (N, H, D) in float64."""
    N, H, D = q.shape
    B = len(start) - 1
    y, by = np.zeros((N, H, D)), np.zeros((N, H, D))
    last, bl = np.zeros((B, H, D, D)), np.zeros((B, H, D, D))
    for b in range(B):
        lo, hi = start[b], start[b + 1]
        given = np.zeros((H, D, D)) if h0 is None else h0[b]
        y[lo:hi], last[b], by[lo:hi], bl[b] = _sweep(q[lo:hi], k[lo:hi], v[lo:hi], _gaps(rate, dt, lo, hi), given, scale, scale,
                                                     1.0, dtype)
    return (y, last), (by, bl)


def attention_bwd(q, k, v, rate, start, dt, h0, scale, gy, glast, dtype):
    """(gq, gk, gv, gh0) and their bounds."""
    N, H, D = q.shape
    B = len(start) - 1
    out = [np.zeros((N, H, D)) for _ in range(3)]
    bound = [np.zeros((N, H, D)) for _ in range(3)]
    g0, b0 = np.zeros((B, H, D, D)), np.zeros((B, H, D, D))
    T = lambda m: m.transpose(0, 2, 1)
    for b in range(B):
        s = slice(start[b], start[b + 1])
        z = _gaps(rate, dt, s.start, s.stop)
        given = np.zeros((H, D, D)) if h0 is None else h0[b]
        out[0][s], _, bound[0][s], _ = _sweep(gy[s], v[s], k[s], z, T(given), scale, scale, 1.0, dtype)
        # from the end a row's decay is that of the token after it, and the window's first gap is left for the end
        n = s.stop - s.start
        zr = np.concatenate([np.zeros((1, H)), z[::-1][:-1]]) if n else z
        r = lambda a: a[s][::-1]
        o, end, bo, be = _sweep(r(k), r(q), r(gy), zr, glast[b], scale, 1.0, scale, dtype)
        out[2][s], bound[2][s] = o[::-1], bo[::-1]
        f = np.exp(-np.minimum(z[0], FORGOTTEN))[:, None, None] if n else 1.0
        grow = (1 + np.abs(np.minimum(z[0], FORGOTTEN)))[:, None, None] if n else 1.0
        g0[b], b0[b] = f * end, f * (be + 8 * U * grow * (np.abs(end) + be))
        o, _, bo, _ = _sweep(r(v), r(gy), r(q), zr, T(glast[b]), scale, 1.0, scale, dtype)
        out[1][s], bound[1][s] = o[::-1], bo[::-1]
    return (*out, g0), (*bound, b0)


def follow(x, y, w, z, given, ps, xs, us):
    """One long window's recurrence token by token, as _sweep's: out and end, and what the same comes to in magnitudes.  With
    at most EXPONENT in any factor, a factor's own rounding is 1 + EXPONENT units of it."""
    n, H, D = x.shape
    out, mag = np.zeros((n, H, D)), np.zeros((n, H, D))
    own, far = np.zeros((H, D, D)), given.astype(np.float64)
    own_a, far_a = np.zeros((H, D, D)), np.abs(far)
    for i in range(n):
        a = np.exp(-z[i])[:, None, None]
        new = y[i][:, :, None] * w[i][:, None, :]
        own, far = a * own + new, a * far
        own_a, far_a = a * own_a + np.abs(new), a * far_a
        out[i] = ps * (x[i][:, None, :] @ own)[:, 0] + xs * (x[i][:, None, :] @ far)[:, 0]
        mag[i] = abs(ps) * (np.abs(x[i])[:, None, :] @ own_a)[:, 0] + abs(xs) * (np.abs(x[i])[:, None, :] @ far_a)[:, 0]
    return out, us * own + far, mag, abs(us) * own_a + far_a


# ------------------------------------------------------------------------------------------- norm and rotation
def _turn(x, angle, sign):
    """(N, H, D) with pairs turned; and the sum of the magnitudes behind every element."""
    P = angle.shape[1]
    c, s = np.cos(angle)[:, None], sign * np.sin(angle)[:, None]
    y, mag = x.copy(), np.abs(x)
    a, b = x[..., 0:2 * P:2], x[..., 1:2 * P:2]
    y[..., 0:2 * P:2], y[..., 1:2 * P:2] = a * c - b * s, a * s + b * c
    both = np.abs(a) + np.abs(b)
    mag[..., 0:2 * P:2] = mag[..., 1:2 * P:2] = both
    return y, mag


def angles(pos, freqs, sections):
    axis = np.repeat(np.arange(len(sections)), sections)
    return pos[:, axis] * freqs[None]


def rotary(x, w, angle, eps):
    """y and its bound: a sum of D squares (D units at most), the root and products (8), the angle in turns rounded to 2^-25
    (2 pi units) and sine and cosine of it (4), the rotation (4)."""
    D = x.shape[-1]
    hat = x if w is None else x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    y, mag = _turn(hat, angle, 1.0)
    return y, (D + 24) * U * mag


def rotary_bwd(x, w, angle, eps, gy):
    """(gx, gw) and their bounds; gw adds all rows in any order."""
    D = x.shape[-1]
    g, mag = _turn(gy, angle, -1.0)
    if w is None:
        return (g, None), (24 * U * mag, None)
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    hat = x * r
    mean = (w * g * hat).mean(-1, keepdims=True)
    gx = r * (w * g - hat * mean)
    big = r * (np.abs(w) * mag + np.abs(hat) * (np.abs(w) * mag * np.abs(hat)).mean(-1, keepdims=True))
    rows = x.shape[0] * x.shape[1]
    return (gx, (g * hat).sum((0, 1))), ((2 * D + 64) * U * big, (rows + D + 64) * U * (mag * np.abs(hat)).sum((0, 1)))


def by_token(q, k, v, rate, start, dt, h0, scale, gy, glast):
    """(y, last, gq, gk, gv, gh0) from the definitions one token after the other, and the same of magnitudes: no product is left
    out or taken apart, so infinities and NaN go where the formulas take them."""
    N, H, D = q.shape
    B = len(start) - 1
    a = np.exp(-(np.ones(N) if dt is None else dt)[:, None] * rate[None])[..., None, None]
    with np.errstate(invalid="ignore", over="ignore"):
        both = []
        for f in (lambda t: t, np.abs):
            Q, K, V, G0, GY, GL = (f(t) for t in (q, k, v, np.zeros((B, H, D, D)) if h0 is None else h0, gy, glast))
            y, gq, gk, gv = (np.zeros((N, H, D)) for _ in range(4))
            last, gh0 = np.zeros((B, H, D, D)), np.zeros((B, H, D, D))
            for b in range(B):
                S = G0[b]
                for i in range(start[b], start[b + 1]):
                    S = a[i] * S + K[i][:, :, None] * V[i][:, None, :]
                    y[i] = f(scale) * (Q[i][:, :, None] * S).sum(1)
                    gq[i] = f(scale) * (S * GY[i][:, None, :]).sum(2)
                last[b], G = S, GL[b]
                for i in reversed(range(start[b], start[b + 1])):
                    G = G + f(scale) * Q[i][:, :, None] * GY[i][:, None, :]
                    gv[i] = (K[i][:, :, None] * G).sum(1)
                    gk[i] = (G * V[i][:, None, :]).sum(2)
                    G = a[i] * G
                gh0[b] = G
            both.append((y, last, gq, gk, gv, gh0))
    return both
