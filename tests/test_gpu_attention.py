"""The attention operators' HIP kernels against the float64 oracle, with its bounds on the kernels' roundings and half a unit of
the output's type: types, widths, lengths, strides, shared heads, empty windows and tokens outside of them, gaps of every size,
NaN and infinities that stay where they are, streams, graphs, offsets past 32 bits, and equal bits on equal calls."""
import numpy as np
import pytest
import torch

from tests import attention_oracle as O
from tests.sequence_oracle import rounding
from x_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _t(a, dtype=F32):
    return None if a is None else torch.as_tensor(a, device=DEV).to(dtype)


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _name(dtype):
    return str(dtype).replace("torch.", "")


def _close(got, want, bound, what=""):
    dtype, got = got.dtype, _np(got)
    assert got.shape == want.shape, (got.shape, want.shape)
    tol = bound + rounding(dtype, np.abs(want) + bound)
    err = np.abs(got - want)
    bad = ~(err <= tol)
    if bad.any():
        pytest.fail(f"{what}: {int(bad.sum())} of {bad.size} off, worst {np.max(np.where(bad, err / tol, 0)):.3g} of the bound")


def _spread(a, how):
    """The same heads in another layout: 'slice' of a wider projection, 'odd' one that starts off alignment, 'heads' with the
    heads before the tokens, 'cols' channels apart (copied by the operator)."""
    N, H, D = a.shape
    if how == "slice":
        wide = torch.zeros(N, H * D + 32, dtype=a.dtype, device=a.device)
        wide[:, 16:16 + H * D] = a.reshape(N, H * D)
        return wide[:, 16:16 + H * D].view(N, H, D)
    if how == "odd":
        wide = torch.zeros(N, H, D + 3, dtype=a.dtype, device=a.device)
        wide[..., 1:1 + D] = a
        return wide[..., 1:1 + D]
    if how == "heads":
        return a.transpose(0, 1).contiguous().transpose(0, 1)
    if how == "cols":
        return a.transpose(0, 2).contiguous().transpose(0, 2)
    return a


# ------------------------------------------------------------------------------------------- attention
def _windows(kind, N, rng):
    if kind == "one":
        return [0, N]
    if kind == "ragged":                                     # with empty windows at both ends and between
        cuts = np.sort(rng.integers(0, N + 1, 5))
        return [0, 0, *np.repeat(cuts, 2).tolist(), N, N]
    if kind == "short":
        return list(range(0, N, 3)) + [N, N]
    if kind == "inside":                                     # tokens of no window before and behind
        return [N // 5, N // 2, N // 2, N - N // 7]
    raise ValueError(kind)


def _case(N, H, D, dtype, kind, with_dt=True, with_h0=True, layout=None, seed=0, grads=("y", "last"), gap=None, size=1.0):
    rng = np.random.default_rng(seed)
    start = _windows(kind, N, rng)
    B = len(start) - 1
    q, k, v, gy = (_t(rng.normal(size=(N, H, D)) * s, dtype) for s in (1, 1, size, 1 / size))
    rate = _t(2.0 ** (-4.0 * np.arange(H) / H) * (1.0 if with_dt else 1 / 64))
    dt = None if not with_dt else _t(rng.exponential(size=N) * (gap or 8 * B / max(N, 1)))
    h0 = _t(rng.normal(size=(B, H, D, D)) * 3 * size) if with_h0 else None
    gl = _t(rng.normal(size=(B, H, D, D)) / size)
    scale = D ** -0.5
    print(f"attention N={N} H={H} D={D} {dtype} {kind} B={B} dt={with_dt} h0={with_h0} {layout}", flush=True)
    qs, ks, vs, gys = (_spread(a, layout).detach() for a in (q, k, v, gy))
    ins = [a.requires_grad_() for a in (qs, ks, vs)] + ([h0.requires_grad_()] if with_h0 else [])
    st = torch.tensor(start, device=DEV)
    y, last = ops.decay_attention(qs, ks, vs, rate, st, dt=dt, h0=h0)
    args = (_np(q), _np(k), _np(v), _np(rate), start, _np(dt), _np(h0), scale)
    (wy, wl), (by, bl) = O.attention(*args, _name(dtype))
    _close(y, wy, by, "y")
    _close(last, wl, bl, "last")
    with torch.no_grad():
        y2, last2 = ops.decay_attention(qs, ks, vs, rate, st, dt=dt, h0=h0, scale=scale)
    assert torch.equal(y, y2) and torch.equal(last, last2)
    outs = [(y, gys)] * ("y" in grads) + [(last, gl)] * ("last" in grads)
    got = torch.autograd.grad([a for a, _ in outs], ins, [b for _, b in outs], retain_graph=True)
    gyn = _np(gy) if "y" in grads else np.zeros((N, H, D))
    gln = _np(gl) if "last" in grads else np.zeros((B, H, D, D))
    want, bound = O.attention_bwd(*args, gyn, gln, _name(dtype))
    for name, a, b, c in zip(("gq", "gk", "gv", "gh0"), got, want, bound):
        _close(a, b, c, name)
    again = torch.autograd.grad([a for a, _ in outs], ins, [b for _, b in outs])
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("N", [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 700, 1400])
@pytest.mark.parametrize("dtype,H,D", [(F32, 2, 5), (BF16, 1, 64), (F16, 3, 32)])
def test_attention_lengths(N, dtype, H, D):
    _case(N, H, D, dtype, "ragged", seed=N)


@pytest.mark.parametrize("D", [1, 2, 3, 4, 7, 8, 12, 16, 31, 32, 33, 45, 48, 63, 64, 65, 72, 96, 100, 127, 128])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_attention_widths(D, dtype):
    _case(300, 2, D, dtype, "ragged", with_dt=D % 2 == 0, with_h0=D % 3 == 0, seed=D)


@pytest.mark.parametrize("layout", ["slice", "odd", "heads", "cols"])
@pytest.mark.parametrize("dtype,D", [(F32, 64), (BF16, 64), (F16, 32), (BF16, 128)])
def test_attention_layouts(layout, dtype, D):
    _case(400, 2, D, dtype, "ragged", layout=layout, with_h0=False, seed=11)


@pytest.mark.parametrize("kind", ["one", "short", "inside"])
@pytest.mark.parametrize("dtype,D", [(F32, 16), (BF16, 32)])
@pytest.mark.parametrize("with_dt", [False, True])
def test_attention_windows(kind, dtype, D, with_dt):
    _case(1100, 2, D, dtype, kind, with_dt=with_dt, seed=12)


@pytest.mark.parametrize("N", [2500, 9000, 20_011])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("among", [False, True])
def test_attention_of_long_windows(N, dtype, among):
    """Windows of ten stretches, of 36 and of 79, alone and between many short ones: the states between stretches joined by one
    thread, and in runs."""
    _long_window(N, 8, dtype, among)


@pytest.mark.parametrize("D", [32, 33, 72, 128])
@pytest.mark.parametrize("N", [1300, 2500])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_attention_of_long_windows_and_wide_heads(N, D, dtype):
    """Windows of six stretches, whose sums a sweep adds up, and of ten, whose sums are joined."""
    _long_window(N, D, dtype, True)


def _long_window(N, D, dtype, among):
    """Exponents stay below 4, so a factor is off by 5 units of itself."""
    H, scale = 1, 0.5
    rng = np.random.default_rng(N)
    short = [3] * 60 if among else []
    lo = sum(short)
    start = np.concatenate([[0], np.cumsum(short + [N] + short)]).astype(int)
    B, T = len(start) - 1, int(start[-1])
    q, k, v, gy = (_t(a, dtype) for a in rng.normal(size=(4, T, H, D)))
    h0, gl = (_t(a) for a in rng.normal(size=(2, B, H, D, D)))
    dt, rate = _t(rng.random(T) * 8 / N), _t([0.9])
    ins = [a.requires_grad_() for a in (q, k, v, h0)]
    print(f"long windows N={N} D={D} {dtype} among={among}", flush=True)
    y, last = ops.decay_attention(*ins[:3], rate, torch.tensor(start, device=DEV), dt=dt, h0=h0, scale=scale)
    grads = torch.autograd.grad((y, last), ins, (gy, gl))
    s, b = slice(lo, lo + N), len(short)
    z = (_np(dt)[s] * _np(rate)[0])[:, None]
    x, key, val, g = (_np(a)[s] for a in (q, k, v, gy))
    units = (3 * D + 300 + 3 * (N // 32 + 1)) * 5 * O.U + O.PIECES[_name(dtype)]
    T_ = lambda m: m.transpose(0, 2, 1)
    out, end, mag, emag = O.follow(x, key, val, z, _np(h0)[b], scale, scale, 1.0)
    _close(y[s], out, units * mag, "y")
    _close(last[b], end, units * emag, "last")
    out, _, mag, _ = O.follow(g, val, key, z, T_(_np(h0)[b]), scale, scale, 1.0)
    _close(grads[0][s], out, units * mag, "gq")
    r, zr = lambda a: a[::-1], np.concatenate([np.zeros((1, 1)), z[::-1][:-1]])
    out, end, mag, emag = O.follow(r(key), r(x), r(g), zr, _np(gl)[b], scale, 1.0, scale)
    _close(grads[2][s], out[::-1], units * mag[::-1], "gv")
    f = np.exp(-z[0])[:, None, None]
    _close(grads[3][b], f * end, units * f * emag, "gh0")
    out, _, mag, _ = O.follow(r(val), r(g), r(x), zr, T_(_np(gl)[b]), scale, 1.0, scale)
    _close(grads[1][s], out[::-1], units * mag[::-1], "gk")


def test_attention_without_windows_and_of_plain_sums():
    """No window: zeros.  32-bit starts, and the gradient of a plain sum (a scalar that is expanded)."""
    q, k, v = (torch.randn(40, 2, 8, device=DEV, requires_grad=True) for _ in range(3))
    rate = torch.ones(2, device=DEV)
    y, last = ops.decay_attention(q, k, v, rate, torch.zeros(1, dtype=torch.int64, device=DEV))
    assert not y.any() and last.shape == (0, 2, 8, 8)
    assert not any(g.any() for g in torch.autograd.grad(y.sum(), (q, k, v)))
    start = torch.tensor([0, 15, 40], device=DEV)
    y, _ = ops.decay_attention(q, k, v, rate, start.int())
    assert torch.equal(y, ops.decay_attention(q, k, v, rate, start)[0])
    for a, b in zip(torch.autograd.grad(y.sum(), (q, k, v), retain_graph=True), torch.autograd.grad(y, (q, k, v), torch.ones_like(y))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("N", [2000, 20_000])
@pytest.mark.parametrize("D", [8, 32, 64, 128])
def test_attention_without_windows_past_the_joined_length(N, D):
    """Tokens and no window, as long as windows whose stretches are joined: zeros, forward and backward."""
    q, k, v = (torch.randn(N, 2, D, device=DEV, requires_grad=True) for _ in range(3))
    h0 = torch.zeros(0, 2, D, D, device=DEV, requires_grad=True)
    print(f"no window: N={N} D={D}", flush=True)
    y, last = ops.decay_attention(q, k, v, torch.ones(2, device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV), h0=h0)
    assert not y.any() and last.shape == (0, 2, D, D)
    *grads, g0 = torch.autograd.grad((y, last), (q, k, v, h0), (torch.randn_like(y), torch.zeros_like(last)))
    assert not any(g.any() for g in grads) and g0.shape == h0.shape


@pytest.mark.parametrize("H", [1, 2, 5, 16, 33])
def test_attention_heads(H):
    _case(600, H, 16, BF16, "ragged", seed=H)


@pytest.mark.parametrize("grads", [("y",), ("last",)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_partial_gradients(grads, dtype):
    _case(600, 2, 24, dtype, "ragged", seed=13, grads=grads)


@pytest.mark.parametrize("D", [8, 32, 45, 128])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("N", [0, 50, 900, 2500])
def test_attention_gradients_of_states_alone(N, D, dtype):
    """Where nothing was made of the outputs, their products have no part in the gradients: queries get zeros, and infinities in
    queries and in the states that they met change no bit of the others."""
    gen = torch.Generator(device=DEV).manual_seed(N + D)
    q, k, v = torch.randn(3, N, 2, D, device=DEV, generator=gen).to(dtype)
    h0, gl = torch.randn(2, 3, 2, D, D, device=DEV, generator=gen)
    rate, start = torch.tensor([0.01, 0.001], device=DEV), torch.tensor([N // 5, N // 5, N // 2, N], device=DEV)
    print(f"gradients of states alone N={N} D={D} {dtype}", flush=True)

    def go(q, h0):
        ins = [t.clone().requires_grad_() for t in (q, k, v, h0)]
        return torch.autograd.grad(ops.decay_attention(*ins[:3], rate, start, h0=ins[3])[1], ins, gl)

    clean = go(q, h0)
    assert not clean[0].any()
    zeros = [t.clone().requires_grad_() for t in (q, k, v, h0)]
    y, last = ops.decay_attention(*zeros[:3], rate, start, h0=zeros[3])
    for a, b in zip(torch.autograd.grad((y, last), zeros, (torch.zeros_like(y), gl)), clean):
        assert torch.equal(a, b)                             # finite inputs: as with a gradient of zeros
    if N:
        q, h0 = q.clone(), h0.clone()
        q[N - N // 3, 0, D - 1], h0[1, 1, 0, D // 2], h0[2, 0, 0, 0] = float("inf"), float("-inf"), float("nan")
        assert all(torch.equal(a, b) for a, b in zip(go(q, h0), clean))


@pytest.mark.parametrize("gap", [1e-6, 1.0, 1e4])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_gaps(gap, dtype):
    """From gaps far below the time constant to gaps that forget everything."""
    _case(900, 2, 16, dtype, "one", seed=14, gap=gap)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("size", [1e-3, 300.0])
def test_attention_of_small_and_large_values(dtype, size):
    """Values of a thousandth and of hundreds: states past half precision's largest number, gradients near its smallest."""
    _case(700, 2, 32, dtype, "one", with_h0=True, seed=15, size=size)


def test_attention_gaps_back_in_time():
    """Events out of order: negative gaps grow the state as the formula has it, within a chunk, over chunks and stretches."""
    rng = np.random.default_rng(21)
    N, H, D = 900, 2, 8
    gap = rng.exponential(size=N) * 0.05
    gap[rng.random(N) < 0.3] *= -1
    gap[400:470] = -np.abs(gap[400:470])
    q, k, v, gy = (_t(a) for a in rng.normal(size=(4, N, H, D)))
    rate, dt, start = _t([1.0, 0.3]), _t(gap), [0, 800, N]
    ins = [a.requires_grad_() for a in (q, k, v)]
    y, last = ops.decay_attention(*ins, rate, torch.tensor(start, device=DEV), dt=dt)
    args = (_np(q), _np(k), _np(v), _np(rate), start, _np(dt), None, D ** -0.5)
    (wy, wl), (by, bl) = O.attention(*args, "float32")
    _close(y, wy, by, "y")
    _close(last, wl, bl, "last")
    want, bound = O.attention_bwd(*args, _np(gy), np.zeros((2, H, D, D)), "float32")
    for a, b, c in zip(torch.autograd.grad(y, ins, gy), want, bound):
        _close(a, b, c)


def test_attention_endless_gaps_forget():
    """A gap without end, and gaps of 1e30, are a fresh start; two in a row too, and at a chunk's and a stretch's edge."""
    N, H, D = 700, 1, 16
    gen = torch.Generator(device=DEV).manual_seed(3)
    q, k, v, gy = torch.randn(4, N, H, D, device=DEV, generator=gen)
    dt = torch.rand(N, device=DEV, generator=gen) * 0.1
    edges = [0, 5, 6, 64, 100, 256, 300, N]
    dt[5] = dt[6] = dt[64] = dt[256] = float("inf")
    dt[100], dt[300] = 1e30, 3e38
    rate = torch.ones(H, device=DEV)
    one = [a.clone().requires_grad_() for a in (q, k, v)]
    y, last = ops.decay_attention(*one, rate, torch.tensor([0, N], device=DEV), dt=dt)
    cut = [a.clone().requires_grad_() for a in (q, k, v)]
    ycut, lcut = ops.decay_attention(*cut, rate, torch.tensor(edges, device=DEV), dt=dt)
    assert torch.allclose(y, ycut, rtol=1e-5, atol=1e-5) and torch.allclose(last[0], lcut[-1], rtol=1e-5, atol=1e-5)
    for a, b in zip(torch.autograd.grad(y, one, gy), torch.autograd.grad(ycut, cut, gy)):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-5)
    state = torch.ones(1, H, D, D, device=DEV)
    ops.decay_attention_step(q[:1], k[:1], v[:1], rate, state, dt=dt[5:6])
    assert torch.equal(state[0, 0], k[0, 0, :, None] * v[0, 0, None])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [32, 64, 100, 128])
def test_attention_rounds_outputs_on_the_right_side(dtype, D):
    """States and pairs' weights meet an output within 2^-17 of themselves at most: next to the middle between two outputs, by 1.5
    times that, each output is still rounded to its own side."""
    step = torch.finfo(dtype).eps                            # between neighbours from one to two
    odd = torch.arange(1, 2 * D, 2, device=DEV, dtype=torch.float64) * (step / 2) + 1
    near = (odd[odd < 2][None, :] + torch.tensor([[-1.5], [1.5]], device=DEV, dtype=torch.float64) * 2.0 ** -17).flatten()
    if dtype == F32:
        near = 1 + torch.arange(2 * D, device=DEV, dtype=torch.float64) * step       # no pieces: the values themselves
    n = len(near)
    want = near.float().to(dtype)
    assert (near.float().double() == near).all()
    rate, start = torch.ones(1, device=DEV), torch.arange(n + 1, device=DEV)
    zero = torch.zeros(n, 1, D, device=DEV, dtype=dtype)
    # a state: every stream asks for its own row, next to other rows and columns of its size
    h0 = near[:, None, None, None].expand(n, 1, D, D).float().contiguous()
    q = zero.clone()
    q[torch.arange(n, device=DEV), 0, torch.arange(n, device=DEV) % D] = 1
    dt = torch.zeros(n, device=DEV)
    y, last = ops.decay_attention(q, zero, zero, rate, start, dt=dt, h0=h0, scale=1.0)
    assert torch.equal(last, h0) and torch.equal(y, want[:, None, None].expand(n, 1, D))
    # a pair's weight: three products of a query and its key that add up to it, times a value of one
    q, k, v = zero.clone(), zero.clone(), zero.clone()
    high = torch.floor((near - 1) / step) * step + 1
    half = torch.where(near - high > step / 4, step / 2, 0.0)
    for c, part in enumerate((high, half, near - high - half)):
        q[:, 0, c], k[:, 0, c] = part.to(dtype), 1
        assert (q[:, 0, c].double() == part).all()
    v[:, 0, 3] = 1
    y, _ = ops.decay_attention(q, k, v, rate, start, dt=dt, scale=1.0)
    assert torch.equal(y[:, 0, 3], want) and not y[:, 0, :3].any()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [8, 32, 64, 128])
def test_attention_of_small_channels_beside_large_ones(dtype, D):
    """A value channel keeps its bits next to one whose states are 2^35 times as large, in outputs and in the gradients that
    have channels of such sizes; the large ones belong to a key channel that no query asks for."""
    N, scale = 400, D ** -0.5
    gen = torch.Generator(device=DEV).manual_seed(D)
    q, k, v, gy = (torch.randn(N, 1, D, device=DEV, generator=gen) for _ in range(4))
    v *= 2.0 ** -12
    gy[..., 1:] *= 2.0 ** 4
    old = torch.arange(N, device=DEV) % 2 == 0               # half of the tokens have the large values
    k[old], v[old] = 0, 0
    k[old, 0, 0], v[old, 0, 0] = 1, 30000
    k[~old, 0, 0], v[~old, 0, 0], q[..., 0], gy[..., 0] = 0, 0, 0, 0
    q, k, v, gy = (t.to(dtype) for t in (q, k, v, gy))
    rate, start = torch.full((1,), 1 / 256, device=DEV), [0, 70, N]
    ins = [t.requires_grad_() for t in (q, k, v)]
    y, last = ops.decay_attention(*ins, rate, torch.tensor(start, device=DEV), scale=scale)
    got = (y, last, *torch.autograd.grad(y, ins, gy))
    zero = np.zeros((2, 1, D, D))
    want, mag = O.by_token(_np(q), _np(k), _np(v), _np(rate), start, None, None, scale, _np(gy), zero)
    units = (3 * D + 300 + 3 * (N // 32 + 1)) * 5 * O.U + O.PIECES[_name(dtype)]
    for name, a, b, c in zip(("y", "last", "gq", "gk", "gv"), got, want, mag):
        _close(a, b, units * c, name)
    assert np.abs(want[0]).max() < 1 and np.abs(want[1]).max() > 2.0 ** 20


def _states(x, dtype, start, dt, scale, rate):
    """last and gh0 of a call in a type, from h0 of zeros."""
    q, k, v, gy = (t.to(dtype) for t in x)
    h0 = torch.zeros(len(start) - 1, q.shape[1], q.shape[2], q.shape[2], device=DEV, requires_grad=True)
    y, last = ops.decay_attention(q, k, v, rate, torch.tensor(start, device=DEV), dt=dt, h0=h0, scale=scale)
    return last.detach(), torch.autograd.grad(y, h0, gy)[0]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [8, 32, 64, 128])
def test_attention_states_hold_24_bits(dtype, D):
    """A token's share of a state is its decay's 24 bits times its key and value: with powers of two for those, and one token a
    window that has any, states and their gradients have the bits of the single-precision call, over chunks and stretches;
    two pieces of the type could not hold them."""
    sizes = [1, 2, 5, 20, 33, 40, 70, 200, 300, 700, 1200, 2000]
    start = np.concatenate([[0], np.cumsum(sizes)]).tolist()
    N, gen = start[-1], torch.Generator(device=DEV).manual_seed(D)
    x = torch.zeros(4, N, 2, D, device=DEV)
    for b, n in enumerate(sizes):
        power = lambda: 2.0 ** torch.randint(-3, 4, (2, D), device=DEV, generator=gen)
        first, end = start[b] + n // 3, start[b + 1] - 1 - n // 3
        x[1, first], x[2, first], x[0, end], x[3, end] = power(), power(), power(), -power()
    dt = torch.rand(N, device=DEV, generator=gen) * 0.01
    rate = torch.tensor([0.9, 0.11], device=DEV)
    wide = _states(x, F32, start, dt, 0.3, rate)
    for a, b in zip(_states(x, dtype, start, dt, 0.3, rate), wide):
        two = b.to(dtype).float()
        two = two + (b - two).to(dtype).float()
        assert torch.equal(a, b) and b.any() and not torch.equal(two, b)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("N,D", [(40, 16), (300, 32), (700, 45), (700, 64), (3000, 128)])
def test_attention_states_are_as_good_as_single_precision(dtype, N, D):
    """last and gh0 next to the definition in 64 bits: sums of N products in 32 bits are off by some 2^-24 times a small number's
    root (2e-7), shares in two pieces of bfloat16 by 2^-17 or a third of it (3e-6) each and so in their root mean square."""
    gen = torch.Generator(device=DEV).manual_seed(N)
    q, k, v, gy = torch.randn(4, N, 1, D, device=DEV, generator=gen).to(dtype)
    dt, rate = torch.rand(N, device=DEV, generator=gen) * 0.01, torch.ones(1, device=DEV)
    got = _states((q, k, v, gy), dtype, [0, N], dt, 0.5, rate)
    zero = np.zeros((1, 1, D, D))
    want, _ = O.by_token(_np(q), _np(k), _np(v), _np(rate), [0, N], _np(dt), None, 0.5, _np(gy), zero)
    for a, b in zip(got, (want[1], want[5])):
        assert np.sqrt(((_np(a) - b) ** 2).mean() / (b ** 2).mean()) < 1e-6


def test_attention_without_decay_adds_up():
    ones = torch.ones(200, 1, 4, device=DEV)
    y, last = ops.decay_attention(ones, ones, ones, torch.zeros(1, device=DEV), torch.tensor([0, 200], device=DEV), scale=1.0)
    assert torch.equal(y[:, 0], 4.0 * torch.arange(1, 201, device=DEV)[:, None].expand(200, 4)) and torch.all(last == 200)


def test_attention_of_shared_heads():
    """Keys and values of one head for three heads of queries, as an expanded view: the results of the copied heads, and
    gradients added over them."""
    N, D = 300, 32
    gen = torch.Generator(device=DEV).manual_seed(5)
    q, gy = torch.randn(2, N, 6, D, device=DEV, generator=gen)
    kv = torch.randn(2, N, 2, D, device=DEV, generator=gen)
    rate, start = torch.rand(6, device=DEV, generator=gen), torch.tensor([0, 100, N], device=DEV)

    def go(copy):
        t = kv.clone().requires_grad_()
        k, v = (a[:, :, None].expand(N, 2, 3, D) for a in t)
        k, v = (a.reshape(N, 6, D).clone() if copy else a.reshape(N, 6, D) for a in (k, v))
        y, _ = ops.decay_attention(q, k, v, rate, start)
        return y, torch.autograd.grad(y, t, gy)[0]

    (a, ga), (b, gb) = go(False), go(True)
    assert torch.equal(a, b) and torch.equal(ga, gb)
    one = kv[:, :, :1].expand(2, N, 6, D)                     # a head stride of zero, taken as it lies
    assert one.stride(2) == 0
    y = ops.decay_attention(q, one[0], one[1], rate, start)[0]
    assert torch.equal(y, ops.decay_attention(q, one[0].contiguous(), one[1].contiguous(), rate, start)[0])


@pytest.mark.parametrize("Hk", [1, 2, 3])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_of_fewer_key_heads_as_documented(Hk, dtype):
    """Keys and values of one head as views, of more as copies, behind a rotation that has Hk heads of keys: the results of
    full heads, and gradients that are their sums."""
    N, H, D = 300, 6, 32
    gen = torch.Generator(device=DEV).manual_seed(Hk)
    q, gy = torch.randn(2, N, H, D, device=DEV, generator=gen).to(dtype)
    kv = torch.randn(2, N, Hk, D, device=DEV, generator=gen).to(dtype)
    rate, start = torch.rand(H, device=DEV, generator=gen), torch.tensor([0, 100, N], device=DEV)
    pos, fr = torch.rand(N, 1, device=DEV, generator=gen), torch.rand(8, device=DEV, generator=gen)
    k, v = (t.clone().requires_grad_() for t in kv)
    wide = (lambda t: t.expand(N, H, D)) if Hk == 1 else (lambda t: t.repeat_interleave(H // Hk, 1))
    qr, kr = ops.head_norm_rotary(q, k, None, None, pos, fr, (8,))
    y, last = ops.decay_attention(qr, wide(kr), wide(v), rate, start)
    full = [t.detach().repeat_interleave(H // Hk, 1).requires_grad_() for t in (kr, v)]
    y1, last1 = ops.decay_attention(qr, *full, rate, start)
    assert torch.equal(y, y1) and torch.equal(last, last1)
    got, per_head = torch.autograd.grad(y, (kr, v), gy, retain_graph=True), torch.autograd.grad(y1, full, gy)
    for a, b in zip(got, per_head):                          # sums of H / Hk numbers, rounded to the type at most that often
        parts = b.view(N, Hk, H // Hk, D).double()
        assert ((a.double() - parts.sum(2)).abs() <= H // Hk * torch.finfo(dtype).eps / 2 * parts.abs().sum(2)).all()
    assert all(g.any() for g in torch.autograd.grad(y, (k, v), gy))


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_attention_bad_values_stay_in_their_window(bad, dtype, which):
    """A NaN or infinity in one token leaves the tokens before it, other windows and other heads alone, in its chunk too; a
    bad query leaves every other token's output alone, a bad value every other channel."""
    N, H, D = 900, 2, 32
    start = torch.tensor([0, 200, 200, 750, N], device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(1)
    x = dict(zip("qkv", torch.randn(3, N, H, D, device=DEV, generator=gen).to(dtype)))
    dt, rate = torch.rand(N, device=DEV, generator=gen) * 0.01, torch.tensor([1.0, 0.1], device=DEV)
    yc, lc = ops.decay_attention(*x.values(), rate, start, dt=dt)
    x[which] = x[which].clone()
    x[which][430, 1, 3] = bad
    y, last = ops.decay_attention(*x.values(), rate, start, dt=dt)
    hit = torch.zeros(N, H, D, dtype=torch.bool, device=DEV)
    if which == "q":
        hit[430, 1] = True
    elif which == "k":
        hit[430:750, 1] = True
    else:
        hit[430:750, 1, 3] = True
    assert torch.equal(y[~hit], yc[~hit]) and not torch.isfinite(y[430, 1, 3])
    lhit = torch.zeros_like(lc, dtype=torch.bool)
    if which == "k":
        lhit[2, 1, 3] = True
    elif which == "v":
        lhit[2, 1, :, 3] = True
    assert torch.equal(last[~lhit], lc[~lhit]) and not torch.isfinite(last[lhit]).any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_attention_bad_gradients_stay_behind_their_token(bad, dtype):
    """A bad gradient of one output reaches the keys and values of no later token, in its chunk too, and no other query."""
    N, H, D = 900, 2, 32
    start = torch.tensor([0, 200, 750, N], device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(2)
    q, k, v, gy = torch.randn(4, N, H, D, device=DEV, generator=gen).to(dtype)
    rate = torch.tensor([0.01, 0.1], device=DEV)

    def go(g):
        ins = [a.clone().requires_grad_() for a in (q, k, v)]
        return torch.autograd.grad(ops.decay_attention(*ins, rate, start)[0], ins, g)

    clean = go(gy)
    gy = gy.clone()
    gy[430, 1, 3] = bad
    for n, (a, b) in enumerate(zip(go(gy), clean)):
        hit = torch.zeros(N, H, D, dtype=torch.bool, device=DEV)
        if n == 0:
            hit[430, 1] = True
        elif n == 1:
            hit[200:431, 1] = True
        else:
            hit[200:431, 1, 3] = True
        assert torch.equal(a[~hit], b[~hit]), n
        assert not torch.isfinite(a[430, 1, 3]), n


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [16, 32, 64, 128])
def test_attention_bad_gradients_reach_the_stretches_before(bad, dtype, D):
    """A bad gradient in a window's second stretch reaches its channel's values and its head's keys of the first one, and
    changes no bit of the others."""
    N, H, at = 900, 2, 700
    start = torch.tensor([0, 200, 750, N], device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(4)
    q, k, v, gy = torch.randn(4, N, H, D, device=DEV, generator=gen).to(dtype)
    rate = torch.tensor([0.01, 0.02], device=DEV)
    print(f"bad gradients {bad} {dtype} D={D}", flush=True)

    def go(g):
        ins = [a.clone().requires_grad_() for a in (q, k, v)]
        return torch.autograd.grad(ops.decay_attention(*ins, rate, start)[0], ins, g)

    clean = go(gy)
    gy = gy.clone()
    gy[at, 1, 3] = bad
    got = go(gy)
    hit = torch.zeros(3, N, H, D, dtype=torch.bool, device=DEV)
    hit[0, at, 1] = hit[1, 200:at + 1, 1] = hit[2, 200:at + 1, 1, 3] = True
    for n, (a, b) in enumerate(zip(got, clean)):
        assert torch.equal(a[~hit[n]], b[~hit[n]]), n
    assert not got[2][200:at + 1, 1, 3].isfinite().any() and not got[1][200:at + 1, 1].isfinite().any()


def _same_kinds(got, want, mag, units, dtype, what):
    """Infinities with their signs and NaN where the definition has them, and finite values within its bound."""
    want32 = want.astype(np.float32).astype(np.float64)      # what single precision can hold
    for kind, of in (("NaN", np.isnan), ("+Inf", np.isposinf), ("-Inf", np.isneginf)):
        a, b = of(_np(got)), of(want32)
        assert (a == b).all(), f"{what}: {kind} in {int((a & ~b).sum())} places too many, {int((b & ~a).sum())} too few"
    fine = np.isfinite(want32) & np.isfinite(mag)
    tol = units * mag[fine] + rounding(dtype, np.abs(want[fine]) + units * mag[fine])
    assert (np.abs(_np(got)[fine] - want[fine]) <= tol).all(), what


def _by_token_case(x, rate, start, dt, dtype, where, scale=0.5, pieces=True):
    """All outputs and gradients against the definition, exponents below 4 (5 units of a factor)."""
    N, H, D = x["q"].shape
    ins = [x[n].clone().requires_grad_() for n in ("q", "k", "v", "h0")]
    y, last = ops.decay_attention(*ins[:3], rate, torch.tensor(start, device=DEV), dt=dt, h0=ins[3], scale=scale)
    grads = torch.autograd.grad((y, last), ins, (x["gy"], x["glast"]))
    want, mag = O.by_token(*(_np(x[n]) for n in "qkv"), _np(rate), start, _np(dt), _np(x["h0"]), scale, _np(x["gy"]), _np(x["glast"]))
    units = (3 * D + 300 + 3 * (N // 32 + 1)) * 5 * O.U + O.PIECES[_name(dtype)]
    for n, (name, got) in enumerate(zip(("y", "last", "gq", "gk", "gv", "gh0"), (y, last, *grads))):
        _same_kinds(got, want[n], mag[n], units, got.dtype, f"{name} ({where})")


@pytest.mark.parametrize("D", [1, 8, 32, 45, 64, 100, 128])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_attention_infinities_go_where_the_formula_takes_them(D, dtype):
    """An infinity in each of the inputs in turn, and in all: signed infinities and NaN are those of the definition, in the
    token's chunk, later chunks, other stretches, states and gradients."""
    N, H, start = 700, 2, [0, 100, 640, 700]
    gen = torch.Generator(device=DEV).manual_seed(D)
    clean = {n: torch.randn(N, H, D, device=DEV, generator=gen).to(dtype) for n in ("q", "k", "v", "gy")}
    clean.update({n: torch.randn(3, H, D, D, device=DEV, generator=gen) for n in ("h0", "glast")})
    dt, rate = torch.rand(N, device=DEV, generator=gen) * 0.01, torch.tensor([1.0, 0.1], device=DEV)
    c, inf = D // 2, float("inf")
    bad = [("q", (150, 0, c), inf), ("k", (131, 1, c), -inf), ("v", (390, 0, D - 1), inf), ("gy", (420, 1, 0), -inf),
           ("h0", (1, 0, c, 0), inf), ("glast", (1, 1, 0, c), -inf), ("k", (99, 0, 0), inf), ("v", (639, 1, c), -inf)]
    for some in [[b] for b in bad] + [bad]:
        print(f"infinities D={D} {dtype} {[b[0] for b in some]}", flush=True)
        x = {n: t.clone() for n, t in clean.items()}
        for name, at, value in some:
            x[name][at] = value
        _by_token_case(x, rate, start, dt, dtype, "+".join(b[0] for b in some))


@pytest.mark.parametrize("N,D", [(2500, 8), (1600, 64), (17_000, 8)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_infinities_cross_joined_stretches(N, D, dtype):
    """Windows whose stretches' sums are joined, by a thread an element and in runs."""
    gen = torch.Generator(device=DEV).manual_seed(N)
    x = {n: torch.randn(N, 1, D, device=DEV, generator=gen).to(dtype) for n in ("q", "k", "v", "gy")}
    x.update({n: torch.randn(1, 1, D, D, device=DEV, generator=gen) for n in ("h0", "glast")})
    x["k"][40, 0, 1], x["gy"][N - 30, 0, 2] = float("inf"), float("-inf")
    dt, rate = torch.rand(N, device=DEV, generator=gen) * 8 / N, torch.ones(1, device=DEV)
    print(f"infinities across joins N={N} D={D} {dtype}", flush=True)
    _by_token_case(x, rate, [0, N], dt, dtype, "joined")


@pytest.mark.parametrize("D", [4, 64])
def test_attention_of_products_past_single_precision(D):
    """Queries and keys whose product is past float32, values so small that the outputs are not; and states past it."""
    N, dtype = 400, F32
    gen = torch.Generator(device=DEV).manual_seed(D)
    x = {n: torch.rand(N, 1, D, device=DEV, generator=gen) + 0.5 for n in ("q", "k", "v", "gy")}
    x.update({n: torch.zeros(1, 1, D, D, device=DEV) for n in ("h0", "glast")})
    x["q"][100:110] *= 1e25
    x["k"][90:95] *= 1e20
    x["v"][90:95] *= 1e-20
    _by_token_case(x, torch.ones(1, device=DEV), [0, N], torch.full((N,), 0.001, device=DEV), dtype, "large products")
    x["k"][300] = x["v"][300] = 1e25
    x["q"][:], x["gy"][:] = 1.0, 1.0
    _by_token_case(x, torch.ones(1, device=DEV), [0, N], torch.full((N,), 0.001, device=DEV), dtype, "large states")


def test_step_of_infinite_states():
    """An infinite state stays so, with its sign, until a factor of zero."""
    N, H, D, inf = 3, 1, 8, float("inf")
    q, k, v = torch.rand(3, N, H, D, device=DEV) + 0.5
    state = torch.zeros(N, H, D, D, device=DEV)
    state[0, 0, 2, 3], state[1, 0, 2, 3], k[2, 0, 1] = inf, -inf, inf
    rate, dt = torch.ones(H, device=DEV), torch.tensor([0.1, 2.0, 1.0], device=DEV)
    for _ in range(2):
        want = torch.exp(-dt.double())[:, None, None, None] * state.double() + k.double()[..., None] * v.double()[:, :, None]
        y = ops.decay_attention_step(q, k, v, rate, state, dt=dt, scale=1.0)
        assert torch.equal(state.isposinf(), want.isposinf()) and torch.equal(state.isneginf(), want.isneginf())
        assert torch.allclose(state, want.float(), rtol=1e-5) and not state.isnan().any()
        out = (q.double()[..., None] * want).sum(2)
        assert torch.equal(y.isposinf(), out.isposinf()) and torch.equal(y.isneginf(), out.isneginf())
        assert torch.allclose(y, out.float(), rtol=1e-5)
    ops.decay_attention_step(q, v, v, rate, state, dt=torch.full((N,), inf, device=DEV))
    assert state[2].isfinite().sum() == 56 and state[0, 0, 2, 3].isnan()       # zero times an infinity


def test_attention_bad_gaps_show():
    """A gap that is not a number makes its token's and the window's later outputs so, and the others' not."""
    N, H, D = 500, 2, 16
    q, k, v = torch.randn(3, N, H, D, device=DEV).to(BF16)
    dt, start = torch.rand(N, device=DEV), torch.tensor([0, 100, 400, N], device=DEV)
    dt[200] = float("nan")
    y, last = ops.decay_attention(q, k, v, torch.ones(H, device=DEV), start, dt=dt)
    hit = torch.zeros(N, dtype=torch.bool, device=DEV)
    hit[200:400] = True
    assert y[hit].isnan().all() and y[~hit].isfinite().all() and last[1].isnan().all() and last[[0, 2]].isfinite().all()


def test_attention_of_very_many_windows():
    """More windows than two steps of the 64-way search cover, empty ones among them, against single windows' sums."""
    rng = np.random.default_rng(15)
    sizes = rng.integers(0, 4, 9000)
    start = np.concatenate([[0], np.cumsum(sizes)])
    N, H, D = int(start[-1]), 1, 8
    q, k, v = (_t(a) for a in rng.normal(size=(3, N, H, D)))
    y, last = ops.decay_attention(q, k, v, torch.full((1,), 0.5, device=DEV), torch.tensor(start, device=DEV))
    args = (_np(q), _np(k), _np(v), np.array([0.5]), start.tolist(), None, None, D ** -0.5)
    (wy, wl), (by, bl) = O.attention(*args, "float32")
    _close(y, wy, by)
    _close(last, wl, bl)


def test_attention_among_a_million_empty_windows():
    N, H, D, empty = 300, 1, 4, 1_000_000
    q, k, v = torch.randn(3, N, H, D, device=DEV)
    rate = torch.ones(1, device=DEV)
    start = torch.cat([torch.zeros(empty, dtype=torch.int64, device=DEV), torch.full((empty,), N, device=DEV)])
    y, last = ops.decay_attention(q, k, v, rate, start)
    y1, l1 = ops.decay_attention(q, k, v, rate, torch.tensor([0, N], device=DEV))
    assert torch.equal(y, y1) and torch.equal(last[empty - 1], l1[0])
    assert not last[:empty - 1].any() and not last[empty:].any()


def test_attention_gradient_is_its_difference():
    N, H, D = 200, 1, 6
    gen = torch.Generator(device=DEV).manual_seed(4)
    x = torch.randn(3, N, H, D, device=DEV, generator=gen)
    h0 = torch.randn(2, H, D, D, device=DEV, generator=gen)
    gy, gl = torch.randn(N, H, D, device=DEV, generator=gen), torch.randn(2, H, D, D, device=DEV, generator=gen)
    rate, start = torch.full((1,), 0.2, device=DEV), torch.tensor([0, 70, N], device=DEV)

    def loss(x, h0):
        y, last = ops.decay_attention(*x, rate, start, h0=h0)
        return (y.double() * gy).sum() + (last.double() * gl).sum()

    a, b = x.clone().requires_grad_(), h0.clone().requires_grad_()
    grads = torch.autograd.grad(loss(a, b), (a, b))
    for t, g, go in ((x, grads[0], lambda s: loss(x + s, h0)), (h0, grads[1], lambda s: loss(x, h0 + s))):
        d = torch.randn(t.shape, device=DEV, generator=gen)
        step = 1e-3                                          # the loss is of third degree: the difference's own error is 1e-6 of it
        diff = (go(step * d) - go(-step * d)) / (2 * step)
        want = (g.double() * d).sum()
        mag = (g.double() * d).abs().sum()
        assert abs(diff - want) < 1e-3 * mag, (float(diff), float(want))


@pytest.mark.parametrize("dtype,N,H,D", [(F32, 1, 1, 1), (F32, 3, 2, 7), (BF16, 256, 4, 64), (F16, 33, 3, 45), (BF16, 0, 1, 8),
                                         (BF16, 70, 2, 128), (F32, 5, 1, 127), (F16, 5, 1, 100)])
@pytest.mark.parametrize("with_dt", [False, True])
@pytest.mark.parametrize("layout", [None, "slice", "odd", "heads"])
def test_step(dtype, N, H, D, with_dt, layout):
    rng = np.random.default_rng(N + D)
    q, k, v = (_t(a, dtype) for a in rng.normal(size=(3, N, H, D)))
    state, rate = _t(rng.normal(size=(N, H, D, D))), _t(rng.random(H))
    dt = _t(rng.exponential(size=N)) if with_dt else None
    was = _np(state)
    print(f"step N={N} H={H} D={D} {dtype} {layout}", flush=True)
    y = ops.decay_attention_step(*(_spread(a, layout) for a in (q, k, v)), rate, state, dt=dt, scale=0.3)
    z = _np(rate)[None] * (np.ones((N, 1)) if dt is None else _np(dt)[:, None])
    old, new = np.exp(-z)[..., None, None] * was, _np(k)[..., :, None] * _np(v)[..., None, :]
    # the factor less one (the exponent's rounding, two units, and one per unit of it), the sum and the product
    bound = O.U * (np.abs(was) * (4 + z)[..., None, None] + 2 * np.abs(new))
    _close(state, old + new, bound, "state")
    mag = np.abs(_np(q))[..., :, None] * (np.abs(old + new) + bound)
    _close(y, 0.3 * (_np(q)[..., :, None] * (old + new)).sum(-2),
           0.3 * ((np.abs(_np(q))[..., :, None] * bound).sum(-2) + (D + 4) * O.U * mag.sum(-2)), "y")


def test_step_follows_attention():
    N, H, D = 90, 2, 32
    q, k, v = torch.randn(3, N, H, D, device=DEV)
    rate, dt = torch.rand(H, device=DEV), torch.rand(N, device=DEV) * 0.1
    y, last = ops.decay_attention(q, k, v, rate, torch.tensor([0, N], device=DEV), dt=dt)
    state = torch.zeros(1, H, D, D, device=DEV)
    for i in range(N):
        out = ops.decay_attention_step(q[i:i + 1], k[i:i + 1], v[i:i + 1], rate, state, dt=dt[i:i + 1])
        assert torch.allclose(out[0], y[i], rtol=1e-4, atol=1e-4)
    assert torch.allclose(state, last, rtol=1e-4, atol=1e-4)


# ------------------------------------------------------------------------------------------- norm and rotation
def _rotary_case(N, H, Hk, D, sections, dtype, norm=True, layout=None, seed=0, far=100.0, pos_type=F32, eps=1e-6):
    rng = np.random.default_rng(seed)
    q, k = _t(rng.normal(size=(N, H, D)) * 2, dtype), _t(rng.normal(size=(N, Hk, D)) * 2, dtype)
    gq, gk = _t(rng.normal(size=(N, H, D)), dtype), _t(rng.normal(size=(N, Hk, D)), dtype)
    wq, wk = (_t(rng.normal(size=D)) for _ in range(2)) if norm else (None, None)
    pos = torch.as_tensor(rng.random((N, len(sections))) * far, device=DEV).to(pos_type)
    freqs = _t(rng.random(sum(sections)) * 2)
    print(f"rotary N={N} H={H},{Hk} D={D} {sections} {dtype} norm={norm} {layout}", flush=True)
    qs, ks, gqs, gks = (_spread(a, layout).detach() for a in (q, k, gq, gk))
    ins = [t.requires_grad_() for t in (qs, ks, wq, wk) if t is not None]
    got = ops.head_norm_rotary(qs, ks, wq, wk, pos, freqs, sections, eps=eps)
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(got, ops.head_norm_rotary(qs, ks, wq, wk, pos, freqs, sections, eps=eps)))
    grads = torch.autograd.grad(got, ins, (gqs, gks), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(got, ins, (gqs, gks))))
    angle = O.angles(_np(pos), _np(freqs), sections)
    for j, (x, w, g, y) in enumerate(((q, wq, gq, got[0]), (k, wk, gk, got[1]))):
        assert y.is_contiguous()
        _close(y, *O.rotary(_np(x), _np(w), angle, eps), "y")
        (gx, gw), (bx, bw) = O.rotary_bwd(_np(x), _np(w), angle, eps, _np(g))
        _close(grads[j], gx, bx, "gx")
        if norm:
            _close(grads[2 + j], gw, bw, "gw")


@pytest.mark.parametrize("D", [1, 2, 3, 7, 8, 9, 24, 32, 46, 64, 65, 100, 128, 200, 255, 256])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("norm", [True, False])
def test_rotary_widths(D, dtype, norm):
    p = D // 2
    _rotary_case(70, 3, 2, D, (p - p // 2, p // 2), dtype, norm, seed=D)


@pytest.mark.parametrize("sections", [(16,), (0, 16), (4, 5, 7), (1, 2, 3, 4), (0,), (0, 0, 3, 0)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rotary_sections(sections, dtype):
    _rotary_case(50, 2, 1, 32, sections, dtype, seed=len(sections))


@pytest.mark.parametrize("N", [0, 1, 2, 31, 257, 5000, 40_001])
@pytest.mark.parametrize("H,Hk", [(1, 1), (4, 2), (13, 5)])
def test_rotary_tokens(N, H, Hk):
    _rotary_case(min(N, 200_000 // (H + Hk)), H, Hk, 32, (8, 8), BF16, seed=N)


@pytest.mark.parametrize("layout", ["slice", "odd", "heads", "cols"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rotary_layouts(layout, dtype):
    _rotary_case(90, 3, 2, 64, (10, 22), dtype, layout=layout, seed=7)


@pytest.mark.parametrize("pos_type", [F32, torch.float64, torch.int64, torch.int32, torch.float16])
def test_rotary_position_types(pos_type):
    _rotary_case(60, 2, 2, 16, (3, 5), F32, seed=8, pos_type=pos_type, far=1000.0)


@pytest.mark.parametrize("far,pos_type", [(1e6, F32), (1e9, torch.float64), (1e9, torch.int64)])
def test_rotary_of_far_positions(far, pos_type):
    """Angles of a billion radians: in 64 bits they are off by 1e9 2^-52 = 2e-7 at most, a few units."""
    _rotary_case(60, 2, 2, 16, (3, 5), F32, seed=9, pos_type=pos_type, far=far)


@pytest.mark.parametrize("pos_type", [F32, torch.float64, torch.int64])
@pytest.mark.parametrize("freq_type", [F32, torch.float64, BF16])
def test_rotary_frequency_types(pos_type, freq_type):
    """Frequencies are taken as they are given: at a position of 2^24 one in 64 bits would be off by half a radian in 32."""
    N, H, D = 40, 2, 12
    gen = torch.Generator().manual_seed(3)
    q, k, gq, gk = (torch.randn(N, H, D, generator=gen).to(DEV) for _ in range(4))
    pos = (torch.rand(N, 2, generator=gen, dtype=torch.float64) * 2 ** 24).floor().to(pos_type).to(DEV)
    fr = torch.rand(6, generator=gen, dtype=torch.float64).to(freq_type).to(DEV)
    ins = [t.requires_grad_() for t in (q, k)]
    got = ops.head_norm_rotary(*ins, None, None, pos, fr, (2, 4))
    grads = torch.autograd.grad(got, ins, (gq, gk))
    angle = O.angles(_np(pos), _np(fr), (2, 4))
    for x, g, y, gx in zip((q, k), (gq, gk), got, grads):
        _close(y, *O.rotary(_np(x), None, angle, 0.0), "y")
        (want, _), (bound, _) = O.rotary_bwd(_np(x), None, angle, 0.0, _np(g))
        _close(gx, want, bound, "gx")


def test_rotary_of_zeros_and_bad_rows():
    """A row of zeros stays zero; a NaN or an infinity in a head or a position leaves the others alone."""
    N, D = 40, 16
    q, k = torch.randn(2, N, 3, D, device=DEV)
    w = torch.ones(D, device=DEV)
    pos, fr = torch.rand(N, 2, device=DEV), torch.rand(6, device=DEV)
    clean = ops.head_norm_rotary(q, k, w, w, pos, fr, (2, 4))
    q[3] = 0
    q[5, 1, 2] = float("nan")
    k[7, 2, 15] = float("inf")
    pos[9, 0] = float("nan")
    got = ops.head_norm_rotary(q, k, w, w, pos, fr, (2, 4))
    assert not got[0][3].any() and got[0][5, 1].isnan().all() and not got[1][7, 2].isfinite().all()
    hit = [torch.zeros(N, 3, D, dtype=torch.bool, device=DEV) for _ in range(2)]
    hit[0][3], hit[0][5, 1], hit[1][7, 2] = True, True, True
    for h in hit:
        h[9, :, :4] = True
    for a, b, h in zip(got, clean, hit):
        assert torch.equal(a[~h], b[~h]) and a[9, :, :4].isnan().all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D,sections", [(16, (1, 2)), (16, (3,)), (15, (2,)), (12, (0,))])
def test_rotary_leaves_unturned_channels_alone(bad, dtype, D, sections):
    """Without norms a channel past the sections is passed on as it is, whatever it holds, and so is its neighbour; in the
    backward pass too, and a norm's weight gradient of the neighbour stays as it was."""
    N, H, turned = 20, 2, 2 * sum(sections)
    q, k, gq, gk = torch.randn(4, N, H, D, device=DEV).to(dtype)
    w = torch.rand(D, device=DEV) + 0.5
    pos, fr = torch.rand(N, len(sections), device=DEV), torch.rand(turned // 2, device=DEV)
    print(f"unturned channels {bad} {dtype} D={D} {sections}", flush=True)

    def go(q, gk):
        ins = [t.clone().requires_grad_() for t in (q, k)]
        out = ops.head_norm_rotary(*ins, None, None, pos, fr, sections)
        return [*out, *torch.autograd.grad(out, ins, (gq, gk))]

    clean, hit = go(q, gk), [torch.zeros(N, H, D, dtype=torch.bool, device=DEV) for _ in range(4)]
    q, gk = q.clone(), gk.clone()
    for n, c in enumerate(range(turned, D)):                 # of the even and of the odd channels, each in a row of its own
        q[n, 0, c], gk[n, 1, c] = bad, bad
        hit[0][n, 0, c] = hit[3][n, 1, c] = True
    for a, b, h in zip(go(q, gk), clean, hit):
        assert torch.equal(a[~h], b[~h]) and not a[h].isfinite().any()
        assert bad != bad or bool((a[h] == bad).all())

    def weights(g):
        ins = [w.clone().requires_grad_() for _ in range(2)]
        out = ops.head_norm_rotary(q0, k, *ins, pos, fr, sections)
        return torch.autograd.grad(out, ins, (g, gk0))

    q0, gk0 = torch.randn(2, N, H, D, device=DEV).to(dtype)
    g = gq.clone()
    g[4, 1, D - 1] = bad
    (a, ak), (b, bk) = weights(g), weights(gq)
    assert torch.equal(a[:-1], b[:-1]) and not a[-1].isfinite() and torch.equal(ak, bk)


def test_rotary_gradients_of_some():
    """Each input's gradient alone, and from one output alone, is the one it has beside the others."""
    N, D = 30, 16
    q, k, gq, gk = torch.randn(4, N, 2, D, device=DEV)
    wq, wk = torch.randn(2, D, device=DEV)
    pos, fr = torch.rand(N, 1, device=DEV), torch.rand(5, device=DEV)
    run = lambda ins: ops.head_norm_rotary(*ins, pos, fr, (5,))
    full = [t.clone().requires_grad_() for t in (q, k, wq, wk)]
    want = torch.autograd.grad(run(full), full, (gq, gk))
    for j in range(4):
        part = [t.clone().requires_grad_(n == j) for n, t in enumerate((q, k, wq, wk))]
        out = run(part)
        assert torch.equal(torch.autograd.grad(out, part[j], (gq, gk))[0], want[j])
    for j in range(2):
        got = torch.autograd.grad(run(full)[j], full, (gq, gk)[j], allow_unused=True)
        assert torch.equal(got[j], want[j]) and torch.equal(got[2 + j], want[2 + j])
        assert got[1 - j] is None or not got[1 - j].any()


# ------------------------------------------------------------------------------------------- together
def _block(N=3000, H=4, D=32, seed=4):
    """A layer as it is used: a projection, its heads normed and rotated, attention; as (step, leaves)."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(N, 64, device=DEV, generator=gen).to(BF16).requires_grad_()
    into = (torch.randn(3 * H * D, 64, device=DEV, generator=gen) / 8).to(BF16).requires_grad_()
    wq, wk = (torch.ones(D, device=DEV, requires_grad=True) for _ in range(2))
    pos, fr = torch.rand(N, 2, device=DEV, generator=gen) * 600, 2.0 ** -torch.arange(D // 2, device=DEV)
    rate, dt = torch.rand(H, device=DEV, generator=gen), torch.rand(N, device=DEV, generator=gen) * 0.01
    start = torch.tensor([0, 900, N], device=DEV)
    gy = torch.randn(N, H, D, device=DEV, generator=gen).to(BF16)
    gl = torch.randn(2, H, D, D, device=DEV, generator=gen)

    def step():
        q, k, v = torch.nn.functional.linear(x, into).view(N, 3, H, D).unbind(1)
        q, k = ops.head_norm_rotary(q, k, wq, wk, pos, fr, (D // 4, D // 4))
        y, last = ops.decay_attention(q, k, v, rate, start, dt=dt)
        return y, last, *torch.autograd.grad((y, last), (x, into, wq, wk), (gy, gl))

    return step, x


def test_operators_on_another_stream():
    step, _ = _block()
    here = step()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        there = step()
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a, b) for a, b in zip(here, there))


def test_operators_in_a_graph():
    """Two blocks recorded and replayed in turn with eager work between: every replay gives the eager bits."""
    blocks = [_block(), _block(N=1500, seed=6)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for step, _ in blocks:
            step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for step, _ in blocks:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for r in range(3):
        for (step, x), g, out in zip(blocks, graphs, outs):
            with torch.no_grad():
                x.add_(0.1 * r)
            want = step()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), r


def test_gradients_of_states_alone_in_a_graph():
    """The zeros that stand for a gradient of y are made in every replay, also where infinities come and go between them."""
    N, H, D = 1500, 2, 32
    gen = torch.Generator(device=DEV).manual_seed(9)
    q, k, v = (torch.randn(N, H, D, device=DEV, generator=gen).to(BF16).requires_grad_() for _ in range(3))
    gl, rate = torch.randn(1, H, D, D, device=DEV, generator=gen), torch.full((H,), 0.01, device=DEV)
    start = torch.tensor([0, N], device=DEV)

    def step():
        last = ops.decay_attention(q, k, v, rate, start)[1]
        return last, *torch.autograd.grad(last, (q, k, v), gl)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for r in range(4):
        with torch.no_grad():
            k.normal_(), v.normal_()
            q[100 * r] = float("inf") if r % 2 else 1.0
            v[700, 0, 3] = float("inf") if r == 2 else 0.5
        want = step()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) or (a.isnan() == b.isnan()).all() and torch.equal(a.nan_to_num(), b.nan_to_num())
                   for a, b in zip(out, want)), r
        assert not out[1].any()


def test_step_in_a_graph():
    """A recorded step follows its state from replay to replay."""
    N, H, D = 40, 2, 32
    q, k, v = torch.randn(3, N, H, D, device=DEV)
    rate, dt = torch.rand(H, device=DEV), torch.rand(N, device=DEV)
    state, eager = torch.zeros(N, H, D, D, device=DEV), torch.zeros(N, H, D, D, device=DEV)
    ops.decay_attention_step(q, k, v, rate, state.clone(), dt=dt)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.decay_attention_step(q, k, v, rate, state, dt=dt)
    for r in range(4):
        q.normal_(), k.normal_()
        want = ops.decay_attention_step(q, k, v, rate, eager, dt=dt)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(state, eager), r


def test_offsets_past_32_bits():
    """Rows whose offsets pass 2^31 elements and 2^32 bytes: the last window against a call on it alone."""
    H, D, tail = 4, 64, 777
    N = 2 ** 31 // (H * D) + 5000
    print(f"past 32 bits: N={N}", flush=True)
    small = torch.randn(4, tail, H, D, device=DEV).to(BF16)
    big = [torch.zeros(N, H, D, dtype=BF16, device=DEV) for _ in range(4)]
    for a, b in zip(big, small):
        a[-tail:] = b
    rate, start = torch.full((H,), 0.01, device=DEV), torch.tensor([0, N - tail, N], device=DEV)
    ins = [a.requires_grad_() for a in big[:3]]
    y, last = ops.decay_attention(*ins, rate, start)
    few = [a.clone().requires_grad_() for a in small[:3]]
    y1, last1 = ops.decay_attention(*few, rate, torch.tensor([0, tail], device=DEV))
    u = torch.finfo(BF16).eps
    near = lambda a, b: (a.float() - b.float()).abs().max() <= 2 * u * b.float().abs().max()
    assert near(y[-tail:], y1) and torch.allclose(last[1], last1[0], rtol=1e-4, atol=1e-3) and not y[:-tail].any()
    for a, b in zip(torch.autograd.grad(y, ins, big[3]), torch.autograd.grad(y1, few, small[3])):
        assert near(a[-tail:], b) and not a[:-tail].any()
    del y, last
    w, pos, fr = torch.ones(D, device=DEV), torch.rand(N, 2, device=DEV), torch.rand(32, device=DEV)
    with torch.no_grad():
        a = ops.head_norm_rotary(big[0], big[1], w, w, pos, fr, (16, 16))
        b = ops.head_norm_rotary(small[0], small[1], w, w, pos[-tail:], fr, (16, 16))
    assert all(torch.equal(x[-tail:], z) for x, z in zip(a, b))


def test_states_past_32_bits():
    """A step of streams whose states pass 2^31 elements."""
    N, H, D, tail = 2 ** 31 // (128 * 128) + 50, 1, 128, 30
    print(f"states past 32 bits: N={N}", flush=True)
    q, k, v = torch.randn(3, N, H, D, device=DEV).to(BF16)
    state = torch.zeros(N, H, D, D, device=DEV)
    few = state[-tail:].clone()
    rate = torch.ones(H, device=DEV)
    y = ops.decay_attention_step(q, k, v, rate, state)
    assert torch.equal(y[-tail:], ops.decay_attention_step(q[-tail:], k[-tail:], v[-tail:], rate, few))
    assert torch.equal(state[-tail:], few)


def test_calls_of_several_launches():
    """More workgroups than a launch takes: windows and streams of the second launch against calls on them alone."""
    tail, D = 300, 1
    N = 2 ** 25 + tail - 7
    print(f"several launches: step N={N}", flush=True)
    x = torch.randn(N, 1, D, device=DEV)
    state, rate = torch.ones(N, 1, D, D, device=DEV), torch.ones(1, device=DEV)
    y = ops.decay_attention_step(x, x, x, rate, state)
    few = torch.ones(tail, 1, D, D, device=DEV)
    assert torch.equal(y[-tail:], ops.decay_attention_step(x[-tail:], x[-tail:], x[-tail:], rate, few))
    assert torch.equal(state[-tail:], few)
    B = 2 ** 23 + 500
    print(f"several launches: attention of {B} windows", flush=True)
    start = torch.arange(B + 1, device=DEV)
    q = torch.randn(B, 1, D, device=DEV)
    y, last = ops.decay_attention(q, q, q, rate, start)
    assert torch.equal(last[..., 0, 0], (q * q)[..., 0]) and torch.allclose(y, q ** 3, rtol=1e-6)
    print("several launches: rotation", flush=True)
    n = 2 ** 24 + 77
    q, pos = torch.randn(n, 1, 128, dtype=BF16, device=DEV), torch.rand(n, 1, device=DEV)
    a, _ = ops.head_norm_rotary(q, q, None, None, pos, torch.ones(4, device=DEV), (4,))
    b, _ = ops.head_norm_rotary(q[-tail:], q[-tail:], None, None, pos[-tail:], torch.ones(4, device=DEV), (4,))
    assert torch.equal(a[-tail:], b)


# ------------------------------------------------------------------------------------------- beside autograd
def test_step_after_a_use_of_its_state_is_noticed():
    q, k, v = torch.randn(3, 6, 2, 8, device=DEV)
    state, rate = torch.randn(6, 2, 8, 8, device=DEV), torch.ones(2, device=DEV)
    w = torch.randn(8, 8, device=DEV, requires_grad=True)
    kq = q.clone().requires_grad_()
    product = torch.nn.functional.linear(state, w)
    y, _ = ops.decay_attention(kq, k, v, rate, torch.arange(7, device=DEV), h0=state)
    before = state._version
    ops.decay_attention_step(q, k, v, rate, state)
    assert state._version > before
    for out, wrt in ((product, w), (y, kq)):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out.sum(), wrt)
    with torch.inference_mode():
        inner = torch.zeros(6, 2, 8, 8, device=DEV)
        assert ops.decay_attention_step(q, k, v, rate, inner).isfinite().all() and inner.any()


def test_second_derivatives_are_refused():
    q, k, v = (torch.randn(10, 1, 8, device=DEV, requires_grad=True) for _ in range(3))
    rate, start = torch.ones(1, device=DEV), torch.tensor([0, 10], device=DEV)
    pos, fr = torch.rand(10, 1, device=DEV), torch.rand(4, device=DEV)
    for out in (ops.decay_attention(q, k, v, rate, start)[0], ops.head_norm_rotary(q, k, None, None, pos, fr, (4,))[0]):
        first, = torch.autograd.grad(out.square().sum(), q, create_graph=True)
        with pytest.raises(RuntimeError):
            first.sum().backward()


def _calls():
    """The operators as functions of one float tensor, and such a tensor."""
    start, rate = torch.tensor([0, 2, 6], device=DEV), torch.rand(2, device=DEV)
    other, w = torch.randn(6, 2, 8, device=DEV), torch.rand(8, device=DEV) + 0.5
    pos, fr = torch.rand(6, 2, device=DEV), torch.rand(4, device=DEV)
    return torch.randn(6, 2, 8, device=DEV), {
        "rotary": lambda t: torch.stack(ops.head_norm_rotary(t, other, w, w, pos, fr, (2, 2))),
        "weight": lambda t: ops.head_norm_rotary(other, other, t[0, 0], w, pos, fr, (2, 2))[0],
        "attention": lambda t: ops.decay_attention(t, other, other, rate, start)[0],
        "values": lambda t: torch.cat([a.flatten() for a in ops.decay_attention(other, other, t, rate, start)]),
        "step": lambda t: ops.decay_attention_step(t, other, other, rate, torch.ones(6, 2, 8, 8, device=DEV)),
    }


@pytest.mark.parametrize("which", ["rotary", "weight", "attention", "values"])
def test_forward_mode_derivatives_are_refused(which):
    t, calls = _calls()
    want = calls[which](t)
    with torch.autograd.forward_ad.dual_level():
        assert torch.equal(calls[which](t), want)
        with pytest.raises((RuntimeError, NotImplementedError)):
            calls[which](torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)))


@pytest.mark.parametrize("which", ["rotary", "weight", "attention", "values", "step"])
@pytest.mark.parametrize("grad", [False, True])
def test_recorded_calls_compute_or_are_refused(which, grad):
    from torch.fx.experimental.proxy_tensor import make_fx
    t, calls = _calls()
    fn = calls[which]
    t.requires_grad_(grad)
    for how in ({}, {"pre_dispatch": True}, {"tracing_mode": "fake"}):
        with pytest.raises(RuntimeError, match="recorded"):
            make_fx(fn, **how)(t)
    if which == "step":
        with pytest.raises(RuntimeError, match="recorded"):
            torch.jit.trace(fn, (t,), check_trace=False)
        return
    traced = torch.jit.trace(fn, (t,), check_trace=False)
    for _ in range(3):
        new = torch.randn_like(t)
        assert torch.equal(traced(new), fn(new))


@pytest.mark.parametrize("which", ["rotary", "attention", "step"])
@pytest.mark.parametrize("grad", [False, True])
def test_compiled_calls_compute(which, grad):
    t, calls = _calls()
    torch._dynamo.reset()
    fn = torch.compile(lambda a: calls[which](a * 2) + 1, backend="eager")
    for _ in range(2):
        t = torch.randn_like(t).requires_grad_(grad)
        got, want = fn(t), calls[which](t * 2) + 1
        assert torch.equal(got, want)
        if grad and want.requires_grad:
            assert torch.equal(torch.autograd.grad(got.sum(), t)[0], torch.autograd.grad(want.sum(), t)[0])


@pytest.mark.parametrize("which", ["rotary", "weight", "attention", "values", "step"])
def test_transforms_raise(which):
    t, calls = _calls()
    fn = calls[which]
    for call in (lambda: torch.func.vmap(fn)(torch.stack([t, t])), lambda: torch.func.grad(lambda a: fn(a).sum())(t),
                 lambda: torch.func.jvp(fn, (t,), (t,)), lambda: torch.func.functionalize(fn)(t)):
        with pytest.raises(RuntimeError):
            call()
    if which != "step":
        x = t.clone().requires_grad_()
        y = fn(x)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, x, torch.stack([torch.ones_like(y)] * 2), is_grads_batched=True)
