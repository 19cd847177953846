"""The sequence operators' HIP kernels against the float64 oracle, with its bounds on single precision's roundings and
half a unit of the output's type: types, widths, lengths, strides, alignments, empty windows and rows, NaN and
infinities that stay where they are, streams, graphs, offsets past 32 bits, and equal bits on equal calls."""
import numpy as np
import pytest
import torch

from tests import sequence_oracle as O
from x_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _t(a, dtype=F32):
    return None if a is None else torch.as_tensor(a, device=DEV).to(dtype)


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _close(got, want, bound, what=""):
    dtype, got = got.dtype, _np(got)
    assert got.shape == want.shape, (got.shape, want.shape)
    tol = bound + O.rounding(dtype, np.abs(want) + bound)
    err = np.abs(got - want)
    bad = ~(err <= tol)
    if bad.any():
        pytest.fail(f"{what}: {int(bad.sum())} of {bad.size} off, worst {np.max(np.where(bad, err / tol, 0)):.3g} of the bound")


def _spread(a, how):
    """The same rows in another layout: 'slice' of wider rows, 'odd' a slice that starts off alignment, 'cols' columns
    apart (copied by the operator)."""
    if how == "slice":
        wide = torch.zeros(a.shape[0], a.shape[1] + 24, dtype=a.dtype, device=a.device)
        wide[:, 8:8 + a.shape[1]] = a
        return wide[:, 8:8 + a.shape[1]]
    if how == "odd":
        wide = torch.zeros(a.shape[0], a.shape[1] + 3, dtype=a.dtype, device=a.device)
        wide[:, 1:1 + a.shape[1]] = a
        return wide[:, 1:1 + a.shape[1]]
    if how == "cols":
        return a.t().contiguous().t()
    return a


# ------------------------------------------------------------------------------------------- recurrence
def _windows(kind, N, rng):
    if kind == "one":
        return [0, N]
    if kind == "ragged":                                     # with empty windows at both ends and between
        cuts = np.sort(rng.integers(0, N + 1, 9))
        return [0, 0, *np.repeat(cuts, 2).tolist(), N, N]
    if kind == "short":                                      # more windows than a wave's search takes in one step
        return list(range(0, N, 3)) + [N, N]
    raise ValueError(kind)


def _scan_case(N, D, dtype, kind, with_dt, with_h0, layout, seed, grads=("y", "last"), gap=None):
    rng = np.random.default_rng(seed)
    start = _windows(kind, N, rng)
    B = len(start) - 1
    x, g, gy = (_t(rng.normal(size=(N, D)) * s - m, dtype) for s, m in ((1, 0), (2, 1), (1, 0)))
    dt = None if not with_dt else _t(rng.exponential(size=N) * (gap or 8 * B / max(N, 1)))
    h0 = _t(rng.normal(size=(B, D))) if with_h0 else None
    gl = _t(rng.normal(size=(B, D)))
    print(f"scan N={N} D={D} {dtype} {kind} B={B} dt={with_dt} h0={with_h0} {layout}", flush=True)
    xs, gs, ys = (_spread(a, layout).detach() for a in (x, g, gy))
    xs.requires_grad_(), gs.requires_grad_()
    if h0 is not None:
        h0.requires_grad_()
    st = torch.tensor(start, device=DEV)
    y, last = ops.gated_scan(xs, gs, st, dt=dt, h0=h0)
    args = (_np(x), _np(g), start)
    wy, wl, E = O.scan(*args, _np(dt), _np(h0))
    _close(y, wy, E, "y")
    tail = np.array(start[1:]) - 1
    some = np.diff(start) > 0
    El = np.where(some[:, None], E[np.maximum(tail, 0)], 0) if N else 0
    _close(last, wl, El, "last")
    with torch.no_grad():
        y2, last2 = ops.gated_scan(xs, gs, st, dt=dt, h0=h0)
    assert torch.equal(y, y2) and torch.equal(last, last2)
    wrt = (xs, gs) if h0 is None else (xs, gs, h0)
    outs = [(y, ys)] * ("y" in grads) + [(last, gl)] * ("last" in grads)
    got = torch.autograd.grad([a for a, _ in outs], wrt, [b for _, b in outs], retain_graph=True)
    gyn = _np(gy) if "y" in grads else np.zeros((N, D))
    gln = _np(gl) if "last" in grads else np.zeros((B, D))
    want, bound = O.scan_bwd(*args, gyn, gln, _np(dt), _np(h0))
    for name, a, b, c in zip(("gx", "gg", "gh0"), got, want, bound):
        _close(a, b, c, name)
    again = torch.autograd.grad([a for a, _ in outs], wrt, [b for _, b in outs])
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("N", [0, 1, 2, 15, 16, 17, 255, 257, 1000, 4099])
@pytest.mark.parametrize("dtype,D", [(F32, 5), (BF16, 64), (F16, 1)])
def test_scan_lengths(N, dtype, D):
    _scan_case(N, D, dtype, "ragged", True, True, None, seed=N)


@pytest.mark.parametrize("D", [1, 2, 3, 4, 7, 8, 12, 31, 32, 48, 65, 128, 130, 256, 257, 300, 520])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_widths(D, dtype):
    _scan_case(700, D, dtype, "ragged", D % 2 == 0, D % 3 == 0, None, seed=D)


@pytest.mark.parametrize("layout", ["slice", "odd", "cols"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_scan_layouts(layout, dtype):
    _scan_case(600, 64, dtype, "ragged", True, False, layout, seed=11)


@pytest.mark.parametrize("kind", ["one", "short"])
@pytest.mark.parametrize("with_dt", [False, True])
def test_scan_windows(kind, with_dt):
    _scan_case(9001, 16, F32, kind, with_dt, True, None, seed=12)


@pytest.mark.parametrize("grads", [("y",), ("last",)])
def test_scan_partial_gradients(grads):
    _scan_case(300, 24, F32, "ragged", True, True, None, seed=13, grads=grads)


@pytest.mark.parametrize("gap", [1e-6, 1.0, 1e4])
def test_scan_gaps(gap):
    """From gaps far below the time constant (decays next to one over all tokens) to gaps that forget everything."""
    _scan_case(5000, 8, F32, "one", True, False, None, seed=14, gap=gap)


def test_scan_gaps_back_in_time():
    """Events out of order: negative gaps grow the state as the formula has it, within a group of tokens, over whole
    groups and over workgroups, forward and backward."""
    N, D = 3000, 8
    rng = np.random.default_rng(21)
    gap = rng.exponential(size=N) * 0.05
    gap[rng.random(N) < 0.3] *= -1
    gap[1000:1100] = -np.abs(gap[1000:1100])
    x, g, gy = (rng.normal(size=(N, D)) for _ in range(3))
    start = [0, 2000, N]
    ins = [_t(a).requires_grad_() for a in (x, g)]
    dt = _t(gap)
    y, last = ops.gated_scan(*ins, torch.tensor(start, device=DEV), dt=dt)
    args = (_np(ins[0]), _np(ins[1]), start)
    wy, wl, E = O.scan(*args, _np(dt))
    _close(y, wy, E, "y")
    _close(last, wl, E[np.array(start[1:]) - 1], "last")
    got = torch.autograd.grad(y, ins, _t(gy))
    want, bound = O.scan_bwd(*args, _np(_t(gy)), np.zeros((2, D)), _np(dt))
    for name, a, b, c in zip(("gx", "gg"), got, want, bound):
        _close(a, b, c, name)
    state = torch.ones(D, D, device=DEV)
    one = O.scan(_np(ins[0][:D]), _np(ins[1][:D]), list(range(D + 1)), _np(-dt[:D].abs()), np.ones((D, D)))
    ops.gated_scan_step(ins[0][:D].detach(), ins[1][:D].detach(), state, dt=-dt[:D].abs())
    _close(state, one[1], one[2], "state")


def test_scan_equal_times_add_up():
    x, g = torch.ones(40, 8, device=DEV), torch.zeros(40, 8, device=DEV)
    y, last = ops.gated_scan(x, g, torch.tensor([0, 40], device=DEV), dt=torch.zeros(40, device=DEV))
    assert torch.equal(y, torch.arange(1, 41, device=DEV)[:, None].expand(40, 8) * 0.5)


def test_scan_extreme_gates():
    """A gate of +-100 and +-infinity: the weight is one or zero, and nothing overflows."""
    N, D = 64, 4
    g = torch.tensor([100.0, -100.0, float("inf"), -float("inf")], device=DEV).expand(N, D)
    x = torch.randn(N, D, device=DEV)
    y, _ = ops.gated_scan(x, g, torch.tensor([0, N], device=DEV))
    assert torch.equal(y[:, 0], x[:, 0]) and torch.equal(y[:, 2], x[:, 2])
    assert y[:, 1].abs().max() < 1e-40 and not y[:, 3].any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_scan_bad_values_stay_in_their_window(bad):
    """A NaN or infinity in one window, channel and token leaves the other windows, channels and earlier tokens alone,
    forward and backward, also across workgroups."""
    N, D = 6000, 8
    start = torch.tensor([0, 2500, 2500, 3100, N], device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(1)
    x, g, gy = torch.randn(3, N, D, device=DEV, generator=gen)
    dt = torch.rand(N, device=DEV, generator=gen) * 0.01
    clean = [a.clone().requires_grad_() for a in (x, g)]
    yc, _ = ops.gated_scan(*clean, start, dt=dt)
    gc = torch.autograd.grad(yc, clean, gy)
    x[2700, 3] = bad
    dirty = [a.clone().requires_grad_() for a in (x, g)]
    y, _ = ops.gated_scan(*dirty, start, dt=dt)
    gd = torch.autograd.grad(y, dirty, gy)
    hit = torch.zeros(N, D, dtype=torch.bool, device=DEV)
    hit[2700:3100, 3] = True
    assert torch.equal(y[~hit], yc[~hit]) and not torch.isfinite(y[hit]).any()
    for a, b in zip(gd, gc):
        assert torch.equal(a[~hit], b[~hit])
    gy2 = gy.clone()
    gy2[2600, 5] = bad
    hit = torch.zeros(N, D, dtype=torch.bool, device=DEV)
    hit[2500:2601, 5] = True
    for a, b in zip(torch.autograd.grad(ops.gated_scan(*clean, start, dt=dt)[0], clean, gy2), gc):
        assert torch.equal(a[~hit], b[~hit]) and not torch.isfinite(a[hit]).any()


def test_scan_gradient_is_its_difference():
    """Central differences of the kernel's own forward along random directions: fp32 states are off by some 1e-6 of
    their size, over a step of 2e-2, and curvature adds the step's square: 2e-3 of the terms' root sum of squares."""
    N, D = 400, 16
    gen = torch.Generator(device=DEV).manual_seed(2)
    x, g, gy = torch.randn(3, N, D, device=DEV, generator=gen)
    start, dt = torch.tensor([0, 150, N], device=DEV), torch.rand(N, device=DEV, generator=gen)
    ins = [a.clone().requires_grad_() for a in (x, g)]
    grads = torch.autograd.grad(ops.gated_scan(*ins, start, dt=dt)[0], ins, gy)
    for k in range(2):
        v = torch.randn(N, D, device=DEV, generator=gen)
        sides = []
        for sgn in (1e-2, -1e-2):
            at = [x, g]
            at[k] = at[k] + sgn * v
            sides.append((ops.gated_scan(*at, start, dt=dt)[0].double() * gy).sum())
        terms = grads[k].double() * v
        assert abs((sides[0] - sides[1]) / 2e-2 - terms.sum()) <= 2e-3 * terms.norm() + 2e-3


@pytest.mark.parametrize("dtype,N,D", [(F32, 1, 1), (F32, 3, 7), (BF16, 256, 256), (F16, 33, 65), (BF16, 0, 8)])
@pytest.mark.parametrize("with_dt", [False, True])
def test_scan_step(dtype, N, D, with_dt):
    rng = np.random.default_rng(N)
    x, g = (_t(rng.normal(size=(N, D)), dtype) for _ in range(2))
    state = _t(rng.normal(size=(N, D)))
    dt = _t(rng.exponential(size=N)) if with_dt else None
    start = list(range(N + 1))
    wy, wl, E = O.scan(_np(x), _np(g), start, _np(dt), _np(state))
    y = ops.gated_scan_step(_spread(x, "slice"), g, state, dt=dt)
    _close(y, wy, E)
    _close(state, wl, E)


def test_scan_step_follows_scan():
    """Streaming token by token gives what the scan gives at once."""
    n, T, D = 5, 40, 32
    gen = torch.Generator(device=DEV).manual_seed(3)
    x, g = torch.randn(2, n * T, D, device=DEV, generator=gen)
    dt = torch.rand(n * T, device=DEV, generator=gen)
    start = torch.arange(n + 1, device=DEV) * T
    y, last = ops.gated_scan(x, g, start, dt=dt)
    state, at = torch.zeros(n, D, device=DEV), start[:-1]
    _, _, E = O.scan(_np(x), _np(g), start.tolist(), _np(dt))
    for k in range(T):
        out = ops.gated_scan_step(x[at + k], g[at + k], state, dt=dt[at + k])
        assert np.all(np.abs(_np(out - y[at + k])) <= 2 * E[(at + k).cpu().numpy()])


# ------------------------------------------------------------------------------------------- norm
def _norm_case(N, D, dtype, rtype, p, layout=None, seed=0, residual=True, eps=1e-5):
    rng = np.random.default_rng(seed)
    x, gy = (_t(rng.normal(size=(N, D)), dtype) for _ in range(2))
    res = _t(rng.normal(size=(N, D)) * 2, rtype) if residual else None
    gs = _t(rng.normal(size=(N, D)), rtype)
    w = _t(rng.normal(size=D)).requires_grad_()
    sd, off = 0xDEAD_BEEF_0BAD_F00D, 2 ** 33 + 5
    print(f"norm N={N} D={D} {dtype} {rtype} p={p} {layout} residual={residual}", flush=True)
    ins = [None if a is None else _spread(a, layout).detach().requires_grad_() for a in (x, res)]
    y, s = ops.residual_rms_norm(*ins, w, eps=eps, p=p, seed=sd, offset=off)
    keep = O.keeps(N, D, p, sd, off) * (65536 / (65536 - round(65536 * p)))
    ws = _np(x) * keep + (0 if res is None else _np(res))
    _close(s, ws, 2 * O.U * (np.abs(_np(x) * keep) + np.abs(ws)), "s")
    assert s.dtype == (rtype if residual else dtype) and y.dtype == dtype
    sn, wn = _np(s), _np(w)
    wy, _ = O.norm(sn, wn, eps)
    _close(y, wy, 64 * O.U * np.abs(wy), "y")
    with torch.no_grad():
        y2, s2 = ops.residual_rms_norm(*ins, w, eps=eps, p=p, seed=sd, offset=off)
    assert torch.equal(y, y2) and torch.equal(s, s2)
    wrt = [a for a in (*ins, w) if a is not None]
    g_s = _spread(gs.to(s.dtype), layout)
    got = torch.autograd.grad((y, s), wrt, (_spread(gy, layout), g_s), retain_graph=True)
    (ds, dw), (bs, bw) = O.norm_bwd(sn, wn, eps, _np(gy), _np(g_s))
    _close(got[0], ds * keep, (bs + 2 * O.U * np.abs(ds)) * keep, "gx")
    if residual:
        _close(got[1], ds, bs, "gres")
    _close(got[-1], dw, bw, "gw")
    again = torch.autograd.grad((y, s), wrt, (_spread(gy, layout), g_s))
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("D", [1, 2, 7, 8, 33, 48, 64, 65, 100, 128, 256, 345, 512, 513, 1000, 1024, 1025, 2048, 2056, 4096, 8191, 8192])
@pytest.mark.parametrize("dtype,rtype", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
def test_norm_widths(D, dtype, rtype):
    _norm_case(5 if D > 512 else 70, D, dtype, rtype, 0.1 if D % 2 else 0.0, seed=D)


@pytest.mark.parametrize("N", [1, 2, 31, 33, 1023, 40_001])
@pytest.mark.parametrize("p", [0.0, 0.5])
def test_norm_rows(N, p):
    _norm_case(N, 64, BF16, BF16, p, seed=N)


@pytest.mark.parametrize("layout", ["slice", "odd", "cols"])
@pytest.mark.parametrize("dtype,rtype", [(F32, F32), (BF16, BF16), (F16, F32)])
def test_norm_layouts(layout, dtype, rtype):
    _norm_case(130, 96, dtype, rtype, 0.25, layout, seed=5)


@pytest.mark.parametrize("p", [0.0, 0.3])
def test_norm_without_residual(p):
    _norm_case(50, 72, F32, F32, p, residual=False)


def test_norm_of_nothing_and_of_zeros():
    w = torch.ones(16, device=DEV, requires_grad=True)
    y, s = ops.residual_rms_norm(torch.zeros(0, 16, device=DEV), None, w)
    assert y.shape == (0, 16)
    assert not torch.autograd.grad(y.sum(), w)[0].any()
    z = torch.zeros(3, 16, device=DEV)
    assert not ops.residual_rms_norm(z, z, w.detach())[0].any()
    q, scale, _ = ops.residual_rms_norm_fp8(z, z, w.detach())
    assert not q.float().any() and torch.all(scale == torch.tensor(1e-30, device=DEV) / 448)


def test_norm_bad_rows_stay_alone():
    x = torch.randn(40, 64, device=DEV)
    w = torch.ones(64, device=DEV)
    want = ops.residual_rms_norm(x, None, w)[0]
    x2 = x.clone()
    x2[7, 3], x2[9, 0] = float("nan"), float("inf")
    got = ops.residual_rms_norm(x2, None, w)[0]
    ok = torch.ones(40, dtype=torch.bool, device=DEV)
    ok[[7, 9]] = False
    assert torch.equal(got[ok], want[ok]) and got[7].isnan().all() and got[9, 0].isnan()
    q, scale, _ = ops.residual_rms_norm_fp8(x2, None, w)
    assert scale[ok].isfinite().all() and scale[7].isnan() and q[7].float().isnan().all()
    # a dropped NaN is dropped
    s = ops.residual_rms_norm(torch.full((64, 64), float("nan"), device=DEV), torch.zeros(64, 64, device=DEV), w, p=0.5, seed=1)[1]
    assert s.isnan().any() and (s == 0).any()


@pytest.mark.parametrize("dtype,rtype", [(F32, F32), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("N,D", [(1, 1), (3, 7), (70, 64), (33, 345), (9, 2048), (5, 5000), (4, 8192)])
def test_norm_fp8(N, D, dtype, rtype):
    rng = np.random.default_rng(D)
    x, res = _t(rng.normal(size=(N, D)), dtype), _t(rng.normal(size=(N, D)), rtype)
    w = _t(rng.normal(size=D))
    q, scale, s = ops.residual_rms_norm_fp8(x, res, w)
    assert q.dtype == torch.float8_e4m3fn and scale.shape == (N, 1)
    ws = _np(x) + _np(res)
    _close(s, ws, 2 * O.U * np.abs(ws), "s")
    y, _ = O.norm(_np(s), _np(w), 1e-6)
    from tests.test_sequence import _fp8_close
    _fp8_close(q, scale, y)


def test_dropout_draws_the_published_bits():
    """The kernel's mask is the restatement's for every width's vectors, whatever the rows' layout."""
    for D in (5, 8, 24, 64, 345):
        for dtype in (F32, BF16):
            x = torch.ones(37, D, device=DEV, dtype=dtype)
            for p in (0.1, 0.5, 1 - 2 ** -16):
                _, s = ops.residual_rms_norm(x, None, torch.ones(D, device=DEV), p=p, seed=-3, offset=12)
                assert np.array_equal((s != 0).cpu().numpy(), O.keeps(37, D, p, (-3) & (2 ** 64 - 1), 12)), (D, dtype, p)


# ------------------------------------------------------------------------------------------- embedding
def _ids(N, V, kind, rng):
    if kind == "uniform":
        return rng.integers(0, V, N)
    if kind == "one":
        return np.full(N, V // 2)
    if kind == "hot":                                        # one id owns half of the tokens, some are none
        ids = rng.integers(-2, V + 2, N)
        ids[rng.random(N) < 0.5] = V - 1
        return ids
    if kind == "none":
        return np.where(rng.random(N) < 0.5, -1, V)
    if kind == "sorted":
        return np.sort(rng.integers(0, V, N))
    raise ValueError(kind)


def _embed_case(N, V, D, kind, ttype, otype, wide=True, layout=None, seed=0, scale=0.5):
    rng = np.random.default_rng(seed)
    ids = _ids(N, V, kind, rng)
    print(f"embed N={N} V={V} D={D} {kind} {ttype} {otype} {layout}", flush=True)
    idt = torch.as_tensor(ids, device=DEV).to(torch.int64 if wide else torch.int32)
    table = _spread(_t(rng.normal(size=(V, D)), ttype), layout).detach().requires_grad_()
    y = ops.embed_tokens(idt, table, scale=scale, dtype=otype)
    ok = (ids >= 0) & (ids < V)
    want = np.where(ok[:, None], _np(table)[np.where(ok, ids, 0)] * scale, 0)
    _close(y, want, O.U * np.abs(want), "rows")
    gy = _spread(_t(rng.normal(size=(N, D)), otype), layout)
    got = torch.autograd.grad(y, table, gy, retain_graph=True)[0]
    wt, bound = O.embed_bwd(ids, V, scale, _np(gy))
    _close(got, wt, bound, "gtable")
    assert torch.equal(got, torch.autograd.grad(y, table, gy)[0])


@pytest.mark.parametrize("N", [0, 1, 63, 64, 65, 1000, 4096, 4097, 20_011])
@pytest.mark.parametrize("kind", ["uniform", "hot", "one", "none", "sorted"])
def test_embed_lengths(N, kind):
    _embed_case(N, 37, 16, kind, F32, F32, seed=N)


@pytest.mark.parametrize("V", [1, 2, 255, 1023, 1024, 9600, 70_001, 1_100_000])
@pytest.mark.parametrize("kind", ["uniform", "hot"])
def test_embed_tables(V, kind):
    _embed_case(9000, V, 8, kind, F32, BF16, seed=V)


@pytest.mark.parametrize("D", [1, 3, 8, 24, 48, 64, 100, 128, 345, 512, 520, 1024])
@pytest.mark.parametrize("ttype,otype", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F32), (F16, F16)])
def test_embed_widths(D, ttype, otype):
    _embed_case(3000, 50, D, "hot", ttype, otype, wide=D % 2 == 0, seed=D)


@pytest.mark.parametrize("layout", ["slice", "odd", "cols"])
@pytest.mark.parametrize("ttype,otype", [(F32, BF16), (BF16, F32)])
def test_embed_layouts(layout, ttype, otype):
    _embed_case(3000, 300, 64, "hot", ttype, otype, layout=layout)


def test_embed_hot_token_of_many_chunks():
    """A run of 300,000 tokens (over 73 workgroups, whose shares one workgroup adds up) between others."""
    rng = np.random.default_rng(1)
    N, V, D = 400_000, 1000, 8
    ids = rng.integers(0, V, N)
    ids[rng.random(N) < 0.75] = 500
    g = rng.normal(size=(N, D)).astype(np.float32)
    table = torch.zeros(V, D, device=DEV, requires_grad=True)
    y = ops.embed_tokens(torch.as_tensor(ids, device=DEV), table)
    got = torch.autograd.grad(y, table, _t(g))[0]
    want, bound = O.embed_bwd(ids, V, 1.0, g.astype(float))
    # 32 rows a group, 128 groups a workgroup, 128 stretches of a share: 32 + 128 + 1 + 128 roundings of the magnitudes,
    # not 300,000
    mag = O.embed_bwd(ids, V, 1.0, np.abs(g).astype(float))[0]
    _close(got, want, np.minimum(bound, 400 * O.U * mag))


@pytest.mark.parametrize("D", [1, 2, 8, 64, 260, 520])
def test_embed_runs_of_all_lengths(D):
    """Tokens that occur from once to 300000 times: runs within a group of lanes, over groups, over up to 16 workgroups
    and over many.  Whole numbers, so every sum is exact."""
    rng = np.random.default_rng(D)
    often = np.array([1, 2, 31, 32, 33, 300_000, 0, 255, 256, 257, 1023, 1024, 1025, 2047, 4099, 1, 17_000, 9_000, 33_000, 0, 40_001, 1])
    if D > 64:
        often = often // 4
    ids = rng.permutation(np.repeat(np.arange(len(often)), often))
    g = rng.integers(-4, 5, size=(len(ids), D)).astype(np.float32)
    print(f"embed runs N={len(ids)} D={D}", flush=True)
    table = torch.zeros(len(often), D, device=DEV, requires_grad=True)
    out = ops.embed_tokens(torch.as_tensor(ids, device=DEV), table)
    got, = torch.autograd.grad(out, table, torch.as_tensor(g, device=DEV))
    want = torch.zeros(len(often), D, dtype=torch.float64).index_add_(0, torch.as_tensor(ids), torch.as_tensor(g).double())
    assert torch.equal(got.double().cpu(), want)


def test_embed_odd_half_precision_table():
    """A table whose gradient is an odd number of 2-byte elements."""
    _embed_case(40, 3, 5, "uniform", BF16, BF16)
    _embed_case(0, 3, 1, "uniform", F16, F16)


def test_embed_keeps_shape_and_bad_values():
    table = torch.randn(5, 8, device=DEV, requires_grad=True)
    ids = torch.tensor([[0, 1, 2], [3, 4, -1]], device=DEV)
    y = ops.embed_tokens(ids, table)
    assert y.shape == (2, 3, 8)
    g = torch.ones_like(y)
    g[0, 1] = float("nan")
    g[1, 2] = float("inf")                                   # of no token: adds nothing
    got = torch.autograd.grad(y, table, g)[0]
    assert got[1].isnan().all() and torch.all(got[[0, 2, 3, 4]] == 1)


# ------------------------------------------------------------------------------------------- together
def test_operators_on_another_stream():
    st = torch.cuda.Stream()
    gen = torch.Generator(device=DEV).manual_seed(4)
    N, V, D = 5000, 200, 64
    ids = torch.randint(0, V, (N,), device=DEV, generator=gen)
    table = torch.randn(V, D, device=DEV, generator=gen, requires_grad=True)
    w = torch.ones(D, device=DEV, requires_grad=True)
    start = torch.tensor([0, 1000, N], device=DEV)

    def step():
        e = ops.embed_tokens(ids, table)
        y, s = ops.residual_rms_norm(e, e, w, p=0.2, seed=1)
        h, last = ops.gated_scan(y, s, start)
        return torch.autograd.grad(h.sum() + last.sum(), (table, w))

    here = step()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        there = step()
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a, b) for a, b in zip(here, there))


def test_operators_in_a_graph():
    """Recorded once and replayed with eager work between: every replay gives the eager bits."""
    gen = torch.Generator(device=DEV).manual_seed(5)
    N, V, D = 9000, 300, 64
    ids = torch.randint(0, V, (N,), device=DEV, generator=gen)
    table = torch.randn(V, D, device=DEV, generator=gen, requires_grad=True)
    w = torch.ones(D, device=DEV, requires_grad=True)
    start = torch.tensor([0, 4000, N], device=DEV)
    gy, gl = torch.randn(N, D, device=DEV, generator=gen), torch.randn(2, D, device=DEV, generator=gen)

    def step():
        e = ops.embed_tokens(ids, table)
        y, s = ops.residual_rms_norm(e, e, w, p=0.2, seed=1)
        h, last = ops.gated_scan(y, s, start)
        return (h, last, *torch.autograd.grad((h, last), (table, w), (gy, gl)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for r in range(3):
        with torch.no_grad():
            table.add_(0.1 * r)
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), r


def test_offsets_past_32_bits():
    """Rows whose offsets pass 2^31 elements and 2^32 bytes: the last window of each operator against a call on it alone."""
    N, D, tail = 2 ** 31 // 64 + 5000, 64, 777
    print(f"past 32 bits: N={N}", flush=True)
    small = torch.randn(2, tail, D, device=DEV).to(BF16)
    x = torch.zeros(N, D, dtype=BF16, device=DEV)
    g = torch.zeros(N, D, dtype=BF16, device=DEV)
    x[-tail:], g[-tail:] = small[0], small[1]
    start = torch.tensor([0, N - tail, N], device=DEV)
    ins = [a.requires_grad_() for a in (x, g)]
    y, last = ops.gated_scan(*ins, start)
    few = [a.clone().requires_grad_() for a in small]
    y1, last1 = ops.gated_scan(*few, torch.tensor([0, tail], device=DEV))
    u = torch.finfo(BF16).eps
    assert torch.allclose(y[-tail:].float(), y1.float(), rtol=u, atol=1e-6) and torch.allclose(last[1], last1[0], atol=1e-5)
    gy = torch.zeros(N, D, dtype=BF16, device=DEV)
    gy[-tail:] = small[1]
    big = torch.autograd.grad(y, ins, gy)
    for a, b in zip(big, torch.autograd.grad(y1, few, small[1])):
        assert torch.allclose(a[-tail:].float(), b.float(), rtol=2 * u, atol=1e-5)
        assert not a[:-tail].any()
    del big, y, last
    w = torch.ones(D, device=DEV)
    with torch.no_grad():
        y, s = ops.residual_rms_norm(x, g, w)
        y1, s1 = ops.residual_rms_norm(small[0], small[1], w)
    assert torch.equal(y[-tail:], y1) and torch.equal(s[-tail:], s1)


def test_calls_of_several_launches():
    """More workgroups than a launch takes: the last rows and streams against a call on them alone, the first of the
    second launch among them."""
    tail, D = 300, 64
    N = 2 ** 31 // D + tail - 7
    print(f"several launches: step N={N}", flush=True)
    few = torch.randn(tail, D, device=DEV)
    state, x = torch.ones(N, D, device=DEV), torch.ones(1, D, dtype=BF16, device=DEV).expand(N, D)
    state[-tail:] = few
    y = ops.gated_scan_step(x, x, state)
    y1 = ops.gated_scan_step(x[-tail:], x[-tail:], few)
    assert torch.equal(y[-tail:], y1) and torch.equal(state[-tail:], few)
    assert torch.equal(y[:-tail:4096], y[:1].expand(y[:-tail:4096].shape))
    del state, y
    N, D = 2 ** 25 + tail - 7, 260
    print(f"several launches: norm N={N}", flush=True)
    x, w = torch.ones(N, D, dtype=BF16, device=DEV), torch.ones(D, device=DEV)
    x[-tail:] = torch.randn(tail, D, device=DEV)
    with torch.no_grad():
        y, _ = ops.residual_rms_norm(x, None, w)
        assert torch.equal(y[-tail:], ops.residual_rms_norm(x[-tail:], None, w)[0])
    assert torch.equal(y[:-tail:4096], torch.ones_like(y[:-tail:4096]))
    del x, y
    N, D = 2 ** 23 + tail - 7, 1031
    print(f"several launches: embedding N={N}", flush=True)
    ids = torch.randint(0, 5, (N,), device=DEV)
    table = torch.randn(5, D, device=DEV)
    y = ops.embed_tokens(ids, table, dtype=BF16)
    assert torch.equal(y[-tail:], table[ids[-tail:]].to(BF16)) and torch.equal(y[::4096], table[ids[::4096]].to(BF16))


def test_scan_of_very_many_windows():
    """More windows than two steps of the 64-way search cover, empty ones among them."""
    rng = np.random.default_rng(15)
    sizes = rng.integers(0, 6, 9000)
    start = [0, *np.cumsum(sizes).tolist()]
    N, D = start[-1], 4
    x, g, gy = (_t(rng.normal(size=(N, D))) for _ in range(3))
    gl = _t(rng.normal(size=(9000, D)))
    ins = [a.requires_grad_() for a in (x, g)]
    y, last = ops.gated_scan(*ins, torch.tensor(start, device=DEV))
    wy, wl, E = O.scan(_np(x), _np(g), start)
    _close(y, wy, E)
    some = sizes > 0
    _close(last, wl, np.where(some[:, None], E[np.array(start[1:]) - 1], 0))
    got = torch.autograd.grad((y, last), ins, (gy, gl))
    want, bound = O.scan_bwd(_np(x), _np(g), start, _np(gy), _np(gl))
    for a, b, c in zip(got, want, bound):
        _close(a, b, c)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_scan_nan_gate_shows(dtype):
    """A gate that is not a number makes its token and the window's later states so, in its channel only."""
    N, D = 100, 8
    x, g = torch.randn(N, D, device=DEV).to(dtype), torch.randn(N, D, device=DEV).to(dtype)
    g[20, 2] = float("nan")
    for dt in (None, torch.rand(N, device=DEV)):
        y, last = ops.gated_scan(x, g, torch.tensor([0, 50, N], device=DEV), dt=dt)
        hit = torch.zeros(N, D, dtype=torch.bool, device=DEV)
        hit[20:50, 2] = True
        assert torch.equal(y.isnan(), hit) and last[0, 2].isnan() and last.isnan().sum() == 1
        state = torch.zeros(N, D, device=DEV)
        ops.gated_scan_step(x, g, state, dt=dt)
        assert state.isnan().sum() == 1


def test_second_derivatives_are_refused():
    x, g = (torch.randn(10, 8, device=DEV, requires_grad=True) for _ in range(2))
    w = torch.ones(8, device=DEV, requires_grad=True)
    table = torch.randn(5, 8, device=DEV, requires_grad=True)
    start, ids = torch.tensor([0, 10], device=DEV), torch.arange(5, device=DEV)
    for out, wrt in ((ops.gated_scan(x, g, start)[0], x), (ops.residual_rms_norm(x, g, w)[0], x),
                     (ops.embed_tokens(ids, table), table)):
        first, = torch.autograd.grad(out.square().sum(), wrt, create_graph=True)
        with pytest.raises(RuntimeError):
            first.sum().backward()


def test_gradients_of_some_inputs():
    """Each input's gradient alone is the one it has beside the others."""
    x, res, gy = torch.randn(3, 40, 24, device=DEV)
    w = torch.randn(24, device=DEV)
    for p in (0.0, 0.4):
        full = [t.clone().requires_grad_() for t in (x, res, w)]
        want = torch.autograd.grad(ops.residual_rms_norm(*full, p=p, seed=2)[0], full, gy)
        for k in range(3):
            part = [t.clone().requires_grad_(j == k) for j, t in enumerate((x, res, w))]
            got, = torch.autograd.grad(ops.residual_rms_norm(*part, p=p, seed=2)[0], part[k], gy)
            assert torch.equal(got, want[k]), (p, k)
        sums = [t.clone().requires_grad_() for t in (x, res, w)]
        gx, gr, gw = torch.autograd.grad(ops.residual_rms_norm(*sums, p=p, seed=2)[1], sums, gy, allow_unused=True)
        assert torch.equal(gr, gy) and (gw is None or not gw.any()) and (p > 0 or torch.equal(gx, gy))
    start = torch.tensor([0, 40], device=DEV)
    full = [t.clone().requires_grad_() for t in (x, res)]
    want = torch.autograd.grad(ops.gated_scan(*full, start)[0], full, gy)
    for k in range(2):
        part = [t.clone().requires_grad_(j == k) for j, t in enumerate((x, res))]
        got, = torch.autograd.grad(ops.gated_scan(*part, start)[0], part[k], gy)
        assert torch.equal(got, want[k])


# ------------------------------------------------------------------------------------------- beside autograd
def test_step_after_a_use_of_its_state_is_noticed():
    """A state that a later backward needs and a step has overwritten: that backward raises, as after any operation in
    place, and a scan from the state as it is works."""
    x, g = torch.randn(2, 6, 16, device=DEV)
    state = torch.randn(6, 16, device=DEV)
    w = torch.randn(16, 16, device=DEV, requires_grad=True)
    start = torch.arange(7, device=DEV)
    gate = g.clone().requires_grad_()
    product = torch.nn.functional.linear(state, w)
    y, _ = ops.gated_scan(x, gate, start, h0=state)
    before = state._version
    ops.gated_scan_step(x, g, state)
    assert state._version > before
    for out, wrt in ((product, w), (y, gate)):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out.sum(), wrt)
    y, _ = ops.gated_scan(x, gate, start, h0=state)
    assert torch.autograd.grad(y.sum(), gate)[0].isfinite().all()
    with torch.inference_mode():
        inner = torch.zeros(6, 16, device=DEV)
        assert torch.equal(ops.gated_scan_step(x, g, inner), inner)


def _calls():
    """The operators as functions of one float tensor, and such a tensor."""
    ids, start = torch.tensor([0, 3, -1, 5, 2], device=DEV), torch.tensor([0, 2, 6], device=DEV)
    w = torch.rand(8, device=DEV) + 0.5
    other = torch.randn(6, 8, device=DEV)
    return torch.randn(6, 8, device=DEV), {
        "embed": lambda t: ops.embed_tokens(ids, t, scale=2.0),
        "norm": lambda t: torch.stack(ops.residual_rms_norm(t, other, w, p=0.25, seed=3)),
        "scan": lambda t: ops.gated_scan(t, other, start)[0],
        "gate": lambda t: torch.cat(ops.gated_scan(other, t, start)),
        "h0": lambda t: torch.cat(ops.gated_scan(other, other, start, h0=t[:2])),
        "fp8": lambda t: ops.residual_rms_norm_fp8(t, other, w)[1],
        "step": lambda t: ops.gated_scan_step(t, other, torch.ones(6, 8, device=DEV)),
    }


@pytest.mark.parametrize("which", ["embed", "norm", "scan", "gate", "h0"])
def test_forward_mode_derivatives_are_refused(which):
    """A tangent is refused, not dropped; without one a call at a forward-mode level is a call as any other."""
    t, calls = _calls()
    want = calls[which](t)
    with torch.autograd.forward_ad.dual_level():
        assert torch.equal(calls[which](t), want)
        with pytest.raises((RuntimeError, NotImplementedError)):
            calls[which](torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)))


@pytest.mark.parametrize("which", ["embed", "norm", "scan", "gate", "h0", "fp8", "step"])
@pytest.mark.parametrize("grad", [False, True])
def test_recorded_calls_compute_or_are_refused(which, grad):
    """A recording that would replay the outputs' memory alone is refused; torch.jit.trace keeps the differentiable
    operators as calls, which compute on the new input."""
    from torch.fx.experimental.proxy_tensor import make_fx
    t, calls = _calls()
    fn = calls[which]
    t.requires_grad_(grad)
    for how in ({}, {"pre_dispatch": True}, {"tracing_mode": "fake"}):
        with pytest.raises(RuntimeError, match="recorded"):
            make_fx(fn, **how)(t)
    if which in ("fp8", "step"):
        with pytest.raises(RuntimeError, match="recorded"):
            torch.jit.trace(fn, (t,), check_trace=False)
        return
    traced = torch.jit.trace(fn, (t,), check_trace=False)
    for _ in range(3):
        new = torch.randn_like(t)
        assert torch.equal(traced(new), fn(new))


@pytest.mark.parametrize("which", ["embed", "norm", "scan", "h0", "fp8", "step"])
@pytest.mark.parametrize("grad", [False, True])
def test_compiled_calls_compute(which, grad):
    """torch.compile breaks its graph at the operators and calls them."""
    t, calls = _calls()
    torch._dynamo.reset()
    fn = torch.compile(lambda a: calls[which](a * 2) + 1, backend="eager")
    for _ in range(2):
        t = torch.randn_like(t).requires_grad_(grad)
        got, want = fn(t), calls[which](t * 2) + 1
        assert torch.equal(got, want)
        if grad and want.requires_grad:
            assert torch.equal(torch.autograd.grad(got.sum(), t)[0], torch.autograd.grad(want.sum(), t)[0])


@pytest.mark.parametrize("dtype,D", [(F32, 24), (BF16, 64), (F16, 64), (F32, 5000)])
@pytest.mark.parametrize("p", [0.0, 0.4])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_of_which_the_sum_alone_is_used(dtype, D, p, residual):
    """The gradient of s alone is gs (through the dropout for x) also in rows whose norm is not finite: a row of zeros
    with eps = 0 and a row with an infinity.  The weight has no part in it."""
    gen = torch.Generator(device=DEV).manual_seed(D)
    x, res, gs = (torch.randn(50, D, device=DEV, generator=gen).to(dtype) for _ in range(3))
    x[3], res[3] = 0, 0
    res[7, 2], x[7, 2] = float("inf"), 1
    if not residual:
        x[7, 2] = float("inf")
    w = torch.ones(D, device=DEV, requires_grad=True)
    ins = [x.requires_grad_(), *([res.requires_grad_()] if residual else [])]
    y, s = ops.residual_rms_norm(x, res if residual else None, w, eps=0.0, p=p, seed=4)
    got = torch.autograd.grad(s, [*ins, w], gs, allow_unused=True)
    keep = torch.as_tensor(O.keeps(50, D, p, 4, 0), device=DEV)
    factor = 65536 / (65536 - round(65536 * p))
    # one product in single precision, rounded to the type
    assert torch.equal(got[0], torch.where(keep, gs.float() * torch.tensor(factor, device=DEV), 0.0).to(dtype))
    if residual:
        assert torch.equal(got[1], gs)
    assert got[-1] is None or not got[-1].any()


@pytest.mark.parametrize("D", [1, 3, 64])
def test_one_row_of_a_very_wide_tensor(D):
    """A single token cut from a row of four million: the stride of one row means nothing."""
    wide = torch.randn(1, 2 ** 22, device=DEV)
    a, b = wide[:, 5:5 + D], wide[:, 900_001:900_001 + D]
    print(f"one row D={D} stride {a.stride(0)}", flush=True)
    few = [t.clone() for t in (a, b)]
    start, w, ids = torch.tensor([0, 1], device=DEV), torch.ones(D, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    grads = [[] for _ in range(2)]
    for k, (x, g) in enumerate(((a, b), few)):
        x, g = x.detach().requires_grad_(), g.detach().requires_grad_()
        y, last = ops.gated_scan(x, g, start)
        n, s = ops.residual_rms_norm(x, g, w)
        e = ops.embed_tokens(ids, x)
        state = torch.ones(1, D, device=DEV)
        ops.gated_scan_step(x.detach(), g.detach(), state)
        grads[k] = [y, last, n, s, e, state, *torch.autograd.grad((y, n, e), (x, g), (b, b, b.expand(3, D)))]
    assert all(torch.equal(p, q) for p, q in zip(*grads))


def _mostly_empty(empty, dtype, seed):
    """Tokens in few windows among ``empty`` windows without any: between the tokens, before them and behind them."""
    rng = np.random.default_rng(seed)
    sizes = np.zeros(empty + 40, np.int64)
    at = np.sort(rng.choice(empty // 8, 20, replace=False)) + empty // 16       # some far apart, and 20 side by side
    at = np.concatenate([at, np.arange(20) + empty // 4 * 3])
    sizes[at] = rng.integers(1, 90, 40)
    start = np.concatenate([[0], np.cumsum(sizes)])
    N, D = int(start[-1]), 8
    x, g, gy = (_t(rng.normal(size=(N, D)), dtype) for _ in range(3))
    dt = _t(rng.exponential(size=N) * 0.1)
    h0, gl = (torch.randn(len(sizes), D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(k)) for k in (1, 2))
    return start, at, x, g, gy, dt, h0, gl


@pytest.mark.parametrize("empty,dtype", [(3000, F32), (1_000_000, F32), (1_000_000, BF16)])
def test_scan_among_very_many_empty_windows(empty, dtype):
    """The windows with tokens against the oracle on them alone; the empty ones hand on h0 and the last state's
    gradient."""
    start, at, x, g, gy, dt, h0, gl = _mostly_empty(empty, dtype, seed=empty)
    print(f"scan among {empty} empty windows, N={x.shape[0]}", flush=True)
    ins = [a.requires_grad_() for a in (x, g, h0)]
    y, last = ops.gated_scan(x, g, torch.as_tensor(start, device=DEV), dt=dt, h0=h0)
    got = torch.autograd.grad((y, last), ins, (gy, gl))
    few = [0, *start[at + 1].tolist()]
    args = (_np(x), _np(g), few)
    wy, wl, E = O.scan(*args, _np(dt), _np(h0[at]))
    _close(y, wy, E, "y")
    _close(last[at], wl, E[np.array(few[1:]) - 1], "last")
    want, bound = O.scan_bwd(*args, _np(gy), _np(gl[at]), _np(dt), _np(h0[at]))
    for name, a, b, c in zip(("gx", "gg", "gh0"), (got[0], got[1], got[2][at]), want, bound):
        _close(a, b, c, name)
    none = torch.ones(len(start) - 1, dtype=torch.bool, device=DEV)
    none[at] = False
    assert torch.equal(last[none], h0[none]) and torch.equal(got[2][none], gl[none])


def test_scan_time_does_not_follow_the_empty_windows():
    """A million empty windows cost a search, not a walk: forward and backward of a few tokens stay within 20 ms (a
    dependent read for each would be a second, writing the windows' states takes under one millisecond)."""
    start, _, x, g, gy, dt, _, _ = _mostly_empty(1_000_000, F32, seed=5)
    start = torch.as_tensor(start, device=DEV)
    ins = [a.requires_grad_() for a in (x, g)]
    best = 1e9
    for _ in range(4):
        e0, e1 = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        e0.record()
        torch.autograd.grad(ops.gated_scan(x, g, start, dt=dt)[0], ins, gy)
        e1.record()
        e1.synchronize()
        best = min(best, e0.elapsed_time(e1))
    print(f"{best:.2f} ms", flush=True)
    assert best < 20


# ------------------------------------------------------------------------------------------- long windows
def _recur(a, u):
    """h_i = a_i h_{i-1} + u_i along the rows in float64, from zero: blocks of about sqrt(N) rows side by side, then
    through their ends one by one."""
    N, D = u.shape
    m = max(1, int(N ** 0.5))
    n = -(-N // m)
    pad = torch.zeros(n * m - N, D, dtype=u.dtype, device=u.device)
    a, u = torch.cat([a, pad]).view(n, m, D), torch.cat([u, pad]).view(n, m, D)
    h, prod = u.clone(), a.clone()
    for j in range(1, m):
        h[:, j] += a[:, j] * h[:, j - 1]
        prod[:, j] *= prod[:, j - 1]
    before = torch.zeros_like(h[:, 0])
    for k in range(1, n):
        before[k] = h[k - 1, -1] + prod[k - 1, -1] * before[k - 1]
    return (h + prod * before[:, None]).view(-1, D)[:N]


def _states(a, z, u, edges, begin):
    """States, their magnitudes M (of |u|) and P = sum of |u_j| decay Z, with Z the rates between j and i; at the rows
    ``edges`` the recurrence begins anew from ``begin``.  A decay counts where the row before hands on."""
    inner = a.clone()
    inner[edges] = 0

    def run(add, first):
        add = add.clone()
        add[edges] += a[edges] * first
        return _recur(inner, add)

    h, M = run(u, begin), run(u.abs(), begin.abs())
    prev = torch.cat([torch.zeros_like(M[:1]), M[:-1]])
    prev[edges] = begin.abs()
    return h, M, _recur(inner, a * z * prev)


def _long_case(N, D, dtype, with_dt, cuts, seed):
    """Against float64 on the device, token by token in blocks.  Bounds: a state's way from its tokens holds at most 16
    steps in a group (4 units of a decay and a sum each), 80 joins of ranges (3 each) and the token's own 8 + |gate|
    (<= 32): 400 units of the magnitudes M.  A rate is off by 8 + |gate| units, one without gaps comes from a product of 16
    decays (50), and sums of rates round at most 90 times: 200 units of each Z, hence of P."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device=DEV, generator=gen)
    start = torch.tensor([0, *cuts, N], device=DEV)
    B = len(start) - 1
    x, gy = (rand(N, D) + 1).to(dtype), (rand(N, D) + 0.5).to(dtype)
    g = (rand(N, D) * 1.5 - 1 if with_dt else rand(N, D) - 11).to(dtype)
    dt = torch.rand(N, device=DEV, generator=gen) * 4e-5 if with_dt else None
    h0, gl = rand(B, D), rand(B, D) * 100
    print(f"scan N={N} D={D} {dtype} dt={with_dt} B={B}", flush=True)
    ins = [t.requires_grad_() for t in (x, g, h0)]
    y, last = ops.gated_scan(x, g, start, dt=dt, h0=h0)
    got = torch.autograd.grad((y, last), ins, (gy, gl))
    with torch.no_grad():
        y2, last2 = ops.gated_scan(x, g, start, dt=dt, h0=h0)
    assert torch.equal(y, y2) and torch.equal(last, last2)

    gd, xd = g.detach().double(), x.detach().double()
    step = torch.ones(N, 1, dtype=torch.float64, device=DEV) if dt is None else dt.double()[:, None]
    z = torch.logaddexp(gd, torch.zeros_like(gd)) * step
    a, w, wc = torch.exp(-z), torch.sigmoid(gd), torch.sigmoid(-gd)
    some = start[1:] > start[:-1]
    head, tail = start[:-1][some], start[1:][some] - 1
    begin = h0.detach().double()[some]
    h, M, P = _states(a, z, w * xd, head, begin)
    E = O.U * (400 * M + 200 * P)
    _close(y, _np(h), _np(E), "y")
    _close(last[some], _np(h[tail]), _np(E[tail]), "last")
    assert torch.equal(last[~some], h0[~some])
    # C_i = a_i (gy_i + C_{i+1}) from the end, H_i = gy_i + C_{i+1}
    back = lambda t: t.flip(0)
    ends = N - 1 - tail
    C, MC, PC = _states(back(a), back(z), back(a * gy.double()), ends, gl.double()[some])
    C, EC, MC = back(C), back(O.U * (400 * MC + 200 * PC)), back(MC)

    def behind(t, edge):
        t = torch.cat([t[1:], torch.zeros_like(t[:1])])
        t[tail] = edge
        return t

    H, mH = gy.double() + behind(C, gl.double()[some]), gy.double().abs() + behind(MC, gl.double()[some].abs())
    eH = behind(EC, 0.0) + O.U * mH
    before = lambda t, first: torch.cat([torch.zeros_like(t[:1]), t[:-1]]).index_put((head,), first)
    hp, ep = before(h, begin), before(E, torch.zeros_like(begin))
    t = xd * wc - step * a * hp
    mt = xd.abs() * wc + step * a * (hp.abs() + ep)
    _close(got[0], _np(H * w), _np((eH + 32 * O.U * mH) * w), "gx")
    _close(got[1], _np(H * w * t), _np(w * (eH * mt + mH * (O.U * (40 + 4 * z) * mt + step * a * ep))), "gg")
    _close(got[2][some], _np(C[head]), _np(EC[head]), "gh0")
    assert torch.equal(got[2][~some], gl[~some])
    return float((last[-1].detach().double() - h[-1]).abs().max() / h[-1].abs().max())


@pytest.mark.parametrize("N,D,dtype", [(40_003, 64, F32), (40_003, 64, BF16), (300_001, 64, F32), (300_001, 64, F16),
                                       (251_117, 65, F32), (300_001, 6, BF16)])
@pytest.mark.parametrize("with_dt", [False, True])
@pytest.mark.parametrize("windows", [1, 4])
def test_scan_of_long_windows(N, D, dtype, with_dt, windows):
    """States that live over many chunks, blocks of chunks and stretches of blocks, forward and backward, from given states,
    also over windows that begin inside them and one without tokens."""
    cuts = [] if windows == 1 else [N // 3, N // 3, N // 2 + 7]
    _long_case(N, D, dtype, with_dt, cuts, seed=N + D)


def test_scan_of_a_million_tokens():
    """The last state after 1M tokens with decays next to one: as near as its ranges' joins allow, not as a product of a
    million factors would be (4e-4)."""
    off = _long_case(1_000_000, 8, F32, True, [], seed=9)
    print(f"last state off by {off:.2g} of its size", flush=True)
    assert off < 5e-6


@pytest.mark.parametrize("which", ["embed", "norm", "scan", "gate", "h0", "fp8", "step"])
def test_transforms_raise(which):
    """torch.func's transforms and batched gradients are refused, whatever the operator has of a gradient."""
    t, calls = _calls()
    fn = calls[which]
    for call in (lambda: torch.func.vmap(fn)(torch.stack([t, t])), lambda: torch.func.grad(lambda a: fn(a).sum())(t),
                 lambda: torch.func.jvp(fn, (t,), (t,)), lambda: torch.func.functionalize(fn)(t)):
        with pytest.raises(RuntimeError):
            call()
    if which not in ("fp8", "step"):
        x = t.clone().requires_grad_()
        y = fn(x)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, x, torch.stack([torch.ones_like(y)] * 2), is_grads_batched=True)
