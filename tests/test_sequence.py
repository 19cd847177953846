"""The sequence operators on the CPU: their pure-torch semantics against the float64 oracle, gradients against central
differences, and what they refuse (the same checks run before a device launch)."""
import numpy as np
import pytest
import torch

from tests import sequence_oracle as O
from x_amd import ops
from x_amd.ops import reference as ref


def _close(got, want, bound, dtype=torch.float32):
    got = got.detach().double().numpy()
    tol = bound + O.rounding(dtype, np.abs(want) + bound)
    assert got.shape == want.shape and np.all(np.abs(got - want) <= tol), float(np.max(np.abs(got - want) / tol))


START = [0, 0, 1, 5, 5, 5, 12, 20, 20]


@pytest.mark.parametrize("with_dt", [False, True])
@pytest.mark.parametrize("with_h0", [False, True])
def test_scan_semantics_and_gradients(with_dt, with_h0):
    rng = np.random.default_rng(3)
    N, D, B = START[-1], 5, len(START) - 1
    x, g, gy = rng.normal(size=(3, N, D)).astype(np.float32)
    dt = rng.exponential(size=N).astype(np.float32) if with_dt else None
    h0 = rng.normal(size=(B, D)).astype(np.float32) if with_h0 else None
    gl = rng.normal(size=(B, D)).astype(np.float32)
    t = lambda a: None if a is None else torch.tensor(a)
    xt, gt, ht = t(x).requires_grad_(), t(g).requires_grad_(), t(h0)
    if ht is not None:
        ht.requires_grad_()
    y, last = ops.gated_scan(xt, gt, torch.tensor(START), dt=t(dt), h0=ht)
    wy, wl, E = O.scan(x.astype(float), g.astype(float), START, dt, h0)
    _close(y, wy, E)
    assert np.allclose(last.detach().numpy(), wl, atol=1e-5)
    wrt = (xt, gt) if ht is None else (xt, gt, ht)
    grads = torch.autograd.grad((y, last), wrt, (t(gy), t(gl)))
    want, bound = O.scan_bwd(x.astype(float), g.astype(float), START, gy.astype(float), gl.astype(float), dt, h0)
    for a, b, c in zip(grads, want, bound):
        _close(a, b, 4 * c + 1e-7)                          # autograd forms the products in another order


def test_scan_oracle_gradients_are_its_differences():
    rng = np.random.default_rng(4)
    N, D, B = START[-1], 3, len(START) - 1
    x, g, gy = rng.normal(size=(3, N, D))
    dt, h0, gl = rng.exponential(size=N), rng.normal(size=(B, D)), rng.normal(size=(B, D))
    grads, _ = O.scan_bwd(x, g, START, gy, gl, dt, h0)

    def loss(x, g, h0):
        y, last, _ = O.scan(x, g, START, dt, h0)
        return (y * gy).sum() + (last * gl).sum()

    at = [x, g, h0]
    for k in range(3):
        v = rng.normal(size=at[k].shape)
        hi, lo = [list(at) for _ in range(2)]
        hi[k], lo[k] = at[k] + 1e-5 * v, at[k] - 1e-5 * v
        # central differences in float64: 1e-10 of curvature, 1e-16 / 1e-5 of rounding, of sums of some hundred terms
        assert abs((loss(*hi) - loss(*lo)) / 2e-5 - (grads[k] * v).sum()) < 1e-6


def test_step_is_the_scan_token_by_token():
    rng = np.random.default_rng(5)
    n, T, D = 3, 6, 4
    x, g = torch.tensor(rng.normal(size=(2, n * T, D)).astype(np.float32))
    dt = torch.tensor(rng.exponential(size=n * T).astype(np.float32))
    y, last = ops.gated_scan(x, g, torch.arange(n + 1) * T, dt=dt)
    state = torch.zeros(n, D)
    at = torch.arange(n) * T
    for k in range(T):
        out = ops.gated_scan_step(x[at + k], g[at + k], state, dt=dt[at + k])
        assert torch.allclose(out, y[at + k], atol=1e-6)
    assert torch.allclose(state, last, atol=1e-6)


@pytest.mark.parametrize("p", [0.0, 0.3])
def test_norm_semantics_and_gradients(p):
    rng = np.random.default_rng(6)
    N, D, eps, seed, off = 7, 11, 1e-3, 0x1234_5678_9ABC_DEF1, 3
    x, res, gy, gs = rng.normal(size=(4, N, D)).astype(np.float32)
    w = rng.normal(size=D).astype(np.float32)
    ts = [torch.tensor(a).requires_grad_() for a in (x, res, w)]
    y, s = ops.residual_rms_norm(*ts, eps=eps, p=p, seed=seed, offset=off)
    keep = O.keeps(N, D, p, seed, off) * (65536 / (65536 - round(65536 * p)))
    _close(s, res + x * keep, 2 * O.U * np.abs(x * keep))
    sd = s.detach().double().numpy()
    wy, _ = O.norm(sd, w.astype(float), eps)
    _close(y, wy, 16 * O.U * np.abs(wy))
    gx, gr, gw = torch.autograd.grad((y, s), ts, (torch.tensor(gy), torch.tensor(gs)))
    (ds, dw), (bs, bw) = O.norm_bwd(sd, w.astype(float), eps, gy.astype(float), gs.astype(float))
    _close(gr, ds, bs)
    _close(gx, ds * keep, (bs + O.U * np.abs(ds)) * keep)
    _close(gw, dw, bw)


def test_norm_oracle_gradients_are_its_differences():
    rng = np.random.default_rng(7)
    s, gy, gs = rng.normal(size=(3, 4, 9))
    w, eps = rng.normal(size=9), 1e-2
    (ds, dw), _ = O.norm_bwd(s, w, eps, gy, gs)
    loss = lambda s, w: (O.norm(s, w, eps)[0] * gy).sum() + (s * gs).sum()
    v, u = rng.normal(size=s.shape), rng.normal(size=9)
    assert abs((loss(s + 1e-5 * v, w) - loss(s - 1e-5 * v, w)) / 2e-5 - (ds * v).sum()) < 1e-6
    assert abs((loss(s, w + 1e-5 * u) - loss(s, w - 1e-5 * u)) / 2e-5 - (dw * u).sum()) < 1e-6


def test_dropout_shares_and_scales():
    x = torch.ones(4000, 32)
    _, s = ops.residual_rms_norm(x, None, torch.ones(32), p=0.25, seed=9)
    kept = s != 0
    assert torch.all(s[kept] == 65536 / (65536 - 16384))
    # 128000 draws: a standard deviation of 0.0012
    assert abs(kept.float().mean().item() - 0.75) < 0.006
    _, other = ops.residual_rms_norm(x, None, torch.ones(32), p=0.25, seed=9, offset=1)
    assert (kept != (other != 0)).any()
    y, same = ops.residual_rms_norm(x, None, torch.ones(32))
    assert same is x


def test_embed_semantics():
    rng = np.random.default_rng(8)
    table = torch.tensor(rng.normal(size=(6, 4)).astype(np.float32), requires_grad=True)
    ids = torch.tensor([[0, 5, -1], [6, 5, 2 ** 40]])
    y = ops.embed_tokens(ids, table, scale=2.0)
    assert torch.equal(y[0, 0], table[0] * 2) and torch.equal(y[0, 1], table[5] * 2)
    assert not y[0, 2].any() and not y[1, 0].any() and not y[1, 2].any()
    g = torch.tensor(rng.normal(size=(2, 3, 4)).astype(np.float32))
    got = torch.autograd.grad(y, table, g)[0]
    want, bound = O.embed_bwd(ids.numpy().ravel(), 6, 2.0, g.double().numpy().reshape(6, 4))
    _close(got, want, bound)


def test_fp8_semantics():
    rng = np.random.default_rng(9)
    x, res = torch.tensor(rng.normal(size=(2, 5, 24)).astype(np.float32))
    x[3], res[3] = 0, 0
    w = torch.tensor(rng.normal(size=24).astype(np.float32))
    q, scale, s = ops.residual_rms_norm_fp8(x, res, w)
    y, _ = O.norm(s.double().numpy(), w.double().numpy(), 1e-6)
    _fp8_close(q, scale, y)


def _fp8_close(q, scale, y):
    """Half a step of e4m3 (a 16th, or 2^-10 below its normal range), and what the value rounds off before."""
    top = np.maximum(np.abs(y).max(1, keepdims=True), 1e-30)
    assert np.all(np.abs(scale.double().cpu().numpy() - top / 448) <= 64 * O.U * top / 448)
    want = y * 448 / top
    err = np.abs(q.float().double().cpu().numpy() - want)
    assert np.all(err <= (np.abs(want) / 16 + 2.0 ** -10) * 1.0001)


def test_reference_philox_is_the_published_generator():
    from tests.test_noise import KAT
    for ctr, key, want in KAT:
        got = ref.philox4x32_10([torch.tensor([c]) for c in ctr], key[0] | key[1] << 32)
        assert tuple(int(v) for v in got) == tuple(want)


def test_refusals():
    f, i = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    st = torch.tensor([0, 4])
    bad = [
        (TypeError, lambda: ops.embed_tokens(i, torch.zeros(4, 8, dtype=torch.int64))),
        (TypeError, lambda: ops.embed_tokens(f, f)),
        (TypeError, lambda: ops.embed_tokens([1], f)),
        (TypeError, lambda: ops.embed_tokens(i, f, dtype=torch.float64)),
        (ValueError, lambda: ops.embed_tokens(i, torch.zeros(8))),
        (ValueError, lambda: ops.embed_tokens(i, torch.zeros(0, 8))),
        (TypeError, lambda: ops.residual_rms_norm(f.double(), None, torch.ones(8))),
        (ValueError, lambda: ops.residual_rms_norm(f, None, torch.ones(7))),
        (ValueError, lambda: ops.residual_rms_norm(f, torch.zeros(3, 8), torch.ones(8))),
        (TypeError, lambda: ops.residual_rms_norm(f, f.half(), torch.ones(8))),
        (ValueError, lambda: ops.residual_rms_norm(f, f, torch.ones(8), p=1.0)),
        (ValueError, lambda: ops.residual_rms_norm(f, f, torch.ones(8), p=-0.1)),
        (ValueError, lambda: ops.residual_rms_norm(f, f, torch.ones(8), p=1 - 2 ** -20)),
        (ValueError, lambda: ops.residual_rms_norm(f, f, torch.ones(8), eps=-1.0)),
        (ValueError, lambda: ops.residual_rms_norm(f, f, torch.ones(8), eps=float("nan"))),
        (ValueError, lambda: ops.residual_rms_norm(torch.zeros(1, 8193), None, torch.ones(8193))),
        (ValueError, lambda: ops.residual_rms_norm_fp8(f, f, torch.ones(9))),
        (TypeError, lambda: ops.gated_scan(f.double(), f.double(), st)),
        (ValueError, lambda: ops.gated_scan(f, f.half(), st)),
        (ValueError, lambda: ops.gated_scan(f, f[:3], st)),
        (ValueError, lambda: ops.gated_scan(f, f, st.float())),
        (ValueError, lambda: ops.gated_scan(f, f, torch.tensor([0]))),
        (ValueError, lambda: ops.gated_scan(f, f, st, dt=torch.zeros(3))),
        (ValueError, lambda: ops.gated_scan(f, f, st, dt=torch.zeros(4, requires_grad=True))),
        (ValueError, lambda: ops.gated_scan(f, f, st, h0=torch.zeros(2, 8))),
        (ValueError, lambda: ops.gated_scan_step(f, f, torch.zeros(4, 8).half())),
        (ValueError, lambda: ops.gated_scan_step(f, f, torch.zeros(8, 4).t())),
        (ValueError, lambda: ops.gated_scan_step(f, f, torch.zeros(3, 8))),
    ]
    for k, (err, fn) in enumerate(bad):
        with pytest.raises(err):
            fn()
            pytest.fail(f"case {k} was accepted")


def test_entries_reject_before_launch():
    """The C entries check sizes, types, settings and workspaces on the host (no device is touched)."""
    import ctypes
    from x_amd.ops import _ext
    L = _ext.load_library()
    fake, n = ctypes.c_void_p(4096), None                    # an aligned, never dereferenced address

    def refused(rc, word):
        assert rc == 1 and word in L.atl_last_error(), (rc, L.atl_last_error())

    refused(L.atl_embed_fwd(fake, 1, -1, fake, 8, 0, 4, 8, 1.0, fake, 0, n), b"bad sizes")
    refused(L.atl_embed_fwd(fake, 1, 5, fake, 8, 3, 4, 8, 1.0, fake, 0, n), b"bad sizes")
    refused(L.atl_embed_fwd(n, 1, 5, fake, 8, 0, 4, 8, 1.0, fake, 0, n), b"null")
    need = L.atl_embed_bwd_ws_bytes(5, 4, 8)
    assert need > 0 and L.atl_embed_bwd_ws_bytes(5, 0, 8) == -1
    refused(L.atl_embed_bwd(fake, 1, 5, fake, 8, 0, 4, 8, 1.0, fake, 0, fake, need - 1, n), b"workspace")
    refused(L.atl_embed_bwd(fake, 1, 5, fake, 8, 0, 4, 8, 1.0, ctypes.c_void_p(4100), 0, fake, need, n), b"aligned")
    refused(L.atl_rms_norm_fwd(fake, 8, 0, n, 0, 1, fake, 5, 8, 1e-6, 0.0, 0, 0, fake, n, n, n), b"bad sizes")
    refused(L.atl_rms_norm_fwd(fake, 8, 0, n, 0, 0, fake, 5, 8, 1e-6, 1.0, 0, 0, fake, n, n, n), b"bad sizes")
    refused(L.atl_rms_norm_fwd(fake, 8, 0, n, 0, 0, fake, 5, 9000, 1e-6, 0.0, 0, 0, fake, n, n, n), b"bad sizes")
    refused(L.atl_rms_norm_fwd(fake, 8, 0, n, 0, 0, n, 5, 8, 1e-6, 0.0, 0, 0, fake, n, n, n), b"null")
    need = L.atl_rms_norm_bwd_ws_bytes(5, 8)
    refused(L.atl_rms_norm_bwd(fake, 8, 0, fake, fake, 8, 0, n, 0, 5, 8, 1e-6, 0.0, 0, 0, fake, fake, fake, fake,
                               need - 1, n), b"workspace")
    need = L.atl_gated_scan_ws_bytes(5, 8, 0)
    assert need > 0 and L.atl_gated_scan_ws_bytes(5, 8, 7) == -1 and L.atl_gated_scan_groups(-1) == -1
    refused(L.atl_gated_scan_fwd(fake, 8, fake, 8, 0, 5, 8, fake, 0, n, n, fake, fake, n, fake, need, n), b"bad sizes")
    refused(L.atl_gated_scan_fwd(fake, 8, fake, 8, 0, 5, 8, fake, 1, n, n, fake, fake, n, fake, need - 1, n), b"workspace")
    refused(L.atl_gated_scan_bwd(fake, 8, fake, 8, 0, 5, 8, fake, 1, n, n, n, fake, 8, n, fake, fake, n, fake, need, n),
            b"null")
    refused(L.atl_gated_scan_step(fake, -1, fake, 8, 0, 5, 8, n, fake, fake, n), b"bad sizes")
