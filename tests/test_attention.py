"""The attention operators on the CPU: the definitions, gradients against differences, the single-token form, refusals."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from tests import attention_oracle as O
from x_amd import ops
from x_amd.ops import reference as ref


def _case(N, H, D, start, seed=0, dt=True, h0=True):
    rng = np.random.default_rng(seed)
    q, k, v, gy = rng.normal(size=(4, N, H, D))
    B = len(start) - 1
    return (q, k, v, rng.random(H) + 0.1, start, rng.random(N) if dt else None,
            rng.normal(size=(B, H, D, D)) if h0 else None), gy, rng.normal(size=(B, H, D, D))


def _torch(args, scale):
    q, k, v, rate, start, dt, h0 = (None if a is None else torch.as_tensor(a) for a in args)
    wrt = [t.requires_grad_() for t in (q, k, v, h0) if t is not None]
    return ref.decay_attention(q, k, v, rate, start, dt, h0, scale), wrt


@pytest.mark.parametrize("with_dt", [False, True])
@pytest.mark.parametrize("with_h0", [False, True])
def test_attention_semantics_and_gradients(with_dt, with_h0):
    start = [0, 7, 7, 8, 30]
    args, gy, gl = _case(30, 2, 5, start, dt=with_dt, h0=with_h0)
    (y, last), wrt = _torch(args, 0.7)
    (wy, wl), _ = O.attention(*args, 0.7, "float32")
    assert np.allclose(y.detach(), wy, atol=1e-12) and np.allclose(last.detach(), wl, atol=1e-12)
    got = torch.autograd.grad((y, last), wrt, (torch.as_tensor(gy), torch.as_tensor(gl)))
    want, _ = O.attention_bwd(*args, 0.7, gy, gl, "float32")
    for a, b in zip(got, want):
        assert np.allclose(a, b, atol=1e-12)


def test_attention_oracle_gradients_are_its_differences():
    args, gy, gl = _case(9, 1, 3, [0, 4, 9], seed=2)
    scale = 0.5
    grads, _ = O.attention_bwd(*args, scale, gy, gl, "float32")

    def loss(a):
        (y, last), _ = O.attention(*a, scale, "float32")
        return (y * gy).sum() + (last * gl).sum()

    step, rng = 1e-5, np.random.default_rng(0)
    for place, g in zip((0, 1, 2, 6), grads):
        for _ in range(5):
            at = tuple(rng.integers(0, n) for n in args[place].shape)
            sides = []
            for sign in (1, -1):
                a = list(args)
                a[place] = args[place].copy()
                a[place][at] += sign * step
                sides.append(loss(a))
            assert abs((sides[0] - sides[1]) / (2 * step) - g[at]) < 1e-7


def test_step_is_the_attention_token_by_token():
    args, _, _ = _case(12, 2, 4, [0, 12], seed=3, h0=False)
    (y, last), _ = _torch(args, 0.5)
    q, k, v, rate, _, dt, _ = args
    state = torch.zeros(1, 2, 4, 4, dtype=torch.float64)
    for i in range(12):
        row = [torch.as_tensor(a[i:i + 1]) for a in (q, k, v)]
        out = ref.decay_attention_step(*row, torch.as_tensor(rate), state, torch.as_tensor(dt[i:i + 1]), 0.5)
        assert torch.allclose(out[0], y[i])
    assert torch.allclose(state, last)


def test_tokens_outside_of_the_windows_are_zeros():
    args, _, _ = _case(20, 2, 4, [3, 9, 15], seed=4)
    (y, last), wrt = _torch(args, 1.0)
    assert not y[:3].any() and not y[15:].any() and y[3:15].all()
    grads = torch.autograd.grad(y.sum(), wrt[:3])
    assert all(not g[:3].any() and not g[15:].any() for g in grads)


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("sections,D", [((2, 1), 8), ((4,), 8), ((0, 3, 0), 7), ((0,), 3)])
def test_rotary_semantics_and_gradients(norm, sections, D):
    rng = np.random.default_rng(D)
    N = 11
    q, k = rng.normal(size=(N, 3, D)), rng.normal(size=(N, 2, D))
    gq, gk = rng.normal(size=q.shape), rng.normal(size=k.shape)
    wq, wk = (rng.normal(size=D), rng.normal(size=D)) if norm else (None, None)
    pos, freqs = rng.random((N, len(sections))) * 100, rng.random(sum(sections))
    ins = [None if a is None else torch.as_tensor(a).requires_grad_() for a in (q, k, wq, wk)]
    got = ref.head_norm_rotary(*ins, torch.as_tensor(pos), torch.as_tensor(freqs), sections, 1e-5)
    grads = torch.autograd.grad(got, [t for t in ins if t is not None], (torch.as_tensor(gq), torch.as_tensor(gk)))
    angle = O.angles(pos, freqs, sections)
    for x, w, g, y, j in ((q, wq, gq, got[0], 0), (k, wk, gk, got[1], 1)):
        assert np.allclose(y.detach(), O.rotary(x, w, angle, 1e-5)[0], atol=1e-12)
        (gx, gw), _ = O.rotary_bwd(x, w, angle, 1e-5, g)
        assert np.allclose(grads[j], gx, atol=1e-12)
        assert gw is None or np.allclose(grads[2 + j], gw, atol=1e-12)


def test_rotary_oracle_gradients_are_its_differences():
    rng = np.random.default_rng(8)
    x, w, gy = rng.normal(size=(4, 2, 6)), rng.normal(size=6), rng.normal(size=(4, 2, 6))
    angle = O.angles(rng.random((4, 2)) * 9, rng.random(3), (1, 2))
    (gx, gw), _ = O.rotary_bwd(x, w, angle, 1e-4, gy)
    loss = lambda a, b: (O.rotary(a, b, angle, 1e-4)[0] * gy).sum()
    step = 1e-6
    for at in ((0, 0, 0), (1, 1, 5), (3, 0, 2)):
        d = np.zeros_like(x)
        d[at] = step
        assert abs((loss(x + d, w) - loss(x - d, w)) / (2 * step) - gx[at]) < 1e-7
    for c in range(6):
        d = np.zeros(6)
        d[c] = step
        assert abs((loss(x, w + d) - loss(x, w - d)) / (2 * step) - gw[c]) < 1e-7


def test_rotated_products_depend_on_distances():
    """Moving all positions leaves the products of queries and keys as they are, on every axis; far positions too."""
    rng = torch.Generator().manual_seed(0)
    q, k = torch.randn(2, 6, 1, 12, generator=rng).double().float()
    pos, freqs = torch.rand(6, 3, generator=rng).double() * 30, torch.rand(6, generator=rng)
    a, b = ops.head_norm_rotary(q, k, None, None, pos, freqs, (1, 2, 3))
    c, d = ops.head_norm_rotary(q, k, None, None, pos + torch.tensor([1e6, -3e5, 12.0]), freqs, (1, 2, 3))
    assert torch.allclose(a[:, 0] @ b[:, 0].t(), c[:, 0] @ d[:, 0].t(), atol=1e-4)
    ints = ops.head_norm_rotary(q, k, None, None, torch.full((6, 1), 2 ** 40, dtype=torch.int64), freqs, (6,))[0]
    same = ops.head_norm_rotary(q, k, None, None, torch.full((6, 1), float(2 ** 40), dtype=torch.float64), freqs, (6,))[0]
    assert torch.equal(ints, same)


def test_refusals():
    f, st = torch.zeros(4, 2, 8), torch.tensor([0, 4])
    r, w, pos, fr = torch.ones(2), torch.ones(8), torch.zeros(4, 2), torch.ones(4)
    S = torch.zeros(4, 2, 8, 8)
    rot = lambda q=f, k=f, wq=w, wk=w, p=pos, fq=fr, s=(2, 2), **kw: ops.head_norm_rotary(q, k, wq, wk, p, fq, s, **kw)
    att = lambda q=f, k=f, v=f, ra=r, s=st, **kw: ops.decay_attention(q, k, v, ra, s, **kw)
    step = lambda q=f, k=f, v=f, ra=r, s=S, **kw: ops.decay_attention_step(q, k, v, ra, s, **kw)
    rot(), att(), step()                                    # as they are, they are taken
    bad = [
        (TypeError, lambda: rot(q=f.double())),
        (TypeError, lambda: rot(k=f.half())),
        (TypeError, lambda: rot(q=[1])),
        (ValueError, lambda: rot(q=f[0])),
        (ValueError, lambda: rot(k=f[:3])),
        (ValueError, lambda: rot(k=f[..., :6])),
        (ValueError, lambda: rot(wq=None)),
        (ValueError, lambda: rot(wk=torch.ones(7))),
        (TypeError, lambda: rot(wk=torch.ones(8, dtype=torch.int32))),
        (ValueError, lambda: rot(s=(2, 3))),
        (ValueError, lambda: rot(s=(5, -1))),
        (ValueError, lambda: rot(s=())),
        (ValueError, lambda: rot(s=(1, 1, 1, 1, 0), p=torch.zeros(4, 5))),
        (ValueError, lambda: rot(s=(4,))),
        (ValueError, lambda: rot(p=torch.zeros(3, 2))),
        (TypeError, lambda: rot(p=torch.zeros(4, 2, dtype=torch.bool))),
        (ValueError, lambda: rot(fq=torch.ones(3))),
        (ValueError, lambda: rot(fq=torch.ones(4, dtype=torch.int64))),
        (ValueError, lambda: rot(p=torch.zeros(4, 2, requires_grad=True))),
        (ValueError, lambda: rot(fq=torch.ones(4, requires_grad=True))),
        (ValueError, lambda: rot(eps=-1.0)),
        (ValueError, lambda: rot(eps=float("nan"))),
        (ValueError, lambda: rot(q=torch.zeros(4, 1, 257), k=torch.zeros(4, 1, 257), wq=None, wk=None)),
        (TypeError, lambda: att(q=f.double())),
        (TypeError, lambda: att(v=f.half())),
        (ValueError, lambda: att(k=f[:, :1])),
        (ValueError, lambda: att(v=f[..., :6])),
        (ValueError, lambda: att(ra=torch.ones(3))),
        (ValueError, lambda: att(ra=torch.ones(2, dtype=torch.int64))),
        (ValueError, lambda: att(ra=torch.ones(2, requires_grad=True))),
        (ValueError, lambda: att(s=st.float())),
        (ValueError, lambda: att(s=torch.zeros(0, dtype=torch.int64))),
        (ValueError, lambda: att(dt=torch.zeros(3))),
        (ValueError, lambda: att(dt=torch.zeros(4, requires_grad=True))),
        (ValueError, lambda: att(h0=torch.zeros(2, 2, 8, 8))),
        (TypeError, lambda: att(h0=torch.zeros(1, 2, 8, 8, dtype=torch.float64))),
        (ValueError, lambda: att(scale=float("inf"))),
        (ValueError, lambda: att(q=torch.zeros(4, 2, 129), k=torch.zeros(4, 2, 129), v=torch.zeros(4, 2, 129))),
        (ValueError, lambda: step(s=S.half())),
        (ValueError, lambda: step(s=S[:3])),
        (ValueError, lambda: step(s=S.transpose(2, 3))),
        (ValueError, lambda: step(s=S.clone().requires_grad_())),
        (ValueError, lambda: step(dt=torch.zeros(3))),
    ]
    for k, (err, fn) in enumerate(bad):
        with pytest.raises(err):
            fn()
            pytest.fail(f"case {k} was accepted")


def test_entries_reject_before_launch():
    """The C entries check sizes, types, settings and workspaces on the host (no device is touched)."""
    from x_amd.ops import _ext
    L = _ext.load_library()
    fake, n = ctypes.c_void_p(4096), None                    # an aligned, never dereferenced address
    rows = (fake, 16, 8)

    def refused(rc, word):
        assert rc == 1 and word in L.atl_last_error(), (rc, L.atl_last_error())

    sec = lambda *m: (ctypes.c_int64 * len(m))(*m)
    rot = lambda N=5, D=8, A=2, s=sec(2, 2), dtype=0, eps=1e-6, pos=fake, out=fake: L.atl_head_norm_rotary_fwd(
        *rows, *rows, dtype, n, n, pos, 0, fake, A, s, N, 2, 2, D, eps, out, out, n)
    refused(rot(N=-1), b"bad sizes")
    refused(rot(D=257), b"bad sizes")
    refused(rot(A=5), b"bad sizes")
    refused(rot(s=sec(2, 3)), b"bad sizes")
    refused(rot(s=sec(5, -1)), b"bad sizes")
    refused(rot(dtype=3), b"bad sizes")
    refused(rot(eps=-1.0), b"bad sizes")
    refused(rot(pos=n), b"null")
    refused(rot(out=n), b"null")
    need = L.atl_head_norm_rotary_bwd_ws_bytes(2, 2, 8)
    assert need > 0 and L.atl_head_norm_rotary_bwd_ws_bytes(2, 2, 0) == -1 and L.atl_head_norm_rotary_bwd_ws_bytes(2, 2, 257) == -1
    back = lambda ws=fake, bytes=need: L.atl_head_norm_rotary_bwd(*rows, *rows, 0, fake, fake, fake, 0, fake, 2, sec(2, 2), 5, 2, 2,
                                                                  8, 1e-6, *rows, *rows, fake, fake, fake, ws, bytes, n)
    refused(back(bytes=need - 1), b"workspace")
    refused(back(ws=n), b"null")
    need = L.atl_decay_attn_states_bytes(100_000, 1, 2, 8)
    assert need > 0 and L.atl_decay_attn_states_bytes(5, 1, 2, 8) == 0
    assert L.atl_decay_attn_states_bytes(5, 1, 2, 129) == L.atl_decay_attn_states_bytes(-1, 1, 2, 8) == -1
    fwd = lambda N=100_000, D=8, dtype=0, B=1, held=fake, bytes=need, sn=16, start=fake: L.atl_decay_attn_fwd(
        fake, sn, 8, *rows, *rows, dtype, N, 2, D, fake, start, B, n, n, 1.0, fake, fake, held, bytes, n)
    refused(fwd(N=-1), b"bad sizes")
    refused(fwd(D=0), b"bad sizes")
    refused(fwd(B=-1), b"bad sizes")
    refused(fwd(dtype=7), b"bad sizes")
    refused(fwd(sn=-1), b"bad sizes")
    refused(fwd(sn=7), b"bad sizes")
    refused(fwd(sn=2 ** 22), b"bad sizes")
    refused(fwd(held=n), b"null")
    refused(fwd(start=n), b"null")
    refused(fwd(bytes=need - 1), b"states")
    bwd = lambda gq=fake, ws=fake, bytes=need: L.atl_decay_attn_bwd(*rows, *rows, *rows, *rows, 0, 100_000, 2, 8, fake, fake, 1, n, n,
                                                                    n, 1.0, fake, gq, fake, fake, n, ws, bytes, n)
    refused(bwd(gq=n), b"null")
    refused(bwd(ws=n), b"null")
    refused(bwd(bytes=need - 1), b"workspace")
    refused(L.atl_decay_attn_step(*rows, *rows, *rows, 0, 5, 2, 200, fake, n, 1.0, fake, fake, n), b"bad sizes")
    refused(L.atl_decay_attn_step(*rows, *rows, *rows, 0, 5, 2, 8, fake, n, 1.0, n, fake, n), b"null")


_NO_WINDOW = """
import ctypes
from x_amd.ops import _ext
L, fake, n = _ext.load_library(), ctypes.c_void_p(4096), None
for D in (8, 64):
    rows, held = (fake, 2 * D, D), L.atl_decay_attn_states_bytes({N}, {B}, 2, D)
    print(L.atl_decay_attn_fwd(*rows, *rows, *rows, 0, {N}, 2, D, fake, fake, {B}, n, n, 1.0, fake, fake, fake, held, n),
          L.atl_decay_attn_bwd(*rows, *rows, *rows, *rows, 0, {N}, 2, D, fake, fake, {B}, n, n, n, 1.0, fake, fake, fake, fake, n,
                               fake, held, n))
"""


@pytest.mark.parametrize("N,B", [(1000, 0), (2000, 0), (20_000, 0), (20_000, 1)])
def test_entries_return_without_windows(N, B):
    """Tokens and no window, past the length from which stretches are joined: the entry points' host part returns (an error
    here, since no device is visible to the process and nothing is launched)."""
    env = {**os.environ, "HIP_VISIBLE_DEVICES": "-1", "ROCR_VISIBLE_DEVICES": "-1"}
    run = subprocess.run([sys.executable, "-c", _NO_WINDOW.format(N=N, B=B)], env=env, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.split() == ["1"] * 4, (run.returncode, run.stdout, run.stderr)
