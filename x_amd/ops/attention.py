"""Attention over event tokens with a state of fixed size, on the HIP library (no counterpart in the reference's package).

* :func:`head_norm_rotary`      RMS norm of every head's queries and keys and their rotation by the token's position, of one
                                or several axes; grads to both and to the norms' weights
* :func:`decay_attention`       linear attention with a decay for each head over ragged windows of tokens; grads to queries,
                                keys, values and h0
* :func:`decay_attention_step`  its single-token form for streams, the state updated in place

Tokens are rows of H heads of D channels in single, bfloat16 or half precision; sums, norms and states are kept in single
precision.  Heads and tokens may lie apart (slices of one projection, heads of one tensor shared by ``expand``) as long as a
head's channels are contiguous; other layouts are copied first.  Device tensors run on the HIP kernels, CPU tensors on
:mod:`x_amd.ops.reference`.
"""
from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd.function import once_differentiable

from . import reference as ref
from ._ext import F32, I64, call, load_library, on_device, raw_stream
from .sequence import _CODE, _at, _float_type, _grads_wanted, _on, _plain, _route, _ws

MAX_ROTARY_WIDTH = 256
MAX_ROTARY_AXES = 4
MAX_ATTENTION_WIDTH = 128
MAX_TOKEN_STRIDE = 2 ** 22


def _heads(t: torch.Tensor) -> torch.Tensor:
    """``t`` (N, H, D) with contiguous heads: itself where they are, else a copy."""
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _chunks(t: torch.Tensor) -> torch.Tensor:
    """``t`` (N, H, D) as the attention over windows takes it: contiguous heads, tokens that lie apart but within reach of a
    chunk's 32-bit offsets (32 tokens); else a copy."""
    t = _heads(t)
    return t if t.shape[0] < 2 or t.shape[2] <= t.stride(0) < MAX_TOKEN_STRIDE else t.contiguous()


def _strides(t: torch.Tensor | None) -> tuple[int, int, int]:
    """Address, token stride and head stride as the entry points take them."""
    return (0, 0, 0) if t is None else (t.data_ptr(), t.stride(0), t.stride(1))


def _head_args(t, name: str, like=None, width: int = 0) -> None:
    _float_type(t, name)
    if t.dim() != 3 or t.shape[1] < 1 or t.shape[2] < 1:
        raise ValueError(f"{name} must be (N, H, D), got {tuple(t.shape)}")
    if width and t.shape[2] > width:
        raise ValueError(f"heads of up to {width} channels, got {t.shape[2]}")
    if like is not None:
        _on(t, name, like.device)
        if t.dtype != like.dtype:
            raise TypeError(f"{name} must be {like.dtype}, got {t.dtype}")


# ------------------------------------------------------------------------------------------- norm and rotation
@functools.lru_cache(maxsize=64)
def _sections(sections: tuple):
    return (ctypes.c_int64 * len(sections))(*sections)


def _doubles(pos, freqs) -> int:
    return (pos.dtype == torch.float64) + 2 * (freqs.dtype == torch.float64)


def _rotary_fwd(q, k, wq, wk, pos, freqs, sections, eps):
    N, H, D = q.shape
    Hk, dev = k.shape[1], q.device
    yq = torch.empty(N, H, D, dtype=q.dtype, device=dev)
    yk = torch.empty(N, Hk, D, dtype=q.dtype, device=dev)
    with on_device(dev):
        call("atl_head_norm_rotary_fwd", *_strides(q), *_strides(k), _CODE[q.dtype], _at(wq), _at(wk), _at(pos),
             _doubles(pos, freqs), _at(freqs), len(sections), _sections(sections), N, H, Hk, D, eps, _at(yq), _at(yk),
             raw_stream(dev))
    return yq, yk


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, pos, freqs, sections, eps):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(*((None, None) if wq is None else (q, k)), wq, wk, pos, freqs)
        ctx.meta = (q.shape, k.shape, q.dtype, sections, eps)
        return _rotary_fwd(q, k, wq, wk, pos, freqs, sections, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, gyq, gyk):
        q, k, wq, wk, pos, freqs = ctx.saved_tensors
        (N, H, D), kshape, dtype, sections, eps = ctx.meta
        if gyq is None and gyk is None:
            return (None,) * 8
        Hk, dev = kshape[1], pos.device
        want = ctx.needs_input_grad
        gyq, gyk = (None if g is None else _heads(g) for g in (gyq, gyk))
        gq = torch.empty(N, H, D, dtype=dtype, device=dev) if want[0] and gyq is not None else None
        gk = torch.empty(N, Hk, D, dtype=dtype, device=dev) if want[1] and gyk is not None else None
        gw = torch.empty(2, D, dtype=F32, device=dev) if want[2] or want[3] else None
        nbytes = int(load_library().atl_head_norm_rotary_bwd_ws_bytes(H, Hk, D)) if gw is not None else 0
        ws = _ws(nbytes, dev, "head_norm_rotary") if gw is not None else None
        with on_device(dev):
            call("atl_head_norm_rotary_bwd", *_strides(q), *_strides(k), _CODE[dtype], _at(wq), _at(wk), _at(pos),
                 _doubles(pos, freqs), _at(freqs), len(sections), _sections(sections), N, H, Hk, D, eps,
                 *_strides(gyq), *_strides(gyk), _at(gq), _at(gk), _at(gw), _at(ws), nbytes, raw_stream(dev))
        gwq = gw[0] if want[2] and gyq is not None else None
        gwk = gw[1] if want[3] and gyk is not None else None
        return gq, gk, gwq, gwk, None, None, None, None


def head_norm_rotary(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                     pos: torch.Tensor, freqs: torch.Tensor, sections, eps: float = 1e-6):
    """(q', k') of queries (N, H, D) and keys (N, Hk, D): every head's root-mean-square norm, x / sqrt(mean(x^2) + eps) *
    weight, and its channel pairs (2p, 2p + 1) turned by the angle pos[:, axis(p)] * freqs[p] (radians).

    ``pos`` (N, A) holds every token's position on up to four axes (time, row and column of an event; float32 or float64,
    integers are taken as float64), ``sections`` how many pairs turn with each axis, in order; channels past the last
    section's stay as the norm leaves them.  The product with a query of a key so turned depends on their distance along
    every axis alone.  Angles are reduced in 64 bits, of float64 frequencies too, so far positions keep them.  Weights (D,), both None: no norm, the
    rotation alone.  Up to 256 channels; the outputs are contiguous.  No gradient flows to pos and freqs."""
    _head_args(q, "q", width=MAX_ROTARY_WIDTH)
    _head_args(k, "k", like=q)
    N, _, D = q.shape
    if k.shape[0] != N or k.shape[2] != D:
        raise ValueError(f"k must be ({N}, Hk, {D}), got {tuple(k.shape)}")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("q_weight and k_weight are both given or both None")
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None:
            _on(w, name, q.device)
            _float_type(w, name)
            if w.shape != (D,):
                raise ValueError(f"{name} must be ({D},), got {tuple(w.shape)}")
    sections = tuple(int(m) for m in sections)
    A, pairs = len(sections), sum(sections)
    if not 1 <= A <= MAX_ROTARY_AXES or min(sections) < 0 or 2 * pairs > D:
        raise ValueError(f"sections must be the pairs of 1 to {MAX_ROTARY_AXES} axes, at most {D // 2} in all, got {sections}")
    _on(pos, "pos", q.device)
    _on(freqs, "freqs", q.device)
    if pos.shape != (N, A):
        raise ValueError(f"pos must be ({N}, {A}), got {tuple(pos.shape)}")
    if pos.is_complex() or pos.dtype == torch.bool:
        raise TypeError(f"pos must hold real positions, got {pos.dtype}")
    if freqs.shape != (pairs,) or not freqs.is_floating_point():
        raise ValueError(f"freqs must be ({pairs},) real numbers, got {tuple(freqs.shape)}, {freqs.dtype}")
    if pos.requires_grad or freqs.requires_grad:
        raise ValueError("no gradient flows to pos and freqs: detach them")
    eps = float(eps)
    if not 0 <= eps < 1e30:
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    through = _route(q, "head_norm_rotary")
    pos = _plain(pos, F32 if pos.dtype in (F32, torch.float16, torch.bfloat16) else torch.float64)
    if through is None:
        return ref.head_norm_rotary(q, k, q_weight, k_weight, pos, freqs, sections, eps)
    freqs = _plain(freqs, F32 if freqs.dtype in (F32, torch.float16, torch.bfloat16) else torch.float64)
    wq, wk = (None if w is None else _plain(w, F32) for w in (q_weight, k_weight))
    q, k = _heads(q), _heads(k)
    if through or _grads_wanted(q, k, wq, wk):
        return _Rotary.apply(q, k, wq, wk, pos, freqs, sections, eps)
    return _rotary_fwd(q, k, wq, wk, pos, freqs, sections, eps)


# ------------------------------------------------------------------------------------------- attention
def _decay_fwd(q, k, v, rate, start, dt, h0, scale):
    N, H, D = q.shape
    B, dev = start.numel() - 1, q.device
    y = torch.empty(N, H, D, dtype=q.dtype, device=dev)
    last = torch.empty(B, H, D, D, dtype=F32, device=dev)
    nbytes = int(load_library().atl_decay_attn_states_bytes(N, B, H, D))
    states = _ws(nbytes, dev, "decay_attention") if nbytes else None
    with on_device(dev):
        call("atl_decay_attn_fwd", *_strides(q), *_strides(k), *_strides(v), _CODE[q.dtype], N, H, D, _at(rate), _at(start), B,
             _at(dt), _at(h0), scale, _at(y), _at(last), _at(states), nbytes, raw_stream(dev))
    return y, last, states


class _Decay(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, rate, start, dt, h0, scale):
        y, last, states = _decay_fwd(q, k, v, rate, start, dt, h0, scale)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, rate, start, dt, h0, states)
        ctx.scale = scale
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, glast):
        q, k, v, rate, start, dt, h0, states = ctx.saved_tensors
        if gy is None and glast is None:
            return (None,) * 8
        N, H, D = q.shape
        B, dev = start.numel() - 1, q.device
        gy = None if gy is None else _chunks(gy)
        glast = None if glast is None else glast.contiguous()
        gq, gk, gv = (torch.empty(N, H, D, dtype=q.dtype, device=dev) for _ in range(3))
        gh0 = torch.empty(B, H, D, D, dtype=F32, device=dev) if ctx.needs_input_grad[6] else None
        nbytes = 0 if states is None else states.numel()
        ws = None if states is None else torch.empty_like(states)
        with on_device(dev):
            call("atl_decay_attn_bwd", *_strides(q), *_strides(k), *_strides(v), *_strides(gy), _CODE[q.dtype], N, H, D,
                 _at(rate), _at(start), B, _at(dt), _at(h0), _at(glast), ctx.scale, _at(states), _at(gq), _at(gk), _at(gv),
                 _at(gh0), _at(ws), nbytes, raw_stream(dev))
        return gq, gk, gv, None, None, None, gh0, None


def _attn_args(q, k, v, rate, dt, scale):
    _head_args(q, "q", width=MAX_ATTENTION_WIDTH)
    for t, name in ((k, "k"), (v, "v")):
        _head_args(t, name, like=q)
        if t.shape != q.shape:
            raise ValueError(f"{name} must be {tuple(q.shape)}, got {tuple(t.shape)}")
    N, H, D = q.shape
    _on(rate, "rate", q.device)
    if rate.shape != (H,) or not rate.is_floating_point():
        raise ValueError(f"rate must be ({H},) real numbers, got {tuple(rate.shape)}, {rate.dtype}")
    if rate.requires_grad:
        raise ValueError("no gradient flows to rate: detach it")
    if dt is not None:
        _on(dt, "dt", q.device)
        if dt.shape != (N,):
            raise ValueError(f"dt must be ({N},), got {tuple(dt.shape)}")
        if dt.requires_grad:
            raise ValueError("no gradient flows to dt: detach it")
        dt = _plain(dt, F32)
    scale = D ** -0.5 if scale is None else float(scale)
    if not abs(scale) < 1e30:
        raise ValueError(f"scale must be finite, got {scale}")
    return _plain(rate, F32), dt, scale


def decay_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rate: torch.Tensor, start: torch.Tensor,
                    dt: torch.Tensor | None = None, h0: torch.Tensor | None = None, scale: float | None = None):
    """(y, last): linear attention of every head over the tokens (N, H, D) of each window,

        y_i = scale sum_{j <= i} exp(-rate (dt_{j+1} + ... + dt_i)) (q_i k_j) v_j  =  scale q_i S_i,
        S_i = exp(-rate dt_i) S_{i-1} + k_i v_i^T,

    from h0 (B, H, D, D) or zero.  y (N, H, D) is in q's type, last (B, H, D, D) each window's last state in float32 (an empty
    window's: h0 or zero), to go on from; its rows are the keys' channels.  ``rate`` (H,) is every head's decay, ``dt`` (N,)
    the gap to the token before in units of a time constant (the first token's: since h0); None stands for ones.  scale is
    1 / sqrt(D) if None.  Up to 128 channels.

    ``start`` (B + 1) holds the windows' first tokens and the last one's end (``EventPacket.offsets``); it must ascend within
    [0, N], which is not checked on the device (no call reads past its tensors if it does not).  Tokens outside of it are in
    no window: zeros, and zero gradients.  A key and a value that all heads share are given as views, ``k.expand(N, H, D)``
    of (N, 1, D), which are read as they lie; those of Hk < H heads as copies, ``k.repeat_interleave(H // Hk, 1)``.  Their
    gradients come out per head, each rounded to their type, and autograd adds them.  An endless gap forgets what was before it (with a
    positive rate), a negative one grows the state as the formula has it.  NaN and infinities go where the formula takes them,
    signs included, but a stretch of tokens that they reach is followed token by token, in some 20 times the time.  No
    gradient flows to rate and dt.

    Products run on the matrix cores.  With 16-bit inputs the pairs' weights and the states that meet a query go in as two
    pieces of that type (within 2^-17 of themselves, a 256th of a bfloat16 output's own rounding; in half precision less of what
    lies 2^28 below the largest of its value channel or token), tokens' shares of a state as three; states are kept and
    returned in single precision."""
    rate, dt, scale = _attn_args(q, k, v, rate, dt, scale)
    N, H, D = q.shape
    _on(start, "start", q.device)
    if start.dim() != 1 or start.numel() < 1 or start.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"start must be (B + 1,) of int64 or int32, got {tuple(start.shape)}, {start.dtype}")
    B = start.numel() - 1
    if h0 is not None:
        _on(h0, "h0", q.device)
        _float_type(h0, "h0")
        if h0.shape != (B, H, D, D):
            raise ValueError(f"h0 must be ({B}, {H}, {D}, {D}), got {tuple(h0.shape)}")
    start = _plain(start, I64)
    through = _route(q, "decay_attention")
    if H * D >= MAX_TOKEN_STRIDE:
        raise ValueError(f"a token of fewer than {MAX_TOKEN_STRIDE} channels in all heads, got {H} x {D}")
    if through is None:
        return ref.decay_attention(q, k, v, rate, start, dt, h0, scale)
    h0 = None if h0 is None else _plain(h0, F32)
    q, k, v = _chunks(q), _chunks(k), _chunks(v)
    if through or _grads_wanted(q, k, v, h0):
        return _Decay.apply(q, k, v, rate, start, dt, h0, scale)
    return _decay_fwd(q, k, v, rate, start, dt, h0, scale)[:2]


def decay_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rate: torch.Tensor, state: torch.Tensor,
                         dt: torch.Tensor | None = None, scale: float | None = None):
    """One token of each of N streams: ``state`` (N, H, D, D) float32 becomes exp(-rate dt) state + k v^T in place; returns
    scale q state (N, H, D) in q's type (:func:`decay_attention` of one token).  For inference (no gradient): a backward
    that needs the state as it was raises."""
    rate, dt, scale = _attn_args(q, k, v, rate, dt, scale)
    (N, H, D), dev = q.shape, q.device
    _on(state, "state", dev)
    if state.dtype != F32 or state.shape != (N, H, D, D) or not state.is_contiguous() or state.requires_grad:
        raise ValueError(f"state must be a contiguous float32 tensor of ({N}, {H}, {D}, {D}) without gradient, got "
                         f"{tuple(state.shape)}, {state.dtype}")
    if _route(q, "decay_attention_step", function=False) is None:
        with torch.no_grad():
            return ref.decay_attention_step(q, k, v, rate, state, dt, scale)
    q, k, v = _heads(q), _heads(k), _heads(v)
    y = torch.empty(N, H, D, dtype=q.dtype, device=dev)
    with on_device(dev):
        call("atl_decay_attn_step", *_strides(q), *_strides(k), *_strides(v), _CODE[q.dtype], N, H, D, _at(rate), _at(dt), scale,
             _at(state), _at(y), raw_stream(dev))
    torch.autograd.graph.increment_version(state)          # written by address: whoever saved it has to know
    return y
