"""Operators of a recurrent model over event tokens, on the HIP library (no counterpart in the reference's package).

* :func:`embed_tokens`           table rows of token ids, scaled; grad to the table, summed by sorted tokens
* :func:`residual_rms_norm`      residual addition with dropout and RMS norm; grads to x, residual and weight
* :func:`residual_rms_norm_fp8`  the same without dropout, the norm in 8 bits (e4m3) with a scale per row
* :func:`gated_scan`             gated linear recurrence over ragged windows of tokens; grads to x, gate and h0
* :func:`gated_scan_step`        its single-token form for streams, the state updated in place

Tokens are rows of D channels in single, bfloat16 or half precision; sums and states are kept in single precision and
every output is rounded once.  Rows may lie apart (a slice of a wider projection) as long as a row is contiguous; other
layouts are copied first.  Device tensors run on the HIP kernels, CPU tensors on :mod:`x_amd.ops.reference`.
"""
from __future__ import annotations

import sys

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import reference as ref
from ._ext import F32, I64, call, load_library, on_device, raw_stream

_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_NORM_WIDTH = 8192
MAX_ROW_STRIDE = 65536
_U64 = 2 ** 64 - 1


def _at(t: torch.Tensor | None) -> int:
    """A tensor's address as the entry points take it (an integer converts faster than a pointer object)."""
    return 0 if t is None else t.data_ptr()


def _float_type(t, name: str) -> int:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    code = _CODE.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


def _on(t, name: str, dev):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.device != dev:
        raise ValueError(f"{name} must be on {dev}, got {t.device}")


def _plain(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """``t`` contiguous in ``dtype``: itself where it is (told in less time than two conversions to nothing)."""
    return t if t.dtype == dtype and t.is_contiguous() else t.to(dtype).contiguous()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as (rows, D) with contiguous rows: a view where its strides allow it (rows less than MAX_ROW_STRIDE elements
    apart), else a copy."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.stride(0) > MAX_ROW_STRIDE and t.shape[0] < 2:
        t = t.reshape(-1).view(t.shape)                # a single row's stride says nothing
    return t if (t.stride(1) == 1 or t.shape[1] == 1) and t.stride(0) <= MAX_ROW_STRIDE else t.contiguous()


def _grads_wanted(*ts) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


# Looked up once: every call asks them.
_compiling, _tracing, _modes = torch.compiler.is_dynamo_compiling, torch._C._get_tracing_state, torch._C._len_torch_dispatch_stack
_key_set, _PRE_DISPATCH = torch._C._dispatch_tls_is_dispatch_key_included, torch._C.DispatchKey.PreDispatch


def _route(t: torch.Tensor, what: str, function: bool = True) -> bool | None:
    """None where the operator runs as torch operations (CPU tensors), else whether the kernels have to be called through
    the operator's autograd function whether a gradient is wanted or not: at a forward-mode level, where the function
    refuses tangents, and under torch.jit.trace, which keeps it as a call.  (Past the function either would take the
    output for memory that nothing was computed into.)  Raises where a recording could not hold the call: operation by
    operation (make_fx; the kernels are none), or by torch.jit.trace without an autograd function.  torch.compile leaves
    the calls outside of its graphs."""
    if not t.is_cuda:
        return None
    if _compiling():
        return False
    if _modes() or _key_set(_PRE_DISPATCH):
        proxies = sys.modules.get("torch.fx.experimental.proxy_tensor")
        if proxies is not None and proxies.get_proxy_mode() is not None:
            raise RuntimeError(f"{what} cannot be recorded operation by operation: call it outside of the recorded program")
    if _tracing() is not None:
        if not function:
            raise RuntimeError(f"{what} cannot be recorded: it has no gradient and no autograd function to keep")
        return True
    return forward_ad._current_level >= 0


def _ws(nbytes: int, dev, what: str) -> torch.Tensor:
    if nbytes < 0:
        raise ValueError(f"{what}: sizes not supported")
    return torch.empty(max(nbytes, 1), dtype=torch.uint8, device=dev)


# ------------------------------------------------------------------------------------------- embedding
def _embed_fwd(ids, table, scale, dtype):
    N, (V, D), dev = ids.numel(), table.shape, table.device
    out = torch.empty(*ids.shape, D, dtype=dtype, device=dev)
    with on_device(dev):
        call("atl_embed_fwd", _at(ids), int(ids.dtype == I64), N, _at(table), table.stride(0), _CODE[table.dtype], V, D,
             scale, _at(out), _CODE[dtype], raw_stream(dev))
    return out


class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale, dtype):
        ctx.save_for_backward(ids)
        ctx.meta = (table.shape, table.dtype, scale)
        return _embed_fwd(ids, table, scale, dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        (ids,) = ctx.saved_tensors
        (V, D), ttype, scale = ctx.meta
        g = _rows(g)
        N = ids.numel()
        gt = torch.empty(V, D, dtype=ttype, device=g.device)
        nbytes = int(load_library().atl_embed_bwd_ws_bytes(N, V, D))
        ws = _ws(nbytes, g.device, "embed_tokens")
        with on_device(g.device):
            call("atl_embed_bwd", _at(ids), int(ids.dtype == I64), N, _at(g), g.stride(0), _CODE[g.dtype], V, D, scale,
                 _at(gt), _CODE[ttype], _at(ws), nbytes, raw_stream(g.device))
        return None, gt, None, None


def embed_tokens(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0, dtype: torch.dtype | None = None):
    """(\\*ids.shape, D) rows ``scale * table[ids]`` of a (V, D) table, in ``dtype`` (the table's if None).  An id outside
    [0, V) is no token, as an event outside the image is no vote: zeros, and no gradient.  The table's gradient adds
    the rows of one id in token order (the tokens are sorted by id, no atomic adds): equal calls give equal bits."""
    _float_type(table, "table")
    _on(ids, "ids", table.device)
    if table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1:
        raise ValueError(f"table must be (V, D), got {tuple(table.shape)}")
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"ids must be int64 or int32, got {ids.dtype}")
    dtype = table.dtype if dtype is None else dtype
    if dtype not in _CODE:
        raise TypeError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
    scale = float(scale)
    through = _route(table, "embed_tokens")
    if through is None:
        return ref.embed_tokens(ids, table, scale, dtype)
    ids, rows = ids.contiguous(), _rows(table)
    if through or _grads_wanted(table):
        return _Embed.apply(ids, rows, scale, dtype)
    return _embed_fwd(ids, rows, scale, dtype)


# ------------------------------------------------------------------------------------------- residual norm
def _norm_fwd(x, res, w, shape, eps, p, seed, offset, fp8=False):
    """(y, s, scale) in the given shape for rows x (N, D) and res (N, D) or None; s None where it would be x itself."""
    N, D = x.shape
    dev, rtype = x.device, (x if res is None else res).dtype
    y = torch.empty(shape, dtype=torch.float8_e4m3fn if fp8 else x.dtype, device=dev)
    s = None if res is None and p == 0 else torch.empty(shape, dtype=rtype, device=dev)
    scale = torch.empty(*shape[:-1], 1, dtype=F32, device=dev) if fp8 else None
    with on_device(dev):
        call("atl_rms_norm_fwd", _at(x), x.stride(0), _CODE[x.dtype], _at(res), 0 if res is None else res.stride(0),
             _CODE[rtype], _at(w), N, D, eps, p, seed, offset, _at(y), _at(s), _at(scale), raw_stream(dev))
    return y, s, scale


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, res, w, eps, p, seed, offset):
        rx, rr = _rows(x), None if res is None else _rows(res)
        y, s, _ = _norm_fwd(rx, rr, w, x.shape, eps, p, seed, offset)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(rx if s is None else s, w)
        ctx.meta = (x.shape, x.dtype, eps, p, seed, offset)
        return y, s

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gs=None):
        s, w = ctx.saved_tensors
        shape, xtype, eps, p, seed, offset = ctx.meta
        want_x, want_r, want_w = ctx.needs_input_grad[:3]
        if gy is None and gs is None:
            return (None,) * 7
        want_w = want_w and gy is not None                 # the weight has no part in the sum
        s = _rows(s)
        N, D = s.shape
        dev = s.device
        gy, gs = None if gy is None else _rows(gy), None if gs is None else _rows(gs)
        same = p == 0 and xtype == s.dtype                 # then both gradients are one tensor
        gr = torch.empty(shape, dtype=s.dtype, device=dev) if want_r or (same and want_x) else None
        gx = torch.empty(shape, dtype=xtype, device=dev) if want_x and not same else None
        gw = torch.empty(D, dtype=F32, device=dev) if want_w else None
        nbytes = int(load_library().atl_rms_norm_bwd_ws_bytes(N, D)) if want_w else 0
        ws = _ws(nbytes, dev, "residual_rms_norm") if want_w else None
        with on_device(dev):
            call("atl_rms_norm_bwd", _at(s), s.stride(0), _CODE[s.dtype], _at(w), _at(gy),
                 0 if gy is None else gy.stride(0), _CODE[xtype], _at(gs), 0 if gs is None else gs.stride(0), N, D, eps,
                 p, seed, offset, _at(gx), _at(gr), _at(gw), _at(ws), nbytes, raw_stream(s.device))
        gx = gr if same else gx
        return gx if want_x else None, gr if want_r else None, gw, None, None, None, None


def _norm_args(x, residual, weight, eps, p=0.0):
    _float_type(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be (..., D), got {tuple(x.shape)}")
    D = x.shape[-1]
    if D > MAX_NORM_WIDTH:
        raise ValueError(f"rows of up to {MAX_NORM_WIDTH} channels, got {D}")
    _on(weight, "weight", x.device)
    _float_type(weight, "weight")
    if weight.shape != (D,):
        raise ValueError(f"weight must be ({D},), got {tuple(weight.shape)}")
    if residual is not None:
        _on(residual, "residual", x.device)
        if residual.dtype not in (x.dtype, F32):
            raise TypeError(f"residual must be {x.dtype} or float32, got {residual.dtype}")
        if residual.shape != x.shape:
            raise ValueError(f"residual must be {tuple(x.shape)}, got {tuple(residual.shape)}")
    eps, p = float(eps), float(p)
    if not 0 <= eps < 1e30:
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    if not (0 <= p < 1 and round(p * 65536) < 65536):
        raise ValueError(f"p must be in [0, 1 - 2^-16], got {p}")
    return eps, round(p * 65536) / 65536


def residual_rms_norm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float = 1e-6,
                      p: float = 0.0, seed: int = 0, offset: int = 0):
    """(y, s): the sum s = residual + dropout(x) and its root-mean-square norm y = s / sqrt(mean(s^2) + eps) * weight
    over the last axis (of up to 8192 channels).  s has the residual's type (x's or float32) and is the next residual;
    y has x's, and is the norm of s as it is returned.  Without a residual s is dropout(x) (x itself where p is 0).

    Dropout zeroes an element with probability p (to the nearest 1 / 65536) and scales the others by 1 / (1 - p).  Its
    bits come from Philox4x32-10 at counter (row, 2^31 + column // 8, ``offset``) under the key ``seed``, so equal
    (seed, offset) give equal masks whatever the launch, the backward draws them again, and no mask is stored."""
    eps, p = _norm_args(x, residual, weight, eps, p)
    seed, offset = int(seed) & _U64, int(offset) & _U64
    through = _route(x, "residual_rms_norm")
    if through is None:
        return ref.residual_rms_norm(x, residual, weight, eps, p, seed, offset)
    w = _plain(weight, F32)
    if through or _grads_wanted(x, residual, w):
        y, s = _Norm.apply(x, residual, w, eps, p, seed, offset)
    else:
        y, s, _ = _norm_fwd(_rows(x), None if residual is None else _rows(residual), w, x.shape, eps, p, seed, offset)
    return y, x if s is None else s


def residual_rms_norm_fp8(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float = 1e-6):
    """(q, scale, s): :func:`residual_rms_norm` without dropout, its norm in e4m3 with a scale per row: y = q * scale,
    scale (..., 1) = max(max |y|, 1e-30) / 448, q = 448 y / max |y| rounded to nearest.  For inference (no gradient): q
    and scale are what a row-scaled 8-bit product takes."""
    eps, _ = _norm_args(x, residual, weight, eps)
    if _route(x, "residual_rms_norm_fp8", function=False) is None:
        with torch.no_grad():
            return ref.residual_rms_norm_fp8(x, residual, weight, eps)
    y, s, scale = _norm_fwd(_rows(x), None if residual is None else _rows(residual), _plain(weight.detach(), F32),
                            x.shape, eps, 0.0, 0, 0, fp8=True)
    return y, scale, x.detach() if s is None else s


# ------------------------------------------------------------------------------------------- recurrence
def _scan_fwd(x, gate, start, dt, h0, save):
    N, D = x.shape
    B, dev = start.numel() - 1, x.device
    lib = load_library()
    y = torch.empty(N, D, dtype=x.dtype, device=dev)
    last = torch.empty(B, D, dtype=F32, device=dev)
    nbytes = int(lib.atl_gated_scan_ws_bytes(N, D, _CODE[x.dtype]))
    ws = _ws(nbytes, dev, "gated_scan")
    states = torch.empty(int(lib.atl_gated_scan_groups(N)), D, dtype=F32, device=dev) if save else None
    with on_device(dev):
        call("atl_gated_scan_fwd", _at(x), x.stride(0), _at(gate), gate.stride(0), _CODE[x.dtype], N, D, _at(start), B,
             _at(dt), _at(h0), _at(y), _at(last), _at(states), _at(ws), nbytes, raw_stream(x.device))
    return y, last, states


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, start, dt, h0):
        y, last, states = _scan_fwd(x, gate, start, dt, h0, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, gate, start, dt, h0, states)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, glast):
        x, gate, start, dt, h0, states = ctx.saved_tensors
        if gy is None and glast is None:
            return (None,) * 5
        N, D = x.shape
        B, dev = start.numel() - 1, x.device
        gy = None if gy is None else _rows(gy)
        glast = None if glast is None else glast.contiguous()
        gx = torch.empty(N, D, dtype=x.dtype, device=dev)
        gg = torch.empty(N, D, dtype=x.dtype, device=dev)
        gh0 = torch.empty(B, D, dtype=F32, device=dev) if ctx.needs_input_grad[4] else None
        nbytes = int(load_library().atl_gated_scan_ws_bytes(N, D, _CODE[x.dtype]))
        ws = _ws(nbytes, dev, "gated_scan")
        with on_device(dev):
            call("atl_gated_scan_bwd", _at(x), x.stride(0), _at(gate), gate.stride(0), _CODE[x.dtype], N, D, _at(start),
                 B, _at(dt), _at(h0), _at(states), _at(gy), 0 if gy is None else gy.stride(0), _at(glast), _at(gx),
                 _at(gg), _at(gh0), _at(ws), nbytes, raw_stream(x.device))
        return gx, gg, None, None, gh0


def _scan_args(x, gate, dt):
    _float_type(x, "x")
    dev, shape = x.device, x.shape
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError(f"x must be (N, D), got {tuple(shape)}")
    _on(gate, "gate", dev)
    if gate.dtype != x.dtype or gate.shape != shape:
        raise ValueError(f"gate must be like x ({tuple(shape)}, {x.dtype}), got {tuple(gate.shape)}, {gate.dtype}")
    if dt is None:
        return None
    _on(dt, "dt", dev)
    if dt.shape != shape[:1]:
        raise ValueError(f"dt must be ({shape[0]},), got {tuple(dt.shape)}")
    if dt.requires_grad:
        raise ValueError("no gradient flows to dt: detach it")
    return _plain(dt, F32)


def gated_scan(x: torch.Tensor, gate: torch.Tensor, start: torch.Tensor, dt: torch.Tensor | None = None,
               h0: torch.Tensor | None = None):
    """(y, last): the gated linear recurrence

        h_i = exp(-dt_i softplus(gate_i)) h_{i-1} + sigmoid(gate_i) x_i

    of every channel over the tokens (N, D) of each window, from h0 (B, D) or zero.  y (N, D) holds every state in x's
    type, last (B, D) each window's last one in float32 (an empty window's: h0 or zero), to go on from.

    ``start`` (B + 1) holds the windows' first tokens and N (``EventPacket.offsets``); it must ascend from 0 to N, which
    is not checked on the device.  ``dt`` (N,) is the gap to the token before, in units of a time constant (the first
    token's: since h0); None stands for ones: then h is a running average.  A negative gap (events out of order) grows the
    state as the formula has it.  No gradient flows to dt."""
    dt = _scan_args(x, gate, dt)
    N, D = x.shape
    _on(start, "start", x.device)
    if start.dim() != 1 or start.numel() < 1 or start.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"start must be (B + 1,) of int64 or int32, got {tuple(start.shape)}, {start.dtype}")
    B = start.numel() - 1
    if B == 0 and N > 0:
        raise ValueError(f"{N} tokens but no window")
    if h0 is not None:
        _on(h0, "h0", x.device)
        if h0.shape != (B, D):
            raise ValueError(f"h0 must be ({B}, {D}), got {tuple(h0.shape)}")
        h0 = _plain(h0, F32)
    start = _plain(start, I64)
    through = _route(x, "gated_scan")
    if through is None:
        return ref.gated_scan(x, gate, start, dt, h0)
    rx, rg = _rows(x), _rows(gate)
    if through or _grads_wanted(x, gate, h0):
        return _Scan.apply(rx, rg, start, dt, h0)
    return _scan_fwd(rx, rg, start, dt, h0, False)[:2]


def gated_scan_step(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor, dt: torch.Tensor | None = None):
    """One token of each of N streams: ``state`` (N, D) float32 becomes exp(-dt softplus(gate)) state + sigmoid(gate) x in
    place; returns it in x's type.  For inference (no gradient): a backward that needs the state as it was raises."""
    dt = _scan_args(x, gate, dt)
    dev, shape = x.device, x.shape
    _on(state, "state", dev)
    if state.dtype != F32 or state.shape != shape or not state.is_contiguous() or state.requires_grad:
        raise ValueError(f"state must be a contiguous float32 tensor of {tuple(shape)} without gradient, got "
                         f"{tuple(state.shape)}, {state.dtype}")
    if _route(x, "gated_scan_step", function=False) is None:
        with torch.no_grad():
            return ref.gated_scan_step(x, gate, state, dt)
    x, gate = _rows(x), _rows(gate)
    N, D = shape
    y = torch.empty(shape, dtype=x.dtype, device=dev)
    with on_device(dev):
        call("atl_gated_scan_step", _at(x), x.stride(0), _at(gate), gate.stride(0), _CODE[x.dtype], N, D, _at(dt),
             _at(state), _at(y), raw_stream(dev))
    torch.autograd.graph.increment_version(state)          # written by address: whoever saved it has to know
    return y
