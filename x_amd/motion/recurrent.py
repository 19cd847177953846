"""A recurrent network from an event packet to trajectory coefficients (no counterpart in the reference's package, whose
network is a convolutional one over voxel grids).

Every event is a token: its cell of the sensor and its polarity.  The tokens of a window run in time order through
layers of norm, projection and gated recurrence, whose decay follows the gaps between events, and the windows' last
states give the coefficients of a grid of trajectories, upsampled to the sensor: what
:class:`x_amd.motion.PixelTrajectories` takes and what the anchored scores train.

    net = EventRecurrence(480, 640).cuda()
    motion = net.motion(ev, p=0.1, seed=step)             # ev: EventPacket; dropout by (seed, layer)
    loss = AnchoredExact(h=1.0, tau=0.2)(ev, motion)["loss"]
    loss.backward()

A stream is followed event by event with :meth:`step`, or window by window by handing on the states and the time since
the last events, which the first gap of the next window adds to its own:

    states, since = net.states(ev, h0=states, since=since), net.idle(ev, since)      # (None, None before the first)
"""
from __future__ import annotations

import math

import torch
from torch import nn

from ..core.events import EventPacket
from ..ops import embed_tokens, gated_scan, gated_scan_step, residual_rms_norm, residual_rms_norm_fp8
from .trajectories import PixelTrajectories

FP8_MAX = 448.0


class EventRecurrence(nn.Module):
    """``cell`` x ``cell`` pixels make a token, ``grid`` trajectories (rows, columns) of K coefficients per axis are
    predicted for a window, ``tau`` is the time constant of the gaps (in windows), ``dtype`` the type of the tokens'
    rows (weights and states are float32)."""

    def __init__(self, height: int, width: int, K: int = 1, dim: int = 64, layers: int = 2, cell: int = 8,
                 grid: tuple[int, int] = (6, 8), tau: float = 1 / 16, dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        if min(height, width, K, dim, layers, cell, *grid) < 1 or not tau > 0:
            raise ValueError("sizes must be positive")
        self.H, self.W, self.K, self.dim, self.cell, self.grid = height, width, K, dim, cell, tuple(grid)
        self.tau, self.dtype = float(tau), dtype
        self.columns = -(-width // cell)
        self.vocab = 2 * self.columns * -(-height // cell)
        self.table = nn.Parameter(torch.randn(self.vocab, dim) / math.sqrt(dim))
        self.norm = nn.ParameterList(nn.Parameter(torch.ones(dim)) for _ in range(layers))
        self.into = nn.ParameterList(nn.Parameter(torch.randn(2 * dim, dim) / math.sqrt(dim)) for _ in range(layers))
        self.out = nn.ParameterList(nn.Parameter(torch.randn(dim, dim) / math.sqrt(dim)) for _ in range(layers - 1))
        self.head = nn.Parameter(torch.zeros(2 * K * grid[0] * grid[1], layers * dim))

    # ------------------------------------------------------------------------------------------ tokens
    def tokens(self, xy: torch.Tensor, p: torch.Tensor) -> torch.Tensor:
        """Ids of events: (row of cells, column of cells, polarity); -1 (no token) outside the sensor or where a position
        is not a number (told before the conversion to integers, which makes a zero of it on the device)."""
        col, row = torch.floor(xy[:, 0] + 0.5), torch.floor(xy[:, 1] + 0.5)
        inside = (col >= 0) & (col < self.W) & (row >= 0) & (row < self.H)
        col, row = torch.where(inside, col, 0.0).long(), torch.where(inside, row, 0.0).long()
        ids = (torch.div(row, self.cell, rounding_mode="floor") * self.columns +
               torch.div(col, self.cell, rounding_mode="floor")) * 2 + (p > 0).long()
        return torch.where(inside, ids, -1)

    def gaps(self, ev: EventPacket, since=None) -> torch.Tensor:
        """Time since the event before in units of tau; the first of a window since the window's start, and with ``since``
        (B,) since the stream's last event, so long (in windows) before the window's start."""
        before = torch.cat([ev.t.new_zeros(1), ev.t[:-1]])[:ev.n]
        fresh = torch.cat([ev.b.new_full((1,), -1), ev.b[:-1]])[:ev.n] != ev.b
        first = 0.0 if since is None else -self._since(ev, since)[ev.b]
        return (ev.t - torch.where(fresh, first, before)) / self.tau

    def idle(self, ev: EventPacket, since=None) -> torch.Tensor:
        """Time (B,) from every window's last event to the window's end, in windows: ``since`` for the windows after these.
        A window without events adds its whole length to its own ``since`` (None: zeros)."""
        since = ev.t.new_zeros(ev.batch_size) if since is None else self._since(ev, since)
        start = ev.offsets
        if ev.n == 0:
            return since + 1
        last = ev.t[(start[1:] - 1).clamp(min=0)]
        return torch.where(start[1:] > start[:-1], 1 - last, since + 1)

    @staticmethod
    def _since(ev: EventPacket, since: torch.Tensor) -> torch.Tensor:
        if since.shape != (ev.batch_size,):
            raise ValueError(f"since must be ({ev.batch_size},), got {tuple(since.shape)}")
        return since.to(ev.t.dtype)

    # ------------------------------------------------------------------------------------------ windows
    def states(self, ev: EventPacket, h0=None, p: float = 0.0, seed: int = 0, since=None) -> list:
        """The layers' last states (B, dim) of every window, from ``h0`` (as returned for the window before) or zero; p
        drops the layers' outputs (masks by (seed, layer)).  ``since`` (B,), with ``h0``: the time from each stream's last
        event to the window's start, in windows (:meth:`idle` of the window before); without it the windows start at
        those events."""
        if since is not None and h0 is None:
            raise ValueError("since says how old the states in h0 are, and h0 is None")
        start, dt = ev.offsets, self.gaps(ev, since)
        s = embed_tokens(self.tokens(ev.xy, ev.p), self.table, scale=math.sqrt(self.dim), dtype=self.dtype)
        x, last = None, []
        for k, (w, into) in enumerate(zip(self.norm, self.into)):
            if x is None:
                y, s = residual_rms_norm(s, None, w)
            else:
                y, s = residual_rms_norm(x, s, w, p=p, seed=seed, offset=k)
            x, gate = nn.functional.linear(y, into.to(y.dtype)).chunk(2, -1)
            h, end = gated_scan(x, gate, start, dt=dt, h0=None if h0 is None else h0[k])
            last.append(end)
            if k < len(self.out):
                x = nn.functional.linear(h, self.out[k].to(h.dtype))
        return last

    def coefficients(self, states: list) -> torch.Tensor:
        """(B, 2K, H, W) coefficients [y_1..y_K, x_1..x_K] in pixels of the windows' trajectories."""
        c = nn.functional.linear(torch.cat(states, 1), self.head).view(-1, 2 * self.K, *self.grid)
        return nn.functional.interpolate(c, size=(self.H, self.W), mode="bilinear", align_corners=False)

    def motion(self, ev: EventPacket, h0=None, p: float = 0.0, seed: int = 0, since=None, **kw) -> PixelTrajectories:
        """The windows' motion (:meth:`states`' arguments); keywords go to :class:`PixelTrajectories`."""
        return PixelTrajectories(self.coefficients(self.states(ev, h0, p, seed, since)), self.K, **kw)

    # ------------------------------------------------------------------------------------------ streams
    def fresh_states(self, streams: int) -> list:
        return [torch.zeros(streams, self.dim, device=self.table.device) for _ in self.norm]

    @torch.no_grad()
    def fp8_weights(self) -> list:
        """The input projections in e4m3 with a scale per output, for :meth:`step` (widths that are multiples of 16)."""
        if self.dim % 16:
            raise ValueError(f"8-bit products need a width that is a multiple of 16, got {self.dim}")
        out = []
        for w in self.into:
            top = w.abs().amax(1, keepdim=True).clamp(min=1e-30)
            out.append(((w * (FP8_MAX / top)).to(torch.float8_e4m3fn), (top / FP8_MAX).t().contiguous()))
        return out

    @staticmethod
    def _projected(x, residual, weight, into, fp8):
        """A layer's norm and input projection for one token of every stream, and the sum the norm is of."""
        if fp8 is None:
            y, s = residual_rms_norm(x, residual, weight)
            return nn.functional.linear(y, into.to(y.dtype)), s
        q, scale, s = residual_rms_norm_fp8(x, residual, weight)
        return torch._scaled_mm(q, fp8[0].t(), scale_a=scale, scale_b=fp8[1], out_dtype=torch.bfloat16).to(s.dtype), s

    @torch.no_grad()
    def step(self, xy: torch.Tensor, p: torch.Tensor, dt: torch.Tensor, states: list, fp8=None) -> list:
        """One event of each of n streams (xy (n, 2), p (n,), dt (n,) gaps in units of tau): the layers' states, updated
        in place.  ``fp8`` (:meth:`fp8_weights`): the input projections in 8 bits (on the GPU), for half the bytes of weights:
        up to widths of 1024 and 4096 streams the step is bound by the host, 305-310 us in 16 bits and 314-339 in 8."""
        s = embed_tokens(self.tokens(xy, p), self.table, scale=math.sqrt(self.dim), dtype=self.dtype)
        x = None
        for k, (w, into) in enumerate(zip(self.norm, self.into)):
            y, s = self._projected(*((s, None) if x is None else (x, s)), w, into, None if fp8 is None else fp8[k])
            x, gate = y.chunk(2, -1)
            h = gated_scan_step(x, gate, states[k], dt=dt)
            if k < len(self.out):
                x = nn.functional.linear(h, self.out[k].to(h.dtype))
        return states
