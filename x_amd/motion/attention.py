"""A network of linear attention from an event packet to trajectory coefficients (no counterpart in the reference's package).

As :class:`x_amd.motion.EventRecurrence`, with layers that remember by content and place: every event's query meets the keys of
the events before it, turned by their rows and columns on the sensor, so a product depends on how far apart two events
are, and forgets them head by head with the time between.  A layer's state is a matrix per head whose size does not grow
with the events, so streams are followed event by event or window by window as there.

    net = EventAttention(480, 640).cuda()
    motion = net.motion(ev, p=0.1, seed=step)             # ev: EventPacket; dropout by (seed, layer)
    loss = AnchoredExact(h=1.0, tau=0.2)(ev, motion)["loss"]
"""
from __future__ import annotations

import math

import torch
from torch import nn

from ..core.events import EventPacket
from ..ops import decay_attention, decay_attention_step, embed_tokens, head_norm_rotary, residual_rms_norm
from ..ops.attention import MAX_ATTENTION_WIDTH
from .recurrent import EventRecurrence


class EventAttention(EventRecurrence):
    """``heads`` heads share the ``dim`` channels; head j forgets with 2^-j per time constant ``tau``.  The other sizes and
    the methods are :class:`EventRecurrence`'s; states are (B, heads, dim / heads, dim / heads) float32 a layer."""

    def __init__(self, height: int, width: int, K: int = 1, dim: int = 64, layers: int = 2, heads: int = 2, cell: int = 8,
                 grid: tuple[int, int] = (6, 8), tau: float = 1 / 16, dtype: torch.dtype = torch.bfloat16):
        super().__init__(height, width, K, dim, layers, cell, grid, tau, dtype)
        if heads < 1 or dim % heads or not 4 <= dim // heads <= MAX_ATTENTION_WIDTH:
            raise ValueError(f"heads must share {dim} channels evenly, 4 to {MAX_ATTENTION_WIDTH} each, got {heads} heads")
        self.heads, D = heads, dim // heads
        # (nothing reads the last layer's outputs, so it has no queries of its own)
        self.into = nn.ParameterList(nn.Parameter(torch.randn((3 if k < layers - 1 else 2) * dim, dim) / math.sqrt(dim))
                                     for k in range(layers))
        self.q_norm = nn.ParameterList(nn.Parameter(torch.ones(D)) for _ in range(layers - 1))
        self.k_norm = nn.ParameterList(nn.Parameter(torch.ones(D)) for _ in range(layers))
        self.read = nn.ParameterList(nn.Parameter(torch.randn(heads, 1, D) / math.sqrt(D)) for _ in range(layers))
        self.read_norm = nn.ParameterList(nn.Parameter(torch.ones(dim)) for _ in range(layers))
        # half of the pairs turn with the row, half with the column: wave lengths from three pixels to a thousand
        self.sections = (D // 4, D // 2 - D // 4)
        self.register_buffer("freqs", torch.cat([2.0 * 300.0 ** -(torch.arange(m) / m) for m in self.sections]), persistent=False)
        self.register_buffer("rate", 2.0 ** -torch.arange(heads), persistent=False)

    def positions(self, xy: torch.Tensor, ids: torch.Tensor) -> torch.Tensor:
        """Rows and columns (n, 2) of events, zero where an event is no token."""
        return torch.where((ids >= 0)[:, None], xy.flip(1), 0.0)

    def _heads(self, y, k, pos):
        """Queries, keys and values (n, heads, D) of a layer's projection, the first two normed and turned."""
        *q, key, v = y.view(len(y), y.shape[1] // self.dim, self.heads, self.dim // self.heads).unbind(1)
        q, q_norm = (q[0], self.q_norm[k]) if q else (key, self.k_norm[k])
        return *head_norm_rotary(q, key, q_norm, self.k_norm[k], pos, self.freqs, self.sections), v

    def states(self, ev: EventPacket, h0=None, p: float = 0.0, seed: int = 0, since=None) -> list:
        if since is not None and h0 is None:
            raise ValueError("since says how old the states in h0 are, and h0 is None")
        start, dt, ids = ev.offsets, self.gaps(ev, since), self.tokens(ev.xy, ev.p)
        pos = self.positions(ev.xy, ids)
        s = embed_tokens(ids, self.table, scale=math.sqrt(self.dim), dtype=self.dtype)
        x, last = None, []
        for k, (w, into) in enumerate(zip(self.norm, self.into)):
            if x is None:
                y, s = residual_rms_norm(s, None, w)
            else:
                y, s = residual_rms_norm(x, s, w, p=p, seed=seed, offset=k)
            q, key, v = self._heads(nn.functional.linear(y, into.to(y.dtype)), k, pos)
            h, end = decay_attention(q, key, v, self.rate, start, dt=dt, h0=None if h0 is None else h0[k])
            last.append(end)
            if k < len(self.out):
                x = nn.functional.linear(h.flatten(1), self.out[k].to(h.dtype))
        return last

    def coefficients(self, states: list) -> torch.Tensor:
        """(B, 2K, H, W) coefficients as :class:`EventRecurrence`'s, from what a learned query of every head reads of the
        states, normed."""
        read = [residual_rms_norm((q @ S).flatten(1), None, w)[0] for q, S, w in zip(self.read, states, self.read_norm)]
        return super().coefficients(read)

    def fresh_states(self, streams: int) -> list:
        D = self.dim // self.heads
        return [torch.zeros(streams, self.heads, D, D, device=self.table.device) for _ in self.norm]

    @torch.no_grad()
    def step(self, xy: torch.Tensor, p: torch.Tensor, dt: torch.Tensor, states: list, fp8=None) -> list:
        """One event of each of n streams, as :meth:`EventRecurrence.step`."""
        ids = self.tokens(xy, p)
        pos = self.positions(xy, ids)
        s = embed_tokens(ids, self.table, scale=math.sqrt(self.dim), dtype=self.dtype)
        x = None
        for k, (w, into) in enumerate(zip(self.norm, self.into)):
            y, s = self._projected(*((s, None) if x is None else (x, s)), w, into, None if fp8 is None else fp8[k])
            h = decay_attention_step(*self._heads(y, k, pos), self.rate, states[k], dt=dt)
            if k < len(self.out):
                x = nn.functional.linear(h.flatten(1), self.out[k].to(h.dtype))
        return states
