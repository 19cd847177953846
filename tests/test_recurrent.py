"""EventRecurrence: the sequence operators together, from an event packet to a motion that the anchored score trains, and
event by event."""
import pytest
import torch

from x_amd import synth
from x_amd.core import EventPacket
from x_amd.motion import EventRecurrence, PixelTrajectories
from x_amd.objectives import AnchoredExact

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


def _net(dev, dtype, dim=32, **kw):
    torch.manual_seed(0)
    net = EventRecurrence(40, 48, dim=dim, layers=2, cell=4, grid=(3, 4), dtype=dtype, **kw)
    with torch.no_grad():
        net.head.normal_(std=0.02)
    return net.to(dev)


def _packet(dev, n=400, B=2, seed=0):
    return EventPacket.from_window(synth.small_window(seed=seed, n=n, B=B), dev)


def test_tokens_and_gaps():
    net = EventRecurrence(40, 48, cell=4, dtype=torch.float32)
    xy = torch.tensor([[0.0, 0.0], [3.6, 0.0], [47.4, 39.4], [47.6, 0.0], [-0.6, 0.0], [5.0, 9.0]])
    ids = net.tokens(xy, torch.tensor([1.0, -1.0, 1.0, 1.0, 1.0, -1.0]))
    assert ids.tolist() == [1, 2, net.vocab - 1, -1, -1, (2 * 12 + 1) * 2]
    ev = EventPacket(torch.zeros(5, 2), torch.tensor([0.1, 0.3, 0.3, 0.25, 0.5]), torch.ones(5),
                     torch.tensor([0, 0, 0, 2, 2]), 3, 40, 48)
    assert torch.allclose(net.gaps(ev) * net.tau, torch.tensor([0.1, 0.2, 0.0, 0.25, 0.25]))
    assert net.gaps(ev.select(torch.zeros(5, dtype=torch.bool))).numel() == 0


@pytest.mark.parametrize("dev", DEVICES)
def test_windows_event_by_event(dev):
    """Following a window with step() ends in the states that the scan has, and handing states on splits a window."""
    net, ev = _net(dev, torch.float32), _packet(dev, n=60, B=2)
    want = net.states(ev)
    dt, start = net.gaps(ev), ev.offsets
    got = net.fresh_states(2)
    for k in range(60):
        at = start[:-1] + k
        got = net.step(ev.xy[at], ev.p[at], dt[at], got)
    for a, b in zip(got, want):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-5)
    one = _packet(dev, n=60, B=1)
    full = net.states(one)
    first = net.states(one.select(torch.arange(25, device=one.device)))
    rest = one.select(torch.arange(25, 60, device=one.device))
    moved = rest._replace(t=rest.t - one.t[24])
    second = net.states(moved, h0=first)
    for a, b in zip(second, full):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("dev", DEVICES)
def test_the_anchored_score_trains_every_parameter(dev):
    ev = _packet(dev, n=600, B=2, seed=3)
    net = _net(dev, torch.float32 if dev == "cpu" else torch.bfloat16)
    motion = net.motion(ev, p=0.1, seed=1)
    assert isinstance(motion, PixelTrajectories)
    AnchoredExact(h=1.5, tau=0.3, n_anchors=None, seed=0)(ev, motion)["loss"].backward()
    for name, q in net.named_parameters():
        assert q.grad is not None and torch.isfinite(q.grad).all() and q.grad.any(), name


@pytest.mark.parametrize("dev", DEVICES)
def test_training_fits_given_motions(dev):
    """Adam on the squared error to a translation per window, with dropout, takes most of the error away."""
    ev = _packet(dev, n=300, B=3, seed=4)
    net = _net(dev, torch.float32 if dev == "cpu" else torch.bfloat16)
    want = torch.tensor([[2.0, -1.0], [-1.5, 0.5], [0.5, 2.5]], device=dev)[:, :, None, None]
    opt = torch.optim.Adam(net.parameters(), lr=3e-3)
    losses = []
    for step in range(40):
        loss = (net.coefficients(net.states(ev, p=0.1, seed=step)) - want).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    assert losses[-1] < 0.3 * losses[0], losses


@pytest.mark.gpu
def test_gpu_states_and_gradients_are_the_cpu_ones():
    net, ev = _net("cpu", torch.float32), _packet("cpu", n=500, B=3)
    gen = torch.Generator().manual_seed(0)
    weights = [torch.randn(3, net.dim, generator=gen) for _ in net.norm]
    params = [net.table, *net.norm, *net.into, *net.out]

    def run(dev):
        states = net.to(dev).states(ev.to(dev), p=0.2, seed=5)
        loss = sum((a * w.to(dev)).sum() for a, w in zip(states, weights))
        return [t.cpu() for t in states], [g.cpu() for g in torch.autograd.grad(loss, params)]

    want, grads = run("cpu")
    got, ggrads = run("cuda:0")
    for a, b in zip(got + ggrads, want + grads):
        assert (a - b).norm() <= 1e-4 * b.norm()


@pytest.mark.gpu
def test_streams_in_8_bits():
    """e4m3 keeps three bits of mantissa: the projections of 64 terms are off by some percent of their size."""
    net = _net("cuda:0", torch.bfloat16, dim=64)
    fp8 = net.fp8_weights()
    gen = torch.Generator(device="cuda:0").manual_seed(0)
    a, b = net.fresh_states(16), net.fresh_states(16)
    for _ in range(20):
        xy = torch.rand(16, 2, device="cuda:0", generator=gen) * 39
        p, dt = torch.ones(16, device="cuda:0"), torch.rand(16, device="cuda:0", generator=gen)
        net.step(xy, p, dt, a)
        net.step(xy, p, dt, b, fp8=fp8)
    for x, y in zip(a, b):
        assert (x - y).norm() < 0.15 * x.norm()


def test_refuses_bad_sizes():
    for kw in (dict(dim=0), dict(layers=0), dict(tau=0.0), dict(grid=(0, 4))):
        with pytest.raises(ValueError):
            EventRecurrence(40, 48, **kw)
    with pytest.raises(ValueError):
        EventRecurrence(40, 48, dim=40).fp8_weights()


def _two_windows(dev, B=3, seed=6):
    """Consecutive windows of B streams, each with times of its own in [0, 1], and idle time on both sides of the
    boundary; the last stream's middle window is empty.  Returns the three windows and all events as one scan's rows
    (xy, p, gaps in windows, start)."""
    gen = torch.Generator().manual_seed(seed)
    windows, events = [], [[] for _ in range(B)]
    for k, sizes in enumerate(([9, 7, 8], [6, 9, 0], [5, 4, 7])):
        parts = []
        for b in range(B):
            n = sizes[b]
            t = torch.sort(torch.rand(n, generator=gen)).values * 0.4 + 0.3
            xy = torch.rand(n, 2, generator=gen) * torch.tensor([47.0, 39.0])
            p = torch.where(torch.rand(n, generator=gen) < 0.5, 1.0, -1.0)
            parts.append((xy, t, p, torch.full((n,), b)))
            events[b].append((xy, t.double() + k, p))
        windows.append(EventPacket(*(torch.cat(v) for v in zip(*parts)), B, 40, 48).to(dev))
    rows = [[torch.cat(v) for v in zip(*e)] for e in events]
    gaps = torch.cat([torch.diff(t, prepend=torch.zeros(1, dtype=t.dtype)) for _, t, _ in rows]).float()
    start = torch.tensor([0, *torch.cumsum(torch.tensor([len(t) for _, t, _ in rows]), 0).tolist()])
    return windows, torch.cat([r[0] for r in rows]).to(dev), torch.cat([r[2] for r in rows]).to(dev), gaps.to(dev), start.to(dev)


@pytest.mark.parametrize("dev", DEVICES)
def test_streams_window_by_window(dev):
    """States handed on over windows, with the time since each stream's last event, are those of all events in one
    scan, event by event too: also over an empty window."""
    net = _net(dev, torch.float32, tau=0.5)
    windows, xy, p, gaps, start = _two_windows(dev)
    want = net.fresh_states(3)
    for k in range(int((start[1:] - start[:-1]).max())):
        on = (start[:-1] + k < start[1:]).nonzero()[:, 0]
        at = start[:-1][on] + k
        part = net.step(xy[at], p[at], gaps[at] / net.tau, [s[on] for s in want])
        for s, q in zip(want, part):
            s[on] = q
    h0 = since = None
    for ev in windows:
        h0, since = net.states(ev, h0=h0, since=since), net.idle(ev, since)
    for a, b in zip(h0, want):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-5)
    last = torch.stack([(1 - windows[2].t[windows[2].b == b][-1]) for b in range(3)])
    assert torch.allclose(since, last)
    # an event at 0.1 of the next window: 0.1 and the idle time after the last one
    late = EventPacket(torch.zeros(1, 2, device=dev), torch.full((1,), 0.1, device=dev), torch.ones(1, device=dev),
                       torch.ones(1, dtype=torch.int64, device=dev), 3, 40, 48)
    assert torch.allclose(net.gaps(late, since) * net.tau, since[1:2] + 0.1)
    assert torch.allclose(net.idle(late, since), torch.stack([since[0] + 1, 1 - late.t[0], since[2] + 1]))


@pytest.mark.parametrize("dev", DEVICES)
def test_time_since_reaches_the_motion(dev):
    net, ev = _net(dev, torch.float32), _packet(dev, n=100, B=2)
    h0 = [torch.ones(2, net.dim, device=dev) for _ in net.norm]
    since = torch.tensor([0.0, 30.0], device=dev)
    near = net.motion(ev, h0=h0).coeff_grid
    far = net.motion(ev, h0=h0, since=since).coeff_grid
    fresh = net.motion(ev).coeff_grid
    assert torch.equal(near[0], far[0]) and not torch.equal(near[1], far[1])
    assert torch.allclose(far[1], fresh[1], atol=1e-6)             # 480 time constants forget everything


def test_time_since_is_checked():
    net, ev = _net("cpu", torch.float32), _packet("cpu", n=20, B=2)
    h0 = net.fresh_states(2)
    for bad in (torch.zeros(3), torch.zeros(2, 1)):
        with pytest.raises(ValueError):
            net.states(ev, h0=h0, since=bad)
        with pytest.raises(ValueError):
            net.idle(ev, bad)
    with pytest.raises(ValueError):
        net.states(ev, since=torch.zeros(2))


@pytest.mark.parametrize("dev", DEVICES)
def test_positions_that_are_not_numbers_are_no_tokens(dev):
    net = _net(dev, torch.float32)
    bad = [float("nan"), float("inf"), -float("inf"), 1e30, -1e30]
    xy = torch.tensor([[v, 3.0] for v in bad] + [[3.0, v] for v in bad] + [[3.0, 3.0]], device=dev)
    ids = net.tokens(xy, torch.ones(11, device=dev))
    assert ids.tolist() == [-1] * 10 + [1]
