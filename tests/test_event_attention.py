"""EventAttention: the attention operators together with the sequence operators, from an event packet to a motion that the
anchored score trains, window by window and event by event."""
import pytest
import torch

from x_amd import synth
from x_amd.core import EventPacket
from x_amd.motion import EventAttention, PixelTrajectories
from x_amd.objectives import AnchoredExact

DEVICES = ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)]


def _net(dev, dtype, dim=32, heads=2, **kw):
    torch.manual_seed(0)
    net = EventAttention(40, 48, dim=dim, heads=heads, layers=2, cell=4, grid=(3, 4), dtype=dtype, **kw)
    with torch.no_grad():
        net.head.normal_(std=0.02)
    return net.to(dev)


def _packet(dev, n=400, B=2, seed=0):
    return EventPacket.from_window(synth.small_window(seed=seed, n=n, B=B), dev)


@pytest.mark.parametrize("dev", DEVICES)
def test_windows_event_by_event(dev):
    """Following a window with step() ends in the states that the windows have, and handing states on splits a window."""
    net, ev = _net(dev, torch.float32), _packet(dev, n=60, B=2)
    want = net.states(ev)
    assert [tuple(w.shape) for w in want] == [(2, 2, 16, 16)] * 2
    dt, start = net.gaps(ev), ev.offsets
    got = net.fresh_states(2)
    for k in range(60):
        at = start[:-1] + k
        got = net.step(ev.xy[at], ev.p[at], dt[at], got)
    for a, b in zip(got, want):
        assert torch.allclose(a, b, rtol=1e-3, atol=1e-4)
    one = _packet(dev, n=60, B=1)
    full = net.states(one)
    first = one.select(torch.arange(25, device=one.device))
    rest = one.select(torch.arange(25, 60, device=one.device))
    second = net.states(rest._replace(t=rest.t - one.t[24]), h0=net.states(first))
    for a, b in zip(second, full):
        assert torch.allclose(a, b, rtol=1e-3, atol=1e-4)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("heads", [1, 4])
def test_the_anchored_score_trains_every_parameter(dev, heads):
    ev = _packet(dev, n=600, B=2, seed=3)
    net = _net(dev, torch.float32 if dev == "cpu" else torch.bfloat16, heads=heads)
    motion = net.motion(ev, p=0.1, seed=1)
    assert isinstance(motion, PixelTrajectories)
    AnchoredExact(h=1.5, tau=0.3, n_anchors=None, seed=0)(ev, motion)["loss"].backward()
    for name, q in net.named_parameters():
        assert q.grad is not None and torch.isfinite(q.grad).all() and q.grad.any(), name


@pytest.mark.gpu
def test_gpu_states_and_gradients_are_the_cpu_ones():
    net, ev = _net("cpu", torch.float32), _packet("cpu", n=500, B=3)
    gen = torch.Generator().manual_seed(0)
    weights = [torch.randn(3, 2, 16, 16, generator=gen) for _ in net.norm]
    params = [net.table, *net.norm, *net.into, *net.out, *net.k_norm, net.q_norm[0]]

    def run(dev):
        states = net.to(dev).states(ev.to(dev), p=0.2, seed=5)
        loss = sum((a * w.to(dev)).sum() for a, w in zip(states, weights))
        return [t.cpu() for t in states], [g.cpu() for g in torch.autograd.grad(loss, params)]

    want, grads = run("cpu")
    got, ggrads = run("cuda:0")
    for a, b in zip(got + ggrads, want + grads):
        assert (a - b).norm() <= 1e-4 * b.norm()


@pytest.mark.parametrize("dev", DEVICES)
def test_streams_window_by_window(dev):
    """A window cut in two, its states and the time since its last event handed on, ends in the states of the whole."""
    net = _net(dev, torch.float32)
    ev = _packet(dev, n=80, B=1)
    half = ev.t < 0.5
    one, two = ev.select(half), ev.select(~half)
    states = net.states(one)
    since = torch.clamp(0.5 - one.t[-1:], min=0)
    got = net.states(two._replace(t=two.t - 0.5), h0=states, since=since)
    for a, b in zip(got, net.states(ev)):
        assert torch.allclose(a, b, rtol=1e-3, atol=1e-4)
    with pytest.raises(ValueError, match="since"):
        net.states(ev, since=since)


@pytest.mark.parametrize("dev", DEVICES)
def test_positions_that_are_not_numbers_are_no_tokens(dev):
    """An event without a place neither asks nor is remembered: the states are those without it, its gap aside."""
    net, ev = _net(dev, torch.float32), _packet(dev, n=40, B=1)
    ev = ev._replace(t=torch.zeros_like(ev.t))
    want = net.states(ev.select(torch.arange(1, 40, device=ev.device)))
    xy = ev.xy.clone()
    xy[0] = float("nan")
    for a, b in zip(net.states(ev._replace(xy=xy)), want):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("dev", DEVICES)
def test_windows_without_events_and_no_streams(dev):
    """A packet without events leaves the states as they were (zeros without any), its windows' whole length goes by, no stream
    steps, and the packet's motion has gradients."""
    net = _net(dev, torch.float32)
    none = _packet(dev, n=60, B=2)
    none = none.select(torch.zeros(0, dtype=torch.int64, device=none.device))
    assert none.n == 0 and none.batch_size == 2
    assert all(tuple(s.shape) == (2, 2, 16, 16) and not s.any() for s in net.states(none))
    h0 = [torch.randn(2, 2, 16, 16, device=dev) for _ in net.norm]
    since = torch.rand(2, device=dev)
    for a, b in zip(net.states(none, h0=h0, p=0.1, since=since), h0):
        assert torch.equal(a, b)
    assert torch.equal(net.idle(none, since), since + 1)
    net.coefficients(net.states(none, h0=h0)).sum().backward()
    assert net.head.grad.isfinite().all() and net.read[0].grad.any()
    empty = torch.zeros(0, device=dev)
    states = net.step(torch.zeros(0, 2, device=dev), empty, empty, net.fresh_states(0))
    assert [tuple(s.shape) for s in states] == [(0, 2, 16, 16)] * 2


@pytest.mark.gpu
def test_streams_in_8_bits():
    """e4m3 keeps three bits of mantissa: the projections of 64 terms are off by some percent of their size, and so are products
    of two of them."""
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
        assert (x - y).norm() < 0.3 * x.norm()


def test_refuses_bad_sizes():
    for kw in (dict(heads=3), dict(heads=0), dict(dim=256, heads=1), dict(dim=4, heads=2)):
        with pytest.raises(ValueError, match="heads"):
            EventAttention(40, 48, **kw)
    with pytest.raises(ValueError, match="positive"):
        EventAttention(40, 0)
