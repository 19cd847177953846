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
