"""alphagpu_amd.learn: the operators together, as a learning step of the network that the engine plays with."""
import numpy as np
import pytest
import torch

import alphagpu_amd as ag
from alphagpu_amd import learn, mcts_gpu as M


def whole_number_network(game, H, T, seed):
    """Weights of -1, 0 and 1, two per row: with planes of 0 and 1 every activation is a small whole number, which 8 bits hold exactly."""
    r = np.random.default_rng(seed)

    def sparse(rows, cols, many=2):
        w = np.zeros((rows, cols), np.float32)
        for i in range(rows):
            w[i, r.choice(cols, many, replace=False)] = r.choice([-1, 1], many)
        return w

    net = ag.SNetwork2(game, H, T, W0=sparse(H, 2 * game.VS), Wres=np.stack([sparse(H, H, 1) for _ in range(T)]), Wp=sparse(game.A, H, 1), Wv=sparse(1, H, 1))
    net.bp[:] = r.integers(-2, 3, game.A)
    return net


def plain(net, planes):
    """The network in 64 bits (DenseNet.jl:294-304), weights as tensors [out, in]."""
    m = lambda w, o, i: torch.from_numpy(w.reshape(i, o).T.copy()).double().requires_grad_()  # noqa: E731
    H = net.H
    ws = [m(net.W0, H, net.inp), *[m(net.Wres[t * H * H:(t + 1) * H * H], H, H) for t in range(net.T)]]
    head, b = torch.cat([m(net.Wp, net.A, H).detach(), m(net.Wv, 1, H).detach()]).requires_grad_(), torch.from_numpy(np.concatenate([net.bp, net.bv])).double().requires_grad_()
    h = (planes.double() @ ws[0].t()).relu()
    for w in ws[1:]:
        h = (h + (h @ w.t()).relu()).relu()
    y = h @ head.t() + b
    return y[:, :net.A], y[:, net.A], [*ws, head, b]


@pytest.mark.gpu
@pytest.mark.parametrize("game,H,T", [(("gobang", 9, 5), 128, 3), (("connect4",), 64, 2), (("hex", 9), 512, 1)])
def test_forward_and_gradients_are_exact_where_8_bits_are(game, H, T):
    """Whole numbers that 8 bits hold, forward and backward: every weight's gradient equals that of the plain network in 64 bits."""
    g = ag.GameSpec(*game)
    net = whole_number_network(g, H, T, 1)
    r = torch.Generator().manual_seed(2)
    n = 37
    planes = (torch.rand(n, 2 * g.VS, generator=r) < 0.3).to(torch.int8)
    dl, dv = torch.randint(-1, 2, (n, g.A), generator=r).float() * (torch.rand(n, g.A, generator=r) < 0.05), torch.randint(-1, 2, (n,), generator=r).float()
    logits, v, ws = plain(net, planes)
    want = torch.autograd.grad([logits, v], ws, [dl.double(), dv.double()])
    le = learn.Learner(net)
    got_l, got_v = le.forward(planes.cuda())
    assert logits.abs().max() <= 16 and torch.equal(got_l.detach().cpu().double(), logits.detach()) and torch.equal(got_v.detach().cpu().double(), v.detach())
    got = torch.autograd.grad([got_l, got_v], le.params, [dl.cuda(), dv.cuda()])
    assert max(w.abs().max().item() for w in want) > 0
    for a, b in zip(got, want):
        assert torch.equal(a.cpu().double(), b)


@pytest.mark.gpu
def test_the_losses_gradient_is_that_of_their_mean():
    """gradients() against autograd of the written-out mean loss through the same layers: the cotangents differ by roundings of 32 bits (at most 16 half steps each:
    a softmax, a sigmoid and a few products), which the layers then hold in 8 bits, where a value next to a border moves by one step (2^-3 of it): equal up to
    that for single entries, and in the whole to 2^-3 of the largest entry."""
    g = ag.GameSpec("gobang", 9, 5)
    le = learn.Learner(ag.SNetwork2.random(g, 128, 2))
    r = torch.Generator().manual_seed(3)
    n = 64
    planes = (torch.rand(n, 2 * g.VS, generator=r) < 0.3).to(torch.int8).cuda()
    policy = torch.rand(n, g.A, generator=r).cuda()
    policy /= policy.sum(1, keepdim=True)
    value = torch.randint(0, 3, (n,), generator=r).cuda() / 2
    pl, vl, grads = le.gradients(planes, policy, value)
    logits, v = le.forward(planes)
    lp, vq = -(policy * torch.log_softmax(logits, 1)).sum(1), (torch.sigmoid(v) - value) ** 2
    want = torch.autograd.grad((lp + vq).mean(), le.params)
    assert (pl - lp).abs().max() < 81 * 2.0 ** -22 * (1 + lp.max()) and (vl - vq).abs().max() < 2.0 ** -20
    for a, b in zip(grads, want):
        assert ((a - b).abs() <= 2.0 ** -3 * b.abs().max()).all() and a.abs().max() > 0


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_from_self_play_to_the_engine_and_back(bits):
    """A generation's samples, a few steps, and the network back into the engine: the weights have moved, nothing is lost on the way, and a captured step
    replays as eager steps do."""
    g = ag.GameSpec("connect4")
    net = ag.SNetwork2.random(g, 64, 2, seed=5)
    buf = ag.PoolSample(g, 4096)
    with M.Engine(g, 64, 16, seed=3) as e:
        _, valid = M.mcts(net, 16, 64, buf, engine=e, seed=3)
        assert valid and buf.length_buffer() > 64
        le = learn.Learner(net, bits=bits)
        same = le.network()
        for k in ("W0", "Wres", "Wp", "bp", "Wv", "bv"):
            assert np.array_equal(getattr(same, k), getattr(net, k)), k
        losses = le.train(buf, steps=3, batch=256)
        assert losses.shape == (3, 2) and np.isfinite(losses).all()
        new = le.network()
        assert all(not np.array_equal(getattr(new, k), getattr(net, k)) and np.isfinite(getattr(new, k)).all() for k in ("W0", "Wres", "Wp", "bp", "Wv", "bv"))
        e.set_network(new)
        e.set_roots(None, L=64)
        e.search(16, cpuct=1.5)
        assert (e.root_visits().sum(1) == 15).all()
    with pytest.raises(ValueError, match="empty"):
        le.train(ag.PoolSample(g, 10), 1, 8)
    with pytest.raises(ValueError, match="planes"):
        le.forward(torch.zeros(3, 5, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_equals_eager_steps(bits):
    g = ag.GameSpec("gobang", 9, 5)
    net = ag.SNetwork2.random(g, 128, 2, seed=6)
    r = torch.Generator().manual_seed(4)
    n = 300
    data = []
    for _ in range(4):
        policy = torch.rand(n, g.A, generator=r)
        data.append(((torch.rand(n, 2 * g.VS, generator=r) < 0.3).to(torch.int8).cuda(), (policy / policy.sum(1, keepdim=True)).cuda(), (torch.randint(0, 3, (n,), generator=r) / 2).cuda()))
    eager, held = learn.Learner(net, bits=bits, capturable=True), learn.Learner(net, bits=bits, capturable=True)
    static = [t.clone() for t in data[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        held.step(*static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    alive = held.forward(data[0][0])                             # a graph over the same weights that lives through the capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        losses = held.step(*static)
    assert alive[0].requires_grad
    first = eager.step(*data[0])
    for d in (data[1], data[2], data[3], data[1]):
        for a, b in zip(static, d):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want = eager.step(*d)
        assert torch.equal(losses[0], want[0]) and torch.equal(losses[1], want[1])
        for a, b in zip(held.params, eager.params):
            assert torch.equal(a, b)
    assert held.optimiser.state()["step"] == eager.optimiser.state()["step"] == 5
