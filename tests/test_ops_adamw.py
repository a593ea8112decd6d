"""alphagpu_amd.ops.AdamW against a plain implementation in 64 bits, states in 32 and 8 bits, refusals and graphs."""
import ctypes as C
import math

import pytest
import torch

from alphagpu_amd import lib, ops

E32 = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
HYPER = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


def step64(p, g, m, v, t, lr, betas, eps, weight_decay):
    """One step in 64 bits -> (p, m, v) and the errors that 32 bits may add."""
    b1, b2 = betas
    p, g, m, v = (x.double() for x in (p, g, m, v))
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    den = (v1 / (1 - b2 ** t)).sqrt() + eps
    up = lr * (m1 / (1 - b1 ** t)) / den
    p1 = p * (1 - lr * weight_decay) - up
    tm = E32 * (2 * (b1 * m).abs() + 2 * ((1 - b1) * g).abs() + m1.abs()) + 2.0 ** -140         # constants and products rounded
    tv = E32 * (2 * b2 * v + 4 * (1 - b2) * g * g + v1) + 2.0 ** -140
    rel_v = torch.where(v1 > 0, tv / v1.clamp_min(1e-300), 0.0)
    tp = E32 * (3 * p.abs() + p1.abs()) + up.abs() * (rel_v + 12 * E32) + lr / (1 - b1 ** t) * tm / den
    return (p1, m1, v1), (tp, tm, tv)


def mix(h):
    h = (h * 0x9E3779B1) & 0xFFFFFFFF
    h ^= h >> 16
    h = (h * 0xB504F335) & 0xFFFFFFFF
    return h ^ (h >> 16)


def tensors(shapes, dtype, gdtype, seed):
    r = torch.Generator().manual_seed(seed)
    ps = [torch.randn(*s, generator=r).to(dtype) for s in shapes]
    gs = [(torch.randn(*s, generator=r) * torch.exp(2 * torch.randn(*s, generator=r))).to(gdtype) for s in shapes]
    return ps, gs


SETS = {"one": [(1,)], "odd": [(3,), (127,), (128,), (129,), (1,), (255,), (640, 3), (81, 128)], "empty": [(5,), (0,), (0, 7), (200,), (0,)],
        "many": [(i % 7 + 1, i % 5 + 1) for i in range(250)], "large": [(1000, 1003), (17,), (2048, 512)]}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,gdtype", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
@pytest.mark.parametrize("which", list(SETS))
def test_32_bits_against_64(which, dtype, gdtype):
    ps, gs = tensors(SETS[which], dtype, gdtype, 1)
    dev = [p.cuda() for p in ps]
    opt = ops.AdamW(dev, **HYPER)
    assert opt.offsets == [sum(-(-q.numel() // 128) * 128 for q in ps[:i]) for i in range(len(ps))]
    for t in (1, 2, 3):
        before = [p.cpu().clone() for p in dev], opt.m.cpu().clone(), opt.v.cpu().clone()
        _, gs = tensors(SETS[which], dtype, gdtype, 10 + t)
        opt.step([g.cuda() for g in gs])
        for i, (p, g, at) in enumerate(zip(before[0], gs, opt.offsets)):
            n = p.numel()
            held = slice(at, at + n)
            (p1, m1, v1), (tp, tm, tv) = step64(p.reshape(-1), g.reshape(-1), before[1][held], before[2][held], t, **HYPER)
            got = dev[i].cpu().reshape(-1).double()
            assert ((got - p1).abs() <= tp * (1 + HALF[dtype]) + HALF[dtype] * p1.abs() + 2.0 ** -25 * (dtype == torch.float16)).all(), (t, i)
            assert ((opt.m.cpu()[held].double() - m1).abs() <= tm).all() and ((opt.v.cpu()[held].double() - v1).abs() <= tv).all(), (t, i)
            rest = slice(at + n, at + -(-n // 128) * 128)
            assert not opt.m[rest].any() and not opt.v[rest].any()


def held_as(codes, scale):
    return (codes.float().view(-1, 128) * scale.float()[:, None]).view(-1).cpu()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,gdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("which", list(SETS))
def test_8_bits_against_64(which, dtype, gdtype):
    """The step itself as in 32 bits from the states that are held; then m and r = sqrt(v) are one of the two neighbours in 8 bits, the one that the hash says
    (unless the place between them is within the error of the step of the border), in the smallest scale that holds the block."""
    ps, gs = tensors(SETS[which], dtype, gdtype, 2)
    dev = [p.cuda() for p in ps]
    opt = ops.AdamW(dev, bits=8, seed=77, **HYPER)
    for t in (1, 2, 3):
        p0, m0, r0 = [p.cpu().clone() for p in dev], held_as(opt.m, opt.m_scale), held_as(opt.r, opt.r_scale)
        _, gs = tensors(SETS[which], dtype, gdtype, 20 + t)
        opt.step([g.cuda() for g in gs])
        q = {"m": (opt.m.cpu().float(), opt.m_scale.view(torch.uint8).cpu().int() - 127), "r": (opt.r.cpu().float(), opt.r_scale.view(torch.uint8).cpu().int() - 127)}
        for i, (p, g, at) in enumerate(zip(p0, gs, opt.offsets)):
            n = p.numel()
            if n == 0:
                continue
            s = slice(at, at + n)
            (p1, m1, v1), (tp, tm, tv) = step64(p.reshape(-1), g.reshape(-1), m0[s], r0[s].double().square(), t, **HYPER)
            got = dev[i].cpu().reshape(-1).double()
            tv = tv + 2 * E32 * v1                                    # (r squared is rounded too)
            tp = tp + 2 * E32 * p1.abs() + 4 * E32 * (p1 - p.reshape(-1).double()).abs()
            assert ((got - p1).abs() <= tp * (1 + HALF[dtype]) + HALF[dtype] * p1.abs()).all(), (t, i)
            key = mix(mix(mix((77 + 0x3C6EF372) & 0xFFFFFFFF) ^ t) + i & 0xFFFFFFFF)
            h = mix(torch.arange(n) ^ key)
            full = -(-n // 128) * 128
            for name, x, tol, u, floor in (("m", m1, tm, h & 0xFFFF, False), ("r", v1.sqrt(), 0.5 * tv / v1.sqrt().clamp_min(1e-30) + 2 * E32 * v1.sqrt(), h >> 16, True)):
                codes, e = q[name]
                codes, e = codes[at:at + full], e[at // 128:(at + full) // 128]
                pad = lambda z: torch.nn.functional.pad(z, (0, full - n)).view(-1, 128)  # noqa: E731
                X, T = pad(x.abs()), pad(tol)
                big = X.amax(1)
                scale = torch.ldexp(torch.ones_like(big), e)
                slack = T.amax(1) + E32 * big
                assert (big <= 448 * scale + slack).all() and ((big >= 224 * scale - slack) | (e == -127) | (big <= slack)).all(), (t, i, name)
                y, c, ty = X / scale[:, None], codes.view(-1, 128).double(), T / scale[:, None]
                assert (c.abs() <= 448).all() and (torch.sign(c) * torch.sign(pad(x)) >= 0).all()
                c = c.abs()
                gap = torch.exp2(torch.floor(torch.log2(y.clamp_min(2.0 ** -6))) - 3)
                place = y / gap
                up = torch.floor(place + pad(u.double()) / 65536)
                want = up * gap
                if floor:
                    want = torch.where(y > 0, want.clamp_min(2.0 ** -9), want)
                near = (place + pad(u.double()) / 65536 - torch.round(place + pad(u.double()) / 65536)).abs() <= ty / gap + 2.0 ** -15
                assert ((c == want) | (near & ((c - want).abs() <= 2 * gap))).all(), (t, i, name)
                assert near.double().mean() < 0.05 or n < 500
            assert not opt.m.view(torch.uint8)[at + n:at + full].any() and not opt.r.view(torch.uint8)[at + n:at + full].any()


@pytest.mark.gpu
def test_8_bits_round_without_a_bias():
    """v under a constant gradient goes to g^2 also with steps far below half a rounding step (b2 = 0.999: each moves v by 0.1 % of the way, a step of 8 bits is
    6 to 12 % of r).  2^17 elements with equal gradients: the mean of r has a standard error of at most 2^-3 / sqrt(2^17) = 0.0004 of r per step; rounding to
    the nearest would leave r where it is.  From r0 = 2 g, 600 steps: v = g^2 (1 + 3 * 0.999^600) in the mean of the exact recurrence; rounding adds the variance of
    r to the mean of v each step, at most (gap / 2)^2 with gap <= r / 8, carried on: v grows by at most a factor (1 + 1/256) per step, so only the direction
    and the order are asked for: r falls by at least half of what the exact recurrence says."""
    n = 1 << 17
    p = torch.zeros(n, device="cuda")
    opt = ops.AdamW([p], lr=0.0, betas=(0.9, 0.999), bits=8, weight_decay=0.0)
    g = torch.full((n,), 0.75, device="cuda")
    opt.r.view(torch.uint8).copy_(torch.full((n,), 1.5).to(torch.float8_e4m3fn).view(torch.uint8))
    means = []
    for _ in range(600):
        opt.step([g])
        means.append(None)
    m, r = held_as(opt.m, opt.m_scale), held_as(opt.r, opt.r_scale)
    exact = 0.75 * math.sqrt(1 + 3 * 0.999 ** 600)
    assert r.mean().item() < 1.5 - 0.5 * (1.5 - exact), r.mean()
    # m under b1 = 0.9 keeps to g: each step's rounding has mean 0 and a size of at most gap = 2^-4 (between 0.5 and 1)
    assert abs(m.mean().item() - 0.75) < 6 * 2.0 ** -4 / math.sqrt(n * 0.19) + 0.75 * 2.0 ** -16


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_zeros_tiny_and_non_finite_gradients(bits):
    n = 512
    p = torch.ones(n, device="cuda")
    opt = ops.AdamW([p], bits=bits, **{**HYPER, "weight_decay": 0.0})
    g = torch.zeros(n)
    opt.step([g.cuda()])
    assert (p == 1).all()
    g[0], g[1], g[2], g[3] = math.nan, math.inf, 1e-30, 1.0
    g[200] = 1e-25                                                # a block of which one element is tiny
    opt.step([g.cuda()])
    got = p.cpu()
    assert torch.isnan(got[0]) and not torch.isfinite(got[1]) and (got[4:128] == 1).all() and torch.isfinite(got[2:]).all() and got[3] < 1
    opt.step([torch.zeros(n, device="cuda")])
    assert torch.isfinite(p.cpu()[2:]).all()
    if bits == 8:                                                 # in one block with a much larger one, v is small but not 0: the step stays bounded
        q = torch.zeros(128, device="cuda")
        opt = ops.AdamW([q], bits=8, **{**HYPER, "weight_decay": 0.0})
        g = torch.full((128,), 1e-6)
        g[0] = 1e3
        for t in range(1, 21):
            # a small element is held as 0 or one unit 2^-9 of its block's scale: m <= b1 u_m + (1 - b1) g, and from the second step on r >= sqrt(b2) u_r, the floor
            # (both from the scales that are held before the step); a step is lr m / (1 - b1^t) / (r / sqrt(1 - b2^t))
            um, ur = (2.0 ** -9 * s[0].float().item() for s in (opt.m_scale, opt.r_scale))
            before = q[1:].clone()
            opt.step([g.cuda()])
            m, r = (0.9 * um + 1e-7, math.sqrt(0.99) * ur) if t > 1 else (1e-7, 0.1 * 1e-6)
            most = HYPER["lr"] * m / (1 - 0.9 ** t) / (r / math.sqrt(1 - 0.99 ** t))
            assert (q[1:] - before).abs().max().item() <= most * 1.001 + 1e-9
        assert (opt.r.float() > 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_missing_gradients_views_and_p_grad(bits):
    """A tensor without a gradient stays as it is; gradients that are not contiguous; parameters that are parts of one buffer, not aligned to 16 bytes; p.grad."""
    flat = torch.randn(1000, device="cuda")
    shapes = [(0, 300), (301, 501), (501, 1000)]
    ps = [flat[a:b] for a, b in shapes]
    gs = [torch.randn(b - a, device="cuda") for a, b in shapes]
    whole = [p.clone() for p in ps]
    one, two = ops.AdamW(ps, bits=bits, **HYPER), ops.AdamW(whole, bits=bits, **HYPER)
    gap = flat[300].clone()
    one.step([gs[0], None, gs[2]])
    assert torch.equal(ps[1], whole[1]) and not one.m[384:640].view(torch.uint8).any() and torch.equal(flat[300], gap)
    two.step([gs[0], None, gs[2]])
    wide = torch.randn(499, 2, device="cuda")
    one.step([gs[0], gs[1], wide[:, 1]])
    two.step([gs[0], gs[1], wide[:, 1].contiguous()])
    for p, g in zip(whole, gs):
        p.grad = g
    two.step()
    one.step(gs)
    assert all(torch.equal(p, q) for p, q in zip(ps, whole))
    assert all(torch.equal(getattr(one, k).view(torch.uint8), getattr(two, k).view(torch.uint8)) for k in one._buffers())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_state_graph_and_another_stream(bits):
    """load_state goes on where state() was taken; a captured step counts on in its replays and equals eager steps bit for bit; a stream of its own."""
    def fresh(capturable):
        ps, _ = tensors(SETS["odd"], torch.float32, torch.float32, 3)
        ps = [p.cuda() for p in ps]
        return ps, ops.AdamW(ps, bits=bits, seed=5, capturable=capturable, **HYPER)

    grads = [[g.cuda() for g in tensors(SETS["odd"], torch.float32, torch.float32, 30 + k)[1]] for k in range(6)]
    ps, opt = fresh(False)
    for g in grads:
        opt.step(g)
    qs, opt2 = fresh(False)
    for g in grads[:3]:
        opt2.step(g)
    kept, at = opt2.state(), [q.clone() for q in qs]
    opt3 = ops.AdamW(at, bits=bits, seed=5, **HYPER)
    opt3.load_state(kept)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for g in grads[3:]:
            opt3.step(g)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(ps, at))
    ws, opt4 = fresh(True)
    held = [g.clone() for g in grads[0]]
    opt4.step(held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt4.step(held)
    for k in range(1, 6):
        for h, g in zip(held, grads[k]):
            h.copy_(g)
        graph.replay()
        torch.cuda.synchronize()
        [w.sum().item() for w in ws]
    assert opt4.state()["step"] == 6 and all(torch.equal(p, w) for p, w in zip(ps, ws))
    with pytest.raises(RuntimeError, match="capturable"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step(grads[0])


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """A tensor of more than 2^32 elements: its last elements take the step that a short tensor's take (in 32 bits: no random numbers)."""
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GiB of free device memory")
    n = (1 << 32) + 300
    p = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    t = torch.randn(300, generator=torch.Generator().manual_seed(2)).bfloat16()
    p[-300:], g[-300:] = t.cuda(), (t * 3).cuda()
    for bits in (32, 8):
        q = t.cuda().clone()
        small, large = ops.AdamW([q], bits=bits, **HYPER), ops.AdamW([p], bits=bits, **HYPER)
        small.step([(t * 3).cuda()])
        large.step([g])
        assert torch.equal(p[-300:], q) and not p[:5].any() and not p[(1 << 32) - 5:1 << 32].any()       # (the first step does not depend on what is held)
        p[-300:] = t.cuda()
        del large


@pytest.mark.gpu
def test_a_step_is_seen_by_autograd():
    p = torch.randn(10, device="cuda", requires_grad=True)
    y = (p * p).sum()
    ops.AdamW([p], **HYPER).step([torch.ones(10, device="cuda")])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    p = torch.randn(40, 4, device="cuda")
    g = torch.randn(40, 4, device="cuda")
    for bad, match in ((lambda: ops.AdamW([]), "none"), (lambda: ops.AdamW([p], bits=16), "bits"), (lambda: ops.AdamW([p], lr=-1), "lr"), (lambda: ops.AdamW([p], betas=(0.9, 1.0)), "betas"),
                       (lambda: ops.AdamW([p.double()]), "float32"), (lambda: ops.AdamW([p, p]), "overlap"), (lambda: ops.AdamW([p[:20], p[10:]]), "overlap"),
                       (lambda: ops.AdamW([p, p.clone().half()]), "one AdamW"), (lambda: ops.AdamW([p.t()]), "contiguous"), (lambda: ops.AdamW([p]).step([g, g]), "gradients"),
                       (lambda: ops.AdamW([p]).step([g[:3]]), "tensor"), (lambda: ops.AdamW([p]).step([g.double()]), "float32"), (lambda: ops.AdamW([p]).step([g.cpu()]), "cpu"),
                       (lambda: ops.AdamW([p, p.clone()]).step([g, g.half()]), "for all"), (lambda: ops.AdamW([p]).load_state({"step": 1, "m": torch.zeros(1)}), "load_state")):
        with pytest.raises(ValueError, match=match):
            bad()


@pytest.mark.gpu
def test_weights_that_have_moved_are_refused():
    """A tensor's memory exchanged behind the optimiser's back: for another place of the same kind it follows, for another device or type it refuses."""
    for move in (lambda p: p.cpu(), lambda p: p.half()):
        p, g = torch.randn(300, device="cuda"), torch.randn(300, device="cuda")
        o = ops.AdamW([p])
        p.data = move(p)
        with pytest.raises(ValueError, match="shape, type or device"):
            o.step([g])
        assert o.steps == 0
    p, q = torch.randn(300, device="cuda"), torch.randn(300, device="cuda")
    one, two = ops.AdamW([p], capturable=True), ops.AdamW([q])
    p.data = q.clone()
    one.step([g])
    two.step([g])
    assert torch.equal(p, q)


def test_refusals_without_a_gpu():
    with pytest.raises(ValueError, match="GPU"):
        ops.AdamW([torch.randn(3)])
    L = lib.load_library()
    buf = (C.c_char * 4096)()
    at = (C.addressof(buf) + 63) // 64 * 64
    good = dict(lr=0.1, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0, param_dtype=0, grad_dtype=0, bits=32, seed=0, tensor_base=0, step=1, step_dev=None)

    def refused(match, count=1, p=at, g=at, n=4, m=at, v=at, ms=None, rs=None, **kw):
        o = lib.AdamWOptions(**{**good, **kw})
        rc = L.agz_adamw_step(0, None, C.byref(o), count, (C.c_void_p * 1)(p), (C.c_void_p * 1)(g), (C.c_int64 * 1)(n), m, v, ms, rs)
        assert rc == -1 and match in L.agz_ops_last_error().decode(), L.agz_ops_last_error()

    refused("null", count=-1)
    refused("null", m=None)
    refused("dtype", param_dtype=3)
    refused("dtype", grad_dtype=-1)
    refused("bits", bits=16)
    refused("2^34", n=2 ** 34 + 1)
    refused("scales", bits=8)
    refused("step", step=0)
    refused("betas", beta1=1.0)
    refused("betas", beta2=math.nan)
    refused("lr", lr=-1.0)
    refused("tensor", n=-1)
    refused("16 bytes", m=at + 4)
    refused("is null", p=None)
    refused("aligned", g=at + 2)
    assert L.agz_adamw_step(0, None, None, 0, None, None, None, None, None, None, None) == -1
    assert L.agz_adamw_state_elements(3, (C.c_int64 * 3)(1, 0, 129)) == 384 and L.agz_adamw_state_elements(1, (C.c_int64 * 1)(-1)) == -1


def late_tensors(calls, capturable=False, bits=32, dense=False, state_at=None, device="cuda"):
    """40 tensors over `calls` calls: tensor i has a gradient from call i on, odd ones not at every fifth call after that; -> weights and optimiser.  dense: every
    tensor has the same gradients one call after the other from the first call on, and none behind its last."""
    sizes = [37 * i % 300 + 1 for i in range(40)]
    r = torch.Generator().manual_seed(9)
    ps = [torch.randn(n, generator=r).to(device) for n in sizes]
    make = lambda: ops.AdamW(ps, bits=bits, seed=3, capturable=capturable, **HYPER)  # noqa: E731
    opt = make()
    has = [[c >= i and not (i % 2 and (c - i) % 5 == 4) for c in range(calls)] for i in range(40)]
    grad = lambda i, k: torch.randn(sizes[i], generator=torch.Generator().manual_seed(100 * i + k)).to(device)  # noqa: E731
    for c in range(calls):
        opt.step([(grad(i, c) if c < sum(has[i]) else None) if dense else (grad(i, sum(has[i][:c])) if has[i][c] else None) for i in range(40)])
        if c == state_at:
            kept = opt.state()
            opt = make()
            opt.load_state(kept)
    return ps, opt


def same_states(one, two):
    return all(torch.equal(getattr(one, k).view(torch.uint8), getattr(two, k).view(torch.uint8)) for k in one._buffers())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_tensor_counts_its_own_steps(bits):
    """What a tensor's steps are depends on the gradients that it had, not on the calls in which it had none: bit for bit the same, with up to 40 different numbers
    of steps in a call, with the numbers on the device, and from a saved state on."""
    want, dense = late_tensors(43, bits=bits, dense=True)
    for form in (dict(), dict(capturable=True), dict(state_at=20), dict(state_at=20, capturable=True)):
        got, opt = late_tensors(43, bits=bits, **form)
        assert all(torch.equal(p, q) for p, q in zip(got, want)) and same_states(opt, dense), form
        assert opt.state()["step"] == 43 and opt.state()["missed"][:4] == [0, 1 + 8, 2, 3 + 8], form


@pytest.mark.gpu
def test_a_late_tensor_against_64_bits():
    """A tensor that gets its first gradient in the 51st call takes the first step of its own, and one that then misses a call the second in the 53rd; calls without
    any gradient count for nobody."""
    p = torch.randn(300, generator=torch.Generator().manual_seed(1))
    gs = [torch.randn(300, generator=torch.Generator().manual_seed(k)) for k in (2, 3)]
    first, late = torch.randn(5, device="cuda"), p.cuda()
    opt = ops.AdamW([first, late], **HYPER)
    for c in range(50):
        opt.step([torch.ones(5, device="cuda") if c % 3 else None, None])
    m = v = torch.zeros(300, dtype=torch.float64)
    want = p
    for t, g in enumerate(gs, 1):
        opt.step([None, g.cuda()])
        (want, m, v), (tp, _, _) = step64(want, g, m, v, t, **HYPER)
        # the states held in 32 bits are what the next step begins with
        assert ((late.cpu().double() - want).abs() <= tp + E32 * want.abs()).all(), t
        want, m, v = late.cpu().clone(), opt.m[128:428].cpu().clone(), opt.v[128:428].cpu().clone()
        opt.step([first, None])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_missing_gradients_in_a_graph(bits):
    """Two graphs of one optimiser, one with a gradient of every tensor and one without the second's, replayed in turns, against a host that counts."""
    sizes = [200, 131, 50]
    start = [torch.randn(n, generator=torch.Generator().manual_seed(n)).cuda() for n in sizes]
    ps, qs = [p.clone() for p in start], [p.clone() for p in start]
    one, two = ops.AdamW(ps, bits=bits, capturable=True, **HYPER), ops.AdamW(qs, bits=bits, **HYPER)
    grads = [torch.randn(n, generator=torch.Generator().manual_seed(n + 1)).cuda() for n in sizes]
    some = [grads[0], None, grads[2]]
    one.step(some)
    two.step(some)
    torch.cuda.synchronize()
    graphs = []
    for g in (grads, some):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            one.step(g)
        graphs.append((graph, g))
    for k in (1, 0, 0, 1, 1, 0):
        graph, g = graphs[k]
        graph.replay()
        torch.cuda.synchronize()
        two.step(g)
        assert all(torch.equal(p, q) for p, q in zip(ps, qs)) and same_states(one, two)
    one.step(grads)
    two.step(grads)
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    a, b = one.state(), two.state()
    assert a["step"] == b["step"] == 8 and a["missed"] == b["missed"] == [0, 4, 0]


@pytest.mark.gpu
def test_states_of_other_lengths_are_refused():
    p = torch.randn(10, device="cuda")
    opt = ops.AdamW([p])
    good = opt.state()
    for bad in ([], [0, 0], [-1], [5]):
        with pytest.raises(ValueError, match="load_state"):
            opt.load_state({**good, "step": 4, "missed": bad})
    opt.load_state({k: v for k, v in good.items() if k != "missed"})
    assert opt.state()["missed"] == [0]


def test_counts_are_refused_without_a_gpu():
    L = lib.load_library()
    buf = (C.c_char * 4096)()
    at = (C.addressof(buf) + 63) // 64 * 64
    good = dict(lr=0.1, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0, param_dtype=0, grad_dtype=0, bits=32, seed=0, tensor_base=0, step=3, step_dev=None)
    for missed, grad in ((-1, at), (3, at), (4, None)):
        o = lib.AdamWOptions(**good)
        assert L.agz_adamw_step_missed(0, None, C.byref(o), (C.c_int64 * 1)(missed), None, 1, (C.c_void_p * 1)(at), (C.c_void_p * 1)(grad), (C.c_int64 * 1)(4), at, at, None, None) == -1
        assert "missed" in L.agz_ops_last_error().decode()
    o = lib.AdamWOptions(**good)                                    # a count on the device belongs to a step on the device
    assert L.agz_adamw_step_missed(0, None, C.byref(o), None, at, 1, (C.c_void_p * 1)(at), (C.c_void_p * 1)(at), (C.c_int64 * 1)(4), at, at, None, None) == -1
    assert "missed_dev" in L.agz_ops_last_error().decode()


@pytest.mark.gpu
@pytest.mark.parametrize("capturable", [False, True])
def test_a_refused_step_counts_nothing(capturable):
    p, g = torch.randn(300, device="cuda"), torch.randn(300, device="cuda")
    opt = ops.AdamW([p], capturable=capturable, **HYPER)
    opt.step([g])
    before = p.clone()
    for name, bad in (("lr", -1.0), ("lr", math.nan), ("betas", (0.9, 1.0)), ("betas", (math.nan, 0.9)), ("betas", (0.9,)), ("eps", -1.0), ("weight_decay", math.nan)):
        good = getattr(opt, name)
        setattr(opt, name, bad)
        with pytest.raises(ValueError, match="needed"):
            opt.step([g])
        setattr(opt, name, good)
        assert opt.state()["step"] == opt.steps == 1 and torch.equal(p, before), name
    with pytest.raises(ValueError, match="betas"):
        ops.AdamW([p], betas=(0.9, 0.99, 0.999))
    opt.betas = [0.9, 0.99]
    opt.lr = torch.tensor(opt.lr)
    for change in (lambda: opt.betas.__setitem__(1, 1.5), lambda: opt.lr.fill_(-1.0)):      # (in place)
        kept = opt.betas[1], opt.lr.item()
        change()
        with pytest.raises(ValueError, match="needed"):
            opt.step([g])
        opt.betas[1] = kept[0]
        opt.lr.fill_(kept[1])
        assert opt.state()["step"] == opt.steps == 1 and torch.equal(p, before)
    opt.step([g])
    assert opt.state()["step"] == opt.steps == 2 and not torch.equal(p, before)


@pytest.mark.gpu
def test_a_tensor_without_a_gradient_stays_unchanged_for_autograd():
    p, q = torch.randn(10, device="cuda", requires_grad=True), torch.randn(10, device="cuda", requires_grad=True)
    y = (q * q).sum()
    ops.AdamW([p, q], **HYPER).step([torch.ones(10, device="cuda"), None])
    y.backward()
    assert torch.equal(q.grad, 2 * q.detach())


def test_nothing_but_empty_tensors_needs_no_states():
    """Tensors without elements have no states, so there is no buffer to name: not an error of the arguments (without a GPU the call ends with the missing device)."""
    L = lib.load_library()
    o = lib.AdamWOptions(lr=0.1, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0, param_dtype=0, grad_dtype=0, bits=8, seed=0, tensor_base=0, step=1)
    rc = L.agz_adamw_step(0, None, C.byref(o), 2, (C.c_void_p * 2)(), (C.c_void_p * 2)(), (C.c_int64 * 2)(0, 0), None, None, None, None)
    assert rc == (0 if torch.cuda.is_available() else -2), L.agz_ops_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_of_empty_tensors(bits):
    p = torch.empty(0, 3, device="cuda")
    opt = ops.AdamW([p], bits=bits)
    opt.step([torch.empty(0, 3, device="cuda")])
    opt.load_state(opt.state())
    assert opt.steps == 1 and p.shape == (0, 3)


@pytest.mark.gpu
def test_8_bits_round_to_both_sides_in_proportion():
    """One step of 2^20 equal elements: m and r lie between two neighbours in 8 bits, and their means keep to the exact values from both sides.  An element is up with the
    probability of its place f (in steps of 2^-16 of a gap), so the mean is off by at most 2^-16 of a gap and six standard errors, gap sqrt(f (1 - f) / n) <= gap / (2 * 2^10),
    beside a few roundings of 32 bits.  The mean of r^2, which the next step begins with, is the square of the mean and the variance of the rounding, gap^2 f (1 - f)."""
    n, b1, b2 = 1 << 20, 0.9, 0.999
    for g, r0, m0 in ((0.6, 0.5625, 0.375), (3e-5, 2.0 ** -15, -(2.0 ** -14)), (700.0, 832.0, 104.0), (0.0, 1.75, 1.625)):
        p = torch.zeros(n, device="cuda")
        opt = ops.AdamW([p], lr=0.0, betas=(b1, b2), bits=8, weight_decay=0.0, seed=11)
        held = ops.AdamW([p], lr=0.0, bits=8)
        for name, x in (("m", m0), ("r", r0)):
            q = ops.quantize_fp8(torch.full((n // 128, 128), x, device="cuda"))
            assert (q.dequantize() == x).all()                      # (all of them are values of 8 bits)
            getattr(held, name).view(torch.uint8).copy_(q.q.view(torch.uint8).view(-1))
            getattr(held, name + "_scale").view(torch.uint8).copy_(q.scale.view(torch.uint8)[:, 0])
        opt.load_state(held.state())
        g32 = torch.full((n,), g, device="cuda")
        opt.step([g32])
        g64 = g32[0].double().item()
        for codes, scale, x in ((opt.m, opt.m_scale, b1 * m0 + (1 - b1) * g64), (opt.r, opt.r_scale, math.sqrt(b2 * r0 * r0 + (1 - b2) * g64 * g64))):
            got = held_as(codes, scale).double()
            gap = 2.0 ** (math.floor(math.log2(abs(x))) - 3)
            tol = gap * (2.0 ** -16 + 6 / 2 ** 11) + 8 * E32 * (abs(x) + abs(m0) + abs(g64))
            assert abs(got.mean().item() - x) <= tol, (g, x, got.mean())
            low = math.floor(abs(x) / gap) * gap
            assert ((got.abs() == low) | (got.abs() == low + gap)).all()
            f = (abs(x) - low) / gap
            # (2 |x| times the mean's own error, and the same six standard errors of the squares' differences, at most 2 (low + gap) gap apart)
            assert abs(got.square().mean().item() - x * x - gap * gap * f * (1 - f)) <= 2 * (abs(x) + gap) * tol, (g, x)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_the_call_without_counts(bits):
    """agz_adamw_step takes the call's t, of the host or of the device, for every tensor: the step that ops.AdamW takes where no gradient was missing."""
    L = lib.load_library()
    ps, gs = tensors(SETS["odd"], torch.float32, torch.bfloat16, 4)
    gs = [g.cuda() for g in gs]
    want = [p.cuda() for p in ps]
    opt = ops.AdamW(want, bits=bits, seed=6, **HYPER)
    opt.load_state({**opt.state(), "step": 2, "missed": [0] * len(ps)})
    opt.step(gs)
    n = len(ps)
    for step_dev in (None, torch.full((), 3, dtype=torch.int64, device="cuda")):
        got = [p.cuda() for p in ps]
        held = ops.AdamW(got, bits=bits)                          # (its buffers)
        second, scales = (held.v, (None, None)) if bits == 32 else (held.r, (held.m_scale.data_ptr(), held.r_scale.data_ptr()))
        o = lib.AdamWOptions(lr=HYPER["lr"], beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.1, param_dtype=0, grad_dtype=1, bits=bits, seed=6, tensor_base=0, step=3 if step_dev is None else 0,
                             step_dev=None if step_dev is None else step_dev.data_ptr())
        rc = L.agz_adamw_step(0, torch.cuda.current_stream().cuda_stream, C.byref(o), n, (C.c_void_p * n)(*[p.data_ptr() for p in got]), (C.c_void_p * n)(*[g.data_ptr() for g in gs]),
                              (C.c_int64 * n)(*[p.numel() for p in ps]), held.m.data_ptr(), second.data_ptr(), *scales)
        assert rc == 0, L.agz_ops_last_error()
        assert all(torch.equal(p, q) for p, q in zip(got, want)) and same_states(held, opt)
