"""alphagpu_amd.ops.log_probs against a plain implementation in 64 bits, its refusals, streams and graphs."""
import ctypes as C
import math

import pytest
import torch
import torch.autograd.forward_ad as fwd
import torch.utils.checkpoint

from alphagpu_amd import lib, ops

E32 = 2.0 ** -24                                     # half a step of float32
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
NINF = -math.inf


def plain(x, moves=None, mask=None, target=None, top=0, g=None):
    """The definition in 64 bits on the CPU, and what its roundings in 32 bits may add up to (by hand, below)."""
    x = x.detach().cpu().double()
    n, a = x.shape
    s = x != NINF                                                     # (NaN is allowed)
    if mask is not None:
        s = s & (mask.cpu() != 0).expand(n, a)
    xm = torch.where(s, x, torch.tensor(NINF, dtype=torch.float64))
    some = s.any(1, keepdim=True)
    mx = torch.where(some, xm.max(1, keepdim=True).values, 0.0)
    d = torch.where(s, xm - mx, torch.tensor(0.0, dtype=torch.float64))
    e = torch.where(s, d.exp(), torch.tensor(0.0, dtype=torch.float64))
    tot = e.sum(1, keepdim=True)
    ls = torch.where(some, tot, 1.0).log()
    p = torch.where(some, e / tot, 0.0)
    logp = torch.where(s, d - ls, torch.tensor(NINF, dtype=torch.float64))
    h = torch.where(some, ls - torch.where(p > 0, p * d, torch.zeros_like(d)).sum(1, keepdim=True), 0.0)
    bad = some & ~torch.isfinite(ls + 0 * mx)
    # a lane adds up at most a / 64 + 24 terms; e^d of a rounded d: relative error (4 |d| + 4) half steps, rescaling included
    adds, ed = a / 64 + 24, (p * d.abs()).sum(1, keepdim=True)
    ed2 = (p * d * d).sum(1, keepdim=True)
    tol_ls = E32 * (adds + 4 * ed + 4 * ls.abs() + 8)
    tol_lp = tol_ls + E32 * (2 * d.abs() + 2 * torch.where(s, logp, 0.0).abs() + 2)
    tol_h = tol_ls + E32 * ((adds + 8) * ed + 8 * ed2 + 4 * h.abs() + 4)
    out, tol = {"entropy": torch.where(bad, math.nan, h)[:, 0]}, {"entropy": tol_h[:, 0]}
    given = None
    if moves is not None:
        mv = moves.cpu().long()
        given = (mv >= 0) & (mv < a)
        at = mv.clamp(0, a - 1)[:, None]
        m = torch.where(given, logp.gather(1, at)[:, 0], 0.0)
        out["move"], tol["move"] = torch.where(bad[:, 0], math.nan, m), tol_lp.gather(1, at)[:, 0]
    if target is not None:
        t = target.cpu().double()
        out["target"] = torch.where(bad[:, 0], math.nan, torch.where(t != 0, t * logp, torch.zeros_like(t)).sum(1))
        ta = t.abs().sum(1)
        tol["target"] = E32 * (adds + 6) * (t * d).abs().sum(1) + ta * (tol_ls[:, 0] + E32 * (adds + 2) * ls[:, 0].abs()) + E32
    if top:
        val, idx = torch.sort(xm, dim=1, descending=True, stable=True)
        val, idx = val[:, :top], idx[:, :top]
        ok = (val != NINF) & ~bad
        out["top_move"] = torch.where(ok, idx, -1).int()
        out["top"] = torch.where(bad, math.nan, torch.where(ok, logp.gather(1, idx), torch.tensor(NINF, dtype=torch.float64)))
        tol["top"] = tol_lp.gather(1, idx)
    if g is not None:
        c, ca = torch.zeros_like(x), torch.zeros_like(x)
        gg = {k: v.cpu().double() for k, v in g.items()}
        if "move" in gg:
            w = torch.where(given, gg["move"], 0.0)[:, None]
            c, ca = c.scatter_add(1, at, w), ca.scatter_add(1, at, w.abs())
        if "target" in gg:
            c, ca = c + t * gg["target"][:, None], ca + (t * gg["target"][:, None]).abs()
        if "top" in gg:
            w = torch.where(ok, gg["top"], 0.0)
            c, ca = c.scatter_add(1, idx, w), ca.scatter_add(1, idx, w.abs())
        gh = gg["entropy"][:, None] if "entropy" in gg else torch.zeros(n, 1, dtype=torch.float64)
        lp0 = torch.where(p > 0, logp, torch.zeros_like(logp))
        dx = c - p * c.sum(1, keepdim=True) - gh * p * (lp0 + h)
        rel = tol_lp + E32 * (4 * lp0.abs() + 4)                      # relative error of p
        tol_g = p * ca.sum(1, keepdim=True) * (rel + E32 * (top + adds + 6)) + 4 * E32 * ca + (gh * p).abs() * ((lp0 + h).abs() * (rel + 4 * E32) + tol_lp + tol_h)
        out["dlogits"] = torch.where(s, torch.where(bad, math.nan, dx), torch.zeros_like(dx))
        tol["dlogits"] = tol_g
    return out, tol


def close(got, want, tol, what=""):
    got, want = got.detach().cpu(), want
    if want.dtype == torch.int32:
        assert torch.equal(got, want), what
        return
    half = HALF[got.dtype]
    got = got.double()
    nan, inf = torch.isnan(want), torch.isinf(want)
    assert torch.equal(torch.isnan(got), nan), what
    assert torch.equal(got[inf], want[inf]), what
    fine = ~nan & ~inf
    small = 2.0 ** -25 if half == HALF[torch.float16] else 2.0 ** -133 if half == HALF[torch.bfloat16] else 2.0 ** -120   # below the normal numbers (32 bits: e^d may flush)
    off = (got - want).abs()[fine] - (tol[fine] * (1 + half) + half * want.abs()[fine] + small)
    assert off.numel() == 0 or off.max() <= 0, (what, off.max().item())


def inputs(n, a, dtype, seed, mask="some", moves=True, target=True, top=0, spread=3.0):
    r = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, a, generator=r) * spread).to(dtype)
    mk = None
    if mask == "some":
        mk = torch.rand(n, a, generator=r) < torch.rand(n, 1, generator=r)
    elif mask == "one":
        mk = torch.rand(1, a, generator=r) < 0.7
    mv = torch.randint(-1, a, (n,), generator=r) if moves else None
    t = None
    if target:
        t = torch.rand(n, a, generator=r)
        if mk is not None:
            t = t * mk
        t = t / t.sum(1, keepdim=True).clamp_min(1e-9)
    g = {"entropy": torch.randn(n, generator=r)}
    if moves:
        g["move"] = torch.randn(n, generator=r)
    if target:
        g["target"] = torch.randn(n, generator=r)
    if top:
        g["top"] = torch.randn(n, top, generator=r)
    return x, mv, mk, t, g


def check(x, mv, mk, t, top, g, what=""):
    dev = [None if v is None else v.cuda() for v in (x, mv, mk, t)]
    leaf = dev[0].detach().requires_grad_()
    r = ops.log_probs(leaf, dev[1], mask=dev[2], target=dev[3], top=top)
    g = {k: v for k, v in g.items() if getattr(r, k) is not None}
    want, tol = plain(x, mv, mk, t, top, g)
    for k in ("move", "entropy", "target", "top", "top_move"):
        if k in want:
            close(getattr(r, k), want[k], tol.get(k), (what, k))
        else:
            assert getattr(r, k) is None
    dx, = torch.autograd.grad([getattr(r, k) for k in g], [leaf], [v.cuda() for v in g.values()])
    assert dx.dtype == x.dtype
    close(dx, want["dlogits"], tol["dlogits"], (what, "dlogits"))


SIZES = [(1, 1), (3, 2), (5, 7), (1, 81), (257, 81), (64, 65), (33, 128), (9, 169), (7, 255), (6, 256), (5, 257), (3, 1000), (2, 1023), (4, 1024), (3, 4097), (2, 8191),
         (1, 16384), (2, 50001), (1, 131072), (3, 33333)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,a", SIZES)
def test_against_64_bits(n, a, dtype):
    top = min(a, 5)
    check(*inputs(n, a, dtype, 1, top=top)[:4], top, inputs(n, a, dtype, 1, top=top)[4], "masked")
    x, mv, mk, t, g = inputs(n, a, dtype, 2, mask=None, target=False)
    check(x, mv, mk, t, 0, g, "moves alone")
    x, mv, mk, t, g = inputs(n, a, dtype, 3, mask="one", moves=False, top=min(a, 32))
    check(x, mv, mk, t, min(a, 32), g, "one mask for all rows")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("a", [2, 81, 130, 700, 20000])
def test_rows_at_the_edges(a, dtype):
    """No allowed entry (by mask and by -inf), one allowed entry, the type's lowest value, large offsets, equal logits, NaN and +inf allowed and masked."""
    x, mv, mk, t, _ = inputs(16, a, dtype, 4, mask=None, top=2)
    mk = torch.ones(16, a, dtype=torch.bool)
    low = torch.finfo(dtype).min
    mk[0] = False
    x[1] = NINF
    mk[2] = False
    mk[2, a - 1] = True
    x[3, : a // 2] = low
    x[4] = low
    x[5] = 1.0e4
    x[6] += 3.0e4
    x[7] = 0.5
    x[8, 1] = math.nan
    x[9, 0] = math.inf
    x[10, 0], mk[10, 0] = math.nan, False
    x[11, 1], mk[11, 1] = math.inf, False
    x[12, 0], mk[12, 0] = NINF, False
    x[13, 0] = NINF
    x[14] = math.nan
    x[15, 0], x[15, 1] = 0.0, -0.0
    mv[:] = torch.arange(16) % a
    mv[13], mv[12], mv[3], mv[2] = 0, 0, 0, a - 1
    t = t * mk * (x != NINF)
    r = torch.Generator().manual_seed(9)
    g = {"entropy": torch.randn(16, generator=r), "move": torch.randn(16, generator=r), "target": torch.randn(16, generator=r), "top": torch.randn(16, 2, generator=r)}
    check(x, mv, mk, t, 2, g)


@pytest.mark.gpu
def test_moves_outside_the_actions_and_targets_on_masked_entries():
    x, mv, mk, t, g = inputs(6, 40, torch.float32, 5, mask="some")
    mv = torch.tensor([-1, 40, 2 ** 40, -2 ** 40, 39, 0])
    mk[:, 3] = False
    t[2, 3] = 0.25                                            # a target on a move that is not allowed: -inf
    check(x, mv, mk, t, 0, {k: v for k, v in g.items() if k != "target"})


@pytest.mark.gpu
def test_strides():
    """Rows of a wider tensor, one row for all (stride 0), unaligned starts, and a gradient that goes back through them."""
    for dtype in (torch.float32, torch.bfloat16):
        for a, first in ((81, 3), (700, 1), (5000, 5)):
            x, mv, mk, t, g = inputs(9, a + 11, dtype, 6, top=3)
            cut = slice(first, first + a)
            mv = mv.clamp(max=a - 1)
            want, tol = plain(x[:, cut], mv, mk[:, cut], t[:, cut], 3, g)
            big, bm, bt = x.cuda().requires_grad_(), mk.cuda(), t.cuda()
            r = ops.log_probs(big[:, cut], mv.cuda(), mask=bm[:, cut], target=bt[:, cut], top=3)
            dx, = torch.autograd.grad([r.move, r.entropy, r.target, r.top], [big], [g[k].cuda() for k in ("move", "entropy", "target", "top")])
            for k in ("move", "entropy", "target", "top", "top_move"):
                close(getattr(r, k), want[k], tol.get(k), (a, k))
            close(dx[:, cut], want["dlogits"], tol["dlogits"])
            assert not dx[:, :first].any() and not dx[:, first + a:].any()
    x = torch.randn(1, 81, device="cuda", requires_grad=True)
    r = ops.log_probs(x.expand(5, 81), torch.arange(5, device="cuda"))
    want, tol = plain(x.expand(5, 81), torch.arange(5))
    close(r.move, want["move"], tol["move"])
    dx, = torch.autograd.grad(r.move.sum(), x)
    p = torch.softmax(x.detach().double(), 1)
    assert (dx.double() - (torch.nn.functional.one_hot(torch.arange(5, device="cuda"), 81).sum(0) - 5 * p)).abs().max() < 5 * 64 * E32


@pytest.mark.gpu
def test_the_gradient_against_differences():
    """Central differences of the kernel's own forward: (f(x + h) - f(x - h)) / 2h is off by h^2 / 6 of the third derivative (at most 6 per unit of
    cotangent for log probabilities and 6 (1 + largest |logp|) for the entropy) and by the two forwards' errors / 2h."""
    n, a, h = 3, 11, 2.0 ** -6
    x, mv, mk, t, g = inputs(n, a, torch.float32, 7, top=2, spread=1.0)
    mv = mk.float().argmax(1)                                         # (an allowed move: no infinity among the outputs; every row has one)
    assert mk.any(1).all() and (mk.sum(1) >= 2).all()
    x = x * 0.5 + torch.randperm(a, generator=torch.Generator().manual_seed(1)) * 0.25
    best = torch.where(mk, x, torch.tensor(-1e30)).sort(1, descending=True).values
    smooth = (best[:, 0] - best[:, 1] > 2 * h) & (best[:, 1] - best[:, 2] > 2 * h)   # rows whose alternatives change places within h have a kink there (row 2: 0.4323 and 0.4315)
    assert smooth.sum() >= 2

    def f(x):
        r = ops.log_probs(x.cuda(), mv.cuda(), mask=mk.cuda(), target=t.cuda(), top=2)
        return sum((getattr(r, k).double().cpu() * g[k].double()).reshape(n, -1).sum(1) for k in g)

    leaf = x.cuda().requires_grad_()
    r = ops.log_probs(leaf, mv.cuda(), mask=mk.cuda(), target=t.cuda(), top=2)
    dx, = torch.autograd.grad([getattr(r, k) for k in g], [leaf], [v.cuda() for v in g.values()])
    want, tol = plain(x, mv, mk, t, 2, g)
    size = sum(v.abs().reshape(n, -1).sum(1) for v in g.values()).double()
    most = torch.where(mk, want["entropy"][:, None] + 8.0, 0.0).max()
    ftol = sum((tol[k].double() * g[k].abs().double()).reshape(n, -1).sum(1) for k in g)
    for j in range(a):
        e = torch.zeros(n, a)
        e[:, j] = h
        num = (f(x + e) - f(x - e)) / (2 * h)
        assert ((dx[:, j].cpu().double() - num).abs() <= size * (1 + most) * h * h + ftol / h + tol["dlogits"][:, j])[smooth].all(), j


def test_the_workspace_holds_every_plan():
    """Rows without mask and target are planned with room for one more block of 2048 at their end, and with longer parts earlier: 4096 rows of 6144 are two
    parts each so, and three with a mask.  32 bytes for each part."""
    L = lib.load_library()
    for n, a, parts in ((4096, 6144, 3), (2731, 6140, 3), (8191, 2049, 2), (1366, 12288, 6), (1, 33552384, 16383)):
        assert L.agz_logprob_workspace(n, a, 0) >= n * parts * 32, (n, a)


@pytest.mark.gpu
def test_many_long_rows_with_a_mask():
    """Numbers of rows from which a masked call is cut into other parts than a plain one."""
    for n, a in ((4096, 6144), (1366, 12288)):
        x, mv, mk, t, g = inputs(n, a, torch.bfloat16, 15, mask="one")
        r = ops.log_probs(x.cuda(), mv.cuda(), mask=mk.cuda(), target=t.cuda())
        rows = torch.tensor([0, 1, n // 2, n - 2, n - 1])
        want, tol = plain(x[rows], mv[rows], mk, t[rows])
        for k in ("move", "entropy", "target"):
            close(getattr(r, k).cpu()[rows], want[k], tol[k], (n, a, k))


@pytest.mark.gpu
def test_equal_logits_come_by_index():
    for a in (81, 300, 9000, 70000):
        x = torch.zeros(2, a)
        x[1, a // 3:] = 1.0
        r = ops.log_probs(x.bfloat16().cuda(), top=32)
        assert r.top_move.cpu().tolist() == [list(range(32)), list(range(a // 3, a // 3 + 32))]
    r = ops.log_probs(torch.randint(0, 3, (4, 5000), generator=torch.Generator().manual_seed(3)).float().cuda(), top=20)
    x = torch.randint(0, 3, (4, 5000), generator=torch.Generator().manual_seed(3)).float()
    assert torch.equal(r.top_move.cpu().long(), torch.sort(x, dim=1, descending=True, stable=True).indices[:, :20])


@pytest.mark.gpu
def test_the_best_in_one_place_and_spread_out():
    """Alternatives that all fall to one lane's or one part's share, ascending and descending rows."""
    for a in (96, 512, 4096, 65536):
        for x in (torch.arange(a).float(), -torch.arange(a).float(), (torch.arange(a) % 64 == 5).float() * torch.arange(a), (torch.arange(a) < 40).float() * torch.arange(a)):
            x = x[None] / a
            r = ops.log_probs(x.cuda(), top=32)
            assert torch.equal(r.top_move.cpu().long(), torch.sort(x, dim=1, descending=True, stable=True).indices[:, :32]), a


@pytest.mark.gpu
def test_equal_calls_give_equal_bits():
    for n, a in ((100, 81), (1, 131072), (3, 50001)):
        x, mv, mk, t, g = (v.cuda() if isinstance(v, torch.Tensor) else v for v in inputs(n, a, torch.bfloat16, 8))
        one = ops.log_probs(x, mv, mask=mk, target=t, top=5)
        for _ in range(3):
            two = ops.log_probs(x, mv, mask=mk, target=t, top=5)
            assert all(torch.equal(p, q) for p, q in zip(one, two))


@pytest.mark.gpu
def test_another_stream_and_a_graph():
    """On a stream of its own, and captured: every replay, with eager work and waits between, equals the eager call."""
    for n, a in ((300, 81), (1, 100000)):
        sets = [[v.cuda() for v in inputs(n, a, torch.float32, s)[:4]] for s in (10, 11, 12)]
        gr = [torch.randn(n, device="cuda") for _ in range(3)]

        def step(x, mv, mk, t):
            leaf = x.detach().requires_grad_()
            r = ops.log_probs(leaf, mv, mask=mk, target=t, top=3)
            dx, = torch.autograd.grad([r.move, r.entropy, r.target], [leaf], gr)
            return [*r, dx]

        eager = [step(*s) for s in sets]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step(*sets[0])
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(p.nan_to_num(7), q.nan_to_num(7)) for p, q in zip(other, eager[0]))
        held = [v.clone() for v in sets[0]]
        with torch.cuda.stream(side):
            step(*held)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*held)
        for k in (1, 2, 0, 1):
            for v, w in zip(held, sets[k]):
                v.copy_(w)
            graph.replay()
            torch.cuda.synchronize()
            again = step(*sets[k])
            for p, q, e in zip(out, again, eager[k]):
                assert torch.equal(p.nan_to_num(7), e.nan_to_num(7)) and torch.equal(q.nan_to_num(7), e.nan_to_num(7))


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """More than 2^32 logits: the last rows, forward and backward."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GiB of free device memory")
    n, a = 33000, 131072
    x = torch.zeros(n, a, dtype=torch.bfloat16, device="cuda")
    tail, mv, _, _, g = inputs(3, a, torch.bfloat16, 14, mask=None, target=False)
    x[-3:] = tail.cuda()
    x.requires_grad_()
    moves = torch.full((n,), -1, device="cuda")
    moves[-3:] = mv.cuda()
    r = ops.log_probs(x, moves, top=3)
    want, tol = plain(tail, mv, top=3, g=g)
    for k in ("move", "entropy", "top", "top_move"):
        close(getattr(r, k)[-3:], want[k], tol.get(k), k)
    gm, ge = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    gm[-3:], ge[-3:] = g["move"].cuda(), g["entropy"].cuda()
    dx, = torch.autograd.grad([r.move, r.entropy], [x], [gm, ge])
    close(dx[-3:], want["dlogits"], tol["dlogits"])
    assert not dx[-5:-3].any() and not dx[:2].any()


@pytest.mark.gpu
def test_two_captured_graphs_side_by_side():
    """Two graphs captured one after the other have workspaces of their own: replayed in any order, on two streams at once, each gives what it gives alone."""
    xs = [torch.randn(1, 90000, device="cuda") + k for k in range(2)]
    graphs, outs = [], []
    for x in xs:
        ops.log_probs(x, top=8)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.log_probs(x, top=8))
        graphs.append(g)
    want = [ops.log_probs(x, top=8) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        for o, w in zip(outs, want):
            assert torch.equal(o.entropy, w.entropy) and torch.equal(o.top_move, w.top_move) and torch.equal(o.top, w.top)


@pytest.mark.gpu
def test_saved_tensors_that_come_back_elsewhere():
    """Hooks that keep what a backward pass needs in host memory, and a part that is computed again (checkpoint): the memory of the first forward pass
    belongs to others by the time of the backward pass."""
    for a in (81, 5000):
        x, mv, mk, t, g = (v.cuda() if isinstance(v, torch.Tensor) else v for v in inputs(40, a, torch.float32, 16, top=3))
        g = {k: v.cuda() for k, v in g.items()}

        def part(x):
            r = ops.log_probs(x * 1.0, mv + 0, mask=mk.clone(), target=t + 0, top=3)
            return [getattr(r, k) for k in g]

        def grad(out, leaf):
            junk = [torch.full_like(v, 1) for v in (x, mv, mk, t) for _ in range(4)]       # what was let go is written to
            return torch.autograd.grad(out, [leaf], list(g.values()))[0], junk

        leaf = x.clone().requires_grad_()
        want, _ = grad(part(leaf), leaf)
        with torch.autograd.graph.save_on_cpu():
            out = part(leaf)
        assert torch.equal(grad(out, leaf)[0], want)
        out = torch.utils.checkpoint.checkpoint(part, leaf, use_reentrant=False)
        assert torch.equal(grad(out, leaf)[0], want)


@pytest.mark.gpu
def test_gradients_of_gradients_are_refused():
    x = torch.randn(4, 9, device="cuda", requires_grad=True)
    r = ops.log_probs(x, torch.zeros(4, dtype=torch.int64, device="cuda"))
    dx, = torch.autograd.grad(r.move.sum(), x, create_graph=True)
    want = torch.nn.functional.one_hot(torch.zeros(4, dtype=torch.int64), 9) - torch.softmax(x.detach().cpu(), 1)
    assert (dx.detach().cpu() - want).abs().max() < 64 * E32
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        dx.sum().backward()


@pytest.mark.gpu
def test_changed_logits_are_noticed():
    x = torch.randn(4, 9, device="cuda", requires_grad=True)
    y = x * 1.0
    r = ops.log_probs(y, torch.zeros(4, dtype=torch.int64, device="cuda"))
    y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.move.sum().backward()


@pytest.mark.gpu
def test_no_rows():
    x = torch.empty(0, 81, device="cuda", requires_grad=True)
    r = ops.log_probs(x, torch.empty(0, dtype=torch.int64, device="cuda"), top=2)
    assert r.move.shape == (0,) and r.top.shape == (0, 2)
    dx, = torch.autograd.grad([r.entropy], [x], [torch.empty(0, device="cuda")])
    assert dx.shape == (0, 81)


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    x = torch.randn(4, 9, device="cuda")
    with pytest.raises(ValueError, match="float32"):
        ops.log_probs(x.double())
    with pytest.raises(ValueError, match="next to each other"):
        ops.log_probs(x.t())
    with pytest.raises(ValueError, match="two dimensions"):
        ops.log_probs(x[0])
    with pytest.raises(ValueError, match="top"):
        ops.log_probs(x, top=10)
    with pytest.raises(ValueError, match="moves"):
        ops.log_probs(x, torch.zeros(3, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="GPU"):
        ops.log_probs(x, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError, match="mask"):
        ops.log_probs(x, mask=torch.ones(4, 8, dtype=torch.bool, device="cuda"))
    with pytest.raises(ValueError, match="constant"):
        ops.log_probs(x, target=torch.rand(4, 9, device="cuda", requires_grad=True))


def test_refusals_without_a_gpu():
    with pytest.raises(ValueError, match="GPU"):
        ops.log_probs(torch.randn(2, 3))
    L = lib.load_library()
    buf = (C.c_char * 4096)()
    at = (C.addressof(buf) + 63) // 64 * 64
    good = dict(n=2, a=4, logits=at, ld=4, dtype=0, top=0, stats=at + 512, entropy=at + 1024)

    def refused(match, fn=L.agz_logprob_forward, more=(), **kw):
        q = lib.LogProbArgs(**{**good, **kw})
        assert fn(0, None, C.byref(q), *more) == -1
        assert match in L.agz_ops_last_error().decode(), L.agz_ops_last_error()

    refused("rows of", n=-1)
    refused("actions", a=0)
    refused("actions", a=2 ** 31)
    refused("dtype", dtype=3)
    refused("alternatives", top=33)
    refused("stride", ld=-1)
    refused("required", logits=None)
    refused("aligned", logits=at + 2)
    refused("aligned", stats=at + 4)
    refused("without moves", move_logp=at)
    refused("without a target", target_logp=at)
    back = L.agz_logprob_backward
    refused("stats are required", back, (None, None, None, None, at, 4), stats=None)
    refused("row stride", back, (None, None, None, None, None, 4))
    refused("row stride", back, (None, None, None, None, at, 3))
    refused("without moves", back, (at, None, None, None, at, 4))
    refused("without a target", back, (None, None, at, None, at, 4))
    refused("without alternatives", back, (None, None, None, at, at, 4))
    assert L.agz_logprob_workspace(-1, 4, 0) < 0 and L.agz_logprob_workspace(1, 4, 33) < 0
    assert L.agz_logprob_forward(0, None, None) == -1


@pytest.mark.gpu
def test_forward_mode_derivatives_are_refused():
    """There is no forward-mode rule: a tangent is refused, never dropped; without one, or where forward mode is off, a level that is open changes nothing."""
    x, t = torch.randn(4, 9, device="cuda"), torch.rand(4, 9, device="cuda")
    want = ops.log_probs(x, target=t)
    with fwd.dual_level():
        d, dt = fwd.make_dual(x, torch.ones_like(x)), fwd.make_dual(t, torch.ones_like(t))
        with pytest.raises(ValueError, match="forward mode"):
            ops.log_probs(d)
        with pytest.raises(ValueError, match="forward mode"):
            ops.log_probs(x, target=dt)
        with torch.no_grad(), pytest.raises(ValueError, match="forward mode"):      # (no_grad is about the other mode)
            ops.log_probs(d, top=2)
        with pytest.raises((ValueError, RuntimeError)):
            ops.log_probs(fwd.make_dual(x.clone().requires_grad_(), torch.ones_like(x)))
        got = ops.log_probs(x, target=t)
        assert torch.equal(got.entropy, want.entropy) and torch.equal(got.target, want.target)
        plain = ops.log_probs(fwd.unpack_dual(d).primal)
        assert torch.equal(plain.entropy, want.entropy)
        with fwd._set_fwd_grad_enabled(False):                     # (as within the forward of a function that has a rule of its own)
            assert torch.equal(ops.log_probs(d).entropy, want.entropy)


def test_many_short_rows_are_not_too_many():
    """A launch holds fewer than 2^32 lanes: nearly 2^29 rows of which each takes eight of them, 2^26 that take a whole wave.  (Without a GPU a call that is not refused ends with
    the missing device; the memory behind the addresses is not read then.)"""
    if torch.cuda.is_available():
        pytest.skip("the addresses here are no device memory")
    L = lib.load_library()
    buf = (C.c_char * 4096)()
    at = (C.addressof(buf) + 63) // 64 * 64
    for n, a, dtype, top, forward, backward in ((1 << 26, 81, 1, 0, True, True), ((1 << 26) + 5, 2, 0, 0, True, True), ((1 << 29) - 32, 81, 1, 0, True, True), ((1 << 29) - 31, 81, 1, 0, False, False),
                                                (1 << 27, 500, 1, 0, True, True), (1 << 28, 500, 1, 0, False, False), ((1 << 26) - 4, 2000, 0, 0, True, True), (1 << 26, 2000, 0, 0, False, False),
                                                (1 << 26, 1000, 0, 9, False, True), (1 << 62, 2, 0, 0, False, False), (1 << 62, 4000, 0, 0, False, False)):
        ws = L.agz_logprob_workspace(n, a, top)
        assert (ws < 0) == (n > (1 << 29) - 32)
        q = lib.LogProbArgs(n=n, a=a, logits=at, ld=a, dtype=dtype, top=top, stats=at, entropy=at, workspace=at, workspace_bytes=max(ws, 0))
        for fits, call in ((forward, lambda: L.agz_logprob_forward(0, None, C.byref(q))), (backward, lambda: L.agz_logprob_backward(0, None, C.byref(q), None, at, None, None, at, a))):
            assert call() == (-2 if fits else -1) and (fits or b"too many rows" in L.agz_ops_last_error()), (n, a, L.agz_ops_last_error())


@pytest.mark.gpu
def test_more_than_2_26_short_rows():
    """Forward and backward where only the last rows and some in between differ from zeros: those as a short call has them, the others all alike."""
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GiB of free device memory")
    n, a = (1 << 26) + 37, 3
    some = torch.tensor([0, 5, 1 << 20, 1 << 25, (1 << 26) - 1, 1 << 26, n - 2, n - 1], device="cuda")
    few = torch.randn(8, a, generator=torch.Generator().manual_seed(4)).cuda()
    x = torch.zeros(n, a, device="cuda")
    x[some] = few
    def both(x):
        x = x.requires_grad_()
        r = ops.log_probs(x, top=1)
        dx, = torch.autograd.grad([r.entropy], [x], [torch.ones_like(r.entropy)])
        return r.entropy.detach(), r.top_move, dx
    want, got = both(few), both(x)
    for w, g in zip(want, got):
        assert torch.equal(g[some], w)
        rest = torch.ones(n, dtype=torch.bool, device="cuda")
        rest[some] = False
        assert (g[rest] == g[1]).all()


@pytest.mark.gpu
def test_too_many_long_rows_are_refused_by_name():
    """Rows that are one row again and again, so that there may be as many as one likes."""
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("needs 8 GiB of free device memory")
    with pytest.raises(ValueError, match="too many"):
        ops.log_probs(torch.zeros(1, 2000, device="cuda").expand(1 << 29, 2000))
    with pytest.raises(lib.AgzError, match="too many rows"):
        ops.log_probs(torch.zeros(1, 81, device="cuda").expand(1 << 29, 81))
