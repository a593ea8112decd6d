"""alphagpu_amd.ops: matrices in 8 bits and their products against plain implementations in 64 bits, refusals, streams and graphs."""
import ctypes as C
import math

import pytest
import torch
import torch.autograd.forward_ad as fwd

from alphagpu_amd import lib, ops

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def blocks(x, rows):
    """x in 8 bits with a power-of-two scale per rows x 128, as the 64-bit values it stands for, and the scales' exponents.  Scaling by powers of two is
    exact, so the values have to be equal bit for bit."""
    R, Cc = x.shape
    x = torch.nn.functional.pad(x.double(), (0, -Cc % 128, 0, -R % rows))
    b = x.view(x.shape[0] // rows, rows, x.shape[1] // 128, 128)
    am = torch.where(torch.isfinite(b), b.abs(), 0.0).amax((1, 3))
    f, e = torch.frexp(am)
    e = torch.where(am > 0, (e - 9 + (f > 0.875)).clamp(min=-127), 0)
    s = torch.ldexp(torch.ones_like(am), e)[:, None, :, None]
    y = b / s
    q = torch.where(torch.isfinite(y), y, 0.0).float().to(torch.float8_e4m3fn).double()      # (|y| <= 448: 24 bits hold y up to ties of inputs of at most 24 bits)
    q = torch.where(torch.isfinite(y), q, math.nan)
    return (q * s).reshape(x.shape)[:R, :Cc], e


def data(m, k, dtype, seed, odd=True):
    r = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=r) * torch.exp(2 * torch.randn(m, 1, generator=r)) * torch.exp(torch.randn(1, k, generator=r))
    if odd and m > 2 and k > 2:
        x[m // 2] = 0
        x[0, 0] = 0.0
        x[1, : k // 2] *= 2.0 ** -20
    return x.to(dtype)


def matrix(x, block_rows=1, transposed=False):
    return ops.quantize_fp8(x.cuda(), block_rows, transposed)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (3, 127), (128, 129), (129, 162), (81, 128), (257, 640), (130, 1025), (31, 64), (33, 3)])
def test_quantize_is_exact(m, k, dtype):
    x = data(m, k, dtype, 1)
    for rows in (1, 128):
        want, e = blocks(x, rows)
        q = matrix(x, rows)
        assert q.q.shape == (m, -(-k // 128) * 128) and q.scale.shape == (m, -(-k // 512) * 4)
        assert torch.equal(q.dequantize().double().cpu(), want)
        assert not q.q.view(torch.uint8)[:, k:].any()
        got = q.scale.view(torch.uint8).cpu().int() - 127
        assert torch.equal(got[:, :e.shape[1]], e.repeat_interleave(rows, 0)[:m].int())
        assert (got[:, e.shape[1]:] == 0).all()
        want, e = blocks(x.t() if rows == 1 else x, rows)
        t = matrix(x, rows, transposed=True)
        assert (t.rows, t.cols) == (k, m)
        assert torch.equal(t.dequantize().double().cpu(), want if rows == 1 else want.t())
        assert not t.q.view(torch.uint8)[:, m:].any()


@pytest.mark.gpu
def test_quantize_at_the_edges():
    """Largest and smallest numbers, ties, the border of a scale (448), zeros of both signs, NaN and infinities."""
    x = torch.zeros(12, 128)
    x[0, 0] = torch.finfo(torch.float32).max
    x[1, 0], x[1, 1] = 2.0 ** -149, -(2.0 ** -140)
    x[2] = torch.linspace(-448, 448, 128)
    x[3, 0], x[3, 1] = 448.0, 447.9
    x[4, 0], x[4, 1] = 448.00003, 1.0
    x[5] = torch.arange(128) / 16 + 1
    x[5, 0] = 256
    x[6, 0], x[6, 1], x[6, 2], x[6, 3] = math.nan, math.inf, -math.inf, 3.0
    x[7, 0] = -0.0
    x[8] = 2.0 ** -126 * torch.linspace(0, 1, 128)
    x[9, :4] = torch.tensor([300.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -11])       # ties below the normal numbers
    x[10] = math.nan
    x[11] = math.inf
    for rows in (1, 128):
        want, _ = blocks(x, rows)
        want = want.float().double()                  # (the largest float rounds to 256 * 2^120 = 2^128, which float32, the type of dequantize(), does not have: infinity)
        got = matrix(x, rows).dequantize().double().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(7), want.nan_to_num(7))


@pytest.mark.gpu
def test_quantize_strides_and_gate():
    for dtype in (torch.float32, torch.bfloat16):
        x = data(200, 300, dtype, 2)
        cut = x.cuda()[3:190, 5:271]
        want, _ = blocks(x[3:190, 5:271], 1)
        assert torch.equal(ops.quantize_fp8(cut).dequantize().double().cpu(), want)
        row = x.cuda()[7:8].expand(40, 300)
        want, _ = blocks(x[7:8].expand(40, 300), 1)
        assert torch.equal(ops.quantize_fp8(row).dequantize().double().cpu(), want)


def product_bound(a, b, want, extra, dtype, relu=False):
    """k products added in 32 bits in any order: at most k steps (2^-23: the matrix unit may cut off) of the sum of their sizes; one rounding to the result's type.
    A 16-bit result (without a relu) comes from the matrix unit's products of 8 bits, which it adds in groups of eight cut off at 2^-13 of the power of two below the
    largest: at most 8 * 2^-13 of the largest in each group, so at most 2^-10 of the sum of all sizes."""
    k = a.shape[1]
    cut = 0.0 if dtype == torch.float32 or relu else 2.0 ** -10
    return ((k + 2) * 2.0 ** -23 + cut) * (a.abs() @ b.abs().t() + extra) + HALF[dtype] * want.abs() * (1 + 1e-3) + 2.0 ** -126 + (2.0 ** -25 if dtype == torch.float16 else 0)


SHAPES = [(1, 1, 1), (1, 128, 128), (2, 81, 162), (16, 16, 128), (17, 33, 130), (64, 64, 64), (65, 63, 512), (128, 128, 128), (129, 257, 384), (300, 82, 162), (1, 1000, 1024), (5, 513, 640),
          (16, 2048, 1100), (33, 31, 2000), (1000, 100, 256), (255, 256, 1280), (256, 512, 515), (700, 300, 30), (2, 700, 9000), (100, 20, 20000)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product_against_64_bits(m, n, k):
    a, b = data(m, k, torch.float32, 3), data(n, k, torch.float32, 4, odd=False) / math.sqrt(k)
    qa, qb = matrix(a), matrix(b, 128)
    va, vb = blocks(a, 1)[0], blocks(b, 128)[0]
    bias = torch.randn(n, generator=torch.Generator().manual_seed(5))
    for dtype, bi, relu in ((torch.float32, None, False), (torch.bfloat16, bias, True), (torch.float16, bias.bfloat16(), False)):
        va_, vb_ = va, vb
        want = va_ @ vb_.t() + (0 if bi is None else bi.double())
        tol = product_bound(va_, vb_, want, 0 if bi is None else bi.double().abs(), dtype, relu)
        if relu:
            want = want.clamp(min=0)
        got = ops.matmul_fp8(qa, qb, None if bi is None else bi.cuda(), relu=relu, dtype=dtype)
        if dtype == torch.float16:                            # beyond its range: infinity
            fine = want.abs() < 6.5e4
            got, want, tol = got.cpu()[fine], want[fine], tol[fine]
        assert got.dtype == dtype and ((got.double().cpu() - want).abs() <= tol).all(), ((got.double().cpu() - want).abs() - tol).max()


@pytest.mark.gpu
def test_product_of_whole_numbers_is_exact():
    """Entries that 8 bits hold and sums that 32 bits hold: every order gives the same number, so a mistake of one product shows."""
    r = torch.Generator().manual_seed(6)
    for m, n, k in ((1, 300, 4096), (37, 45, 777), (128, 256, 1024), (513, 129, 256), (300, 260, 130), (16, 1024, 2048), (1024, 512, 128), (260, 520, 3000)):
        a = torch.randint(-8, 9, (m, k), generator=r).float()
        b = torch.randint(-8, 9, (n, k), generator=r).float()
        bias = torch.randint(-50, 50, (n,), generator=r).float()
        got = ops.matmul_fp8(matrix(a), matrix(b, 128), bias.cuda(), dtype=torch.float32)
        want = a.double() @ b.double().t() + bias.double()
        assert torch.equal(got.cpu().double(), want), (m, n, k)
        for t in (torch.bfloat16, torch.float16):             # (products of at most 2^6, in groups cut off at 2^-7: exact too)
            got = ops.matmul_fp8(matrix(a), matrix(b, 128), bias.cuda(), dtype=t)
            assert torch.equal(got.cpu(), want.float().to(t)), (m, n, k, t)


@pytest.mark.gpu
def test_every_block_has_its_scale():
    """Blocks of very different size: row i, block j scaled by powers of two of its own; exact again."""
    r = torch.Generator().manual_seed(7)
    for m, n, k in ((70, 50, 1300), (1, 200, 2600), (300, 300, 700)):
        kb = -(-k // 128)
        sa = torch.randint(-3, 4, (m, kb), generator=r).repeat_interleave(128, 1)[:, :k]
        sb = torch.randint(-3, 4, (-(-n // 128), kb), generator=r).repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
        a = torch.ldexp(torch.randint(-4, 5, (m, k), generator=r).float(), sa)
        b = torch.ldexp(torch.randint(-4, 5, (n, k), generator=r).float(), sb)
        got = ops.matmul_fp8(matrix(a), matrix(b, 128), dtype=torch.float32)
        want = a.double() @ b.double().t()
        assert torch.equal(got.cpu().double(), want), (m, n, k)
        got = ops.matmul_fp8(matrix(a), matrix(b, 128))
        assert ((got.cpu().double() - want).abs() <= HALF[torch.bfloat16] * want.abs()).all(), (m, n, k)     # (the scale is one for a group of eight)


@pytest.mark.gpu
def test_product_with_nan_and_nothing_to_sum():
    a, b = torch.ones(20, 200), torch.ones(30, 200)
    a[3, 150] = math.nan
    got = ops.matmul_fp8(matrix(a), matrix(b), relu=True, dtype=torch.float32).cpu()
    assert torch.isnan(got[3]).all() and (got[torch.arange(20) != 3] == 200).all()
    b[4, 2] = math.inf
    got = ops.matmul_fp8(matrix(a), matrix(b), dtype=torch.bfloat16).cpu()
    assert torch.isnan(got[:, 4]).all() and (got[0, :4] == 200).all()
    got = ops.matmul_fp8(matrix(torch.empty(3, 0)), matrix(torch.empty(4, 0)), torch.arange(4.0).cuda(), dtype=torch.float32)
    assert torch.equal(got.cpu(), torch.arange(4.0).expand(3, 4))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,relu", [(torch.float32, False), (torch.bfloat16, True), (torch.float16, True)])
@pytest.mark.parametrize("m,n,k", [(1, 8, 16), (5, 81, 128), (130, 128, 162), (257, 82, 512), (1000, 200, 90), (4000, 64, 72)])
def test_linear_and_its_gradients_against_64_bits(m, n, k, dtype, relu):
    x, w = data(m, k, dtype, 8), (data(n, k, torch.float32, 9, odd=False) / math.sqrt(k))
    bias, dy = torch.randn(n, generator=torch.Generator().manual_seed(1)), data(m, n, dtype, 10)
    lx, lw, lb = (t.cuda().requires_grad_() for t in (x, w, bias))
    y = ops.linear_fp8(lx, lw, lb, relu=relu)
    assert y.dtype == dtype and y.shape == (m, n)
    dx, dw, db = torch.autograd.grad([y], [lx, lw, lb], [dy.cuda()])
    assert dx.dtype == dtype and dw.dtype == torch.float32 and db.dtype == torch.float32
    d = dy.double()
    if relu:
        d = torch.where(y.detach().cpu() > 0, d, 0.0)
    vd, vdt, vw, vxt = blocks(d, 1)[0], blocks(d.t(), 1)[0], blocks(w, 128)[0], blocks(x.t().contiguous(), 1)[0]
    for got, p, q, t in ((dx, vd, vw.t(), dtype), (dw, vdt, vxt, torch.float32)):
        want = p @ q.t()
        tol = product_bound(p, q, want, 0, t)
        fine = want.abs() < (6.5e4 if t == torch.float16 else math.inf)
        assert ((got.cpu().double() - want).abs()[fine] <= tol[fine]).all()
    assert ((db.cpu().double() - d.sum(0)).abs() <= m * 2.0 ** -24 * d.abs().sum(0) + 1e-30).all()


@pytest.mark.gpu
def test_linear_gradients_are_the_differences_where_8_bits_are_exact():
    """Small whole numbers: the product is linear and exact, so gradients equal differences quotients (h = 1) exactly."""
    r = torch.Generator().manual_seed(2)
    m, n, k = 6, 5, 140
    x, w, b = (torch.randint(-6, 7, s, generator=r).float() for s in ((m, k), (n, k), (n,)))
    dy = torch.randint(-4, 5, (m, n), generator=r).float()
    lx, lw, lb = (t.cuda().requires_grad_() for t in (x, w, b))
    f = lambda x, w, b: (ops.linear_fp8(x.cuda(), w.cuda(), b.cuda()).cpu() * dy).sum().item()  # noqa: E731
    dx, dw, db = torch.autograd.grad([ops.linear_fp8(lx, lw, lb)], [lx, lw, lb], [dy.cuda()])
    for leaf, grad in ((0, dx), (1, dw), (2, db)):
        for _ in range(8):
            args = [x.clone(), w.clone(), b.clone()]
            at = tuple(int(torch.randint(0, d, (1,), generator=r)) for d in args[leaf].shape)
            before = f(*args)
            args[leaf][at] += 1
            assert f(*args) - before == grad[at].item(), (leaf, at)


@pytest.mark.gpu
def test_linear_forms():
    """More dimensions, weights laid out once, gradients of some arguments only, a weight in 16 bits, no rows."""
    x, w, b = data(24, 160, torch.bfloat16, 1).cuda().view(2, 3, 4, 160), data(48, 160, torch.float32, 2).cuda(), torch.randn(48, device="cuda")
    y = ops.linear_fp8(x, w, b, relu=True)
    assert y.shape == (2, 3, 4, 48)
    assert torch.equal(y, ops.linear_fp8(x, ops.Fp8Weight(w), b, relu=True))
    full = [t.detach().clone().requires_grad_() for t in (x, w, b)]
    g = torch.randn(2, 3, 4, 48, device="cuda").bfloat16()
    want = torch.autograd.grad([ops.linear_fp8(*full)], full, [g])
    for k in range(3):
        some = [t.detach().clone().requires_grad_(i == k) for i, t in enumerate((x, w, b))]
        got, = torch.autograd.grad([ops.linear_fp8(*some)], [some[k]], [g])
        assert torch.equal(got, want[k]), k
    half = w.bfloat16().requires_grad_()
    assert torch.autograd.grad(ops.linear_fp8(x, half).float().sum(), half)[0].dtype == torch.bfloat16
    none = torch.empty(0, 160, device="cuda", requires_grad=True)
    lw, lb = w.clone().requires_grad_(), b.clone().requires_grad_()
    y = ops.linear_fp8(none, lw, lb)
    dx, dw, db = torch.autograd.grad([y], [none, lw, lb], [torch.empty(0, 48, device="cuda")])
    assert y.shape == (0, 48) and dx.shape == (0, 160) and not dw.any() and not db.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_few_rows_on_ready_weights(dtype):
    """Up to 16 rows are held in 8 bits on the way: the same bits as in two steps, with rows of a wider tensor, NaN, infinities and zeros among them."""
    for m, n, k in ((1, 300, 1024), (2, 17, 5), (5, 33, 700), (16, 128, 130), (16, 64, 2049), (7, 1000, 128), (17, 40, 300), (3, 16, 31)):
        x = data(m, k + 3, dtype, 20)[:, 1:k + 1]
        if m > 4 and k > 600:
            x = x.clone()
            x[2, 600], x[3, 0], x[4, :128] = math.nan, -math.inf, 0.0
        w, b = data(n, k, torch.float32, 21), torch.randn(n, generator=torch.Generator().manual_seed(1)).cuda()
        ready = ops.Fp8Weight(w.cuda())
        wide = torch.zeros(m, k + 3, dtype=dtype, device="cuda")
        wide[:, 1:k + 1] = x.cuda()
        for relu in (False, True):
            got = ops.linear_fp8(wide[:, 1:k + 1], ready, b, relu=relu)
            want = ops.matmul_fp8(ops.quantize_fp8(x.cuda()), ready.matrix, b, relu=relu, dtype=dtype)
            assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(7), want.nan_to_num(7)), (m, n, k, relu)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_short_rows_in_one_launch(dtype):
    """Up to 512 columns and more than 16 rows, x held in 8 bits on the way: the same bits as in two steps at either side of the rule that takes it (rows, columns, a second
    tile of columns, four steps), with rows of a wider tensor, NaN, infinities, zeros and rows behind the last."""
    for m, n, k in ((17, 128, 128), (64, 129, 1), (65, 1, 7), (63, 300, 129), (200, 127, 256), (130, 256, 257), (1000, 82, 384), (129, 130, 511), (8192, 256, 512), (8256, 256, 512),
                    (20001, 128, 162), (66, 1030, 300), (32769, 260, 100)):
        x = data(m, k + 3, dtype, 22)[:, 1:k + 1]
        x[2, 0], x[3, k - 1], x[4, :] = math.nan, -math.inf, 0.0
        w, b = data(n, k, torch.float32, 23), torch.randn(n, generator=torch.Generator().manual_seed(2)).cuda()
        ready = ops.Fp8Weight(w.cuda())
        wide = torch.full((m, k + 3), math.nan, dtype=dtype, device="cuda")
        wide[:, 1:k + 1] = x.cuda()
        for relu in (False, True):
            got = ops.linear_fp8(wide[:, 1:k + 1], ready, b, relu=relu)
            want = ops.matmul_fp8(ops.quantize_fp8(x.cuda()), ready.matrix, b, relu=relu, dtype=dtype)
            assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(7), want.nan_to_num(7)), (m, n, k, relu)
            assert torch.equal(ops.linear_fp8(wide[:, 1:k + 1], w.cuda(), b, relu=relu).nan_to_num(7), want.nan_to_num(7)), (m, n, k, relu)
        leaf = wide[:, 1:k + 1].detach().requires_grad_()             # weights without a gradient
        y = ops.linear_fp8(leaf, w.cuda(), b)
        full = ops.linear_fp8(leaf, w.cuda().requires_grad_(), b)
        dy = torch.randn(m, n, device="cuda").to(dtype)
        assert torch.equal(y.nan_to_num(7), full.nan_to_num(7))
        assert torch.equal(torch.autograd.grad(y, leaf, dy)[0], torch.autograd.grad(full, leaf, dy)[0])


@pytest.mark.gpu
def test_another_stream_and_a_graph():
    def step(x, w, b, g):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = ops.linear_fp8(*leaves, relu=True)
        return [y.detach(), *torch.autograd.grad([y], leaves, [g])]

    for m, n, k in ((200, 96, 162), (1500, 64, 64)):
        sets = [[data(m, k, torch.bfloat16, s).cuda(), data(n, k, torch.float32, s + 1).cuda(), torch.randn(n, device="cuda"), data(m, n, torch.bfloat16, s + 2).cuda()] for s in (1, 5, 9)]
        eager = [step(*s) for s in sets]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step(*sets[0])
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(p, q) for p, q in zip(other, eager[0]))
        held = [v.clone() for v in sets[0]]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*held)
        for i in (1, 2, 0, 1):
            for v, s in zip(held, sets[i]):
                v.copy_(s)
            graph.replay()
            torch.cuda.synchronize()
            again = step(*sets[i])
            assert all(torch.equal(p, e) and torch.equal(q, e) for p, q, e in zip(out, again, eager[i]))


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """More than 2^32 entries: the last rows of a quantised matrix, of its transpose and of a result."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GiB of free device memory")
    m, k = 70000, 65536
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    tail = data(3, k, torch.bfloat16, 12)
    x[-3:] = tail.cuda()
    q = ops.quantize_fp8(x)
    want = blocks(tail, 1)[0]
    last = ops.Fp8Matrix.of(q.q[-3:].clone(), q.scale[-3:].clone(), 3, k)
    assert torch.equal(last.dequantize().double().cpu(), want) and not q.q[-9:-3].view(torch.uint8).any()
    t = ops.quantize_fp8(x, transposed=True)
    got = ops.Fp8Matrix.of(t.q[-3:].clone(), t.scale[-3:].clone(), 3, m).dequantize()[:, -3:].double().cpu()
    full = torch.zeros(3, 128)
    full[:, m % 128 - 3:m % 128] = tail[:, -3:].t().float()       # the last block along the rows
    assert torch.equal(got, blocks(full, 1)[0][:, m % 128 - 3:m % 128])
    del x, q, t
    r = torch.Generator().manual_seed(3)
    a, b = torch.randint(-4, 5, (m, 40), generator=r).float(), torch.randint(-4, 5, (k, 40), generator=r).float()
    out = ops.matmul_fp8(matrix(a), matrix(b))
    assert torch.equal(out[-300:].cpu().double(), (a[-300:].double() @ b.double().t()))
    assert torch.equal(out[:, -3:].cpu().double(), (a.double() @ b[-3:].double().t()))


@pytest.mark.gpu
def test_gradients_of_gradients_are_refused():
    x, w = torch.randn(4, 32, device="cuda", requires_grad=True), torch.randn(8, 32, device="cuda", requires_grad=True)
    dx, = torch.autograd.grad(ops.linear_fp8(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        dx.sum().backward()


@pytest.mark.gpu
def test_changed_results_are_noticed():
    """Behind a relu the result itself says where the gradient passes: changed in place, it is refused."""
    x, w = torch.randn(4, 32, device="cuda", requires_grad=True), torch.randn(8, 32, device="cuda")
    y = ops.linear_fp8(x, w, relu=True)
    z = (y * 2).sum()
    y.detach().add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    x, w = torch.randn(4, 64, device="cuda"), torch.randn(8, 64, device="cuda")
    q = matrix(x)
    assert torch.equal(ops.Fp8Matrix.of(q.q, q.scale, 4, 64).dequantize(), q.dequantize())
    for bad, match in ((lambda: ops.Fp8Matrix.of(q.q, q.scale, 5, 64), "q:"), (lambda: ops.Fp8Matrix.of(q.q, q.scale, 4, 129), "q:"), (lambda: ops.Fp8Matrix.of(q.q, q.scale[:, :3], 4, 64), "scale:"),
                       (lambda: ops.Fp8Matrix.of(q.q.view(torch.uint8), q.scale, 4, 64), "q:"), (lambda: ops.Fp8Matrix.of(q.q, q.scale.cpu(), 4, 64), "GPU"), (lambda: ops.quantize_fp8(x.double()), "float32"), (lambda: ops.quantize_fp8(x, 64), "block_rows"), (lambda: ops.quantize_fp8(x.t()), "next to each other"),
                       (lambda: ops.quantize_fp8(x[0]), "two dimensions"), (lambda: ops.matmul_fp8(x, w), "Fp8Matrix"),
                       (lambda: ops.matmul_fp8(matrix(x), matrix(w[:, :32].contiguous())), "columns"), (lambda: ops.matmul_fp8(matrix(x), matrix(w), dtype=torch.float64), "dtype"),
                       (lambda: ops.matmul_fp8(matrix(x), matrix(w), torch.randn(7, device="cuda")), "bias"), (lambda: ops.linear_fp8(x, w[:, :32]), "columns"),
                       (lambda: ops.linear_fp8(x, w.cpu()), "GPU"), (lambda: ops.linear_fp8(x.clone().requires_grad_(), ops.Fp8Weight(w)), "weights themselves")):
        with pytest.raises(ValueError, match=match):
            bad()


def test_refusals_without_a_gpu():
    with pytest.raises(ValueError, match="GPU"):
        ops.quantize_fp8(torch.randn(2, 3))
    with pytest.raises(ValueError, match="GPU"):
        ops.linear_fp8(torch.randn(2, 3), torch.randn(4, 3))
    L = lib.load_library()
    buf = (C.c_char * 4096)()
    at = (C.addressof(buf) + 63) // 64 * 64
    err = lambda: L.agz_ops_last_error().decode()  # noqa: E731
    ok = dict(x=at, dtype=0, rows=2, cols=4, ld=4, gate=None, br=1, q=at, s=at, qt=None, st=None, colsum=None, ws=None, n=0)
    for change, match in (({"dtype": 5}, "dtype"), ({"rows": -1}, "x"), ({"cols": 1 << 31}, "x"), ({"ld": -4}, "stride"), ({"br": 2}, "blocks"), ({"s": None}, "q with s"), ({"q": None, "s": None}, "q with s"),
                          ({"colsum": at}, "colsum"), ({"qt": at, "st": at, "colsum": at, "ws": at, "n": 4}, "colsum")):
        a = {**ok, **change}
        assert L.agz_fp8_quantize(0, None, *a.values()) == -1 and match in err(), (change, err())
    mm = dict(m=2, n=2, k=4, qa=at, sa=at, qb=at, sb=at, bias=None, bt=0, relu=0, out=at, ot=0, ldo=2, ws=None, wsn=0)
    for change, match in (({"m": -1}, "-1"), ({"k": 1 << 31}, "x"), ({"ot": 7}, "dtype"), ({"bias": at, "bt": 9}, "dtype")):
        a = {**mm, **change}
        assert L.agz_fp8_matmul(0, None, *a.values()) == -1 and match in err(), (change, err())
    lin = dict(m=2, n=2, k=4, x=at, ldx=4, w=at, ldw=4, bias=None, dtype=0, w_dtype=0, bias_dtype=0, relu=0)
    big = (C.c_char * 65536)()
    ws = (C.addressof(big) + 255) // 256 * 256
    fwd = lambda ch, y=at, saved=ws, dx=1, dw=1, w=ws, n=60000: L.agz_linear_fp8_forward(0, None, C.byref(lib.LinearFp8Args(**{**lin, **ch})), y, saved, dx, dw, w, n)  # noqa: E731
    bwd = lambda ch, dy=at, y=at, saved=ws, sdx=1, sdw=1, dx=at, dw=at, db=at, w=ws, n=60000: L.agz_linear_fp8_backward(  # noqa: E731
        0, None, C.byref(lib.LinearFp8Args(**{**lin, **ch})), dy, y, saved, sdx, sdw, dx, dw, db, w, n)
    for call, match in ((lambda: fwd({"m": -1}), "-1"), (lambda: fwd({"k": 1 << 24}), "x"), (lambda: fwd({"n": 65536 * 128}), "x"), (lambda: fwd({"dtype": 4}), "dtype"), (lambda: fwd({"w_dtype": -1}), "dtype"),
                        (lambda: fwd({"bias": at, "bias_dtype": 3}), "dtype"), (lambda: fwd({"ldw": -1}), "stride"), (lambda: fwd({"x": at + 2}), "aligned"), (lambda: fwd({"x": None}), "required"),
                        (lambda: fwd({}, y=None), "required"), (lambda: fwd({}, saved=None), "saved"), (lambda: fwd({}, n=10), "workspace"), (lambda: fwd({}, w=ws + 16), "workspace"),
                        (lambda: bwd({}, sdx=0), "did not save"), (lambda: bwd({}, sdw=0), "did not save"), (lambda: bwd({}, saved=None), "saved"), (lambda: bwd({}, dy=None), "required"),
                        (lambda: bwd({"relu": 1}, y=None), "required"), (lambda: bwd({}, n=0), "workspace"), (lambda: bwd({}, dx=at + 1), "aligned"), (lambda: bwd({"bias_dtype": 7}), "aligned")):
        assert call() == -1 and match in err(), err()
    app = lambda ch, qw=at, sw=at, y=at, w=ws, n=60000: L.agz_linear_fp8_apply(0, None, C.byref(lib.LinearFp8Args(**{**lin, **ch})), qw, sw, y, w, n)  # noqa: E731
    for call, match in ((lambda: app({"m": -1}), "-1"), (lambda: app({"dtype": 3}), "dtype"), (lambda: app({"x": None}), "required"), (lambda: app({}, qw=None), "required"), (lambda: app({}, sw=at + 1), "required"),
                        (lambda: app({}, y=at + 1), "required"), (lambda: app({"m": 20, "k": 600}, n=3), "workspace"), (lambda: app({"m": 20, "k": 600}, w=None), "workspace")):
        assert call() == -1 and match in err(), err()
    assert L.agz_linear_fp8_apply_workspace(1, -1, 1) < 0 and L.agz_linear_fp8_apply_workspace(16, 100, 100) == 0
    assert L.agz_linear_fp8_apply_workspace(20, 100, 100) == 0 and L.agz_linear_fp8_apply_workspace(20, 100, 600) > 0
    assert L.agz_linear_fp8_forward(0, None, None, None, None, 0, 0, None, 0) == -1
    assert L.agz_linear_fp8_workspace(-1, 1, 1) < 0 and L.agz_linear_fp8_saved(1, 1, -1, 1, 1) < 0 and L.agz_linear_fp8_backward_workspace(1, 1 << 31, 1, 1, 1, 1) < 0
    assert L.agz_linear_fp8_saved(5, 6, 7, 0, 0) == 0
    assert L.agz_fp8_pitch(-1) == -1 and L.agz_fp8_pitch(129) == 256 and L.agz_fp8_scale_pitch(129) == 4 and L.agz_fp8_scale_pitch(513) == 8
    assert L.agz_fp8_matmul_workspace(-1, 1, 1) < 0 and L.agz_fp8_colsum_ws(-1, 1) < 0


@pytest.mark.gpu
def test_forward_mode_derivatives_are_refused():
    """There is no forward-mode rule: a tangent of any argument is refused, never dropped; without one a level that is open changes nothing."""
    x, w, b = torch.randn(4, 64, device="cuda"), torch.randn(8, 64, device="cuda"), torch.randn(8, device="cuda")
    ready = ops.Fp8Weight(w)
    want = ops.linear_fp8(x, w, b)
    with fwd.dual_level():
        d, dw, db = (fwd.make_dual(t, torch.ones_like(t)) for t in (x, w, b))
        for bad in (lambda: ops.linear_fp8(d, w, b), lambda: ops.linear_fp8(x, dw, b), lambda: ops.linear_fp8(x, w, db), lambda: ops.linear_fp8(d, ready), lambda: ops.linear_fp8(x, ready, db),
                    lambda: ops.linear_fp8(d.view(2, 2, 64), w), lambda: ops.matmul_fp8(ops.quantize_fp8(x), ready.matrix, db)):
            with pytest.raises(ValueError, match="forward mode"):
                bad()
        assert torch.equal(ops.linear_fp8(x, w, b), want) and torch.equal(ops.linear_fp8(x, ready, b), want)


@pytest.mark.gpu
def test_a_product_without_gradients_refuses_a_bias_that_wants_one():
    x, w = matrix(torch.randn(4, 64)), matrix(torch.randn(8, 64), 128)
    b = torch.randn(8, device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="linear_fp8"):
        ops.matmul_fp8(x, w, b)
    want = ops.matmul_fp8(x, w, b.detach())
    with torch.no_grad():
        assert torch.equal(ops.matmul_fp8(x, w, b), want)


def test_an_empty_matrix_stands_for_no_values():
    for rows, cols in ((0, 128), (0, 0), (0, 5), (3, 0)):
        got = ops.Fp8Matrix(rows, cols, "cpu").dequantize()
        assert got.shape == (rows, cols) and got.dtype == torch.float32


@pytest.mark.gpu
def test_quantizing_nothing():
    for rows, cols in ((0, 128), (0, 0), (0, 5), (3, 0)):
        for block in (1, 128):
            x = torch.empty(rows, cols, device="cuda")
            assert ops.quantize_fp8(x, block).dequantize().shape == (rows, cols)
            assert ops.quantize_fp8(x, block, transposed=True).dequantize().shape == (cols, rows)


@pytest.mark.gpu
def test_more_dimensions_with_nothing_to_sum():
    """x [..., 0]: the bias alone, and gradients of nothing, with any number of dimensions."""
    b = torch.arange(4.0, device="cuda")
    for shape in ((2, 3, 0), (0,), (2, 0, 0), (5, 0)):
        x, w, lb = torch.empty(shape, device="cuda", requires_grad=True), torch.empty(4, 0, device="cuda", requires_grad=True), b.clone().requires_grad_()
        y = ops.linear_fp8(x, w, lb, relu=True)
        assert y.shape == (*shape[:-1], 4) and torch.equal(y, b.expand_as(y))
        assert torch.equal(ops.linear_fp8(x.detach(), ops.Fp8Weight(w.detach()), b), y)
        dx, dw, db = torch.autograd.grad([y], [x, w, lb], [torch.ones_like(y)])
        assert dx.shape == shape and dw.shape == (4, 0) and torch.equal(db, y.new_tensor([0.0, 1, 1, 1]) * (y.numel() // 4))


@pytest.mark.gpu
def test_a_product_that_is_too_deep_is_refused_by_name():
    q = ops.quantize_fp8(torch.zeros(1, 1 << 24, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError, match="too large"):
        ops.matmul_fp8(q, q)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("block", [1, 128])
def test_gate_and_column_sums(block, dtype):
    """agz_fp8_quantize with a gate and column sums, both ways and each way alone: entries behind a gate that is not above 0 (NaN is not) count as 0, whatever they are; sums of what is
    left, rows x half a step of 32 bits of the sum of their sizes off at most; few columns, odd ends, rows of a wider tensor."""
    L = lib.load_library()
    for rows, cols in ((1, 1), (3, 5), (130, 7), (128, 128), (129, 131), (300, 515), (40, 8)):
        x, gate = data(rows, cols, dtype, 30), torch.randn(rows, cols, generator=torch.Generator().manual_seed(31)).to(dtype)
        gate[0, 0] = math.nan
        if rows > 2:
            gate[2, cols - 1], gate[1, 0], x[2, cols - 1], x[1, 0] = -1.0, 0.0, math.nan, math.inf      # (closed, with NaN and infinity behind)
        wide = torch.full((2, rows, cols + 3), math.nan, dtype=dtype, device="cuda")
        wide[0, :, 1:cols + 1], wide[1, :, 1:cols + 1] = x.cuda(), gate.cuda()
        xs, gs = wide[0, :, 1:cols + 1], wide[1, :, 1:cols + 1]
        passed = torch.where(gate > 0, x, torch.zeros_like(x))
        straight = blocks(passed, block)[0]
        across = blocks(passed.t(), 1)[0] if block == 1 else straight.t()
        for both in ((True, True), (True, False), (False, True)):
            a, t = ops.Fp8Matrix(rows, cols, "cuda") if both[0] else None, ops.Fp8Matrix(cols, rows, "cuda") if both[1] else None
            sums = torch.full((cols,), math.nan, device="cuda") if both[1] else None
            ws = torch.empty(L.agz_fp8_colsum_ws(rows, cols), dtype=torch.uint8, device="cuda")
            at = lambda m, k: getattr(m, k).data_ptr() if m is not None else None  # noqa: E731
            rc = L.agz_fp8_quantize(0, torch.cuda.current_stream().cuda_stream, xs.data_ptr(), ops._CODE[dtype], rows, cols, cols + 3, gs.data_ptr(), block,
                                    at(a, "q"), at(a, "scale"), at(t, "q"), at(t, "scale"), sums.data_ptr() if both[1] else None, ws.data_ptr(), ws.numel())
            assert rc == 0, L.agz_ops_last_error()
            if both[0]:
                assert torch.equal(a.dequantize().double().cpu(), straight) and not a.q.view(torch.uint8)[:, cols:].any()
            if both[1]:
                assert torch.equal(t.dequantize().double().cpu(), across) and not t.q.view(torch.uint8)[:, rows:].any()
                d = passed.double()
                assert ((sums.double().cpu() - d.sum(0)).abs() <= rows * 2.0 ** -24 * d.abs().sum(0)).all()
