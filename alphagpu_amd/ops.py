"""Operators on device tensors: what a network learns with (include/agz.h "operators on tensors in DEVICE memory").

    log_probs(logits, moves, ...)            log probabilities of given moves, entropy, best alternatives, expected log probability; differentiable
    linear_fp8                               a layer with its product in 8 bits, a scale for each block of 128; differentiable
    quantize_fp8, matmul_fp8                 matrices in 8 bits and their products by themselves; without gradients
    AdamW                                    one step over many tensors, states in 32 or 8 bits

The reference does this in Flux (train.jl:12-15, :50; DenseNet.jl:161-198).  Tensors are torch tensors on a GPU; the work runs on the current
stream of their device, nothing waits for it, and it can be captured into a graph.  Wrong arguments raise ValueError before anything is
queued, errors of the library AgzError.  There is no CPU path, and no forward-mode rule (a tangent is refused).  A backward pass that is captured into a graph needs leaves of its own
(detach().requires_grad_(), and autograd.grad): gradients that another, living autograd graph accumulates into the same leaves are torch's to order.
"""
import ctypes as C
import functools
import math
import struct
from collections import namedtuple

import torch
import torch.autograd.forward_ad as _forward_ad
from torch._C import _cuda_getCurrentRawStream as _raw_stream     # the current stream's handle without a Stream object around it
from torch._C import _cuda_isCurrentStreamCapturing as _capturing

from . import lib as _lib

_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
TOP_MAX = 32
FP8, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _lib_call(rc, L):
    if rc != 0:
        raise _lib.AgzError(rc, L.agz_ops_last_error().decode())


def _need(ok, text):
    if not ok:
        raise ValueError(text)


def _on_gpu(t, name, device=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name}: a tensor on a GPU is needed (there is no CPU path)")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the others on {device}")


def _float_type(t, name):
    if t.dtype not in _CODE:
        raise ValueError(f"{name}: float32, bfloat16 or float16, not {t.dtype}")


def _rows(t, name):
    """[rows][cols] with the columns next to each other; the row stride."""
    if t.dim() != 2:
        raise ValueError(f"{name}: two dimensions are needed, not {t.dim()}")
    if t.shape[1] > 1 and t.stride(1) != 1 and t.numel():
        raise ValueError(f"{name}: the columns of a row have to lie next to each other (stride {t.stride(1)}): use contiguous()")
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def _no_tangent(**tensors):
    """Refuses tensors that carry a forward-mode derivative (called where a level is open)."""
    for name, t in tensors.items():
        if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f"{name}: no derivatives in forward mode (give the primal, without a tangent)")


def _ptr(t):
    return None if t is None else t.data_ptr()


# ---------------------------------------------------------------------------------------------------------------------------------------
# log probabilities
# ---------------------------------------------------------------------------------------------------------------------------------------
LogProbs = namedtuple("LogProbs", "move entropy target top top_move")


# agz_logprob_args as bytes (a ctypes.Structure takes several times as long to fill)
_LP = struct.Struct("=qqqqii13q")
assert _LP.size == C.sizeof(_lib.LogProbArgs)


def _log_probs_head(logits, moves, mask, target, top):
    """The first fields of agz_logprob_args: sizes, pointers, row strides."""
    ld = _rows(logits, "logits")
    n, a = logits.shape
    mask_at = mask_ld = target_at = target_ld = 0
    if mask is not None:
        mask_ld, mask_at = _rows(mask, "mask"), mask.data_ptr()
        if mask.shape[0] == 1:
            mask_ld = 0
    if target is not None:
        target_ld, target_at = _rows(target, "target"), target.data_ptr()
    return n, a, logits.data_ptr(), ld, _CODE[logits.dtype], top, mask_at, mask_ld, 0 if moves is None else moves.data_ptr(), target_at, target_ld


def _log_probs_forward(logits, head, moves, target, top, stats):
    """head: the inputs, checked and packed -> move, entropy, target, top, top_move; stats [n, 4] (None: not wanted): what the backward pass reads."""
    n, a = logits.shape
    dev, f32 = logits.device, torch.float32
    entropy = torch.empty(n, dtype=f32, device=dev)
    move = None if moves is None else torch.empty(n, dtype=f32, device=dev)
    expected = None if target is None else torch.empty(n, dtype=f32, device=dev)
    tops = top_move = None
    if top:
        tops, top_move = torch.empty(n, top, dtype=f32, device=dev), torch.empty(n, top, dtype=torch.int32, device=dev)
    L, need, ws = _lib.load_library(), 0, None
    if a > 1024:                                             # (shorter rows need no workspace)
        need = L.agz_logprob_workspace(n, a, top)
        if need < 0:
            raise ValueError(f"logits: {n} rows of {a} actions are too many")
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
    q = _LP.pack(*head, 0 if move is None else move.data_ptr(), entropy.data_ptr(), 0 if expected is None else expected.data_ptr(),
                 tops.data_ptr() if top else 0, top_move.data_ptr() if top else 0, 0 if stats is None else stats.data_ptr(), ws.data_ptr() if need else 0, need)
    i = dev.index
    rc = L.agz_logprob_forward(i, _raw_stream(i), q)
    if rc:
        _lib_call(rc, L)
    return move, entropy, expected, tops, top_move


def _log_probs_backward(ctx, g_move, g_entropy, g_target, g_top, _):
    logits, stats, top_move, moves, mask, target = ctx.saved_tensors
    head = ctx.head
    if head != (now := _log_probs_head(logits, moves, mask, target, head[5])):      # (hooks on saved tensors may give back copies of them)
        head = now
    g = [None if x is None else x.contiguous() for x in (g_move, g_entropy, g_target, g_top)]     # (held here until the call is queued)
    dx = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    L, i = _lib.load_library(), logits.get_device()
    rc = L.agz_logprob_backward(i, _raw_stream(i), _LP.pack(*head, 0, 0, 0, 0, 0 if top_move is None else top_move.data_ptr(), stats.data_ptr(), 0, 0),
                                _ptr(g[0]), _ptr(g[1]), _ptr(g[2]), _ptr(g[3]), dx.data_ptr(), head[1])
    if rc:
        _lib_call(rc, L)
    return dx, None, None


class _LogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, head, rest):
        moves, mask, target, top = rest
        stats = torch.empty(logits.shape[0], 4, dtype=torch.float32, device=logits.device)
        out = _log_probs_forward(logits, head, moves, target, top, stats)
        ctx.set_materialize_grads(False)
        ctx.head = head
        ctx.save_for_backward(logits, stats, out[4], moves, mask, target)
        if top:
            ctx.mark_non_differentiable(out[4])
        return out

    @staticmethod
    def backward(ctx, *g):
        if g[0] is None and g[1] is None and g[2] is None and g[3] is None:
            return None, None, None
        # a backward pass that is recorded itself (create_graph): its own gradient is refused where it is asked for
        return (_LogProbs._once if torch.is_grad_enabled() else _log_probs_backward)(ctx, *g)

    _once = staticmethod(torch.autograd.function.once_differentiable(_log_probs_backward))


def log_probs(logits, moves=None, mask=None, target=None, top=0):
    """Log probabilities of moves under rows of logits [n, a] (float32, bfloat16 or float16) -> LogProbs of float32 tensors:

        move      [n]       of the given `moves` (whole numbers [n]; 0 where the move is < 0 or >= a: none given; -inf where it is not allowed)
        entropy   [n]       of the distribution
        target    [n]       sum_j target_j logp_j: minus the cross entropy against `target` [n, a] (float32; a constant for the gradient)
        top       [n, top]  of the `top` (at most 32) most probable moves, most probable first, equal logits by index
        top_move  [n, top]  those moves (int32; -1, with -inf, where fewer are allowed)

    None for what was not asked for.  `mask` (bool or uint8; [n, a], or [1, a] / [a] for all rows): the moves that are allowed; a logit of -inf
    is not allowed either.  A row without an allowed move has entropy 0 and gradient 0; a row with NaN or +inf among the allowed is NaN.
    Differentiable in the logits through move, entropy, target and top."""
    _on_gpu(logits, "logits")
    if logits.dtype not in _CODE:
        _float_type(logits, "logits")
    if logits.dim() != 2:
        _rows(logits, "logits")
    n, a = logits.shape
    dev = logits.device
    if not 1 <= a <= 1 << 30:
        raise ValueError(f"logits: {a} actions (1 to 2^30)")
    if not (isinstance(top, int) and 0 <= top <= TOP_MAX and top <= a):
        raise ValueError(f"top: 0 to {TOP_MAX} and at most the number of actions, not {top!r}")
    if moves is not None:
        _on_gpu(moves, "moves", dev)
        if moves.shape != (n,) or moves.dtype not in (torch.int64, torch.int32):
            raise ValueError(f"moves: int64 or int32 [{n}], not {moves.dtype} {list(moves.shape)}")
        if moves.dtype != torch.int64 or not moves.is_contiguous():
            moves = moves.long().contiguous()
    if mask is not None:
        _on_gpu(mask, "mask", dev)
        if mask.dtype not in (torch.bool, torch.uint8):
            raise ValueError(f"mask: bool or uint8, not {mask.dtype}")
        if mask.dim() == 1:
            mask = mask[None]
        if mask.shape != (n, a) and mask.shape != (1, a):
            raise ValueError(f"mask: [{n}, {a}], [1, {a}] or [{a}], not {list(mask.shape)}")
    if target is not None:
        _on_gpu(target, "target", dev)
        if target.dtype != torch.float32 or target.shape != (n, a):
            raise ValueError(f"target: float32 [{n}, {a}], not {target.dtype} {list(target.shape)}")
        if target.requires_grad:
            raise ValueError("target: a constant is needed (detach() it)")
    if _forward_ad._current_level >= 0:
        _no_tangent(logits=logits, target=target)
    head = _log_probs_head(logits, moves, mask, target, top)
    if logits.requires_grad and torch.is_grad_enabled():
        return LogProbs(*_LogProbs.apply(logits, head, (moves, mask, target, top)))
    return LogProbs(*_log_probs_forward(logits, head, moves, target, top, None))


# ---------------------------------------------------------------------------------------------------------------------------------------
# products in 8 bits
# ---------------------------------------------------------------------------------------------------------------------------------------
class Fp8Matrix:
    """A matrix [rows, cols] in 8 bits: q [rows, cols rounded up to 128] (float8_e4m3fn; zeros behind cols) and scale [rows, blocks of 128
    columns rounded up to 4] (float8_e8m0fnu).  Entry (i, j) is q[i, j] * scale[i, j // 128]."""
    __slots__ = ("q", "scale", "rows", "cols")

    def __init__(self, rows, cols, device):
        self.rows, self.cols = rows, cols
        self.q = torch.empty((rows, -(-cols // 128) * 128), dtype=FP8, device=device)
        self.scale = torch.empty((rows, -(-cols // 512) * 4), dtype=E8M0, device=device)

    def dequantize(self):
        """The values it stands for, in float32."""
        pitch = self.q.shape[1]
        s = self.scale.float()[:, :pitch // 128]
        return (self.q.float().view(self.rows, pitch // 128, 128) * s[:, :, None]).view(self.rows, pitch)[:, :self.cols]

    @classmethod
    def of(cls, q, scale, rows, cols):
        """From tensors that are laid out as above already (no scale of NaN)."""
        for t, name, shape, kind in ((q, "q", (rows, -(-cols // 128) * 128), FP8), (scale, "scale", (rows, -(-cols // 512) * 4), E8M0)):
            _on_gpu(t, name, q.device)
            _need(t.shape == shape and t.dtype == kind and t.is_contiguous() and t.data_ptr() % 16 == 0, f"{name}: {kind} {list(shape)}, contiguous and aligned to 16 bytes, is needed, not {t.dtype} {list(t.shape)}")
        m = cls.__new__(cls)
        m.q, m.scale, m.rows, m.cols = q, scale, rows, cols
        return m


def quantize_fp8(x, block_rows=1, transposed=False):
    """x [rows, cols] (float32, bfloat16 or float16) -> Fp8Matrix, of x or (transposed) of its transpose, with one scale per block of
    block_rows (1, or 128 for weights) x 128 along the columns of the result.  Scales are the smallest powers of two with |x| <= 448 scale; NaN
    and infinities become NaN.  No gradient passes: what is held in 8 bits is a constant."""
    _on_gpu(x, "x")
    _float_type(x, "x")
    _need(block_rows in (1, 128), f"block_rows: 1 or 128, not {block_rows!r}")
    L, dev, ld = _lib.load_library(), x.device, _rows(x, "x")
    r, c = x.shape
    q = Fp8Matrix(c, r, dev) if transposed else Fp8Matrix(r, c, dev)
    at = (q.q.data_ptr(), q.scale.data_ptr())
    _lib_call(L.agz_fp8_quantize(dev.index, _raw_stream(dev.index), x.data_ptr(), _CODE[x.dtype], r, c, ld, None, block_rows,
                                 *((None, None, *at) if transposed else (*at, None, None)), None, None, 0), L)
    return q


def _product(a, b, bias, relu, dtype):
    L = _lib.load_library()
    dev = a.q.device
    need = L.agz_fp8_matmul_workspace(a.rows, b.rows, a.cols)
    if need < 0:
        raise ValueError(f"matmul_fp8: {a.rows} x {b.rows} x {a.cols} is too large")
    out = torch.empty((a.rows, b.rows), dtype=dtype, device=dev)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _lib_call(L.agz_fp8_matmul(dev.index, _raw_stream(dev.index), a.rows, b.rows, a.cols, a.q.data_ptr(), a.scale.data_ptr(), b.q.data_ptr(), b.scale.data_ptr(),
                               _ptr(bias), 0 if bias is None else _CODE[bias.dtype], int(relu), out.data_ptr(), _CODE[dtype], max(b.rows, 1), _ptr(ws), need), L)
    return out


def _check_bias(bias, n, dev):
    if bias is not None:
        _on_gpu(bias, "bias", dev)
        _float_type(bias, "bias")
        if bias.shape != (n,) or (n > 1 and bias.stride(0) != 1):
            raise ValueError(f"bias: [{n}], contiguous, not {list(bias.shape)}")


def matmul_fp8(a, b, bias=None, relu=False, dtype=torch.bfloat16):
    """relu?(a b^T + bias) of two Fp8Matrix with the same number of columns: [a.rows, b.rows] in `dtype`; sums in 32 bits, rounded once.
    No gradient passes, so a bias that wants one is refused (linear_fp8 has one)."""
    _need(isinstance(a, Fp8Matrix) and isinstance(b, Fp8Matrix), "a and b: Fp8Matrix (quantize_fp8) are needed")
    _need(a.cols == b.cols, f"a has {a.cols} columns, b {b.cols}")
    _need(a.q.device == b.q.device, "a and b are on different devices")
    _need(dtype in _CODE, f"dtype: float32, bfloat16 or float16, not {dtype}")
    _check_bias(bias, b.rows, a.q.device)
    _need(bias is None or not (bias.requires_grad and torch.is_grad_enabled()), "bias: a constant is needed (detach() it; linear_fp8 has gradients)")
    if _forward_ad._current_level >= 0:
        _no_tangent(bias=bias)
    with torch.no_grad():
        return _product(a, b, None if bias is None else bias.detach(), relu, dtype)


class Fp8Weight:
    """Weights [out, in] laid out once for linear_fp8 calls that need no gradient of them."""
    __slots__ = ("matrix",)

    def __init__(self, w):
        self.matrix = quantize_fp8(w, block_rows=128)


_LIN = struct.Struct("=qqqqqqqqiiii")               # agz_linear_fp8_args
assert _LIN.size == C.sizeof(_lib.LinearFp8Args)


@functools.lru_cache(maxsize=4096)
def _linear_sizes(m, n, k, need_x, need_w, need_b):
    """Bytes of (the forward call's workspace, what it saves, the backward call's workspace) of a product of this size."""
    L = _lib.load_library()
    sizes = L.agz_linear_fp8_workspace(m, n, k), L.agz_linear_fp8_saved(m, n, k, need_x, need_w), L.agz_linear_fp8_backward_workspace(m, n, k, need_x, need_w, need_b)
    if min(sizes) < 0:
        raise ValueError(f"linear_fp8: {m} x {n} x {k} is too large")
    return sizes


def _linear_forward(x, w, bias, relu, need_x, need_w, need_b):
    (m, k), n, dev = x.shape, w.shape[0], x.device
    need, keep, _ = _linear_sizes(m, n, k, need_x, need_w, need_b)
    y = torch.empty(m, n, dtype=x.dtype, device=dev)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    saved = torch.empty(keep, dtype=torch.uint8, device=dev) if need_x or need_w else None
    q = _LIN.pack(m, n, k, x.data_ptr(), _rows(x, "x"), w.data_ptr(), _rows(w, "w"), 0 if bias is None else bias.data_ptr(),
                  _CODE[x.dtype], _CODE[w.dtype], 0 if bias is None else _CODE[bias.dtype], relu)
    L, i = _lib.load_library(), dev.index
    rc = L.agz_linear_fp8_forward(i, _raw_stream(i), q, y.data_ptr(), _ptr(saved), need_x, need_w, ws.data_ptr(), need)
    if rc:
        _lib_call(rc, L)
    return y, saved, q


def _linear_apply(x, w, bias, relu):
    L = _lib.load_library()
    (m, k), n, dev, i = x.shape, w.rows, x.device, x.get_device()
    y = torch.empty(m, n, dtype=x.dtype, device=dev)
    need = L.agz_linear_fp8_apply_workspace(m, n, k)
    if need < 0:
        raise ValueError(f"linear_fp8: {m} x {n} x {k} is too large")
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    q = _LIN.pack(m, n, k, x.data_ptr(), _rows(x, "x"), 0, 0, 0 if bias is None else bias.data_ptr(), _CODE[x.dtype], 0, 0 if bias is None else _CODE[bias.dtype], relu)
    rc = L.agz_linear_fp8_apply(i, _raw_stream(i), q, w.q.data_ptr(), w.scale.data_ptr(), y.data_ptr(), _ptr(ws), need)
    if rc:
        _lib_call(rc, L)
    return y


def _linear_backward(ctx, dy):
    saved, y = ctx.saved_tensors
    need_x, need_w, need_b = need_grad = ctx.needs_input_grad[:3]
    (m, n, k), w_type, b_type, q, kept = ctx.call
    dev = dy.device
    dy = dy.contiguous()
    dx = torch.empty(m, k, dtype=dy.dtype, device=dev) if need_x else None
    dw = torch.empty(n, k, dtype=w_type, device=dev) if need_w else None
    db = torch.empty(n, dtype=b_type, device=dev) if need_b else None
    need = _linear_sizes(m, n, k, *need_grad)[2]
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    L, i = _lib.load_library(), dev.index
    rc = L.agz_linear_fp8_backward(i, _raw_stream(i), q, dy.data_ptr(), _ptr(y), _ptr(saved), kept[0], kept[1], _ptr(dx), _ptr(dw), _ptr(db), ws.data_ptr(), need)
    if rc:
        _lib_call(rc, L)
    return dx, dw, db, None


class _LinearFp8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, relu):
        need = ctx.needs_input_grad[:3]
        y, saved, q = _linear_forward(x, w, bias, relu, *need)
        ctx.call = (x.shape[0], *w.shape), w.dtype, None if bias is None else bias.dtype, q, need
        ctx.save_for_backward(saved, y if relu else None)
        return y

    @staticmethod
    def backward(ctx, dy):
        return (_LinearFp8._once if torch.is_grad_enabled() else _linear_backward)(ctx, dy)

    _once = staticmethod(torch.autograd.function.once_differentiable(_linear_backward))


def linear_fp8(x, w, bias=None, relu=False):
    """relu?(x w^T + bias) with x [..., in] and w [out, in] held in 8 bits for the product: x in blocks of 1 x 128, w in blocks of 128 x 128.
    The result has the type of x.  w: a tensor (float32, bfloat16 or float16; quantised in the call), or Fp8Weight.  Differentiable in x, w and bias:
    dx = dy w and dw = dy^T x are products in 8 bits too (dy in blocks of 1 x 128 along what is summed over), dbias sums in 32 bits."""
    _on_gpu(x, "x")
    _float_type(x, "x")
    dev = x.device
    _need(x.dim() >= 1, "x: at least one dimension is needed")
    ready = isinstance(w, Fp8Weight)
    if ready:
        n, k = w.matrix.rows, w.matrix.cols
        _need(w.matrix.q.device == dev, f"w is on {w.matrix.q.device}, x on {dev}")
    else:
        _on_gpu(w, "w", dev)
        _float_type(w, "w")
        _rows(w, "w")
        n, k = w.shape
    if x.shape[-1] != k:
        raise ValueError(f"x has {x.shape[-1]} columns, w {k}")
    _check_bias(bias, n, dev)
    if _forward_ad._current_level >= 0:
        _no_tangent(x=x, w=None if ready else w, bias=bias)
    two = x if x.dim() == 2 else x.reshape(math.prod(x.shape[:-1]), k)
    _rows(two, "x")
    if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad) or (not ready and w.requires_grad)):
        _need(not ready, "w: gradients need the weights themselves, not Fp8Weight")
        y = _LinearFp8.apply(two, w, bias, bool(relu))
    elif ready:
        y = _linear_apply(two, w.matrix, bias, bool(relu))
    else:
        y = _linear_forward(two, w, bias, bool(relu), False, False, False)[0]
    return y if x.dim() == 2 else y.view(*x.shape[:-1], n)


# ---------------------------------------------------------------------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------------------------------------------------------------------
_ADAMW = struct.Struct("=dddddiiiIi4xqq")           # agz_adamw_options
assert _ADAMW.size == C.sizeof(_lib.AdamWOptions)


def _check_adamw(lr, betas, eps, weight_decay):
    if not (lr >= 0 and eps >= 0 and weight_decay >= 0 and len(betas) == 2 and all(0 <= b < 1 for b in betas)):
        raise ValueError(f"lr, eps, weight_decay >= 0 and two betas in [0, 1) are needed, not {lr}, {eps}, {weight_decay}, {betas}")


class AdamW:
    """AdamW (decoupled weight decay) over many tensors in one launch, in place:

        m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  p = p (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    t is the number of steps that a tensor has taken: those in which it has no gradient are not among them, and leave it as it is.

    params: contiguous tensors of one type on one device that do not overlap.  bits = 32: states m, v in float32.  bits = 8: m and r = sqrt(v) in
    float8_e4m3fn with one power-of-two scale per 128 elements, rounded up or down at random in proportion (from `seed`, the step and the
    element: equal calls give equal results; the mean of r^2 gains the variance of that, about 4 % of v under normal gradients, more for entries far below the others
    of their block).  The states of all tensors lie in the buffers m, v (or m, m_scale, r, r_scale), tensor i from element offsets[i] on.
    capturable: the number of the step is kept on the device, so that a step captured into a graph counts on in its replays (with the lr, betas, eps
    and weight_decay it was captured with)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, bits=32, seed=0, capturable=False):
        self.params = list(params)
        _need(self.params, "params: none")
        _need(bits in (8, 32), f"bits: 8 or 32, not {bits!r}")
        self._options = None
        _check_adamw(lr, betas, eps, weight_decay)
        dev, kind, ends = self.params[0].device if isinstance(self.params[0], torch.Tensor) else None, None, []
        for i, p in enumerate(self.params):
            _on_gpu(p, f"params[{i}]", dev)
            _float_type(p, f"params[{i}]")
            kind = kind or p.dtype
            _need(p.dtype == kind, f"params[{i}] is {p.dtype}, the first {kind}: one AdamW for each type")
            _need(p.is_contiguous(), f"params[{i}] is not contiguous")
            if p.numel():
                ends.append((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size(), i))
        ends.sort()
        for (_, end, i), (start, _, j) in zip(ends, ends[1:]):
            _need(end <= start, f"params[{i}] and params[{j}] overlap")
        self.device, self.dtype, self.lr, self.betas, self.eps, self.weight_decay, self.bits, self.seed = dev, kind, lr, tuple(betas), eps, weight_decay, bits, int(seed)
        count = len(self.params)
        self._numel, self._pointers, self._shapes = (C.c_int64 * count)(*[p.numel() for p in self.params]), struct.Struct(f"={count}q"), [p.shape for p in self.params]
        self.offsets, at = [], 0
        for p in self.params:
            self.offsets.append(at)
            at += -(-p.numel() // 128) * 128
        if bits == 32:
            self.m, self.v = (torch.zeros(at, dtype=torch.float32, device=dev) for _ in range(2))
        else:
            self.m, self.r = (torch.zeros(at, dtype=torch.uint8, device=dev).view(FP8) for _ in range(2))
            self.m_scale, self.r_scale = (torch.full((at // 128,), 127, dtype=torch.uint8, device=dev).view(E8M0) for _ in range(2))
        self.steps = 0                                       # calls; a tensor's own steps are these less the ones that it missed
        self._missed, self._any_missed = (C.c_int64 * count)(), False
        self.step_dev = torch.zeros((), dtype=torch.int64, device=dev) if capturable else None
        self._missed_dev = torch.zeros(count, dtype=torch.int64, device=dev) if capturable else None

    def _buffers(self):
        return ("m", "v") if self.bits == 32 else ("m", "m_scale", "r", "r_scale")

    def state(self):
        """{"step": steps taken, "missed": how many of them each tensor missed, and the buffers of the states}: copies, for load_state."""
        step, missed = (self.steps, list(self._missed)) if self.step_dev is None else (int(self.step_dev.item()), self._missed_dev.tolist())
        return {"step": step, "missed": missed, **{k: getattr(self, k).clone() for k in self._buffers()}}

    def load_state(self, state):
        """What state() returned, of this or an equal optimiser; without "missed" no tensor has missed a step."""
        step, missed = int(state["step"]), [int(k) for k in state.get("missed", [0] * len(self.params))]
        _need(step >= 0 and len(missed) == len(self.params) and all(0 <= k <= step for k in missed), f"load_state: step {step}, and as many numbers of missed steps, at most {step}, as tensors ({len(self.params)})")
        for k in self._buffers():
            mine = getattr(self, k)
            _need(k in state and state[k].shape == mine.shape and state[k].dtype == mine.dtype, f"load_state: {k} has to be {mine.dtype} {list(mine.shape)}")
        for k in self._buffers():
            getattr(self, k).view(torch.uint8).copy_(state[k].view(torch.uint8))
        self.steps, self._missed[:], self._any_missed = step, missed, any(missed)
        if self.step_dev is not None:
            self.step_dev.fill_(step)
            self._missed_dev.copy_(torch.tensor(missed, dtype=torch.int64))

    def zero_grad(self):
        for p in self.params:
            p.grad = None

    def step(self, grads=None):
        """One step with `grads` (one per tensor, of one type; None: p.grad).  A tensor whose gradient is None is left as it is and misses the step."""
        params = self.params
        grads = [p.grad for p in params] if grads is None else list(grads)
        if len(grads) != len(params):
            raise ValueError(f"{len(grads)} gradients for {len(params)} tensors")
        options = (self.lr, self.betas, self.eps, self.weight_decay)
        if options != self._options:                         # (changed since they were last looked at)
            _check_adamw(*options)
            self._options = (float(self.lr), tuple(float(b) for b in self.betas), float(self.eps), float(self.weight_decay))      # (values: a list may change in place)
        kind, own, device, at = None, self.dtype, self.device.index, []
        for i, (p, g, shape) in enumerate(zip(params, grads, self._shapes)):
            if p.shape != shape or p.get_device() != device or p.dtype is not own or not p.is_contiguous():
                raise ValueError(f"params[{i}] has changed its shape, type or device")
            if g is None:
                at.append(0)
                continue
            if g.get_device() != device:
                raise ValueError(f"grads[{i}] is on {g.device}, the tensors on {self.device}")
            if g.dtype is not kind:
                if kind is not None or g.dtype not in _CODE:
                    raise ValueError(f"grads[{i}] is {g.dtype}: one of float32, bfloat16, float16 for all")
                kind = g.dtype
            if g.shape != shape:
                raise ValueError(f"grads[{i}] is {list(g.shape)}, the tensor {list(shape)}")
            if not g.is_contiguous():
                g = grads[i] = g.contiguous()
            at.append(g.data_ptr())
        missed = missed_dev = None
        if self.step_dev is None:
            if _capturing():
                raise RuntimeError("AdamW.step in a graph: capturable=True is needed (a replay has to count its step on the device)")
            counter = 0
            if self._any_missed:
                missed = C.addressof(self._missed)
        else:
            counter, missed_dev = self.step_dev.data_ptr(), self._missed_dev.data_ptr()
        t = self.steps + 1
        o = _ADAMW.pack(self.lr, *self.betas, self.eps, self.weight_decay, _CODE[own], _CODE[kind or torch.float32], self.bits, self.seed & 0xFFFFFFFF, 0, t, counter)
        if counter:
            self.step_dev.add_(1)                            # (behind everything that can refuse the call)
        second, ms, rs = (self.v, None, None) if self.bits == 32 else (self.r, self.m_scale, self.r_scale)
        L = _lib.load_library()
        rc = L.agz_adamw_step_missed(device, _raw_stream(device), o, missed, missed_dev, len(params), self._pointers.pack(*[p.data_ptr() for p in params]), self._pointers.pack(*at), self._numel,
                              self.m.data_ptr(), second.data_ptr(), _ptr(ms), _ptr(rs))
        if rc:
            _lib_call(rc, L)
        self.steps = t
        if 0 not in at:
            torch.autograd.graph.increment_version(params)
            return
        torch.autograd.graph.increment_version([p for p, g in zip(params, at) if g])
        if self.step_dev is None:
            for i, g in enumerate(at):
                if not g:
                    self._missed[i] += 1
                    self._any_missed = True


__all__ = ["log_probs", "LogProbs", "quantize_fp8", "matmul_fp8", "linear_fp8", "Fp8Matrix", "Fp8Weight", "AdamW", "TOP_MAX"]
