"""Times and checks the operators of the learning side: log probabilities of moves with their gradient, products in 8 bits with a scale for each
block of 128 and their backward pass, and AdamW over many tensors.  `own` chooses between the framework's kernels (alphagpu_amd.ops) and the same
mathematics in elementary torch operations.

    listed()               the cases, by name
    draw(rng)              one more case of the same ranges
    prepare(case, seed)    inputs and handles on the GPU
    run(state)             one pass through the operator
    work(case)             the bytes and operations that a pass cannot do without
    exact(case, seed)      what run() returns, from the definitions in 64 bits
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
DEV = "cuda"
LR, BETA1, BETA2, EPS, DECAY = 1e-4, 0.9, 0.999, 1e-8, 1e-2      # AdamW
STEPS_BEFORE = 100                                               # steps an optimiser has taken before the one that is measured


# ---------------------------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the leaf batch of a full-size search (32768 games, Gobang 9x9): log probability of the move played, entropy, five best alternatives
        {"name": "moves of a leaf batch", "op": "log_probs", "rows": 32768, "actions": 81, "dtype": "f32", "mask": True, "target": False, "top": 5, "grad": False},
        # the policy head of a learning step over two plies of a generation: policy loss against the search's policy, and its gradient
        {"name": "policy loss and gradient", "op": "log_probs", "rows": 65536, "actions": 81, "dtype": "f32", "mask": True, "target": True, "top": 0, "grad": True},
        # one row over a very large set of actions, as an answer is given move by move
        {"name": "one wide row", "op": "log_probs", "rows": 1, "actions": 131072, "dtype": "bf16", "mask": False, "target": False, "top": 20, "grad": False},
        # many wide rows of an odd length (their starts are not aligned), with the gradient
        {"name": "wide rows and gradient", "op": "log_probs", "rows": 4096, "actions": 50001, "dtype": "bf16", "mask": False, "target": False, "top": 0, "grad": True},
        # the first layer of the 128-wide network on the planes of Gobang 9x9 (162 of them), an odd number of positions, weights laid out once
        {"name": "first layer", "op": "product", "m": 20001, "k": 162, "n": 128, "dtype": "bf16", "relu": True, "grad": False},
        # one position through a wide layer: the weights are read once and that is all
        {"name": "one row through a wide layer", "op": "product", "m": 1, "k": 8192, "n": 8192, "dtype": "bf16", "relu": False, "grad": False},
        # a learning step of one trunk layer of the 512x8 network: forward, both gradients, from weights in 32 bits
        {"name": "trunk layer, learning", "op": "product", "m": 32768, "k": 512, "n": 512, "dtype": "bf16", "relu": True, "grad": True},
        # a learning step of a wide layer
        {"name": "wide layer, learning", "op": "product", "m": 8192, "k": 4096, "n": 8192, "dtype": "bf16", "relu": False, "grad": True},
        # the optimiser over the 128x6 network of Gobang 9x9 in 32 bits: launch bound
        {"name": "adamw 128x6", "op": "adamw", "tensors": "128x162,128x128,128x128,128x128,128x128,128x128,128x128,81x128,81,128,1", "bits": 32, "param": "f32", "grads": "f32"},
        # ... over the 512x8 network, states in 8 bits
        {"name": "adamw 512x8, 8 bits", "op": "adamw", "tensors": "512x162,8x512x512,81x512,81,512,1", "bits": 8, "param": "f32", "grads": "f32"},
        # ... over large networks: a few wide matrices among small vectors
        {"name": "adamw large, 32 bits", "op": "adamw", "tensors": _large(), "bits": 32, "param": "f32", "grads": "f32"},
        {"name": "adamw large, 8 bits", "op": "adamw", "tensors": _large(), "bits": 8, "param": "f32", "grads": "bf16"},
    ]


def _large():
    return ",".join(["4096x4096", "4096", "8191x2048", "8191"] * 2)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["log_probs", "product", "adamw"])
    if op == "log_probs":
        rows = _log(rng, 1, 200000)
        grad = rng.random() < 0.5
        top = rng.choice([0, 1, 5, 20]) if rows <= 40000 else rng.choice([0, 1, 5])
        most = 100_000_000 if not top else 20_000_000            # (the plain form sorts the rows for the alternatives)
        actions = _log(rng, 2, max(3, min(131072, most // rows)))
        return {"op": op, "rows": rows, "actions": actions, "dtype": rng.choice(["f32", "bf16", "f16"]), "mask": rng.random() < 0.5,
                "target": rng.random() < 0.4, "top": min(top, actions), "grad": grad}
    if op == "product":
        grad = rng.random() < 0.5
        k, n = _log(rng, 24, 8192), _log(rng, 24, 8192)
        m = _log(rng, 1, max(2, min(65536, (1 << 37) // (k * n))))
        return {"op": op, "m": m, "k": k, "n": n, "dtype": rng.choice(["f32", "bf16", "f16"]), "relu": rng.random() < 0.5, "grad": grad}
    count, total = rng.randint(1, 40), _log(rng, 1000, 60_000_000)
    parts = [rng.random() ** 3 for _ in range(count)]
    sizes = [max(1, int(total * p / sum(parts))) for p in parts]
    return {"op": op, "tensors": ",".join(map(str, sizes)), "bits": rng.choice([8, 32]), "param": rng.choice(["f32", "f32", "bf16"]),
            "grads": rng.choice(["f32", "bf16"])}


def _shapes(case):
    return [tuple(int(d) for d in t.split("x")) for t in case["tensors"].split(",")]


def work(case):
    op = case["op"]
    if op == "log_probs":
        n, a, es = case["rows"], case["actions"], SIZE[case["dtype"]]
        read = n * a * (es + (1 if case["mask"] else 0) + (4 if case["target"] else 0)) + 8 * n
        out = n * 4 * (2 + case["target"] + 2 * case["top"])
        return {"bytes": read + out + (n * a * es + n * 4 * (2 + case["target"] + case["top"]) if case["grad"] else 0), "flops": n * a * (10 + 8 * case["grad"])}
    if op == "product":
        m, k, n, es = case["m"], case["k"], case["n"], SIZE[case["dtype"]]
        if not case["grad"]:
            return {"bytes": m * k * es + n * k + m * n * es, "flops": 2 * m * n * k}
        return {"bytes": (2 * m * k + 2 * m * n) * es + 8 * n * k + 8 * n, "flops": 6 * m * n * k}
    total = sum(math.prod(s) for s in _shapes(case))
    held = 16 if case["bits"] == 32 else 4 + 4 / 128
    return {"bytes": total * (2 * SIZE[case["param"]] + SIZE[case["grads"]] + held), "flops": total * 14}


# ---------------------------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 17)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device=DEV)


def _log_probs_inputs(case, seed):
    g, n, a = _gen(seed), case["rows"], case["actions"]
    s = {"logits": (_randn(g, n, a) * (0.5 + 3 * _rand(g, n, 1))).to(DTYPES[case["dtype"]]), "mask": None, "target": None}
    free = None
    if case["mask"]:                                              # moves that are legal: a different share in each row, none in a few
        s["mask"] = _rand(g, n, a) < (0.1 + 0.9 * _rand(g, n, 1))
        if n > 8:
            s["mask"][_rand(g, n) < 0.001] = False
        free = s["mask"]
    score = _rand(g, n, a) if free is None else _rand(g, n, a).masked_fill_(~free, -1.0)
    s["moves"] = score.argmax(1)
    s["moves"][_rand(g, n) < 0.01] = -1                           # rows without a move
    if case["target"]:                                            # a search's policy: sharper than the logits, zero on illegal moves
        score.mul_(8.0).exp_()
        if free is not None:
            score.mul_(free)
        s["target"] = score / score.sum(1, keepdim=True).clamp_min(1e-30)
    if case["grad"]:                                              # of a mean over the rows (16 bits with 5 of exponent: of their sum)
        size = 1 if case["dtype"] == "f16" else 1 / n
        s["g_move"] = size * _randn(g, n)
        s["g_entropy"] = 0.01 * size * _randn(g, n)
        s["g_target"] = -size * (1 + 0.1 * _randn(g, n)) if case["target"] else None
        s["g_top"] = size * _randn(g, n, case["top"]) if case["top"] else None
    return s


def _product_inputs(case, seed):
    g, m, k, n = _gen(seed), case["m"], case["k"], case["n"]
    t = DTYPES[case["dtype"]]
    x = _randn(g, m, k) * torch.exp(0.7 * _randn(g, 1, k))        # channels of different scale, as activations have
    s = {"x": x.relu_().to(t), "w": _randn(g, n, k) * (1.5 / math.sqrt(k)), "bias": 0.1 * _randn(g, n)}
    if case["grad"]:
        s["dy"] = (_randn(g, m, n) * torch.exp(_randn(g, m, 1)) * (1 if case["dtype"] == "f16" else 1 / m)).to(t)
    return s


def _offsets(shapes):
    """Where each tensor's states begin in the buffers that hold all of them (every tensor starts a new block of 128), and their length."""
    at, out = 0, []
    for s in shapes:
        out.append(at)
        at += -(-math.prod(s) // 128) * 128
    return out, at


def _adamw_inputs(case, seed):
    g, shapes = _gen(seed), _shapes(case)
    at, total = _offsets(shapes)
    s = {"params": [], "grads": []}
    m, v = torch.zeros(total, device=DEV), torch.zeros(total, device=DEV)
    for sh, o in zip(shapes, at):
        n = math.prod(sh)
        s["params"].append((_randn(g, *sh) * 0.05).to(DTYPES[case["param"]]))
        size = 1e-3 * torch.exp(_randn(g, n))                     # gradients' sizes differ from weight to weight
        s["grads"].append((size * _randn(g, n)).to(DTYPES[case["grads"]]).view(sh))
        m[o:o + n] = size * 0.3 * _randn(g, n)
        v[o:o + n] = size.square() * (0.5 + _rand(g, n))
    return s, m, v


def prepare(case, seed):
    op = case["op"]
    if op == "log_probs":
        s = _log_probs_inputs(case, seed)
        if case["grad"]:
            s["logits"].requires_grad_(own)
    elif op == "product":
        s = _product_inputs(case, seed)
        if case["grad"]:                                          # weights in 32 bits, quantised in every pass
            for t in ("x", "w", "bias"):
                s[t].requires_grad_(own)
        elif own:                                                 # weights laid out once
            from alphagpu_amd import ops
            s["w"] = ops.Fp8Weight(s["w"])
        else:
            q, e = _to_blocks(s["w"], 128)
            s["w"] = (q.to(torch.float8_e4m3fn), e)
    else:
        s, m, v = _adamw_inputs(case, seed)
        s["bits"], s["seed"], s["step"] = case["bits"], 1234, STEPS_BEFORE
        held = {"m": m, "v": v}
        if case["bits"] == 8:
            mq, me = _to_blocks(m.view(-1, 128), 1)
            rq, re = _to_blocks(v.sqrt().view(-1, 128), 1)
            rq = torch.where((v.view(-1, 128) > 0) & (rq == 0), 2.0 ** -9, rq)
            held = {"m": mq.view(-1).to(torch.float8_e4m3fn), "m_scale": _e8m0(me.view(-1)),
                    "r": rq.view(-1).to(torch.float8_e4m3fn), "r_scale": _e8m0(re.view(-1))}
        if own:
            from alphagpu_amd import ops
            s["opt"] = ops.AdamW(s["params"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, bits=case["bits"], seed=s["seed"])
            s["opt"].load_state({"step": STEPS_BEFORE, **held})
        else:
            s["held"] = held
            s["at"] = _offsets(_shapes(case))[0]
    s["case"] = dict(case)
    return s


# ---------------------------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return {"log_probs": _own_log_probs, "product": _own_product, "adamw": _own_adamw}[case["op"]](state, case)
    return {"log_probs": _plain_log_probs, "product": _plain_product, "adamw": _plain_adamw}[case["op"]](state, case)


def _own_log_probs(s, case):
    from alphagpu_amd import ops
    r = ops.log_probs(s["logits"], s["moves"], mask=s["mask"], target=s["target"], top=case["top"])
    out = {"move": r.move, "entropy": r.entropy}
    if case["target"]:
        out["target"] = r.target
    if case["top"]:
        out["top"], out["top_move"] = r.top, r.top_move
    if case["grad"]:
        names = ["move", "entropy"] + (["target"] if case["target"] else []) + (["top"] if case["top"] else [])
        out["dlogits"], = torch.autograd.grad([out[k] for k in names], [s["logits"]], [s["g_" + k] for k in names])
    return out


def _own_product(s, case):
    from alphagpu_amd import ops
    y = ops.linear_fp8(s["x"], s["w"], s["bias"], relu=case["relu"])
    if not case["grad"]:
        return {"y": y}
    dx, dw, db = torch.autograd.grad([y], [s["x"], s["w"], s["bias"]], [s["dy"]])
    return {"y": y, "dx": dx, "dw": dw, "dbias": db}


def _own_adamw(s, case):
    opt = s["opt"]
    opt.step(s["grads"])
    held = {"m": opt.m, "v": opt.v} if case["bits"] == 32 else {"m": opt.m, "m_scale": opt.m_scale, "r": opt.r, "r_scale": opt.r_scale}
    return {"params": s["params"], **held}


def _plain_log_probs(s, case):
    lowest = float("-inf")
    x = s["logits"].float()
    free = x > lowest if s["mask"] is None else (s["mask"] & (x > lowest))
    x = torch.where(free, x, lowest)
    top = x.max(1, keepdim=True).values
    d = torch.where(free, x - top, 0.0)
    e = torch.where(free, d.exp(), 0.0)
    total = e.sum(1, keepdim=True)
    some = free.any(1, keepdim=True)
    ls = torch.where(some, total, 1.0).log()
    logp = torch.where(free, d - ls, lowest)
    p = torch.where(some, e / total, 0.0)
    entropy = ls - (p * d).sum(1, keepdim=True)
    moves = s["moves"]
    given = (moves >= 0) & (moves < x.shape[1])
    at = moves.clamp(0, x.shape[1] - 1)[:, None]
    out = {"move": torch.where(given, logp.gather(1, at)[:, 0], 0.0), "entropy": entropy[:, 0]}
    if case["target"]:
        t = s["target"]
        out["target"] = torch.where(t != 0, t * logp, 0.0).sum(1)
    if case["top"]:
        best, which = torch.sort(x, dim=1, descending=True, stable=True)
        best, which = best[:, :case["top"]], which[:, :case["top"]]
        out["top"] = torch.where(best > lowest, best - top - ls, lowest)
        out["top_move"] = torch.where(best > lowest, which, -1).to(torch.int32)
    if case["grad"]:
        g = torch.where(given, s["g_move"], 0.0)[:, None]
        whole = g
        if case["top"]:
            valid = out["top_move"] >= 0
            g_top = torch.where(valid, s["g_top"], 0.0)
            whole = g + g_top.sum(1, keepdim=True)
        dx = -p * (whole + s["g_entropy"][:, None] * torch.where(free, logp + entropy, 0.0))
        if case["target"]:
            dx += s["g_target"][:, None] * (s["target"] - p * s["target"].sum(1, keepdim=True))
        dx.scatter_add_(1, at, g)
        if case["top"]:
            dx.scatter_add_(1, out["top_move"].long().clamp_min(0), g_top)
        out["dlogits"] = torch.where(free, dx, 0.0).to(s["logits"].dtype)
    return out


def _exponent(amax):
    """The smallest e (from -127 on) with amax <= 448 * 2^e; 0 for a block of zeros."""
    f, e = torch.frexp(amax)
    e = e - 9 + (f > 0.875).to(e.dtype)
    return torch.where(amax > 0, e.clamp_min(-127), 0)


def _power(e):
    return torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)


def _e8m0(e):
    return (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _pad(x, rows, cols):
    return torch.nn.functional.pad(x, (0, -x.shape[1] % cols, 0, -x.shape[0] % rows))


def _to_blocks(x, rows):
    """x [R, C] -> (x / 2^e rounded to e4m3, as float32 [R, C]; e [ceil(R / rows), ceil(C / 128)]) for blocks of `rows` x 128."""
    R, C = x.shape
    b = _pad(x.float(), rows, 128)
    b = b.view(b.shape[0] // rows, rows, b.shape[1] // 128, 128)
    e = _exponent(torch.where(b.isfinite(), b.abs(), 0.0).amax((1, 3)))
    q = (b / _power(e)[:, None, :, None]).to(torch.float8_e4m3fn).float()
    return q.reshape(q.shape[0] * rows, -1)[:R, :C], e


def _from_blocks(q, e, rows):
    R, C = q.shape
    b = _pad(q.float(), rows, 128)
    b = b.view(b.shape[0] // rows, rows, b.shape[1] // 128, 128) * _power(e)[:, None, :, None]
    return b.reshape(b.shape[0] * rows, -1)[:R, :C]


def _rounded(x, rows):
    return _from_blocks(*_to_blocks(x, rows), rows)


def _plain_product(s, case):
    t = s["x"].dtype
    wq = _from_blocks(*s["w"], 128) if isinstance(s["w"], tuple) else _rounded(s["w"], 128)
    y = _rounded(s["x"], 1) @ wq.t() + s["bias"]
    if case["relu"]:
        y = y.relu()
    y = y.to(t)
    if not case["grad"]:
        return {"y": y}
    dy = s["dy"].float()
    if case["relu"]:
        dy = torch.where(y > 0, dy, 0.0)
    dx = (_rounded(dy, 1) @ wq).to(t)
    dw = _rounded(dy.t(), 1) @ _rounded(s["x"].t(), 1).t()
    return {"y": y, "dx": dx, "dw": dw, "dbias": dy.sum(0)}


M32 = 0xFFFFFFFF


def _mix(h):
    """The hash behind the rounding of 8-bit states: 32 bits to 32 bits (ints or int64 tensors)."""
    h = (h * 0x9E3779B1) & M32
    h = h ^ (h >> 16)
    h = (h * 0xB504F335) & M32
    return h ^ (h >> 16)


def _key(seed, step, tensor):
    return _mix(_mix(_mix((seed + 0x3C6EF372) & M32) ^ (step & M32)) + tensor & M32)


def _stochastic(y, u):
    """y in [0, 448] to e4m3: up with the probability of its place between its neighbours; u: whole numbers below 2^16."""
    low = torch.where(y < 2.0 ** -6, 2.0 ** -6, 0.0)              # below the normal numbers the steps are those of 2^-6
    t = (y + low).view(torch.int32) + (u.to(torch.int32) << 4)
    return (t & ~0xFFFFF).view(torch.float32) - low


def _hold(x, u, floor):
    b = x.view(-1, 128)
    e = _exponent(torch.where(b.isfinite(), b.abs(), 0.0).amax(1))
    y = b.abs() / _power(e)[:, None]
    q = torch.where(y.isfinite(), _stochastic(torch.where(y.isfinite(), y, 0.0), u.view(-1, 128)), float("nan"))
    if floor:
        q = torch.where(y > 0, q.clamp_min(2.0 ** -9), q)
    return (q * b.sign()).to(torch.float8_e4m3fn).view(-1), _e8m0(e)


def _plain_adamw(s, case):
    s["step"] += 1
    c1, c2 = 1 - BETA1 ** s["step"], 1 - BETA2 ** s["step"]
    held = s["held"]
    for i, (p, g, o) in enumerate(zip(s["params"], s["grads"], s["at"])):
        n = p.numel()
        full = -(-n // 128) * 128
        g = torch.nn.functional.pad(g.reshape(-1).float(), (0, full - n))
        if case["bits"] == 32:
            m, v = held["m"][o:o + full], held["v"][o:o + full]
        else:
            b = slice(o // 128, (o + full) // 128)
            m = (held["m"][o:o + full].float().view(-1, 128) * held["m_scale"][b].float()[:, None]).view(-1)
            v = (held["r"][o:o + full].float().view(-1, 128) * held["r_scale"][b].float()[:, None]).view(-1).square()
        m = m * BETA1 + g * (1 - BETA1)
        v = v * BETA2 + (g * g) * (1 - BETA2)
        root = v.sqrt()
        step = (m * (LR / c1)) / (root * (1 / math.sqrt(c2)) + EPS)
        p.copy_((p.reshape(-1).float() * (1 - LR * DECAY) - step[:n]).view(p.shape))
        if case["bits"] == 32:
            held["m"][o:o + full], held["v"][o:o + full] = m, v
        else:
            h = _mix(torch.arange(full, device=DEV) ^ _key(s["seed"], s["step"], i))
            held["m"][o:o + full], held["m_scale"][b] = _hold(m, h & 0xFFFF, False)
            held["r"][o:o + full], held["r_scale"][b] = _hold(root, h >> 16, True)
    return {"params": s["params"], **held}


# ---------------------------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    return {"log_probs": _exact_log_probs, "product": _exact_product, "adamw": _exact_adamw}[case["op"]](case, seed)


def _exact_log_probs(case, seed):
    s = _log_probs_inputs(case, seed)
    out = {"move": [], "entropy": [], "target": [], "top": [], "dlogits": []}
    n, step = case["rows"], max(1, 20_000_000 // case["actions"])
    for a in range(0, n, step):                                   # some rows at a time: memory
        part = slice(a, a + step)
        x = s["logits"][part].double()
        if s["mask"] is not None:
            x = x.masked_fill(~s["mask"][part], -math.inf)
        lse = torch.logsumexp(x, 1, keepdim=True)
        lp = torch.where(x == -math.inf, -math.inf, x - lse)
        p = lp.exp()
        plp = torch.where(p > 0, p * lp, 0.0)
        h = -plp.sum(1, keepdim=True)
        mv = s["moves"][part]
        hot = torch.zeros_like(x)
        given = (mv >= 0).nonzero()[:, 0]
        hot[given, mv[given]] = 1.0
        out["move"].append(torch.where(hot > 0, lp, 0.0).sum(1))
        out["entropy"].append(h[:, 0])
        if case["target"]:
            t = s["target"][part].double()
            out["target"].append(torch.where(t > 0, t * lp, 0.0).sum(1))
        if case["top"]:
            best = torch.topk(lp, case["top"], dim=1)
            out["top"].append(best.values)
        if case["grad"]:                                          # d/dx of sum_k c_k lp_k is c - p sum(c); d/dx of the entropy is -p (lp + H)
            c = hot * s["g_move"][part].double()[:, None]
            if case["target"]:
                c = c + t * s["g_target"][part].double()[:, None]
            if case["top"]:                                       # equal logits: the lowest index comes first
                order = torch.sort(lp, dim=1, descending=True, stable=True).indices[:, :case["top"]]
                live = best.values > -math.inf
                c = c.scatter_add(1, order, torch.where(live, s["g_top"][part].double(), 0.0))
            dx = c - p * c.sum(1, keepdim=True) - s["g_entropy"][part].double()[:, None] * (plp + p * h)
            out["dlogits"].append(torch.where(x == -math.inf, 0.0, dx))
    got = {k: torch.cat(v) for k, v in out.items() if v}
    if case["top"]:
        got["top_move"] = None
    return got


def _grid(x, axis_rows):
    """The value that each entry of x (64 bits) stands for once it is held in e4m3 with a power-of-two scale per block."""
    R, C = x.shape
    full = torch.zeros(-(-R // axis_rows) * axis_rows, -(-C // 128) * 128, dtype=torch.float64, device=x.device)
    full[:R, :C] = x
    blocks = full.unflatten(0, (-1, axis_rows)).unflatten(2, (-1, 128))
    biggest = blocks.abs().amax(dim=(1, 3), keepdim=True)
    scale = torch.exp2(torch.ceil(torch.log2(biggest.clamp_min(1e-300) / 448)).clamp_min(-127))
    scale = torch.where(biggest > 448 * scale, scale * 2, scale)
    y = blocks / scale
    spacing = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(y / spacing) * spacing * scale).flatten(2, 3).flatten(0, 1)[:R, :C]


def _exact_product(case, seed):
    s = _product_inputs(case, seed)
    w, x = _grid(s["w"].double(), 128), _grid(s["x"].double(), 1)
    y = torch.addmm(s["bias"].double(), x, w.t())
    if case["relu"]:
        y.clamp_(min=0)
    if not case["grad"]:
        return {"y": y}
    dy = s["dy"].double()
    if case["relu"]:
        dy = dy * (y > 0)
    dx = _grid(dy, 1) @ w
    dw = _grid(dy.t(), 1) @ _grid(s["x"].double().t(), 1).t()
    return {"y": y, "dx": dx, "dw": dw, "dbias": dy.sum(0)}


def _exact_adamw(case, seed):
    s, m_all, v_all = _adamw_inputs(case, seed)
    t = STEPS_BEFORE + 1
    at, total = _offsets(_shapes(case))
    out = {"params": []}
    if case["bits"] == 32:
        out["m"], out["v"] = (torch.zeros(total, dtype=torch.float64, device=DEV) for _ in range(2))
    else:
        out["m"] = out["m_scale"] = out["r"] = out["r_scale"] = None
        m_all = _grid(m_all.double().view(-1, 128), 1).view(-1)
        r = v_all.sqrt().double().view(-1, 128)
        held = _grid(r, 1)
        unit = torch.exp2(torch.ceil(torch.log2(r.amax(1, keepdim=True).clamp_min(1e-300) / 448)) - 9)
        v_all = torch.where((held == 0) & (r > 0), unit, held).square().view(-1)
    for p, g, o in zip(s["params"], s["grads"], at):
        n = p.numel()
        g, p64 = g.double().view(-1), p.double().view(-1)
        m = BETA1 * m_all[o:o + n].double() + (1 - BETA1) * g
        v = BETA2 * v_all[o:o + n].double() + (1 - BETA2) * g ** 2
        new = p64 * (1 - LR * DECAY) - LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
        out["params"].append(new.view(p.shape))
        if case["bits"] == 32:
            out["m"][o:o + n], out["v"][o:o + n] = m, v
    return out
