"""Measured cases of the language-model operators: the root-mean-square norm
(``autodrive_b200.ops.rmsnorm``), the 8-bit product with a scale for each block
of 128 (``autodrive_b200.ops.fp8``) and the log-probabilities of given tokens
(``autodrive_b200.ops.token_logprobs``).

``run`` computes a case in plain torch operations, or, where ``own`` is true,
with the framework's kernels; ``exact`` computes it in 64 bits.
"""
from __future__ import annotations

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.
TINY = 2. ** -126
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one robot's context token on its way into a head: launch latency
        {"name": "norm one token", "op": "norm", "mode": "forward", "rows": 1, "d": 256, "dtype": "bf16",
         "residual": True},
        # a minibatch of packed entity tokens, forward and backward, an odd number of them
        {"name": "norm train tokens", "op": "norm", "mode": "train", "rows": 40001, "d": 256, "dtype": "bf16",
         "residual": True},
        # a wide model in single precision, no residual, an odd width
        {"name": "norm train fp32 odd", "op": "norm", "mode": "train", "rows": 4099, "d": 4099, "dtype": "fp32",
         "residual": False},
        # a prompt's activations on their way into an 8-bit product
        {"name": "norm to 8 bits", "op": "norm", "mode": "fp8", "rows": 16384, "d": 4096, "dtype": "bf16",
         "residual": True},
        # one decision through the raster network's widest layer (128 channels x 8 x 16 cells + 256 scalars)
        {"name": "product one row", "op": "product", "m": 1, "n": 1408, "k": 16640, "out": "bf16", "bias": True},
        # a few decisions at a time through a wide square layer
        {"name": "product few rows", "op": "product", "m": 18, "n": 4096, "k": 4096, "out": "bf16", "bias": False},
        # a rollout step of 2048 worlds x 3 robots through the raster network's widest layer
        {"name": "product rollout", "op": "product", "m": 6144, "n": 1408, "k": 16640, "out": "bf16", "bias": True},
        # sides that end inside a block, results in single precision
        {"name": "product ragged", "op": "product", "m": 1537, "n": 1000, "k": 2008, "out": "fp32", "bias": True},
        # a training step of the entity network's head layer 1536 -> 1024
        {"name": "linear step", "op": "linear", "m": 8192, "n": 1024, "k": 1536, "dtype": "bf16"},
        # a PPO minibatch of masked strategic actions, with gradients
        {"name": "score actions", "op": "score", "rows": 4096, "v": 8, "dtype": "fp32", "mask": True, "top": 0,
         "grad": True, "temperature": 1.},
        # the next token of two sequences and its alternatives
        {"name": "score next token", "op": "score", "rows": 2, "v": 131072, "dtype": "bf16", "mask": False, "top": 20,
         "grad": False, "temperature": .7},
        # a batch of sampled tokens, with gradients and alternatives
        {"name": "score tokens", "op": "score", "rows": 4095, "v": 32003, "dtype": "bf16", "mask": False, "top": 5,
         "grad": True, "temperature": 1.},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(("norm", "norm", "product", "product", "linear", "score", "score"))
    if op == "norm":
        d = _log_int(rng, 32, 8192)
        return {"op": op, "mode": rng.choice(("forward", "train", "fp8")),
                "rows": _log_int(rng, 1, min(65536, 16384 * 4096 // d)), "d": d,
                "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32")), "residual": rng.random() < .6}
    if op == "product":
        n, k = _log_int(rng, 32, 8192), 8 * _log_int(rng, 4, 2080)
        return {"op": op, "m": _log_int(rng, 1, min(16384, 140_000_000_000 // (n * k))), "n": n, "k": k,
                "out": rng.choice(("bf16", "bf16", "fp32")), "bias": rng.random() < .5}
    if op == "linear":
        return {"op": op, "m": _log_int(rng, 16, 8192), "n": _log_int(rng, 64, 2048), "k": _log_int(rng, 64, 2048),
                "dtype": rng.choice(("bf16", "fp32"))}
    v = _log_int(rng, 2, 200_000)
    return {"op": op, "rows": _log_int(rng, 1, min(65536, 4095 * 32003 // v)), "v": v,
            "dtype": rng.choice(("bf16", "fp32", "fp16")), "mask": rng.random() < .5,
            "top": rng.choice((0, 0, 1, 5, 20)), "grad": rng.random() < .5, "temperature": rng.choice((1., .7, 1.3))}


# ------------------------------------------------------------------ inputs
def _to_e4m3(t):
    """The e4m3 value nearest to each 64-bit value of `t`, ties to even: rounded in one step, as a cast by way of
    32 bits would round a value next to a tie twice. `t` is at most 448, but for the rounding of its scale."""
    _, exponent = torch.frexp(t)
    step = torch.ldexp(torch.ones_like(t), exponent.clamp_min(-5) - 4)
    return (torch.round(t / step) * step).to(torch.float8_e4m3fn)


def _scale_of(amax):
    """amax / 448, held in 32 bits (rounded once: the quotient is taken in 64 bits)."""
    return (amax.clamp_min(E4M3_MAX * TINY).double() / E4M3_MAX).float()


def _quantize_rows(x):
    """(e4m3 values, scales): one scale for each row and group of 128 columns. The quotient by the scale decides
    between two neighbours, so it is taken in 64 bits."""
    m, k = x.shape
    groups = -(-k // BLOCK)
    padded = torch.zeros((m, groups * BLOCK), dtype=torch.float32, device=x.device)
    padded[:, :k] = x
    padded = padded.view(m, groups, BLOCK)
    scale = _scale_of(padded.abs().amax(-1))
    q = _to_e4m3(padded.double() / scale[..., None])
    return q.view(m, -1)[:, :k], scale


def _quantize_blocks(w):
    """(e4m3 values, scales): one scale for each 128 x 128 block."""
    n, k = w.shape
    bn, bk = -(-n // BLOCK), -(-k // BLOCK)
    padded = torch.zeros((bn * BLOCK, bk * BLOCK), dtype=torch.float32, device=w.device)
    padded[:n, :k] = w
    padded = padded.view(bn, BLOCK, bk, BLOCK)
    scale = _scale_of(padded.abs().amax((1, 3)))
    q = _to_e4m3(padded.double() / scale[:, None, :, None])
    return q.view(bn * BLOCK, bk * BLOCK)[:n, :k], scale


def _rows_16(q):
    """`q` in storage whose rows start 16 bytes apart, as the quantisers lay it out."""
    m, k = q.shape
    buf = torch.zeros((m, -(-k // 16) * 16), dtype=torch.uint8, device=q.device).view(q.dtype)
    buf[:, :k] = q
    return buf[:, :k]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(shape, device=dev, generator=g)

    op, s = case["op"], {"case": case}
    if op == "norm":
        dt, rows, d = DTYPES[case["dtype"]], case["rows"], case["d"]
        train = case["mode"] == "train"
        s["x"] = normal(rows, d).to(dt).requires_grad_(train)
        s["weight"] = (1. + .2 * normal(d)).requires_grad_(train)
        s["residual"] = (2. * normal(rows, d)).to(dt).requires_grad_(train) if case["residual"] else None
        if train:
            s["dy"] = normal(rows, d).to(dt)
            s["dh"] = normal(rows, d).to(dt) if case["residual"] else None
    elif op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        # activations with rows and channels of different size, weights near 1 / sqrt(k)
        x = normal(m, k) * (.5 * normal(m, 1)).exp() * (.5 * normal(1, k)).exp()
        a, s["a_scale"] = _quantize_rows(x)
        b, s["b_scale"] = _quantize_blocks(normal(n, k) * k ** -.5)
        s["a"], s["b"] = _rows_16(a), _rows_16(b)
        s["bias"] = normal(n) if case["bias"] else None
    elif op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        # bf16 values also where they are held in fp32: the weight gradient takes its operands in bf16
        s["x"] = normal(m, k).bfloat16().to(DTYPES[case["dtype"]]).requires_grad_(True)
        s["weight"] = (normal(n, k) * k ** -.5).requires_grad_(True)
        s["bias"] = normal(n).requires_grad_(True)
        s["dy"] = (normal(m, n) / m).bfloat16().to(DTYPES[case["dtype"]])
    else:
        rows, v = case["rows"], case["v"]
        s["logits"] = (3. * normal(rows, v)).to(DTYPES[case["dtype"]]).requires_grad_(case["grad"])
        s["tokens"] = torch.randint(v, (rows,), device=dev, generator=g)
        s["mask"] = None
        if case["mask"]:
            # about a third of the entries is invalid; the taken token is valid, and one row in 64 has none at all
            mask = torch.rand((rows, v), device=dev, generator=g) < .66
            mask.scatter_(1, s["tokens"][:, None], True)
            mask[5::64] = False
            s["mask"] = mask
        if case["grad"]:
            s["g_log_prob"], s["g_entropy"] = normal(rows) / rows, .01 * normal(rows) / rows
    return s


# ------------------------------------------------------------------ one pass
EPS = 1e-6


def _plain_norm(s):
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    x, w = s["x"].detach(), s["weight"].detach()
    h = x if s["residual"] is None else (x.float() + s["residual"].detach().float()).to(dt)
    hf = h.float()
    rstd = (hf.square().mean(-1, keepdim=True) + EPS).rsqrt()
    out = {} if s["residual"] is None else {"h": h}
    y = hf * rstd * w
    if case["mode"] == "fp8":
        out["q"], out["scale"] = _quantize_rows(y)
        return out
    out["y"] = y.to(dt)
    if case["mode"] == "train":
        dy, n = s["dy"].float(), hf * rstd
        g = dy * w
        dx = rstd * (g - n * (g * n).mean(-1, keepdim=True))
        if s["dh"] is not None:
            dx = dx + s["dh"].float()
        out["dx"], out["dweight"] = dx.to(dt), (dy * n).sum(0)
    return out


def _own_norm(s):
    from autodrive_b200.ops.rmsnorm import rms_norm, rms_norm_fp8
    case, res = s["case"], s["residual"]
    if case["mode"] == "fp8":
        q, scale, *h = rms_norm_fp8(s["x"], s["weight"], res, eps=EPS)
        return {"q": q, "scale": scale, **({} if res is None else {"h": h[0]})}
    if res is None:
        y = rms_norm(s["x"], s["weight"], eps=EPS)
        out, ends, grads = {"y": y}, (y,), (s["dy"] if case["mode"] == "train" else None,)
    else:
        y, h = rms_norm(s["x"], s["weight"], res, eps=EPS)
        out, ends, grads = {"y": y, "h": h}, (y, h), (s.get("dy"), s.get("dh"))
    if case["mode"] == "train":
        out["dx"], out["dweight"] = torch.autograd.grad(ends, (s["x"], s["weight"]), grads)
    return out


def _spread_rows(scale, k):
    return scale.repeat_interleave(BLOCK, 1)[:, :k]


def _spread_blocks(scale, n, k):
    return scale.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]


def _plain_product(s):
    a, b, k = s["a"].float(), s["b"].float(), s["case"]["k"]
    y = (a * _spread_rows(s["a_scale"], k)) @ (b * _spread_blocks(s["b_scale"], b.shape[0], k)).t()
    if s["bias"] is not None:
        y = y + s["bias"]
    return {"y": y.to(DTYPES[s["case"]["out"]])}


def _own_product(s):
    from autodrive_b200.ops.fp8 import fp8_matmul
    return {"y": fp8_matmul(s["a"], s["a_scale"], s["b"], s["b_scale"], bias=s["bias"],
                            out_dtype=DTYPES[s["case"]["out"]])}


def _plain_linear(s):
    case = s["case"]
    n, k = case["n"], case["k"]
    x, w, dy = s["x"].detach(), s["weight"].detach(), s["dy"]
    xq, xs = _quantize_rows(x)
    wq, ws = _quantize_blocks(w)
    gq, gs = _quantize_rows(dy)
    wd = wq.float() * _spread_blocks(ws, n, k)
    y = (xq.float() * _spread_rows(xs, k)) @ wd.t() + s["bias"].detach()
    dx = (gq.float() * _spread_rows(gs, n)) @ wd
    return {"y": y.to(x.dtype), "dx": dx.to(x.dtype), "dweight": dy.float().t() @ x.float(),
            "dbias": dy.float().sum(0)}


def _own_linear(s):
    from autodrive_b200.ops.fp8 import fp8_linear
    y = fp8_linear(s["x"], s["weight"], s["bias"])
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
    return {"y": y, "dx": dx, "dweight": dw, "dbias": db}


def _plain_score(s):
    case = s["case"]
    logits, tokens, mask = s["logits"].detach().float(), s["tokens"][:, None], s["mask"]
    z = logits / case["temperature"]
    if mask is not None:
        z = torch.where(mask, z, torch.full_like(z, -torch.inf))
    top = z.amax(-1, keepdim=True)
    empty = top == -torch.inf
    top = torch.where(empty, torch.zeros_like(top), top)
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True)
    log_p = z - top - torch.log(total)
    p = e / torch.where(empty, torch.ones_like(total), total)
    terms = torch.where(p > 0, p * log_p, torch.zeros_like(p))
    entropy = -terms.sum(-1, keepdim=True)
    log_prob = torch.where(empty, torch.full_like(entropy, -torch.inf), log_p.gather(1, tokens))
    out = {"log_prob": log_prob[:, 0], "entropy": entropy[:, 0]}
    if case["top"]:
        k = case["top"]
        order = logits if mask is None else torch.where(mask, logits, torch.full_like(logits, -torch.inf))
        _, index = torch.sort(order, dim=-1, descending=True, stable=True)
        index = index[:, :k]
        value = log_p.gather(1, index)
        missing = order.gather(1, index) == -torch.inf
        value = torch.where(missing, torch.full_like(value, -torch.inf), value)
        index = torch.where(missing, torch.full_like(index, -1), index)
        short = k - index.shape[1]
        if short > 0:
            value = torch.cat((value, torch.full_like(value[:, :1], -torch.inf).expand(-1, short)), 1)
            index = torch.cat((index, torch.full_like(index[:, :1], -1).expand(-1, short)), 1)
        out["top_log_prob"], out["top_token"] = value, index
    if case["grad"]:
        gl, ge = s["g_log_prob"][:, None], s["g_entropy"][:, None]
        d = p * -gl - ge * (terms + p * entropy)
        d = d.scatter_add(1, tokens, gl)
        d = torch.where(empty, torch.zeros_like(d), d) / case["temperature"]
        out["dlogits"] = d.to(s["logits"].dtype)
    return out


def _own_score(s):
    from autodrive_b200.ops.token_logprobs import token_log_probs
    case = s["case"]
    r = token_log_probs(s["logits"], s["tokens"], mask=s["mask"], temperature=case["temperature"], top=case["top"])
    out = {"log_prob": r.log_prob, "entropy": r.entropy}
    if case["top"]:
        out["top_log_prob"], out["top_token"] = r.top_log_prob, r.top_token
    if case["grad"]:
        out["dlogits"], = torch.autograd.grad((r.log_prob, r.entropy), s["logits"], (s["g_log_prob"], s["g_entropy"]))
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "product": _own_product, "linear": _own_linear, "score": _own_score}[op](state)
    return {"norm": _plain_norm, "product": _plain_product, "linear": _plain_linear, "score": _plain_score}[op](state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "norm":
        n, size = case["rows"] * case["d"], DTYPES[case["dtype"]].itemsize
        read = write = size * n
        if case["residual"]:
            read, write = read + size * n, write + size * n
        flops = 5 * n
        if case["mode"] == "fp8":
            write += n * (1 - size) + 4 * case["rows"] * -(-case["d"] // BLOCK)
            flops += 3 * n
        if case["mode"] == "train":
            # x and residual, dy and dh in; y and h, dx and the weight's gradient out
            read += size * n * (2 if case["residual"] else 1)
            write += size * n + 4 * case["d"]
            flops += 11 * n
        return {"bytes": read + write + 4 * case["d"], "flops": flops}
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        groups = -(-k // BLOCK)
        return {"bytes": m * k + n * k + 4 * groups * (m + -(-n // BLOCK)) + m * n * DTYPES[case["out"]].itemsize
                + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    if op == "linear":
        m, n, k, size = case["m"], case["n"], case["k"], DTYPES[case["dtype"]].itemsize
        return {"bytes": size * (2 * m * k + 2 * m * n) + 8 * n * k + 8 * n, "flops": 6 * m * n * k}
    rows, v, size = case["rows"], case["v"], DTYPES[case["dtype"]].itemsize
    n = rows * v
    b = size * n + (n if case["mask"] else 0) + 16 * rows + 12 * rows * case["top"]
    f = 5 * n
    if case["grad"]:
        b, f = b + size * n + 8 * rows, f + 6 * n
    return {"bytes": b, "flops": f}


# ------------------------------------------------------------------ the definition in 64 bits
def _group_scale(y, axis):
    """amax / 448 as it is held, in 32 bits."""
    amax = torch.maximum(y.abs().amax(axis), torch.tensor(E4M3_MAX * TINY, dtype=torch.float64, device=y.device))
    return (amax / E4M3_MAX).float().double()


def _e4m3(t):
    """Nearest e4m3 value (ties to even): steps of 2^(exponent - 3), the exponent at least -6."""
    step = torch.exp2(torch.floor(torch.log2(t.abs().clamp_min(2. ** -6))) - 3)
    return torch.round(t / step) * step


def _exact_rows(x):
    """(8-bit values, scales) of the rows of a 64-bit matrix, group by group."""
    q, scales = torch.empty_like(x), []
    for g in range(0, x.shape[1], BLOCK):
        part = x[:, g:g + BLOCK]
        sc = _group_scale(part, 1)
        q[:, g:g + BLOCK] = _e4m3(part / sc[:, None])
        scales.append(sc)
    return q, torch.stack(scales, 1)


def _exact_norm(s):
    case = s["case"]
    x, w = s["x"].detach().double(), s["weight"].detach().double()
    out = {}
    if s["residual"] is not None:
        out["h"] = (x + s["residual"].detach().double())
        h = out["h"].to(DTYPES[case["dtype"]]).double()
    else:
        h = x
    w = w.requires_grad_(True)
    h = h.requires_grad_(True)
    y = h / torch.sqrt((h * h).sum(-1, keepdim=True) / case["d"] + EPS) * w
    if case["mode"] == "fp8":
        out["q"], out["scale"] = _exact_rows(y.detach())
        return out
    out["y"] = y.detach()
    if case["mode"] == "train":
        dx, out["dweight"] = torch.autograd.grad(y, (h, w), s["dy"].double())
        out["dx"] = dx if s["dh"] is None else dx + s["dh"].double()
    return out


def _exact_blocks_product(a, a_scale, b, b_scale):
    """sum over groups of 128 of the 64-bit products, each times its two scales."""
    y = torch.zeros((a.shape[0], b.shape[0]), dtype=torch.float64, device=a.device)
    row_block = torch.arange(b.shape[0], device=b.device) // BLOCK
    for g in range(a_scale.shape[1]):
        c = slice(g * BLOCK, (g + 1) * BLOCK)
        y += (a[:, c].double() @ b[:, c].double().t()) * a_scale[:, g, None].double() * b_scale[row_block, g].double()
    return y


def _exact_linear(s):
    x, w, dy = s["x"].detach().double(), s["weight"].detach().double(), s["dy"].double()
    n, k = w.shape
    wd = torch.empty_like(w)
    for i in range(0, n, BLOCK):
        for j in range(0, k, BLOCK):
            part = w[i:i + BLOCK, j:j + BLOCK]
            sc = _group_scale(part, (0, 1))
            wd[i:i + BLOCK, j:j + BLOCK] = _e4m3(part / sc) * sc

    def rounded(t):
        q, sc = _exact_rows(t)
        return torch.cat([q[:, g * BLOCK:(g + 1) * BLOCK] * sc[:, g, None] for g in range(sc.shape[1])], 1)

    return {"y": rounded(x) @ wd.t() + s["bias"].detach().double(), "dx": rounded(dy) @ wd, "dweight": dy.t() @ x,
            "dbias": dy.sum(0)}


def _exact_score(s):
    case = s["case"]
    parts = []
    for r in range(0, case["rows"], max(1, 30_000_000 // case["v"])):
        c = slice(r, r + max(1, 30_000_000 // case["v"]))
        x = s["logits"].detach()[c].double().requires_grad_(True)
        mask = None if s["mask"] is None else s["mask"][c]
        none = torch.zeros(x.shape[0], dtype=torch.bool, device=x.device) if mask is None else ~mask.any(-1)
        z = x / case["temperature"]
        if mask is not None:   # rows that hold nothing are computed as if unmasked and put right below
            z = z.masked_fill(~(mask | none[:, None]), -torch.inf)
        lp = torch.log_softmax(z, -1)
        finite = lp.masked_fill(lp == -torch.inf, 0.)
        lp_t, ent = lp.gather(1, s["tokens"][c, None])[:, 0], -(lp.exp() * finite).sum(-1)
        out = {"log_prob": lp_t.detach().masked_fill(none, -torch.inf), "entropy": ent.detach().masked_fill(none, 0.)}
        if case["top"]:
            best = lp.detach().masked_fill(none[:, None], -torch.inf).topk(min(case["top"], case["v"]), -1).values
            fill = best.new_full((best.shape[0], case["top"] - best.shape[1]), -torch.inf)
            out["top_log_prob"] = torch.cat((best, fill), 1)
        if case["grad"]:
            keep = (~none).double()
            d, = torch.autograd.grad((lp_t, ent), x, (s["g_log_prob"][c].double() * keep, s["g_entropy"][c].double() * keep))
            out["dlogits"] = d.to(torch.float64)
        parts.append(out)
    return {key: torch.cat([p[key] for p in parts]) for key in parts[0]}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        return _exact_norm(s)
    if op == "product":
        y = _exact_blocks_product(s["a"].float(), s["a_scale"], s["b"].float(), s["b_scale"])
        return {"y": y if s["bias"] is None else y + s["bias"].double()}
    if op == "linear":
        return _exact_linear(s)
    return {"top_token": None, **_exact_score(s)} if case["top"] else _exact_score(s)
