"""Measured cases of the operators of a training iteration: sampling of tokens
or actions (``autodrive_b200.ops.sampling``), the group norm with an activation
(``autodrive_b200.ops.groupnorm``) and the AdamW step over many tensors
(``autodrive_b200.ops.adamw``).

``run`` computes a case in plain torch operations, or, where ``own`` is true,
with the framework's kernels; ``exact`` computes it in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 256            # elements of a tensor that share a scale of the 8-bit moments
E4M3_MAX = 448.

# the parameters of the raster scorer with a recurrent context, of the entity network and of the large raster network
RASTER_SCORER = (
    [(24, 6, 3, 3), (24,), (24,), (24,), (24, 24, 3, 3), (24,), (24,), (24,), (32, 24, 3, 3), (32,), (32,), (32,),
     (32, 32, 3, 3), (32,), (32,), (32,), (64, 32, 3, 3), (64,), (64,), (64,), (64, 64, 3, 3), (64,), (64,), (64,),
     (64, 7), (64,), (64, 64), (64,), (192, 64), (192, 64), (192,), (192,), (64, 128, 1, 1), (64,), (32, 96, 3, 3),
     (32,), (32,), (32,), (32, 32, 3, 3), (32,), (32,), (32,), (24, 56, 3, 3), (24,), (24,), (24,), (24, 24, 3, 3),
     (24,), (24,), (24,), (16, 24, 1, 1), (16,), (5, 64), (5,)])
ENTITY_NETWORK = (
    [(256, 137), (256,), (256, 12), (256,)]
    + 2 * [(256,), (256,), (768, 256), (768,), (256, 256), (256,), (256,), (256,), (1024, 256), (1024,), (256, 1024),
           (256,)]
    + [(256,), (256,), (1536, 256), (1536,), (1024, 1536), (1024,), (8, 1024), (8,), (1, 1024), (1,)])
RASTER_NETWORK = (
    [(128, 12, 3, 3), (128,)] + 5 * [(128, 128, 3, 3), (128,)]
    + [(256, 137), (256,), (1408, 16640), (1408,), (256, 1408), (256,), (8, 256), (8,), (1, 256), (1,)])
# a few wide layers with odd widths among them
WIDE_LAYERS = 8 * [(4096, 4096), (4096,)] + [(4096, 8191), (8191, 4096), (8191,), (1001, 4096), (1,)]
TENSORS = {"raster scorer": RASTER_SCORER, "entity network": ENTITY_NETWORK, "raster network": RASTER_NETWORK,
           "wide layers": WIDE_LAYERS}


def listed():
    return [
        # one robot's strategic action among the valid ones: launch latency
        {"name": "sample one action", "op": "sample", "rows": 1, "v": 8, "dtype": "fp32", "mask": True,
         "temperature": 1., "top_k": 0, "top_p": 1., "min_p": 0., "per_row": False},
        # a rollout step of 2048 worlds x 3 robots, each robot with a temperature and cut-offs of its own
        {"name": "sample rollout actions", "op": "sample", "rows": 6144, "v": 8, "dtype": "fp32", "mask": True,
         "temperature": .7, "top_k": 5, "top_p": .9, "min_p": .02, "per_row": True},
        # the next token of two sequences
        {"name": "sample next token", "op": "sample", "rows": 2, "v": 131072, "dtype": "bf16", "mask": False,
         "temperature": .7, "top_k": 50, "top_p": .9, "min_p": 0., "per_row": False},
        # a batch of next tokens whose cut-off falls among thousands of entries
        {"name": "sample tokens", "op": "sample", "rows": 2047, "v": 32003, "dtype": "bf16", "mask": False,
         "temperature": 1., "top_k": 0, "top_p": .95, "min_p": 0., "per_row": False},
        # one raster on its way through the raster scorer: launch latency
        {"name": "group norm one raster", "op": "group_norm", "mode": "forward", "n": 1, "c": 24, "groups": 8, "h": 25,
         "w": 51, "dtype": "fp32", "act": "silu"},
        # a minibatch of rasters through the raster scorer's first level, forward and backward
        {"name": "group norm rasters", "op": "group_norm", "mode": "train", "n": 512, "c": 24, "groups": 8, "h": 25,
         "w": 51, "dtype": "fp32", "act": "silu"},
        # a layer of the large raster network's width
        {"name": "group norm wide", "op": "group_norm", "mode": "train", "n": 384, "c": 128, "groups": 32, "h": 32,
         "w": 64, "dtype": "bf16", "act": "silu"},
        # few large images with an odd side and channels that fill no vector
        {"name": "group norm images", "op": "group_norm", "mode": "train", "n": 3, "c": 36, "groups": 4, "h": 257,
         "w": 263, "dtype": "fp16", "act": "relu"},
        # a step of the raster scorer, its gradients clipped: many small tensors
        {"name": "step raster scorer", "op": "adamw", "tensors": "raster scorer", "dtype": "fp32", "grad": "fp32",
         "bits": 32, "clip": .5},
        # a step of the entity network
        {"name": "step entity network", "op": "adamw", "tensors": "entity network", "dtype": "fp32", "grad": "fp32",
         "bits": 32, "clip": .5},
        # a step of the large raster network with its moments in 8 bits
        {"name": "step raster network 8 bits", "op": "adamw", "tensors": "raster network", "dtype": "fp32",
         "grad": "fp32", "bits": 8, "clip": 0.},
        # a step of wide 16-bit layers with the moments in 8 bits
        {"name": "step wide layers 8 bits", "op": "adamw", "tensors": "wide layers", "dtype": "bf16", "grad": "bf16",
         "bits": 8, "clip": 1.},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(("sample", "group_norm", "adamw"))
    if op == "sample":
        v = _log_int(rng, 2, 200_000)
        return {"op": op, "rows": _log_int(rng, 1, min(16384, 2047 * 32003 // v)), "v": v,
                "dtype": rng.choice(("bf16", "fp32", "fp16")), "mask": rng.random() < .4,
                "temperature": rng.choice((.3, .7, 1., 1.5)), "top_k": rng.choice((0, 0, 1, 5, 50, 1000)),
                "top_p": rng.choice((1., .5, .9, .95)), "min_p": rng.choice((0., 0., .02, .2)),
                "per_row": rng.random() < .3}
    if op == "group_norm":
        groups, per = rng.choice((1, 2, 4, 8, 32)), _log_int(rng, 1, 40)
        h, w = _log_int(rng, 1, 300), _log_int(rng, 1, 300)
        w = max(1, min(w, 50_000_000 // (groups * per * h)))
        most = 50_000_000 // (groups * per * h * w)
        return {"op": op, "mode": rng.choice(("forward", "train", "train")), "n": _log_int(rng, 1, max(1, min(4096, most))),
                "c": groups * per, "groups": groups, "h": h, "w": w, "dtype": rng.choice(("bf16", "fp16", "fp32")),
                "act": rng.choice(("silu", "silu", "relu", "gelu", "none"))}
    # `count` tensors of all sizes between one element and `largest`
    dtype = rng.choice(("fp32", "fp32", "bf16", "fp16"))
    return {"op": op, "tensors": "drawn", "count": _log_int(rng, 1, 300), "largest": _log_int(rng, 100, 4_000_000),
            "sizes": rng.randrange(1 << 30), "dtype": dtype, "grad": rng.choice((dtype, dtype, "fp32")),
            "bits": rng.choice((32, 8)), "clip": rng.choice((0., .5))}


def _shapes(case):
    if case["tensors"] != "drawn":
        return TENSORS[case["tensors"]]
    g = torch.Generator().manual_seed(case["sizes"])
    return [(int(case["largest"] ** u),) for u in torch.rand(case["count"], generator=g, dtype=torch.float64).tolist()]


# ------------------------------------------------------------------ inputs
def _to_e4m3(t):
    """The e4m3 value nearest to each 64-bit value, of at most 448."""
    _, exponent = torch.frexp(t)
    step = torch.ldexp(torch.ones_like(t), exponent.clamp_min(-5) - 4)
    return (torch.round(t / step) * step).float().to(torch.float8_e4m3fn)


def _block_scale(t):
    """(blocks of 256, largest magnitude / 448 of each, at least the smallest normal number, held in 32 bits)."""
    blocks = t.view(-1, BLOCK)
    amax = blocks.abs().amax(-1, keepdim=True).clamp_min(E4M3_MAX * 2. ** -126)
    return blocks, (amax.double() / E4M3_MAX).float()


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(shape, device=dev, generator=g)

    def uniform(*shape):
        return torch.rand(shape, device=dev, generator=g)

    op, s = case["op"], {"case": case}
    if op == "sample":
        rows, v = case["rows"], case["v"]
        s["logits"] = (3. * normal(rows, v)).to(DTYPES[case["dtype"]])
        s["uniforms"] = uniform(rows)
        s["mask"] = None
        if case["mask"]:
            # about a third of the entries is invalid, and one row in 64 has none at all
            s["mask"] = uniform(rows, v) < .66
            s["mask"][5::64] = False
        s["temperature"], s["top_k"], s["top_p"], s["min_p"] = (case[k] for k in ("temperature", "top_k", "top_p", "min_p"))
        if case["per_row"]:
            # requests of their own: about a tenth takes the most probable entry, some have no cut-off
            s["temperature"] = torch.where(uniform(rows) < .1, 0., case["temperature"] * (.5 + uniform(rows)))
            s["top_k"] = torch.randint(0, 2 * case["top_k"] + 2, (rows,), device=dev, generator=g)
            s["top_p"] = torch.where(uniform(rows) < .2, 1., case["top_p"] * (.6 + .4 * uniform(rows)))
            s["min_p"] = case["min_p"] * uniform(rows)
    elif op == "group_norm":
        dt, n, c, train = DTYPES[case["dtype"]], case["n"], case["c"], case["mode"] == "train"
        # channels of different size and offset, in channels-last memory
        def image():
            return normal(n, case["h"], case["w"], c)
        x = image() * (.5 * normal(c)).exp() + normal(c)
        s["x"] = x.to(dt).permute(0, 3, 1, 2).requires_grad_(train)
        s["weight"] = (1. + .2 * normal(c)).requires_grad_(train)
        s["bias"] = (.2 * normal(c)).requires_grad_(train)
        if train:
            s["dy"] = image().to(dt).permute(0, 3, 1, 2)
    else:
        # parameters, gradients and moments as views of one buffer each, every tensor at a multiple of 256 elements
        shapes = _shapes(case)
        sizes = [math.prod(shape) for shape in shapes]
        starts, total = [], 0
        for n in sizes:
            starts.append(total)
            total += -(-n // BLOCK) * BLOCK
        # each tensor's own magnitude of gradients, and what pads a tensor to whole blocks is zero
        blocks = torch.tensor([-(-n // BLOCK) for n in sizes], device=dev)
        size_of = (2. * normal(len(sizes)) - 6.).exp().repeat_interleave(blocks)[:, None]
        left = (torch.tensor(sizes, device=dev).repeat_interleave(blocks)
                - BLOCK * (torch.arange(total // BLOCK, device=dev) - torch.tensor(starts, device=dev).div(BLOCK, rounding_mode="floor").repeat_interleave(blocks)))
        real = torch.arange(BLOCK, device=dev) < left[:, None]

        def flat(t):
            return torch.where(real, t, 0.).view(-1)

        def views(t):
            return [t[o:o + n].view(shape) for o, n, shape in zip(starts, sizes, shapes)]

        each = (total // BLOCK, BLOCK)
        s["flat"] = {"param": flat(.05 * normal(*each)).to(DTYPES[case["dtype"]]),
                     "grad": flat(size_of * normal(*each)).to(DTYPES[case["grad"]])}
        m = flat(.3 * size_of * normal(*each))
        # the square root of the second moment
        r = flat(size_of * (.3 * normal(*each)).exp())
        if case["bits"] == 32:
            s["flat"]["exp_avg"], s["flat"]["exp_avg_sq"] = m, r.square()
        else:
            for name, t in (("exp_avg", m), ("exp_avg_sq", r)):
                b, scale = _block_scale(t)
                s["flat"][name] = _to_e4m3(b.double() / scale.double()).view(-1)
                s["flat"][name + "_scale"] = scale.view(-1)
        s["lists"] = {k: views(t) for k, t in s["flat"].items() if not k.endswith("_scale")}
        for k in ("exp_avg_scale", "exp_avg_sq_scale"):
            if k in s["flat"]:
                s["lists"][k] = [s["flat"][k][o // BLOCK:o // BLOCK - (-n // BLOCK)] for o, n in zip(starts, sizes)]
        s["step"] = 20
    return s


# ------------------------------------------------------------------ one pass
EPS = {"group_norm": 1e-5, "adamw": 1e-5}
LR, BETAS, DECAY, SEED = 3e-4, (.9, .999), .01, 7


def _plain_sample(s):
    case = s["case"]
    rows, v = case["rows"], case["v"]
    dev = s["logits"].device

    def column(value, dtype):
        return torch.as_tensor(value, dtype=dtype, device=dev).expand(rows)[:, None]

    z = s["logits"].float()
    if s["mask"] is not None:
        z = torch.where(s["mask"], z, -torch.inf)
    top = z.amax(-1, keepdim=True)
    empty = top == -torch.inf
    top = torch.where(empty, 0., top)
    temperature = column(s["temperature"], torch.float64)
    greedy = temperature == 0
    # weights and their sums in 64 bits: which entry holds a given number hangs on the last bits of 32-bit ones
    scaled = (z.double() - top) / torch.where(greedy, 1., temperature)
    w = torch.where(greedy, (z == top).double(), torch.exp(scaled))
    w = torch.where(w >= column(s["min_p"], torch.float64), w, 0.)
    if case["top_k"] or case["top_p"] < 1 or case["per_row"]:
        _, index = torch.sort(z, dim=-1, descending=True, stable=True)
        ordered = w.gather(1, index)
        rank = torch.arange(v, device=dev)
        k = torch.where(greedy, 1, column(s["top_k"], torch.int64))
        ordered = torch.where((k == 0) | (rank < k), ordered, 0.)
        before = ordered.cumsum(-1)
        limit = column(s["top_p"], torch.float64)
        before, least = torch.nn.functional.pad(before[:, :-1], (1, 0)), limit * before[:, -1:]
        ordered = torch.where((limit >= 1) | (rank == 0) | (before < least), ordered, 0.)
        w = torch.zeros_like(w).scatter_(1, index, ordered)
    running = w.cumsum(-1)
    total = running[:, -1:]
    token = (running <= s["uniforms"].double()[:, None] * total).sum(-1, keepdim=True)
    # a number at the upper end takes the last kept entry
    token = torch.minimum(token, (running < total).sum(-1, keepdim=True)).clamp(max=v - 1)
    log_prob = torch.where(greedy, 0., scaled.gather(1, token)) - torch.log(total)
    return {"token": torch.where(empty, -1, token)[:, 0],
            "log_prob": torch.where(empty, -torch.inf, log_prob)[:, 0].float()}


def _own_sample(s):
    from autodrive_b200.ops.sampling import sample_tokens
    r = sample_tokens(s["logits"], s["uniforms"], mask=s["mask"], temperature=s["temperature"], top_k=s["top_k"],
                      top_p=s["top_p"], min_p=s["min_p"])
    return {"token": r.token, "log_prob": r.log_prob}


def _act(z, act):
    """(value, derivative) of the activation."""
    if act == "silu":
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p))
    if act == "relu":
        return z.clamp_min(0.), (z > 0).float()
    if act == "gelu":
        p = .5 * (1 + torch.erf(z * math.sqrt(.5)))
        return z * p, p + z * torch.exp(-.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return z, torch.ones_like(z)


def _plain_group_norm(s):
    case = s["case"]
    groups = (case["groups"], case["c"] // case["groups"])
    x, shape = s["x"].detach().float(), s["x"].shape
    x = x.unflatten(1, groups)
    centred = x - x.mean((2, 3, 4), keepdim=True)
    rstd = (centred.square().mean((2, 3, 4), keepdim=True) + EPS["group_norm"]).rsqrt()
    n = centred * rstd
    w, b = (s[k].detach().view(*groups, 1, 1) for k in ("weight", "bias"))
    y, slope = _act(n * w + b, case["act"])
    out = {"y": y.reshape(shape).to(s["x"].dtype)}
    if case["mode"] == "train":
        dz = s["dy"].float().unflatten(1, groups) * slope
        g = dz * w
        dx = rstd * (g - g.mean((2, 3, 4), keepdim=True) - n * (g * n).mean((2, 3, 4), keepdim=True))
        out["dx"] = dx.reshape(shape).to(s["x"].dtype)
        out["dweight"], out["dbias"] = (dz * n).sum((0, 3, 4)).flatten(), dz.sum((0, 3, 4)).flatten()
    return out


def _own_group_norm(s):
    from autodrive_b200.ops.groupnorm import group_norm
    case = s["case"]
    y = group_norm(s["x"], case["groups"], s["weight"], s["bias"], eps=EPS["group_norm"],
                   activation=None if case["act"] == "none" else case["act"])
    out = {"y": y}
    if case["mode"] == "train":
        out["dx"], out["dweight"], out["dbias"] = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
    return out


def _mix(x):
    """32 mixed bits of each 32-bit number (held in 64), by two rounds of multiplication and shifted exclusive or."""
    x = ((x ^ (x >> 16)) * 0x7feb352d) & 0xffffffff
    x = ((x ^ (x >> 15)) * 0x846ca68b) & 0xffffffff
    return x ^ (x >> 16)


def _dithered(t, bits):
    """The e4m3 number below or above each magnitude `t`, above with the probability of its distance from the one
    below: `bits` (16 random ones) are added below the last bit that stays."""
    normal = ((t.view(torch.int32) + (bits << 4)) & ~0xfffff).view(torch.float32)
    small = torch.floor(t * 512 + bits.float() / 65536) / 512
    return torch.where(t < 2. ** -6, small, normal).clamp(max=E4M3_MAX)


def _plain_adamw(s):
    case, f = s["case"], s["flat"]
    s["step"] += 1
    g = f["grad"].float()
    b1, b2 = BETAS
    out = {"params": f["param"]}
    if case["clip"]:
        norm = f["grad"].double().square().sum().sqrt()
        g = g * (case["clip"] / (norm + 1e-6)).clamp(max=1.).float()
        out["norm"] = norm.float()
    if case["bits"] == 8:
        m = (f["exp_avg"].float().view(-1, BLOCK) * f["exp_avg_scale"][:, None]).view(-1)
        v = (f["exp_avg_sq"].float().view(-1, BLOCK) * f["exp_avg_sq_scale"][:, None]).view(-1).square()
    else:
        m, v = f["exp_avg"], f["exp_avg_sq"]
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    root = v.sqrt()
    p = f["param"].float() * (1 - LR * DECAY)
    p = p - (LR / (1 - b1 ** s["step"])) * m / (root / math.sqrt(1 - b2 ** s["step"]) + EPS["adamw"])
    f["param"].copy_(p)
    if case["bits"] == 32:
        f["exp_avg"].copy_(m)
        f["exp_avg_sq"].copy_(v)
    else:
        h = _mix((torch.arange(m.numel(), device=m.device) + _mix(_mix(SEED) ^ s["step"])) & 0xffffffff).to(torch.int32).view(-1, BLOCK)
        bm, scale = _block_scale(m)
        code = _dithered(bm.abs() / scale, h & 0xffff)
        f["exp_avg"].copy_(torch.where(bm < 0, -code, code).view(-1))
        f["exp_avg_scale"].copy_(scale.view(-1))
        br, scale = _block_scale(root)
        code = _dithered(br / scale, (h >> 16) & 0xffff)
        # a root that is not zero stays so: it is divided by
        code = torch.where((br > 0) & (code == 0), 2. ** -9, code)
        f["exp_avg_sq"].copy_(code.view(-1))
        f["exp_avg_sq_scale"].copy_(scale.view(-1))
    out.update({k: t for k, t in f.items() if k.startswith("exp_")})
    return out


def _own_adamw(s):
    from autodrive_b200.ops.adamw import adamw_step
    case, lists, f = s["case"], s["lists"], s["flat"]
    s["step"] += 1
    norm = adamw_step(lists["param"], lists["grad"], lists["exp_avg"], lists["exp_avg_sq"],
                      lists.get("exp_avg_scale"), lists.get("exp_avg_sq_scale"), step=s["step"], lr=LR, betas=BETAS,
                      eps=EPS["adamw"], weight_decay=DECAY, max_grad_norm=case["clip"], seed=SEED)
    out = {"params": f["param"], **{k: t for k, t in f.items() if k.startswith("exp_")}}
    if case["clip"]:
        out["norm"] = norm
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"sample": _own_sample, "group_norm": _own_group_norm, "adamw": _own_adamw}[op](state)
    return {"sample": _plain_sample, "group_norm": _plain_group_norm, "adamw": _plain_adamw}[op](state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "sample":
        rows, n = case["rows"], case["rows"] * case["v"]
        return {"bytes": n * DTYPES[case["dtype"]].itemsize + (n if case["mask"] else 0) + 16 * rows
                + (20 * rows if case["per_row"] else 0), "flops": 6 * n}
    if op == "group_norm":
        n = case["n"] * case["c"] * case["h"] * case["w"]
        size, train = DTYPES[case["dtype"]].itemsize, case["mode"] == "train"
        # x in and y out; a training step reads dy and writes dx as well
        return {"bytes": size * n * (4 if train else 2) + case["c"] * (16 if train else 8),
                "flops": n * (30 if train else 12)}
    n = sum(math.prod(shape) for shape in _shapes(case))
    moments = 16 * n if case["bits"] == 32 else 4 * n + 16 * -(-n // BLOCK)
    return {"bytes": n * (2 * DTYPES[case["dtype"]].itemsize + DTYPES[case["grad"]].itemsize) + moments,
            "flops": n * (16 if case["bits"] == 32 else 50)}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_sample(s):
    """Row by row of a chunk: the entries that stay are found by their order, and the chosen one among them in the
    order of their indices."""
    case, parts = s["case"], []
    rows, v = case["rows"], case["v"]
    dev = s["logits"].device
    step = max(1, 8_000_000 // v)
    each = {k: torch.as_tensor(s[k], dtype=torch.float64, device=dev).expand(rows) for k in ("temperature", "top_k", "top_p", "min_p")}
    for r in range(0, rows, step):
        c = slice(r, min(rows, r + step))
        value = s["logits"][c].double()
        valid = torch.ones_like(value, dtype=torch.bool) if s["mask"] is None else s["mask"][c]
        none = ~valid.any(-1)
        value = value.masked_fill(~valid, -torch.inf).masked_fill(none[:, None], 0.)
        t, k, p, least = (each[n][c, None] for n in ("temperature", "top_k", "top_p", "min_p"))
        k = torch.where(t == 0, 1., torch.where(k == 0, float(v), k))
        value, index = torch.sort(value / torch.where(t == 0, 1., t), dim=-1, descending=True, stable=True)
        log_w = value - value[:, :1]
        weight = log_w.exp() * (log_w.exp() >= least) * (torch.arange(v, device=dev) < k)
        share = weight / weight.sum(-1, keepdim=True)
        above = share.cumsum(-1) - share
        keep = (weight > 0) & ((p >= 1) | (above < p) | (torch.arange(v, device=dev) == 0))
        share = share * keep / (share * keep).sum(-1, keepdim=True)
        place = index.argsort(-1)                              # of each index in the order
        by_index = share.gather(1, place)
        chosen = (by_index.cumsum(-1) > s["uniforms"][c, None].double()).double().argmax(-1, keepdim=True)
        log_prob = by_index.gather(1, chosen).log()[:, 0]
        parts.append(log_prob.masked_fill(none, -torch.inf))
    return {"token": None, "log_prob": torch.cat(parts)}


def _exact_group_norm(s):
    case = s["case"]
    x, w, b = (s[k].detach().double().contiguous().requires_grad_(True) for k in ("x", "weight", "bias"))
    rows = x.reshape(case["n"] * case["groups"], -1)
    mean = rows.sum(-1, keepdim=True) / rows.shape[1]
    var = ((rows - mean) ** 2).sum(-1, keepdim=True) / rows.shape[1]
    z = ((rows - mean) / torch.sqrt(var + EPS["group_norm"])).reshape(x.shape) * w[:, None, None] + b[:, None, None]
    y = {"silu": lambda: z / (1 + torch.exp(-z)), "relu": lambda: z * (z > 0), "none": lambda: z,
         "gelu": lambda: z * (1 - torch.special.erfc(z / 2 ** .5) / 2)}[case["act"]]()
    out = {"y": y.detach()}
    if case["mode"] == "train":
        out["dx"], out["dweight"], out["dbias"] = torch.autograd.grad(y, (x, w, b), s["dy"].double())
    return out


def _exact_code(t, scale, bits):
    """The e4m3 number at or below t / scale (`t` not negative), or the next one where 16 random bits say so."""
    q = t / scale
    exponent = torch.floor(torch.log2(q.clamp_min(2. ** -6)))
    grid = torch.exp2(exponent - 3)
    return torch.minimum(torch.floor(q / grid + bits.double() / 65536) * grid, torch.full_like(q, E4M3_MAX))


def _exact_adamw(s):
    case, lists = s["case"], s["lists"]
    step, bits8 = s["step"] + 1, case["bits"] == 8
    norm = torch.stack([g.double().square().sum() for g in lists["grad"]]).sum().sqrt()
    factor = (case["clip"] / (norm + 1e-6)).clamp(max=1.) if case["clip"] else 1.
    out = {k: torch.zeros(t.shape, dtype=torch.float64, device=t.device) for k, t in s["flat"].items() if k != "grad"}
    out["params"] = out.pop("param")
    # the random bits are counted over the tensors' whole blocks
    number = torch.arange(out["params"].numel(), device=norm.device)
    random = _mix((number + _mix(_mix(SEED) ^ step)) & 0xffffffff)
    at = 0
    for i, g in enumerate(lists["grad"]):
        n = g.numel()
        blocks = -(-n // BLOCK)
        of = torch.arange(n, device=norm.device) // BLOCK
        m, v = lists["exp_avg"][i].double().view(-1), lists["exp_avg_sq"][i].double().view(-1)
        if bits8:
            m = m * lists["exp_avg_scale"][i].double()[of]
            v = (v * lists["exp_avg_sq_scale"][i].double()[of]) ** 2
        g = g.double().view(-1) * factor
        m, v = m * BETAS[0] + (1 - BETAS[0]) * g, v * BETAS[1] + (1 - BETAS[1]) * g * g
        update = (m / (1 - BETAS[0] ** step)) / ((v / (1 - BETAS[1] ** step)).sqrt() + EPS["adamw"])
        out["params"][at:at + n] = lists["param"][i].double().view(-1) * (1 - LR * DECAY) - LR * update
        if bits8:
            h = random[at:at + n]
            for name, t, b in (("exp_avg", m, h & 0xffff), ("exp_avg_sq", v.sqrt(), h >> 16)):
                amax = torch.zeros(blocks, dtype=torch.float64, device=g.device).scatter_reduce_(0, of, t.abs(), "amax")
                scale = (amax.clamp_min(E4M3_MAX * 2. ** -126) / E4M3_MAX).float().double()
                code = _exact_code(t.abs(), scale[of], b)
                if name == "exp_avg_sq":
                    code = torch.where((t > 0) & (code == 0), 2. ** -9, code)
                out[name][at:at + n] = torch.where(t < 0, -code, code)
                out[name + "_scale"][at // BLOCK:at // BLOCK + blocks] = scale
        else:
            out["exp_avg"][at:at + n], out["exp_avg_sq"][at:at + n] = m, v
        at += blocks * BLOCK
    if case["clip"]:
        out["norm"] = norm
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"sample": _exact_sample, "group_norm": _exact_group_norm, "adamw": _exact_adamw}[case["op"]](s)
