"""Workloads of the row operators of a training step: layer norm over feature rows, products with one weight matrix per row group, and the
AdamW step over many tensors with states in 32 or 8 bits.

A case is a dict of plain values.  ``run`` is one pass through an operator: with ``own`` false in elementary tensor operations, with ``own``
true through this package's entry points.  ``exact`` is the same result from the definition, in float64."""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS_NORM = 1e-5
LR, BETAS, EPS_ADAM, DECAY, STEP, SEED = 2e-3, (0.9, 0.99), 1e-8, 0.01, 400, 20
BLOCK = 128     # elements that share an exponent in the 8-bit states


def listed():
    return [
        # a head's pooled features of one frame at inference: 512 proposals of 256 channels, all launch latency
        {"name": "norm_proposals", "op": "norm", "rows": 512, "cols": 256, "type": "f32", "params": "f32", "train": False},
        # the first-stage voxel rows of a 4-frame training batch (133 578 rows) at the backbone's widest 64 channels: short rows, many of them
        {"name": "norm_voxels", "op": "norm", "rows": 133578, "cols": 64, "type": "f32", "params": "f32", "train": True},
        # wide rows in 16 bits with fp32 weights, an odd number of rows: the bandwidth case, forward and backward
        {"name": "norm_wide", "op": "norm", "rows": 16381, "cols": 4096, "type": "bf16", "params": "f32", "train": True},
        # one weight matrix per class over a frame's proposals, odd sizes in every direction, inference
        {"name": "group_classes", "op": "group", "groups": 3, "rows": 517, "inner": 250, "outer": 129, "type": "f16", "train": False, "spread": 1.0},
        # voxel rows grouped by frame at 64 channels, trained in fp32: few flops a byte
        {"name": "group_voxels", "op": "group", "groups": 4, "rows": 133578, "inner": 64, "outer": 64, "type": "f32", "train": True, "spread": 4.0},
        # the pooled-grid features of the RoI head (27 648 = 6 x 6 x 6 cells x 128) into 256 channels, per class: a long inner axis, few rows
        {"name": "group_pooled", "op": "group", "groups": 3, "rows": 480, "inner": 27648, "outer": 256, "type": "f32", "train": True, "spread": 4.0},
        # one row for most of 64 weight matrices: single tokens, the weights' bandwidth
        {"name": "group_single", "op": "group", "groups": 64, "rows": 64, "inner": 2048, "outer": 2048, "type": "bf16", "train": False, "spread": 4.0},
        # routed rows in training: ragged groups, matrix-unit work in all three products
        {"name": "group_routed", "op": "group", "groups": 16, "rows": 32749, "inner": 1024, "outer": 4096, "type": "bf16", "train": True, "spread": 3.0},
        # the backbone's parameters: a few dozen weights and as many channel vectors, 0.4 M elements: launch latency
        {"name": "adamw_backbone", "op": "adamw", "bits": 32, "tensors": 87, "elements": 420_000, "type": "f32", "pattern": 1},
        # a whole detector, 13 M parameters, most of them in the head's first matrix
        {"name": "adamw_detector", "op": "adamw", "bits": 32, "tensors": 193, "elements": 13_000_000, "type": "f32", "pattern": 2},
        # the same with states in 8 bits
        {"name": "adamw_detector_8bit", "op": "adamw", "bits": 8, "tensors": 193, "elements": 13_000_000, "type": "f32", "pattern": 2},
        # a large model held in bf16 with states in 8 bits: 6 bytes of model and state an element
        {"name": "adamw_large_8bit", "op": "adamw", "bits": 8, "tensors": 291, "elements": 200_000_000, "type": "bf16", "pattern": 3},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "group", "group", "adamw"])
    if op == "norm":
        cols = _log(rng, 4, 16384)
        kind = rng.choice(["f32", "f16", "bf16"])
        return {"op": op, "rows": _log(rng, 1, min(500_000, 16381 * 4096 // (2 * cols))), "cols": cols, "type": kind,
                "params": rng.choice(["f32", kind]), "train": rng.random() < 0.7}
    if op == "group":
        inner, outer = (_log(rng, 1024, 27648), _log(rng, 16, 256)) if rng.random() < 0.2 else (_log(rng, 8, 4096), _log(rng, 8, 4096))
        kind = rng.choice(["f32", "f16", "bf16"])
        most = (32749 * 1024 * 4096 // (4 if kind == "f32" else 1)) // (inner * outer)
        # the weights stay below 64 x 2048 x 2048 elements (16-bit) however many groups there are
        groups = _log(rng, 1, max(1, min(128, (64 << 22) // (2 * inner * outer))))
        return {"op": op, "groups": groups, "rows": _log(rng, 1, max(1, min(133578, most))), "inner": inner,
                "outer": outer, "type": kind, "train": rng.random() < 0.6, "spread": rng.choice([0.3, 1.0, 4.0])}
    elements = _log(rng, 10_000, 100_000_000)
    return {"op": op, "bits": rng.choice([8, 32]), "tensors": _log(rng, 1, min(400, elements // 100)), "elements": elements,
            "type": rng.choice(["f32", "bf16"]), "pattern": rng.randrange(1 << 20)}


def work(case):
    if case["op"] == "norm":
        n, s, c = case["rows"] * case["cols"], DTYPES[case["type"]].itemsize, case["cols"] * DTYPES[case["params"]].itemsize
        # forward: x in, y out, weight and bias in; backward: x and dy in, dx out, weight in, two gradients out
        return {"bytes": (5 * n * s + 5 * c) if case["train"] else (2 * n * s + 2 * c), "flops": 20 * n if case["train"] else 8 * n}
    if case["op"] == "group":
        s = DTYPES[case["type"]].itemsize
        x, y = case["rows"] * case["inner"] * s, case["rows"] * case["outer"] * s
        w, b = case["groups"] * case["inner"] * case["outer"] * s, case["groups"] * case["outer"] * s
        one = 2 * case["rows"] * case["inner"] * case["outer"]
        if not case["train"]:
            # a group without rows needs no weights: the share of groups that have some, over a few seeds
            used = [sum(a < b for a, b in zip(e, e[1:])) for e in (_group_sizes(case, seed) for seed in range(8))]
            w = w * sum(used) // (8 * case["groups"])
            return {"bytes": x + w + b + y, "flops": one}
        # forward; then dy and w in, dx out; dy and x in, dw and db out
        return {"bytes": (x + w + b + y) + (y + w + x) + (y + x + w + b), "flops": 3 * one}
    n, s = case["elements"], DTYPES[case["type"]].itemsize
    state = 8 if case["bits"] == 32 else 2 + 2 / BLOCK
    return {"bytes": int(n * (3 * s + 2 * state)), "flops": 15 * n}


def _sizes(case):
    """Sizes of the tensors of a model: half of them channel vectors, the others weights over two decades, their sum as asked."""
    rng = random.Random(case["pattern"])
    t, left = case["tensors"], case["elements"]
    vectors = [min(rng.choice([16, 32, 64, 64, 128, 256, 77]), left // (2 * t)) for _ in range(t // 2)]
    left -= sum(vectors)
    share = [math.exp(rng.uniform(0.0, 4.6)) for _ in range(t - t // 2)]
    weights = [max(1, int(left * s / sum(share))) for s in share]
    weights[0] += left - sum(weights)
    sizes = vectors + weights
    rng.shuffle(sizes)
    return [max(1, n) for n in sizes]


def _group_sizes(case, seed):
    """Rows of each group: gamma-distributed shares (`spread` below 1 leaves some groups empty), their sum as asked."""
    rng = random.Random(seed * 7919 + 13)
    share = [rng.gammavariate(case["spread"], 1.0) + 1e-9 for _ in range(case["groups"])]
    total, ends, at = sum(share), [0], 0.0
    for s in share:
        at += s
        ends.append(int(round(case["rows"] * at / total)))
    ends[-1] = case["rows"]
    return ends


def _power(k):
    """2^k in fp32, exactly, for integers -126 <= k <= 127."""
    return ((k + 127) << 23).to(torch.int32).view(torch.float32)


def _to_8bit(x):
    """An fp32 vector of whole blocks as (e4m3 values, a power of two per block), to nearest: what a checkpoint holds."""
    blocks = x.view(-1, BLOCK)
    exponent = torch.frexp(blocks.abs().amax(1))[1].clamp(-118, 127) - 1
    return (blocks * _power(7 - exponent[:, None])).to(torch.float8_e4m3fn).view(-1), exponent.to(torch.int8)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return torch.empty(shape, device=dev).normal_(0.0, scale, generator=g).to(dtype)

    state = {"case": case}
    dtype = DTYPES[case["type"]]
    if case["op"] == "norm":
        rows, cols, pdt = case["rows"], case["cols"], DTYPES[case["params"]]
        # features with a channel-dependent offset, as they leave a convolution or a residual sum
        state["x"] = (normal(rows, cols) * 1.5 + normal(cols)).to(dtype)
        state["weight"] = (1.0 + normal(cols, scale=0.1)).to(pdt)
        state["bias"] = normal(cols, scale=0.1, dtype=pdt)
        if case["train"]:
            state["dy"] = normal(rows, cols, scale=1e-2, dtype=dtype)
            for k in ("x", "weight", "bias"):
                state[k].requires_grad_()
    elif case["op"] == "group":
        ends = _group_sizes(case, seed)
        state["most"] = max(b - a for a, b in zip(ends, ends[1:]))
        state["offsets"] = torch.tensor(ends, dtype=torch.int32, device=dev)
        state["x"] = normal(case["rows"], case["inner"], dtype=dtype)
        state["weight"] = normal(case["groups"], case["outer"], case["inner"], scale=case["inner"] ** -0.5, dtype=dtype)
        state["bias"] = normal(case["groups"], case["outer"], scale=0.1, dtype=dtype)
        if case["train"]:
            state["dy"] = normal(case["rows"], case["outer"], scale=1e-1, dtype=dtype)
            for k in ("x", "weight", "bias"):
                state[k].requires_grad_()
    else:
        # the tensors of a model lie in one allocation, each from a multiple of BLOCK elements on, with zeros between them
        sizes = _sizes(case)
        padded = [n + -n % BLOCK for n in sizes]
        rng = random.Random(seed)

        def apart(flat):
            return [t[:n] for t, n in zip(flat.split(padded), sizes)]

        inside = torch.zeros(sum(padded), dtype=torch.bool, device=dev)
        torch._foreach_add_(apart(inside), True)
        # each tensor's gradients have a scale of their own, and within a tensor they spread over a few binades
        scale = torch.tensor([10.0 ** rng.uniform(-5, -2) for _ in sizes], device=dev).repeat_interleave(torch.tensor(padded, device=dev))
        m, v = (normal(sum(padded)) * torch.exp(normal(sum(padded))) * scale * inside for _ in range(2))
        grad = (normal(sum(padded)) * torch.exp(normal(sum(padded))) * scale * inside).to(dtype)
        m, v = 0.3 * m, (0.5 * v * v + 0.1 * scale * scale) * inside
        state.update(step=STEP, sizes=sizes, padded=padded, flat={"params": normal(sum(padded), scale=0.05).mul_(inside).to(dtype)})
        state["grads"], state["flat_grads"] = apart(grad), grad
        if case["bits"] == 32:
            state["flat"].update(exp_avgs=m, exp_avg_sqs=v)
        else:
            (m, a), (r, b) = _to_8bit(m), _to_8bit(v.sqrt())
            state["flat"].update(exp_avgs=m, exp_avg_rmss=r, exponents=torch.stack((a, b), 1))
            state["exponents"] = list(state["flat"]["exponents"].split([n // BLOCK for n in padded]))
        for k in ("params", "exp_avgs", "exp_avg_sqs", "exp_avg_rmss"):
            if k in state["flat"]:
                state[k] = apart(state["flat"][k])
    return state


# ---------------------------------------------------------------------------------------------------------------- passes
def run(state):
    case = state["case"]
    if case["op"] == "norm":
        return _norm(state, case["train"])
    if case["op"] == "group":
        return _group(state, case["train"])
    state["step"] += 1
    return _adamw_32(state) if case["bits"] == 32 else _adamw_8(state)


def _norm(state, train):
    x, weight, bias = state["x"], state["weight"], state["bias"]
    if own:
        from virconv_amd import ops
        y = ops.layer_norm(x, weight, bias, EPS_NORM)
        if not train:
            return y
        return (y.detach(), *torch.autograd.grad(y, (x, weight, bias), state["dy"]))
    with torch.no_grad():
        a, w = x.float(), weight.float()
        mean = a.mean(1, keepdim=True)
        a = a - mean
        rstd = torch.rsqrt((a * a).mean(1, keepdim=True) + EPS_NORM)
        hat = a * rstd
        y = (hat * w + bias.float()).to(x.dtype)
        if not train:
            return y
        dy = state["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
        return y, dx.to(x.dtype), (dy * hat).sum(0).to(weight.dtype), dy.sum(0).to(bias.dtype)


def _group(state, train):
    x, weight, bias, offsets = state["x"], state["weight"], state["bias"], state["offsets"]
    if own:
        from virconv_amd import ops
        y = ops.grouped_linear(x, weight, offsets, bias)
        if not train:
            return y
        return (y.detach(), *torch.autograd.grad(y, (x, weight, bias), state["dy"]))
    with torch.no_grad():
        # every group padded to the largest one, so that each product is one batch of products
        first, last = offsets[:-1].long(), offsets[1:].long()
        at = first[:, None] + torch.arange(state["most"], device=x.device)
        inside = (at < last[:, None])[:, :, None]
        at = at.clamp(max=x.shape[0] - 1)
        rows = torch.arange(x.shape[0], device=x.device)
        group = torch.searchsorted(last, rows, right=True)
        place = rows - first[group]
        a, w = x.float()[at] * inside, weight.float()
        y = (torch.bmm(a, w.transpose(1, 2)) + bias.float()[:, None])[group, place].to(x.dtype)
        if not train:
            return y
        d = state["dy"].float()[at] * inside
        dx = torch.bmm(d, w)[group, place]
        dw = torch.bmm(d.transpose(1, 2), a)
        return y, dx.to(x.dtype), dw.to(weight.dtype), d.sum(1).to(bias.dtype)


def _scalars(step):
    """(1 - lr wd, step size, 1 / sqrt(1 - beta2^t)) of a step."""
    return 1.0 - LR * DECAY, LR / (1.0 - BETAS[0] ** step), 1.0 / math.sqrt(1.0 - BETAS[1] ** step)


def _optimizer(state, bits, **moments):
    """The optimizer that a program keeps, made at the first pass, with the moments that it has by then."""
    if "optimizer" not in state:
        from virconv_amd import optim
        state["optimizer"] = optim.AdamW(state["params"], lr=LR, betas=BETAS, eps=EPS_ADAM, weight_decay=DECAY, state_bits=bits, seed=SEED)
        for k, (p, g) in enumerate(zip(state["params"], state["grads"])):
            p.grad = g
            state["optimizer"].state[p].update(step=state["step"] - 1, **{name: t[k] for name, t in moments.items()})
    return state["optimizer"]


def _adamw_32(state):
    flat = state["flat"]
    if own:
        _optimizer(state, 32, exp_avg=state["exp_avgs"], exp_avg_sq=state["exp_avg_sqs"]).step()
        return flat
    keep, size, scale = _scalars(state["step"])
    g = state["flat_grads"].float()
    m = flat["exp_avgs"].mul_(BETAS[0]).add_(g * (1.0 - BETAS[0]))
    v = flat["exp_avg_sqs"].mul_(BETAS[1]).add_(g * g * (1.0 - BETAS[1]))
    flat["params"].copy_(flat["params"].float() * keep - size * (m / (v.sqrt() * scale + EPS_ADAM)))
    return flat


def _mix(x):
    """The 32-bit mixing function of the rounding's random numbers, on int64 tensors or Python numbers in [0, 2^32)."""
    x = x ^ (x >> 16)
    x = (x * 0x85EBCA6B) & 0xFFFFFFFF
    x = x ^ (x >> 13)
    x = (x * 0xC2B2AE35) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _random(sizes, padded, step, device):
    """32 random bits for every element: a function of the seed, the step, the tensor's place in the list and the element's in the tensor."""
    key = _mix(_mix(SEED) + step & 0xFFFFFFFF)
    keys = torch.tensor([_mix(key + k & 0xFFFFFFFF) for k in range(len(sizes))], device=device)
    blocks = torch.tensor(padded, device=device) // BLOCK
    tensor = torch.repeat_interleave(torch.arange(len(sizes), device=device), blocks, output_size=sum(padded) // BLOCK)
    first = (torch.cumsum(blocks, 0) - blocks)[tensor]
    at = (torch.arange(sum(padded) // BLOCK, device=device) - first)[:, None] * BLOCK + torch.arange(BLOCK, device=device)
    return _mix(keys[tensor][:, None] ^ at)


def _round_e4m3(y, bits):
    """|y| < 256 to a neighbouring e4m3 value, up with the probability of its distance from the lower one; 16 random bits each.
    Below 2^-6 the values are 2^-9 apart, as they are in the binade above it: there the rounding is done with 2^-6 added."""
    low = y < 2.0 ** -6
    z = torch.where(low, y + 2.0 ** -6, y)
    z = ((z.view(torch.int32) + (bits << 4).to(torch.int32)) & ~0xFFFFF).view(torch.float32)
    return torch.where(low, z - 2.0 ** -6, z)


def _encode(x, top, bits):
    """Blocks of fp32 values as e4m3 values over 2^exponent; `top`: the block's exponent."""
    return torch.copysign(_round_e4m3(x.abs() * _power(7 - top[:, None]), bits), x).to(torch.float8_e4m3fn)


def _adamw_8(state):
    flat = state["flat"]
    if own:
        _optimizer(state, 8, exp_avg=state["exp_avgs"], exp_avg_rms=state["exp_avg_rmss"], exponents=state["exponents"]).step()
        return flat
    keep, size, scale = _scalars(state["step"])
    p, g, m, r = (t.view(-1, BLOCK).float() for t in (flat["params"], state["flat_grads"], flat["exp_avgs"], flat["exp_avg_rmss"]))
    unit = _power(flat["exponents"].int() - 7)
    m, r = m * unit[:, :1], r * unit[:, 1:]
    m = m * BETAS[0] + g * (1.0 - BETAS[0])
    v = r * r * BETAS[1] + g * g * (1.0 - BETAS[1])
    r = v.sqrt()
    p = p * keep - size * (m / (r * scale + EPS_ADAM))
    # the exponent of a block: its largest magnitude lies in [2^e, 2^(e + 1)); -119 or more, so that the scale of its values stays a number
    most = torch.stack((m.abs().amax(1), r.amax(1)), 1)
    top = torch.where(most > 0, torch.frexp(most)[1] - 1, -119).clamp(min=-119)
    bits = _random(state["sizes"], state["padded"], state["step"], p.device)
    flat["params"].view(-1, BLOCK).copy_(p)
    flat["exp_avgs"].view(-1, BLOCK).copy_(_encode(m, top[:, 0], bits & 0xFFFF))
    flat["exp_avg_rmss"].view(-1, BLOCK).copy_(_encode(r, top[:, 1], bits >> 16))
    flat["exponents"].copy_(top)
    return flat


# ---------------------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "group": _exact_group, "adamw": _exact_adamw}[case["op"]](case, state)


def _exact_norm(case, state):
    x, w, b = (state[k].double() for k in ("x", "weight", "bias"))
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    sd = torch.sqrt(var + EPS_NORM)
    hat = (x - mean) / sd
    y = torch.addcmul(b, hat, w)
    if not case["train"]:
        return y
    dy = state["dy"].double()
    inner = (dy * w).sum(1, keepdim=True), (dy * w * hat).sum(1, keepdim=True)
    dx = (case["cols"] * dy * w - inner[0] - hat * inner[1]) / (case["cols"] * sd)
    return y, dx, torch.einsum("rc,rc->c", dy, hat), dy.sum(0)


def _exact_group(case, state):
    x, w, b = (state[k].double() for k in ("x", "weight", "bias"))
    ends = state["offsets"].tolist()
    y = torch.empty(case["rows"], case["outer"], dtype=torch.float64, device=x.device)
    for g, (i, j) in enumerate(zip(ends, ends[1:])):
        y[i:j] = x[i:j] @ w[g].T + b[g]
    if not case["train"]:
        return y
    dy = state["dy"].double()
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    for g, (i, j) in enumerate(zip(ends, ends[1:])):
        dx[i:j], dw[g], db[g] = dy[i:j] @ w[g], dy[i:j].T @ x[i:j], dy[i:j].sum(0)
    return y, dx, dw, db


def _exact_adamw(case, state):
    step = state["step"] + 1
    out = {k: torch.zeros(t.shape, dtype=torch.float64, device=t.device) for k, t in state["flat"].items()}
    key, at = _mix(_mix(SEED) + step & 0xFFFFFFFF), 0
    for k, (p, g, m, n) in enumerate(zip(state["params"], state["grads"], state["exp_avgs"], state["padded"])):
        here = slice(at, at + p.numel())
        p, g, m = p.double(), g.double(), m.double()
        if case["bits"] == 8:
            e = (2.0 ** (state["exponents"][k].double() - 7)).repeat_interleave(BLOCK, 0)[:p.numel()]
            m, v = m * e[:, 0], (state["exp_avg_rmss"][k].double() * e[:, 1]) ** 2
        else:
            v = state["exp_avg_sqs"][k].double()
        m = m + (1.0 - BETAS[0]) * (g - m)
        v = v + (1.0 - BETAS[1]) * (g ** 2 - v)
        out["params"][here] = p - LR * DECAY * p - LR * (m / (1.0 - BETAS[0] ** step)) / (torch.sqrt(v / (1.0 - BETAS[1] ** step)) + EPS_ADAM)
        if case["bits"] == 8:
            chance = _mix(torch.arange(p.numel(), device=p.device) ^ _mix(key + k & 0xFFFFFFFF))
            blocks = slice(at // BLOCK, (at + n) // BLOCK)
            out["exp_avgs"][here], out["exponents"][blocks, 0] = _exact_8bit(m, (chance & 0xFFFF).double() / 65536)
            out["exp_avg_rmss"][here], out["exponents"][blocks, 1] = _exact_8bit(torch.sqrt(v), (chance >> 16).double() / 65536)
        else:
            out["exp_avgs"][here], out["exp_avg_sqs"][here] = m, v
        at += n
    if case["bits"] == 8:
        out["exponents"] = out["exponents"].to(torch.int8)
    return out


def _exact_8bit(x, chance):
    """The definition of the 8-bit form: the block's largest magnitude scaled into [128, 256), every value rounded down to a multiple of
    its spacing (an eighth of its power of two, 2^-9 at the least) after `chance` of that spacing was added."""
    n = x.numel()
    most = torch.nn.functional.pad(x.abs(), (0, -n % BLOCK)).view(-1, BLOCK).amax(1)
    top = torch.where(most > 0, torch.floor(torch.log2(most.clamp(min=1e-300))), torch.full_like(most, -119.0)).clamp(min=-119.0)
    y = x.abs() * 2.0 ** (7 - top).repeat_interleave(BLOCK)[:n]
    spacing = 2.0 ** (torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)
    return torch.sign(x) * torch.floor(y / spacing + chance) * spacing, top
