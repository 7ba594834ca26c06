"""Group normalisation with an activation (channels last, forward and backward) and the AdamW step over many tensors (moments in
32 or in 8 bits, gradients clipped by their global norm): the calls of raft_amd, and the same operators in elementary torch
operations.

What the cases stand for: the norms of RAFT's encoders (instance norm = one channel a group, group norm with width // 8 groups)
at 1/2, 1/4 and 1/8 of the image, in inference and in training, and the optimizer step of a training run, from a handful of
small tensors to models some twenty times RAFT's size."""
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS_NORM = 1e-5
LR, BETAS, EPS, DECAY, SEED = 2e-4, (0.9, 0.999), 1e-8, 5e-5, 0
TILE, BLOCK = 512, 64           # a parameter's moments start at a multiple of TILE; 8-bit moments share one exponent a BLOCK


def _norm(name, n, c, h, w, groups, act, dtype, train):
    return {"name": name, "op": "norm", "n": n, "c": c, "h": h, "w": w, "groups": groups, "act": act, "dtype": dtype, "train": train}


def _adamw(name, tensors, total, bits, dtype, clip):
    return {"name": name, "op": "adamw", "tensors": tensors, "total": total, "bits": bits, "dtype": dtype, "clip": clip}


def listed():
    return [
        # the last stage of RAFT-small's feature encoder on a 200 x 320 frame: latency
        _norm("norm_small_map", 1, 96, 25, 40, 96, "relu", "fp32", False),
        # the stem of the feature encoder on a frame pair of 440 x 1024: instance norm + ReLU, inference
        _norm("norm_stem", 2, 64, 220, 512, 64, "relu", "fp32", False),
        # the second stage on a pair of 1088 x 1920 frames with 16-bit activations
        _norm("norm_hd_16bit", 2, 96, 272, 480, 96, "relu", "bf16", False),
        # the third stage in training on six pairs of 400 x 720 crops, 16-bit activations
        _norm("norm_train_stage3", 12, 128, 50, 90, 16, "relu", "fp16", True),
        # an odd map, channel count and group size
        _norm("norm_train_odd", 3, 42, 47, 157, 7, "silu", "bf16", True),
        # the stem in training on six pairs of 400 x 720 crops: the largest activation of the model
        _norm("norm_train_stem", 12, 64, 200, 360, 8, "relu", "fp32", True),
        # fine-tuning the flow head alone
        _adamw("adamw_head", 4, 300_000, 8, "bf16", 0.0),
        # RAFT-small and RAFT-basic: 106 and 124 tensors, clipped as in the training recipe
        _adamw("adamw_raft_small", 106, 990_162, 32, "fp32", 1.0),
        _adamw("adamw_raft_basic", 124, 5_257_536, 32, "fp32", 1.0),
        _adamw("adamw_raft_basic_8bit", 124, 5_257_536, 8, "fp32", 1.0),
        # a model of a hundred million parameters
        _adamw("adamw_large", 310, 100_000_000, 32, "fp32", 1.0),
        _adamw("adamw_large_8bit", 310, 100_000_000, 8, "bf16", 1.0),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        c = rng.choice([_log_uniform(rng, 3, 256), 8 * rng.randint(1, 32)])
        groups = rng.choice([g for g in range(1, c + 1) if c % g == 0])
        n = rng.randint(1, 12)
        rows = _log_uniform(rng, 60, min(500_000, 40_000_000 // (n * c)))
        h = max(1, min(rows, int(math.sqrt(rows * rng.uniform(0.3, 1.0)))))
        case = _norm("", n, c, h, max(1, rows // h), groups, rng.choice(["none", "relu", "relu", "silu"]),
                     rng.choice(list(DTYPES)), rng.random() < 0.6)
    else:
        total = _log_uniform(rng, 2_000, 60_000_000)
        case = _adamw("", _log_uniform(rng, 1, 400), total, rng.choice([8, 32]), rng.choice(["fp32", "bf16"]), rng.choice([0.0, 1.0]))
    del case["name"]
    return case


def _sizes(case):
    """The tensors' lengths: as in a convolutional model half of them are short vectors, the others hold the rest."""
    tensors, total = case["tensors"], case["total"]
    rng = random.Random(tensors * 1_000_003 + total)
    small = [min(rng.choice([2, 32, 64, 96, 126, 128, 192, 256, 576]), max(1, total // (2 * tensors))) for _ in range(tensors // 2)]
    share = [rng.uniform(0.05, 1.0) ** 2 for _ in range(tensors - len(small))]
    rest = total - sum(small)
    large = [max(1, int(rest * s / sum(share))) for s in share]
    large[-1] += max(0, rest - sum(large))
    sizes = small + large
    rng.shuffle(sizes)
    return sizes


def _inputs(case, seed):
    """What both the operators and their definition in 64 bits start from."""
    g = torch.Generator("cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if case["op"] == "norm":
        n, c, h, w, dtype = case["n"], case["c"], case["h"], case["w"], DTYPES[case["dtype"]]
        spread, shift = torch.exp(0.5 * randn(c)), randn(c)           # a convolution's outputs: each channel has its own mean and width
        x = (randn(n, h, w, c) * spread + shift).to(dtype).permute(0, 3, 1, 2)
        affine = case["groups"] < c                                    # instance norm has no weights
        weight = (1 + 0.3 * randn(c)) if affine else None
        bias = 0.3 * randn(c) if affine else None
        dy = (1e-3 * randn(n, h, w, c)).to(dtype).permute(0, 3, 1, 2) if case["train"] else None
        return {"x": x, "weight": weight, "bias": bias, "dy": dy}
    sizes, dtype = _sizes(case), DTYPES[case["dtype"]]
    starts, total = [], 0
    for n in sizes:
        starts.append(total)
        total += (n + TILE - 1) // TILE * TILE
    index, level = torch.arange(total, device="cuda"), torch.zeros(total, device="cuda")
    widths = torch.exp(torch.linspace(math.log(1e-5), math.log(1e-2), len(sizes))[torch.randperm(len(sizes), generator=torch.Generator().manual_seed(seed))]).tolist()
    for start, n, width in zip(starts, sizes, widths):
        level[start:start + n] = width                                 # gradients differ by layer ...
    p = (0.05 * randn(total) * (level > 0)).to(dtype)
    grad = randn(total) * torch.exp(randn(total)) * level              # ... have long tails ...
    grad = (grad * ((index // 96) % 11 != 5)).to(dtype)                # ... and units that never fired have none
    return {"p": p, "grad": grad, "starts": starts, "sizes": sizes}


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if case["op"] == "norm":
        if case["train"]:
            state["x"].requires_grad_(True)
            if state["weight"] is not None:
                state["weight"].requires_grad_(True)
                state["bias"].requires_grad_(True)
        return state
    if own:
        import raft_amd
        params = []
        for start, n in zip(state["starts"], state["sizes"]):
            p = torch.nn.Parameter(state["p"][start:start + n])
            p.grad = state["grad"][start:start + n]
            params.append(p)
        state["optimizer"] = raft_amd.AdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=case["bits"],
                                            max_norm=case["clip"] or None, seed=SEED)
    else:
        state.update(step=0, m=torch.zeros(state["p"].numel(), device="cuda"), v=torch.zeros(state["p"].numel(), device="cuda"))
    return state


def run(state):
    case = state["case"]
    if case["op"] == "norm":
        return _own_norm(state) if own else _plain_norm(state)
    return _own_adamw(state) if own else _plain_adamw(state)


def work(case):
    if case["op"] == "norm":
        size = 4 if case["dtype"] == "fp32" else 2
        count = case["n"] * case["c"] * case["h"] * case["w"]
        return {"bytes": count * size * (4 if case["train"] else 2), "flops": count * (28 if case["train"] else 8)}
    size = 4 if case["dtype"] == "fp32" else 2
    # p and g read, p written; 32-bit moments read and written; 8-bit ones read, written and given out in 16 bits
    return {"bytes": case["total"] * (3 * size + (16 if case["bits"] == 32 else 4 + 4)), "flops": case["total"] * 20}


# ---- the framework's calls -------------------------------------------------------------------------------------------

def _own_norm(state):
    import raft_amd
    case = state["case"]
    y = raft_amd.group_norm(state["x"], case["groups"], state["weight"], state["bias"], eps=EPS_NORM, activation=case["act"])
    if not case["train"]:
        return {"y": y}
    leaves = [t for t in (state["x"], state["weight"], state["bias"]) if t is not None]
    return {"y": y, "grads": list(torch.autograd.grad(y, leaves, state["dy"]))}


def _own_adamw(state):
    optimizer = state["optimizer"]
    optimizer.step()
    if state["case"]["bits"] == 32:
        (m, v), = optimizer.packed_moments()
    else:
        (m, v), = optimizer.packed_moments(torch.bfloat16)            # four significant bits: 16 bits hold them exactly
    out = {"p": state["p"], "m": m, "v": v}
    if state["case"]["clip"]:
        out["norm"] = optimizer.grad_norm
    return out


# ---- the same in elementary operations -------------------------------------------------------------------------------

def _activate(z, act):
    return z if act == "none" else torch.clamp_min(z, 0) if act == "relu" else z / (1 + torch.exp(-z))


def _slope(z, act):
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).to(z.dtype)
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def _plain_norm(state):
    case, x = state["case"], state["x"].detach()
    n, c, h, w = x.shape
    groups, act = case["groups"], case["act"]

    def rows(t):
        return t.permute(0, 2, 3, 1).reshape(n, h * w, groups, c // groups).float()

    def maps(t, dtype):
        return t.reshape(n, h, w, c).to(dtype).permute(0, 3, 1, 2)

    xf = rows(x)
    centred = xf - xf.mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt((centred * centred).mean((1, 3), keepdim=True) + EPS_NORM)
    xh = centred * rstd
    affine = state["weight"] is not None
    weight = state["weight"].detach().view(groups, -1) if affine else torch.ones(groups, c // groups, device=x.device)
    z = xh * weight + (state["bias"].detach().view(groups, -1) if affine else 0)
    y = maps(_activate(z, act), x.dtype)
    if not case["train"]:
        return {"y": y}
    g = rows(state["dy"]) * _slope(z, act)
    gw = g * weight
    dx = rstd * (gw - gw.mean((1, 3), keepdim=True) - xh * (gw * xh).mean((1, 3), keepdim=True))
    grads = [maps(dx, x.dtype)]
    if affine:
        grads += [(g * xh).sum((0, 1)).reshape(c), g.sum((0, 1)).reshape(c)]
    return {"y": y, "grads": grads}


_LOW = 0xFFFFFFFF
_GOLDEN, _ROOT2, _ROOT3 = 0x9E3779B9, 0x6A09E667, 0xBB67AE85          # the leading binary digits of the golden ratio, sqrt 2, sqrt 3


def _mix(x):
    x = x ^ (x >> 16)
    x = (x * _ROOT2) & _LOW
    x = x ^ (x >> 15)
    x = (x * _ROOT3) & _LOW
    return x ^ (x >> 16)


def _random(step, count, device):
    """32 random bits for each position, from the seed, the step and the position alone."""
    key = _mix((_mix((SEED + _GOLDEN * step) & _LOW)) & _LOW)
    return _mix((torch.arange(count, device=device) * _GOLDEN + key) & _LOW)


def _bits(x):
    return x.view(torch.int32).long() & _LOW


def _quantised(x, bits16, top):
    """x >= 0 in 32 bits -> the value of its 8-bit code. The block's largest value has exponent `top` in the code's units; below 8
    units codes are whole units, above they are a float with 3 bits after the leading one. bits16: 16 random bits each."""
    blocks = x.view(-1, BLOCK)
    field = _bits(blocks.amax(1, keepdim=True)) >> 23
    scale = torch.exp2((127 + top - field).double())
    scaled = (blocks.double() * scale).float()
    low = scaled < 8
    word = _bits(torch.where(low, scaled + 8, scaled))
    code = ((word + (bits16.view(-1, BLOCK) << 4)) >> 20) - (0x41000000 >> 20) + torch.where(low, 0, 8)
    if top == 32:
        code = torch.maximum(code, (blocks > 0).long())               # a second moment that is not zero never becomes zero
    value = torch.where(code < 8, code, (8 + (code & 7)) << ((code >> 3) - 1).clamp_min(0)).double() / scale
    return torch.where(field == 0, 0.0, value).view(-1)


def _plain_adamw(state):
    case, p, g = state["case"], state["p"], state["grad"]
    state["step"] += 1
    t, (b1, b2) = state["step"], BETAS
    wide = torch.float64 if case["bits"] == 8 else torch.float32      # 8-bit codes have borders that 32-bit sums miss
    out, g = {"p": p}, g.to(wide)
    if case["clip"]:
        norm = torch.sqrt(g.double().square().sum())
        g = g * torch.clamp(case["clip"] / (norm + 1e-6), max=1.0)
        out["norm"] = norm.float()
    m = b1 * state["m"].to(wide) + (1 - b1) * g
    v = b2 * state["v"].to(wide) + (1 - b2) * g * g
    mf, vf = m.float(), v.float()
    new = p.float() * (1 - LR * DECAY) - (LR / (1 - b1 ** t)) * mf / (torch.sqrt(vf) / math.sqrt(1 - b2 ** t) + EPS)
    if p.dtype == torch.bfloat16 or case["bits"] == 8:
        bits = _random(t, p.numel(), p.device)
    if p.dtype == torch.bfloat16:
        word = _bits(new) + (_mix((bits + _GOLDEN) & _LOW) & 0xFFFF)
        new = ((word & 0xFFFF0000) - ((word & 0x80000000) << 1)).int().view(torch.float32)
    p.copy_(new)
    if case["bits"] == 32:
        state["m"], state["v"] = m, v
        return dict(out, m=m, v=v)
    state["m"] = (torch.sign(mf) * _quantised(mf.abs(), bits & 0xFFFF, 16)).float()
    state["v"] = _quantised(vf, bits >> 16, 32).float()
    return dict(out, m=state["m"].bfloat16(), v=state["v"].bfloat16())


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------

def exact(case, seed):
    inputs = _inputs(case, seed)
    return _exact_norm(case, inputs) if case["op"] == "norm" else _exact_adamw(case, inputs)


def _exact_norm(case, inputs):
    n, c, h, w = inputs["x"].shape
    x = inputs["x"].double().contiguous().requires_grad_(case["train"])
    leaves = [x]
    groups = x.reshape(n, case["groups"], -1)
    moment1 = groups.sum(2, keepdim=True) / groups.shape[2]
    moment2 = ((groups - moment1) ** 2).sum(2, keepdim=True) / groups.shape[2]
    z = ((groups - moment1) * (moment2 + EPS_NORM) ** -0.5).reshape(n, c, h, w)
    if inputs["weight"] is not None:
        weight = inputs["weight"].double().requires_grad_(case["train"])
        bias = inputs["bias"].double().requires_grad_(case["train"])
        leaves += [weight, bias]
        z = z * weight[None, :, None, None] + bias[None, :, None, None]
    y = torch.where(z > 0, z, 0.0) if case["act"] == "relu" else z * torch.sigmoid(z) if case["act"] == "silu" else z * 1
    if not case["train"]:
        return {"y": y}
    return {"y": y.detach(), "grads": list(torch.autograd.grad(y, leaves, inputs["dy"].double()))}


def _exact_code_value(x, fraction, top):
    """The definition of the 8-bit codes in sums and products: steps of one unit up to 8, then of 2^e units between 2^(e+3) and
    2^(e+4); rounded up where the rest plus the random fraction reaches a whole step."""
    x = x.reshape(-1, BLOCK)
    largest = x.amax(1, keepdim=True)
    exponent = torch.frexp(largest)[1].double() - 1
    unit = torch.exp2(exponent - top)
    u = x / unit
    step = torch.exp2((torch.frexp(u)[1].double() - 4).clamp_min(0))
    value = torch.floor(u / step + fraction.reshape(-1, BLOCK)) * step
    if top == 32:
        value = torch.where((x > 0) & (value < 1), 1.0, value)
    return torch.where(largest >= 2.0 ** -126, value * unit, 0.0).reshape(-1)


def _exact_adamw(case, inputs):
    p, g, t, (b1, b2) = inputs["p"].double(), inputs["grad"].double(), 1, BETAS
    out = {}
    if case["clip"]:
        out["norm"] = torch.linalg.vector_norm(g)
        g = g * min(1.0, case["clip"] / (float(out["norm"]) + 1e-6))
    m, v = (1 - b1) * g, (1 - b2) * g ** 2                             # the first step, from moments of zero
    out["p"] = p - LR * DECAY * p - LR * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)) ** 0.5 + EPS)
    if case["dtype"] == "bf16" or case["bits"] == 8:
        bits = _random(t, p.numel(), p.device)
    if case["dtype"] == "bf16":
        q = out["p"].float().double()
        step = torch.exp2(torch.frexp(q)[1].double() - 8)
        out["p"] = torch.sign(q) * step * torch.floor(q.abs() / step + (_mix((bits + _GOLDEN) & _LOW) & 0xFFFF) / 65536.0)
    if case["bits"] == 32:
        return dict(out, m=m, v=v)
    m, v = m.float().double(), v.float().double()                      # moments are rounded to 32 bits, then to 8
    return dict(out, m=torch.sign(m) * _exact_code_value(m.abs(), (bits & 0xFFFF) / 65536.0, 16), v=_exact_code_value(v, (bits >> 16) / 65536.0, 32))
