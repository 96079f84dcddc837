"""The optimizer operators as a training program meets them, for timing and comparing.

  adamw    one AdamW step over many tensors, both moments in 32 bits, optionally with the gradients clipped to a
           joint norm
  adamw8   the same step with both moments in 8 bits, one scale per moment and block of 256 elements
  norm     the 2-norm of every gradient and of all of them together

`own` chooses between elementary torch operations and the calls into pir_amd.optim; both get what prepare() gives.

The 8-bit moments of a block of 256 consecutive elements (the last one of a tensor filled up with zeros) are

  first    int8 q in [-127, 127],  m = a (q / 127) |q / 127|,   a = the block's largest |m|
  second   uint8 c in [0, 255],    v = b (c / 255)^4,           b = the block's largest v

rounded to the nearest code (ties to even), except that a v above zero has c >= 1.  A block whose largest is below
2^-126 is all zeros; one that holds a value that is not finite has a scale of NaN.
"""
import math
import random

import torch

own = False

BLOCK = 256
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
TINY = 2.0 ** -126


# ---------------------------------------------------------------------------------------------------- the tensors
def _numels(case):
    kind = case["tensors"]
    if kind == "networks":     # weight-normed linear layers as in scene.MODEL_CONFIG: bias, weight_g, weight_v of each
        dims = [case["d_in"]] + [case["width"]] * (case["layers"] - 1) + [case["d_out"]]
        one = [n for i, o in zip(dims[:-1], dims[1:]) for n in (o, o, o * i)]
        return one * case["copies"]
    if kind == "blocks":       # a table of rows, then blocks of four square matrices, two of ratio 4, and two vectors
        d = case["width"]
        return [case["rows"] * d] + [d * d] * 4 * case["layers"] + [4 * d * d] * 2 * case["layers"] + [d] * 2 * case["layers"]
    rng = random.Random(case["shape_seed"])   # "ragged": anything from one element up, spread over the logarithm
    return [int(math.exp(rng.uniform(0.0, math.log(case["largest"] + 0.5)))) for _ in range(case["count"])]


def _offsets(numels, packed):
    """Where each tensor starts in the buffer of all: at every 256th element, or back to back from an odd place on."""
    at, off = (1, []) if packed else (0, [])
    for n in numels:
        off.append(at)
        at += n if packed else -(-n // BLOCK) * BLOCK
    return off, at


def _blocks(numels):
    return [-(-n // BLOCK) for n in numels]


# ----------------------------------------------------------------------------------------------------------- cases
def _case(name, op, dtype, clip=0.0, packed=False, step=500, lr=1e-4, decay=0.01, **tensors):
    return {"name": name, "op": op, "dtype": dtype, "clip": clip, "packed": packed, "step": step, "lr": lr,
            "decay": decay, **tensors}


def _networks(copies, layers=9, width=256, d_in=39, d_out=257):
    return {"tensors": "networks", "copies": copies, "layers": layers, "width": width, "d_in": d_in, "d_out": d_out}


def _layers(layers, width, rows):
    return {"tensors": "blocks", "layers": layers, "width": width, "rows": rows}


def _ragged(count, largest, shape_seed):
    return {"tensors": "ragged", "count": count, "largest": largest, "shape_seed": shape_seed}


def listed():
    return [
        # the SDF network alone: what every iteration steps, and the call where the launch itself counts
        _case("adamw sdf network", "adamw", "float32", lr=1e-5, decay=0.0, **_networks(1)),
        # all seven networks of a training run in one step, gradients clipped to a joint norm
        _case("adamw all networks, clipped", "adamw", "float32", clip=0.5, decay=0.0, **_networks(7, layers=6)),
        # many tensors of odd sizes, views of one gradient bucket, none of them aligned
        _case("adamw ragged fp16", "adamw", "float16", clip=2.0, packed=True, **_ragged(301, 200_000, 3)),
        # a larger model in bfloat16, clipped: the norm's pass over the gradients and the step's
        _case("adamw 88M bf16, clipped", "adamw", "bfloat16", clip=0.5, **_layers(6, 1024, 12_007)),
        # the largest 32-bit one: 28 bytes an element, nothing but memory
        _case("adamw 284M fp32", "adamw", "float32", **_layers(5, 2048, 16_001)),
        # the SDF network with 8-bit moments
        _case("adamw8 sdf network", "adamw8", "float32", lr=1e-5, decay=0.0, **_networks(1)),
        # tensors of odd sizes whose last blocks are partly filled
        _case("adamw8 ragged fp32, clipped", "adamw8", "float32", clip=0.5, packed=True, **_ragged(257, 300_000, 5)),
        _case("adamw8 88M bf16, clipped", "adamw8", "bfloat16", clip=0.5, **_layers(6, 1024, 12_007)),
        # the largest 8-bit one: where the states' 2 bytes an element in place of 8 matter most
        _case("adamw8 435M bf16", "adamw8", "bfloat16", **_layers(8, 2048, 16_001)),
        # gradient norms of all networks, as a run logs them
        _case("norm all networks", "norm", "float32", **_networks(7, layers=6)),
        _case("norm ragged bf16", "norm", "bfloat16", packed=True, **_ragged(301, 200_000, 7)),
        _case("norm 284M fp32", "norm", "float32", **_layers(5, 2048, 16_001)),
    ]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    op = rng.choice(("adamw", "adamw8", "norm"))
    kind = rng.choice(("networks", "blocks", "ragged"))
    if kind == "networks":
        tensors = _networks(rng.randint(1, 8), rng.randint(1, 9), log(1, 640), log(1, 700), log(1, 384))
    elif kind == "blocks":
        tensors = _layers(rng.randint(1, 6), log(16, 1900), log(1, 20_000))
    else:
        tensors = _ragged(log(1, 500), log(1, 1_000_000), rng.randrange(1 << 20))
    c = _case("", op, rng.choice(tuple(DTYPES)), clip=rng.choice((0.0, 0.0, 0.3, 3.0)), packed=rng.random() < 0.4,
              step=log(1, 100_000) - 1, lr=math.exp(rng.uniform(math.log(1e-5), math.log(2e-4))),
              decay=rng.choice((0.0, 0.01, 0.1)), **tensors)
    del c["name"]
    return c


def work(case):
    """A pass reads the gradients and the parameters, writes the parameters, and reads and writes both moments: 4 bytes
    each, or 1 and two 4-byte scales a block.  The 8-bit step's moments are also read back as bfloat16 values.  The joint
    norm has to be known before the first update: where it is asked for, the gradients are read twice."""
    numels = _numels(case)
    n, item, nb = sum(numels), DTYPES[case["dtype"]].itemsize, sum(_blocks(numels))
    if case["op"] == "norm":
        return {"bytes": n * item, "flops": 2 * n}
    data = n * 3 * item + (n * item if case["clip"] else 0) + 8 * len(numels)
    if case["op"] == "adamw":
        return {"bytes": data + 16 * n, "flops": 16 * n + (2 * n if case["clip"] else 0)}
    return {"bytes": data + nb * (BLOCK * 4 + 16) + nb * (BLOCK * (2 + 4) + 8),
            "flops": 40 * n + (2 * n if case["clip"] else 0)}


# ---------------------------------------------------------------------------------------------------------- inputs
def _pad(numels, pieces, zeros):
    """The tensors back to back, each filled up with zeros to a whole number of blocks."""
    return torch.cat([x for n, t in zip(numels, pieces) for x in (t, zeros[:-n % BLOCK])])


def _encode(m, v):
    """[blocks, 256] moments of floating type -> codes and scales."""
    a, b = m.abs().amax(1), v.amax(1)
    a = torch.where(torch.isfinite(a), torch.where(a < TINY, 0.0, a), math.nan)
    b = torch.where(torch.isfinite(b), torch.where(b < TINY, 0.0, b), math.nan)
    q = (127 * (m.abs() / a[:, None]).sqrt()).round().clamp(max=127) * m.sign()
    c = (255 * (v / b[:, None]).sqrt().sqrt()).round().clamp(max=255)
    c = torch.where(v > 0, c.clamp(min=1), c)
    q = torch.where(a[:, None] > 0, q, 0.0)
    c = torch.where(b[:, None] > 0, c, 0.0)
    return q.to(torch.int8), c.to(torch.uint8), torch.stack([a, b], 1)


def _decode(q, c, scales, dtype):
    q, c, a, b = q.to(dtype) / 127, c.to(dtype) / 255, scales[:, :1].to(dtype), scales[:, 1:].to(dtype)
    return a * (q * q.abs()), b * (c * c * (c * c))


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    host = random.Random(seed)
    numels, dtype = _numels(case), DTYPES[case["dtype"]]
    off, total = _offsets(numels, case["packed"])
    view = lambda buf: [buf[o:o + n] for o, n in zip(off, numels)]  # noqa: E731
    noise = lambda n: torch.randn(n, device="cuda", generator=gen)  # noqa: E731
    # each tensor's gradients have a size of their own; float16 cannot hold the smallest without a loss scale
    size = [math.exp(host.uniform(math.log(1e-6), math.log(1e-2))) * (2.0 ** 7 if dtype == torch.float16 else 1.0) for _ in numels]
    g = noise(total)
    for t, s in zip(view(g), size):
        t.mul_(s)
    if case["op"] != "adamw":   # a unit that was not reached has gradients of zero
        g.mul_(torch.rand(total, device="cuda", generator=gen) > 0.05)
    s = {"op": case["op"], "numels": numels, "grad_buffer": g.to(dtype), "max_norm": None}
    s["grads"] = view(s["grad_buffer"])
    if case["op"] == "norm":
        return s
    if case["clip"]:
        s["max_norm"] = case["clip"] * math.sqrt(sum(n * x * x for n, x in zip(numels, size)))
    s["param_buffer"] = (0.05 * noise(total)).to(dtype)
    s["params"] = view(s["param_buffer"])
    # tensors join a run at different times: their step counts differ
    s["steps"] = torch.tensor([float(max(0, case["step"] - host.randrange(3))) for _ in numels], device="cuda")
    s["hyper"] = {"lr": case["lr"], "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": case["decay"]}
    m, v = noise(total), noise(total)
    for a, b, x in zip(view(m), view(v), size):
        a.mul_(0.25 * x)
        b.square_().add_(0.05).mul_(x * x)
    if case["op"] == "adamw":
        s["m_buffer"], s["v_buffer"] = m, v
        s["exp_avgs"], s["exp_avg_sqs"] = view(m), view(v)
        return s
    zeros = torch.zeros(BLOCK, device="cuda")
    s["q"], s["c"], s["scale"] = _encode(_pad(numels, view(m), zeros).view(-1, BLOCK), _pad(numels, view(v), zeros).view(-1, BLOCK))
    nb = _blocks(numels)
    s["exp_avgs"], s["exp_avg_sqs"], s["scales"] = (list(s[k].split(nb)) for k in ("q", "c", "scale"))
    return s


# ------------------------------------------------------------------------------------------------- the plain forms
def _flat(tensors):
    return torch.cat([t.reshape(-1) for t in tensors]).float()


def _clip(g, max_norm):
    norm = g.double().square().sum().sqrt()
    return norm.float(), (max_norm / (norm + 1e-6)).clamp(max=1.0).float()


def _factors(s):
    """The step counts, moved on by one, and lr / (1 - beta1^t) and 1 / sqrt(1 - beta2^t) of each tensor."""
    (b1, b2), lr = s["hyper"]["betas"], s["hyper"]["lr"]
    s["steps"].add_(1)
    t = s["steps"].double()
    return (lr / (1 - b1 ** t)).float(), (1 - b2 ** t).rsqrt().float()


def _spread(x, counts):
    """One value a tensor -> one an element (or block) of all of them."""
    return torch.cat([t.expand(n) for t, n in zip(x.unbind(), counts)])


def _update(s, p, g, m, v, size, root):
    """The moments of this step and the parameters after it."""
    (b1, b2), lr = s["hyper"]["betas"], s["hyper"]["lr"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    p = p * (1 - lr * s["hyper"]["weight_decay"]) - size * m / (v.sqrt() * root + s["hyper"]["eps"])
    return p, m, v


def _adamw(s):
    numels = s["numels"]
    size, root = (_spread(x, numels) for x in _factors(s))
    p, g, m, v = (_flat(s[k]) for k in ("params", "grads", "exp_avgs", "exp_avg_sqs"))
    norm = None
    if s["max_norm"]:
        norm, coef = _clip(g, s["max_norm"])
        g = g * coef
    p, m, v = _update(s, p, g, m, v, size, root)
    torch._foreach_copy_(s["params"], list(p.to(s["param_buffer"].dtype).split(numels)))
    torch._foreach_copy_(s["exp_avgs"], list(m.split(numels)))
    torch._foreach_copy_(s["exp_avg_sqs"], list(v.split(numels)))
    return norm


def _adamw8(s):
    numels, nb = s["numels"], _blocks(s["numels"])
    zeros = torch.zeros(BLOCK, device="cuda", dtype=s["param_buffer"].dtype)
    size, root = (_spread(x, nb)[:, None] for x in _factors(s))
    p, g = (_pad(numels, s[k], zeros).float().view(-1, BLOCK) for k in ("params", "grads"))
    norm = None
    if s["max_norm"]:
        norm, coef = _clip(g, s["max_norm"])
        g = g * coef
    m, v = _decode(torch.cat(s["exp_avgs"]), torch.cat(s["exp_avg_sqs"]), torch.cat(s["scales"]), torch.float32)
    p, m, v = _update(s, p, g, m, v, size, root)
    torch._foreach_copy_(s["params"], [t[:n] for t, n in zip(p.to(zeros.dtype).view(-1).split([BLOCK * k for k in nb]), numels)])
    q, c, scale = _encode(m, v)
    torch._foreach_copy_(s["exp_avgs"], list(q.split(nb)))
    torch._foreach_copy_(s["exp_avg_sqs"], list(c.split(nb)))
    torch._foreach_copy_(s["scales"], list(scale.split(nb)))
    return norm


def _norms(grads):
    each = torch.stack([g.double().square().sum() for g in grads])
    return each.sum().sqrt().float(), each.sqrt().float()


# ------------------------------------------------------------------------------------------------------------- run
def run(state):
    s = state
    if s["op"] == "norm":
        if own:
            from pir_amd import optim
            return optim.grad_norm(s["grads"])
        return _norms(s["grads"])
    if s["op"] == "adamw":
        if own:
            from pir_amd import optim
            norm = optim.adamw_step(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"], s["steps"],
                                    max_norm=s["max_norm"], **s["hyper"])
        else:
            norm = _adamw(s)
        return {"params": s["param_buffer"], "exp_avg": s["m_buffer"], "exp_avg_sq": s["v_buffer"], "steps": s["steps"],
                "norm": norm}
    # 8-bit moments come back as the values they stand for.  A code says no more than 8 bits of one, which is what
    # bfloat16 holds.
    if own:
        from pir_amd import optim
        norm = optim.adamw8_step(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"], s["scales"], s["steps"],
                                 max_norm=s["max_norm"], **s["hyper"])
        m, v = optim.moments8_decode(s["q"], s["c"], s["scale"], dtype=torch.bfloat16)
    else:
        norm = _adamw8(s)
        m, v = (t.bfloat16() for t in _decode(s["q"], s["c"], s["scale"], torch.float32))
    return {"params": s["param_buffer"], "exp_avg": m, "exp_avg_sq": v, "steps": s["steps"], "norm": norm}


# ----------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """run()'s answer tensor by tensor in 64 bits, from the formulas."""
    s = prepare(case, seed)
    grads = [g.double() for g in s["grads"]]
    squares = [torch.dot(g, g) for g in grads]
    norm = math.sqrt(math.fsum(x.item() for x in squares))
    if case["op"] == "norm":
        return torch.tensor(norm, dtype=torch.float64, device="cuda"), torch.stack([x.sqrt() for x in squares])
    h, (beta1, beta2) = s["hyper"], s["hyper"]["betas"]
    shrink = min(1.0, s["max_norm"] / (norm + 1e-6)) if s["max_norm"] else 1.0
    params, moments1, moments2 = s["param_buffer"].double(), [], []
    off, _ = _offsets(s["numels"], case["packed"])
    first = s["m_buffer"].double() if case["op"] == "adamw" else None
    second = s["v_buffer"].double() if case["op"] == "adamw" else None
    for k, (at, n) in enumerate(zip(off, s["numels"])):
        t = int(s["steps"][k].item()) + 1
        here = slice(at, at + n)
        g = grads[k] * shrink
        grads[k] = None
        if case["op"] == "adamw":
            m, v = first[here], second[here]
        else:
            q, c, ab = s["exp_avgs"][k].double(), s["exp_avg_sqs"][k].double(), s["scales"][k].double()
            m = (torch.sign(q) * (q / 127) ** 2 * ab[:, 0, None]).reshape(-1)[:n]
            v = ((c / 255) ** 4 * ab[:, 1, None]).reshape(-1)[:n]
        m = beta1 * m + (1 - beta1) * g
        v = beta2 * v + (1 - beta2) * g ** 2
        step = (m / -math.expm1(t * math.log(beta1))) / ((v / -math.expm1(t * math.log(beta2))) ** 0.5 + h["eps"])
        params[here] = params[here] - h["lr"] * (h["weight_decay"] * params[here] + step)
        if case["op"] == "adamw":
            first[here], second[here] = m, v
            continue
        rows = -(-n // BLOCK)
        full = lambda x: torch.cat([x, x.new_zeros(rows * BLOCK - n)]).view(rows, BLOCK)  # noqa: E731
        m, v = full(m), full(v)
        top1, top2 = m.abs().max(1, keepdim=True).values, v.max(1, keepdim=True).values
        top1, top2 = top1 * (top1 >= TINY), top2 * (top2 >= TINY)
        level1 = torch.round(127 * (m.abs() / top1.clamp(min=TINY)) ** 0.5).clamp(0, 127)
        level2 = torch.round(255 * (v / top2.clamp(min=TINY)) ** 0.25).clamp(0, 255)
        level2 = torch.maximum(level2, ((v > 0) & (top2 > 0)).double())
        moments1.append(torch.sign(m) * top1 * (level1 / 127) ** 2)
        moments2.append(top2 * (level2 / 255) ** 4)
    if case["op"] == "adamw8":
        first, second = torch.cat(moments1), torch.cat(moments2)
    return {"params": params, "exp_avg": first, "exp_avg_sq": second, "steps": s["steps"].double() + 1,
            "norm": torch.tensor(norm, dtype=torch.float64, device="cuda") if s["max_norm"] else None}
