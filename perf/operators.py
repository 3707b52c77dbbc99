"""Operators for training with small optimiser states and for serving in 8-bit integers: the cases that are measured, the plain form of each
operator, and the calls a user makes of ``controllable_agent_amd``.

* ``adamw``: one AdamW step over a list of tensors (``controllable_agent_amd.AdamW``), moments in 32 or in 8 bits, with or without clipping by
  the global gradient norm;
* ``linear_i8``: y = relu?(x W^T + bias) with x quantised per token inside the call and W held in 8 bits per channel (``kernels.linear_i8``);
* ``gemm_i8``: the product alone, on codes that are 8-bit integers already (``kernels.gemm_i8``).

The tensors of an AdamW case are views of one flat buffer, each starting on a multiple of 256 elements (the networks of this package live in flat
buffers too), so that the parameters come back as one output.  The gaps hold zeros and no step changes them.
"""
import math
import random

import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
BLOCK = 256                     # elements that share a scale of an 8-bit moment
LR, BETA1, BETA2, EPS, DECAY, MAX_NORM, STEP0, SEED = 1e-4, 0.9, 0.999, 1e-8, 0.01, 1.0, 100, 1234


# ------------------------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one optimiser step of the walker agent's ForwardMap + BackwardMap (28 tensors, 3.7 M parameters), as the package trains them: fp32
        dict(name="adamw32 walker nets", op="adamw", layout="walker", count=28, total=3681694, bits=32, p="fp32", g="fp32", clip=False),
        # the same networks with 8-bit moments and clipping
        dict(name="adamw8 walker nets clip", op="adamw", layout="walker", count=28, total=3681694, bits=8, p="fp32", g="fp32", clip=True),
        # many small odd tensors: biases, norms, small heads.  Launches and host work count
        dict(name="adamw8 many small", op="adamw", layout="odd", count=200, total=400003, bits=8, p="fp32", g="fp32", clip=False),
        # a large network in bf16 with fp32 moments and clipping
        dict(name="adamw32 large bf16 clip", op="adamw", layout="even", count=24, total=1 << 26, bits=32, p="bf16", g="bf16", clip=True),
        # the largest: fp32 master weights, bf16 gradients, 8-bit moments
        dict(name="adamw8 large", op="adamw", layout="even", count=40, total=1 << 27, bits=8, p="fp32", g="bf16", clip=False),
        # acting: one token through a hidden layer
        dict(name="linear_i8 one token", op="linear_i8", m=1, n=1024, k=1024, x="fp32", y="fp32", bias=True, relu=True),
        # a few environments stepped together through a wide layer: the weights' bytes count
        dict(name="linear_i8 16 tokens", op="linear_i8", m=16, n=4096, k=4096, x="bf16", y="bf16", bias=True, relu=False),
        # a batch through the walker agent's head layer (both heads' hidden layers are one product)
        dict(name="linear_i8 batch", op="linear_i8", m=1024, n=2048, k=1024, x="fp32", y="fp32", bias=True, relu=True),
        # odd sizes in every direction: BackwardMap's hidden width 526
        dict(name="linear_i8 odd", op="linear_i8", m=777, n=526, k=1051, x="fp16", y="fp16", bias=True, relu=False),
        # relabelling a replay buffer: many rows through a large layer
        dict(name="linear_i8 large", op="linear_i8", m=8192, n=8192, k=8192, x="bf16", y="bf16", bias=True, relu=False),
        # codes in hand: several products share one quantised input
        dict(name="gemm_i8 medium", op="gemm_i8", m=4096, n=2048, k=2048, x="int8", y="fp32", bias=False, relu=False),
        dict(name="gemm_i8 ragged", op="gemm_i8", m=2500, n=5001, k=1999, x="int8", y="bf16", bias=True, relu=True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.5:
        total = _spread(rng, 2000, 1 << 26)
        count = _spread(rng, 1, min(300, max(1, total // 16)))
        return dict(op="adamw", layout=rng.choice(["odd", "even"]), count=count, total=total, bits=rng.choice([8, 32]),
                    p=rng.choice(["fp32", "fp32", "bf16"]), g=rng.choice(["fp32", "bf16", "fp16"]), clip=rng.random() < 0.5)
    op = rng.choice(["linear_i8", "linear_i8", "gemm_i8"])
    m = rng.choice([1, rng.randint(2, 64), _spread(rng, 64, 8192)])
    return dict(op=op, m=m, n=_spread(rng, 6, 8192), k=_spread(rng, 24, 8192), x="int8" if op == "gemm_i8" else rng.choice(list(TYPES)),
                y=rng.choice(list(TYPES)), bias=rng.random() < 0.7, relu=rng.random() < 0.5)


def _shapes(case):
    """The tensors of an AdamW case: fixed by the case alone."""
    if case["layout"] == "walker":
        linear = lambda i, o: [(o, i), (o,)]  # noqa: E731
        norm = lambda n: [(n,), (n,)]  # noqa: E731
        trunk = lambda i: linear(i, 1024) + norm(1024) + linear(1024, 512)  # noqa: E731
        head = linear(1024, 1024) + linear(1024, 50)
        return trunk(30) + trunk(74) + head + head + linear(24, 526) + norm(526) + linear(526, 526) + linear(526, 50)
    count, total = case["count"], case["total"]
    if case["layout"] == "even":
        each = total // count
        return [(each,)] * (count - 1) + [(total - each * (count - 1),)]
    r = random.Random(total)
    shares = [math.exp(r.gauss(0, 1.2)) for _ in range(count)]
    sizes = [max(1, int(total * s / sum(shares))) | 1 for s in shares]
    return [(n,) for n in sizes]


# ------------------------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen, device=DEVICE)  # noqa: E731
    return _prepare_adamw(case, randn) if case["op"] == "adamw" else _prepare_product(case, randn)


def _prepare_adamw(case, randn):
    shapes = _shapes(case)
    starts, at = [], 0
    for s in shapes:
        starts.append(at)
        at += -(-math.prod(s) // BLOCK) * BLOCK
    live = torch.zeros(at, device=DEVICE, dtype=torch.bool)
    for b, s in zip(starts, shapes):
        live[b:b + math.prod(s)] = True
    views = lambda flat: [flat[b:b + math.prod(s)].view(s) for b, s in zip(starts, shapes)]  # noqa: E731
    # gradients whose size differs from one element to the next, as a network's do; moments as a hundred steps on such gradients leave them
    size = 1e-2 * torch.exp(0.7 * randn(at)) * live
    flat_p = (0.03 * randn(at) * live).to(TYPES[case["p"]])
    flat_g = (size * randn(at)).to(TYPES[case["g"]])
    m, root = 0.3 * size * randn(at), 0.3 * size
    state = dict(case=case, p=flat_p, g=flat_g, params=views(flat_p), grads=views(flat_g), step=STEP0)
    if case["bits"] == 32:
        moments = dict(m=m, v=root * root)
    else:
        moments = {}
        for name, x in (("m", m), ("r", root)):
            _, e = torch.frexp(x.view(-1, BLOCK).abs().amax(1).clamp_min(1e-30) / 448)
            scale = torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)
            moments[name + "8"] = (x.view(-1, BLOCK) / scale[:, None]).to(torch.float8_e4m3fn).view(-1)
            moments[name + "_scale"] = scale
    state.update(moments)
    if own:
        from controllable_agent_amd import AdamW
        state["optimizer"] = AdamW(state["params"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, state_bits=case["bits"], seed=SEED)
        state["optimizer"].load_state_dict(dict(moments, step=STEP0, seed=SEED))
    return state


def _prepare_product(case, randn):
    m, n, k = case["m"], case["n"], case["k"]
    # the weights as a server holds them: 8-bit codes and a scale for each output channel, rows on multiples of 16 bytes
    rows = lambda r: torch.zeros(r, -(-k // 16) * 16, device=DEVICE, dtype=torch.int8)[:, :k]  # noqa: E731
    w = randn(n, k) * torch.exp(0.3 * randn(n, 1)) / math.sqrt(k)
    w_scale = w.abs().amax(1) / 127
    state = dict(case=case, w=rows(n), w_scale=w_scale, bias=0.1 * randn(n) if case["bias"] else None)
    state["w"].copy_(torch.round(w / w_scale[:, None]))
    x = randn(m, k) * torch.exp(0.5 * randn(m, 1))
    if case["op"] == "gemm_i8":
        state["x_scale"] = x.abs().amax(1) / 127
        state["x"] = rows(m)
        state["x"].copy_(torch.round(x / state["x_scale"][:, None]))
    else:
        state["x"] = x.to(TYPES[case["x"]])
    return state


# --------------------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if case["op"] == "adamw":
        if own:
            opt = state["optimizer"]
            norm = opt.step(state["grads"], max_norm=MAX_NORM if case["clip"] else None)
            moments = (opt.m, opt.v) if case["bits"] == 32 else (opt.m8, opt.m_scale, opt.r8, opt.r_scale)
            return [state["p"], *moments, *([norm] if case["clip"] else [])]
        return _plain_adamw(state)
    if own:
        from controllable_agent_amd import kernels
        kw = dict(bias=state["bias"], relu=case["relu"], out_dtype=TYPES[case["y"]])
        if case["op"] == "gemm_i8":
            return kernels.gemm_i8(state["x"], state["x_scale"], state["w"], state["w_scale"], **kw)
        return kernels.linear_i8(state["x"], state["w"], state["w_scale"], **kw)
    return _plain_product(state)


def _plain_product(state):
    case = state["case"]
    x = state["x"].float()
    if case["op"] == "gemm_i8":
        codes, scale = x, state["x_scale"]
    else:
        scale = x.abs().amax(1) / 127
        codes = torch.where(scale[:, None] > 0, torch.round(x / scale[:, None]), 0.0).clamp(-127, 127)
    y = (codes @ state["w"].float().t()) * scale[:, None] * state["w_scale"]
    if state["bias"] is not None:
        y = y + state["bias"]
    return (torch.relu(y) if case["relu"] else y).to(TYPES[case["y"]])


def _words(n, step):
    """A 32-bit word for each element from its place, the seed and the step number, as int64."""
    low = 0xFFFFFFFF

    def finish(h):
        h = (h ^ (h >> 16)) * 0x85EBCA6B & low
        h = (h ^ (h >> 13)) * 0xC2B2AE35 & low
        return h ^ (h >> 16)

    key = finish((SEED ^ (step * 0x27D4EB2F)) & low)
    return finish((torch.arange(n, device=DEVICE) * 0x9E3779B1 + key) & low)


def _encode(x, bits16, keep_positive):
    """e4m3 codes of x (as float8) and their power-of-two scales: rounded down or up by 16 random bits, so that the mean is x."""
    mag = x.abs().view(-1, BLOCK)
    top = mag.amax(1).view(torch.int32)
    field = (((top + 0x1FFFFF) >> 23) - 8).clamp_min(1)
    y = (mag * ((254 - field) << 23).view(torch.float32)[:, None]).view(-1)
    small = y < 2.0 ** -6
    z = torch.where(small, y + 2.0 ** -6, y)
    code = ((z.view(torch.int32) + (bits16 << 4).int()) >> 20) - torch.where(small, 968, 960).int()
    if keep_positive:
        code = torch.where((code == 0) & (x > 0), 1, code)
    code = code | torch.where(torch.signbit(x), 128, 0).int()
    return code.to(torch.uint8).view(torch.float8_e4m3fn), (field << 23).view(torch.float32)


def _decode(codes, scale):
    return (codes.float().view(-1, BLOCK) * scale[:, None]).view(-1)


def _plain_adamw(state):
    case = state["case"]
    state["step"] += 1
    t = state["step"]
    g = state["g"].float()
    norm = None
    if case["clip"]:
        norm = g.double().square().sum().sqrt().float()
        g = g * (MAX_NORM / torch.clamp_min(norm, MAX_NORM))
    if case["bits"] == 32:
        m, v = state["m"], state["v"]
    else:
        m, v = _decode(state["m8"], state["m_scale"]), _decode(state["r8"], state["r_scale"]).square()
    m = m + (1 - BETA1) * (g - m)
    v = v * BETA2 + ((1 - BETA2) * g) * g
    root = torch.sqrt(v)
    den = root * (1 / math.sqrt(1 - BETA2 ** t)) + EPS
    p = state["p"].float() * (1 - LR * DECAY) - (LR / (1 - BETA1 ** t)) * (m / den)
    words = _words(p.numel(), t) if case["bits"] == 8 or case["p"] == "bf16" else None
    if case["p"] == "bf16":      # rounded to 16 bits up or down at random: updates below half a step still move the parameter on average
        bits = p.view(torch.int32) + ((words * 0x9E3779B1 & 0xFFFFFFFF) >> 16).int()
        p = (bits & -65536).view(torch.float32)
    state["p"].copy_(p)
    if case["bits"] == 32:
        state["m"], state["v"] = m, v
        moments = [m, v]
    else:
        state["m8"], state["m_scale"] = _encode(m, words >> 16, False)
        state["r8"], state["r_scale"] = _encode(root, words & 0xFFFF, True)
        moments = [state["m8"], state["m_scale"], state["r8"], state["r_scale"]]
    return [state["p"], *moments, *([norm] if case["clip"] else [])]


# ----------------------------------------------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(case))
        moments = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
        return {"bytes": n * (2 * BYTES[case["p"]] + BYTES[case["g"]] + moments), "flops": 16 * n}
    m, n, k = case["m"], case["n"], case["k"]
    x = 1 if case["x"] == "int8" else BYTES[case["x"]]
    return {"bytes": m * k * x + n * k + m * n * BYTES[case["y"]] + 4 * n, "flops": 2 * m * n * k}


# ---------------------------------------------------------------------------------------------------------------- the definition, 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return _exact_adamw(case, state) if case["op"] == "adamw" else _exact_product(case, state)


def _exact_product(case, state):
    x = state["x"].double()
    if case["op"] == "gemm_i8":
        q, sx = x, state["x_scale"].double()
    else:
        # the scale is a 32-bit number, and a code the nearest whole number to the 32-bit quotient, ties to even
        sx = (x.abs().max(1).values / 127).float().double()
        quotient = (x / sx.clamp_min(1e-300).unsqueeze(1)).float().double()
        q = quotient.round().clamp(-127, 127)
    y = torch.mm(q, state["w"].double().t()) * (sx.unsqueeze(1) * state["w_scale"].double().unsqueeze(0))
    if case["bias"]:
        y += state["bias"].double()
    return y.clamp_min(0) if case["relu"] else y


def _exact_adamw(case, state):
    t = STEP0 + 1
    g = state["g"].double()
    total = g.pow(2).sum().sqrt()
    if case["clip"] and float(total) > MAX_NORM:
        g = g * (MAX_NORM / total)
    p = state["p"].double()
    n = p.numel()
    if case["bits"] == 32:
        m0, v0 = state["m"].double(), state["v"].double()
    else:
        per = lambda s: s.double().repeat_interleave(BLOCK)  # noqa: E731
        m0, v0 = state["m8"].double() * per(state["m_scale"]), (state["r8"].double() * per(state["r_scale"])).pow(2)
    m1 = BETA1 * m0 + (1 - BETA1) * g
    v1 = BETA2 * v0 + (1 - BETA2) * g.pow(2)
    p1 = p - LR * DECAY * p - LR * (m1 / (1 - BETA1 ** t)) / ((v1 / (1 - BETA2 ** t)).sqrt() + EPS)

    def word32(h):      # the same words from 32-bit halves
        for shift, factor in ((16, 0x85EBCA6B), (13, 0xC2B2AE35)):
            h = torch.bitwise_xor(h, h >> shift)
            h = torch.remainder((h % 65536) * factor + (((h >> 16) * (factor % 65536)) % 65536) * 65536, 2 ** 32)
        return torch.bitwise_xor(h, h >> 16)

    key = word32(torch.tensor((SEED ^ (t * 0x27D4EB2F)) % 2 ** 32, device=p.device))
    place = torch.remainder(torch.arange(n, device=p.device) * 0x9E3779B1 + key, 2 ** 32)
    need = case["bits"] == 8 or case["p"] == "bf16"
    word = word32(place) if need else None
    if case["p"] == "bf16":
        u = torch.div(torch.remainder((word % 65536) * 0x9E3779B1 + (((word >> 16) * 0x79B1) % 65536) * 65536, 2 ** 32), 65536, rounding_mode="floor").double() / 65536
        _, e = torch.frexp(p1)
        grid = torch.ldexp(torch.ones_like(p1), (e - 8).to(torch.int32))
        p1 = torch.sign(p1) * torch.floor(p1.abs() / grid + u) * grid
    out = [p1]
    if case["bits"] == 32:
        out += [m1, v1]
    else:
        for x, u, floor_one in ((m1, torch.div(word, 65536, rounding_mode="floor"), False), (v1.sqrt(), word % 65536, True)):
            top = x.abs().view(-1, BLOCK).max(1).values
            k = torch.ceil(torch.log2(top.clamp_min(2.0 ** -117) / 448))     # the least power of two under which the block fits
            scale = torch.pow(torch.full_like(k, 2.0), k).clamp_min(2.0 ** -126)
            scale = torch.where(top > 0, scale, torch.full_like(scale, 2.0 ** -126))
            y = x.abs() / scale.repeat_interleave(BLOCK)
            grid = torch.pow(torch.full_like(y, 2.0), torch.floor(torch.log2(y.clamp_min(2.0 ** -6))) - 3)
            y = torch.floor(y / grid + u.double() / 65536) * grid
            if floor_one:
                y = torch.where((y == 0) & (x > 0), torch.full_like(y, 2.0 ** -9), y)
            out += [torch.copysign(y, x), scale]
    return out + ([total] if case["clip"] else [])
