"""Cases and plain forms of the low-precision training operators: 4-bit microscaled quantisation, the encoder product on
it, and the AdamW step with moments in 32 or 8 bits.

``run`` computes them with elementary torch operations, or (``own``) through the package's entry points; ``exact`` gives
their definition in 64 bits.  The 4-bit format is MXFP4: 32 consecutive values of a row share one scale 2^(s - 127) (one
byte s), each value is one of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}; two codes a byte, the even column in the low half; rows are
padded with zeros to a multiple of 128 columns.  The 8-bit moments are e4m3 with one power of two for 128 elements."""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp32": 4}
HYPER = {"lr": 2e-4, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01}
FIRST_STEP = 100
BLOCK, BLOCK8 = 32, 128


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token through a GPT-2 layer's dictionary (expansion 128): serving, bound by reading W
        {"name": "linear one token", "op": "linear", "n": 1, "m": 98304, "d": 768, "x": "bf16", "out": "bf16", "bias": True, "relu": True},
        # a few sequences' last tokens, an odd dictionary and width, full-precision activations
        {"name": "linear ragged", "op": "linear", "n": 77, "m": 6151, "d": 1000, "x": "fp32", "out": "fp32", "bias": True, "relu": False},
        # the training batch of the 12-layer GPT-2 transcoder: 8192 tokens, 98304 latents
        {"name": "linear gpt2 batch", "op": "linear", "n": 8192, "m": 98304, "d": 768, "x": "bf16", "out": "bf16", "bias": True, "relu": True},
        # a residual-stream SAE of width 4096, expansion 32, while a prompt is read
        {"name": "linear wide prompt", "op": "linear", "n": 509, "m": 131072, "d": 4096, "x": "bf16", "out": "bf16", "bias": True, "relu": True},
        # width 2048, expansion 64: a training batch
        {"name": "linear 2048 batch", "op": "linear", "n": 4096, "m": 131072, "d": 2048, "x": "bf16", "out": "bf16", "bias": False, "relu": True},
        # activations of a training batch to 4 bits and back
        {"name": "quantise activations", "op": "quantise", "n": 8192, "d": 768, "x": "bf16", "out": "bf16"},
        # an encoder table after an optimizer step
        {"name": "quantise table", "op": "quantise", "n": 98304, "d": 768, "x": "fp32", "out": "bf16"},
        # a ragged batch of an odd width
        {"name": "quantise ragged", "op": "quantise", "n": 1021, "d": 1001, "x": "bf16", "out": "fp32"},
        # biases and post-encoder vectors of a transcoder: many small tensors, latency counts
        {"name": "adamw vectors", "op": "adamw", "count": 0, "rows": 24576, "cols": 768, "vectors": 20, "p": "bf16", "g": "bf16", "bits": 32},
        # one GPT-2 layer's encoder and three of its decoders in bf16 with 32-bit moments
        {"name": "adamw tables 32", "op": "adamw", "count": 4, "rows": 98304, "cols": 768, "vectors": 4, "p": "bf16", "g": "bf16", "bits": 32},
        # the same with 8-bit moments
        {"name": "adamw tables 8", "op": "adamw", "count": 4, "rows": 98304, "cols": 768, "vectors": 4, "p": "bf16", "g": "bf16", "bits": 8},
        # full-precision parameters, an odd shape, 8-bit moments
        {"name": "adamw odd 8", "op": "adamw", "count": 3, "rows": 4099, "cols": 769, "vectors": 2, "p": "fp32", "g": "fp32", "bits": 8},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("linear", "linear", "quantise", "adamw", "adamw"))
    if op == "linear":
        n, m, d = _spread(rng, 1, 8192), _spread(rng, 500, 131072), _spread(rng, 64, 4096)
        if rng.random() < 0.5:  # widths of models are whole blocks
            d = -(-d // 64) * 64
        while n * m * d > 4096 * 131072 * 1024:
            n = max(1, n // 2)
        return {"op": op, "n": n, "m": m, "d": d, "x": rng.choice(("bf16", "bf16", "fp32")), "out": rng.choice(("bf16", "bf16", "fp32")),
                "bias": rng.random() < 0.7, "relu": rng.random() < 0.7}
    if op == "quantise":
        return {"op": op, "n": _spread(rng, 1, 98304), "d": _spread(rng, 32, 768), "x": rng.choice(("bf16", "fp32")), "out": rng.choice(("bf16", "fp32"))}
    return {"op": op, "count": rng.randint(1, 5), "rows": _spread(rng, 64, 49152), "cols": _spread(rng, 64, 768), "vectors": rng.randint(0, 9),
            "p": rng.choice(("bf16", "fp32")), "g": rng.choice(("bf16", "fp32")), "bits": rng.choice((8, 32))}


# ------------------------------------------------------------------------------------------------------------ inputs
def _activations(n, d, gen, dtype):
    """Hidden states: widths of their own per column, a few columns with very large values, now and then an empty row."""
    x = torch.randn(n, d, generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn(d, generator=gen, device="cuda"))
    x[:, :: max(1, d // 4)] *= 30.0
    if n > 8:
        x *= torch.rand(n, 1, generator=gen, device="cuda") > 0.01
    return x.to(dtype)


def _grad_like(rows, cols, gen):
    """A table's gradient: rows of latents that did not fire are zero, the others differ widely in size."""
    size = torch.exp(1.5 * torch.randn(rows, 1, generator=gen, device="cuda")) * (torch.rand(rows, 1, generator=gen, device="cuda") > 0.3)
    return torch.randn(rows, cols, generator=gen, device="cuda") * size * 1e-4


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["op"] == "linear":
        state["x"] = _activations(case["n"], case["d"], gen, DT[case["x"]])
        bound = 1 / math.sqrt(case["d"])
        W = torch.empty(case["m"], case["d"], device="cuda").uniform_(-bound, bound, generator=gen)
        W *= torch.exp(0.3 * torch.randn(case["m"], 1, generator=gen, device="cuda"))
        parts = [_plain_quantise(w) for w in W.split(16384)]  # (in parts: the temporaries of a whole table are large)
        state["codes"], state["scales"] = torch.cat([c for c, _ in parts]), torch.cat([s for _, s in parts])
        state["bias"] = 0.1 * torch.randn(case["m"], generator=gen, device="cuda") if case["bias"] else None
    elif case["op"] == "quantise":
        state["x"] = _activations(case["n"], case["d"], gen, DT[case["x"]])
    else:
        state.update(params=[], grads=[], first=[], second=[], step=FIRST_STEP - 1, seed=seed)
        for shape in [(case["rows"], case["cols"])] * case["count"] + [(case["rows"],)] * case["vectors"]:
            matrix = len(shape) == 2
            size = shape if matrix else (1, shape[0])
            p = 0.03 * torch.randn(size, generator=gen, device="cuda")
            g = _grad_like(size[0], size[1], gen) if matrix else 1e-3 * torch.randn(size, generator=gen, device="cuda")
            m = 0.3 * _grad_like(size[0], size[1], gen) + 0.1 * g
            r = (g.abs() + m.abs()) * (0.5 + torch.rand(size, generator=gen, device="cuda"))
            state["params"].append(p.to(DT[case["p"]] if matrix else torch.float32).reshape(shape))
            state["grads"].append(g.to(DT[case["g"]] if matrix else torch.float32).reshape(shape))
            eight = case["bits"] == 8 and matrix
            for name, value in (("first", m), ("second", r)):
                state[name].append(_nearest_e4m3(value.reshape(shape)) if eight else (value if name == "first" else value * value).reshape(shape))
    return state


# -------------------------------------------------------------------------------------------------------- plain forms
def _power(e):
    """2^e in 32 bits, exactly, for whole e in [-126, 127]."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _plain_quantise(x):
    n, d = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -d % 128)).view(n, -1, BLOCK)
    e = (torch.frexp(x.abs().amax(-1)).exponent - 3).clamp(-127, 127)
    e = torch.where((x == 0).all(-1), -127, e)
    y = (x.abs() * _power(-e).unsqueeze(-1)).clamp(max=6.0)
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))
    q = (torch.round(y / step) * step).clamp(max=6.0)
    code = torch.where(q < 2, 2 * q, torch.where(q < 4, q + 2, q / 2 + 4)).to(torch.uint8) | (torch.signbit(x).to(torch.uint8) << 3)
    code = code.view(n, -1, 2)
    return code[..., 0] | (code[..., 1] << 4), (e + 127).to(torch.uint8)


def _plain_values(codes, scales, d):
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    v = table[torch.stack((codes & 15, codes >> 4), -1).view(codes.shape[0], -1).int()]
    s = scales.int() - 127
    half = torch.where(s < -100, s + 64, s)  # 2^-127 is below the least normal number: in two factors
    v = v.view(codes.shape[0], -1, BLOCK) * _power(half).unsqueeze(-1) * _power(s - half).unsqueeze(-1)
    return v.view(codes.shape[0], -1)[:, :d]


def _nearest_e4m3(value):
    flat = torch.nn.functional.pad(value.reshape(-1).float(), (0, -value.numel() % BLOCK8)).view(-1, BLOCK8)
    e = _scale8(flat)
    codes = (flat * _power(-e).unsqueeze(-1)).to(torch.float8_e4m3fn)
    codes = torch.where((flat != 0) & (codes.float() == 0), 2.0**-9, codes.float()).to(torch.float8_e4m3fn)
    return codes.view(-1)[: value.numel()].view(value.shape), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _scale8(blocks):
    """The least e with max |x| 2^-e <= 448 = 1.75 * 2^8 for each row (an empty row: -127)."""
    top = blocks.abs().amax(-1)
    mantissa, e = torch.frexp(top)
    e = torch.where(mantissa <= 0.875, e - 9, e - 8)
    return torch.where(top > 0, e.clamp(-126, 127), -127 + 0 * e)


def _mix(x):
    """Two rounds of xor-shift and multiply on 32 bits (held in 64)."""
    x = ((x ^ (x >> 16)) * 0x21F0AAAD) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x735A2D97) & 0xFFFFFFFF
    return x ^ (x >> 15)


def _dither(seed, tensor, step, numel, device):
    """Two times 16 random bits for every element: (for the first moment, for the second)."""
    key = _mix((_mix((seed + 0x9E3779B9 * (tensor + 1)) & 0xFFFFFFFF) + step) & 0xFFFFFFFF)
    h = _mix(torch.arange(numel, device=device) ^ key)  # (fewer than 2^32 elements)
    return h & 0xFFFF, h >> 16


def _stochastic_e4m3(y, bits, keep):
    """|y| <= 448 to e4m3 with 16 random bits: up with the probability of the part that is cut off.  keep: no value but 0 becomes 0."""
    a = y.abs()
    low = a < 2.0**-6
    t = torch.where(low, a + 2.0**-6, a)
    t = ((t.view(torch.int32) + (bits << 4).int()) & -0x100000).view(torch.float32)
    t = torch.where(low, t - 2.0**-6, t)
    if keep:
        t = torch.where((t == 0) & (a > 0), 2.0**-9, t)
    return torch.copysign(t, y).to(torch.float8_e4m3fn)


def _plain_adamw(state, i):
    b1, b2 = HYPER["betas"]
    p, g, t = state["params"][i], state["grads"][i], state["step"]
    gf = g.reshape(-1).float()
    eight = isinstance(state["first"][i], tuple)
    if eight:
        n = gf.numel()
        blocks = lambda v: torch.nn.functional.pad(v, (0, -n % BLOCK8)).view(-1, BLOCK8)  # noqa: E731
        m, r = ((blocks(c.view(-1).float()) * s.view(torch.float8_e8m0fnu).float().unsqueeze(-1)).view(-1)[:n] for c, s in (state["first"][i], state["second"][i]))
        v = r * r
    else:
        m, v = state["first"][i].view(-1), state["second"][i].view(-1)
    m = m + (gf - m) * (1 - b1)
    v = v * b2 + gf * gf * (1 - b2)
    r = v.sqrt()
    new = p.reshape(-1).float() * (1 - HYPER["lr"] * HYPER["weight_decay"]) - HYPER["lr"] / (1 - b1**t) * m / (r / math.sqrt(1 - b2**t) + HYPER["eps"])
    p.copy_(new.view(p.shape))
    if eight:
        for value, bits, (codes, scales), keep in zip((m, r), _dither(state["seed"], i, t, n, p.device), (state["first"][i], state["second"][i]), (False, True)):
            e = _scale8(blocks(value))
            y = (blocks(value) * _power(-e.clamp(max=126)).unsqueeze(-1)).view(-1)[:n]
            codes.copy_(_stochastic_e4m3(y, bits, keep).view(codes.shape))
            scales.view(torch.uint8).copy_((e + 127).to(torch.uint8))
    else:
        state["first"][i].view(-1).copy_(m)
        state["second"][i].view(-1).copy_(v)


def run(state):
    case = state["case"]
    if case["op"] == "adamw":
        state["step"] += 1
        if own:
            from clt_training_amd import hip_ops as ops

            ops.adamw_step(state["params"], state["grads"], state["first"], state["second"], step=state["step"], seed=state["seed"], **HYPER)
        else:
            for i in range(len(state["params"])):
                _plain_adamw(state, i)
        return {"p": state["params"], "m": state["first"], "v": state["second"]}
    if case["op"] == "quantise":
        if own:
            from clt_training_amd import hip_ops as ops

            return ops.mxfp4_quantize(state["x"]).dequantize(DT[case["out"]])
        codes, scales = _plain_quantise(state["x"])
        return _plain_values(codes, scales, case["d"]).to(DT[case["out"]])
    if own:
        from clt_training_amd import hip_ops as ops

        W = ops.MXFP4Tensor(state["codes"], state["scales"], case["d"])
        return ops.mxfp4_linear(state["x"], W, state["bias"], relu=case["relu"], out_dtype=DT[case["out"]])
    x = _plain_values(*_plain_quantise(state["x"]), case["d"])
    y = x @ _plain_values(state["codes"], state["scales"], case["d"]).t()
    if state["bias"] is not None:
        y += state["bias"]
    return (y.relu_() if case["relu"] else y).to(DT[case["out"]])


def work(case):
    if case["op"] == "adamw":
        table, vector = case["count"] * case["rows"] * case["cols"], case["vectors"] * case["rows"]
        moments = 16 if case["bits"] == 32 else 4 + 4 / BLOCK8
        return {"bytes": table * (2 * SIZE[case["p"]] + SIZE[case["g"]] + moments) + vector * 28, "flops": 14 * (table + vector)}
    packed = (case["d"] + -case["d"] % 128) * (1 / 2 + 1 / BLOCK)
    if case["op"] == "quantise":
        values = case["n"] * case["d"]
        return {"bytes": values * (SIZE[case["x"]] + SIZE[case["out"]]) + 2 * case["n"] * packed, "flops": 4 * values}
    n, m, d = case["n"], case["m"], case["d"]
    return {"bytes": n * d * SIZE[case["x"]] + m * packed + 4 * m * case["bias"] + n * m * SIZE[case["out"]], "flops": 2 * n * m * d}


# ---------------------------------------------------------------------------------------------------------- in 64 bits
def _exact_quantised(x):
    """The values that a row's blocks of 32 stand for once they are held in 4 bits."""
    n, d = x.shape
    x = torch.nn.functional.pad(x.double(), (0, -d % BLOCK)).view(n, -1, BLOCK)
    top = x.abs().amax(-1, keepdim=True)
    unit = torch.exp2((torch.floor(torch.log2(top.clamp(min=1e-300))) - 2).clamp(-127, 127))
    # borders between neighbours; a tie goes to the neighbour with an even last bit, so three of them belong to the upper one
    above = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    above = [b if b in (0.75, 1.75, 3.5) else math.nextafter(b, 9.0) for b in above]
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    at = torch.bucketize((x / unit).abs().contiguous(), torch.tensor(above, dtype=torch.float64, device=x.device), right=True)
    return (torch.sign(x) * grid[at] * unit).view(n, -1)[:, :d]


def _exact_table(codes, scales, d):
    c = torch.stack((codes % 16, codes // 16), -1).view(codes.shape[0], -1, BLOCK).double()
    sign = torch.where(c >= 8, -1.0, 1.0).double()
    c = c % 8
    power = torch.floor(c / 2)  # two exponent bits, one bit of mantissa
    value = torch.where(power == 0, c / 2, (1 + (c % 2) / 2) * torch.exp2(power - 1))
    return (sign * value * torch.exp2(scales.double() - 127).unsqueeze(-1)).view(codes.shape[0], -1)[:, :d]


def _exact_random(seed, tensor, step, numel, device):
    def scramble(z):
        for shift, factor in ((16, 0x21F0AAAD), (15, 0x735A2D97)):
            z = (z ^ (z >> shift)) * factor % 2**32
        return z ^ (z >> 15)

    key = scramble((scramble((seed + (tensor + 1) * 0x9E3779B9) % 2**32) + step) % 2**32)
    z = torch.arange(numel, dtype=torch.int64, device=device)
    z = scramble(z ^ key)
    return (z % 65536).double() / 65536, torch.div(z, 65536, rounding_mode="floor").double() / 65536


def _exact_rounded(value, chance, keep):
    n = value.numel()
    blocks = torch.nn.functional.pad(value, (0, -n % BLOCK8)).view(-1, BLOCK8)
    top = blocks.abs().amax(-1)
    e = torch.ceil(torch.log2(top.clamp(min=1e-300) / 448)).clamp(-126, 127)
    e = torch.where(top > 0, e, -127.0)
    y = (blocks / torch.exp2(e).unsqueeze(-1)).view(-1)[:n]
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)
    q = torch.floor(y.abs() / step + chance) * step
    if keep:
        q = torch.where((q == 0) & (y != 0), 2.0**-9, q)
    return torch.sign(y) * q, torch.exp2(e)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "quantise":
        return _exact_quantised(state["x"])
    if case["op"] == "linear":
        y = _exact_quantised(state["x"]) @ _exact_table(state["codes"], state["scales"], case["d"]).t()
        y = y if state["bias"] is None else y + state["bias"].double()
        return y.clamp(min=0) if case["relu"] else y
    out, (b1, b2), t = {"p": [], "m": [], "v": []}, HYPER["betas"], FIRST_STEP
    for i, (p, g) in enumerate(zip(state["params"], state["grads"])):
        m, v, g = state["first"][i], state["second"][i], g.double().view(-1)
        eight = isinstance(m, tuple)
        if eight:
            spread = lambda s: s.view(torch.uint8).double().sub(127).exp2().repeat_interleave(BLOCK8)[: g.numel()]  # noqa: E731
            m = m[0].view(-1).float().double() * spread(m[1])
            v = (v[0].view(-1).float().double() * spread(v[1])) ** 2
        m, v = b1 * m.double().view(-1) + (1 - b1) * g, b2 * v.double().view(-1) + (1 - b2) * g * g
        step = HYPER["lr"] * (m / (1 - b1**t)) / (torch.sqrt(v / (1 - b2**t)) + HYPER["eps"])
        out["p"].append((p.double().view(-1) * (1 - HYPER["lr"] * HYPER["weight_decay"]) - step).view(p.shape))
        if eight:
            chances = _exact_random(state["seed"], i, t, g.numel(), g.device)
            m, v = (tuple(x if k else x.view(p.shape) for k, x in enumerate(_exact_rounded(value, c, keep))) for value, c, keep in ((m, chances[0], False), (v.sqrt(), chances[1], True)))
        else:
            m, v = m.view(p.shape), v.view(p.shape)
        out["m"].append(m)
        out["v"].append(v)
    return out
