"""Performance cases of a training step's other halves in 8 bits: the optimiser's, the norms of convolution nets and the
products of linear layers.

``op`` of a case:
  adamw   one AdamW step over all tensors of a model, moments in 8 bits or in fp32
  norm    group norm with an activation, channels last: forward and backward pass; backward reads the 8-bit checkpoint of
          the input (or the input as it is)
  linear  a product in 8-bit floating point (e4m3) with a power of two for each 128 values of a row of activations and for each
          128 x 128 weights.  ``train``: weights laid out, y = x W^T + b, dx = dy W; else y alone from weights laid out before

Moments in 8 bits: 32 consecutive values share a power of two 2^e, e = floor(log2 of the largest) - 6, a byte; a value's
magnitude y = |x| / 2^e is held by the sign, exponent and three bits of y + T (T = 2^-8 for the first moment, 2^-24 for the second, which has no
sign): code c stands for (2^(c / 8) (1 + (c mod 8) / 8) T - T) 2^e.  What is cut off is carried up where it and the step's
offset u (an element's place in its tensor and the step's number, each times a constant) make a whole: over the steps every value
between two codes is held by both in its proportion.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
MOST_BYTES = 1.6e9
MOST_FLOPS = 2.8e11

GROUP = 32                                # values of a moment or of a checkpoint that share a power of two
OFFSET_A, OFFSET_B = 0xC13FA9A9, 0x91E10DA5   # 2^32 over the plastic number and over its square
LR, BETAS, EPS, DECAY = 1e-3, (0.9, 0.999), 1e-8, 1e-2
BLOCK = 128                               # values of a row, and rows and columns of weights, that share one in a product


def listed():
    return [
        # a classifier's head being fine-tuned: two small tensors, latency
        adamw("adamw_head", "f32", 8, False, 512, 0, 10),
        # a 16-bit encoder's parameters, moments in 8 bits
        adamw("adamw_encoder_8bit", "bf16", 8, False, 1024, 8, 1000),
        # an fp32 model with fp32 moments, as checkpoints of other frameworks hold them
        adamw("adamw_encoder_32bit", "f32", 32, False, 1024, 4, 1000),
        # odd widths, fp32 copies of fp16 parameters: no size a multiple of a group
        adamw("adamw_odd", "f16", 8, True, 193, 3, 1000),
        # last layer of a small convolution net at batch 2: latency
        norm("norm_small", "f32", 2, 64, 8, 8, 8, "silu", True),
        # an image model's middle, 16 bits
        norm("norm_image", "bf16", 16, 256, 64, 64, 32, "silu", True),
        # the first block of a VGG net on 64 x 64 images at batch 128: the largest activation
        norm("norm_first", "f32", 128, 64, 64, 64, 32, "gelu", True),
        # an inception block's odd image, 12 channels to a group, input kept as it is
        norm("norm_odd_plain", "f16", 7, 288, 35, 35, 24, "none", False),
        # one token through a feed-forward layer whose weights were laid out before
        linear("linear_token", "bf16", 1, 4096, 1024, False),
        # a feed-forward layer of a 16-bit model at batch 32, sequence 512
        linear("linear_ffn", "bf16", 32 * 512, 4096, 1024, True),
        # the attention projections of an fp32 model
        linear("linear_hidden", "f32", 32 * 512, 768, 768, True),
        # a classifier on image tokens: no size a multiple of anything
        linear("linear_odd", "f16", 8 * 197, 1000, 193, True),
    ]


def adamw(name, dtype, bits, master, hidden, layers, classes):
    return {"name": name, "op": "adamw", "dtype": dtype, "bits": bits, "master": master, "hidden": hidden, "layers": layers,
            "classes": classes}


def norm(name, dtype, batch, channels, height, width, groups, act, checkpoint):
    return {"name": name, "op": "norm", "dtype": dtype, "batch": batch, "channels": channels, "height": height, "width": width,
            "groups": groups, "act": act, "checkpoint": checkpoint}


def linear(name, dtype, rows, out_features, in_features, train):
    return {"name": name, "op": "linear", "dtype": dtype, "rows": rows, "n": out_features, "k": in_features, "train": train}


def draw(rng):
    op = rng.choice(["adamw", "norm", "norm", "linear", "linear", "linear"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    while True:
        if op == "adamw":
            case = adamw("", dtype, rng.choice([8, 8, 32]), dtype != "f32" and rng.random() < 0.3, odd_or_even(rng, 16, 2048),
                         rng.choice([0, 1, 2, 4, 6, 12]), odd_or_even(rng, 2, 32768))
        elif op == "norm":
            groups = rng.choice([1, 3, 8, 16, 32])
            case = norm("", dtype, log_uniform(rng, 1, 128), groups * log_uniform(rng, 1, 1024 // groups), log_uniform(rng, 1, 128),
                        log_uniform(rng, 1, 128), groups, rng.choice(["none", "gelu", "gelu_tanh", "silu", "silu"]),
                        rng.random() < 0.7)
        else:
            train = rng.random() < 0.6
            case = linear("", dtype, log_uniform(rng, 1, 65536 if train else 256), odd_or_even(rng, 16, 8192),
                          odd_or_even(rng, 16, 8192), train)
        need = work(case)
        if op == "norm" and case["height"] * case["width"] * case["channels"] < 16 * case["groups"]:
            continue                # a few values to a group: their gradient all but cancels, and nobody norms them so
        if need["bytes"] <= MOST_BYTES and need["flops"] <= MOST_FLOPS:
            del case["name"]
            return case


def log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def odd_or_even(rng, low, high):
    """Widths as models have them (multiples of 32 or 64), and any other."""
    v = log_uniform(rng, low, high)
    step = rng.choice([1, 1, 8, 32, 64, 128])
    return max(low, v // step * step)


def parameters(case):
    """Sizes of a model's tensors: encoder layers (four projections, a feed-forward pair of four times the width, two norms), a classifier."""
    h, c = case["hidden"], case["classes"]
    layer = [h * h, h] * 4 + [4 * h * h, 4 * h, 4 * h * h, h] + [h] * 4
    return layer * case["layers"] + [c * h, c]


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"adamw": prepare_adamw, "norm": prepare_norm, "linear": prepare_linear}[case["op"]](case, gen)


def randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def prepare_adamw(case, gen):
    """Parameters and gradients as views of two buffers, each from a multiple of 256 values on (there are zeros between them, which a step
    leaves zeros), and the moments that 100 steps have left."""
    sizes = parameters(case)
    dtype = TYPES[case["dtype"]]
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + -(-n // 256) * 256)
    total = starts.pop()
    place = torch.full((total,), -1, dtype=torch.int64, device="cuda")     # of an element in its tensor
    for s, n in zip(starts, sizes):
        place[s:s + n] = torch.arange(n, device="cuda")
    there = (place >= 0).float()
    # gradients differ in size from place to place, smoothly and by outliers
    size = torch.exp(0.7 * randn(gen, total)) * (1e-3 * there)
    grad = (randn(gen, total) * size).to(dtype)
    master = 0.02 * randn(gen, total) * there
    param = master.to(dtype)
    m = 0.25 * randn(gen, total) * size
    v = size * size * torch.exp(0.3 * randn(gen, total)) * 0.1
    state = {"op": "adamw", "bits": case["bits"], "sizes": sizes, "starts": starts, "place": place, "param": param, "grad": grad,
             "master": master if case["master"] else None, "step": 100,
             "out": [torch.zeros(total, device="cuda") for _ in range(2)]}
    if case["bits"] == 8:
        none = torch.full((total,), 1 << 31, dtype=torch.int64, device="cuda")
        v_codes, v_scales = pack_moment(v, none, False)
        m_codes, m_scales = pack_moment(m, none, True)
        state["m"], state["v"] = [m_codes * (v_codes != 0), m_scales], [v_codes, v_scales]
    else:
        state["m"], state["v"] = m, v
    return state


def prepare_norm(case, gen):
    dtype = TYPES[case["dtype"]]
    n, c, h, w = (case[k] for k in ("batch", "channels", "height", "width"))
    scale = torch.exp(0.5 * randn(gen, c))
    scale[:: max(1, c // 3)] *= 10.0
    x = randn(gen, n, h, w, c).mul_(scale).add_(scale * randn(gen, c))
    return {"op": "norm", "dtype": dtype, "groups": case["groups"], "act": case["act"], "checkpoint": case["checkpoint"],
            "x": x.to(dtype).permute(0, 3, 1, 2), "dy": (0.01 * randn(gen, n, h, w, c)).to(dtype).permute(0, 3, 1, 2),
            "weight": (1.0 + 0.1 * randn(gen, c)).to(dtype), "bias": (0.1 * randn(gen, c)).to(dtype)}


def prepare_linear(case, gen):
    dtype, rows, n, k = TYPES[case["dtype"]], case["rows"], case["n"], case["k"]
    scale = torch.exp(0.5 * randn(gen, k))
    scale[:: max(1, k // 3)] *= 10.0
    w = (randn(gen, n, k) / math.sqrt(k)).to(dtype)
    state = {"op": "linear", "dtype": dtype, "train": case["train"], "n": n, "k": k, "w": w,
             "x": randn(gen, rows, k).mul_(scale).to(dtype), "bias": (0.1 * randn(gen, n)).to(dtype)}
    if case["train"]:
        state["dy"] = (0.01 * randn(gen, rows, n)).to(dtype)
    else:
        state["codes"], state["scales"] = pack_weight(w)
    return state


# ---------------------------------------------------------------- one pass
def run(state):
    return (run_own if own else run_plain)(state)


def run_own(state):
    if state["op"] == "adamw":
        return own_adamw(state)
    if state["op"] == "norm":
        from cswap_amd import q8

        act = None if state["act"] == "none" else state["act"]
        y, mean, rstd, held = q8.group_norm(state["x"], state["groups"], state["weight"], state["bias"], 1e-5, act=act,
                                            checkpoint=state["checkpoint"])
        return [y, *q8.group_norm_backward(state["dy"], held, mean, rstd, state["groups"], state["weight"], state["bias"], act=act)]
    from cswap_amd import f8

    if state["train"]:
        held = f8.f8_weight(state["w"])
        return [f8.f8_linear(state["x"], held, state["bias"]), f8.f8_linear_backward(state["dy"], held)]
    held = f8.F8Weight(state["codes"], state["scales"], (state["n"], state["k"]), state["dtype"])
    return [f8.f8_linear(state["x"], held, state["bias"])]


def own_adamw(state):
    from cswap_amd import adamw8

    optimizer = state.get("optimizer")
    if optimizer is None:           # a program makes its optimiser once; its moments are read from a checkpoint
        optimizer = state["optimizer"] = own_optimizer(state)
    optimizer.step()
    if state["bits"] == 8:          # moments as the values that they stand for
        adamw8.unpack_moments(optimizer, state["views"])
        return [state["param"], *state["out"], *masters(state)]
    return [state["param"], state["m"], state["v"], *masters(state)]


def own_optimizer(state):
    from cswap_amd import adamw8

    params, views = [], []
    for s, n in zip(state["starts"], state["sizes"]):
        p = torch.nn.Parameter(state["param"][s:s + n])
        p.grad = state["grad"][s:s + n]
        params.append(p)
        views.append([out[s:s + n] for out in state["out"]])
    state["views"] = views
    optimizer = adamw8.AdamW8(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, bits=state["bits"],
                              master=state["master"] is not None)
    for p, s, n in zip(params, state["starts"], state["sizes"]):
        held = {"step": state["step"]}
        for key, kept in (("exp_avg", state["m"]), ("exp_avg_sq", state["v"])):
            if state["bits"] == 8:      # 32 codes of each group of the tensor, then their scales
                a, b = s // GROUP, s // GROUP + -(-n // GROUP)
                held[key] = torch.cat([kept[0].view(-1, GROUP)[a:b].reshape(-1), kept[1][a:b]])
            else:
                held[key] = kept[s:s + n]
        if state["master"] is not None:
            held["master"] = state["master"][s:s + n]
        optimizer.state[p].update(held)
    return optimizer


def masters(state):
    return [] if state["master"] is None else [state["master"]]


def run_plain(state):
    if state["op"] == "adamw":
        return plain_adamw(state)
    if state["op"] == "norm":
        return plain_norm(state)
    x = unpack_rows(*pack_rows(state["x"]), state["k"])
    w8 = pack_weight(state["w"]) if state["train"] else (state["codes"], state["scales"])
    w = unpack_weight(*w8, state["n"], state["k"])
    out = [(x @ w.t() + state["bias"].float()).to(state["dtype"])]
    if state["train"]:
        dy = unpack_rows(*pack_rows(state["dy"]), state["n"])
        out.append((dy @ w).to(state["dtype"]))
    return out


# ---------------------------------------------------------------- AdamW
def moment_limits(signed):
    """bits(T), T and the number of magnitudes of a code."""
    exponent = 119 if signed else 103
    return exponent << 23, 2.0 ** (exponent - 127)


def pack_moment(x, offset, signed):
    first, least = moment_limits(signed)
    g = x.abs().view(-1, GROUP)
    bits = g.amax(dim=1).view(torch.int32) >> 23
    scale = (bits - 6).clamp_(min=1)
    inverse = ((254 - scale) << 23).view(torch.float32)
    y = (g * inverse.unsqueeze(1) + least).view(torch.int32).view(-1)
    code = ((y - first + (offset >> 12).to(torch.int32)) >> 20).to(torch.uint8)
    if signed:
        code |= (x < 0).to(torch.uint8) << 7
    return code, scale.to(torch.uint8)


def unpack_moment(code, scale, signed):
    first, least = moment_limits(signed)
    c = code.to(torch.int32)
    y = ((((c & 127) if signed else c) << 20) + first).view(torch.float32) - least
    unit = (scale.to(torch.int32) << 23).view(torch.float32)
    x = (y.view(-1, GROUP) * unit.unsqueeze(1)).view(-1)
    return torch.where(c >= 128, -x, x) if signed else x


def plain_adamw(state):
    state["step"] += 1
    t, (b1, b2) = state["step"], BETAS
    small = state["bits"] == 8
    p = (state["param"] if state["master"] is None else state["master"]).float()
    g = state["grad"].float()
    m = unpack_moment(*state["m"], True) if small else state["m"]
    v = unpack_moment(*state["v"], False) if small else state["v"]
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + (g * g) * (1.0 - b2)
    denominator = v.sqrt() * (1.0 / math.sqrt(1.0 - b2 ** t)) + EPS
    p = p * (1.0 - LR * DECAY) - m / denominator * (LR / (1.0 - b1 ** t))
    state["param"].copy_(p)
    if state["master"] is not None:
        state["master"].copy_(p)
    if not small:
        state["m"].copy_(m)
        state["v"].copy_(v)
        return [state["param"], state["m"], state["v"], *masters(state)]
    at = state["place"].clamp(min=0)
    state["v"] = pack_moment(v, (at * OFFSET_B + t * OFFSET_A) & 0xFFFFFFFF, False)
    codes, scales = pack_moment(m, (at * OFFSET_A + t * OFFSET_B) & 0xFFFFFFFF, True)
    state["m"] = codes * (state["v"][0] != 0), scales         # nothing over nothing: no first moment without a second
    return [state["param"], unpack_moment(*state["m"], True), unpack_moment(*state["v"], False), *masters(state)]


# ---------------------------------------------------------------- group norm
def rows_of(x):
    """[N, C, H, W] in channels-last memory as [N, H W, C]."""
    return x.permute(0, 2, 3, 1).flatten(1, 2)


def checkpoint8(x):
    """What the 8-bit checkpoint of rows stands for: 32 values share 2^e, e = floor(log2 of the largest) - 6."""
    n = x.shape[-1]
    g = torch.nn.functional.pad(x, (0, -n % GROUP)).unflatten(-1, (-1, GROUP))
    biased = ((g.abs().amax(dim=-1, keepdim=True).view(torch.int32) >> 23) - 6).clamp_(min=1)
    q = (g * ((254 - biased) << 23).view(torch.float32)).round_().clamp_(-127, 127)
    return (q * (biased << 23).view(torch.float32)).flatten(-2)[..., :n]


def plain_act(z, kind):
    """The function's value and its derivative."""
    if kind == "none":
        return z, torch.ones_like(z)
    if kind == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if kind == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 0.134145 * z * z)
    s = 1.0 / (1.0 + torch.exp(-z))
    return z * s, s * (1.0 + z * (1.0 - s))


def plain_norm(state):
    dtype, groups, shape = state["dtype"], state["groups"], state["x"].shape
    x, dy = rows_of(state["x"]).float(), rows_of(state["dy"]).float()
    w, b = (state[k].float().view(groups, -1) for k in ("weight", "bias"))
    back = lambda t: t.reshape(shape[0], *shape[2:], shape[1]).to(dtype).permute(0, 3, 1, 2)  # noqa: E731
    split = lambda t: t.unflatten(-1, (groups, -1))                                         # noqa: E731
    g = split(x)
    mean = g.mean(dim=(1, 3), keepdim=True)
    rstd = 1.0 / torch.sqrt(((g - mean) ** 2).mean(dim=(1, 3), keepdim=True) + 1e-5)
    y = plain_act((g - mean) * rstd * w + b, state["act"])[0]
    h = (split(checkpoint8(x)) - mean) * rstd if state["checkpoint"] else (g - mean) * rstd
    dz = split(dy) * plain_act(h * w + b, state["act"])[1]
    u = dz * w
    dx = rstd * (u - u.mean(dim=(1, 3), keepdim=True) - h * (u * h).mean(dim=(1, 3), keepdim=True))
    return [back(y), back(dx), (dz * h).sum(dim=(0, 1)).view(-1).to(dtype), dz.sum(dim=(0, 1)).view(-1).to(dtype)]


# ---------------------------------------------------------------- products in 8-bit floating point
def block_scale(largest):
    """The byte of the least power of two (2^-126 at least) that makes the largest magnitude at most 448."""
    bits = largest.view(torch.int32)
    return ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000)).clamp_(min=1)


def to_e4m3(x, scale):
    return (x * ((254 - scale) << 23).view(torch.float32)).to(torch.float8_e4m3fn)


def pack_rows(x):
    rows, k = x.shape
    g = torch.nn.functional.pad(x.float(), (0, -k % BLOCK)).view(rows, -1, BLOCK)
    scale = block_scale(g.abs().amax(dim=2, keepdim=True))
    return to_e4m3(g, scale), scale


def unpack_rows(codes, scale, k):
    return (codes.float() * (scale << 23).view(torch.float32)).flatten(1)[:, :k]


def pack_weight(w):
    """Codes (rows and columns filled up with zeros to whole blocks) and scales, block rows x block columns."""
    n, k = w.shape
    g = torch.nn.functional.pad(w.float(), (0, -k % BLOCK, 0, -n % BLOCK))
    g = g.view(-(-n // BLOCK), BLOCK, -1, BLOCK)
    scale = block_scale(g.abs().amax(dim=(1, 3), keepdim=True))
    return to_e4m3(g, scale).flatten(2).flatten(0, 1), scale.view(scale.shape[0], -1).to(torch.uint8)


def unpack_weight(codes, scales, n, k):
    unit = (scales.to(torch.int32) << 23).view(torch.float32)
    g = codes.float().view(scales.shape[0], BLOCK, scales.shape[1], BLOCK) * unit[:, None, :, None]
    return g.flatten(2).flatten(0, 1)[:n, :k]


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    """Every input read once, every output written once; a checkpoint made and used within the pass is both."""
    size = SIZE[case["dtype"]]
    if case["op"] == "adamw":
        n = sum(parameters(case))
        moments = 4 * n * (GROUP + 1) / GROUP if case["bits"] == 8 else 16 * n      # read and written
        values = 8 * n if case["bits"] == 8 else 0                                   # as which the 8-bit ones come back
        return {"bytes": 3 * size * n + moments + values + (8 - size) * n * case["master"], "flops": 0}
    if case["op"] == "norm":
        c, rows = case["channels"], case["batch"] * case["height"] * case["width"]
        kept = 2 * rows * (c + -(-c // GROUP)) if case["checkpoint"] else size * rows * c
        return {"bytes": 4 * size * rows * c + kept + 6 * size * c, "flops": 0}
    rows, n, k = case["rows"], case["n"], case["k"]
    if case["train"]:
        return {"bytes": size * (2 * rows * (n + k) + n * k + n), "flops": 4 * rows * n * k}
    return {"bytes": size * (rows * (n + k) + n) + n * k, "flops": 2 * rows * n * k}


# ---------------------------------------------------------------- from the definitions, in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return {"adamw": exact_adamw, "norm": exact_norm, "linear": exact_linear}[case["op"]](case, state)


def power(e):
    """2^e to the bit: a library's power may not be."""
    return (e.long() + 1023 << 52).view(torch.float64)


def moment_value(code, scale, signed):
    c = code.long()
    size = c % 128 if signed else c
    t = 2.0 ** (-8 if signed else -24)
    y = (power(torch.div(size, 8, rounding_mode="floor")) * (1 + (size % 8).double() / 8) - 1) * t
    return torch.where(c >= 128, -1.0, 1.0) * y * unit_of(scale) if signed else y * unit_of(scale)


def unit_of(scale):
    return power(scale.long() - 127).repeat_interleave(GROUP)


def moment_held(x, offset, signed, keep=None):
    """What x is held as: the code below or above (x + T) that the offset, a share of 2^32, decides for."""
    t = 2.0 ** (-8 if signed else -24)
    _, exponent = torch.frexp(x.abs().view(-1, GROUP).amax(dim=1))
    unit = power((exponent.long() - 7).clamp(min=-126)).repeat_interleave(GROUP)
    mantissa, exponent = torch.frexp(single(x.abs() / unit + t) / t)          # at least 1: 1/2 <= mantissa < 1
    eighths = torch.floor(16 * mantissa + torch.div(offset, 4096, rounding_mode="floor").double() / 2 ** 20) - 8
    code = 8 * (exponent.long() - 1) + eighths.long()
    if keep is not None:
        code = code * keep
    y = (power(torch.div(code, 8, rounding_mode="floor")) * (1 + (code % 8).double() / 8) - 1) * t * unit
    return torch.where(x < 0, -y, y), code != 0


def single(x):
    """Rounded to fp32, where the definition says so."""
    return x.float().double()


def exact_adamw(case, state):
    t, (b1, b2) = state["step"] + 1, BETAS
    p = (state["param"] if state["master"] is None else state["master"]).double()
    g = state["grad"].double()
    if case["bits"] == 8:
        m, v = moment_value(*state["m"], True), moment_value(*state["v"], False)
    else:
        m, v = state["m"].double(), state["v"].double()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g ** 2
    p = (1 - LR * DECAY) * p - LR * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + EPS)
    if case["bits"] == 8:
        at = state["place"].clamp(min=0)
        m0, v0, (c1, c2) = moment_value(*state["m"], True), moment_value(*state["v"], False), single(torch.tensor(BETAS, dtype=torch.float64)).tolist()
        d1, d2 = single(torch.tensor([1 - b1, 1 - b2], dtype=torch.float64)).tolist()
        v = single(single(c2 * single(v0)) + single(d2 * single(g * g)))
        m = single(single(c1 * single(m0)) + single(d1 * g))
        v, there = moment_held(v, (at * OFFSET_B + t * OFFSET_A) % 2 ** 32, False)
        m, _ = moment_held(m, (at * OFFSET_A + t * OFFSET_B) % 2 ** 32, True, there)
    return [p, m, v] + ([p] if case["master"] else [])


def exact_norm(case, state):
    n, c, h, w = state["x"].shape
    groups, act = case["groups"], case["act"]
    x = state["x"].permute(0, 2, 3, 1).double().reshape(n, h * w, groups, c // groups)
    dy = state["dy"].permute(0, 2, 3, 1).double().reshape(x.shape)
    gamma, beta = (state[k].double().reshape(groups, -1) for k in ("weight", "bias"))
    variance, mean = torch.var_mean(x, dim=(1, 3), correction=0, keepdim=True)
    deviation = torch.sqrt(variance + 1e-5)
    kept = held_exactly(x.reshape(-1, c)).reshape(x.shape) if case["checkpoint"] else x
    y = act_exactly((x - mean) / deviation * gamma + beta, act)[0]
    hat = (kept - mean) / deviation
    dz = dy * act_exactly(hat * gamma + beta, act)[1]
    u = dz * gamma
    count = h * w * (c // groups)
    dx = (u - (u.sum(dim=(1, 3), keepdim=True) + hat * (u * hat).sum(dim=(1, 3), keepdim=True)) / count) / deviation
    image = lambda t: t.reshape(n, h, w, c).permute(0, 3, 1, 2)  # noqa: E731
    return [image(y), image(dx), (dz * hat).sum(dim=(0, 1)).reshape(-1), dz.sum(dim=(0, 1)).reshape(-1)]


def held_exactly(x):
    """What a checkpoint of rows x stands for."""
    rows, cols = x.shape
    count = -(-cols // GROUP)
    filled = torch.zeros(rows, count * GROUP, dtype=torch.float64, device=x.device)
    filled[:, :cols] = x
    filled = filled.view(rows, count, GROUP)
    _, exponent = torch.frexp(filled.abs().amax(dim=2, keepdim=True))    # a = m 2^exponent, 1/2 <= m < 1
    step = power((exponent.long() - 7).clamp(min=-126))
    return (torch.round(filled / step).clamp(-127, 127) * step).view(rows, -1)[:, :cols]


def act_exactly(x, kind):
    if kind == "none":
        return x, torch.ones_like(x)
    if kind == "gelu":
        cdf = 0.5 * torch.special.erfc(-x / math.sqrt(2.0))
        return x * cdf, cdf + x * torch.exp(-x * x / 2.0) / math.sqrt(2.0 * math.pi)
    if kind == "gelu_tanh":
        # (1 + tanh z) / 2 = 1 / (1 + exp(-2 z))
        c = 2.0 * math.sqrt(2.0 / math.pi)
        s = torch.sigmoid(c * (x + 0.044715 * x ** 3))
        return x * s, s + x * s * (1.0 - s) * c * (1.0 + 3.0 * 0.044715 * x ** 2)
    s = torch.sigmoid(x)
    return x * s, s + x * s * (1.0 - s)


def e4m3_exactly(x, block_rows):
    """x in blocks of block_rows x 128, each a power of two times values of four significant bits, 2^-9 at the least and 448 at the most."""
    rows, cols = x.shape
    full = torch.zeros(-(-rows // block_rows) * block_rows, -(-cols // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    full[:rows, :cols] = x
    g = full.view(-1, block_rows, full.shape[1] // BLOCK, BLOCK)
    mantissa, exponent = torch.frexp(g.abs().amax(dim=(1, 3), keepdim=True) / 448.0)
    unit = power((exponent.long() - (mantissa == 0.5).long()).clamp(min=-126))
    g = g / unit
    _, exponent = torch.frexp(g)
    step = power((exponent.long() - 4).clamp(min=-9))
    return (torch.round(g / step) * step * unit).view(full.shape)[:rows, :cols].contiguous()


def exact_linear(case, state):
    x = e4m3_exactly(state["x"].double(), 1)
    w = e4m3_exactly(state["w"].double(), BLOCK)
    out = [torch.matmul(x, w.t().contiguous()) + state["bias"].double()]
    if case["train"]:
        out.append(torch.matmul(e4m3_exactly(state["dy"].double(), 1), w))
    return out
