"""Performance cases of the 8-bit activation checkpoints and of the backward passes that read them.

A checkpoint holds an activation of ``rows x cols`` values for the backward pass: groups of 32 consecutive values
of a row (the last one of a row may be shorter) share a power of two, each value is a signed byte.  With a the
largest magnitude of a group and e = floor(log2 a) - 6 (at least -126), a value x is held as
q = clamp(round(x / 2^e), -127, 127) and stands for q * 2^e.

``op`` of a case:
  codec         activation -> checkpoint -> activation
  act           an activation function's forward pass, which leaves the checkpoint of its input, and its backward pass
  norm          layer norm's forward and backward pass; backward reads the checkpoint (or the input as it is)
  weight_grad   the gradients of a linear layer's weight and bias, from the checkpoint of its input
"""
import math

import torch

own = False

GROUP = 32
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
MOST_BYTES = 1.0e9
MOST_FLOPS = 1.3e11


def listed():
    return [
        # one token's hidden state: nothing but the calls' latency
        codec("codec_token", "bf16", 1, 768),
        # attention probabilities of a transformer layer (batch 32, 12 heads, sequence 512): the largest tensor that is saved
        codec("codec_attention", "f32", 32 * 12 * 512, 512),
        # hidden states behind a GELU, as the benchmark's dense activations have them
        act("gelu_hidden", "gelu", "f32", 32 * 512, 768),
        # a feed-forward layer's inner activation in a 16-bit model: the largest elementwise pass
        act("gelu_tanh_ffn", "gelu_tanh", "bf16", 32 * 512, 4096),
        # image tokens (7 of 197) of an odd width
        act("silu_odd", "silu", "f16", 7 * 197, 1111),
        # the norm in front of each sublayer of the same model
        norm("norm_hidden", "bf16", 32 * 512, 768, True),
        # few wide rows
        norm("norm_wide", "f32", 2048, 8192, True),
        # image tokens of an odd width, the input kept as it is
        norm("norm_odd_plain", "f32", 8 * 197, 193, False),
        # fine-tuning on one short sequence: latency
        weight_grad("weight_grad_short", "bf16", 64, 256, 256),
        # the attention projections of an fp32 model
        weight_grad("weight_grad_f32", "f32", 32 * 512, 768, 768),
        # a feed-forward layer of a 16-bit model
        weight_grad("weight_grad_ffn", "bf16", 32 * 512, 4096, 1024),
        # a classifier's head on image tokens: no size a multiple of anything
        weight_grad("weight_grad_odd", "f16", 8 * 197, 1000, 193),
    ]


def codec(name, dtype, rows, cols):
    return {"name": name, "op": "codec", "dtype": dtype, "rows": rows, "cols": cols}


def act(name, kind, dtype, rows, cols):
    return {"name": name, "op": "act", "kind": kind, "dtype": dtype, "rows": rows, "cols": cols}


def norm(name, dtype, rows, cols, checkpoint):
    return {"name": name, "op": "norm", "dtype": dtype, "rows": rows, "cols": cols, "checkpoint": checkpoint}


def weight_grad(name, dtype, rows, out_features, in_features):
    return {"name": name, "op": "weight_grad", "dtype": dtype, "rows": rows, "n": out_features, "cols": in_features}


def draw(rng):
    op = rng.choice(["codec", "act", "norm", "weight_grad", "weight_grad"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    while True:
        rows = log_uniform(rng, 1, 65536)
        cols = odd_or_even(rng, 16, 16384 if op != "weight_grad" else 8192)
        if op == "codec":
            case = codec("", dtype, rows, cols)
        elif op == "act":
            case = act("", rng.choice(["gelu", "gelu_tanh", "silu"]), dtype, rows, cols)
        elif op == "norm":
            case = norm("", dtype, rows, cols, rng.random() < 0.7)
        else:
            case = weight_grad("", dtype, rows, odd_or_even(rng, 16, 8192), cols)
        need = work(case)
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


# ---------------------------------------------------------------- inputs
def hidden(rows, cols, gen):
    """A hidden state: channels of different scale, a few of them far outliers, and small offsets."""
    scale = torch.exp(0.5 * torch.randn(cols, generator=gen, device="cuda"))
    scale[:: max(1, cols // 3)] *= 10.0
    shift = 0.1 * torch.randn(cols, generator=gen, device="cuda")
    return torch.randn(rows, cols, generator=gen, device="cuda").mul_(scale).add_(shift)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, rows, cols = TYPES[case["dtype"]], case["rows"], case["cols"]
    state = {"op": case["op"], "dtype": dtype, "kind": case.get("kind"), "checkpoint": case.get("checkpoint")}
    if case["op"] == "codec":
        x = torch.randn(rows, cols, generator=gen, device="cuda")
        state["x"] = (torch.softmax(x, dim=-1) if dtype == torch.float32 else x).to(dtype)
        return state
    x = hidden(rows, cols, gen).to(dtype)
    if case["op"] == "weight_grad":
        # what the forward pass left: the checkpoint of the layer's input, as its two arrays
        state["codes"], state["scales"] = pack(x)
        state["cols"] = cols
        state["dy"] = (0.01 * torch.randn(rows, case["n"], generator=gen, device="cuda")).to(dtype)
        return state
    state["x"] = x
    state["dy"] = (0.01 * torch.randn(rows, cols, generator=gen, device="cuda")).to(dtype)
    if case["op"] == "norm":
        state["weight"] = (1.0 + 0.1 * torch.randn(cols, generator=gen, device="cuda")).to(dtype)
        state["bias"] = (0.1 * torch.randn(cols, generator=gen, device="cuda")).to(dtype)
    return state


# ---------------------------------------------------------------- one pass
def run(state):
    return (run_own if own else run_plain)(state)


def run_own(state):
    from cswap_amd import q8

    op = state["op"]
    if op == "codec":
        return [q8.q8_decompress(q8.q8_compress(state["x"]))]
    if op == "act":
        y, held = q8.q8_act(state["x"], state["kind"])
        return [y, q8.q8_act_backward(state["dy"], held, state["kind"])]
    if op == "norm":
        y, mean, rstd, held = q8.layer_norm(state["x"], state["weight"], state["bias"], 1e-5,
                                            checkpoint=state["checkpoint"])
        dx, dw, db = q8.layer_norm_backward(state["dy"], held, mean, rstd, state["weight"])
        return [y, dx, dw, db]
    held = q8.Checkpoint8(state["codes"], state["scales"], (state["dy"].shape[0], state["cols"]), state["dtype"])
    return list(q8.q8_weight_grad(state["dy"], held))


def run_plain(state):
    op, dtype = state["op"], state["dtype"]
    if op == "codec":
        x = state["x"]
        return [unpack(*pack(x), x.shape[1]).to(dtype)]
    if op == "act":
        x, dy = state["x"].float(), state["dy"].float()
        held = unpack(*pack(state["x"]), x.shape[1])
        return [plain_act(x, state["kind"])[0].to(dtype), (dy * plain_act(held, state["kind"])[1]).to(dtype)]
    if op == "norm":
        return plain_norm(state)
    x = unpack(state["codes"], state["scales"], state["cols"])
    dy = state["dy"].float()
    return [(dy.t() @ x).to(dtype), dy.sum(dim=0).to(dtype)]


def groups(x):
    """rows x groups x 32, the last group of a row filled up with zeros."""
    rows, cols = x.shape
    return torch.nn.functional.pad(x, (0, -cols % GROUP)).view(rows, -1, GROUP)


def pack(x):
    g = groups(x.float())
    biased = (g.abs().amax(dim=-1).view(torch.int32) >> 23) - 6          # floor(log2) + 127 - 6
    biased = biased.clamp_(min=1)
    inverse = ((254 - biased) << 23).view(torch.float32)                 # at most 2^126: the scaling is exact
    codes = (g * inverse.unsqueeze(-1)).round_().clamp_(-127, 127).to(torch.int8)
    return codes.view(x.shape[0], -1), biased.to(torch.uint8)


def unpack(codes, scales, cols):
    unit = (scales.to(torch.int32) << 23).view(torch.float32)
    g = codes.view(codes.shape[0], -1, GROUP).float() * unit.unsqueeze(-1)
    return g.view(codes.shape[0], -1)[:, :cols]


def plain_act(x, kind):
    """The function's value and its derivative."""
    if kind == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(x * math.sqrt(0.5)))
        return x * cdf, cdf + x * torch.exp(-0.5 * x * x) / math.sqrt(2.0 * math.pi)
    if kind == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (x + 0.044715 * x * x * x))
        return 0.5 * x * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * x * (1.0 - t * t) * c * (1.0 + 0.134145 * x * x)
    s = 1.0 / (1.0 + torch.exp(-x))
    return x * s, s * (1.0 + x * (1.0 - s))


def plain_norm(state):
    dtype = state["dtype"]
    x, dy, w, b = (state[k].float() for k in ("x", "dy", "weight", "bias"))
    mean = x.mean(dim=1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((x - mean) ** 2).mean(dim=1, keepdim=True) + 1e-5)
    y = (x - mean) * rstd * w + b
    if state["checkpoint"]:
        x = unpack(*pack(state["x"]), x.shape[1])
    h = (x - mean) * rstd
    u = dy * w
    dx = rstd * (u - u.mean(dim=1, keepdim=True) - h * (u * h).mean(dim=1, keepdim=True))
    return [y.to(dtype), dx.to(dtype), (dy * h).sum(dim=0).to(dtype), dy.sum(dim=0).to(dtype)]


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    """Every input read once, every output written once; a checkpoint made and used within the pass is both."""
    size, rows, cols = SIZE[case["dtype"]], case["rows"], case["cols"]
    held = rows * (cols + -(-cols // GROUP))
    n = rows * cols
    if case["op"] == "codec":
        return {"bytes": 2 * size * n + 2 * held, "flops": 0}
    if case["op"] == "act":
        return {"bytes": 4 * size * n + 2 * held, "flops": 0}
    if case["op"] == "norm":
        kept = 2 * held if case["checkpoint"] else size * n
        return {"bytes": 4 * size * n + kept + 16 * rows + 4 * size * cols, "flops": 0}
    out = case["n"]
    return {"bytes": size * rows * out + held + size * out * (cols + 1), "flops": 2 * rows * out * cols}


# ---------------------------------------------------------------- from the definitions, in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "weight_grad":
        # the bytes as they are: a signed byte times a power of two
        power = torch.pow(2.0, state["scales"].double() - 127.0)
        x = (state["codes"].double() * power.repeat_interleave(GROUP, dim=1))[:, : case["cols"]]
        dy = state["dy"].double()
        return [torch.matmul(dy.t().contiguous(), x.contiguous()), dy.sum(dim=0)]
    x = state["x"].double()
    if op == "codec":
        return [held_exactly(x)]
    dy = state["dy"].double()
    if op == "act":
        value, _ = act_exactly(x, case["kind"])
        _, slope = act_exactly(held_exactly(x), case["kind"])
        return [value, dy * slope]
    w, b = state["weight"].double(), state["bias"].double()
    variance, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    deviation = torch.sqrt(variance + 1e-5)
    y = (x - mean) / deviation * w + b
    kept = held_exactly(x) if case["checkpoint"] else x
    h = (kept - mean) / deviation
    u = dy * w
    cols = x.shape[1]
    dx = (u - (u.sum(dim=1, keepdim=True) + h * (u * h).sum(dim=1, keepdim=True)) / cols) / deviation
    return [y, dx, (dy * h).sum(dim=0), dy.sum(dim=0)]


def held_exactly(x):
    """What a checkpoint of x stands for."""
    rows, cols = x.shape
    count = -(-cols // GROUP)
    filled = torch.zeros(rows, count * GROUP, dtype=torch.float64, device=x.device)
    filled[:, :cols] = x
    filled = filled.view(rows, count, GROUP)
    _, exponent = torch.frexp(filled.abs().amax(dim=2, keepdim=True))    # a = m 2^exponent, 1/2 <= m < 1
    step = ((exponent.long() - 7).clamp(min=-126) + 1023 << 52).view(torch.float64)     # 2^e to the bit: a library's power may not be
    return (torch.round(filled / step).clamp(-127, 127) * step).view(rows, -1)[:, :cols]


def act_exactly(x, kind):
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
