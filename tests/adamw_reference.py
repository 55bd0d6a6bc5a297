"""AdamW and its moments in 8 bits from their definitions, element by element in 64 bits with the roundings to fp32 that the definition names;
on the CPU, without the package."""
import math

import torch

GROUP = 32
A, B = 0xC13FA9A9, 0x91E10DA5
NEAREST = 1 << 31


def single(x):
    """Rounded to fp32."""
    return x.to(torch.float32).to(torch.float64)


def power(e):
    return torch.ldexp(torch.ones((), dtype=torch.float64), e.to(torch.int32)) if isinstance(e, torch.Tensor) else 2.0 ** e


def least(signed):
    return 2.0 ** (-8 if signed else -24)


def groups(x):
    n = x.numel()
    return torch.nn.functional.pad(x.reshape(-1), (0, -n % GROUP)).view(-1, GROUP)


def offsets(n, step, signed):
    """u of every value of a tensor, its group padding included."""
    i = torch.arange(-(-n // GROUP) * GROUP, dtype=torch.int64)
    a, b = (A, B) if signed else (B, A)
    return (i * a + step * b) % (1 << 32)


def pack(x, u, signed):
    """Codes (uint8, whole groups) and scales of fp32 values x; u: offsets of whole groups, or one for all."""
    g = groups(x.double())
    top = g.abs().amax(dim=1)
    finite = torch.isfinite(g).all(dim=1)
    _, exponent = torch.frexp(torch.where(finite, top, torch.ones_like(top)))
    e = torch.where(top == 0, -126, (exponent - 7).clamp(min=-126))          # floor(log2 top) - 6; frexp gives 0 the exponent 0
    t = least(signed)
    y = single(torch.where(finite[:, None], g.abs(), 0.0) / power(e)[:, None] + t) / t
    mantissa, k = torch.frexp(y)                             # y = 2 mantissa 2^(k - 1), 1 <= 2 mantissa < 2
    u = torch.as_tensor(u).reshape(-1, GROUP) if isinstance(u, torch.Tensor) else torch.full(g.shape, u)
    code = 8 * (k - 1) + torch.floor(8 * (2 * mantissa - 1) + torch.div(u, 4096, rounding_mode="floor").double() / 2 ** 20).long()
    if signed:
        code = code + 128 * torch.signbit(g).long()
    code = torch.where(finite[:, None], code, 0)
    return code.view(-1).to(torch.uint8), torch.where(finite, e + 127, 255).to(torch.uint8)


def pack_pair(m, v, um, uv):
    """Both moments: where v's code is 0 m's is."""
    vc, vs = pack(v, uv, False)
    mc, ms = pack(m, um, True)
    return (torch.where(vc != 0, mc, torch.zeros_like(mc)), ms), (vc, vs)


def unpack(codes, scales, n, signed):
    c = codes.long()
    size = c % 128 if signed else c
    t = least(signed)
    y = single(torch.ldexp(1 + (size % 8).double() / 8, torch.div(size, 8, rounding_mode="floor").to(torch.int32)) * t - t)
    unit = torch.where(scales == 255, torch.nan, power(scales.int() - 127)).repeat_interleave(GROUP)
    y = y * unit
    return (torch.where(c >= 128, -y, y) if signed else y)[:n]


def room(codes, scales):
    """As the optimiser keeps them."""
    return torch.cat([codes, scales])


def split(held, n):
    count = -(-n // GROUP)
    return held[:count * GROUP], held[count * GROUP:]


def moments(m, v, g, betas):
    """m' and v', rounded to fp32 after each product and sum."""
    b = single(torch.tensor([betas[0], 1 - betas[0], betas[1], 1 - betas[1]], dtype=torch.float64))
    m = single(single(m.double() * b[0]) + single(g.double() * b[1]))
    v = single(single(v.double() * b[2]) + single(single(g.double() * g.double()) * b[3]))
    return m, v


def update(p, m, v, step, lr, betas, eps, decay):
    """p' from the new moments, and the size of the terms it is made of."""
    c1, c2 = 1 - betas[0] ** step, 1 - betas[1] ** step
    change = lr / c1 * m / (torch.sqrt(v) / math.sqrt(c2) + eps)
    return p.double() * (1 - lr * decay) - change, p.double().abs() + change.abs()
