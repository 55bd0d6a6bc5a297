"""Plain 64-bit forms of the 8-bit checkpoints and of what reads them, and the error that fp32 arithmetic may
leave around them.  U = 2^-24 is half a step of fp32; a sum of k terms in any order is off by at most k U sum|terms|."""
import math

import torch

U = 2.0 ** -24
GROUP = 32


def half_step(value, dtype):
    """What rounding ``value`` (64 bits) to ``dtype`` may add: half a step, or half the smallest subnormal."""
    least = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}[dtype]
    return torch.clamp(value.abs() * (torch.finfo(dtype).eps / 2), min=least / 2)


def power_of_two(e):
    """2^e to the bit, -1022 <= e <= 1023 (a library's power need not be)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def pack(x, keep_sign=False):
    """codes (rows x pitch, int8), scales (rows x groups, uint8) of a 2-D tensor of any type."""
    x = x.detach().cpu().double()
    rows, cols = x.shape
    groups = -(-cols // GROUP)
    full = torch.zeros(rows, groups * GROUP, dtype=torch.float64)
    full[:, :cols] = x
    g = full.view(rows, groups, GROUP)
    finite = torch.isfinite(g).all(dim=2, keepdim=True)
    g = torch.where(finite, g, torch.zeros_like(g))
    _, ex = torch.frexp(g.abs().amax(dim=2, keepdim=True))          # a = m 2^ex, 1/2 <= m < 1; 0 for a = 0
    zero = g.abs().amax(dim=2, keepdim=True) == 0
    e = torch.where(zero, torch.full_like(ex, -126), (ex - 7).clamp(-126, 121))
    q = torch.round(g * power_of_two(-e)).clamp(-127, 127)
    if keep_sign:
        q = torch.where(q == 0, torch.sign(g), q)
    scales = torch.where(finite, e + 127, torch.full_like(e, 255)).to(torch.uint8)
    return q.to(torch.int8).view(rows, -1), scales.view(rows, groups)


def unpack(codes, scales, cols):
    """What they stand for, 64 bits (NaN for groups that held what is not finite)."""
    codes, scales = codes.cpu().double(), scales.cpu()
    unit = power_of_two(scales.long() - 127)
    unit = torch.where(scales == 255, torch.full_like(unit, math.nan), unit)
    return (codes.view(*scales.shape, GROUP) * unit.unsqueeze(2)).view(codes.shape)[:, :cols]


def held(x, keep_sign=False):
    return unpack(*pack(x, keep_sign), x.shape[1])


# ---------------------------------------------------------------- activation functions: value, slope
def act(x, kind):
    if kind == "gelu":
        cdf = 0.5 * torch.special.erfc(-x / math.sqrt(2.0))
        pdf = torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
        return x * cdf, cdf + x * pdf
    if kind == "gelu_tanh":
        c = 2.0 * math.sqrt(2.0 / math.pi)
        z, dz = c * (x + 0.044715 * x ** 3), c * (1 + 3 * 0.044715 * x ** 2)
    else:
        z, dz = x, torch.ones_like(x)
    s, o = torch.sigmoid(z), torch.sigmoid(-z)
    return x * s, s * (1 + x * o * dz)


def act_error(x, kind, dtype):
    """Bounds on the fp32 error of value and slope.

    gelu: the tail T = Phi(-|x|) is exp(-x^2/2) R; R is off by 4.2e-7 (fp32) or 1.2e-5 (16-bit types) of itself, the
    exponential by one unit (2 U) and by its argument's three roundings, 3 U x^2/2, and below 2^-126 it is 0: R <= 1/2 and
    phi's factor 0.4 make that |x| 2^-126 of the value and (1 + |x|) 2^-126 of the slope at most.
    The sigmoid forms: e = 2^(-z log2 e) has an argument off by 8 U |z| (roundings of z and of the product), the exponential,
    the sum and the reciprocal 6 U: s is off by s (1 - s) of the first and by 6 U of itself.
    Products and sums that follow: 4 U of their terms."""
    a = x.abs()
    if kind == "gelu":
        fit = 4.2e-7 if dtype == torch.float32 else 1.2e-5
        tail = 0.5 * torch.special.erfc(a / math.sqrt(2.0))
        pdf = torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
        arg = 1.5 * U * x * x + 4 * U
        return (a * tail * (fit + arg) + 4 * U * (a * tail + act(x, kind)[0].abs()) + a * 2.0 ** -126,
                tail * (fit + arg) + a * pdf * (arg + 4 * U) + 4 * U + (1 + a) * 2.0 ** -126)
    z = 2.0 * math.sqrt(2.0 / math.pi) * (x + 0.044715 * x ** 3) if kind == "gelu_tanh" else x
    dz = 2.0 * math.sqrt(2.0 / math.pi) * (1 + 3 * 0.044715 * x ** 2) if kind == "gelu_tanh" else torch.ones_like(x)
    s, o = torch.sigmoid(z), torch.sigmoid(-z)
    rel = 8 * U * z.abs() * o + 6 * U                                # of s
    rel_o = 8 * U * z.abs() + 12 * U                                 # of 1 - s = e s
    value = a * s * (rel + 4 * U) + 1e-35                            # what the lowest s, 2^-126, leaves
    term = a * o * dz
    return value, s * (1 + term) * (rel + 4 * U) + s * term * (rel_o + 6 * U) + 1e-35


# ---------------------------------------------------------------- layer norm
def norm(x, kept, dy, w, b, eps):
    """y, mean, rstd, dx, dw, db in 64 bits: statistics of ``x``, the backward pass from ``kept``."""
    mu = x.mean(dim=1, keepdim=True)
    r = 1.0 / torch.sqrt(((x - mu) ** 2).mean(dim=1, keepdim=True) + eps)
    y = (x - mu) * r * w + b
    h = (kept - mu) * r
    u = dy * w
    dx = r * (u - u.mean(dim=1, keepdim=True) - h * (u * h).mean(dim=1, keepdim=True))
    return y, mu[:, 0], r[:, 0], dx, (dy * h).sum(0), dy.sum(0)


def norm_error(x, kept, dy, w, b, eps):
    """Bounds on what fp32 leaves of them.  A row's sums have at most 16 terms in a lane and 4 + 2 + 16 joins, or 24 and 5:
    k = 40 with the factor 1 / cols.  The parameters' sums: one rounding a row at most, and 80 for the joins."""
    k = 40
    mu = x.mean(dim=1, keepdim=True)
    d = x - mu
    var = (d ** 2).mean(dim=1, keepdim=True)
    r = 1.0 / torch.sqrt(var + eps)
    e_mu = k * U * x.abs().mean(dim=1, keepdim=True)
    # d is off by e_mu + U |d|, the mean of squares by 2 |d| of that and k roundings, the root halves it
    e_var = 2 * (d.abs() * (e_mu + U * d.abs())).mean(dim=1, keepdim=True) + e_mu ** 2 + k * U * var
    rho = 0.5 * e_var * r * r + 4 * U

    def h_of(v):
        h = (v - mu) * r
        return h, h.abs() * (rho + 3 * U) + r * e_mu

    h, e_h = h_of(x)
    y = h * w + b
    e_y = w.abs() * e_h + 2 * U * ((h * w).abs() + y.abs())
    h, e_h = h_of(kept)
    u = dy * w
    s1, s2 = u.mean(dim=1, keepdim=True), (u * h).mean(dim=1, keepdim=True)
    e1 = k * U * u.abs().mean(dim=1, keepdim=True)
    e2 = (u.abs() * e_h).mean(dim=1, keepdim=True) + (k + 2) * U * (u * h).abs().mean(dim=1, keepdim=True)
    inner = u - s1 - h * s2
    e_dx = r * (3 * U * (u.abs() + s1.abs() + (h * s2).abs()) + e1 + h.abs() * e2 + e_h * (s2.abs() + e2)) + inner.abs() * r * (rho + 2 * U)
    n = x.shape[0] + 80
    e_dw = (dy.abs() * e_h).sum(0) + n * U * (dy * h).abs().sum(0)
    e_db = n * U * dy.abs().sum(0)
    return e_y, e_mu[:, 0], r[:, 0] * rho[:, 0], e_dx, e_dw, e_db


# ---------------------------------------------------------------- weight gradient
def weight_grad(dy, kept):
    return dy.t() @ kept, dy.sum(0)


def weight_grad_error(dy, kept):
    """Exact products, summed in fp32 in any order: one rounding a term."""
    n = dy.shape[0] + 8
    return n * U * (dy.abs().t() @ kept.abs()), n * U * dy.abs().sum(0)


def check(got, want, error, dtype, what):
    """|got - want| within the fp32 error and the rounding to ``dtype``."""
    got = got.detach().cpu().double()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)}, not {tuple(want.shape)}"
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN in other places"
    allowed = error + half_step(want.abs() + error, dtype)
    over = ((got - want).abs() - allowed)[~nan]
    assert over.numel() == 0 or float(over.max()) <= 0, \
        f"{what}: off by {float((got - want).abs()[~nan].max()):.3g}, {float(over.max()):.3g} more than allowed"
