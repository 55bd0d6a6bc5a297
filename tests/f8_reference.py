"""Blocks of 128 in 8-bit floating point, and linear layers' products of them, in 64 bits; on the CPU, without the package."""
import torch

BLOCK = 128
U = 2.0 ** -24


def power(e):
    return torch.ldexp(torch.ones((), dtype=torch.float64), e.to(torch.int32))


def held(x, rows):
    """What blocks of `rows` x 128 values stand for, and their scale bytes: e4m3 by its definition (four significant bits, 2^-9 the least step)."""
    x = x.double()
    n, k = x.shape
    full = torch.nn.functional.pad(x, (0, -k % BLOCK, 0, -n % rows)).view(-(-n // rows), rows, -(-k // BLOCK), BLOCK)
    finite = torch.isfinite(full).all(dim=3, keepdim=True).all(dim=1, keepdim=True)
    top = torch.where(finite, full.abs(), 0.0).amax(dim=(1, 3), keepdim=True)
    mantissa, exponent = torch.frexp(top / 448)                               # top / 448 = m 2^e, 1/2 <= m < 1
    s = torch.where(top == 0, -126, torch.where(mantissa == 0.5, exponent - 1, exponent).clamp(min=-126))
    y = torch.where(finite, full, 0.0) / power(s)
    _, exponent = torch.frexp(y)
    step = power((exponent - 4).clamp(min=-9))
    value = torch.where(finite, torch.round(y / step) * step * power(s), torch.nan)      # torch rounds to even
    scales = torch.where(finite, s + 127, 127)[:, 0, :, 0].to(torch.uint8)
    return value.view(-(-n // rows) * rows, -1)[:n, :k].contiguous(), scales


def linear(x, w, bias, turned=False):
    """x @ w.T + bias of held x and w (turned: x @ w), and bounds on the error of results in 16 bits and in fp32.

    fp32: exact products, one rounding a term.  16 bits: an instruction cuts each of its 64 (few rows: 128) products below 2^-13 of its largest, which is at
    most the product of the blocks' largest values: 128 * 2^-13 of that for a block; sums with what was there before are fp32."""
    xh = held(x, 1)[0]
    wh = held(w, BLOCK)[0]
    wh = wh.t().contiguous() if turned else wh
    y = xh @ wh.t()
    size = xh.nan_to_num().abs() @ wh.nan_to_num().abs().t()
    ax, aw = (torch.nn.functional.pad(t.nan_to_num().abs(), (0, -t.shape[1] % BLOCK)).unflatten(1, (-1, BLOCK)).amax(dim=2) for t in (xh, wh))
    exact = (x.shape[1] + 16) * U * size
    cut = 128 * 2.0 ** -13 * (ax @ aw.t()) + exact
    if bias is not None:
        y = y + bias.double()
        exact, cut = (e + 2 * U * y.nan_to_num().abs() for e in (exact, cut))
    return y, cut, exact
