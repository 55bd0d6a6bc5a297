"""Products of linear layers in 8-bit floating point, a power of two for each block of 128 (``include/cswap_hip.h``, "f8").

The reference's layers multiply in fp32 (CIFAR10/models/vgg.py:23-45).  Here both operands of a linear layer's product are held as e4m3 with
a scale for each 128 values of a row of activations and for each 128 x 128 weights, and meet in the matrix cores' 8-bit rate:

    held = f8_weight(w)                     # F8Weight: 1 byte a weight, 2 with what the backward pass reads
    y    = f8_linear(x, held, bias)         # x @ w.T + bias; x is held so within the call
    dx   = f8_linear_backward(dy, held)     # dy @ w

Tensors are float32, bfloat16 or float16 in device memory, ``[..., features]`` with one distance between rows, on the current stream of
their device; nothing waits.  A value is off by at most 2^-4 of itself (2^-18 of its block's largest below that).  Results in float32 are fp32
sums of exact products; results in 16 bits come from the 8-bit matrix instructions, which cut each of eight neighbouring products to a multiple of 2^-13 of the
power of two in the largest of them (as a rule 3e-5 of the products' norm in all) and add up the eights in fp32: ``out_dtype=torch.float32`` where that matters.  A NaN or an
infinity makes the results of its block's rows (of weights: columns) NaN.  The weight's gradient comes from the input's 8-bit checkpoint
(``q8.q8_weight_grad``); ``layers8.LinearF8`` has all three.
"""
from __future__ import annotations

import torch

from . import q8
from ._lib import check, lib

BLOCK = 128
MAX_FEATURES = 1 << 20


class F8Weight:
    """A weight in 8-bit floating point: ``codes`` (float8_e4m3fn, features rounded up to multiples of 128, out x in), ``scales`` (uint8, a byte
    for each 128 x 128) and, for ``f8_linear_backward``, ``turned``: the codes as in x out.  ``shape`` and ``dtype`` are the weight's."""
    __slots__ = ("shape", "dtype", "device", "codes", "scales", "turned")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape, dtype: torch.dtype, turned: torch.Tensor | None = None):
        n, k = shape
        nb, kb = -(-n // BLOCK), -(-k // BLOCK)
        if dtype not in q8._DTYPE:
            raise TypeError(f"weights are float32, bfloat16 or float16, not {dtype}")
        for what, t, want in (("codes", codes, (nb * BLOCK, kb * BLOCK)), ("turned", turned, (kb * BLOCK, nb * BLOCK))):
            if t is None and what == "turned":
                continue
            if t.dtype is not torch.float8_e4m3fn or t.shape != want or not t.is_contiguous() or t.device != codes.device or t.data_ptr() % 16:
                raise ValueError(f"expected {what} of {(n, k)} weights as contiguous {want} float8_e4m3fn, 16-byte aligned, on one device, not "
                                 f"{tuple(t.shape)} {t.dtype} on {t.device}")
        if scales.dtype is not torch.uint8 or scales.shape != (nb, kb) or not scales.is_contiguous() or scales.device != codes.device:
            raise ValueError(f"expected scales of {(n, k)} weights as contiguous {(nb, kb)} uint8, not {tuple(scales.shape)} {scales.dtype}")
        self.shape, self.dtype, self.device = torch.Size(shape), dtype, codes.device
        self.codes, self.scales, self.turned = codes, scales, turned

    def record_stream(self, stream) -> None:
        """As ``torch.Tensor.record_stream``."""
        for t in (self.codes, self.scales, self.turned):
            if t is not None:
                t.record_stream(stream)

    def __repr__(self):
        return f"F8Weight(shape={tuple(self.shape)}, dtype={self.dtype}{', turned' if self.turned is not None else ''})"


def f8_weight(w: torch.Tensor, backward: bool = True) -> F8Weight:
    """``w`` (out x in features) in 8-bit floating point; ``backward=False``: without what ``f8_linear_backward`` reads."""
    kind, device, stream = q8._begin(w, "f8_weight")
    if stream is None:
        with torch.cuda.device(device):
            return f8_weight(w, backward)
    if w.dim() != 2 or 0 in w.shape:
        raise ValueError(f"f8_weight: expected out x in features, not {tuple(w.shape)}")
    if w.is_neg():
        raise ValueError("f8_weight: a view with its sign turned (resolve_neg)")
    stride = q8._row_stride(w, "f8_weight")
    n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    codes = torch.empty((nb * BLOCK, kb * BLOCK), dtype=torch.float8_e4m3fn, device=device)
    turned = torch.empty((kb * BLOCK, nb * BLOCK), dtype=torch.float8_e4m3fn, device=device) if backward else None
    scales = torch.empty((nb, kb), dtype=torch.uint8, device=device)
    check(lib().cswap_f8_pack_weight(w.data_ptr(), kind, n, k, stride, codes.data_ptr(), turned.data_ptr() if backward else 0, scales.data_ptr(),
                                     stream), "cswap_f8_pack_weight")
    return F8Weight(codes, scales, (n, k), w.dtype, turned)


def f8_weight_values(held: F8Weight, dtype: torch.dtype | None = None) -> torch.Tensor:
    """What ``held`` stands for, in its own type or in ``dtype``."""
    n, k = held.shape
    nb, kb = held.scales.shape
    unit = (held.scales.to(torch.int32) << 23).view(torch.float32)
    values = held.codes.float().view(nb, BLOCK, kb, BLOCK) * unit[:, None, :, None]
    return values.view(nb * BLOCK, kb * BLOCK)[:n, :k].to(dtype or held.dtype).contiguous()


def _product(what: str, x: torch.Tensor, held: F8Weight, codes: torch.Tensor, k: int, n: int, turned: int, bias, out_dtype):
    kind, device, stream = q8._begin(x, what, bias)
    if device != held.device:
        raise ValueError(f"{what}: a tensor on {device}, weights on {held.device}")
    if stream is None:
        with torch.cuda.device(device):
            return _product(what, x, held, codes, k, n, turned, bias, out_dtype)
    shape = x.shape
    if len(shape) == 0 or shape[-1] != k:
        raise ValueError(f"{what}: rows of {k} values, not {tuple(shape)}")
    if x.is_neg():
        raise ValueError(f"{what}: a view with its sign turned (resolve_neg)")
    stride = 0 if x.is_contiguous() else q8._row_stride(x, what)
    rows, _ = q8._rows_cols(shape)
    b, bk = q8._param(bias, n, device, f"{what}: bias")
    out_dtype = out_dtype or x.dtype
    out_kind = q8._DTYPE.get(out_dtype)
    if out_kind is None:
        raise TypeError(f"{what}: out_dtype {out_dtype}")
    y = torch.empty((*shape[:-1], n), dtype=out_dtype, device=device)
    room = lib().cswap_f8_linear_workspace_bytes(rows, k)
    ws = torch.empty(room, dtype=torch.uint8, device=device) if room else None
    check(lib().cswap_f8_linear(x.data_ptr(), kind, rows, k, stride, codes.data_ptr(), held.scales.data_ptr(), n, turned, b, bk or 0, y.data_ptr(),
                                out_kind, 0, ws.data_ptr() if room else 0, room, stream), "cswap_f8_linear")
    return y


def f8_linear(x: torch.Tensor, held: F8Weight, bias: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x @ w.T + bias`` in ``out_dtype`` (x's type)."""
    n, k = held.shape
    return _product("f8_linear", x, held, held.codes, k, n, 0, bias, out_dtype)


def f8_linear_backward(dy: torch.Tensor, held: F8Weight, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``dy @ w`` in ``out_dtype`` (dy's type): the gradient of ``f8_linear``'s input."""
    n, k = held.shape
    if held.turned is None:
        raise ValueError("f8_linear_backward: weights made with backward=False")
    return _product("f8_linear_backward", dy, held, held.turned, n, k, 1, None, out_dtype)
