"""8-bit activation checkpoints and the backward passes that read them, for torch (``include/cswap_hip.h``, "q8").

The reference compresses an activation to move it to the host and back (CSWAP+/Execution.h:70-127).
An activation that stays on the device can be held in one byte a value instead and be read in that
form by its layer's backward pass:

    held = q8_compress(x)                         # Checkpoint8: 1.03 bytes a value
    x    = q8_decompress(held)
    y, held = q8_act(x, "gelu");                    dx = q8_act_backward(dy, held, "gelu")
    y, mean, rstd, held = layer_norm(x, w, b);      dx, dw, db = layer_norm_backward(dy, held, mean, rstd, w)
    dw, db = q8_weight_grad(dy, held)             # of y = x @ w.T + b, held made from x

Tensors are float32, bfloat16 or float16 in device memory, ``[..., features]``: the last dimension is
contiguous and the dimensions before it have one distance between rows.  Every function launches on the
current stream of the tensor's device and returns without synchronising.  ``cswap_amd.layers8`` has them
as layers with gradients, ``cswap_amd.hooks.hold_saved_tensors`` for whatever a model saves.
"""
from __future__ import annotations

import contextlib
import math

import torch

from ._lib import check, lib
from .api import _stream

GROUP = 32
KINDS = {"gelu": 0, "gelu_tanh": 1, "silu": 2}
_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_NO_GUARD = contextlib.nullcontext()


class Checkpoint8:
    """An activation in 8 bits: ``codes`` (int8, rows x pitch) and ``scales`` (uint8, rows x groups), and the
    ``shape`` and ``dtype`` of what it was made from.  ``rows`` is the product of the leading dimensions and
    ``cols`` the last one, or 1 and all of it if it was made with ``flat=True``."""
    __slots__ = ("codes", "scales", "shape", "dtype", "rows", "cols")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape, dtype: torch.dtype):
        shape = tuple(shape)
        rows, cols = _rows_cols(shape)
        if codes.dim() != 2 or scales.dim() != 2 or codes.dtype != torch.int8 or scales.dtype != torch.uint8:
            raise ValueError("expected codes as a 2-D int8 tensor and scales as a 2-D uint8 tensor")
        if codes.shape[0] != rows and codes.shape[0] == 1:
            rows, cols = 1, rows * cols
        groups = -(-cols // GROUP)
        if codes.shape != (rows, groups * GROUP) or scales.shape != (rows, groups):
            raise ValueError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not hold a tensor of shape {shape}")
        if not (codes.is_contiguous() and scales.is_contiguous() and codes.device == scales.device):
            raise ValueError("codes and scales are contiguous and on one device")
        if dtype not in _DTYPE:
            raise TypeError(f"checkpoints are made of float32, bfloat16 and float16 tensors, not {dtype}")
        self.codes, self.scales, self.shape, self.dtype, self.rows, self.cols = codes, scales, shape, dtype, rows, cols

    @property
    def device(self):
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def __repr__(self):
        return f"Checkpoint8(shape={self.shape}, dtype={self.dtype}, {self.nbytes} bytes)"


# ------------------------------------------------------------------- what the calls have in common
def _rows_cols(shape):
    if len(shape) == 0:
        return 1, 1
    return math.prod(shape[:-1]), shape[-1]


def _on(device: torch.device):
    """The device's current stream is the one to launch on, whichever device is current."""
    if device.index is None or device.index == torch.cuda.current_device():
        return _NO_GUARD
    return torch.cuda.device(device)


def _need(t: torch.Tensor, what: str) -> int:
    kind = _DTYPE.get(t.dtype)
    if kind is None:
        raise TypeError(f"{what}: float32, bfloat16 or float16, not {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{what}: expected a tensor in device memory")
    return kind


def _row_stride(t: torch.Tensor, what: str) -> int:
    """The distance between rows, in elements; 0 (the library's default) where there are no gaps."""
    if t.is_contiguous():
        return 0
    shape, stride = t.shape, t.stride()
    if shape[-1] > 1 and stride[-1] != 1:
        raise ValueError(f"{what}: the last dimension has to be contiguous")
    outer = [(n, s) for n, s in zip(shape[:-1], stride[:-1]) if n != 1]
    if not outer or t.numel() == 0:
        return 0
    for (_, a), (n, b) in zip(outer, outer[1:]):
        if a != n * b:
            raise ValueError(f"{what}: the dimensions before the last have no one distance between rows")
    if outer[-1][1] < shape[-1]:
        raise ValueError(f"{what}: rows overlap")
    return outer[-1][1]


def _same(t: torch.Tensor, like, what: str) -> None:
    if t.device != like.device:
        raise ValueError(f"{what}: on {t.device}, not on {like.device}")


def _params(p, cols: int, like: torch.Tensor, what: str):
    if p is None:
        return 0, None
    kind = _need(p, what)
    _same(p, like, what)
    if p.numel() != cols or not p.is_contiguous():
        raise ValueError(f"{what}: expected {cols} contiguous values")
    return p.data_ptr(), kind


def _empty_checkpoint(x: torch.Tensor, flat: bool = False) -> Checkpoint8:
    rows, cols = _rows_cols(x.shape)
    if flat:
        rows, cols = 1, rows * cols
    groups = -(-cols // GROUP)
    codes = torch.empty((rows, groups * GROUP), dtype=torch.int8, device=x.device)
    scales = torch.empty((rows, groups), dtype=torch.uint8, device=x.device)
    return Checkpoint8(codes, scales, x.shape, x.dtype)


# ------------------------------------------------------------------- codec
def q8_compress(x: torch.Tensor, flat: bool = False) -> Checkpoint8:
    """The checkpoint of ``x``.  ``flat`` (contiguous tensors): groups run through the whole tensor instead of
    starting at each row, which saves the padding of short rows; a tensor whose last dimension is a multiple of 32
    is the same either way, and only such a flat checkpoint has rows for ``q8_weight_grad``."""
    kind = _need(x, "q8_compress")
    stride = _row_stride(x, "q8_compress")
    if x.numel() == 0 and (x.dim() == 0 or x.shape[-1] == 0):
        raise ValueError("q8_compress: rows without values")
    if flat and not x.is_contiguous():
        raise ValueError("q8_compress: flat checkpoints are made of contiguous tensors")
    if flat and x.numel() == 0:
        flat = False
    held = _empty_checkpoint(x, flat and x.shape[-1:].numel() % GROUP != 0)
    with _on(x.device):
        check(lib().cswap_q8_pack(x.data_ptr(), kind, held.rows, held.cols, stride, held.codes.data_ptr(),
                                  held.scales.data_ptr(), _stream()), "cswap_q8_pack")
    return held


def q8_decompress(held: Checkpoint8, out: torch.Tensor | None = None, dtype: torch.dtype | None = None) -> torch.Tensor:
    """What ``held`` stands for, in its own type or in ``dtype`` (rounded once where that does not hold it)."""
    if not held.codes.is_cuda:
        raise ValueError("q8_decompress: expected a checkpoint in device memory")
    if out is None:
        out = torch.empty(held.shape, dtype=dtype or held.dtype, device=held.device)
    elif tuple(out.shape) != held.shape or (dtype is not None and out.dtype != dtype):
        raise ValueError(f"q8_decompress: out is {tuple(out.shape)} {out.dtype}")
    kind = _need(out, "q8_decompress")
    _same(out, held, "q8_decompress: out")
    stride = _row_stride(out, "q8_decompress")
    if stride and held.rows == 1 and out.numel() != out.shape[-1]:
        raise ValueError("q8_decompress: a flat checkpoint goes into a contiguous tensor")
    with _on(held.device):
        check(lib().cswap_q8_unpack(held.codes.data_ptr(), held.scales.data_ptr(), held.rows, held.cols, out.data_ptr(),
                                    kind, stride, _stream()), "cswap_q8_unpack")
    return out


# ------------------------------------------------------------------- activation functions
def _kind_of(kind: str) -> int:
    if kind not in KINDS:
        raise ValueError(f"activation function {kind!r}: one of {', '.join(KINDS)}")
    return KINDS[kind]


def q8_act(x: torch.Tensor, kind: str = "gelu"):
    """``(f(x), checkpoint of x)`` in one pass; ``kind``: "gelu", "gelu_tanh" or "silu"."""
    k, dtype = _kind_of(kind), _need(x, "q8_act")
    stride = _row_stride(x, "q8_act")
    rows, cols = _rows_cols(x.shape)
    if cols == 0:
        raise ValueError("q8_act: rows without values")
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    held = _empty_checkpoint(x)
    with _on(x.device):
        check(lib().cswap_q8_act_forward(k, x.data_ptr(), dtype, rows, cols, stride, y.data_ptr(), 0, held.codes.data_ptr(),
                                         held.scales.data_ptr(), _stream()), "cswap_q8_act_forward")
    return y, held


def _need_gradient(dy: torch.Tensor, held, what: str):
    """dy's type and row stride; it goes with an input of held's shape and type."""
    kind = _need(dy, f"{what}: dy")
    _same(dy, held, f"{what}: dy")
    if tuple(dy.shape) != tuple(held.shape) or dy.dtype != held.dtype:
        raise ValueError(f"{what}: dy is {tuple(dy.shape)} {dy.dtype}, the input was {tuple(held.shape)} {held.dtype}")
    return kind, _row_stride(dy, f"{what}: dy")


def _need_rows(held: Checkpoint8, what: str):
    """rows and cols of a checkpoint by its shape: a flat one has them where its rows are whole groups."""
    rows, cols = _rows_cols(held.shape)
    if held.rows != rows and cols % GROUP:
        raise ValueError(f"{what}: a flat checkpoint of rows of {cols} values has no rows of its own")
    return rows, cols


def q8_act_backward(dy: torch.Tensor, held: Checkpoint8, kind: str = "gelu") -> torch.Tensor:
    """``dy * f'(x)``, x as ``held`` has it."""
    k = _kind_of(kind)
    dtype, stride = _need_gradient(dy, held, "q8_act_backward")
    rows, cols = _need_rows(held, "q8_act_backward")
    dx = torch.empty(dy.shape, dtype=dy.dtype, device=dy.device)
    with _on(dy.device):
        check(lib().cswap_q8_act_backward(k, dy.data_ptr(), dtype, rows, cols, stride, held.codes.data_ptr(),
                                          held.scales.data_ptr(), dx.data_ptr(), 0, _stream()), "cswap_q8_act_backward")
    return dx


# ------------------------------------------------------------------- layer norm
def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5,
               checkpoint: bool = True):
    """``(y, mean, rstd, held)``: layer norm over the last dimension, the rows' statistics in fp32, and what the
    backward pass reads: the checkpoint of ``x``, or ``x`` itself with ``checkpoint=False``."""
    dtype = _need(x, "layer_norm")
    stride = _row_stride(x, "layer_norm")
    rows, cols = _rows_cols(x.shape)
    if cols == 0 or x.dim() == 0:
        raise ValueError("layer_norm: rows without values")
    w, wk = _params(weight, cols, x, "layer_norm: weight")
    b, bk = _params(bias, cols, x, "layer_norm: bias")
    if wk is not None and bk is not None and wk != bk:
        raise TypeError("layer_norm: weight and bias have one type")
    pk = wk if wk is not None else bk if bk is not None else 0
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty((2, rows), dtype=torch.float32, device=x.device)
    held = _empty_checkpoint(x) if checkpoint else x
    codes, scales = (held.codes.data_ptr(), held.scales.data_ptr()) if checkpoint else (0, 0)
    at = stats.data_ptr()
    with _on(x.device):
        check(lib().cswap_layer_norm_forward(x.data_ptr(), dtype, rows, cols, stride, w, b, pk, eps, y.data_ptr(), 0, at,
                                             at + 4 * rows, codes, scales, _stream()), "cswap_layer_norm_forward")
    return y, stats[0], stats[1], held


def layer_norm_backward(dy: torch.Tensor, held, mean: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor | None = None,
                        param_dtype: torch.dtype | None = None):
    """``(dx, dweight, dbias)``; ``held`` is what ``layer_norm`` returned last.  The parameters' gradients come in
    ``param_dtype`` (the weight's type, else dy's)."""
    dtype, stride = _need_gradient(dy, held, "layer_norm_backward")
    if isinstance(held, Checkpoint8):
        rows, cols = _need_rows(held, "layer_norm_backward")
        x, x_stride, codes, scales = 0, 0, held.codes.data_ptr(), held.scales.data_ptr()
    else:
        rows, cols = _rows_cols(held.shape)
        x, x_stride, codes, scales = held.data_ptr(), _row_stride(held, "layer_norm_backward: x"), 0, 0
    for s in (mean, rstd):
        if s.dtype != torch.float32 or s.numel() != rows or not s.is_contiguous() or s.device != dy.device:
            raise ValueError(f"layer_norm_backward: mean and rstd are {rows} contiguous fp32 values on {dy.device}")
    w, wk = _params(weight, cols, dy, "layer_norm_backward: weight")
    param_dtype = param_dtype or (weight.dtype if weight is not None else dy.dtype)
    if param_dtype not in _DTYPE or (weight is not None and param_dtype != weight.dtype):
        raise TypeError(f"layer_norm_backward: param_dtype {param_dtype}")
    dx = torch.empty(dy.shape, dtype=dy.dtype, device=dy.device)
    grads = torch.empty((2, cols), dtype=param_dtype, device=dy.device)
    room = lib().cswap_layer_norm_workspace_bytes(rows, cols)
    ws = torch.empty(room, dtype=torch.uint8, device=dy.device)
    at = grads.data_ptr()
    with _on(dy.device):
        check(lib().cswap_layer_norm_backward(dy.data_ptr(), dtype, rows, cols, stride, x, x_stride, codes, scales,
                                              mean.data_ptr(), rstd.data_ptr(), w, _DTYPE[param_dtype], dx.data_ptr(), 0, at,
                                              at + cols * grads.element_size(), ws.data_ptr(), room, _stream()),
              "cswap_layer_norm_backward")
    return dx, grads[0], grads[1]


# ------------------------------------------------------------------- weight gradient
def q8_weight_grad(dy: torch.Tensor, held: Checkpoint8, bias: bool = True, out_dtype: torch.dtype | None = None):
    """``(dW, db)`` of ``y = x @ W.T + b`` from ``dy`` and the checkpoint of ``x``: ``dy.T @ x`` and ``dy.sum(0)`` over
    all rows, in ``out_dtype`` (dy's type); ``db`` is None without ``bias``."""
    kind = _need(dy, "q8_weight_grad: dy")
    _same(dy, held, "q8_weight_grad: dy")
    rows, k = _need_rows(held, "q8_weight_grad")
    if dy.dim() == 0 or tuple(dy.shape[:-1]) != held.shape[:-1]:
        raise ValueError(f"q8_weight_grad: dy is {tuple(dy.shape)}, the input was {held.shape}")
    if dy.dtype == torch.float16 and held.dtype != torch.float16:
        raise TypeError("q8_weight_grad: a float16 dy goes with the checkpoint of a float16 input")
    stride = _row_stride(dy, "q8_weight_grad: dy")
    n = dy.shape[-1]
    out_dtype = out_dtype or dy.dtype
    if out_dtype not in _DTYPE:
        raise TypeError(f"q8_weight_grad: out_dtype {out_dtype}")
    dw = torch.empty((n, k), dtype=out_dtype, device=dy.device)
    db = torch.empty(n, dtype=out_dtype, device=dy.device) if bias else None
    room = lib().cswap_q8_weight_grad_workspace_bytes(kind, rows, n, k)
    ws = torch.empty(room, dtype=torch.uint8, device=dy.device)
    with _on(dy.device):
        check(lib().cswap_q8_weight_grad(dy.data_ptr(), kind, rows, n, stride, held.codes.data_ptr(), held.scales.data_ptr(),
                                         k, dw.data_ptr(), db.data_ptr() if bias else 0, _DTYPE[out_dtype], ws.data_ptr(),
                                         room, _stream()), "cswap_q8_weight_grad")
    return dw, db
