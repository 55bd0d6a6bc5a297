"""8-bit activation checkpoints and the backward passes that read them, for torch (``include/cswap_hip.h``, "q8").

The reference compresses an activation to move it to the host and back (CSWAP+/Execution.h:70-127).
An activation that stays on the device can be held in one byte a value instead and be read in that
form by its layer's backward pass:

    held = q8_compress(x)                         # Checkpoint8: 1.03 bytes a value
    x    = q8_decompress(held)
    y, held = q8_act(x, "gelu");                    dx = q8_act_backward(dy, held, "gelu")
    y, mean, rstd, held = layer_norm(x, w, b);      dx, dw, db = layer_norm_backward(dy, held, mean, rstd, w)
    y, mean, rstd, held = group_norm(x, 32, w, b, act="silu")          # x: images, channels last
    dx, dw, db = group_norm_backward(dy, held, mean, rstd, 32, w, b, act="silu")
    dw, db = q8_weight_grad(dy, held)             # of y = x @ w.T + b, held made from x

Tensors are float32, bfloat16 or float16 in device memory, ``[..., features]``: the last dimension is
contiguous and the dimensions before it have one distance between rows (images of a group norm: ``[N, C, ...]`` that lie so in memory
with C last, as ``torch.channels_last`` has them).  Every function launches on the
current stream of the tensor's device and returns without synchronising.  Torch sees the outputs but not what makes
them: functions here refuse to be traced, and tensors with forward-mode derivatives.  ``cswap_amd.layers8`` has them
as layers with gradients, ``cswap_amd.hooks.hold_saved_tensors`` for whatever a model saves.
"""
from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from . import api
from ._lib import check, lib

GROUP = 32
MAX_VALUES = ((1 << 31) // 4 - 1) * GROUP   # of a flat checkpoint: 2^31 - 1 pieces of 8, in whole groups
MAX_FEATURES = 1 << 20                      # on either side of a weight gradient
MAX_NORM = 16384                            # values of a layer norm's row
MAX_CHANNELS, MAX_GROUPS = 4096, 2048       # of a group norm
KINDS = {"gelu": 0, "gelu_tanh": 1, "silu": 2}
_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_HOLD = 2    # keep_sign of the saved-tensor hooks: few signs, and minus infinity, which only _give_back knows


class Checkpoint8:
    """An activation in 8 bits: ``codes`` (int8, rows x pitch) and ``scales`` (uint8, rows x groups), and the
    ``shape`` and ``dtype`` of what it was made from.  ``rows`` is the product of the leading dimensions and
    ``cols`` the last one, or 1 and all of it if it was made with ``flat=True``."""
    __slots__ = ("shape", "dtype", "device", "rows", "cols", "_codes", "_scales", "_room", "_at", "_scales_at")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape, dtype: torch.dtype):
        rows, cols = _rows_cols(shape)
        if codes.dtype is not torch.int8 or scales.dtype is not torch.uint8 or codes.dim() != 2 or scales.dim() != 2:
            raise ValueError("expected codes as a 2-D int8 tensor and scales as a 2-D uint8 tensor")
        held, pitch = codes.shape
        if held != rows and held == 1:
            rows, cols = 1, rows * cols
        groups = -(-cols // GROUP)
        if held != rows or pitch != groups * GROUP or scales.shape != (rows, groups):
            raise ValueError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not hold a tensor of shape "
                             f"{tuple(shape)}")
        if not (codes.is_contiguous() and scales.is_contiguous() and codes.device == scales.device):
            raise ValueError("codes and scales are contiguous and on one device")
        if dtype not in _DTYPE:
            raise TypeError(f"checkpoints are made of float32, bfloat16 and float16 tensors, not {dtype}")
        self.shape, self.dtype, self.device, self.rows, self.cols = torch.Size(shape), dtype, codes.device, rows, cols
        self._codes, self._scales, self._room = codes, scales, None
        self._at, self._scales_at = codes.data_ptr(), scales.data_ptr()

    @classmethod
    def _over(cls, room: torch.Tensor, shape, dtype: torch.dtype, rows: int, cols: int) -> "Checkpoint8":
        """The checkpoint in ``room``: codes, and scales behind them; the tensors over either are made when they are
        asked for."""
        self = cls.__new__(cls)
        self.shape, self.dtype, self.device, self.rows, self.cols = torch.Size(shape), dtype, room.device, rows, cols
        self._codes = self._scales = None
        self._room = room
        self._at = at = room.data_ptr()
        self._scales_at = at + rows * -(-cols // GROUP) * GROUP
        return self

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            pitch = -(-self.cols // GROUP) * GROUP
            self._codes = self._room[:self.rows * pitch].view(self.rows, pitch)
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            groups = -(-self.cols // GROUP)
            self._scales = self._room[self.rows * groups * GROUP:].view(torch.uint8).view(self.rows, groups)
        return self._scales

    @property
    def nbytes(self) -> int:
        return self.rows * -(-self.cols // GROUP) * (GROUP + 1)

    def record_stream(self, stream) -> None:
        """As ``torch.Tensor.record_stream``: the arrays are used on ``stream``, too."""
        for t in (self._room, self._codes, self._scales):
            if t is not None:
                t.record_stream(stream)

    def __repr__(self):
        return f"Checkpoint8(shape={tuple(self.shape)}, dtype={self.dtype}, {self.nbytes} bytes)"


# ------------------------------------------------------------------- what the calls have in common
def _rows_cols(shape):
    n = len(shape)
    if n == 2:
        return shape
    return (math.prod(shape[:-1]), shape[-1]) if n else (1, 1)


# torch's own short cut to the current device's number, as api has one to the stream's handle
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_is_tracing = getattr(torch._C, "_is_tracing", torch.jit.is_tracing)
_modes = getattr(torch._C, "_len_torch_dispatch_stack", lambda: 0)


def _traced() -> bool:
    return _is_tracing() or torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None


def _have_tangents(*tensors) -> bool:
    return forward_ad._current_level >= 0 and any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None
                                                  for t in tensors)


def _refuse_what_torch_would_lose(what: str, *tensors) -> None:
    """Called where something watches: a trace records the outputs' allocation alone and would give back memory as it
    was, and outputs have no tangent."""
    if _traced():
        raise RuntimeError(f"{what}: cannot be traced")
    if _have_tangents(*tensors):
        raise RuntimeError(f"{what}: no forward-mode derivatives")


def _watched() -> bool:
    """Something sees more of a tensor than its values: forward-mode differentiation, a trace, a dispatch mode."""
    return forward_ad._current_level >= 0 or _is_tracing() or _modes() > 0


def _begin(t: torch.Tensor, what: str, *others):
    """Type and device of a tensor in device memory, and the stream to launch on: the current one of its device, if that
    is the current device, else None. The call is then made again with its device current."""
    if forward_ad._current_level >= 0 or _is_tracing() or _modes():     # _watched, without the call: it is on every path
        _refuse_what_torch_would_lose(what, t, *others)
    kind = _DTYPE.get(t.dtype)
    if kind is None:
        raise TypeError(f"{what}: float32, bfloat16 or float16, not {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{what}: expected a tensor in device memory")
    device = t.device
    return kind, device, _stream_of(device)


def _stream_of(device: torch.device):
    index = device.index
    if index != _current_device():
        return None
    return api._raw_stream(index) if api._raw_stream is not None else api._stream()


def _row_stride(t: torch.Tensor, what: str) -> int:
    """The distance between rows, in elements; 0 (the library's default) where there are no gaps."""
    if t.is_contiguous():
        return 0
    if t.is_neg():
        raise ValueError(f"{what}: a view with its sign turned (resolve_neg)")
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


def _empty_checkpoint(x: torch.Tensor, rows: int, cols: int, device: torch.device) -> Checkpoint8:
    """Room for the checkpoint of x, in one allocation (``Checkpoint8._over``, without the call: it is on every path)."""
    codes = rows * -(-cols // GROUP) * GROUP
    held = _new_checkpoint(Checkpoint8)
    held._room = room = torch.empty(codes + codes // GROUP, dtype=torch.int8, device=device)
    held._at = at = room.data_ptr()
    held._scales_at = at + codes
    held._codes = held._scales = None
    held.shape, held.dtype, held.device, held.rows, held.cols = x.shape, x.dtype, device, rows, cols
    return held


_new_checkpoint = object.__new__


def _like(t: torch.Tensor, stride: int) -> torch.Tensor:
    """A contiguous tensor of t's shape and type."""
    return torch.empty_like(t) if stride == 0 else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _param(p, cols: int, device: torch.device, what: str):
    """Address and type of a parameter (0 and None: there is none)."""
    if p is None:
        return 0, None
    kind = _DTYPE.get(p.dtype)
    if kind is None or p.device != device:
        raise TypeError(f"{what}: a float32, bfloat16 or float16 tensor on {device}, not {p.dtype} on {p.device}")
    if p.numel() != cols or not p.is_contiguous():
        raise ValueError(f"{what}: expected {cols} contiguous values")
    return p.data_ptr(), kind


# ------------------------------------------------------------------- codec
def q8_compress(x: torch.Tensor, flat: bool = False, keep_sign: bool = False) -> Checkpoint8:
    """The checkpoint of ``x``.  ``flat`` (contiguous tensors): groups run through the whole tensor instead of
    starting at each row, which saves the padding of short rows; a tensor whose last dimension is a multiple of 32
    is the same either way, and only such a flat checkpoint has rows for the backward passes.  ``keep_sign``: what is
    not 0 but rounds to 0 is held as the smallest value with its sign, off by up to 2^-6 of the group's largest magnitude."""
    kind, device, stream = _begin(x, "q8_compress")
    if stream is None:
        with torch.cuda.device(device):
            return q8_compress(x, flat, keep_sign)
    stride = 0 if x.is_contiguous() else _row_stride(x, "q8_compress")
    rows, cols = _rows_cols(x.shape)
    if cols == 0:
        raise ValueError("q8_compress: rows without values")
    if flat and stride:
        raise ValueError("q8_compress: flat checkpoints are made of contiguous tensors")
    if flat and rows and cols % GROUP:
        rows, cols = 1, rows * cols
    held = _empty_checkpoint(x, rows, cols, device)
    check(lib().cswap_q8_pack(x.data_ptr(), kind, rows, cols, stride, keep_sign, held._at, held._scales_at, stream),
          "cswap_q8_pack")
    return held


def q8_decompress(held: Checkpoint8, out: torch.Tensor | None = None, dtype: torch.dtype | None = None) -> torch.Tensor:
    """What ``held`` stands for, in its own type or in ``dtype`` (rounded once where that does not hold it)."""
    device = held.device
    if _watched():
        _refuse_what_torch_would_lose("q8_decompress", out)
    if device.type != "cuda":
        raise ValueError("q8_decompress: expected a checkpoint in device memory")
    stream = _stream_of(device)
    if stream is None:
        with torch.cuda.device(device):
            return q8_decompress(held, out, dtype)
    if out is None:
        dtype = dtype or held.dtype
        out = torch.empty(held.shape, dtype=dtype, device=device)
        kind, stride = _DTYPE.get(dtype), 0
        if kind is None:
            raise TypeError(f"q8_decompress: float32, bfloat16 or float16, not {dtype}")
    else:
        if out.shape != held.shape or (dtype is not None and out.dtype != dtype):
            raise ValueError(f"q8_decompress: out is {tuple(out.shape)} {out.dtype}")
        if out.device != device:
            raise ValueError(f"q8_decompress: out on {out.device}, not on {device}")
        kind, stride = _begin(out, "q8_decompress: out")[0], _row_stride(out, "q8_decompress")
        if stride and held.rows != _rows_cols(held.shape)[0]:
            raise ValueError("q8_decompress: a flat checkpoint goes into a contiguous tensor")
    check(lib().cswap_q8_unpack(held._at, held._scales_at, held.rows, held.cols, out.data_ptr(), kind,
                                stride, stream), "cswap_q8_unpack")
    return out


def _give_back(held: Checkpoint8) -> torch.Tensor:
    """The tensor that the saved-tensor hooks' checkpoint was made of, as far as that holds it."""
    stream = _stream_of(held.device)
    if stream is None:
        with torch.cuda.device(held.device):
            return _give_back(held)
    out = torch.empty(held.shape, dtype=held.dtype, device=held.device)
    check(lib().cswap_q8_unpack_held(held._at, held._scales_at, held.rows, held.cols, out.data_ptr(), _DTYPE[held.dtype], 0,
                                     stream), "cswap_q8_unpack_held")
    return out


# ------------------------------------------------------------------- activation functions
def _kind_of(kind: str) -> int:
    if kind not in KINDS:
        raise ValueError(f"activation function {kind!r}: one of {', '.join(KINDS)}")
    return KINDS[kind]


def q8_act(x: torch.Tensor, kind: str = "gelu", checkpoint: bool = True):
    """``(f(x), checkpoint of x)`` in one pass; ``kind``: "gelu", "gelu_tanh" or "silu".  The second is None with
    ``checkpoint=False``."""
    k = _kind_of(kind)
    dtype, device, stream = _begin(x, "q8_act")
    if stream is None:
        with torch.cuda.device(device):
            return q8_act(x, kind, checkpoint)
    stride = 0 if x.is_contiguous() else _row_stride(x, "q8_act")
    rows, cols = _rows_cols(x.shape)
    if cols == 0:
        raise ValueError("q8_act: rows without values")
    y = _like(x, stride)
    if checkpoint:
        held = _empty_checkpoint(x, rows, cols, device)
        codes, scales = held._at, held._scales_at
    else:
        held, codes, scales = None, 0, 0
    check(lib().cswap_q8_act_forward(k, x.data_ptr(), dtype, rows, cols, stride, y.data_ptr(), 0, codes, scales,
                                     stream), "cswap_q8_act_forward")
    return y, held


def _need_gradient(dy: torch.Tensor, held, what: str, *others):
    """``_begin`` of dy, and its row stride; it goes with an input of held's shape and type."""
    kind, device, stream = _begin(dy, what, held, *others)
    if dy.shape != held.shape or dy.dtype != held.dtype or device != held.device:
        raise ValueError(f"{what}: dy is {tuple(dy.shape)} {dy.dtype} on {dy.device}, the input was {tuple(held.shape)} "
                         f"{held.dtype} on {held.device}")
    return kind, device, stream, 0 if dy.is_contiguous() else _row_stride(dy, what)


def _need_rows(held: Checkpoint8, what: str):
    """rows and cols of a checkpoint by its shape: a flat one has them where its rows are whole groups."""
    rows, cols = _rows_cols(held.shape)
    if held.rows != rows and cols % GROUP:
        raise ValueError(f"{what}: a flat checkpoint of rows of {cols} values has no rows of its own")
    return rows, cols


def q8_act_backward(dy: torch.Tensor, held: Checkpoint8, kind: str = "gelu") -> torch.Tensor:
    """``dy * f'(x)``, x as ``held`` has it."""
    k = _kind_of(kind)
    dtype, device, stream, stride = _need_gradient(dy, held, "q8_act_backward")
    if stream is None:
        with torch.cuda.device(device):
            return q8_act_backward(dy, held, kind)
    rows, cols = _need_rows(held, "q8_act_backward")
    dx = _like(dy, stride)
    check(lib().cswap_q8_act_backward(k, dy.data_ptr(), dtype, rows, cols, stride, held._at, held._scales_at, dx.data_ptr(), 0,
                                      stream), "cswap_q8_act_backward")
    return dx


# ------------------------------------------------------------------- layer norm
def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5,
               checkpoint: bool = True):
    """``(y, mean, rstd, held)``: layer norm over the last dimension, the rows' statistics in fp32, and what the
    backward pass reads: the checkpoint of ``x``, or ``x`` itself with ``checkpoint=False``.  A checkpoint is off by up to
    2^-7 of the largest magnitude nearby, mean included: rows whose mean is many times their deviation are better kept
    as they are."""
    dtype, device, stream = _begin(x, "layer_norm", weight, bias)
    if stream is None:
        with torch.cuda.device(device):
            return layer_norm(x, weight, bias, eps, checkpoint)
    stride = 0 if x.is_contiguous() else _row_stride(x, "layer_norm")
    rows, cols = _rows_cols(x.shape)
    if cols == 0 or x.dim() == 0:
        raise ValueError("layer_norm: rows without values")
    w, wk = _param(weight, cols, device, "layer_norm: weight")
    b, bk = _param(bias, cols, device, "layer_norm: bias")
    if wk is not None and bk is not None and wk != bk:
        raise TypeError("layer_norm: weight and bias have one type")
    y = _like(x, stride)
    mean = torch.empty(rows, dtype=torch.float32, device=device)
    rstd = torch.empty_like(mean)
    if checkpoint:
        held = _empty_checkpoint(x, rows, cols, device)
        codes, scales = held._at, held._scales_at
    else:
        held, codes, scales = x, 0, 0
    check(lib().cswap_layer_norm_forward(x.data_ptr(), dtype, rows, cols, stride, w, b, wk or bk or 0, eps, y.data_ptr(), 0,
                                         mean.data_ptr(), rstd.data_ptr(), codes, scales, stream),
          "cswap_layer_norm_forward")
    return y, mean, rstd, held


def layer_norm_backward(dy: torch.Tensor, held, mean: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor | None = None,
                        param_dtype: torch.dtype | None = None):
    """``(dx, dweight, dbias)``; ``held`` is what ``layer_norm`` returned last.  The parameters' gradients come in
    ``param_dtype`` (the weight's type, else dy's)."""
    dtype, device, stream, stride = _need_gradient(dy, held, "layer_norm_backward", mean, rstd, weight)
    if stream is None:
        with torch.cuda.device(device):
            return layer_norm_backward(dy, held, mean, rstd, weight, param_dtype)
    if isinstance(held, Checkpoint8):
        rows, cols = _need_rows(held, "layer_norm_backward")
        x, x_stride, codes, scales = 0, 0, held._at, held._scales_at
    else:
        rows, cols = _rows_cols(held.shape)
        x, x_stride, codes, scales = held.data_ptr(), _row_stride(held, "layer_norm_backward: x"), 0, 0
    for s in (mean, rstd):
        if s.dtype is not torch.float32 or s.numel() != rows or not s.is_contiguous() or s.device != device:
            raise ValueError(f"layer_norm_backward: mean and rstd are {rows} contiguous fp32 values on {device}")
    w, wk = _param(weight, cols, device, "layer_norm_backward: weight")
    if wk is not None and param_dtype not in (None, weight.dtype):
        raise TypeError(f"layer_norm_backward: param_dtype {param_dtype}, the weight has {weight.dtype}")
    param_dtype = param_dtype or (dy.dtype if weight is None else weight.dtype)
    pk = _DTYPE.get(param_dtype)
    if pk is None:
        raise TypeError(f"layer_norm_backward: param_dtype {param_dtype}")
    dx = _like(dy, stride)
    dw = torch.empty(cols, dtype=param_dtype, device=device)
    db = torch.empty_like(dw)
    room = lib().cswap_layer_norm_workspace_bytes(rows, cols)
    ws = torch.empty(room, dtype=torch.uint8, device=device) if room else None
    check(lib().cswap_layer_norm_backward(dy.data_ptr(), dtype, rows, cols, stride, x, x_stride, codes, scales, mean.data_ptr(),
                                          rstd.data_ptr(), w, pk, dx.data_ptr(), 0, dw.data_ptr(), db.data_ptr(),
                                          ws.data_ptr() if room else 0, room, stream), "cswap_layer_norm_backward")
    return dx, dw, db


# ------------------------------------------------------------------- group norm
def _images(x: torch.Tensor, what: str):
    """Samples, positions and channels of ``[N, C, ...]``, and the distance between positions (0: no gaps)."""
    shape, stride, n = x.shape, x.stride(), x.dim()
    if n < 2:
        raise ValueError(f"{what}: expected [N, C, ...], not {tuple(shape)}")
    if x.is_neg():
        raise ValueError(f"{what}: a view with its sign turned (resolve_neg)")
    samples, channels = shape[0], shape[1]
    positions = math.prod(shape[2:])
    if channels == 0 or positions == 0:
        raise ValueError(f"{what}: images without values, {tuple(shape)}")
    if samples == 0:        # wherever its values would lie
        return samples, positions, channels, 0
    if channels > 1 and stride[1] != 1:
        raise ValueError(f"{what}: channels have to lie next to each other (torch.channels_last)")
    outer = [(shape[d], stride[d]) for d in (0, *range(2, n)) if shape[d] != 1]
    if not outer:
        return samples, positions, channels, 0
    for (_, a), (size, b) in zip(outer, outer[1:]):
        if a != size * b:
            raise ValueError(f"{what}: positions have no one distance (torch.channels_last)")
    step = outer[-1][1]
    if step < channels:
        raise ValueError(f"{what}: positions overlap")
    return samples, positions, channels, 0 if step == channels else step


def _like_images(t: torch.Tensor, stride: int) -> torch.Tensor:
    """A tensor of t's shape and type, channels last without gaps."""
    if stride == 0 and t.dim() == 4 and t.is_contiguous(memory_format=torch.channels_last):
        return torch.empty_like(t)
    shape = t.shape
    return torch.empty((shape[0], *shape[2:], shape[1]), dtype=t.dtype, device=t.device).movedim(-1, 1)


_NO_ACT = 3


def group_norm(x: torch.Tensor, groups: int, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5,
               act: str | None = None, checkpoint: bool = True):
    """``(y, mean, rstd, held)``: group norm of images ``[N, C, ...]`` that lie channels last, then the activation function ``act``
    ("gelu", "gelu_tanh", "silu"; None: none), in one call; the groups' statistics ``[N, groups]`` in fp32, and what the backward pass reads:
    the checkpoint of ``x`` as ``[N, ..., C]``, or ``x`` itself with ``checkpoint=False``.  Up to 4096 channels in up to 2048 groups.  What
    ``layer_norm`` says of means far from 0 holds here, too."""
    k = _NO_ACT if act is None else _kind_of(act)
    dtype, device, stream = _begin(x, "group_norm", weight, bias)
    if stream is None:
        with torch.cuda.device(device):
            return group_norm(x, groups, weight, bias, eps, act, checkpoint)
    samples, positions, channels, stride = _images(x, "group_norm")
    if groups <= 0 or channels % groups:
        raise ValueError(f"group_norm: {channels} channels in {groups} groups")
    w, wk = _param(weight, channels, device, "group_norm: weight")
    b, bk = _param(bias, channels, device, "group_norm: bias")
    if wk is not None and bk is not None and wk != bk:
        raise TypeError("group_norm: weight and bias have one type")
    y = _like_images(x, stride)
    mean = torch.empty((samples, groups), dtype=torch.float32, device=device)
    rstd = torch.empty_like(mean)
    if checkpoint:
        held = _empty_checkpoint(x, samples * positions, channels, device)
        shape = x.shape
        held.shape = torch.Size((shape[0], *shape[2:], channels))
        codes, scales = held._at, held._scales_at
    else:
        held, codes, scales = x, 0, 0
    room = lib().cswap_group_norm_workspace_bytes(samples, positions, channels, groups, 0)
    ws = torch.empty(room, dtype=torch.uint8, device=device) if room else None
    check(lib().cswap_group_norm_forward(k, x.data_ptr(), dtype, samples, positions, channels, groups, stride, w, b, wk or bk or 0, eps,
                                         y.data_ptr(), 0, mean.data_ptr(), rstd.data_ptr(), codes, scales, ws.data_ptr() if room else 0, room,
                                         stream), "cswap_group_norm_forward")
    return y, mean, rstd, held


def group_norm_backward(dy: torch.Tensor, held, mean: torch.Tensor, rstd: torch.Tensor, groups: int, weight: torch.Tensor | None = None,
                        bias: torch.Tensor | None = None, act: str | None = None, param_dtype: torch.dtype | None = None):
    """``(dx, dweight, dbias)``; ``held`` is what ``group_norm`` returned last, ``weight``, ``bias`` and ``act`` are what it was given.
    The parameters' gradients come in ``param_dtype`` (the weight's type, else the bias's, else dy's)."""
    k = _NO_ACT if act is None else _kind_of(act)
    dtype, device, stream = _begin(dy, "group_norm_backward", held, mean, rstd, weight, bias)
    if stream is None:
        with torch.cuda.device(device):
            return group_norm_backward(dy, held, mean, rstd, groups, weight, bias, act, param_dtype)
    samples, positions, channels, stride = _images(dy, "group_norm_backward")
    if groups <= 0 or channels % groups:
        raise ValueError(f"group_norm_backward: {channels} channels in {groups} groups")
    shape = dy.shape
    if isinstance(held, Checkpoint8):
        fits = held.shape == (shape[0], *shape[2:], channels)
        x, x_stride, codes, scales = 0, 0, held._at, held._scales_at
        if fits and held.rows != samples * positions and channels % GROUP:
            raise ValueError(f"group_norm_backward: a flat checkpoint of rows of {channels} values has no rows of its own")
    else:
        fits = held.shape == shape
        x, codes, scales = held.data_ptr(), 0, 0
        x_stride = _images(held, "group_norm_backward: x")[3] if fits else 0
    if not fits or held.dtype != dy.dtype or held.device != device:
        raise ValueError(f"group_norm_backward: dy is {tuple(shape)} {dy.dtype} on {device}, the input was held as {tuple(held.shape)} "
                         f"{held.dtype} on {held.device}")
    for s in (mean, rstd):
        if s.dtype is not torch.float32 or s.numel() != samples * groups or not s.is_contiguous() or s.device != device:
            raise ValueError(f"group_norm_backward: mean and rstd are {samples} x {groups} contiguous fp32 values on {device}")
    w, wk = _param(weight, channels, device, "group_norm_backward: weight")
    b, bk = _param(bias, channels, device, "group_norm_backward: bias")
    if wk is not None and bk is not None and wk != bk:
        raise TypeError("group_norm_backward: weight and bias have one type")
    given = weight if weight is not None else bias
    if given is not None and param_dtype not in (None, given.dtype):
        raise TypeError(f"group_norm_backward: param_dtype {param_dtype}, the parameters have {given.dtype}")
    param_dtype = param_dtype or (dy.dtype if given is None else given.dtype)
    pk = _DTYPE.get(param_dtype)
    if pk is None:
        raise TypeError(f"group_norm_backward: param_dtype {param_dtype}")
    dx = _like_images(dy, stride)
    dw = torch.empty(channels, dtype=param_dtype, device=device)
    db = torch.empty_like(dw)
    room = lib().cswap_group_norm_workspace_bytes(samples, positions, channels, groups, 1)
    ws = torch.empty(room, dtype=torch.uint8, device=device) if room else None
    check(lib().cswap_group_norm_backward(k, dy.data_ptr(), dtype, samples, positions, channels, groups, stride, x, x_stride, codes, scales,
                                          mean.data_ptr(), rstd.data_ptr(), w, b, pk, dx.data_ptr(), 0, dw.data_ptr(), db.data_ptr(),
                                          ws.data_ptr() if room else 0, room, stream), "cswap_group_norm_backward")
    return dx, dw, db


# ------------------------------------------------------------------- weight gradient
def q8_weight_grad(dy: torch.Tensor, held: Checkpoint8, bias: bool = True, out_dtype: torch.dtype | None = None):
    """``(dW, db)`` of ``y = x @ W.T + b`` from ``dy`` and the checkpoint of ``x``: ``dy.T @ x`` and ``dy.sum(0)`` over
    all rows, in ``out_dtype`` (dy's type); ``db`` is None without ``bias``."""
    kind, device, stream = _begin(dy, "q8_weight_grad: dy")
    if device != held.device:
        raise ValueError(f"q8_weight_grad: dy on {device}, the input's checkpoint on {held.device}")
    if stream is None:
        with torch.cuda.device(device):
            return q8_weight_grad(dy, held, bias, out_dtype)
    rows, k = _need_rows(held, "q8_weight_grad")
    shape = dy.shape
    if len(shape) == 0 or shape[:-1] != held.shape[:-1]:
        raise ValueError(f"q8_weight_grad: dy is {tuple(dy.shape)}, the input was {tuple(held.shape)}")
    if dy.dtype == torch.float16 and held.dtype != torch.float16:
        raise TypeError("q8_weight_grad: a float16 dy goes with the checkpoint of a float16 input")
    stride = 0 if dy.is_contiguous() else _row_stride(dy, "q8_weight_grad: dy")
    n = shape[-1]
    if n == 0:
        raise ValueError("q8_weight_grad: rows without values")
    out_dtype = out_dtype or dy.dtype
    out_kind = _DTYPE.get(out_dtype)
    if out_kind is None:
        raise TypeError(f"q8_weight_grad: out_dtype {out_dtype}")
    dw = torch.empty((n, k), dtype=out_dtype, device=device)
    db = torch.empty(n, dtype=out_dtype, device=device) if bias else None
    room = lib().cswap_q8_weight_grad_workspace_bytes(kind, rows, n, k)
    ws = torch.empty(room, dtype=torch.uint8, device=device) if room else None
    check(lib().cswap_q8_weight_grad(dy.data_ptr(), kind, rows, n, stride, held._at, held._scales_at, k, dw.data_ptr(),
                                     db.data_ptr() if bias else 0, out_kind, ws.data_ptr() if room else 0, room, stream),
          "cswap_q8_weight_grad")
    return dw, db
