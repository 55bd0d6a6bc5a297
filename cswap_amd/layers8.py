"""Layers that keep what their backward pass needs in 8 bits (``cswap_amd.q8``), with gradients.

The reference swaps the inputs of selected layers out and back in (CSWAP+/Execution.h:70-127,
CIFAR10/models/vgg.py:23-45).  Here the input of a linear layer, a layer norm or an activation function
stays on the device in one byte a value, and the layer's backward pass reads it in that form:

    import cswap_amd.layers8 as layers8
    layers8.checkpoint_layers(model)        # nn.Linear, nn.LayerNorm, nn.GELU, nn.SiLU of a model, in place
    layers8.checkpoint_layers(model, group_norm=True)                   # and nn.GroupNorm, for images that lie channels last
    layers8.checkpoint_layers(model, f8=True)                           # linear layers whose products are in 8-bit floating point, too
    y = layers8.group_norm(x, 32, weight, bias, act="silu")            # with an activation function in the same call
    y = layers8.linear(x, weight, bias)     # or function by function

Outputs are those of the layers without checkpoints (linear layers run torch's own product, those with ``f8=True`` that of ``cswap_amd.f8``, whose
operands are held to 2^-4; norms and activation functions are computed in fp32 and rounded once, which may differ from torch's in the last place); gradients are
computed from inputs that are off by at most 2^-7 of the largest magnitude among 32 neighbours (a layer norm whose
rows have a mean of many times their deviation is better left as it is).  Without gradients to come nothing is
kept.  Layers that share an input (the projections of an attention layer) can
share its checkpoint: ``held = layers8.hold(x)``, then ``linear(x, w, b, held=held)`` for each.  Double
backward, forward-mode derivatives and traces are refused, as are tensors that ``cswap_amd.q8`` refuses.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F
from torch import nn
from torch.autograd.function import once_differentiable

from . import f8 as _f8
from . import q8
from .f8 import F8Weight
from .q8 import Checkpoint8

__all__ = ["hold", "linear", "linear_f8", "layer_norm", "group_norm", "activation", "Linear8", "LinearF8", "LayerNorm8", "GroupNorm8", "GELU8", "SiLU8", "checkpoint_layers"]


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t, or a contiguous copy where its rows have no one distance (a gradient that was expanded, a transposed view)."""
    try:
        q8._row_stride(t, "")
        return t
    except ValueError:
        return t.contiguous()


def _keep(ctx, held: Checkpoint8 | None, *others) -> None:
    """Through autograd, which lets them go when backward has used them.  Parameters come detached, as leaves: hooks that
    take a model's saved activations leave those alone, also where they are a cast or a view of a parameter."""
    if held is None:
        ctx.held = None
        ctx.save_for_backward(*others)
    else:
        room = held._room if held._room is not None else held.codes
        ctx.held = (held.shape, held.dtype, held.rows, held.cols, held._room is not None)
        ctx.save_for_backward(*others, *((room,) if held._room is not None else (room, held.scales)))


def _kept(ctx, count: int):
    """What ``_keep`` was given: ``count`` tensors and the checkpoint."""
    saved = ctx.saved_tensors
    shape, dtype, rows, cols, own = ctx.held
    held = Checkpoint8._over(saved[count], shape, dtype, rows, cols) if own else Checkpoint8(*saved[count:], shape, dtype)
    return (*saved[:count], held)


def hold(x: torch.Tensor) -> Checkpoint8:
    """The checkpoint of x for several ``linear`` layers of x."""
    return q8.q8_compress(_rows(x.detach()))


# ------------------------------------------------------------------- linear
class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, held):
        if ctx.needs_input_grad[1]:
            if max(weight.shape) > q8.MAX_FEATURES:
                raise ValueError(f"linear: up to {q8.MAX_FEATURES} features on either side, not {tuple(weight.shape)}")
            if held is None:
                held = hold(x)
            elif tuple(held.shape) != tuple(x.shape) or held.dtype != x.dtype or held.device != x.device:
                raise ValueError(f"linear: held is the checkpoint of a {tuple(held.shape)} {held.dtype} tensor on {held.device}, x is "
                                 f"{tuple(x.shape)} {x.dtype} on {x.device}")
            _keep(ctx, held, weight.detach())
        else:
            _keep(ctx, None, weight.detach())
        return F.linear(x, weight, bias)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        dx = dw = db = None
        dy = _rows(dy)
        if need_w:
            weight, held = _kept(ctx, 1)
            dw, db = q8.q8_weight_grad(dy, held, bias=need_b, out_dtype=weight.dtype)
        else:
            weight, = ctx.saved_tensors
            if need_b:
                db = dy.reshape(-1, dy.shape[-1]).sum(dim=0)
        if need_x:
            dx = dy @ weight
        return dx, dw, db, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, held: Checkpoint8 | None = None):
    """``x @ weight.T + bias``; ``held``: x's checkpoint, if there is one already.  Under autocast in its type, as
    torch's linear is (``held`` is then of x in that type)."""
    if not torch.is_grad_enabled():
        return F.linear(x, weight, bias)
    if torch.is_autocast_enabled("cuda"):
        dtype = torch.get_autocast_dtype("cuda")
        x, weight, bias = (t if t is None or t.dtype == torch.float64 else t.to(dtype) for t in (x, weight, bias))
        with torch.autocast("cuda", enabled=False):
            return _Linear.apply(x, weight, bias, held)
    return _Linear.apply(x, weight, bias, held)


def _same_weight(weight8: F8Weight, weight: torch.Tensor, turned: bool) -> None:
    if tuple(weight8.shape) != tuple(weight.shape) or weight8.device != weight.device or turned and weight8.turned is None:
        raise ValueError(f"linear_f8: weight8 is {weight8} on {weight8.device}, the weight {tuple(weight.shape)} on {weight.device}")


class _LinearF8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, held, weight8):
        need_x, need_w = ctx.needs_input_grad[:2]
        if weight8 is None:
            weight8 = _f8.f8_weight(_rows(weight.detach()), backward=need_x)
        else:
            _same_weight(weight8, weight, need_x)
        if need_w:
            if held is None:
                held = hold(x)
            elif tuple(held.shape) != tuple(x.shape) or held.dtype != x.dtype or held.device != x.device:
                raise ValueError(f"linear_f8: held is the checkpoint of a {tuple(held.shape)} {held.dtype} tensor on {held.device}, x is "
                                 f"{tuple(x.shape)} {x.dtype} on {x.device}")
        # codes go through autograd as bytes, which hooks that take activations leave alone
        codes = (weight8.turned.view(torch.uint8), weight8.scales) if need_x else (None, None)
        _keep(ctx, held if need_w else None, *codes)
        ctx.weight = weight.shape, weight.dtype
        return _f8.f8_linear(_rows(x), weight8, bias)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx = dw = db = None
        dy = _rows(dy)
        (n, k), dtype = ctx.weight
        codes, scales, *held = _kept(ctx, 2) if need_w else ctx.saved_tensors
        if need_w:
            dw, db = q8.q8_weight_grad(dy, held[0], bias=need_b, out_dtype=dtype)
        elif need_b:
            db = dy.reshape(-1, n).sum(dim=0)
        if need_x:
            dx = _f8._product("linear_f8: dy", dy, _Scales(scales, dy.device), codes, n, k, 1, None, None)
        return dx, dw, db, None, None


class _Scales:
    """What a product reads of an ``F8Weight`` besides its codes."""
    __slots__ = ("scales", "device")

    def __init__(self, scales, device):
        self.scales, self.device = scales, device


def linear_f8(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, held: Checkpoint8 | None = None,
              weight8: F8Weight | None = None):
    """``x @ weight.T + bias`` in 8-bit floating point (``cswap_amd.f8``), and so the gradient of x; that of the weight comes from x's 8-bit checkpoint.
    ``held``: that checkpoint, ``weight8``: the weight as ``f8.f8_weight`` lays it out, where they are there already (a weight that several
    micro-batches meet is laid out once).  Under autocast in its type."""
    if torch.is_autocast_enabled("cuda") and x.dtype != torch.float64:
        dtype = torch.get_autocast_dtype("cuda")
        x, weight, bias = (t if t is None else t.to(dtype) for t in (x, weight, bias))
    if not torch.is_grad_enabled():
        if weight8 is None:
            weight8 = _f8.f8_weight(_rows(weight), backward=False)
        else:
            _same_weight(weight8, weight, False)
        return _f8.f8_linear(_rows(x), weight8, bias)
    return _LinearF8.apply(x, weight, bias, held, weight8)


# ------------------------------------------------------------------- layer norm
class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        need = any(ctx.needs_input_grad)
        y, mean, rstd, held = q8.layer_norm(_rows(x), weight, bias, eps, checkpoint=need)
        if need:
            _keep(ctx, held, mean, rstd, None if weight is None else weight.detach())
            ctx.params = weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        mean, rstd, weight, held = _kept(ctx, 3)
        dx, dw, db = q8.layer_norm_backward(_rows(dy), held, mean, rstd, weight, ctx.params)
        need = ctx.needs_input_grad
        return dx if need[0] else None, dw if need[1] else None, db if need[2] else None, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5):
    """Layer norm over the last dimension; under autocast in fp32, as torch's is."""
    if torch.is_autocast_enabled("cuda") and x.dtype != torch.float64:
        x = x.float()
    if not torch.is_grad_enabled():
        return q8.layer_norm(_rows(x), weight, bias, eps, checkpoint=False)[0]
    return _LayerNorm.apply(x, weight, bias, eps)


# ------------------------------------------------------------------- group norm
def _channels_last(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy of it that lies channels last."""
    try:
        q8._images(t, "")
        return t
    except ValueError:
        if t.dim() < 2:
            raise
        return t.movedim(1, -1).contiguous().movedim(-1, 1)


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act):
        need = any(ctx.needs_input_grad)
        y, mean, rstd, held = q8.group_norm(_channels_last(x), groups, weight, bias, eps, act, checkpoint=need)
        if need:
            _keep(ctx, held, mean, rstd, None if weight is None else weight.detach(), None if bias is None else bias.detach())
            ctx.params = weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype
            ctx.how = groups, act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        mean, rstd, weight, bias, held = _kept(ctx, 4)
        groups, act = ctx.how
        dx, dw, db = q8.group_norm_backward(_channels_last(dy), held, mean, rstd, groups, weight, bias, act, ctx.params)
        need = ctx.needs_input_grad
        return dx if need[0] else None, dw if need[1] else None, db if need[2] else None, None, None, None


def group_norm(x: torch.Tensor, groups: int, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5,
               act: str | None = None):
    """Group norm of images ``[N, C, ...]``, then ``act`` ("gelu", "gelu_tanh", "silu"; None: none); under autocast in fp32, as torch's is.
    Images that do not lie channels last are copied so first; the result and the gradient lie so in any case."""
    if torch.is_autocast_enabled("cuda") and x.dtype != torch.float64:
        x = x.float()
    if not torch.is_grad_enabled():
        return q8.group_norm(_channels_last(x), groups, weight, bias, eps, act, checkpoint=False)[0]
    return _GroupNorm.apply(x, weight, bias, groups, eps, act)


# ------------------------------------------------------------------- activation functions
class _Act(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kind):
        y, held = q8.q8_act(_rows(x), kind, checkpoint=ctx.needs_input_grad[0])
        if held is not None:
            _keep(ctx, held)
            ctx.kind = kind
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        held, = _kept(ctx, 0)
        return q8.q8_act_backward(_rows(dy), held, ctx.kind), None


def activation(x: torch.Tensor, kind: str = "gelu"):
    """"gelu", "gelu_tanh" or "silu" of x."""
    if not torch.is_grad_enabled():
        return q8.q8_act(_rows(x), kind, checkpoint=False)[0]
    return _Act.apply(x, kind)


# ------------------------------------------------------------------- modules
class Linear8(nn.Linear):
    """``nn.Linear`` whose input is kept in 8 bits."""

    def forward(self, x):
        return linear(x, self.weight, self.bias)


class LinearF8(nn.Linear):
    """``nn.Linear`` whose products are in 8-bit floating point and whose input is kept in 8 bits.  The weight is laid out in each call; a
    program that serves with weights that stay lays them out once and calls ``f8.f8_linear``."""

    def forward(self, x):
        return linear_f8(x, self.weight, self.bias)


class LayerNorm8(nn.LayerNorm):
    """``nn.LayerNorm`` whose input is kept in 8 bits."""

    def forward(self, x):
        shape = self.normalized_shape
        if tuple(x.shape[-len(shape):]) != tuple(shape):
            raise ValueError(f"LayerNorm8: the last dimensions are {tuple(x.shape[-len(shape):])}, not {tuple(shape)}")
        weight, bias = self.weight, self.bias
        if len(shape) == 1:
            return layer_norm(x, weight, bias, self.eps)
        flat = x.reshape(*x.shape[:-len(shape)], math.prod(shape))
        return layer_norm(flat, None if weight is None else weight.reshape(-1), None if bias is None else bias.reshape(-1),
                          self.eps).view(x.shape)


class GroupNorm8(nn.GroupNorm):
    """``nn.GroupNorm`` whose input is kept in 8 bits; images lie channels last (others are copied so).  ``act``: an activation function behind it
    in the same call."""
    act = None

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, device=None, dtype=None, *, act: str | None = None):
        super().__init__(num_groups, num_channels, eps, affine, device, dtype)
        if act is not None:
            q8._kind_of(act)
        self.act = act

    def forward(self, x):
        if x.dim() < 2 or x.shape[1] != self.num_channels:
            raise ValueError(f"GroupNorm8: images of {self.num_channels} channels, not {tuple(x.shape)}")
        return group_norm(x, self.num_groups, self.weight, self.bias, self.eps, self.act)


class GELU8(nn.GELU):
    """``nn.GELU`` whose input is kept in 8 bits."""

    def forward(self, x):
        return activation(x, "gelu_tanh" if self.approximate == "tanh" else "gelu")


class SiLU8(nn.SiLU):
    """``nn.SiLU`` whose input is kept in 8 bits."""

    def forward(self, x):
        if self.inplace:
            raise ValueError("SiLU8: not in place")
        return activation(x, "silu")


_KINDS = {nn.Linear: Linear8, nn.LayerNorm: LayerNorm8, nn.GELU: GELU8, nn.SiLU: SiLU8}


def checkpoint_layers(model: nn.Module, group_norm: bool = False, f8: bool = False) -> nn.Module:
    """Every ``nn.Linear``, ``nn.LayerNorm``, ``nn.GELU`` and ``nn.SiLU`` of ``model`` (itself among them) becomes its form here, in place:
    parameters, hooks and state stay as they are.  Classes derived from them are left alone, and so are a SiLU that works
    in place, a layer norm over more than 16384 values, a linear layer with more than 2^20 features on one side, and either over
    none.  ``group_norm=True``: every ``nn.GroupNorm`` of up to 4096 channels in up to 2048 groups, too, for models whose images lie channels last.
    ``f8=True``: linear layers become ``LinearF8``, those that are ``Linear8`` already among them."""
    kinds = dict(_KINDS)
    if group_norm:
        kinds[nn.GroupNorm] = GroupNorm8
    if f8:
        kinds[nn.Linear] = kinds[Linear8] = LinearF8
    for m in model.modules():
        to = kinds.get(type(m))
        if to is not None and _fits(m):
            m.__class__ = to
    return model


def _fits(m: nn.Module) -> bool:
    if type(m) is nn.SiLU:
        return not m.inplace
    if type(m) is nn.LayerNorm:
        return 0 < math.prod(m.normalized_shape) <= q8.MAX_NORM
    if type(m) is nn.GroupNorm:
        return 0 < m.num_channels <= q8.MAX_CHANNELS and m.num_groups <= q8.MAX_GROUPS
    return type(m) not in (nn.Linear, Linear8) or 0 < min(m.weight.shape) and max(m.weight.shape) <= q8.MAX_FEATURES
