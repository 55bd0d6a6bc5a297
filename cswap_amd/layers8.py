"""Layers that keep what their backward pass needs in 8 bits (``cswap_amd.q8``), with gradients.

The reference swaps the inputs of selected layers out and back in (CSWAP+/Execution.h:70-127,
CIFAR10/models/vgg.py:23-45).  Here the input of a linear layer, a layer norm or an activation function
stays on the device in one byte a value, and the layer's backward pass reads it in that form:

    import cswap_amd.layers8 as layers8
    layers8.checkpoint_layers(model)        # nn.Linear, nn.LayerNorm, nn.GELU, nn.SiLU of a model, in place
    y = layers8.linear(x, weight, bias)     # or function by function

Outputs are those of the layers without checkpoints (linear layers run torch's own product; norms and activation
functions are computed in fp32 and rounded once, which may differ from torch's in the last place); gradients are
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

from . import q8
from .q8 import Checkpoint8

__all__ = ["hold", "linear", "layer_norm", "activation", "Linear8", "LayerNorm8", "GELU8", "SiLU8", "checkpoint_layers"]


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


def checkpoint_layers(model: nn.Module) -> nn.Module:
    """Every ``nn.Linear``, ``nn.LayerNorm``, ``nn.GELU`` and ``nn.SiLU`` of ``model`` (itself among them) becomes its form here, in place:
    parameters, hooks and state stay as they are.  Classes derived from them are left alone, and so are a SiLU that works
    in place, a layer norm over more than 16384 values, a linear layer with more than 2^20 features on one side, and either over
    none."""
    for m in model.modules():
        to = _KINDS.get(type(m))
        if to is not None and _fits(m):
            m.__class__ = to
    return model


def _fits(m: nn.Module) -> bool:
    if type(m) is nn.SiLU:
        return not m.inplace
    if type(m) is nn.LayerNorm:
        return 0 < math.prod(m.normalized_shape) <= q8.MAX_NORM
    return type(m) is not nn.Linear or 0 < min(m.weight.shape) and max(m.weight.shape) <= q8.MAX_FEATURES
