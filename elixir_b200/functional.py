"""Operators of the wrapped model with their gradients: layer norm, and the embedding lookup with a scale.

``ElixirModule(use_fused_kernels=True)`` runs the ``nn.LayerNorm`` and ``nn.Embedding`` layers of its module through
them (``use_kernels``), where the reference swaps in a fused layer norm (``elixir/kernels/layernorm.py:4``,
``elixir/hook/parameter.py:69-70``).  Statistics and sums are fp32, every output is rounded once, and both parameter
gradients are summed in an order that the inputs alone fix.  CUDA tensors only.  ``layer_norm`` and ``embedding`` have first
derivatives in reverse mode only; for anything else the layers of a module stay with torch (``use_kernels``).  As with
every autograd function, a backward pass is captured into a CUDA graph only while no eager graph of the same parameters is
alive.
"""
from functools import partial
from math import prod
from typing import Optional

import torch
import torch.nn as nn
from torch.autograd import Function, forward_ad
from torch.autograd.function import once_differentiable
from torch.utils._device import DeviceContext

from . import _abi, kernels

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


class _LayerNorm(Function):

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = kernels.layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias_shape = None if bias is None else bias.shape
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        dx, dweight, dbias = kernels.layer_norm_backward(dy.contiguous(), x, weight, mean, rstd,
                                                         weight_grad=ctx.needs_input_grad[1],
                                                         bias_grad=ctx.needs_input_grad[2])
        return (dx if ctx.needs_input_grad[0] else None, None if dweight is None else dweight.view(weight.shape),
                None if dbias is None else dbias.view(ctx.bias_shape), None)


class _LayerNormOfLayer(_LayerNorm):
    """A backward pass that is going to be differentiated itself (``create_graph``) is torch's."""

    @staticmethod
    def backward(ctx, dy):
        if not torch.is_grad_enabled():
            return _LayerNorm.backward(ctx, dy)
        x, weight, mean, rstd = ctx.saved_tensors
        need_x, need_weight = ctx.needs_input_grad[0], ctx.needs_input_grad[1] and weight is not None
        need_bias = ctx.needs_input_grad[2] and ctx.bias_shape is not None
        rows = x.shape[:-1] + (1, )
        dx, dweight, _ = torch.ops.aten.native_layer_norm_backward(dy, x, x.shape[-1:], mean.view(rows), rstd.view(rows),
                                                                   None if weight is None else weight.flatten(), None,
                                                                   [need_x, need_weight, False])
        return (dx if need_x else None, dweight.view(weight.shape) if need_weight else None,
                dy.reshape(-1, dy.shape[-1]).sum(0).view(ctx.bias_shape) if need_bias else None, None)


def layer_norm(x: torch.Tensor, normalized_shape, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """``torch.nn.functional.layer_norm`` on this package's kernels.  ``weight`` and ``bias`` have the type of ``x``."""
    return _apply_layer_norm(_LayerNorm, x, normalized_shape, weight, bias, eps)


def _apply_layer_norm(function, x, normalized_shape, weight, bias, eps):
    shape = (normalized_shape, ) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    if not shape or x.shape[-len(shape):] != shape or x.dim() < len(shape):
        raise ValueError(f'normalized_shape {shape} does not end the shape {tuple(x.shape)}')
    for name, t in (('weight', weight), ('bias', bias)):
        if t is not None and t.shape != shape:
            raise ValueError(f'{name} must have the shape {shape}')
    flat = x.contiguous()
    if len(shape) > 1:
        flat = flat.flatten(-len(shape))
    # the parameters themselves, not views of them: the memory of a chunk may be another by the time of the backward pass
    weight, bias = (t if t is None else t.contiguous() for t in (weight, bias))
    return function.apply(flat, weight, bias, eps).view(x.shape)


class _Embedding(Function):

    @staticmethod
    def forward(ctx, tokens, weight, padding_idx, scale):
        ctx.save_for_backward(tokens)
        ctx.vocab, ctx.padding_idx, ctx.scale = weight.shape[0], padding_idx, scale
        return kernels.embedding_forward(tokens, weight, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        tokens, = ctx.saved_tensors
        return None, kernels.embedding_backward(tokens, dout.contiguous(), ctx.vocab, ctx.scale, ctx.padding_idx), None, None


class _EmbeddingOfLayer(_Embedding):
    """As ``_LayerNormOfLayer``: torch's, for a scale of 1."""

    @staticmethod
    def backward(ctx, dout):
        if not torch.is_grad_enabled():
            return _Embedding.backward(ctx, dout)
        tokens, = ctx.saved_tensors
        keep = (tokens >= 0) & (tokens < ctx.vocab)    # torch's operator takes tokens of the table only
        if ctx.padding_idx is not None:
            keep &= tokens != ctx.padding_idx
        dout = torch.where(keep.unsqueeze(-1), dout, torch.zeros_like(dout))
        return None, torch.ops.aten.embedding_dense_backward(dout, torch.where(keep, tokens, 0), ctx.vocab, -1, False), None, None


def embedding(tokens: torch.Tensor, weight: torch.Tensor, padding_idx: Optional[int] = None, scale: float = 1.0) -> torch.Tensor:
    """``scale * weight[tokens]``.  As with ``torch.nn.functional.embedding``, ``padding_idx`` (negative values count from
    the end) names the token whose row gets no gradient; the gradient is dense.  A token outside the table, which torch
    answers with a device assertion, reads as a row of NaN here: the overflow probe then skips the step."""
    return _apply_embedding(_Embedding, tokens, weight, padding_idx, scale)


def _apply_embedding(function, tokens, weight, padding_idx, scale=1.0):
    if padding_idx is not None:
        if not -weight.shape[0] <= padding_idx < weight.shape[0]:
            raise ValueError('padding_idx outside the table')
        padding_idx %= weight.shape[0]
    return function.apply(tokens.contiguous(), weight.contiguous(), padding_idx, float(scale))


# ---------------------------------------------------------------------------------------------------
# the layers of a module
# ---------------------------------------------------------------------------------------------------


def _watched():
    """Whether something has to see torch's own operations: a compiler, a trace, a functional transform, forward-mode
    derivatives, a dispatch or function mode (fake tensors, counters; a default device changes no operation here)."""
    return (torch.compiler.is_compiling() or torch._C._is_tracing() or torch._C._are_functorch_transforms_active()
            or forward_ad._current_level >= 0 or torch._C._len_torch_dispatch_stack() > 0
            or (torch._C._len_torch_function_stack() > 0 and any(
                not isinstance(torch._C._get_function_stack_at(i), DeviceContext)
                for i in range(torch._C._len_torch_function_stack()))))


def _plain_cuda(x, *params):
    """The kernels take CUDA tensors of one supported type, no subclasses of torch's, outside autocast (which would change
    the types) and where nothing watches torch's operations."""
    return (not _watched() and x.is_cuda and type(x) in (torch.Tensor, nn.Parameter)
            and all(p is None or (p.is_cuda and type(p) in (torch.Tensor, nn.Parameter) and p.dtype in _DTYPES
                                  and p.device == x.device) for p in params) and not torch.is_autocast_enabled('cuda'))


def _torch_forward(kind):
    """The ``forward`` of a class of torch's, or None where a program has given it another one."""
    home = getattr(kind.forward, '__globals__', {}).get('__name__')
    return kind.forward if home == kind.__module__ else None


# as they are when this module is imported: a class that has been given another one, before or after, keeps that
_TORCH_FORWARD = {kind: _torch_forward(kind) for kind in (nn.LayerNorm, nn.Embedding)}


def _layer_norm_layer(layer: nn.LayerNorm, x):
    shape, weight, bias = layer.normalized_shape, layer.weight, layer.bias
    if (type(layer).forward is _TORCH_FORWARD[nn.LayerNorm] and _plain_cuda(x, weight, bias) and x.dtype in _DTYPES
            and all(p is None or p.dtype == x.dtype for p in (weight, bias)) and 0 < prod(shape) <= _abi.NORM_MAX_COLS
            and x.shape[-len(shape):] == shape):
        return _apply_layer_norm(_LayerNormOfLayer, x, shape, weight, bias, layer.eps)
    return type(layer).forward(layer, x)


def _embedding_layer(layer: nn.Embedding, tokens):
    if (type(layer).forward is _TORCH_FORWARD[nn.Embedding] and _plain_cuda(tokens, layer.weight)
            and tokens.dtype in (torch.int32, torch.int64) and layer.max_norm is None and not layer.sparse
            and not layer.scale_grad_by_freq and layer.weight.numel() > 0):
        return _apply_embedding(_EmbeddingOfLayer, tokens, layer.weight, layer.padding_idx)
    return type(layer).forward(layer, tokens)


def use_kernels(module: nn.Module) -> int:
    """Run every ``nn.LayerNorm`` and ``nn.Embedding`` of ``module`` (subclasses that keep their ``forward`` included)
    through this package's kernels wherever those apply: CUDA tensors, one type for input and parameters, no autocast;
    embeddings without ``max_norm``, ``sparse`` and ``scale_grad_by_freq``.  Other calls stay with torch: tensor subclasses,
    forward-mode derivatives and functional transforms, compilation and tracing, calls under a dispatch or function mode; so
    do the operations of a backward pass with ``create_graph``.  A layer with a ``forward`` of its own, set on the layer or
    on its class, keeps that.  (``torch.jit.script`` takes a module before this, not after; a shallow copy of a layer needs a
    call of its own.)  Returns the number of layers."""
    count = 0
    for layer in module.modules():
        for kind, forward in ((nn.LayerNorm, _layer_norm_layer), (nn.Embedding, _embedding_layer)):
            if not isinstance(layer, kind) or type(layer).forward is not _TORCH_FORWARD[kind]:
                continue
            own = layer.__dict__.get('forward')    # None, or what a call before this one put there
            if own is None or (isinstance(own, partial) and own.func is forward):
                layer.forward = partial(forward, layer)
                count += 1
    return count
