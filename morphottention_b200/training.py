"""The operators of a training step around the attention layer, on hand-written kernels: layer norm with
the residual add, softmax cross entropy over a large vocabulary without keeping the logits, and the
global gradient norm with clipping.

Each has an autograd form (:func:`layer_norm`, :class:`LayerNorm`, :func:`linear_cross_entropy`) and the
pair of calls behind it (``*_forward`` / ``*_backward``, thin over ``torch.ops.morphottention``), for
callers that keep their own graph.  They run on the current stream, allocate through torch and never
wait on the host, so a step that uses them can be captured in a CUDA graph.  There is no CPU form.
"""

from __future__ import annotations

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from ._ops import add_op_namespace_prefix, ops

REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}

# the overloads themselves: a call through the packet looks them up every time
_norm_forward, _norm_backward = ops.layer_norm_forward.default, ops.layer_norm_backward.default
_loss_forward, _loss_backward = ops.linear_cross_entropy_forward.default, ops.linear_cross_entropy_backward.default
_clip = ops.clip_grad_norm.default


@torch.library.register_fake(add_op_namespace_prefix("layer_norm_forward"))
def _layer_norm_forward_fake(x, weight, bias, eps, residual=None):
    stat = x.new_empty(x.shape[:-1], dtype=torch.float32)
    out = [x.new_empty(x.shape), stat, torch.empty_like(stat)]
    return out if residual is None else out + [x.new_empty(x.shape)]


@torch.library.register_fake(add_op_namespace_prefix("layer_norm_backward"))
def _layer_norm_backward_fake(grad_y, h, weight, mean, rstd, grad_h=None):
    w = h.new_empty(h.shape[-1:]) if weight is None else weight
    return [h.new_empty(h.shape), torch.empty_like(w), torch.empty_like(w)]


@torch.library.register_fake(add_op_namespace_prefix("linear_cross_entropy_forward"))
def _linear_cross_entropy_forward_fake(hidden, weight, target, ignore_index=-100, reduction=1):
    lse = hidden.new_empty(target.shape, dtype=torch.float32)
    return [torch.empty_like(lse) if reduction == 0 else hidden.new_empty((), dtype=torch.float32), lse]


@torch.library.register_fake(add_op_namespace_prefix("linear_cross_entropy_backward"))
def _linear_cross_entropy_backward_fake(grad_loss, hidden, weight, target, lse, ignore_index=-100, reduction=1):
    return [hidden.new_empty(hidden.shape), weight.new_empty(weight.shape)]


@torch.library.register_fake(add_op_namespace_prefix("clip_grad_norm"))
def _clip_grad_norm_fake(grads, out, max_norm, loss_scale=1.0):
    return grads[0].new_empty((), dtype=torch.float32)


# ---- layer norm --------------------------------------------------------------------------------------

def layer_norm_forward(x, weight=None, bias=None, eps: float = 1e-5, residual=None):
    """``[y, mean, rstd]``, or ``[y, mean, rstd, h]`` with a ``residual``: ``h = x + residual`` in their
    type, ``y = (h - mean) * rstd * weight + bias`` over the last dimension.

    :param x: float16, bfloat16 or float32 CUDA tensor ``[..., dim]``; rows may have any common stride.
    :param weight, bias: ``[dim]`` in ``x``'s type or float32 (both in one), or None (a bias needs a weight).
    :returns: ``y`` and ``h`` contiguous in ``x``'s type, ``mean`` and ``rstd`` float32 ``[...]``."""
    return _norm_forward(x, weight, bias, eps, residual)


def layer_norm_backward(grad_y, h, weight, mean, rstd, grad_h=None):
    """``[dx, dweight, dbias]`` for the gradients of ``y`` and, with a residual, of ``h`` (``grad_h`` may be
    None).  ``dx`` is the gradient of the residual as well.  ``h`` is the forward's (``x`` without a
    residual).  Deterministic."""
    return _norm_backward(grad_y, h, weight, mean, rstd, grad_h)


class LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps: float, residual):
        if not x.is_cuda:
            raise ValueError("layer_norm expects a CUDA tensor")
        ctx.set_materialize_grads(False)
        y, mean, rstd, *h = _norm_forward(x, weight, bias, eps, residual)
        ctx.save_for_backward(h[0] if h else x, weight, mean, rstd)
        ctx.has_bias = bias is not None
        ctx.has_residual = residual is not None
        return (y, h[0]) if h else y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y, grad_h=None):
        h, weight, mean, rstd = ctx.saved_tensors
        if grad_y is None:  # only h was used
            if grad_h is None:
                return None, None, None, None, None
            return grad_h, None, None, None, grad_h if ctx.has_residual else None
        dx, dw, db = _norm_backward(grad_y, h, weight, mean, rstd, grad_h)
        return (dx, dw if weight is not None else None, db if ctx.has_bias else None, None,
                dx if ctx.has_residual else None)


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, *, residual=None):
    """Layer norm over the last dimension, with gradients for ``x``, ``weight`` and ``bias``.  With a
    ``residual`` it returns ``(y, h)``: ``h = x + residual`` and its norm, the step every pre-norm block
    takes, in one pass over memory; both results carry gradients."""
    return LayerNormFunction.apply(x, weight, bias, eps, residual)


class LayerNorm(nn.Module):
    """:func:`layer_norm` with its parameters (ones and zeros at the start; ``state_dict`` as
    ``torch.nn.LayerNorm``).  ``forward(x)`` gives ``y``, ``forward(x, residual)`` gives ``(y, h)``.

    :param dim: width of the last dimension.
    :param bias: False leaves the bias out.
    :param dtype: parameter type: the inputs' or float32."""

    def __init__(self, dim: int, eps: float = 1e-5, *, bias: bool = True, dtype: torch.dtype = torch.float16,
                 device=None) -> None:
        super().__init__()
        if dim <= 0:
            raise ValueError(f"dim must be positive (got {dim})")
        self.dim, self.eps = dim, eps
        self.weight = nn.Parameter(torch.ones(dim, dtype=dtype, device=device))
        self.register_parameter("bias", nn.Parameter(torch.zeros(dim, dtype=dtype, device=device)) if bias else None)

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        return LayerNormFunction.apply(x, self.weight, self.bias, self.eps, residual)


# ---- vocabulary loss -----------------------------------------------------------------------------------

def _reduction(reduction) -> int:
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction must be one of {tuple(REDUCTIONS)}")
    return REDUCTIONS[reduction]


def linear_cross_entropy_forward(hidden, weight, target, ignore_index: int = -100, reduction: str = "mean"):
    """``[loss, lse]`` of ``z = hidden @ weight.T``: ``lse = logsumexp(z)`` per token (float32) and the
    cross entropy ``lse - z[target]``, zero where ``target == ignore_index``.

    :param hidden: float16 or bfloat16 ``[..., dim]``, ``dim`` a multiple of 8.
    :param weight: ``[vocab, dim]`` in the same type (the output embedding).
    :param target: int64 ``[...]``.  One outside ``[0, vocab)`` that is not ignored makes its token's
        loss NaN (no device assert).
    :param reduction: ``"none"`` (``[...]``), ``"sum"``, or ``"mean"`` over the tokens that are not
        ignored (0, not NaN, if all are)."""
    return _loss_forward(hidden, weight, target, ignore_index, _reduction(reduction))


def linear_cross_entropy_backward(grad_loss, hidden, weight, target, lse, ignore_index: int = -100,
                                  reduction: str = "mean"):
    """``[dhidden, dweight]`` for the loss's float32 gradient (``target``'s shape for ``"none"``, else one
    element) and the forward's ``lse``.  Tokens that are ignored, or whose gradient is zero, add nothing to
    either, whatever their hidden rows hold (NaN and infinities included).  Deterministic."""
    return _loss_backward(grad_loss, hidden, weight, target, lse, ignore_index,
                                             _reduction(reduction))


class LinearCrossEntropyFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, target, ignore_index: int, reduction: int):
        if not hidden.is_cuda:
            raise ValueError("linear_cross_entropy expects CUDA tensors")
        loss, lse = _loss_forward(hidden, weight, target, ignore_index, reduction)
        ctx.save_for_backward(hidden, weight, target, lse)
        ctx.options = ignore_index, reduction
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss):
        hidden, weight, target, lse = ctx.saved_tensors
        dh, dw = _loss_backward(grad_loss, hidden, weight, target, lse, *ctx.options)
        return dh, dw, None, None, None


def linear_cross_entropy(hidden, weight, target, *, ignore_index: int = -100, reduction: str = "mean"):
    """Softmax cross entropy of ``hidden @ weight.T`` with gradients for ``hidden`` and ``weight``; the
    logits are never stored (see :func:`linear_cross_entropy_forward`)."""
    return LinearCrossEntropyFunction.apply(hidden, weight, target, ignore_index, _reduction(reduction))


# ---- gradient clipping -----------------------------------------------------------------------------------

def clip_grad_norm(grads, max_norm: float, *, out=None, loss_scale: float = 1.0) -> torch.Tensor:
    """2-norm over all ``grads`` (float32, on the device, not read on the host), and the clipped gradients
    in ``out``:

        norm = sqrt(sum |g|^2) / loss_scale,   out = g * min(1, max_norm / (norm + 1e-6)) / loss_scale

    :param grads: CUDA tensors, float16, bfloat16 or float32, mixed as they come, dense.
    :param out: as many tensors of the same shapes, in any of the three types (float32 masters of
        16-bit gradients, say); None writes ``grads`` in place.
    :param loss_scale: the factor that the loss was multiplied by, removed here.

    An infinite gradient makes the norm infinite: finite gradients become zero, infinite ones NaN.  With
    a NaN among them the norm and every result are NaN."""
    grads = list(grads)
    return _clip(grads, grads if out is None else list(out), max_norm, loss_scale)


def clip_grad_norm_(parameters, max_norm: float, *, loss_scale: float = 1.0) -> torch.Tensor:
    """:func:`clip_grad_norm` in place on the gradients of ``parameters`` (those that have one); zero if
    none has."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.zeros(())
    return clip_grad_norm(grads, max_norm, loss_scale=loss_scale)
