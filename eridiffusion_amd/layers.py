"""Layers at a transformer's entry, on kernels of their own: embedding lookup with scaling, dropout from a counter-based
generator, and the residual's addition with root-mean-square norm, each with its gradient (include/eri_layers.h).

Tensors are float32 or bfloat16 on the GPU; the calls run on the current stream of their device and wait for nothing.
`embedding`, `dropout` and `rms_norm` are differentiable: where an input requires a gradient, autograd records them.
Forward-mode tangents are refused, and so are tracers (`torch.jit.trace`, `make_fx`, fake tensors): they record torch's operations,
and these kernels are none.  An `out` that overlaps an input is refused too; only `dropout` may write over x itself.
`embedding_grad` and `rms_norm_grad` are the backward passes themselves, for trainers that keep their own: the
table's gradient may be float32 beside a bfloat16 table and may be accumulated over micro-batches, which is what
`Adam8bit` takes as `.grad` as it stands.
"""
from typing import NamedTuple, Optional, Tuple, Union

import torch
from torch import Tensor

from . import _layers_face
from ._lib import lib

lib()  # torch's HIP runtime and the library, before the first call

Offset = Union[int, Tensor]


class RmsNorm(NamedTuple):
    """What rms_norm() returns."""
    y: Tensor
    h: Tensor                 # what was normed: residual + dropped x; x itself where nothing was added or dropped
    rstd: Tensor              # 1 / sqrt(mean of h^2 + eps) of each row, float32
    scales: Optional[Tensor]  # of an 8-bit y, float32


class RmsNormGrad(NamedTuple):
    """What rms_norm_grad() returns; None for what is not needed.  x and residual may be one tensor."""
    x: Optional[Tensor]
    residual: Optional[Tensor]
    weight: Optional[Tensor]


def embedding(ids: Tensor, weight: Tensor, scale: float = 1.0, *, out: Optional[Tensor] = None, padding_id: Optional[int] = None) -> Tensor:
    """scale * weight[ids], of shape ids.shape + (dim,); a row of zeros for an id outside the table.

    Rows named padding_id are looked up like others, but get no gradient."""
    if padding_id is not None and not 0 <= padding_id < weight.shape[0]:
        raise ValueError("padding_id is no row of the table")
    rows = _layers_face.embedding(ids, weight, scale, out)
    return _Embedding.apply(ids, weight, scale, padding_id) if rows is None else rows


def embedding_grad(ids: Tensor, grad: Tensor, vocab: int, scale: float = 1.0, *, padding_id: Optional[int] = None,
                   dtype: Optional[torch.dtype] = None, out: Optional[Tensor] = None, accumulate: bool = False) -> Tensor:
    """The table's gradient, (vocab, dim): in row v, scale times the sum of the rows of grad whose id is v.

    Tokens with padding_id or an id outside the table add nothing.  dtype: float32 or bfloat16, grad's by default.
    accumulate: added to what out holds.  The same inputs give the same bits."""
    return _layers_face.embedding_grad(ids, grad, vocab, scale, padding_id, dtype, out, accumulate)


def dropout(x: Tensor, p: float, seed: int, offset: Offset = 0, *, out: Optional[Tensor] = None) -> Tensor:
    """x with a share p of its elements set to zero and the others divided by the share that is kept.

    Which ones goes by seed, offset and the element's place in x alone, so that nothing has to be stored: the backward
    pass is the same call on the gradient.  Calls that shall be independent differ in seed or offset.  The offset may be an
    int64 tensor of one element on the device, read when the kernel runs: a captured graph draws anew where the tensor is
    advanced between replays.  p counts in steps of 1/65536."""
    y = _layers_face.dropout(x, p, seed, offset, out)
    return _Dropout.apply(x, p, seed, offset) if y is None else y


def rms_norm(x: Tensor, weight: Optional[Tensor] = None, eps: float = 1e-6, *, residual: Optional[Tensor] = None, p: float = 0.0,
             seed: int = 0, offset: Offset = 0, dtype: Optional[torch.dtype] = None, scale_group: int = 0) -> RmsNorm:
    """h = residual + dropout(x, p, seed, offset);  y = h / sqrt(mean(h^2) + eps) * weight over the last dimension.

    dtype of y: float32, bfloat16 (x's by default) or float8_e4m3fn, which comes with float32 scales: one for each row, or
    for each 128 columns of it with scale_group=128, so that y * scale is the norm's output.  h has the residual's dtype."""
    got = _layers_face.rms_norm(x, weight, eps, residual, p, seed, offset, dtype, scale_group)
    if got is not None:
        return RmsNorm._make(got)
    if residual is None and p == 0:
        y, rstd = _RmsNorm.apply(x, weight, None, eps, 0.0, 0, 0, dtype)
        return RmsNorm(y, x, rstd, None)
    y, rstd, h = _RmsNorm.apply(x, weight, residual, eps, p, seed, offset, dtype)
    return RmsNorm(y, h, rstd, None)


def rms_norm_grad(grad: Tensor, h: Tensor, rstd: Tensor, weight: Optional[Tensor] = None, *, grad_h: Optional[Tensor] = None, p: float = 0.0,
                  seed: int = 0, offset: Offset = 0, dtype: Optional[torch.dtype] = None,
                  needs: Tuple[bool, bool, bool] = (True, True, True)) -> RmsNormGrad:
    """Gradients of rms_norm's x, residual and weight (`needs`: which of them) from that of y, and grad_h, what reaches h
    besides the norm.  h and rstd are what rms_norm returned; dtype is x's (grad's by default), weight's gradient has weight's
    dtype.  The same inputs give the same bits."""
    return RmsNormGrad._make(_layers_face.rms_norm_grad(grad, h, rstd, weight, grad_h, p, seed, offset, dtype, needs))


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_id):
        ctx.save_for_backward(ids)
        ctx.rest = weight.shape[0], scale, padding_id, weight.dtype
        return embedding(ids, weight, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        vocab, scale, padding_id, dtype = ctx.rest
        return None, embedding_grad(*ctx.saved_tensors, grad, vocab, scale, padding_id=padding_id, dtype=dtype), None, None


def _keep_offset(ctx, offset, *tensors):
    """A tensor that is advanced before the backward pass has run is noticed there."""
    ctx.offset = None if isinstance(offset, Tensor) else offset
    ctx.save_for_backward(*tensors, offset if ctx.offset is None else None)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, offset):
        ctx.rest = p, seed
        _keep_offset(ctx, offset)
        return dropout(x, p, seed, offset)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        offset, = ctx.saved_tensors
        return dropout(grad, *ctx.rest, ctx.offset if offset is None else offset), None, None, None


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps, p, seed, offset, dtype):
        r = rms_norm(x, weight, eps, residual=residual, p=p, seed=seed, offset=offset, dtype=dtype)
        ctx.rest = p, seed, x.dtype
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(r.rstd)
        _keep_offset(ctx, offset, r.h, r.rstd, weight)
        return (r.y, r.rstd) if r.h is x else (r.y, r.rstd, r.h)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _, grad_h=None):
        h, rstd, weight, offset = ctx.saved_tensors
        p, seed, dtype = ctx.rest
        if grad is None:
            grad = torch.zeros_like(h)
        need = ctx.needs_input_grad
        g = rms_norm_grad(grad, h, rstd, weight, grad_h=grad_h, p=p, seed=seed, offset=ctx.offset if offset is None else offset, dtype=dtype,
                          needs=(need[0], need[2], need[1]))
        return g.x, g.weight, g.residual, None, None, None, None, None
