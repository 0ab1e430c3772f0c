"""What stands between a model's logits and its gradients, on kernels of their own: log probabilities of given tokens with
entropy and top alternatives, and distillation from a teacher of which only the top tokens are kept (include/eri_losses.h).

Logits are float32 or bfloat16 on the GPU, the vocabulary their last dimension; the calls run on the current stream of their
device and wait for nothing.  One pass reads the logits, one more writes their gradient; nothing of their size is made besides.
`token_logprobs` and `distill_top` are differentiable with respect to the logits; `token_logprobs_grad` and `distill_top_grad`
are the backward passes themselves, for trainers that keep their own: there the gradient may be written over the logits (`out=logits`).

Minus infinity is a token that cannot occur, and an id outside the vocabulary names no token: it counts for nothing in a loss, as an
ignore index does.  A row whose logits are all minus infinity has log probabilities of minus infinity, entropy 0 and gradient 0; one that
holds NaN or plus infinity gives NaN.  Forward-mode tangents, tracers and overlapping outputs are refused as in `layers`.
"""
from typing import NamedTuple, Optional

import torch
from torch import Tensor

from . import _losses_face
from ._lib import lib

lib()  # torch's HIP runtime and the library, before the first call


class TokenLogprobs(NamedTuple):
    """What token_logprobs() returns, float32 but for the ids; None for what was not asked for."""
    logprob: Optional[Tensor]  # of the given token in each row, 0 where none is named
    entropy: Optional[Tensor]  # of each row
    top: Optional[Tensor]      # log probabilities of the row's largest logits, in descending order
    top_ids: Optional[Tensor]  # int64; of equal logits the lowest id comes first
    stats: Tensor              # (..., 2): the largest logit m, and the log of the sum of exp((x - m) / temperature)


class DistillTop(NamedTuple):
    """What distill_top() returns, float32."""
    loss: Tensor   # of each row
    stats: Tensor  # (..., 6): what distill_top_grad() takes


def token_logprobs(logits: Tensor, ids: Optional[Tensor] = None, *, temperature: float = 1.0, entropy: bool = False, top: int = 0) -> TokenLogprobs:
    """Log probabilities of the tokens `ids` (int32 or int64, one for each row) under softmax(logits / temperature).

    entropy: that of each row too.  top: the log probabilities and ids of that many largest logits, up to 64.  `logprob` and
    `entropy` are differentiable; cross entropy is the sum of -logprob over the number of ids that name a token."""
    got = _losses_face.token_logprobs(logits, ids, temperature, entropy, top)
    if got is not None:
        return TokenLogprobs._make(got)
    return TokenLogprobs._make(_TokenLogprobs.apply(logits, ids, temperature, entropy, top))


def token_logprobs_grad(logits: Tensor, ids: Optional[Tensor], stats: Tensor, grad: Optional[Tensor], *, grad_entropy: Optional[Tensor] = None,
                        entropy: Optional[Tensor] = None, temperature: float = 1.0, dtype: Optional[torch.dtype] = None, out: Optional[Tensor] = None) -> Tensor:
    """The logits' gradient from that of the log probabilities and, with the entropies themselves, from that of the entropies.

    stats is what token_logprobs returned.  Rows that get nothing from either are zeros.  dtype: float32 or bfloat16, the logits' by
    default.  out: rows to write, the logits themselves among them."""
    return _losses_face.token_logprobs_grad(logits, ids, stats, grad, grad_entropy, entropy, temperature, dtype, out)


def distill_top(logits: Tensor, ids: Tensor, teacher: Tensor, *, temperature: float = 1.0, rest: bool = False) -> DistillTop:
    """The divergence of softmax(logits / temperature) from a teacher whose top tokens are `ids` (..., k), k up to 64, with the log
    probabilities `teacher`, at that temperature: the `top_ids` and `top` of token_logprobs.

    rest=False: the teacher's probabilities are renormalised over its tokens.  rest=True: all other tokens are one more class, to which the
    teacher gives what its tokens leave.  The loss of each row is the sum of q (ln q - ln p); multiply by temperature ** 2 to
    keep gradients of one size.  Differentiable with respect to the logits."""
    got = _losses_face.distill_top(logits, ids, teacher, temperature, rest)
    if got is not None:
        return DistillTop._make(got)
    return DistillTop._make(_DistillTop.apply(logits, ids, teacher, temperature, rest))


def distill_top_grad(logits: Tensor, ids: Tensor, teacher: Tensor, stats: Tensor, grad: Tensor, *, temperature: float = 1.0,
                     dtype: Optional[torch.dtype] = None, out: Optional[Tensor] = None) -> Tensor:
    """The logits' gradient from that of distill_top's loss; stats is what distill_top returned.

    Rows whose gradient is 0 are zeros.  dtype: float32 or bfloat16, the logits' by default.  out: rows to write, the logits themselves
    among them."""
    return _losses_face.distill_top_grad(logits, ids, teacher, stats, grad, temperature, dtype, out)


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, temperature, entropy, top):
        r = token_logprobs(logits, ids, temperature=temperature, entropy=entropy, top=top)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*[t for t in (r.top, r.top_ids, r.stats) if t is not None])
        ctx.save_for_backward(logits, ids, r.stats, r.entropy)
        return tuple(r)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, grad_entropy, *_):
        logits, ids, stats, entropy = ctx.saved_tensors
        if grad is None and grad_entropy is None:
            return None, None, None, None, None
        dx = token_logprobs_grad(logits, None if grad is None else ids, stats, grad, grad_entropy=grad_entropy,
                                 entropy=None if grad_entropy is None else entropy, temperature=ctx.temperature)
        return dx, None, None, None, None


class _DistillTop(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, teacher, temperature, rest):
        r = distill_top(logits, ids, teacher, temperature=temperature, rest=rest)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(r.stats)
        ctx.save_for_backward(logits, ids, teacher, r.stats)
        return tuple(r)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _):
        logits, ids, teacher, stats = ctx.saved_tensors
        if grad is None:
            return None, None, None, None, None
        return distill_top_grad(logits, ids, teacher, stats, grad, temperature=ctx.temperature), None, None, None, None
