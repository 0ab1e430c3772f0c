"""The losses where their numbers leave the usual range, and the launches that only certain layouts reach, against the 64-bit oracle.

The bounds are those of test_gpu_losses.py unless a test says otherwise."""
import math

import pytest
import torch

import test_gpu_losses as tl
from oracle import losses_f64 as of
from test_gpu_layers import BF, F32
from test_gpu_losses import losses  # noqa: F401

INF = math.inf


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,vocab", [(4, 70), (5, 9003), (1100, 2003)])
@pytest.mark.parametrize("temperature,size", [(1e-4, 1e7), (1.0, 1e11), (1.0, 1e30), (1e4, 1e32)])
def test_entropy_gradients_of_any_size_leave_masked_logits_at_zero(losses, dtype, rows, vocab, temperature, size):  # noqa: F811
    """grad_entropy has no limit but float32's: what stands at minus infinity or at the type's lowest value gets nothing."""
    gen = torch.Generator().manual_seed(vocab)
    x = torch.randn(rows, vocab, generator=gen) * 2 * temperature  # a softmax over many tokens at any temperature
    masked = torch.rand(rows, vocab, generator=gen) < 0.5
    masked[:, vocab // 3] = False
    x[masked] = -INF
    x[1::2] = x[1::2].clamp(min=torch.finfo(dtype).min)
    x = x.to(dtype)
    ids, g, gh = torch.full((rows,), vocab // 3), tl._gen(rows), tl._gen(rows, seed=1) * size
    m, log_s, _, _ = of.softmax(x, temperature)
    stats, entropy = torch.stack((m, log_s), -1).float(), of.token_logprobs(x, None, temperature)[1].float()
    for out in (BF, F32):
        got = losses.token_logprobs_grad(x.cuda(), ids.cuda(), stats.cuda(), g.cuda(), grad_entropy=gh.cuda(), entropy=entropy.cuda(), temperature=temperature, dtype=out)
        assert bool((got.cpu()[masked] == 0).all())
        tl._check_token_grad(got, x, ids, g, gh, temperature, out)
