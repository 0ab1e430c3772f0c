"""The losses of include/eri_losses.h in 64 bits, one formula a line, on the device of their inputs: what the kernels are tested against.

Temperatures are those that the kernels get, rounded to 32 bits.  Each function also gives what the errors of 32-bit arithmetic
are measured by."""
import math

import numpy as np
import torch

INF = math.inf


def t32(temperature):
    return float(np.float32(temperature))


def softmax(logits, temperature):
    """m, ln s, p, ln p; {-inf, -inf, 0, -inf} where nothing is left, NaN where there is NaN or plus infinity."""
    x, t = logits.double(), t32(temperature)
    m = torch.where(x.isnan(), -INF, x).amax(-1, keepdim=True)
    none = (m == -INF) & ~x.isnan().any(-1, keepdim=True)
    d = torch.where(x == -INF, -INF, x - torch.where(none, 0.0, m))
    e = (d / t).exp()
    log_s = e.sum(-1, keepdim=True).log()
    logp = torch.where(none, -INF, torch.where(log_s.isnan(), math.nan, d / t - log_s))
    return m.squeeze(-1), log_s.squeeze(-1), torch.where(none, 0.0, logp.exp()), logp


def plogp(p, logp):
    return torch.where(p == 0, 0.0, p * logp)


def largest(logits, k):
    """Values and places of the k largest; of equal ones the first comes first."""
    x, places = torch.sort(torch.where(logits == 0, 0.0, logits.double()), dim=-1, descending=True, stable=True)
    return x[..., :k], places[..., :k]


def token_logprobs(logits, ids=None, temperature=1.0, top=0):
    """logprob, entropy, top, top_ids, m, ln s."""
    m, log_s, p, logp = softmax(logits, temperature)
    one = None
    if ids is not None:
        fits = (ids >= 0) & (ids < logits.shape[-1])
        one = torch.where(fits, logp.gather(-1, torch.where(fits, ids, 0).long()[..., None]).squeeze(-1), 0.0)
    h = -plogp(p, logp).sum(-1)
    nan = log_s.isnan()[..., None]
    places = values = None
    if top:
        places = largest(torch.nan_to_num(logits.double(), 0.0, INF, -INF), top)[1]
        places = torch.where(nan, torch.arange(top, device=logits.device), places)
        values = torch.where(nan, math.nan, logp.gather(-1, places))
    return one, h, values, places, torch.where(log_s == -INF, -INF, m), log_s


def token_logprobs_grad(logits, ids, grad, grad_entropy=None, temperature=1.0):
    """The gradient, p and ln p."""
    _, log_s, p, logp = softmax(logits, temperature)
    fits = torch.zeros_like(grad, dtype=torch.bool) if ids is None else (ids >= 0) & (ids < logits.shape[-1])
    g = torch.where(fits, grad.double(), 0.0)[..., None]
    one = torch.zeros_like(p)
    if ids is not None:
        one.scatter_(-1, torch.where(fits, ids, 0).long()[..., None], fits.double()[..., None])
    dz = g * (one - p)
    h = torch.zeros_like(g) if grad_entropy is None else grad_entropy.double()[..., None]
    terms = plogp(p, logp)
    dz = dz - torch.where(h == 0, 0.0, h * (terms - p * terms.sum(-1, keepdim=True)))
    dz = torch.where((log_s == -INF)[..., None] | ((g == 0) & (h == 0)), 0.0, dz)
    return dz / t32(temperature), p, logp


def distill_top(logits, ids, teacher, temperature=1.0, rest=False):
    """loss, stats (.., 6), the loss's gradient, p of the named tokens (.., k), q (.., k)."""
    t, vocab = t32(temperature), logits.shape[-1]
    m, log_s, p, logp = softmax(logits, temperature)
    fits = (ids >= 0) & (ids < vocab)
    at = torch.where(fits, ids, 0).long()
    named = torch.zeros_like(p).scatter_add_(-1, at, fits.double()) > 0
    outside = torch.where(named, -INF, logits.double())
    m_o, log_o, p_o, _ = softmax(outside, temperature)
    apart = (log_o != -INF) if rest else torch.zeros_like(log_o, dtype=torch.bool)
    value = torch.where(fits, teacher.double(), -INF)
    norm = torch.logsumexp(value, -1)
    norm = torch.where(torch.isposinf(value).any(-1), math.nan, norm)
    divisor = torch.where(apart & (norm <= 0), 0.0, norm)
    q = torch.where(value == -INF, 0.0, (value - divisor[..., None]).exp())
    lp = logp.gather(-1, at)
    terms = torch.where(q == 0, 0.0, q * (value - divisor[..., None] - lp))
    held = torch.where(named, p, 0.0).sum(-1)
    qr = torch.where(apart & ~(norm > 0), (1 - q.sum(-1)).clamp(min=0.0), 0.0)  # none where q is divided by its sum, whatever that rounds to
    log_r = (m_o - m) / t + log_o - log_s
    log_r = torch.where(held < 0.5, torch.log1p(-held.clamp(max=0.5)), log_r)
    loss = terms.sum(-1) + torch.where(apart & (qr != 0), qr * (qr.log() - log_r), 0.0)
    loss = torch.where(apart & log_s.isnan(), math.nan, loss)
    some = (value != -INF).any(-1)
    over = torch.where(apart, torch.where(held < 0.5, q.sum(-1) - held, log_r.exp() - qr), torch.where(some, torch.where(norm.isnan(), math.nan, 1.0), 0.0))
    dz = torch.where(apart[..., None], p_o, p) * over[..., None]
    total = torch.zeros_like(p).scatter_add_(-1, at, torch.where(fits, q, 0.0))
    # where the teacher leaves nothing and there is no rest, nothing is asked of the named tokens either
    dz = torch.where(named, torch.where((norm == -INF) & ~apart, 0.0, 1.0)[..., None] * p - total, dz)
    dz = torch.where((log_s == -INF)[..., None], 0.0, dz)
    empty = log_s == -INF
    stats = torch.stack((torch.where(empty, -INF, m), log_s, torch.where(empty, -INF, torch.where(apart, m_o, m)), torch.where(apart, log_o, log_s), divisor, over), -1)
    return loss, stats, dz / t, lp.exp(), q
