"""The layers of include/eri_layers.h in 64 bits on the CPU, one formula a line: what the kernels are tested against."""
import numpy as np
import torch

F8_MAX = 448.0


def philox(counters, seed, offset):
    """Philox4x32-10 of Salmon, Moraes, Dror and Shaw (2011): four 32-bit words for each 64-bit counter, as uint64."""
    low, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [counters & low, counters >> shift, np.full_like(counters, offset & 0xFFFFFFFF), np.full_like(counters, offset >> 32)]
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> shift) ^ c[1] ^ np.uint64(key[0]), b & low, (a >> shift) ^ c[3] ^ np.uint64(key[1]), a & low]
        key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1)


def kept(shape, p, seed, offset):
    """1 / (share that is kept) for elements that stay, 0 for the others."""
    n = int(np.prod(shape))
    words = philox(np.arange((n + 7) // 8, dtype=np.uint64), seed, offset)
    bits = np.stack((words & np.uint64(0xFFFF), words >> np.uint64(16)), 2).reshape(-1)[:n]
    below = int(np.floor(p * 65536 + 0.5))
    factor = 65536 / (65536 - below) if below < 65536 else 0.0
    return torch.from_numpy(np.where(bits >= below, factor, 0.0).reshape(shape))


def dropout(x, p, seed, offset):
    if p == 0:
        return x.double()
    k = kept(tuple(x.shape), p, seed, offset)
    return torch.where(k == 0, 0.0, x.double() * k)


def embedding(ids, weight, scale):
    fits = (ids >= 0) & (ids < weight.shape[0])
    return torch.where(fits[..., None], weight.double()[torch.where(fits, ids, 0).long()] * scale, 0.0)


def embedding_grad(ids, grad, vocab, scale, padding_id=None):
    """The sums, and the sums of their terms' magnitudes."""
    ids, rows = ids.reshape(-1).long(), grad.double().reshape(-1, grad.shape[-1])
    use = (ids >= 0) & (ids < vocab)
    if padding_id is not None:
        use &= ids != padding_id
    total, size = torch.zeros(2, vocab, rows.shape[1], dtype=torch.float64)
    total.index_add_(0, ids[use], rows[use] * scale)
    size.index_add_(0, ids[use], (rows[use] * scale).abs())
    return total, size


def rms_norm(x, weight, eps, residual=None, p=0.0, seed=0, offset=0):
    """y, h, rstd."""
    h = dropout(x, p, seed, offset)
    if residual is not None:
        h = h + residual.double()
    rstd = 1 / torch.sqrt((h * h).mean(-1) + eps)
    y = h * rstd[..., None]
    return y if weight is None else y * weight.double(), h, rstd


def scales_of(y, group):
    """The scale of each group of columns, NaN left out of the largest magnitude."""
    parts = y.split(group or y.shape[-1], -1)
    most = torch.stack([torch.nan_to_num(q.abs(), 0.0, float("inf")).amax(-1) for q in parts], -1)
    return torch.where(most >= 2.0 ** -100, most / F8_MAX, 1.0)


def rms_norm_grad(grad, h, rstd, weight, grad_h=None, p=0.0, seed=0, offset=0):
    """Gradients of x, residual and weight, and the sums of the magnitudes that the last two are made of."""
    g, h, q = grad.double(), h.double(), rstd.double()[..., None]
    gw = g if weight is None else g * weight.double()
    back = h * q ** 3 * (gw * h).mean(-1, keepdim=True)
    dh, size = gw * q - back, (gw * q).abs() + h.abs() * q ** 3 * (gw * h).abs().mean(-1, keepdim=True)
    if grad_h is not None:
        dh, size = dh + grad_h.double(), size + grad_h.double().abs()
    parts = (g * h * q).reshape(-1, h.shape[-1])
    return dropout(dh, p, seed, offset), dh, parts.sum(0), size, parts.abs().sum(0)
