"""The losses where their numbers leave the usual range, and the launches that only certain layouts reach, against the 64-bit oracle.

The bounds are those of test_gpu_losses.py unless a test says otherwise."""
import importlib.util
import math
import os

import pytest
import torch

import test_gpu_losses as tl
from oracle import losses_f64 as of
from test_gpu_layers import BF, F32, U, U32, _near
from test_gpu_losses import losses  # noqa: F401
from test_losses_host import ROOT

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


# ---------------------------------------------------------------------------------------------------------------
# what little the student leaves to the rest
# ---------------------------------------------------------------------------------------------------------------

def _small_rest(rows, vocab, dtype, lift, over):
    """Students whose named tokens stand `lift` above the others, and a teacher that leaves the rest nothing (its values come to more
    than one) or next to nothing (to one, but for roundings)."""
    gen = torch.Generator().manual_seed(vocab + int(lift))
    x = torch.randn(rows, vocab, generator=gen)
    ids = torch.stack([torch.randperm(vocab, generator=gen)[:6] for _ in range(rows)])
    x.scatter_add_(1, ids, torch.full((rows, 6), lift))
    teacher = torch.randn(rows, 6, generator=gen)
    return x.to(dtype), ids, torch.log_softmax(teacher, 1) + (0.5 if over else 0.0)


def _check_small_rest(over, dx, x, ids, teacher, grad, temperature):
    """stats[5] = pr - qr, and the gradient of the tokens that are not named, whose every factor has it.

    pr is exp of a difference of maxima, over T, and two sums' logs, in 64 bits from 32-bit parts: relative to itself it is off by what the two sums
    are, by the rounding of 1 / T times that difference, and by what the named tokens' sum takes in of the others', together at most
    4 u far + 8 u.  qr is one minus six doubles.  Both are rounded together.  A token's share of the rest is off as any p is."""
    t, g = of.t32(temperature), grad.double()[:, None]
    _, stats, dz, _, _ = of.distill_top(x, ids, teacher, temperature, True)
    m, log_s, whole, _ = of.softmax(x, temperature)
    named = torch.zeros(x.shape, dtype=torch.bool).scatter_(1, ids, True)
    others = x.double().masked_fill(named, -INF)
    m_o, log_o, part, _ = of.softmax(others, temperature)
    far = (m - m_o) / t
    pr = (log_o - log_s - far).exp()
    assert bool((torch.where(named, whole, 0.0).sum(1) >= 0.5).all())
    want = stats[:, 5]
    qr = (1 - teacher.double().exp().sum(1)).clamp(min=0.0)
    rel = tl._sum_off(x, whole, m, t) + tl._sum_off(others, part, m_o, t) + U32 * (4 * far + 8)
    off = pr * rel + torch.where(qr > 0, 1e-14, 0.0) + U32 * want.abs()
    _near(over, want, off)
    rel_j = U32 * (4 * tl._distance(others, m_o, t) + 4 * log_o.abs()[:, None] + 10)
    size = part * g.abs() / t
    bound = size * (want.abs()[:, None] * (rel_j + 3 * U32) + off[:, None]) + U[dx.dtype] * (dz * g).abs() + 2.0 ** -120
    rest = ~named
    _near(dx.cpu()[rest], (dz * g)[rest], bound[rest])


SMALL = [(lift, over, t) for lift in (20.0, 35.0, 52.0) for over in (True, False) for t in (1.0, 1.3)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,vocab", [(7, 90), (5, 5003), (2, 70001), (1050, 1501)])
@pytest.mark.parametrize("lift,over,temperature", SMALL)
def test_a_small_rest_keeps_its_digits(losses, dtype, rows, vocab, lift, over, temperature):  # noqa: F811
    x, ids, teacher = _small_rest(rows, vocab, dtype, lift, over)
    got = losses.distill_top(x.cuda(), ids.cuda(), teacher.cuda(), temperature=temperature, rest=True)
    g = tl._gen(rows)
    for out in (BF, F32):
        dx = losses.distill_top_grad(x.cuda(), ids.cuda(), teacher.cuda(), got.stats, g.cuda(), temperature=temperature, dtype=out)
        _check_small_rest(got.stats[:, 5], dx, x, ids, teacher, g, temperature)
        tl._check_distill_grad(dx, x, ids, teacher, g, temperature, True, out)


@pytest.mark.parametrize("lift,pr", [(20.0, 1e-5), (52.0, 1e-19)])
def test_the_check_of_a_small_rest_refuses_one_minus_the_rest(lift, pr):
    """The oracle's own values pass; what one minus the named tokens' share in 32 bits leaves does not."""
    x, ids, teacher = _small_rest(7, 90, F32, lift, True)
    g = tl._gen(7)
    _, stats, dz, _, _ = of.distill_top(x, ids, teacher, 1.0, True)
    dx = (dz * g.double()[:, None]).float()
    assert bool((stats[:, 5] < pr).all())
    _check_small_rest(stats[:, 5].float(), dx, x, ids, teacher, g, 1.0)
    p = torch.softmax(x, 1)
    wrong = 1 - p.gather(1, ids).sum(1)
    with pytest.raises(AssertionError):
        _check_small_rest(wrong, dx, x, ids, teacher, g, 1.0)
    factor = 1 + 1e-3
    with pytest.raises(AssertionError):
        _check_small_rest(stats[:, 5].float(), dx * factor, x, ids, teacher, g, 1.0)


@pytest.mark.gpu
def test_the_examples_mean_is_over_the_targets_that_name_a_token():
    """A target past the vocabulary counts for nothing, as a negative one: neither in the sum nor in what it is divided by."""
    spec = importlib.util.spec_from_file_location("train_tokens", os.path.join(ROOT, "examples", "train_tokens.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    torch.manual_seed(4)
    model = example.Model(0.0)
    target = torch.randint(0, example.VOCAB, (4, 16), device="cuda")
    target[:, -3:] = -100
    got = []
    for other in (-100, example.VOCAB, example.VOCAB + 77):
        rows = torch.randn(4, 16, example.DIM, device="cuda", dtype=BF, generator=torch.Generator(device="cuda").manual_seed(5)).requires_grad_()
        target[:, :5] = other
        loss = model.loss(rows, target, 0)
        got.append((loss.detach(), torch.autograd.grad(loss, rows)[0]))
    assert all(torch.equal(a, b) for other in got[1:] for a, b in zip(got[0], other))


# ---------------------------------------------------------------------------------------------------------------
# launches that rows of certain lengths and places reach
# ---------------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows,vocab", [(BF, 1100, 131072), (F32, 520, 131072), (BF, 2100, 65536), (F32, 2100, 32768)])
def test_even_rows_that_the_caches_do_not_hold(losses, dtype, rows, vocab):  # noqa: F811
    """Rows that all begin on 128 bytes: the gradients run with fewer workgroups to a unit where such rows are long."""
    tl.test_logits_that_the_caches_do_not_hold(losses, dtype, rows, vocab)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,out", [(BF, BF), (F32, F32), (F32, BF), (BF, F32)])
@pytest.mark.parametrize("vocab", [33000, 131072])
def test_gradients_into_rows_that_begin_elsewhere(losses, dtype, out, vocab):  # noqa: F811
    """Past the caches too: the logits begin on 128 bytes, the gradient's rows anywhere."""
    rows = (288 << 20) // (vocab * (2 if dtype == BF else 4)) + 1
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    x = (torch.randn(rows, vocab, generator=gen, device="cuda") * 2).to(dtype)
    ids = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    few = torch.randint(0, vocab, (rows, 9), generator=gen, device="cuda")
    values = torch.log_softmax(torch.randn(rows, 10, generator=gen, device="cuda"), 1)[:, :9].contiguous()
    g, gh = torch.randn(rows, generator=gen, device="cuda"), torch.randn(rows, generator=gen, device="cuda")
    r, d = losses.token_logprobs(x, ids, entropy=True), losses.distill_top(x, few, values, rest=True)
    wide = torch.empty(rows, vocab + 9, dtype=out, device="cuda")
    for call in (lambda **k: losses.token_logprobs_grad(x, ids, r.stats, g, **k), lambda **k: losses.distill_top_grad(x, few, values, d.stats, g, **k),
                 lambda **k: losses.token_logprobs_grad(x, ids, r.stats, g, grad_entropy=gh, entropy=r.entropy, **k)):
        want = call(dtype=out)
        for at in (1, 4):
            wide.fill_(7.0)
            call(out=wide[:, at:at + vocab])
            assert torch.equal(wide[:, at:at + vocab], want)
            assert bool((wide[:, :at] == 7).all()) and bool((wide[:, at + vocab:] == 7).all())
