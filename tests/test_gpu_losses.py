"""The losses' kernels against the 64-bit oracle.

Bounds, with u = 2^-24: a logit's distance to the row's largest is rounded once (u |d|), scaled by log2(e) / T (three roundings:
the product, the constant and T's inverse), and its exponential is at most two units off; the log of it is off by what these come to, 4 u |d| / T + 4 u.
A sum over the row is made of sums of 32 terms, one for each batch of a thread's vectors, rescaled where the maximum grows (4 u each time), and of the
threads' sums in at most 24 additions: with at most vocab / 2048 + 8 batches the sum's relative error is u (4 sum of p |d| / T + 5 (vocab / 2048 + 8) + 64).
A result is rounded once to its type, u |result| or 2^-8 |result|."""
import ctypes as C
import math
import random

import pytest
import torch

from oracle import losses_f64 as of
from test_gpu_layers import BF, F32, U, U32, _near
from test_losses_host import Distill, DistillGrad, Logprobs, LogprobsGrad, _sized

pytestmark = pytest.mark.gpu
INF = math.inf


@pytest.fixture
def losses():
    from eridiffusion_amd import losses
    return losses


def _logits(rows, vocab, dtype, seed=0, masked=0.0, std=3.0):
    g = torch.Generator().manual_seed(rows * 1000003 + vocab * 31 + seed)
    x = torch.randn(rows, vocab, generator=g) * std
    if masked:
        x[torch.rand(rows, vocab, generator=g) < masked] = -INF
    x[:, vocab // 3] = 9.5
    return x.to(dtype)


def _ids(rows, vocab, seed=0, dtype=torch.long):
    ids = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(rows + vocab + seed))
    if rows > 3:
        ids[0], ids[2], ids[3] = vocab - 1, -100, vocab
    return ids.to(dtype)


def _gen(rows, *more, seed=0):
    return torch.randn(rows, *more, generator=torch.Generator().manual_seed(rows * 7 + seed))


def _finite(x):
    return torch.nan_to_num(x, 0.0, 0.0, 0.0)


def _distance(x, m, t):
    """|x - m| / T of the logits that can occur."""
    return _finite((x.double() - m[..., None]).abs() / t)


def _sum_off(x, p, m, t):
    """The relative error of the sum of exp, and so the absolute one of its log."""
    return U32 * (4 * (_finite(p) * _distance(x, m, t)).sum(-1) + 5 * (x.shape[-1] // 2048 + 8) + 64)


def _check_scores(got, x, ids, temperature, top, what=""):
    """A TokenLogprobs against the oracle, on the device of x."""
    t = of.t32(temperature)
    one, h, values, places, m, log_s = of.token_logprobs(x, ids, temperature, top)
    _, _, p, logp = of.softmax(x, temperature)
    off = _sum_off(x, p, m, t)
    log_off = off + 2 * U32 * _finite(log_s.abs())
    _near(got.stats[..., 0], m.cpu(), 0.0, what)
    _near(got.stats[..., 1], log_s.cpu(), log_off.cpu(), what)

    def term(lp):
        # the distance is the log probability and the log of the sum apart: both are rounded
        return 4 * U32 * (_finite(lp.abs()) + _finite(log_s.abs()).reshape(log_s.shape + (1,) * (lp.dim() - log_s.dim())))
    if ids is not None:
        _near(got.logprob, one.cpu(), (term(one) + log_off).cpu(), what)
    if got.entropy is not None:
        d = _distance(x, m, t)
        terms = (_finite(p) * d * (4 * U32 * d)).sum(-1) + (_finite(p) * d).sum(-1) * (off + U32 * (5 * (x.shape[-1] // 2048 + 8) + 64))
        _near(got.entropy, h.cpu(), (log_off + terms + 2 * U32 * _finite(h.abs())).cpu(), what)
    if top:
        assert got.top_ids.dtype == torch.long and torch.equal(got.top_ids.cpu(), places.cpu()), what
        _near(got.top, values.cpu(), (term(values) + log_off[..., None]).cpu(), what)


SHAPES = [(1, 1), (3, 2), (5, 7), (4, 8), (2, 9), (7, 63), (3, 64), (5, 65), (2, 513), (9, 2048), (3, 2049), (2, 4101), (1, 8192), (1, 10007), (600, 4099), (5, 33000), (2, 70001), (67, 66003)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_scores(losses, dtype, rows, vocab):
    for masked, temperature in ((0.0, 1.0), (0.3, 0.7), (0.97, 3.0)):
        x = _logits(rows, vocab, dtype, masked=masked)
        for k, ids in ((0, _ids(rows, vocab)), (min(20, vocab), _ids(rows, vocab, dtype=torch.int32)), (min(64, vocab), None), (1, _ids(rows, vocab, 1))):
            got = losses.token_logprobs(x.cuda(), None if ids is None else ids.cuda(), temperature=temperature, entropy=k != 1, top=k)
            assert (got.logprob is None) == (ids is None) and (got.entropy is None) == (k == 1) and (got.top is None) == (k == 0) == (got.top_ids is None)
            _check_scores(got, x, ids, temperature, k, (masked, temperature, k))


def _odd_rows(vocab, dtype):
    """Rows where a softmax goes wrong, one of each kind."""
    low = torch.finfo(dtype).min
    x = _logits(12, vocab, F32)
    x[0] = -INF
    x[1] = low
    x[2, : vocab - 1] = -INF  # one token left
    x[3, : vocab - 1] = low
    x[4, 0] = math.nan
    x[5, vocab - 1] = INF
    x[6] = 0.25
    x[7] = torch.where(torch.arange(vocab) % 2 == 0, 0.0, -0.0)
    x[8] = x[8] * 1e30
    x[9] = torch.finfo(dtype).max
    x[10] = -1e30
    x[10, vocab // 2] = -1.01e30
    x[11] = torch.where(torch.arange(vocab) % 2 == 0, 1.5e38, -1.5e38)
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab", [2, 13, 500, 2056, 5003, 9000])
@pytest.mark.parametrize("temperature", [1.0, 2.5])
def test_scores_of_masked_infinite_and_nan_logits(losses, dtype, vocab, temperature):
    x, ids = _odd_rows(vocab, dtype), torch.arange(12) % vocab
    for many in (1, 60):  # rows that are cut into slices, and rows that are not
        top = min(64, vocab)
        got = losses.token_logprobs(x.repeat(many, 1).cuda(), ids.repeat(many).cuda(), temperature=temperature, entropy=True, top=top)
        for at in (0, 12 * (many - 1)):
            part = type(got)(*[t[at:at + 12] for t in got])
            _check_scores(part, x, ids, temperature, top, many)
        assert bool((got.entropy[0] == 0).all()) and bool((got.logprob[0] == -INF).all())


@pytest.mark.parametrize("kind", ["few values", "ascending", "descending", "one thread", "many ties", "all equal"])
@pytest.mark.parametrize("rows,vocab", [(1, 65536), (2, 40001), (1100, 32768), (1030, 10007), (3, 2047), (66, 70000), (1, 600011)])
def test_alternatives_of_rows_in_any_order(losses, kind, rows, vocab):
    """Ties go to the lowest id; rows that put many elements above the bound, or all of them with one thread."""
    j = torch.arange(vocab)
    row = {"few values": (j * 7919 % 13).float(), "ascending": j.float() / 8, "descending": -j.float() / 8,
           "one thread": torch.where(j // 8 % 256 == 5, j % 100, -5.0 - j % 3),
           "many ties": torch.where(j // 8 % 256 < 63, 2.0, 1.0), "all equal": torch.full((vocab,), -1.5)}[kind]
    x = row.float().expand(min(rows, 3), vocab).contiguous()
    x[-1] = x[-1].flip(0)
    for dtype in (BF, F32):
        y = x.to(dtype)
        _, places = of.largest(y, 64)
        z = y.cuda()[torch.arange(rows) % len(x)]
        for k in (1, 20, 64):
            got = losses.token_logprobs(z, top=k)
            assert torch.equal(got.top_ids.cpu(), places[torch.arange(rows) % len(x), :k]), (dtype, k)
        _check_scores(type(got)(*[None if t is None else t[: len(x)] for t in got]), y[:rows], None, 1.0, 64, dtype)


def _check_token_grad(got, x, ids, grad, grad_entropy, temperature, what=""):
    t = of.t32(temperature)
    want, p, logp = of.token_logprobs_grad(x, ids, grad, grad_entropy, temperature)
    m, log_s = of.softmax(x, temperature)[:2]
    _, h = of.token_logprobs(x, None, temperature)[:2]
    lp, log_s, h = _finite(logp.abs()), _finite(log_s.abs())[..., None], _finite(h.abs())[..., None]
    rel = U32 * (4 * _distance(x, m, t) + 4 * log_s + 10)  # of p: its log's parts, rounded statistics, the exponential and three products
    size = _finite(p) * ((grad.double().abs() if ids is not None else torch.zeros_like(grad).double())[..., None]) / t
    off = size * rel
    if grad_entropy is not None:
        gh = grad_entropy.double().abs()[..., None] / t
        off = off + _finite(p) * gh * ((lp + h) * rel + U32 * (4 * _distance(x, m, t) + 4 * log_s + 4 * lp + 4 * h))
    # next to its token both parts count: the sum of two rounded ones
    off = off + 3 * U32 * (want.abs() + (grad.double().abs()[..., None] / t if ids is not None else 0.0) * (torch.arange(x.shape[-1], device=x.device) == (
        ids[..., None] if ids is not None else -1)))
    _near(got, want.cpu(), (U[got.dtype] * _finite(want.abs()) + _finite(off)).cpu() + 2.0 ** -120, what)




@pytest.mark.parametrize("dtype,out", [(BF, BF), (BF, F32), (F32, F32), (F32, BF)])
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_scores_gradient(losses, dtype, out, rows, vocab):
    for masked, temperature in ((0.0, 1.0), (0.5, 0.7)):
        x, ids, g, gh = _logits(rows, vocab, dtype, masked=masked), _ids(rows, vocab), _gen(rows), _gen(rows, seed=1)
        ids = torch.where((ids >= 0) & (ids < vocab) & x.float().gather(1, ids.clamp(0, vocab - 1)[:, None]).squeeze(1).isinf(), vocab // 3, ids)
        g[-1], gh[rows // 2] = 0.0, 0.0
        r = losses.token_logprobs(x.cuda(), ids.cuda(), temperature=temperature, entropy=True)
        for e, i, w in ((None, ids, g), (gh, ids.int(), g), (gh, None, torch.zeros(rows))):
            given = dict(grad_entropy=None if e is None else e.cuda(), entropy=None if e is None else r.entropy, temperature=temperature)
            i_, w_ = (None, None) if i is None else (i.cuda(), w.cuda())
            got = losses.token_logprobs_grad(x.cuda(), i_, r.stats, w_, dtype=out, **given)
            assert got.dtype == out
            _check_token_grad(got, x, i, w, e, temperature, (masked, e is None, i is None))
            if out == dtype:
                y = x.cuda()
                assert losses.token_logprobs_grad(y, i_, r.stats, w_, out=y, **given) is y and torch.equal(y, got)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab", [13, 2056, 9000])
def test_scores_gradient_of_masked_infinite_and_nan_logits(losses, dtype, vocab):
    x, ids, g, gh = _odd_rows(vocab, dtype), torch.arange(12) % vocab, _gen(12), _gen(12, seed=1)
    ids[0], ids[2], ids[3] = 5, vocab - 1, vocab - 1
    r = losses.token_logprobs(x.cuda(), ids.cuda(), entropy=True)
    for e in (None, gh):
        got = losses.token_logprobs_grad(x.cuda(), ids.cuda(), r.stats, g.cuda(), grad_entropy=None if e is None else e.cuda(), entropy=None if e is None else r.entropy, dtype=F32)
        _check_token_grad(got, x, ids, g, e, 1.0, e is None)
    assert bool((got[0] == 0).all()) and bool(got[4].isnan().all()) and bool(got[5].isnan().all())
    zero = losses.token_logprobs_grad(x.cuda(), torch.full((12,), -1).cuda(), r.stats, g.cuda())
    assert bool((zero == 0).all())  # rows of NaN too: nothing is asked of them


# ---------------------------------------------------------------------------------------------------------------
# distillation
# ---------------------------------------------------------------------------------------------------------------

def _teacher(rows, vocab, k, dtype=F32, seed=0, temperature=1.0):
    """k distinct tokens and their log probabilities."""
    g = torch.Generator().manual_seed(rows * 13 + vocab + k + seed)
    full = torch.log_softmax(torch.randn(rows, vocab, generator=g) * 3 / temperature, 1)
    values, ids = full.topk(k, 1)
    return ids, values.to(dtype)


def _check_distill(got, x, ids, teacher, temperature, rest, what=""):
    t = of.t32(temperature)
    loss, stats, _, p, q = of.distill_top(x, ids, teacher, temperature, rest)
    m, log_s, whole, _ = of.softmax(x, temperature)
    off = _sum_off(x, whole, m, t)
    # the others' sum is over a part of the row, against its own maximum
    fits = (ids >= 0) & (ids < x.shape[-1])
    named = torch.zeros(x.shape, dtype=torch.float64, device=x.device).scatter_add_(-1, torch.where(fits, ids, 0).long(), fits.double()) > 0
    others = x.double().masked_fill(named, -INF)
    m_o, _, part, _ = of.softmax(others, temperature)
    off_o = _sum_off(others, part, m_o, t)
    lp = _finite(torch.where(q > 0, p, 1.0).log().abs())
    far = _finite((m - m_o).abs() / t)
    # each term's log: the sum's error, its distance times the rounded inverse of T, and the share of the rest: what is held, or what is left
    bound = off + (_finite(q) * 2 * U32 * lp).sum(-1) + 3 * (off + off_o + U32 * (4 * far + 8)) + U32 * _finite(loss.abs())
    _near(got.loss, loss.cpu(), bound.cpu(), what)
    _near(got.stats[..., 0], stats[..., 0].cpu(), 0.0, what)
    _near(got.stats[..., 1], stats[..., 1].cpu(), (off + U32 * _finite(stats[..., 1].abs())).cpu(), what)
    _near(got.stats[..., 2], stats[..., 2].cpu(), 0.0, what)
    _near(got.stats[..., 3], stats[..., 3].cpu(), (off + off_o + U32 * _finite(stats[..., 3].abs())).cpu(), what)
    _near(got.stats[..., 4], stats[..., 4].cpu(), U32 * _finite(stats[..., 4].abs()).cpu() + 1e-12, what)
    _near(got.stats[..., 5], stats[..., 5].cpu(), (U32 * _finite(stats[..., 5].abs()) + 2 * (off + off_o + U32 * (4 * far + 8))).cpu(), what)


def _check_distill_grad(got, x, ids, teacher, grad, temperature, rest, what=""):
    t, g = of.t32(temperature), grad.double()[..., None]
    _, stats, dx, p, q = of.distill_top(x, ids, teacher, temperature, rest)
    want = torch.where(g == 0, 0.0, dx * g)
    m, log_s, whole, _ = of.softmax(x, temperature)
    fits = (ids >= 0) & (ids < x.shape[-1])
    at = torch.where(fits, ids, 0).long()
    named = torch.zeros(x.shape, dtype=torch.float64, device=x.device).scatter_add_(-1, at, fits.double()) > 0
    rel = U32 * (4 * _distance(x, m, t) + 4 * _finite(log_s.abs())[..., None] + 10)
    # the others: their share, and the difference that it is multiplied by, which the forward pass has to within a few sums' errors
    m_o, log_o = stats[..., 2], stats[..., 3]
    share = torch.where(named, 0.0, _finite(torch.exp((x.double() - m_o[..., None]) / t - log_o[..., None])))
    rel_o = U32 * (4 * _distance(x, m_o, t) + 4 * _finite(log_o.abs())[..., None] + 10)
    far = _finite((m - m_o).abs() / t)
    over_off = 2 * (_sum_off(x, whole, m, t) + _sum_off(x.double().masked_fill(named, -INF), torch.where(named, 0.0, _finite(share)), m_o, t) + U32 * (4 * far + 8))
    off = share * (rel_o * _finite(stats[..., 5].abs())[..., None] + over_off[..., None])
    q_off = torch.zeros_like(off).scatter_add_(-1, at, torch.where(fits, _finite(q) * U32 * (4 * _finite(teacher.double().abs()) + 4 * _finite(stats[..., 4].abs())[..., None] + 70), 0.0))
    off = torch.where(named, _finite(whole) * rel + q_off, off) * g.abs() / t
    _near(got, want.cpu(), (U[got.dtype] * _finite(want.abs()) + 3 * U32 * _finite(want.abs()) + _finite(off)).cpu() + 2.0 ** -120, what)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,vocab", [s for s in SHAPES if s != (1, 1)] + [(530, 5000)])
@pytest.mark.parametrize("rest", [False, True])
def test_distillation_and_its_gradient(losses, dtype, rows, vocab, rest):
    for k, kind, temperature, masked in ((1, F32, 1.0, 0.0), (min(20, vocab - 1), F32, 2.0, 0.0), (min(64, vocab), BF, 0.7, 0.0), (min(5, vocab), F32, 1.0, 0.6)):
        x = _logits(rows, vocab, dtype, masked=masked)
        ids, teacher = _teacher(rows, vocab, k, kind, temperature=temperature)
        if k == 5:
            ids = ids.int()
        got = losses.distill_top(x.cuda(), ids.cuda(), teacher.cuda(), temperature=temperature, rest=rest)
        _check_distill(got, x, ids, teacher, temperature, rest, (k, masked))
        g = _gen(rows)
        g[rows // 2] = 0.0
        for out in (BF, F32):
            dx = losses.distill_top_grad(x.cuda(), ids.cuda(), teacher.cuda(), got.stats, g.cuda(), temperature=temperature, dtype=out)
            _check_distill_grad(dx, x, ids, teacher, g, temperature, rest, (k, masked, out))
            if out == dtype:
                y = x.cuda()
                assert losses.distill_top_grad(y, ids.cuda(), teacher.cuda(), got.stats, g.cuda(), temperature=temperature, out=y) is y and torch.equal(y, dx)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab", [13, 700, 2056, 9000])
@pytest.mark.parametrize("rest", [False, True])
def test_distillation_at_its_edges(losses, dtype, vocab, rest):
    """Entries that name no token, the same token twice, a teacher that leaves nothing, that sums to more than one, that holds NaN;
    students without a rest, without anything, with NaN."""
    x = _logits(16, vocab, dtype, std=1.0)
    ids, teacher = _teacher(16, vocab, 6)
    ids[0, 2], ids[0, 5], ids[0, 0] = -1, vocab, -100
    ids[1, 1] = ids[1, 4] = ids[1, 0]
    ids[2] = -1
    teacher[3] = -INF
    teacher[4, 2] = -INF
    teacher[5] = torch.tensor([3.0, 2.5, 1.0, 0.0, -1.0, -8.0])
    teacher[6, 1] = math.nan
    keep = torch.zeros(vocab, dtype=torch.bool)
    keep[ids[7]] = True
    x[7, ~keep] = -INF
    x[8] = -INF
    x[9, 3] = math.nan
    x[10, ids[10, 1]] = -INF  # the teacher gives it something
    x[11, ids[11, 5]], teacher[11, 5] = -INF, -INF  # and here nothing
    x[12] = torch.finfo(dtype).min
    x[13, ids[13]] = 60.0  # the rest is far below what fp32 has beside one
    x[14, ids[14]] = -60.0
    x[15, vocab - 1] = INF
    for many in (1, 40):
        xx, ii, tt = x.repeat(many, 1), ids.repeat(many, 1), teacher.repeat(many, 1)
        got = losses.distill_top(xx.cuda(), ii.cuda(), tt.cuda(), rest=rest)
        g = _gen(16).abs() + 0.1
        dx = losses.distill_top_grad(xx.cuda(), ii.cuda(), tt.cuda(), got.stats, g.repeat(many).cuda(), dtype=F32)
        for at in (0, 16 * (many - 1)):
            for row in range(16):  # so that a row's name stands in the failure
                s, one = slice(at + row, at + row + 1), slice(row, row + 1)
                _check_distill(type(got)(got.loss[s], got.stats[s]), x[one], ids[one], teacher[one], 1.0, rest, row)
                _check_distill_grad(dx[s], x[one], ids[one], teacher[one], g[one], 1.0, rest, row)
    assert bool((dx[8] == 0).all()) and (rest or bool((dx[2] == 0).all())) and bool(dx[9].isnan().any())


def test_distillation_over_several_segments_of_a_row(losses):
    """More vectors than a thread has bits for, in rows that are not cut; tokens at every end."""
    for dtype, vocab in ((BF, 262147), (F32, 131080)):
        rows, k = 515, 64
        g = torch.Generator(device="cuda").manual_seed(5)
        x = (torch.randn(rows, vocab, generator=g, device="cuda") * 2).to(dtype)
        ids = torch.randint(0, vocab, (rows, k), generator=g, device="cuda")
        ids[:, :6] = torch.tensor([0, vocab - 1, 131071, 131072, 131079, 8], device="cuda")
        teacher = torch.log_softmax(torch.randn(rows, k + 1, generator=g, device="cuda"), 1)[:, :k].contiguous()
        got = losses.distill_top(x, ids, teacher, temperature=1.5, rest=True)
        w = torch.rand(rows, generator=g, device="cuda")
        dx = losses.distill_top_grad(x, ids, teacher, got.stats, w, temperature=1.5)
        for at in (0, 200, rows - 4):
            s = slice(at, at + 4)
            _check_distill(type(got)(got.loss[s], got.stats[s]), x[s], ids[s], teacher[s], 1.5, True, at)
            _check_distill_grad(dx[s], x[s], ids[s], teacher[s], w[s], 1.5, True, at)


def test_small_divergences_are_not_lost(losses):
    """A teacher and a student that agree, both nearly flat: the loss is far below its terms, and the others' gradient far below their share."""
    vocab, t = 50000, 4.0
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(40, vocab, generator=g, device="cuda")
    near = x + 0.05 * torch.randn(40, vocab, generator=g, device="cuda")
    r = losses.token_logprobs(near, temperature=t, top=20)
    got = losses.distill_top(x, r.top_ids, r.top, temperature=t, rest=True)
    want, stats, dx, _, _ = of.distill_top(x, r.top_ids, r.top, t, True)
    held = r.top.double().exp().sum(1)
    # of the order of 1e-7; the errors are those of numbers of the size of what the named tokens hold, 1e-3, and not of one
    assert bool((want < 1e-5).all()) and bool((held < 5e-3).all())
    off = _sum_off(x, of.softmax(x, t)[2], x.double().amax(1), t)
    _near(got.loss, want.cpu(), (4 * held * (off + 8 * U32)).cpu())
    _near(got.stats[:, 5], stats[:, 5].cpu(), (2 * held * (off + 8 * U32)).cpu())


# ---------------------------------------------------------------------------------------------------------------
# layouts, streams, autograd
# ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab", [50, 2053, 5001])
def test_rows_with_gaps_and_other_layouts(losses, dtype, vocab):
    whole = torch.randn(30, vocab + 21, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    for at in (0, 1, 3, 8):
        x, ids = whole[:, at:at + vocab], _ids(30, vocab).cuda()
        want = losses.token_logprobs(x.contiguous(), ids, entropy=True, top=9)
        got = losses.token_logprobs(x, ids, entropy=True, top=9)  # rows that begin elsewhere are summed in another order
        _check_scores(got, x.cpu(), ids.cpu(), 1.0, 9, at)
        assert torch.equal(got.top_ids, want.top_ids)
        g, gh = _gen(30).cuda(), _gen(30, seed=1).cuda()
        dx = losses.token_logprobs_grad(x.contiguous(), ids, got.stats, g, grad_entropy=gh, entropy=got.entropy)
        back = whole.clone()
        rows = back[:, at:at + vocab]
        losses.token_logprobs_grad(rows, ids, got.stats, g, grad_entropy=gh, entropy=got.entropy, out=rows)
        assert torch.equal(rows, dx)
        rows.copy_(x)
        assert torch.equal(back, whole)  # nothing beside the rows
        few, values = want.top_ids, want.top
        wide_ids, wide = torch.full((30, 12), -1, device="cuda"), torch.zeros(30, 14, device="cuda")
        wide_ids[:, 2:11], wide[:, 5:] = few, values
        d = losses.distill_top(x, wide_ids[:, 2:11], wide[:, 5:], rest=True)
        _check_distill(d, x.cpu(), few.cpu(), values.cpu(), 1.0, True, at)
        dx = losses.distill_top_grad(x.contiguous(), few, values, d.stats, g)
        back = whole.clone()
        rows = back[:, at:at + vocab]
        losses.distill_top_grad(rows, wide_ids[:, 2:11], wide[:, 5:], d.stats, g, out=rows)
        assert torch.equal(rows, dx)
        rows.copy_(x)
        assert torch.equal(back, whole)
    x = whole[:24, :vocab].reshape(2, 3, 4, vocab)
    ids = _ids(24, vocab).view(2, 3, 4).cuda()
    flat = losses.token_logprobs(x.reshape(24, vocab), ids.reshape(24), entropy=True, top=3)
    for y, i in ((x, ids), (x.transpose(0, 2), ids.transpose(0, 2))):  # rows at any distances, ids in any order
        got = losses.token_logprobs(y, i, entropy=True, top=3)
        assert got.top.shape == y.shape[:-1] + (3,) and got.stats.shape == y.shape[:-1] + (2,)
        back = (lambda t: t.transpose(0, 2) if y is not x else t)
        assert torch.equal(back(got.top_ids).reshape(24, 3), flat.top_ids)
        _check_scores(type(got)(*[back(p).reshape(f.shape) for p, f in zip(got, flat)]), x.reshape(24, vocab).cpu(), ids.reshape(24).cpu(), 1.0, 3)
        d = losses.distill_top(y, got.top_ids, got.top)
        _check_distill(type(d)(back(d.loss).reshape(24), back(d.stats).reshape(24, 6)), x.reshape(24, vocab).cpu(), back(got.top_ids).reshape(24, 3).cpu(),
                       back(got.top).reshape(24, 3).cpu(), 1.0, False)
    t = whole[:, :30].float().t()  # columns as rows: copied first
    assert torch.equal(losses.token_logprobs(t, top=2).top, losses.token_logprobs(t.contiguous(), top=2).top)
    one = losses.token_logprobs(whole[0, :vocab], torch.tensor(3, device="cuda"))
    assert one.logprob.shape == () and one.stats.shape == (2,)
    few, row = got.top_ids.reshape(24, 3)[0], got.top.reshape(24, 3)[0]
    shared = losses.distill_top(x.reshape(24, vocab), few.expand(24, 3), row.expand(24, 3))  # one teacher for all
    assert torch.equal(shared.loss, losses.distill_top(x.reshape(24, vocab), few.expand(24, 3).contiguous(), row.expand(24, 3).contiguous()).loss)


def test_no_rows(losses):
    x, none = torch.zeros(0, 40, device="cuda"), torch.zeros(0, dtype=torch.long, device="cuda")
    r = losses.token_logprobs(x, none, entropy=True, top=4)
    assert r.logprob.shape == (0,) and r.top.shape == (0, 4)
    assert losses.token_logprobs_grad(x, none, r.stats, r.logprob).shape == (0, 40)
    d = losses.distill_top(x, r.top_ids, r.top)
    assert losses.distill_top_grad(x, r.top_ids, r.top, d.stats, d.loss, out=x) is x


def test_past_32_bit_offsets(losses):
    rows, vocab = 33000, 131072  # 2^32 elements and more
    x = torch.zeros(rows, vocab, dtype=BF, device="cuda")
    some = torch.tensor([0, 1, 16383, 16384, 32767, 32768, rows - 1], device="cuda")
    x[some] = _logits(7, vocab, BF).cuda()
    ids = torch.full((rows,), 3, device="cuda")
    ids[some] = _ids(7, vocab).cuda()
    r = losses.token_logprobs(x, ids, entropy=True, top=8)
    y, i = x[some], ids[some]
    _check_scores(type(r)(*[t[some] for t in r]), y, i, 1.0, 8)
    assert bool((r.top_ids[5:16000] == torch.arange(8, device="cuda")).all())
    few, values = _teacher(7, vocab, 10)
    teacher_ids, teacher = torch.zeros(rows, 10, dtype=torch.long, device="cuda"), torch.full((rows, 10), -INF, device="cuda")
    teacher_ids[some], teacher[some] = few.cuda(), values.cuda()
    d = losses.distill_top(x, teacher_ids, teacher, rest=True)
    _check_distill(type(d)(d.loss[some], d.stats[some]), y, few.cuda(), values.cuda(), 1.0, True)
    g = torch.zeros(rows, device="cuda")
    g[some] = _gen(7).cuda()
    dx = losses.distill_top_grad(x, teacher_ids, teacher, d.stats, g)
    _check_distill_grad(dx[some], y, few.cuda(), values.cuda(), g[some], 1.0, True)
    g[16000] = 1.0
    losses.token_logprobs_grad(x, ids, r.stats, g, out=x)
    _check_token_grad(x[some], y, i, g[some], None, 1.0)
    assert float(x[16000, 3]) == pytest.approx(1.0, abs=2 ** -7) and float(x[16000, 4]) == pytest.approx(-1 / vocab, rel=2 ** -7)
    assert int((x[:16000] != 0).any(1).sum()) == 2


@pytest.mark.parametrize("dtype,rows,vocab", [(BF, 140001, 1001), (BF, 70001, 2507), (BF, 36000, 5003), (BF, 20001, 7003), (BF, 1100, 131071), (F32, 70001, 1003),
                                              (F32, 33001, 2100), (F32, 2100, 33333), (F32, 500, 140003)])
def test_logits_that_the_caches_do_not_hold(losses, dtype, rows, vocab):
    """More than 256 MB, in rows of all the lengths that are dealt with differently."""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    x = (torch.randn(rows, vocab, generator=gen, device="cuda") * 2).to(dtype)
    assert x.numel() * x.element_size() > 2 ** 28
    ids = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    few = torch.randint(0, vocab, (rows, 9), generator=gen, device="cuda")
    values = torch.log_softmax(torch.randn(rows, 10, generator=gen, device="cuda"), 1)[:, :9].contiguous()
    g, gh = torch.randn(rows, generator=gen, device="cuda"), torch.randn(rows, generator=gen, device="cuda")
    parts = [slice(at, at + 3) for at in (0, rows // 2, rows - 3)]
    for top, entropy in ((0, True), (7, False), (50, True)):
        r = losses.token_logprobs(x, ids, entropy=entropy, top=top)
        for s in parts:
            _check_scores(type(r)(*[None if t is None else t[s] for t in r]), x[s], ids[s], 1.0, top, (top, s))
    for rest in (False, True):
        d = losses.distill_top(x, few, values, rest=rest)
        for s in parts:
            _check_distill(type(d)(d.loss[s], d.stats[s]), x[s], few[s], values[s], 1.0, rest, s)
        for out in (BF, F32):
            dx = losses.distill_top_grad(x, few, values, d.stats, g, dtype=out)
            for s in parts:
                _check_distill_grad(dx[s], x[s], few[s], values[s], g[s], 1.0, rest, (out, s))
    for e in (None, gh):
        given = dict(grad_entropy=e, entropy=None if e is None else r.entropy)
        for out in (BF, F32):
            dx = losses.token_logprobs_grad(x, ids, r.stats, g, dtype=out, **given)
            for s in parts:
                _check_token_grad(dx[s], x[s], ids[s], g[s], None if e is None else e[s], 1.0, (out, s))
    whole = losses.token_logprobs_grad(x, ids, r.stats, g)
    losses.token_logprobs_grad(x, ids, r.stats, g, out=x)
    assert torch.equal(x, whole)


@pytest.mark.parametrize("seed", range(24))
def test_any_sizes_and_places(losses, seed):
    """Rows of any length that begin anywhere, all calls on one batch."""
    rng = random.Random(seed)
    dtype, out = rng.choice([BF, F32]), rng.choice([BF, F32])
    vocab = round(math.exp(rng.uniform(math.log(1), math.log(90000))))
    rows = max(1, min(round(math.exp(rng.uniform(0, math.log(3000)))), 6000000 // vocab))
    gap, at, t, rest = rng.choice([0, 1, 7, 64]), rng.choice([0, 1, 2, 5, 8, 33]), rng.choice([1.0, 0.6, 2.5]), rng.random() < 0.5
    gen = torch.Generator(device="cuda").manual_seed(seed)
    flat = (torch.randn(rows * (vocab + gap) + at, generator=gen, device="cuda") * 3).to(dtype)
    flat[torch.rand(flat.shape, generator=gen, device="cuda") < rng.choice([0.0, 0.4, 0.95])] = -INF
    x = flat[at:].as_strided((rows, vocab), (vocab + gap, 1))
    ids = torch.randint(-1, vocab + 1, (rows,), generator=gen, device="cuda")
    top, k = rng.randint(0, min(64, vocab)), rng.randint(1, 64)
    r = losses.token_logprobs(x, ids, temperature=t, entropy=True, top=top)
    _check_scores(r, x, ids, t, top)
    ids[(r.logprob == -INF)] = -100
    g, gh = torch.randn(rows, generator=gen, device="cuda"), torch.randn(rows, generator=gen, device="cuda")
    _check_token_grad(losses.token_logprobs_grad(x, ids, r.stats, g, grad_entropy=gh, entropy=r.entropy, temperature=t, dtype=out), x, ids, g, gh, t)
    few = torch.randint(-1, vocab + 1, (rows, k), generator=gen, device="cuda")  # some of them twice
    teacher = (torch.log_softmax(torch.randn(rows, k + 1, generator=gen, device="cuda") * 2, 1)[:, :k]).to(rng.choice([BF, F32]))
    d = losses.distill_top(x, few, teacher, temperature=t, rest=rest)
    _check_distill(d, x, few, teacher, t, rest)
    _check_distill_grad(losses.distill_top_grad(x, few, teacher, d.stats, g, temperature=t, dtype=out), x, few, teacher, g, t, rest)


def test_the_longest_row(losses):
    """2^31 - 1 columns: places that just fit.  Equal logits but for a few: the sums of powers of two are exact."""
    vocab = 2 ** 31 - 1
    x = torch.full((1, vocab), -5.0, dtype=BF, device="cuda")
    peaks = {0: 3.0, 7: 2.0, 2 ** 20 + 3: 2.0, 2 ** 30: 4.0, vocab - 2: 2.0, vocab - 1: 5.0}
    for col, v in peaks.items():
        x[0, col] = v
    order = [vocab - 1, 2 ** 30, 0, 7, 2 ** 20 + 3, vocab - 2, 1, 2]
    total = sum(math.exp(v + 5.0) for v in peaks.values()) + vocab - len(peaks)  # in units of a peak-less token
    r = losses.token_logprobs(x, torch.tensor([vocab - 1], device="cuda"), entropy=True, top=8)
    assert r.top_ids[0].tolist() == order
    lp = lambda v: v + 5.0 - math.log(total)  # noqa: E731
    want = [lp(peaks.get(c, -5.0)) for c in order]
    # 2^31 terms: a thread's 2^21 are added 32 at a time, half a unit lost each time at most
    near = 2 ** 16 * U32 + 64 * U32
    assert all(abs(a - b) < near for a, b in zip(r.top[0].tolist(), want)) and abs(r.logprob.item() - lp(5.0)) < near
    entropy = -sum(math.exp(lp(v)) * lp(v) for v in peaks.values()) - (vocab - len(peaks)) * math.exp(lp(-5.0)) * lp(-5.0)
    assert abs(r.entropy.item() - entropy) < 30 * near
    few, q = torch.tensor([[vocab - 1, 0, 2 ** 30]], device="cuda"), torch.tensor([[0.5, 0.25, 0.125]], device="cuda").log()
    d = losses.distill_top(x, few, q, rest=True)
    p = [math.exp(lp(v)) for v in (5.0, 3.0, 4.0)]
    loss = sum(w * (math.log(w) - math.log(v)) for w, v in zip((0.5, 0.25, 0.125), p)) + 0.125 * (math.log(0.125) - math.log1p(-sum(p)))
    assert abs(d.loss.item() - loss) < 4 * near
    cols = torch.tensor([0, 1, 7, 2 ** 20 + 3, 2 ** 30, 2 ** 30 + 1, vocab - 2, vocab - 1], device="cuda")
    one = torch.ones(1, device="cuda")
    dx = losses.distill_top_grad(x, few, q, d.stats, one)[0, cols].tolist()
    others = (1 - sum(p) - 0.125) / (1 - sum(p))
    named = dict(zip(few[0].tolist(), zip(p, (0.5, 0.25, 0.125))))
    for col, got in zip(cols.tolist(), dx):
        pj = math.exp(lp(peaks.get(col, -5.0)))
        exact = named[col][0] - named[col][1] if col in named else pj * others
        assert abs(got - exact) < abs(exact) * (U[BF] + 8 * near), col
    losses.token_logprobs_grad(x, torch.tensor([vocab - 1], device="cuda"), r.stats, one, out=x)
    for col, got in zip(cols.tolist(), x[0, cols].tolist()):
        exact = (1.0 if col == vocab - 1 else 0.0) - math.exp(lp(peaks.get(col, -5.0)))
        assert abs(got - exact) < abs(exact) * (U[BF] + 8 * near), col


def _steps(losses, x, near, ids, g):
    r = losses.token_logprobs(x, ids, temperature=1.5, entropy=True, top=12)
    teacher = losses.token_logprobs(near, temperature=1.5, top=12)
    d = losses.distill_top(x, teacher.top_ids, teacher.top, temperature=1.5, rest=True)
    return (*r, *d, losses.token_logprobs_grad(x, ids, r.stats, g, grad_entropy=g, entropy=r.entropy, temperature=1.5),
            losses.distill_top_grad(x, teacher.top_ids, teacher.top, d.stats, g, temperature=1.5))


@pytest.mark.parametrize("rows,vocab", [(2, 70003), (700, 5003), (90, 500)])
def test_together_on_another_stream_captured_and_replayed(losses, rows, vocab):
    """A teacher's run, both losses and both gradients, as they follow each other in a training step; twice in one graph, so that two
    sets of workspaces live side by side, and with the program's own work between the replays."""
    x, near, ids, g = _logits(rows, vocab, BF).cuda(), _logits(rows, vocab, F32, seed=1).cuda(), _ids(rows, vocab).cuda(), _gen(rows).cuda()
    want = [t.clone() for t in _steps(losses, x, near, ids, g)]
    assert all(torch.equal(a, b) for a, b in zip(want, _steps(losses, x, near, ids, g)))  # the same bits
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _steps(losses, x, near, ids, g)
        s.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            first = _steps(losses, x, near, ids, g)
            second = _steps(losses, x, near, ids, g)
    for k in range(4):
        x.copy_(x.roll(1, 1))
        near.mul_(1.1)
        g.mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        kept = [[t.clone() for t in part] for part in (first, second)]
        torch.cuda.synchronize()
        want = _steps(losses, x, near, ids, g)
        for part in kept:
            assert all(torch.equal(a, b) for a, b in zip(part, want)), k


@pytest.mark.parametrize("rows,vocab", [(6, 40), (5, 2500)])
def test_autograd_is_the_backward_call(losses, rows, vocab):
    x, ids = _logits(rows, vocab, BF).cuda().requires_grad_(), _ids(rows, vocab).cuda()
    few, values = (t.cuda() for t in _teacher(rows, vocab, 7))
    g, gh = _gen(rows).cuda(), _gen(rows, seed=1).cuda()
    r = losses.token_logprobs(x, ids, temperature=0.5, entropy=True, top=3)
    assert not r.top.requires_grad and not r.stats.requires_grad and r.logprob.requires_grad and r.entropy.requires_grad
    y = x.detach()

    def back(*parts):
        x.grad = None
        sum((a * b).sum() for a, b in parts).backward(retain_graph=True)
        return x.grad
    call = lambda *a, **k: losses.token_logprobs_grad(y, *a, temperature=0.5, **k)  # noqa: E731
    assert torch.equal(back((r.logprob, g), (r.entropy, gh)), call(ids, r.stats, g, grad_entropy=gh, entropy=r.entropy.detach()))
    assert torch.equal(back((r.logprob, g)), call(ids, r.stats, g))
    assert torch.equal(back((r.entropy, gh)), call(None, r.stats, None, grad_entropy=gh, entropy=r.entropy.detach()))
    for rest in (False, True):
        d = losses.distill_top(x, few, values, temperature=0.5, rest=rest)
        assert torch.equal(back((d.loss, g)), losses.distill_top_grad(y, few, values, d.stats, g, temperature=0.5)) and not d.stats.requires_grad
    # the mean of a batch: one gradient for all rows, which autograd hands over as a broadcast one
    x.grad = None
    (-losses.token_logprobs(x, ids).logprob.mean()).backward()
    assert torch.equal(x.grad, losses.token_logprobs_grad(y, ids, losses.token_logprobs(y, ids).stats, torch.full((rows,), -1 / rows, device="cuda")))
    assert not losses.token_logprobs(x, top=3).top.requires_grad  # nothing that has a gradient is asked for
    with torch.no_grad():
        assert not losses.token_logprobs(x, ids).logprob.requires_grad
    with torch.inference_mode():
        losses.token_logprobs(y, ids)
    d = losses.distill_top(x, few, values)
    with torch.no_grad():
        x.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        d.loss.sum().backward()


@pytest.mark.parametrize("rows,vocab", [(3, 70001), (300, 2500)])
def test_a_captured_autograd_pass_replays(losses, rows, vocab):
    x, ids = _logits(rows, vocab, BF).cuda().requires_grad_(), _ids(rows, vocab).cuda()
    few, values = (t.cuda() for t in _teacher(rows, vocab, 7))
    g, gh = _gen(rows).cuda(), _gen(rows, seed=1).cuda()

    def step():
        r = losses.token_logprobs(x, ids, entropy=True)
        d = losses.distill_top(x, few, values, rest=True)
        return torch.autograd.grad([r.logprob, r.entropy, d.loss], [x], [g, gh, g])[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = step()
    for k in range(4):
        with torch.no_grad():
            x.copy_(x.roll(1, 1))
        g.mul_(1.5)
        ids.copy_(ids.roll(1))
        graph.replay()
        torch.cuda.synchronize()
        kept = got.clone()
        torch.cuda.synchronize()
        assert torch.equal(kept, step()), k


def test_two_streams_at_once(losses):
    """Each call has a workspace of its own."""
    inputs = [(_logits(5, 90001, F32, seed=i).cuda(), _ids(5, 90001, i).cuda()) for i in range(2)]
    few, values = (t.cuda() for t in _teacher(5, 90001, 11))
    want = [(losses.token_logprobs(x, ids, entropy=True, top=30), losses.distill_top(x, few, values, rest=True)) for x, ids in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((losses.token_logprobs(*inputs[i], entropy=True, top=30), losses.distill_top(inputs[i][0], few, values, rest=True)))
    torch.cuda.synchronize()
    for i in range(2):
        for pair in got[i]:
            assert all(torch.equal(a, b) for one, other in zip(pair, want[i]) for a, b in zip(one, other))


def test_autograd_against_differences(losses):
    """The chain's gradient against differences of the oracle's forward in 64 bits."""
    x, ids = _logits(5, 300, F32, std=1.0).cuda().requires_grad_(), _ids(5, 300).cuda()
    few, values = (t.cuda() for t in _teacher(5, 300, 9))
    r, d = losses.token_logprobs(x, ids, entropy=True, temperature=2.0), losses.distill_top(x, few, values, rest=True, temperature=2.0)
    (r.logprob.sum() - 0.3 * r.entropy.sum() + 4.0 * d.loss.sum()).backward()

    def loss(z):
        one, h = of.token_logprobs(z, ids, 2.0)[:2]
        return (one.sum() - 0.3 * h.sum() + 4.0 * of.distill_top(z, few, values, 2.0, True)[0].sum()).item()
    step = torch.randn(5, 300, generator=torch.Generator().manual_seed(2), dtype=torch.float64).cuda()
    z, h = x.detach().double(), 1e-5
    want, got = (loss(z + h * step) - loss(z - h * step)) / (2 * h), (x.grad.double() * step).sum().item()
    # 1500 terms, each a few roundings of a gradient whose parts are at most a few units
    assert abs(got - want) < 1e-6 * (x.grad.double() * step).abs().sum().item() + 1e-7


def test_outputs_that_overlap_inputs_are_refused(losses):
    x = torch.zeros(6, 40, device="cuda")
    wide = torch.zeros(6, 90, device="cuda")
    ids, one, few = torch.zeros(6, dtype=torch.long, device="cuda"), torch.zeros(6, device="cuda"), torch.zeros(6, 3, dtype=torch.long, device="cuda")
    r, d = losses.token_logprobs(x, ids), losses.distill_top(x, few, one[:, None].expand(6, 3))
    flat = torch.zeros(1000, device="cuda")
    for what, call in [
            ("logits", lambda: losses.token_logprobs_grad(x[:5], ids[:5], r.stats[:5], one[:5], out=x[1:])),
            ("logits", lambda: losses.token_logprobs_grad(wide[:, :40], ids, r.stats, one, out=wide[:, 39:79])),
            ("logits", lambda: losses.token_logprobs_grad(x.view(BF)[:, :40], ids, r.stats, one, out=x)),
            ("stats", lambda: losses.token_logprobs_grad(x, ids, flat[:12].view(6, 2), one, out=flat[11:251].view(6, 40))),
            ("grad", lambda: losses.token_logprobs_grad(x, ids, r.stats, flat[240:246], out=flat[:250].narrow(0, 5, 240).view(6, 40))),
            ("grad", lambda: losses.distill_top_grad(x, few, one[:, None].expand(6, 3), d.stats, flat[:6], out=flat[:240].view(6, 40))),
            ("teacher", lambda: losses.distill_top_grad(x, few, flat[:18].view(6, 3), d.stats, one, out=flat[10:250].view(6, 40))),
            ("logits", lambda: losses.distill_top_grad(x[1:], few[1:], flat[:15].view(5, 3), d.stats[1:], one[1:], out=x[:5]))]:
        with pytest.raises(ValueError, match="out overlaps " + what):
            call()
    beside = losses.token_logprobs_grad(wide[:, :40], ids, r.stats, one, out=wide[:, 40:80])
    assert beside.data_ptr() == wide[:, 40:80].data_ptr()
    version = x._version
    losses.token_logprobs_grad(x, ids, r.stats, one, out=x)
    assert x._version > version


def test_refusals_on_the_device(losses):
    x, ids, one = torch.zeros(4, 8, device="cuda"), torch.zeros(4, dtype=torch.long, device="cuda"), torch.zeros(4, device="cuda")
    few, values = torch.zeros(4, 3, dtype=torch.long, device="cuda"), torch.zeros(4, 3, device="cuda")
    r, d = losses.token_logprobs(x, ids, entropy=True), losses.distill_top(x, few, values)
    from eridiffusion_amd import EriError
    for error, call in [(TypeError, lambda: losses.token_logprobs(x.half(), ids)), (TypeError, lambda: losses.token_logprobs(x, one)),
                        (ValueError, lambda: losses.token_logprobs(x, ids[:3])), (ValueError, lambda: losses.token_logprobs(x, ids.cpu())),
                        (ValueError, lambda: losses.token_logprobs(x, ids[:, None])), (ValueError, lambda: losses.token_logprobs(x, top=9)),
                        (ValueError, lambda: losses.token_logprobs(x.expand(4, 8).repeat(1, 20), top=65)), (ValueError, lambda: losses.token_logprobs(x, top=-1)),
                        (TypeError, lambda: losses.token_logprobs(x, top=1.5)), (TypeError, lambda: losses.token_logprobs(x, ids, temperature="hot")),
                        (ValueError, lambda: losses.token_logprobs(torch.tensor(1.0, device="cuda"))),
                        (EriError, lambda: losses.token_logprobs(x, ids, temperature=0.0)), (EriError, lambda: losses.token_logprobs(x, ids, temperature=math.nan)),
                        (EriError, lambda: losses.token_logprobs(x[:, :0], ids)),
                        (ValueError, lambda: losses.token_logprobs_grad(x, ids, r.stats, None)), (ValueError, lambda: losses.token_logprobs_grad(x, None, r.stats, one)),
                        (ValueError, lambda: losses.token_logprobs_grad(x, None, r.stats, None)),
                        (ValueError, lambda: losses.token_logprobs_grad(x, ids, r.stats, one, grad_entropy=one)),
                        (ValueError, lambda: losses.token_logprobs_grad(x, ids, d.stats, one)), (ValueError, lambda: losses.token_logprobs_grad(x, ids, r.stats.bfloat16(), one)),
                        (ValueError, lambda: losses.token_logprobs_grad(x, ids, r.stats, one.bfloat16())), (ValueError, lambda: losses.token_logprobs_grad(x, ids, r.stats, one[:3])),
                        (TypeError, lambda: losses.token_logprobs_grad(x, ids, r.stats, one, dtype=torch.float16)),
                        (ValueError, lambda: losses.token_logprobs_grad(x, ids, r.stats, one, out=x[:3])),
                        (ValueError, lambda: losses.token_logprobs_grad(x, ids, r.stats, one, dtype=BF, out=torch.zeros_like(x))),
                        (ValueError, lambda: losses.token_logprobs_grad(x, ids, r.stats, one, out=torch.zeros(8, 4, device="cuda").t())),
                        (ValueError, lambda: losses.distill_top(x, few[:, :0], values[:, :0])), (ValueError, lambda: losses.distill_top(x, few, values[:, :2])),
                        (ValueError, lambda: losses.distill_top(x, few[:3], values[:3])), (ValueError, lambda: losses.distill_top(x, ids, one)),
                        (ValueError, lambda: losses.distill_top(x, few.repeat(1, 22), values.repeat(1, 22))), (TypeError, lambda: losses.distill_top(x, values, values)),
                        (TypeError, lambda: losses.distill_top(x, few, values.half())), (ValueError, lambda: losses.distill_top(x, few, values.cpu())),
                        (ValueError, lambda: losses.distill_top(x, few, values.clone().requires_grad_())),
                        (EriError, lambda: losses.distill_top(x, few, values, temperature=1e5)),
                        (ValueError, lambda: losses.distill_top_grad(x, few, values, r.stats, one)), (ValueError, lambda: losses.distill_top_grad(x, few, values, d.stats, one[:2])),
                        (ValueError, lambda: losses.distill_top_grad(x, few, values, d.stats, one, out=x.bfloat16().float()[:, :7]))]:
        with pytest.raises(error):
            call()


def test_the_c_calls_write_nothing_behind_their_outputs():
    """One workspace for batches of all sizes, made for the largest; outputs with a guard behind them."""
    from eridiffusion_amd import _lib as L
    most, vocab, k = 40, 70011, 13
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    size = max(_sized("eri_token_logprobs_workspace", most, vocab, k), _sized("eri_distill_top_workspace", most, vocab))
    ws = torch.full((size + 64,), 77, dtype=torch.uint8, device="cuda")
    for rows in (most, most - 1, 7, 1):
        x, ids = _logits(rows, vocab, BF), _ids(rows, vocab)
        dev, dids = x.cuda(), ids.cuda()
        new = lambda *n, dtype=F32: torch.full((rows + 1, *n), 5, dtype=dtype, device="cuda")  # noqa: E731
        logprob, entropy, stats, top, places = new(), new(), new(2), new(k), new(k, dtype=torch.long)
        a = Logprobs(logits=dev.data_ptr(), ids=dids.data_ptr(), logprob=logprob.data_ptr(), entropy=entropy.data_ptr(), stats=stats.data_ptr(), top=top.data_ptr(),
                     top_ids=places.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=size, rows=rows, vocab=vocab, temperature=1.0, ids_64=1, dtype_tag=2, top_n=k)
        L.check(L.lib().eri_token_logprobs(C.byref(a), stream), "eri_token_logprobs")
        from eridiffusion_amd.losses import DistillTop, TokenLogprobs
        _check_scores(TokenLogprobs(logprob[:rows], entropy[:rows], top[:rows], places[:rows], stats[:rows]), x, ids, 1.0, k, rows)
        loss, more, out = new(), new(6), new(vocab, dtype=BF)
        d = Distill(logits=dev.data_ptr(), ids=places.data_ptr(), teacher=top.data_ptr(), loss=loss.data_ptr(), stats=more.data_ptr(), workspace=ws.data_ptr(),
                    workspace_bytes=size, rows=rows, vocab=vocab, temperature=1.0, ids_64=1, dtype_tag=2, teacher_dtype=0, k=k, rest=1)
        L.check(L.lib().eri_distill_top(C.byref(d), stream), "eri_distill_top")
        _check_distill(DistillTop(loss[:rows], more[:rows]), x, places[:rows].cpu(), top[:rows].cpu(), 1.0, True, rows)
        grad = _gen(rows)
        dgrad = grad.cuda()
        e = DistillGrad(logits=dev.data_ptr(), ids=places.data_ptr(), teacher=top.data_ptr(), stats=more.data_ptr(), grad=dgrad.data_ptr(), out=out.data_ptr(), rows=rows,
                        vocab=vocab, temperature=1.0, ids_64=1, dtype_tag=2, teacher_dtype=0, out_dtype=2, k=k)
        L.check(L.lib().eri_distill_top_grad(C.byref(e), stream), "eri_distill_top_grad")
        _check_distill_grad(out[:rows], x, places[:rows].cpu(), top[:rows].cpu(), grad, 1.0, True, rows)
        f = LogprobsGrad(logits=dev.data_ptr(), ids=dids.data_ptr(), stats=stats.data_ptr(), grad=dgrad.data_ptr(), out=out.data_ptr(), rows=rows, vocab=vocab,
                         temperature=1.0, ids_64=1, dtype_tag=2, out_dtype=2)
        L.check(L.lib().eri_token_logprobs_grad(C.byref(f), stream), "eri_token_logprobs_grad")
        _check_token_grad(out[:rows], x, ids, grad, None, 1.0, rows)
        assert bool((ws[size:] == 77).all()) and all(bool((t[rows] == 5).all()) for t in (logprob, entropy, stats, top, places, loss, more, out))


def test_the_examples_loss_and_its_gradients_are_those_of_cross_entropy():
    """The example runs, and its loss, which it reads off bf16 logits, is the mean over the tokens that are asked for."""
    import importlib.util
    import os

    from test_losses_host import ROOT
    spec = importlib.util.spec_from_file_location("train_tokens", os.path.join(ROOT, "examples", "train_tokens.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    torch.manual_seed(3)
    model = example.Model(0.0)
    rows = torch.randn(4, 16, example.DIM, device="cuda", dtype=BF).requires_grad_()
    target = torch.randint(0, example.VOCAB, (4, 16), device="cuda")
    target[:, -3:] = -100
    loss = model.loss(rows, target, 0)
    loss.backward()
    with torch.no_grad():  # the same model up to its logits, whose gradient is then taken in 64 bits
        from eridiffusion_amd import layers
        h = layers.dropout(rows, 0.0, seed=1)
        y = layers.rms_norm(h, model.norms[0]).y
        for i in range(example.BLOCKS):
            branch = torch.nn.functional.gelu(y @ model.up[i]) @ model.down[i]
            y, h, _, _ = layers.rms_norm(branch, model.norms[i + 1], residual=h)
        logits = (y @ model.head).double().flatten(0, 1)
    real = target.flatten() >= 0
    logp = torch.log_softmax(logits, 1)
    want = -logp[real, target.flatten()[real]].mean()
    assert abs(loss.item() - want.item()) < 64 * 2 * U32 * 64 * abs(want.item())  # means of 52 numbers, each a few roundings off
    p = logp.exp()
    p[real, target.flatten()[real]] -= 1
    dz = torch.where(real[:, None], p / real.sum(), 0.0)
    dw = y.double().flatten(0, 1).t() @ dz
    # each term's gradient is rounded to bf16, and so is their sum
    size = y.double().flatten(0, 1).abs().t() @ dz.abs()
    _near(model.head.grad, dw.cpu(), (U[BF] * dw.abs() + (U[BF] + 100 * U32) * size).cpu())
