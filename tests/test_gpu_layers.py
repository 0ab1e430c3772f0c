"""The layers' kernels against the 64-bit oracle.

Bounds, with u = 2^-24 for float32 and 2^-8 for bfloat16: one rounding to the output's type is u |result|, a sum of n
float32 terms in any order (n + 2) 2^-24 times the sum of their magnitudes.  Eight-bit values are half a step of their grid off."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import layers_f64 as of
from test_layers_host import Norm, NormGrad

pytestmark = pytest.mark.gpu
BF, F32, F8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
U = {BF: 2.0 ** -8, F32: 2.0 ** -24}
U32 = 2.0 ** -24
SEED, OFFSET = 0x9E3779B97F4A7C15, 2 ** 33 + 5


@pytest.fixture
def layers():
    from eridiffusion_amd import layers
    return layers


def _new(*shape, dtype=F32, seed=0, std=1.0, mean=0.0):
    g = torch.Generator().manual_seed(hash((shape, seed)) % 2 ** 31)
    return (torch.randn(*shape, generator=g) * std + mean).to(dtype)


def _near(got, want, bound, what=""):
    got, bound = got.cpu().double(), torch.as_tensor(bound, dtype=torch.float64) + 1e-37
    assert got.shape == want.shape, (got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), what
    off = torch.nan_to_num((got - want).abs(), 0.0, float("inf"))
    off = torch.where(got == want, 0.0, off)
    assert bool((off <= bound).all()), "%s: off by %g times the bound" % (what, (off / bound).max())


# ---------------------------------------------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (3, 5, 8), (33, 257), (1000, 64), (0, 8), (2, 0)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.75, 1.0])
def test_dropout(layers, dtype, shape, p):
    x = _new(*shape, dtype=dtype)
    want = of.dropout(x, p, SEED, OFFSET)
    y = layers.dropout(x.cuda(), p, SEED, OFFSET)
    assert torch.equal(y.cpu() == 0, want == 0)
    _near(y, want, (U[dtype] + 2 * U32) * want.abs())
    z = x.cuda()
    assert layers.dropout(z, p, SEED, OFFSET, out=z) is z and torch.equal(z, y)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cols", [8, 13, 129])
def test_dropout_of_rows_with_gaps(layers, dtype, cols):
    """The mask goes by an element's place in the tensor, not in memory; nothing beside the rows is written."""
    whole = _new(70, 200, dtype=dtype).cuda()
    for at in (0, 1, 3):
        x = whole[:, at:at + cols]
        want = of.dropout(x.cpu(), 0.3, 1, 2)
        _near(layers.dropout(x, 0.3, 1, 2), want, (U[dtype] + 2 * U32) * want.abs())
        back = whole.clone()
        out = back[:, at:at + cols]
        layers.dropout(x, 0.3, 1, 2, out=out)
        _near(out, want, (U[dtype] + 2 * U32) * want.abs())
        out.copy_(x)
        assert torch.equal(back, whole)
    t = _new(20, 30, dtype=dtype).cuda().t()  # no rows: copied first
    _near(layers.dropout(t, 0.3, 1, 2), of.dropout(t.cpu(), 0.3, 1, 2), 2 * U[dtype] * t.cpu().abs().double())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_dropped_infinities_and_nan_are_zero(layers, dtype):
    x = _new(4096, dtype=dtype)
    x[::3], x[1::3], x[5::7] = float("nan"), float("inf"), -float("inf")
    want = of.dropout(x, 0.5, 3, 4)
    y = layers.dropout(x.cuda(), 0.5, 3, 4).cpu()
    keep = of.kept((4096,), 0.5, 3, 4) != 0
    assert bool((y[~keep] == 0).all()) and torch.equal(y[keep].isnan(), x[keep].isnan())
    _near(y, want, 2 * U[dtype] * torch.nan_to_num(want.abs(), 0, 0, 0))


def test_dropout_past_32_bit_counts(layers):
    n = 2 ** 32 + 1003
    x = torch.ones(n, dtype=BF, device="cuda")
    layers.dropout(x, 0.5, 11, 12, out=x)
    for first in (0, 2 ** 31 - 8, 2 ** 32 - 8, n - 1003 - 5):
        first -= first % 8
        words = of.philox(np.arange(first // 8, first // 8 + 16, dtype=np.uint64), 11, 12)
        bits = np.stack((words & np.uint64(0xFFFF), words >> np.uint64(16)), 2).reshape(-1)
        assert np.array_equal(x[first:first + 128].float().cpu().numpy(), np.where(bits >= 32768, 2.0, 0.0))
    last = n - n % 8
    words = of.philox(np.array([last // 8], np.uint64), 11, 12)
    bits = np.stack((words & np.uint64(0xFFFF), words >> np.uint64(16)), 2).reshape(-1)[:n % 8]
    assert np.array_equal(x[last:].float().cpu().numpy(), np.where(bits >= 32768, 2.0, 0.0))


def test_an_offset_on_the_device_is_read_when_the_kernel_runs(layers):
    x = _new(50, 40).cuda()
    step = torch.tensor([17], dtype=torch.long, device="cuda")
    assert torch.equal(layers.dropout(x, 0.2, 5, step), layers.dropout(x, 0.2, 5, 17))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        layers.dropout(x, 0.2, 5, step)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            y = layers.dropout(x, 0.2, 5, step)
            n = layers.rms_norm(y, residual=x, p=0.4, seed=6, offset=step)
            step.add_(1)
    for k in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, layers.dropout(x, 0.2, 5, 17 + k)), k
        assert torch.equal(n.y, layers.rms_norm(y, residual=x, p=0.4, seed=6, offset=17 + k).y), k


# ---------------------------------------------------------------------------------------------------------------
# lookup
# ---------------------------------------------------------------------------------------------------------------

def _ids(n, vocab, seed=0, dtype=torch.long, common=0.0, outside=True):
    g = torch.Generator().manual_seed(n * 31 + vocab + seed)
    ids = torch.randint(0, vocab, (n,), generator=g)
    ids[torch.rand(n, generator=g) < common] = vocab // 2
    if outside and n > 4:
        ids[1], ids[3], ids[4] = -1, vocab, -100
    return ids.to(dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("tokens,vocab,dim", [(0, 5, 8), (1, 1, 1), (2, 9, 3), (77, 300, 64), (77, 1000, 65), (5, 7, 768), (333, 50, 257), (600, 99, 1280),
                                              (40, 11, 4097), (20000, 500, 40), (9000, 40, 520)])
def test_lookup(layers, dtype, tokens, vocab, dim):
    w = _new(vocab, dim + 3, dtype=dtype)
    for ids in (_ids(tokens, vocab), _ids(tokens, vocab, dtype=torch.int32)):
        for scale in (1.0, 27.7):
            for table in (w[:, :dim].contiguous().cuda(), w.cuda()[:, 3:]):
                want = of.embedding(ids, table.cpu(), np.float32(scale).item())
                _near(layers.embedding(ids.cuda(), table, scale), want, 0.0 if scale == 1 else (U[dtype] + U32) * want.abs())
    back = torch.full((tokens, dim + 5), 7.0, dtype=dtype).cuda()
    layers.embedding(ids.cuda(), table, 1.0, out=back[:, 2:dim + 2])
    assert torch.equal(back[:, 2:dim + 2].double().cpu(), of.embedding(ids, table.cpu(), 1.0)) and bool((back[:, :2] == 7).all()) and bool((back[:, dim + 2:] == 7).all())


def test_lookup_shapes_and_long_tables(layers):
    w = _new(50, 16, dtype=BF).cuda()
    ids = _ids(24, 50).view(2, 3, 4).cuda()
    assert layers.embedding(ids, w).shape == (2, 3, 4, 16)
    assert torch.equal(layers.embedding(ids.transpose(0, 2), w), layers.embedding(ids, w).transpose(0, 2))
    assert layers.embedding(torch.tensor(3, device="cuda"), w).shape == (16,)
    big = torch.empty(2 ** 21 + 7, 2048, dtype=BF, device="cuda")  # offsets over 2^32
    at = torch.tensor([0, 2 ** 20, 2 ** 21 - 1, 2 ** 21, 2 ** 21 + 6], device="cuda")
    big[at] = _new(5, 2048, dtype=BF).cuda()
    assert torch.equal(layers.embedding(at, big), big[at])


def test_refusals_on_the_device(layers):
    x, ids = torch.zeros(4, 8, device="cuda"), torch.zeros(4, dtype=torch.long, device="cuda")
    for error, call in [(TypeError, lambda: layers.embedding(ids.float(), x)), (TypeError, lambda: layers.embedding(ids, x.half())),
                        (ValueError, lambda: layers.embedding(ids, x[0])), (ValueError, lambda: layers.embedding(ids.cpu(), x)),
                        (ValueError, lambda: layers.embedding(ids, x, out=x[:3])), (ValueError, lambda: layers.embedding(ids, x, out=x.bfloat16())),
                        (ValueError, lambda: layers.embedding(ids, x, out=torch.zeros(8, 4, device="cuda").t())),
                        (ValueError, lambda: layers.embedding_grad(ids[:3], x, 9)), (ValueError, lambda: layers.embedding_grad(ids, x, 9, padding_id=9)),
                        (ValueError, lambda: layers.embedding_grad(ids, x, 9, accumulate=True)), (ValueError, lambda: layers.embedding_grad(ids, x, 2 ** 31)),
                        (ValueError, lambda: layers.embedding_grad(ids, x, 9, out=x)), (TypeError, lambda: layers.embedding_grad(ids, x, 9, dtype=F8)),
                        (ValueError, lambda: layers.embedding_grad(ids, x, 4, out=x, dtype=BF)), (ValueError, lambda: layers.dropout(x, 1.5, 0)),
                        (ValueError, lambda: layers.dropout(x, 0.5, -1)), (ValueError, lambda: layers.dropout(x, 0.5, 2 ** 64)),
                        (TypeError, lambda: layers.dropout(x, 0.5, 1.5)), (ValueError, lambda: layers.dropout(x, 0.5, 1, ids)),
                        (ValueError, lambda: layers.dropout(x, 0.5, 1, out=x[:2])), (ValueError, lambda: layers.rms_norm(x, x[0, :4])),
                        (ValueError, lambda: layers.rms_norm(x, residual=x[:2])), (TypeError, lambda: layers.rms_norm(x, dtype=torch.float16)),
                        (ValueError, lambda: layers.rms_norm(x, scale_group=128)), (ValueError, lambda: layers.rms_norm(x, dtype=F8, scale_group=64)),
                        (ValueError, lambda: layers.rms_norm_grad(x, x, x[:, 0].bfloat16())), (ValueError, lambda: layers.rms_norm_grad(x, x[:2], x[:, 0])),
                        (ValueError, lambda: layers.rms_norm_grad(x, x, x[:, 0], grad_h=x.bfloat16())), (TypeError, lambda: layers.rms_norm_grad(x, x, x[:, 0], needs=True)),
                        (ValueError, lambda: layers.rms_norm(x.requires_grad_(), dtype=F8))]:
        with pytest.raises(error):
            call()
    from eridiffusion_amd import EriError
    with pytest.raises(EriError, match="rows without elements"):
        layers.rms_norm(torch.zeros(3, 0, device="cuda"))
    with pytest.raises(EriError, match="eps"):
        layers.rms_norm(x.detach(), eps=-1.0)
    with pytest.raises(EriError, match="without rows"):
        layers.embedding(ids, x.detach()[:0])


# ---------------------------------------------------------------------------------------------------------------
# the table's gradient
# ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,out", [(BF, BF), (BF, F32), (F32, F32), (F32, BF)])
@pytest.mark.parametrize("tokens,vocab,dim,common", [
    (0, 5, 8, 0), (1, 1, 1, 0), (64, 1, 24, 0), (65, 1, 24, 0), (500, 3, 7, 0), (300, 256, 64, 0), (300, 257, 65, 0.5), (2000, 700, 130, 0.2),
    (4097, 1023, 257, 0.1), (5000, 40, 520, 0.6), (3000, 100, 1156, 1.0), (2000, 262144, 8, 0.1), (1000, 263000, 9, 0.1), (20000, 5000, 16, 0.3)])
def test_table_gradient(layers, dtype, out, tokens, vocab, dim, common):
    ids, grad = _ids(tokens, vocab, common=common), _new(tokens, dim, dtype=dtype)
    scale = np.float32(1.7).item()
    deep = int(torch.bincount(ids[(ids >= 0) & (ids < vocab)], minlength=1).max()) + 4 if tokens else 4
    for pad in (None, vocab // 2):
        want, size = of.embedding_grad(ids, grad, vocab, scale, pad)
        got = layers.embedding_grad(ids.cuda(), grad.cuda(), vocab, scale, padding_id=pad, dtype=out)
        _near(got, want, U[out] * want.abs() + deep * U32 * size, "pad %s" % pad)
        assert torch.equal(got, layers.embedding_grad(ids.int().cuda(), grad.cuda(), vocab, scale, padding_id=pad, dtype=out))  # the same bits
        old = _new(vocab, dim, dtype=out, seed=3)
        into = old.cuda()
        assert layers.embedding_grad(ids.cuda(), grad.cuda(), vocab, scale, padding_id=pad, out=into, accumulate=True) is into
        _near(into, want + old.double(), U[out] * (want + old.double()).abs() + (deep + 1) * U32 * (size + old.double().abs()), "accumulate")
        untouched = size.sum(1) == 0
        assert torch.equal(into.cpu()[untouched], old[untouched])


def test_table_gradient_of_strided_broadcast_and_shaped_inputs(layers):
    ids = _ids(600, 37, common=0.3).view(3, 200)
    wide = _new(3, 200, 50, dtype=BF)
    want, size = of.embedding_grad(ids, wide[..., 5:45], 37, 1.0)
    bound = U32 * 700 * size
    back = torch.full((37, 48), 9.0, device="cuda")
    got = layers.embedding_grad(ids.cuda(), wide.cuda()[..., 5:45], 37, out=back[:, 4:44])
    _near(got, want, bound)
    assert bool((back[:, :4] == 9).all()) and bool((back[:, 44:] == 9).all())
    row = _new(40, dtype=BF)
    want, size = of.embedding_grad(ids, row.expand(3, 200, 40), 37, 1.0)
    _near(layers.embedding_grad(ids.cuda(), row.cuda().expand(3, 200, 40), 37, dtype=F32), want, U32 * 700 * size)
    want, size = of.embedding_grad(ids.t(), wide.transpose(0, 1)[..., 5:45], 37, 1.0)
    _near(layers.embedding_grad(ids.cuda().t(), wide.cuda().transpose(0, 1)[..., 5:45], 37, dtype=F32), want, U32 * 700 * size)


def test_table_gradient_past_32_bit_offsets(layers):
    vocab, dim = 2 ** 20 + 11, 4100  # 2^32 elements and more
    ids = torch.tensor([vocab - 1, 5, vocab - 1, 2 ** 20, -1])
    grad = _new(5, dim, dtype=BF)
    out = torch.empty(vocab, dim, dtype=BF, device="cuda").fill_(3.0)
    layers.embedding_grad(ids.cuda(), grad.cuda(), vocab, out=out)
    for v, rows in [(vocab - 1, [0, 2]), (5, [1]), (2 ** 20, [3]), (0, []), (vocab - 2, []), (2 ** 19, [])]:
        want = grad.double()[rows].sum(0)
        _near(out[v], want, (U[BF] + 4 * U32) * want.abs() + 4 * U32)
    assert int((out != 0).any(1).sum()) == 3


@pytest.mark.parametrize("vocab,dim", [(70000, 1000), (300000, 256)])
def test_table_gradient_of_no_token(layers, vocab, dim):
    """A large table, which takes the sort, with an empty batch: zeros, or what was there."""
    ids, grad = torch.zeros(0, dtype=torch.long, device="cuda"), torch.zeros(0, dim, dtype=BF, device="cuda")
    out = torch.full((vocab, dim), 3.0, dtype=BF, device="cuda")
    layers.embedding_grad(ids, grad, vocab, out=out, accumulate=True)
    assert bool((out == 3).all())
    layers.embedding_grad(ids, grad, vocab, out=out)
    assert bool((out == 0).all())


# ---------------------------------------------------------------------------------------------------------------
# norm
# ---------------------------------------------------------------------------------------------------------------

def _depth(cols):
    """Terms that one of the float32 sums over a row adds up, one after the other."""
    return cols / 64 + 40


def _norm_bounds(x, w, res, p, want_y, want_h, want_rstd, cols):
    """What float32 may be off before the last rounding: of h, and of y."""
    size = of.dropout(x, p, SEED, OFFSET).abs() + (res.double().abs() if res is not None else 0)
    h = 3 * U32 * size
    scale = want_rstd[..., None] * (w.double().abs() if w is not None else 1)
    return h, h * scale + want_y.abs() * U32 * (_depth(cols) + 8) + want_y.abs() * (h * want_h.abs()).mean(-1, keepdim=True) * want_rstd[..., None] ** 2


COLS = [1, 7, 64, 129, 512, 520, 1000, 1281, 2048, 2056, 4096, 5001, 8192, 9001, 16384, 20000, 33000, 40001]


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype,res,w,out", [(BF, BF, BF, BF), (BF, F32, F32, BF), (F32, F32, F32, F32), (BF, None, BF, F32), (F32, BF, None, BF), (F32, None, F32, BF)])
def test_norm(layers, cols, dtype, res, w, out):
    rows = 70 if cols < 600 else 6
    x, weight = _new(rows, cols, dtype=dtype), None if w is None else _new(cols, dtype=w, std=0.3, mean=1.0)
    r = None if res is None else _new(rows, cols, dtype=res, std=2.0, seed=1)
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    for p in (0.0, 0.3):
        y, h, rstd = of.rms_norm(x, weight, 1e-6, r, p, SEED, OFFSET)
        off_h, off_y = _norm_bounds(x, weight, r, p, y, h, rstd, cols)
        given = x.cuda()
        got = layers.rms_norm(given, dev(weight), 1e-6, residual=dev(r), p=p, seed=SEED, offset=OFFSET, dtype=out)
        assert got.y.dtype == out and got.scales is None
        _near(got.y, y, U[out] * y.abs() + off_y, "y, p %g" % p)
        _near(got.rstd, rstd, rstd * U32 * (_depth(cols) + 8) + rstd ** 3 * (off_h * h.abs()).mean(-1), "rstd")
        if r is None and p == 0:
            assert got.h is given
        else:
            assert got.h.dtype == (res or dtype)
            _near(got.h, h, U[got.h.dtype] * h.abs() + off_h, "h")


@pytest.mark.parametrize("cols", [1, 9, 127, 128, 130, 700, 1280, 2500, 5120, 16000, 20000, 33001])
@pytest.mark.parametrize("group", [0, 128])
@pytest.mark.parametrize("dtype,res", [(BF, BF), (F32, None)])
def test_norm_in_eight_bits(layers, cols, group, dtype, res):
    rows = 9
    x, w = _new(rows, cols, dtype=dtype), _new(cols, dtype=dtype, std=0.5, mean=1.0)
    x[2] = 0
    r = None if res is None else _new(rows, cols, dtype=res, std=2.0, seed=1)
    if r is not None:
        r[2] = 0
    p = 0.2 if res else 0.0
    y, h, rstd = of.rms_norm(x, w, 1e-6, r, p, SEED, OFFSET)
    _, off = _norm_bounds(x, w, r, p, y, h, rstd, cols)
    got = layers.rms_norm(x.cuda(), w.cuda(), 1e-6, residual=None if r is None else r.cuda(), p=p, seed=SEED, offset=OFFSET, dtype=F8, scale_group=group)
    scales = of.scales_of(y, group)
    assert got.y.dtype == F8 and got.scales.shape == scales.shape == (rows, -(-cols // group) if group else 1)
    wide = lambda s: s.repeat_interleave(group or cols, -1)[:, :cols]  # noqa: E731
    assert bool((scales[2] == 1).all()) and bool((got.scales[2] == 1).all())
    off_scales = torch.stack([q.amax(-1) for q in off.split(group or cols, -1)], -1) / of.F8_MAX + 2 * U32 * scales
    _near(got.scales, scales, off_scales, "scales")
    q = y / wide(scales)
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)  # between neighbours of that size
    _near(got.y.float(), q, 0.5 * step + 2 * (off / wide(scales) + q.abs() * (wide(off_scales / scales) + 3 * U32)), "codes")


@pytest.mark.parametrize("cols", [100, 3000, 40000])
def test_norm_of_zeros_infinities_and_nan(layers, cols):
    x = _new(6, cols, dtype=BF)
    x[0] = 0
    x[1, 5] = float("nan")
    x[2, 7] = float("inf")
    x[3] *= 1e-20
    w = torch.ones(cols, dtype=BF)
    w[9] = float("nan")
    y, h, rstd = of.rms_norm(x, w, 1e-6)
    got = layers.rms_norm(x.cuda(), w.cuda(), 1e-6)
    _near(got.y, y, U[BF] * 1.01 * torch.nan_to_num(y.abs(), 0, 0, 0) + 1e-30)
    _near(got.rstd, rstd, torch.nan_to_num(rstd, 0) * U32 * (_depth(cols) + 8))
    f8 = layers.rms_norm(x.cuda(), w.cuda(), 1e-6, dtype=F8, scale_group=128)
    assert torch.equal(f8.y.float().cpu().isnan(), y.isnan())
    assert torch.equal(f8.scales.isnan().cpu(), torch.zeros_like(f8.scales.cpu(), dtype=torch.bool))
    z = layers.rms_norm(torch.zeros(2, cols, device="cuda"), eps=0.0)  # 0 * infinity
    assert bool(z.y.isnan().all()) and bool(z.rstd.isinf().all())


@pytest.mark.parametrize("group", [0, 128])
def test_eight_bits_of_very_small_values(layers, group):
    """Where 448 / max|y| would leave float32 the group counts as zeros; just above, it is scaled like any other."""
    x = torch.ones(4, 300)
    x[0], x[1], x[2, 10:] = 1e-38, 2.0 ** -110, 0
    w = torch.full((300,), 2.0 ** -95)
    got = layers.rms_norm(x.cuda(), w.cuda(), 1.0, dtype=F8, scale_group=group)
    y, _, _ = of.rms_norm(x, w, 1.0)
    scales = of.scales_of(y, group)
    _near(got.scales, scales, 16 * U32 * scales)
    assert bool((got.scales[:2] == 1).all()) and bool((got.y[:2].float() == 0).all())
    assert bool((got.y[3].float() == 448).all()) and not bool(got.y.float().isnan().any())


def test_norm_of_a_single_row_without_other_dimensions(layers):
    x, r, w = _new(40).cuda(), _new(40, seed=1).cuda(), _new(40, seed=2).cuda()
    got, want = layers.rms_norm(x, w, residual=r), layers.rms_norm(x[None], w, residual=r[None])
    assert got.rstd.shape == () and torch.equal(got.y, want.y[0]) and torch.equal(got.h, want.h[0]) and torch.equal(got.rstd, want.rstd[0])
    assert layers.rms_norm(x, w, dtype=F8).scales.shape == (1,)
    back, rows = layers.rms_norm_grad(x, got.h, got.rstd, w), layers.rms_norm_grad(x[None], want.h, want.rstd, w)
    assert torch.equal(back.x, rows.x[0]) and torch.equal(back.weight, rows.weight)


def test_norm_of_strided_shaped_and_empty_inputs(layers):
    wide = _new(5, 7, 90, dtype=BF).cuda()
    for x in (wide[..., 3:83], wide[:, 2:5, :80], wide[::2, 1, 10:90], wide.transpose(0, 1)[..., :80], wide[:1, :1, 5:85], wide[0, 0, :80].expand(4, 80)):
        r = _new(*x.shape, seed=8).cuda()
        y, h, rstd = of.rms_norm(x.cpu(), None, 1e-5, r.cpu())
        got = layers.rms_norm(x, eps=1e-5, residual=r, dtype=F32)
        assert got.y.shape == x.shape and got.rstd.shape == x.shape[:-1]
        _near(got.y, y, 1e-5 * y.abs() + 1e-6)
        _near(got.h, h, U32 * h.abs() + U32)
    empty = layers.rms_norm(torch.zeros(0, 16, device="cuda"), dtype=F8, scale_group=128)
    assert empty.y.shape == (0, 16) and empty.scales.shape == (0, 1) and empty.rstd.shape == (0,)


@pytest.mark.parametrize("cols", [96, 1001, 5000, 34000])
def test_norm_in_place_and_with_gaps_through_the_c_call(cols):
    """y over x and h over the residual, rows with gaps: what lies between them stays."""
    from eridiffusion_amd import _lib as L
    x, r, w = _new(11, cols + 9, dtype=BF), _new(11, cols + 4, seed=2), _new(cols, dtype=F32)
    y, h, rstd = of.rms_norm(x[:, :cols], w, 1e-6, r[:, :cols], 0.25, SEED, OFFSET)
    off_h, off_y = _norm_bounds(x[:, :cols], w, r[:, :cols], 0.25, y, h, rstd, cols)
    dx, dr, dw = x.cuda(), r.cuda(), w.cuda()
    a = Norm(x=dx.data_ptr(), residual=dr.data_ptr(), weight=dw.data_ptr(), y=dx.data_ptr(), h=dr.data_ptr(), rows=11, cols=cols, x_stride=cols + 9,
             residual_stride=cols + 4, y_stride=cols + 9, h_stride=cols + 4, eps=1e-6, x_dtype=2, residual_dtype=0, weight_dtype=0, y_dtype=2)
    a.key.seed, a.key.offset, a.key.p = SEED, OFFSET, 0.25
    L.check(L.lib().eri_rms_norm(C.byref(a), C.c_void_p(torch.cuda.current_stream().cuda_stream)), "eri_rms_norm")
    _near(dx[:, :cols], y, U[BF] * y.abs() + off_y)
    _near(dr[:, :cols], h, U32 * h.abs() + off_h)
    assert torch.equal(dx[:, cols:].cpu(), x[:, cols:]) and torch.equal(dr[:, cols:].cpu(), r[:, cols:])


# ---------------------------------------------------------------------------------------------------------------
# its gradient
# ---------------------------------------------------------------------------------------------------------------

def _grad_inputs(rows, cols, dtype, stream, w):
    x, gy, gh = _new(rows, cols, dtype=stream, std=2.0), _new(rows, cols, dtype=dtype, seed=1), _new(rows, cols, dtype=stream, seed=2)
    weight = None if w is None else _new(cols, dtype=w, std=0.3, mean=1.0)
    rstd = (1 / torch.sqrt((x.double() ** 2).mean(-1) + 1e-6)).float()
    return gy, x, rstd, weight, gh


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype,stream,w", [(BF, BF, BF), (F32, F32, F32), (BF, F32, F32), (F32, BF, None)])
@pytest.mark.parametrize("p,more", [(0.0, True), (0.3, True), (0.0, False)])
def test_norm_gradient(layers, cols, dtype, stream, w, p, more):
    rows = 1100 if cols < 100 else 131 if cols < 1100 else 5
    gy, h, rstd, weight, gh = _grad_inputs(rows, cols, dtype, stream, w)
    if not more:
        gh = None
    dx, dr, dw, size, size_w = of.rms_norm_grad(gy, h, rstd, weight, gh, p, SEED, OFFSET)
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    got = layers.rms_norm_grad(dev(gy), dev(h), dev(rstd), dev(weight), grad_h=dev(gh), p=p, seed=SEED, offset=OFFSET, dtype=dtype)
    off = U32 * (_depth(cols) + 12) * size
    _near(got.residual, dr, U[stream] * dr.abs() + off, "residual")
    share = 1 / (1 - int(p * 65536 + 0.5) / 65536)
    _near(got.x, dx, U[dtype] * dx.abs() + off * share + 2 * U32 * dx.abs(), "x")
    assert (got.weight is None) == (w is None) and (got.x is got.residual) == (p == 0 and dtype == stream)
    if w is not None:
        assert got.weight.dtype == w
        _near(got.weight, dw, U[w] * dw.abs() + U32 * (rows + 130) * size_w, "weight")
        again = layers.rms_norm_grad(dev(gy), dev(h), dev(rstd), dev(weight), grad_h=dev(gh), p=p, seed=SEED, offset=OFFSET, dtype=dtype)
        assert torch.equal(got.weight, again.weight)  # the same bits
    for needs in [(True, False, False), (False, True, False), (False, False, True), (False, False, False)]:
        part = layers.rms_norm_grad(dev(gy), dev(h), dev(rstd), dev(weight), grad_h=dev(gh), p=p, seed=SEED, offset=OFFSET, dtype=dtype, needs=needs)
        for need, a, b in zip(needs, part, got):
            assert (a is not None) == (need and b is not None) and (a is None or torch.equal(a, b))


@pytest.mark.parametrize("rows,cols", [(0, 50), (1, 1), (3000, 72), (2100, 600), (1300, 2100), (300, 17000), (280, 33001)])
def test_norm_gradient_of_few_and_many_rows(layers, rows, cols):
    gy, h, rstd, w, _ = _grad_inputs(rows, cols, BF, BF, F32)
    dx, _, dw, size, size_w = of.rms_norm_grad(gy, h, rstd, w)
    got = layers.rms_norm_grad(gy.cuda(), h.cuda(), rstd.cuda(), w.cuda())
    _near(got.x, dx, U[BF] * dx.abs() + U32 * (_depth(cols) + 12) * size)
    _near(got.weight, dw, U32 * dw.abs() + U32 * (rows + 130) * size_w)


@pytest.mark.parametrize("cols", [96, 1001, 5000, 34000])
def test_norm_gradient_in_place_and_with_gaps_through_the_c_call(cols):
    from eridiffusion_amd import _lib as L
    gy, h, rstd, w, gh = _grad_inputs(9, cols + 7, BF, F32, BF)
    v = slice(0, cols)
    dx, dr, dw, size, size_w = of.rms_norm_grad(gy[:, v], h[:, v], rstd, w[v], gh[:, v], 0.25, SEED, OFFSET)
    g, hh, q, ww, r = gy.cuda(), h.cuda(), rstd.cuda(), w.cuda(), gh.cuda()
    need, s = C.c_uint64(), C.c_void_p(torch.cuda.current_stream().cuda_stream)
    L.check(L.lib().eri_rms_norm_grad_workspace(C.c_uint64(9), C.c_uint64(cols), C.byref(need)), "workspace")
    ws, weight = torch.empty(need.value + 16, dtype=torch.uint8, device="cuda"), torch.empty(cols + 1, device="cuda").fill_(5)
    ws[need.value:] = 77
    a = NormGrad(grad=g.data_ptr(), h=hh.data_ptr(), rstd=q.data_ptr(), weight=ww.data_ptr(), grad_h=r.data_ptr(), grad_x=g.data_ptr(),
                 grad_residual=r.data_ptr(), grad_weight=weight.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=need.value, rows=9, cols=cols,
                 grad_stride=cols + 7, h_stride=cols + 7, grad_h_stride=cols + 7, grad_x_stride=cols + 7, grad_residual_stride=cols + 7, grad_dtype=2,
                 h_dtype=0, x_dtype=2, weight_dtype=2, grad_weight_dtype=0)
    a.key.seed, a.key.offset, a.key.p = SEED, OFFSET, 0.25
    L.check(L.lib().eri_rms_norm_grad(C.byref(a), s), "eri_rms_norm_grad")
    off = U32 * (_depth(cols) + 12) * size
    _near(r[:, v], dr, U32 * dr.abs() + off)
    _near(g[:, v], dx, U[BF] * dx.abs() + 1.4 * off + 2 * U32 * dx.abs())
    _near(weight[:cols], dw, U32 * dw.abs() + U32 * 139 * size_w)
    assert torch.equal(g[:, cols:].cpu(), gy[:, cols:]) and torch.equal(r[:, cols:].cpu(), gh[:, cols:])
    assert weight[cols].item() == 5 and bool((ws[need.value:] == 77).all())


# ---------------------------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------------------------

def test_autograd_against_differences(layers):
    """lookup -> dropout -> lookup's rows added and normed, in float32: the gradients along a direction against central
    differences of the same chain in 64 bits.  The kernels' error is that of sums of at most 330 float32 terms, the
    difference's own of the order 1e-8; the products with the direction are summed in 64 bits."""
    ids = _ids(60, 40, common=0.2)
    w, n, d_w, d_n = _new(40, 24), _new(24, std=0.2, mean=1.0), _new(40, 24, seed=1), _new(24, seed=2)
    gy, gh = _new(60, 24, seed=3), _new(60, 24, seed=4)
    scale, eps = 1.25, 1e-3

    def chain(t):
        rows = of.embedding(ids, w.double() + t * d_w.double(), scale)
        y, h, _ = of.rms_norm(of.dropout(rows, 0.2, 1, 1), n.double() + t * d_n.double(), eps, rows, 0.3, 2, 2)
        return (y * gy.double()).sum() + (h * gh.double()).sum()
    table, norm = w.cuda().requires_grad_(), n.cuda().requires_grad_()
    rows = layers.embedding(ids.cuda(), table, scale)
    got = layers.rms_norm(layers.dropout(rows, 0.2, 1, 1), norm, eps, residual=rows, p=0.3, seed=2, offset=2)
    ((got.y * gy.cuda()).sum() + (got.h * gh.cuda()).sum()).backward()
    a, b = table.grad.cpu().double() * d_w.double(), norm.grad.cpu().double() * d_n.double()
    want = (chain(1e-4) - chain(-1e-4)) / 2e-4
    size = a.abs().sum() + b.abs().sum()
    assert abs(a.sum() + b.sum() - want) < 400 * U32 * 10 * size + 1e-6 * size


def test_autograd_takes_what_is_needed(layers):
    x, w = _new(6, 40, dtype=BF).cuda(), _new(40, dtype=BF).cuda().requires_grad_()
    got = layers.rms_norm(x, w)
    assert got.h is x and not got.rstd.requires_grad
    got.y.float().sum().backward()
    want = layers.rms_norm_grad(torch.ones_like(x), x, got.rstd, w.detach())
    assert torch.equal(w.grad, want.weight) and x.grad is None
    x.requires_grad_()
    got = layers.rms_norm(x, w.detach(), residual=x.detach(), p=0.5, seed=1)
    got.h.float().sum().backward()  # only h is used
    assert torch.equal(x.grad, layers.dropout(torch.ones_like(x), 0.5, 1))
    with torch.no_grad():
        assert not layers.dropout(x, 0.5, 1).requires_grad
    step = torch.ones(1, dtype=torch.long, device="cuda")
    y = layers.dropout(x, 0.5, 1, step)
    step.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()


def test_outputs_that_are_given_count_as_changed(layers):
    """A value that autograd has saved is not overwritten unnoticed, and a parameter is no output."""
    x = _new(6, 40).cuda()
    w = _new(40).cuda().requires_grad_()
    loss = (x * w).sum()
    layers.dropout(x, 0.5, 1, out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    ids = torch.zeros(6, dtype=torch.long, device="cuda")
    p = torch.nn.Parameter(x.clone())
    for call in [lambda: layers.dropout(x, 0.5, 1, out=p), lambda: layers.embedding(ids, x, out=p), lambda: layers.embedding_grad(ids, x, 6, out=p),
                 lambda: layers.embedding(ids, p, out=x), lambda: layers.dropout(p, 0.5, 1, out=x), lambda: layers.embedding(ids, x, padding_id=6)]:
        with pytest.raises(ValueError):
            call()
    with torch.no_grad():
        assert torch.equal(layers.dropout(x, 0.5, 1, out=p), layers.dropout(x, 0.5, 1))
    with torch.inference_mode():
        y = torch.zeros(6, 40, device="cuda")
        assert torch.equal(layers.dropout(x, 0.5, 1, out=y), layers.dropout(x, 0.5, 1))


def test_norm_and_its_gradient_past_32_bit_offsets(layers):
    rows, cols = 2 ** 18 + 3, 16390  # 2^32 elements and more
    x = torch.zeros(rows, cols, dtype=BF, device="cuda")
    at = torch.tensor([0, 1, 2 ** 17, 2 ** 18 - 1, 2 ** 18 + 2])
    some, w = _new(5, cols, dtype=BF), _new(cols, dtype=BF, std=0.3, mean=1.0)
    x[at.cuda()] = some.cuda()
    r = layers.rms_norm(x, w.cuda(), 1e-6, p=0.5, seed=3)
    first = [int(i) * cols for i in at]
    keep = []
    for f in first:
        words = of.philox(np.arange(f // 8, (f + cols) // 8 + 1, dtype=np.uint64), 3, 0)
        bits = np.stack((words & np.uint64(0xFFFF), words >> np.uint64(16)), 2).reshape(-1)[f % 8:f % 8 + cols]
        keep.append(torch.from_numpy(np.where(bits >= 32768, 2.0, 0.0)))
    keep = torch.stack(keep)
    h = some.double() * keep
    rstd = 1 / torch.sqrt((h * h).mean(-1) + 1e-6)
    y = h * rstd[:, None] * w.double()
    _near(r.h[at.cuda()], h, U[BF] * h.abs())
    _near(r.y[at.cuda()], y, U[BF] * y.abs() + U32 * (_depth(cols) + 8) * y.abs())
    g = layers.rms_norm_grad(r.y, r.h, r.rstd, w.cuda(), p=0.5, seed=3, needs=(True, False, True))
    y, h, q = r.y[at.cuda()].cpu(), r.h[at.cuda()].cpu(), r.rstd[at.cuda()].cpu()
    _, dh, dw, size, size_w = of.rms_norm_grad(y, h, q, w)
    _near(g.x[at.cuda()], dh * keep, U[BF] * (dh * keep).abs() + 2 * U32 * (_depth(cols) + 12) * size)
    _near(g.weight, dw, U[BF] * dw.abs() + U32 * 800 * size_w)  # five rows' terms, and zeros, in sums of at most 513 + 130


def test_on_another_stream(layers):
    """Work queued on a side stream, its inputs made there: the calls follow it."""
    s = torch.cuda.Stream()
    ids, w = _ids(3000, 500, outside=False).cuda(), _new(500, 256, dtype=BF).cuda()
    base = layers.embedding(ids, w)
    want = layers.rms_norm(base * 2, residual=base)
    want_g = layers.embedding_grad(ids, want.y, 500)
    want_n = layers.rms_norm_grad(want.y, want.h, want.rstd, torch.ones(256, device="cuda"))
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(3):
            rows = layers.embedding(ids, w)
            for _ in range(20):
                rows = rows * 1
            got = layers.rms_norm(rows * 2, residual=rows)
            g = layers.embedding_grad(ids, got.y, 500)
            n = layers.rms_norm_grad(got.y, got.h, got.rstd, torch.ones(256, device="cuda"))
    s.synchronize()
    assert torch.equal(got.y, want.y) and torch.equal(got.h, want.h) and torch.equal(g, want_g)
    assert torch.equal(n.weight, want_n.weight) and torch.equal(n.x, want_n.x)


def test_a_captured_training_pass_replays(layers):
    ids, w = _ids(700, 90, common=0.3).cuda(), _new(90, 200, dtype=BF).cuda()
    n = _new(200, dtype=BF, std=0.1, mean=1.0).cuda()
    grad = _new(700, 200, dtype=BF, seed=5).cuda()
    table = torch.zeros(90, 200, device="cuda")

    def step():
        rows = layers.embedding(ids, w, 3.0)
        got = layers.rms_norm(rows, n, residual=rows, p=0.1, seed=9)
        back = layers.rms_norm_grad(grad, got.h, got.rstd, n, p=0.1, seed=9)
        return layers.embedding_grad(ids, back.x, 90, 3.0, out=table), back.weight
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got, weight = step()
    for k in range(4):
        w.mul_(1.5)
        ids.copy_(ids.roll(1))
        graph.replay()
        torch.cuda.synchronize()
        first, second = got.clone(), weight.clone()
        torch.cuda.synchronize()
        want, want_n = step()
        assert torch.equal(first, want) and torch.equal(second, want_n), k


def test_the_example_learns():
    import importlib.util
    import os

    from test_layers_host import ROOT
    spec = importlib.util.spec_from_file_location("train_tokens", os.path.join(ROOT, "examples", "train_tokens.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses = example.train(steps=30, log=None)
    assert abs(losses[0] - np.log(example.VOCAB)) < 1 and losses[-1] < 0.5 * losses[0] and all(np.isfinite(losses))
    assert losses[0] == example.train(steps=1, log=None)[0]
