"""The layers' kernels where their ranges, launches and memory end, against the 64-bit oracle; bounds as in test_gpu_layers.py."""
import ctypes as C

import pytest
import torch
import torch.utils.checkpoint

from oracle import layers_f64 as of
from test_gpu_layers import (BF, F8, F32, OFFSET, SEED, U, U32, _depth, _grad_inputs, _ids, _near, _new, _norm_bounds,
                             layers)  # noqa: F401
from test_layers_host import EmbeddingGrad, Norm, NormGrad

pytestmark = pytest.mark.gpu


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _need(query, *sizes):
    from eridiffusion_amd import _lib as L
    need = C.c_uint64()
    L.check(getattr(L.lib(), query)(*[C.c_uint64(n) for n in sizes], C.byref(need)), query)
    return need.value


@pytest.mark.parametrize("rows,cols", [(9, 100), (1600, 200), (900, 520), (5, 2100), (3, 17000)])
@pytest.mark.parametrize("stream", [BF, F32])
@pytest.mark.parametrize("size", [1e15, 3e17, 1e-14])
def test_norm_gradient_of_large_and_small_rows(layers, rows, cols, stream, size):  # noqa: F811
    """rstd^3 does not fit in float32 for the small rows (without eps) and is lost for the large ones; the gradient does."""
    gy, h, w = _new(rows, cols, dtype=F32, seed=1), _new(rows, cols, dtype=stream, std=size), _new(cols, std=0.3, mean=1.0)
    h[:, 0] = size / 4
    gy[:, 0] += 50.0  # the mean of the products is of their order, so that its term counts
    rstd = (1 / torch.sqrt((h.double() ** 2).mean(-1))).float()
    for gh in (None, _new(rows, cols, dtype=stream, seed=2, std=1 / size)):
        dx, dr, dw, terms, terms_w = of.rms_norm_grad(gy, h, rstd, w, gh, 0.3, SEED, OFFSET)
        got = layers.rms_norm_grad(gy.cuda(), h.cuda(), rstd.cuda(), w.cuda(), grad_h=None if gh is None else gh.cuda(), p=0.3, seed=SEED, offset=OFFSET)
        off = U32 * (_depth(cols) + 12) * terms
        _near(got.residual, dr, U[stream] * dr.abs() + off, "residual")
        _near(got.x, dx, 3 * U32 * dx.abs() + 1.5 * off, "x")
        _near(got.weight, dw, U32 * dw.abs() + U32 * (rows + 130) * terms_w, "weight")


@pytest.mark.parametrize("cols", [40, 200, 1000, 1281, 5000, 9000, 20000])
def test_the_norm_gradients_workspace_does_for_fewer_rows(cols):
    most = 0
    for rows in list(range(0, 1100)) + [2 ** k + d for k in range(11, 31) for d in (-1, 0, 1)]:
        need = _need("eri_rms_norm_grad_workspace", rows, cols)
        assert need >= most, rows
        most = need


def test_one_workspace_for_batches_of_all_sizes():
    """Made for the largest; nothing is written behind it."""
    from eridiffusion_amd import _lib as L
    vocab, dim, most = 5000, 768, 16384
    size = _need("eri_embedding_grad_workspace", most, vocab, dim)
    ws, out = torch.empty(size + 64, dtype=torch.uint8, device="cuda"), torch.empty(vocab, dim, device="cuda")
    ws[size:] = 77
    for tokens in (most, most - 1, 9000, 8192, 4095, 1025):
        ids, grad = _ids(tokens, vocab, common=0.2), _new(tokens, dim, dtype=BF)
        want, terms = of.embedding_grad(ids, grad, vocab, 1.0)
        di, dg = ids.cuda(), grad.cuda()
        a = EmbeddingGrad(ids=di.data_ptr(), grad=dg.data_ptr(), out=out.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=size, tokens=tokens, vocab=vocab,
                          dim=dim, padding_id=-1, ids_64=1, grad_dtype=2, out_dtype=0, scale=1.0)
        L.check(L.lib().eri_embedding_grad(C.byref(a), _stream()), "eri_embedding_grad")
        deep = int(torch.bincount(ids[(ids >= 0) & (ids < vocab)]).max()) + 4
        _near(out, want, U32 * want.abs() + deep * U32 * terms, tokens)
        assert bool((ws[size:] == 77).all())


@pytest.mark.parametrize("rows,cols", [(1, 40), (300, 200), (70, 1281), (40, 9001), (900, 1281), (5, 20000)])
@pytest.mark.parametrize("over", ["weight", "x on h", "x on grad_h, residual on grad", "all"])
def test_norm_gradient_over_each_of_its_inputs(rows, cols, over):
    """Every pair that the header allows, with grad_weight wanted, in one launch and in two."""
    from eridiffusion_amd import _lib as L
    (gy, h, gh), w = (_new(rows, cols, seed=s) for s in range(3)), _new(cols, std=0.3, mean=1.0)
    rstd = (1 / torch.sqrt((h.double() ** 2).mean(-1) + 1e-6)).float()
    dx, dr, dw, size, size_w = of.rms_norm_grad(gy, h, rstd, w, gh, 0.25, SEED, OFFSET)
    g, hh, r, q, ww = gy.cuda(), h.cuda(), gh.cuda(), rstd.cuda(), w.cuda()
    new = lambda t: torch.empty_like(t)  # noqa: E731
    x, res, weight = {"weight": (new(g), new(g), ww), "x on h": (hh, new(g), new(ww)), "x on grad_h, residual on grad": (r, g, new(ww)), "all": (hh, g, ww)}[over]
    need = _need("eri_rms_norm_grad_workspace", rows, cols)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    a = NormGrad(grad=g.data_ptr(), h=hh.data_ptr(), rstd=q.data_ptr(), weight=ww.data_ptr(), grad_h=r.data_ptr(), grad_x=x.data_ptr(), grad_residual=res.data_ptr(),
                 grad_weight=weight.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=need, rows=rows, cols=cols)
    a.key.seed, a.key.offset, a.key.p = SEED, OFFSET, 0.25
    L.check(L.lib().eri_rms_norm_grad(C.byref(a), _stream()), "eri_rms_norm_grad")
    off = U32 * (_depth(cols) + 12) * size
    _near(res, dr, U32 * dr.abs() + off, "residual")
    _near(x, dx, 3 * U32 * dx.abs() + 1.4 * off, "x")
    _near(weight, dw, U32 * dw.abs() + U32 * (rows + 130) * size_w, "weight")


@pytest.mark.parametrize("cols", [40, 1001, 6000, 34000])
@pytest.mark.parametrize("y_on,h_on", [("residual", "x"), ("residual", None), (None, "x")])
def test_norm_over_each_of_its_inputs(cols, y_on, h_on):
    from eridiffusion_amd import _lib as L
    x, r, w = _new(9, cols), _new(9, cols, seed=1), _new(cols, std=0.3, mean=1.0)
    y, h, rstd = of.rms_norm(x, w, 1e-6, r, 0.25, SEED, OFFSET)
    dev = {"x": x.cuda(), "residual": r.cuda(), None: torch.empty(9, cols, device="cuda")}
    dw = w.cuda()
    a = Norm(x=dev["x"].data_ptr(), residual=dev["residual"].data_ptr(), weight=dw.data_ptr(), y=dev[y_on].data_ptr(), h=dev[h_on].data_ptr(), rows=9, cols=cols, eps=1e-6)
    a.key.seed, a.key.offset, a.key.p = SEED, OFFSET, 0.25
    L.check(L.lib().eri_rms_norm(C.byref(a), _stream()), "eri_rms_norm")
    off_h, off_y = _norm_bounds(x, w, r, 0.25, y, h, rstd, cols)
    _near(dev[h_on], h, U32 * h.abs() + off_h, "h")
    _near(dev[y_on], y, U32 * y.abs() + off_y, "y")


def test_under_a_dispatch_mode_that_only_looks_on(layers):  # noqa: F811
    from torch.utils._python_dispatch import TorchDispatchMode

    class Count(TorchDispatchMode):
        seen = 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen += 1
            return func(*args, **(kwargs or {}))
    x, w = _new(5, 40).cuda(), _new(40).cuda().requires_grad_()
    want = layers.rms_norm(x, w, residual=x, p=0.2, seed=1)
    with Count() as mode:
        got = layers.rms_norm(x, w, residual=x, p=0.2, seed=1)
    assert mode.seen and torch.equal(got.y, want.y) and torch.equal(got.h, want.h)

    def block(x, w):
        return layers.rms_norm(torch.nn.functional.gelu(x), w, residual=x, p=0.2, seed=1).y
    grads = []
    for run in (block, lambda *a: torch.utils.checkpoint.checkpoint(block, *a, use_reentrant=False)):
        xs, ws = x.clone().requires_grad_(), w.detach().clone().requires_grad_()
        run(xs, ws).square().sum().backward()
        grads.append((xs.grad, ws.grad))
    assert torch.equal(grads[0][0], grads[1][0]) and torch.equal(grads[0][1], grads[1][1])


def test_outputs_that_overlap_inputs_are_refused(layers):  # noqa: F811
    w, g = _new(12, 40).cuda(), _new(12, 40).cuda()
    ids = torch.randperm(12).cuda()
    flat = _new(1000).cuda()
    wide = _new(12, 90).cuda()
    for what, call in [
            ("weight", lambda: layers.embedding(ids, w, out=w)), ("weight", lambda: layers.embedding(ids[:5], w, out=w[:5])),
            ("weight", lambda: layers.embedding(ids[:1], w, out=w[11:])), ("weight", lambda: layers.embedding(ids, wide[:, :40], out=wide[:, 39:79])),
            ("weight", lambda: layers.embedding(ids, wide[:, 50:], out=wide[:, 11:51])), ("weight", lambda: layers.embedding(ids[:3], wide[:, :40], out=wide[::2][:3, 50:])),
            ("ids", lambda: layers.embedding(flat[:24].view(torch.long), w, out=flat[20:500].view(12, 40))),
            ("grad", lambda: layers.embedding_grad(ids, g, 12, out=g)), ("grad", lambda: layers.embedding_grad(ids[:6], g[:6], 6, out=g[5:11])),
            ("grad", lambda: layers.embedding_grad(ids, g.view(BF)[:, :40], 12, out=g)),
            ("grad", lambda: layers.embedding_grad(ids, wide[:, 45:85], 12, out=wide[:, 10:50], accumulate=True)),
            ("ids", lambda: layers.embedding_grad(flat[476:500].view(torch.long), g, 12, out=flat[:480].view(12, 40))),
            ("x", lambda: layers.dropout(w[1:], 0.5, 1, out=w[:-1])), ("x", lambda: layers.dropout(flat[1:], 0.5, 1, out=flat[:-1])),
            ("x", lambda: layers.dropout(wide[:, :40], 0.5, 1, out=wide[:, 1:41])), ("x", lambda: layers.dropout(wide[:6, :40], 0.5, 1, out=wide[::2, :40])),
            ("x", lambda: layers.dropout(flat[:480].view(12, 40), 0.5, 1, out=flat[:960].view(12, 80)[:, :40])),
            ("offset", lambda: layers.dropout(w, 0.5, 1, flat[500:502].view(torch.long), out=flat[30:510].view(12, 40)))]:
        before = [t.clone() for t in (w, g, flat, wide)]
        with pytest.raises(ValueError, match="out overlaps " + what):
            call()
        assert all(torch.equal(a, b) for a, b in zip(before, (w, g, flat, wide)))


def test_outputs_beside_their_inputs_are_not_refused(layers):  # noqa: F811
    wide, ids = _new(12, 90).cuda(), torch.randperm(12).cuda()
    a, b, one = wide[:, :40], wide[:, 40:80], wide[3, 80:].clone()
    want = a[ids]
    assert torch.equal(layers.embedding(ids, a, out=b), want)
    want = layers.embedding_grad(ids, b, 12)
    assert torch.equal(layers.embedding_grad(ids, b, 12, out=a), want)
    want = layers.dropout(a, 0.5, 1)
    assert torch.equal(layers.dropout(a, 0.5, 1, out=b), want) and torch.equal(layers.dropout(a, 0.5, 1, out=a), want)  # beside it, then over itself
    assert torch.equal(layers.dropout(wide[:6, :40], 0.5, 2, out=wide[6:, :40]), layers.dropout(wide[:6, :40], 0.5, 2))  # rows behind
    assert torch.equal(layers.embedding(ids[:1], a, out=wide[5:6, 50:]), a[ids[:1]]) and torch.equal(wide[3, 80:], one)  # one row between the others
    assert torch.equal(layers.embedding(ids, wide[2:3, :40], out=wide[:, 45:85])[ids != 0], torch.zeros(11, 40, device="cuda"))  # and several beside one
    square = _new(30, 30).cuda()
    want = layers.dropout(square.t(), 0.5, 1)  # no rows: what the kernel reads is a copy
    assert torch.equal(layers.dropout(square.t(), 0.5, 1, out=square), want)
    empty = wide[:0]
    assert layers.dropout(empty, 0.5, 1, out=empty) is empty


@pytest.mark.parametrize("cols", [2 ** 27 + 70, 2 ** 28 + 100])
def test_weight_gradient_of_a_very_long_row(layers, cols):  # noqa: F811
    """16 threads to a column, and a launch counts its threads in 32 bits.  One row: each element is a product of three."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    g, h = (torch.randn(1, cols, generator=gen, device="cuda", dtype=BF) for _ in range(2))
    got = layers.rms_norm_grad(g, h, torch.full((1,), 0.75, device="cuda"), torch.ones(cols, device="cuda"), needs=(False, False, True)).weight
    for at in range(0, cols, 2 ** 26):
        part = slice(at, at + 2 ** 26)
        want = g[0, part].double() * h[0, part].double() * 0.75
        assert bool(((got[part].double() - want).abs() <= 4 * U32 * want.abs()).all()), at


def test_table_gradient_of_the_most_tokens(layers):  # noqa: F811
    """2^31 - 1 of them, and the last to be joined stand in a launch of their own.  Sums of ones below 2^24 are exact."""
    tokens, vocab = 2 ** 31 - 1, 1000
    ids = torch.randint(0, vocab, (tokens,), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda", dtype=torch.int32)
    ids[-5:] = vocab - 1
    grad = torch.ones(tokens, 1, device="cuda", dtype=BF)
    grad[-5:] = 3
    got = layers.embedding_grad(ids, grad, vocab, dtype=F32)[:, 0]
    want = sum(torch.bincount(part, minlength=vocab) for part in ids.split(2 ** 27))
    want[vocab - 1] += 10
    assert torch.equal(got.double(), want.double())


# ---------------------------------------------------------------------------------------------------------------
# launches and layouts that only certain sizes reach
# ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,out", [(BF, BF), (BF, F32), (F32, F32)])
@pytest.mark.parametrize("tokens,vocab,dim,common", [(20000, 5000, 16, 0.9), (12000, 900, 40, 1.0), (30001, 3000, 300, 0.6)])
def test_table_gradient_of_a_batch_with_most_tokens_on_one_id(layers, dtype, out, tokens, vocab, dim, common):  # noqa: F811
    """More than 512 tokens of a bucket in a wave's share of the ids: the sort looks at them a second time."""
    ids, grad = _ids(tokens, vocab, common=common), _new(tokens, dim, dtype=dtype)
    share = (tokens + 1023) // 1024 * 64
    assert int((ids[share:2 * share] == vocab // 2).sum()) > 512
    deep = int((ids == vocab // 2).sum()) + 4
    for pad in (None, 3):
        want, size = of.embedding_grad(ids, grad, vocab, 0.75, pad)
        got = layers.embedding_grad(ids.cuda(), grad.cuda(), vocab, 0.75, padding_id=pad, dtype=out)
        _near(got, want, U[out] * want.abs() + deep * U32 * size, pad)
        assert torch.equal(got, layers.embedding_grad(ids.int().cuda(), grad.cuda(), vocab, 0.75, padding_id=pad, dtype=out))
        old = _new(vocab, dim, dtype=out, seed=3)
        into = layers.embedding_grad(ids.cuda(), grad.cuda(), vocab, 0.75, padding_id=pad, out=old.cuda(), accumulate=True)
        _near(into, want + old.double(), U[out] * (want + old.double()).abs() + (deep + 1) * U32 * (size + old.double().abs()), "accumulate")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("out,vocab", [(BF, 270000), (F32, 140000)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_table_gradient_that_reads_grad_past_the_caches(layers, dtype, out, vocab, accumulate):  # noqa: F811
    """A table of more than 256 MB, rows of an odd length in two tiles, runs of one piece and of many."""
    tokens, dim, some = 3000, 513, 400
    rows = torch.randperm(vocab, generator=torch.Generator().manual_seed(1))[:some].sort().values  # the rows that are named
    local, grad = _ids(tokens, some, common=0.3, outside=False), _new(tokens, dim, dtype=dtype)
    ids = torch.where(torch.arange(tokens) % 97 == 5, -1, rows[local])
    want, size = of.embedding_grad(torch.where(ids < 0, -1, local), grad, some, 1.5)
    deep = int(torch.bincount(local).max()) + 5
    table = torch.full((vocab, dim), 2.0, dtype=out, device="cuda") if accumulate else None
    got = layers.embedding_grad(ids.cuda(), grad.cuda(), vocab, 1.5, dtype=out, out=table, accumulate=accumulate)
    base = 2.0 if accumulate else 0.0
    _near(got[rows.cuda()], want + base, U[out] * (want + base).abs() + deep * U32 * (size + base))
    rest = torch.ones(vocab, dtype=torch.bool, device="cuda")
    rest[ids[ids >= 0].cuda()] = False
    assert bool((got[rest] == base).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("tokens,dim", [(140000, 40), (140000, 7), (40000, 200), (4500, 1300), (5000, 4099), (2 ** 22 + 5, 8), (2 ** 22 + 5, 70)])
def test_lookup_of_many_tokens(layers, dtype, tokens, dim):  # noqa: F811
    """Several rows at a time in a thread, for each number of lanes to a row, and more tokens than a launch takes."""
    w, ids = _new(300, dim, dtype=dtype).cuda(), _ids(tokens, 300).cuda()
    fits = (ids >= 0) & (ids < 300)
    want = torch.where(fits[:, None], w[torch.where(fits, ids, 0)], 0)
    for some in (ids, ids.int()):
        assert torch.equal(layers.embedding(some, w), want)
    back = torch.full((tokens, dim + 3), 7.0, dtype=dtype, device="cuda")
    layers.embedding(ids, w, 2.0, out=back[:, 1:dim + 1])
    assert torch.equal(back[:, 1:dim + 1], want * 2) and bool((back[:, 0] == 7).all()) and bool((back[:, dim + 1:] == 7).all())


@pytest.mark.parametrize("group", [0, 128])
def test_norm_of_more_rows_than_a_launch_takes(layers, group):  # noqa: F811
    rows, cols = 2 ** 21 + 5, 8
    x, r, w = _new(rows, cols, dtype=BF), _new(rows, cols, dtype=BF, seed=1), _new(cols, std=0.3, mean=1.0)
    y, h, rstd = of.rms_norm(x, w, 1e-6, r, 0.3, SEED, OFFSET)
    off_h, off_y = _norm_bounds(x, w, r, 0.3, y, h, rstd, cols)
    got = layers.rms_norm(x.cuda(), w.cuda(), 1e-6, residual=r.cuda(), p=0.3, seed=SEED, offset=OFFSET)
    _near(got.y, y, U[BF] * y.abs() + off_y, "y")
    _near(got.h, h, U[BF] * h.abs() + off_h, "h")
    _near(got.rstd, rstd, rstd * U32 * (_depth(cols) + 8) + rstd ** 3 * (off_h * h.abs()).mean(-1), "rstd")
    whole = layers.rms_norm(x.cuda(), w.cuda(), dtype=F8, scale_group=group)
    for part in (slice(0, 70), slice(2 ** 21 - 9, 2 ** 21 + 5)):
        some = layers.rms_norm(x[part].cuda(), w.cuda(), dtype=F8, scale_group=group)
        assert torch.equal(whole.y[part].view(torch.uint8), some.y.view(torch.uint8))
        assert torch.equal(whole.scales[part], some.scales) and torch.equal(whole.rstd[part], some.rstd)


@pytest.mark.parametrize("cols", [1025, 1281, 2048, 2500, 4095, 5001, 6144, 6150, 8192, 9001, 12288, 12290])
@pytest.mark.parametrize("dtype,out", [(BF, BF), (BF, F8), (F32, BF), (F32, F32)])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_norm_without_a_residual(layers, cols, dtype, out, p):  # noqa: F811
    """Layouts of their own where the row moves few bytes."""
    rows = 5
    x, w = _new(rows, cols, dtype=dtype), _new(cols, dtype=dtype, std=0.3, mean=1.0)
    y, h, rstd = of.rms_norm(x, w, 1e-6, None, p, SEED, OFFSET)
    off_h, off_y = _norm_bounds(x, w, None, p, y, h, rstd, cols)
    got = layers.rms_norm(x.cuda(), w.cuda(), 1e-6, p=p, seed=SEED, offset=OFFSET, dtype=out)
    _near(got.rstd, rstd, rstd * U32 * (_depth(cols) + 8) + rstd ** 3 * (off_h * h.abs()).mean(-1), "rstd")
    _near(got.h, h, U[dtype] * h.abs() + off_h, "h")
    if out != F8:
        _near(got.y, y, U[out] * y.abs() + off_y, "y")
        return
    scales = of.scales_of(y, 0)
    off_scales = off_y.amax(-1, keepdim=True) / of.F8_MAX + 2 * U32 * scales
    _near(got.scales, scales, off_scales, "scales")
    q = y / scales
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
    _near(got.y.float(), q, 0.5 * step + 2 * (off_y / scales + q.abs() * (off_scales / scales + 3 * U32)), "codes")


@pytest.mark.parametrize("rows,cols", [(2000, 200), (2000, 400), (1537, 129), (1600, 512), (600, 9001), (800, 9001), (770, 16384)])
@pytest.mark.parametrize("dtype,stream,w", [(BF, BF, F32), (F32, F32, F32), (BF, F32, BF)])
def test_norm_gradient_of_more_rows_than_workgroups(layers, rows, cols, dtype, stream, w):  # noqa: F811
    """Every width whose sums the waves of a workgroup join, and long rows several to a workgroup, in one launch and in two."""
    gy, h, rstd, weight, gh = _grad_inputs(rows, cols, dtype, stream, w)
    dx, dr, dw, size, size_w = of.rms_norm_grad(gy, h, rstd, weight, gh, 0.3, SEED, OFFSET)
    got = layers.rms_norm_grad(gy.cuda(), h.cuda(), rstd.cuda(), weight.cuda(), grad_h=gh.cuda(), p=0.3, seed=SEED, offset=OFFSET, dtype=dtype)
    off = U32 * (_depth(cols) + 12) * size
    _near(got.residual, dr, U[stream] * dr.abs() + off, "residual")
    _near(got.x, dx, U[dtype] * dx.abs() + 1.5 * off + 2 * U32 * dx.abs(), "x")
    _near(got.weight, dw, U[w] * dw.abs() + U32 * (rows + 130) * size_w, "weight")
