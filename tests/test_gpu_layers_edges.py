"""The layers' kernels where their ranges, launches and memory end, against the 64-bit oracle; bounds as in test_gpu_layers.py."""
import ctypes as C

import pytest
import torch

from oracle import layers_f64 as of
from test_gpu_layers import BF, F32, OFFSET, SEED, U, U32, _depth, _ids, _near, _new, layers  # noqa: F401
from test_layers_host import EmbeddingGrad

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
