"""The layers' kernels where their ranges, launches and memory end, against the 64-bit oracle; bounds as in test_gpu_layers.py."""
import ctypes as C

import pytest
import torch

from oracle import layers_f64 as of
from test_gpu_layers import BF, F32, OFFSET, SEED, U, U32, _depth, _near, _new, layers  # noqa: F401

pytestmark = pytest.mark.gpu


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
