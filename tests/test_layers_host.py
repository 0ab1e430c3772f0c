"""The layers' host side without a GPU: exported symbols, refusals of the C functions with their codes, the oracle's
generator against its published vectors and the oracle's gradients against differences."""
import ctypes as C
import os
import re

import numpy as np
import pytest
import torch

import oracle_c as oc
from eridiffusion_amd import _lib as L
from eridiffusion_amd import _layers_face, layers
from oracle import layers_f64 as of

ROOT = oc.ROOT
NULL, ALIGN, EMPTY, DTYPE, ARG, TOO_LARGE = -1, -2, -3, -4, -6, -7
F32, F16, BF16, F8 = 0, 1, 2, 16


class Key(C.Structure):
    _fields_ = [("seed", C.c_uint64), ("offset", C.c_uint64), ("offset_ptr", C.c_void_p), ("p", C.c_double)]


def _struct(fields):
    kinds = {"p": C.c_void_p, "u": C.c_uint64, "i": C.c_int32, "l": C.c_int64, "f": C.c_float, "k": Key}
    return type("S", (C.Structure,), {"_fields_": [(n, kinds[k]) for n, k in (w.split(":") for w in fields.split())]})


Embedding = _struct("ids:p table:p out:p tokens:u vocab:u dim:u table_stride:u out_stride:u ids_64:i dtype_tag:i scale:f reserved:i")
EmbeddingGrad = _struct("ids:p grad:p out:p workspace:p workspace_bytes:u tokens:u vocab:u dim:u grad_stride:u out_stride:u padding_id:l ids_64:i "
                        "grad_dtype:i out_dtype:i accumulate:i scale:f reserved:i")
Dropout = _struct("x:p y:p rows:u cols:u x_stride:u y_stride:u key:k dtype_tag:i reserved:i")
Norm = _struct("x:p residual:p weight:p y:p h:p rstd:p scales:p rows:u cols:u x_stride:u residual_stride:u y_stride:u h_stride:u key:k eps:f "
               "x_dtype:i residual_dtype:i weight_dtype:i y_dtype:i scale_group:i")
NormGrad = _struct("grad:p h:p rstd:p weight:p grad_h:p grad_x:p grad_residual:p grad_weight:p workspace:p workspace_bytes:u rows:u cols:u "
                   "grad_stride:u h_stride:u grad_h_stride:u grad_x_stride:u grad_residual_stride:u key:k grad_dtype:i h_dtype:i x_dtype:i "
                   "weight_dtype:i grad_weight_dtype:i reserved:i")


def _header():
    return open(os.path.join(ROOT, "include", "eri_layers.h")).read()


def _declared():
    return set(re.findall(r"^int (eri_[a-z0-9_]+)\s*\(", _header(), re.M))


def test_library_exports_every_declared_symbol():
    lib = L.lib()
    assert len(_declared()) == 7
    for name in _declared():
        assert hasattr(lib, name), name


def test_rust_declares_the_same_functions():
    rust = open(os.path.join(ROOT, "eridiffusion_amd", "rust", "eri_layers_sys.rs")).read()
    assert set(re.findall(r"pub fn (eri_[a-z0-9_]+)\s*\(", rust)) == _declared()


@pytest.mark.parametrize("kind,name", [(Embedding, "EriEmbedding"), (EmbeddingGrad, "EriEmbeddingGrad"), (Dropout, "EriDropout"),
                                       (Norm, "EriRmsNorm"), (NormGrad, "EriRmsNormGrad")])
def test_structs_of_these_tests_and_of_rust_have_the_headers_fields(kind, name):
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), re.sub(r"/\*.*?\*/", "", _header(), flags=re.S), re.S).group(1)
    fields = [n.strip().lstrip("*") for line in body.split(";") if line.strip() for n in re.sub(r"^\s*(const )?\w+ ", "", line.strip()).split(",")]
    assert fields == [f for f, _ in kind._fields_]
    rust = open(os.path.join(ROOT, "eridiffusion_amd", "rust", "eri_layers_sys.rs")).read()
    assert re.findall(r"pub (\w+):", re.search(r"pub struct %s \{(.*?)\}" % name, rust, re.S).group(1)) == fields


def _refused(call, args):
    fn = getattr(L.lib(), call)
    fn.restype, fn.argtypes = C.c_int, [C.c_void_p, C.c_void_p]
    rc = fn(C.byref(args) if args is not None else None, None)
    message = L.lib().eri_last_error().decode()
    assert rc == 0 or message.startswith(call + ":"), message
    return rc


def _with(kind, base, **changes):
    a = kind(**base)
    for k, v in changes.items():
        if k in ("p", "offset_ptr"):
            setattr(a.key, k, v)
        else:
            setattr(a, k, v)
    return a


def test_refusals_of_the_lookup():
    base = dict(ids=0x1000, table=0x2000, out=0x3000, tokens=4, vocab=8, dim=16, ids_64=1, dtype_tag=BF16, scale=1.0)
    assert _refused("eri_embedding", None) == NULL
    for code, change in [(NULL, dict(ids=0)), (NULL, dict(table=0)), (NULL, dict(out=0)), (ALIGN, dict(ids=0x1004)), (ALIGN, dict(table=0x2001)),
                         (ALIGN, dict(out=0x3002, dtype_tag=F32)), (EMPTY, dict(vocab=0)), (EMPTY, dict(dim=0)), (DTYPE, dict(dtype_tag=F16)),
                         (DTYPE, dict(ids_64=2)), (DTYPE, dict(dtype_tag=F8)), (ARG, dict(table_stride=15)), (ARG, dict(out_stride=1)),
                         (ARG, dict(out_stride=2 ** 41)), (TOO_LARGE, dict(tokens=2 ** 31)), (TOO_LARGE, dict(vocab=2 ** 31)),
                         (TOO_LARGE, dict(dim=2 ** 40))]:
        assert _refused("eri_embedding", _with(Embedding, base, **change)) == code, change
    assert _refused("eri_embedding", _with(Embedding, base, tokens=0, ids=0, table=0, out=0)) == 0  # nothing to do


def test_refusals_of_the_tables_gradient():
    need = C.c_uint64()
    fn = L.lib().eri_embedding_grad_workspace
    fn.restype, fn.argtypes = C.c_int, [C.c_uint64] * 3 + [C.c_void_p]
    assert fn(4, 8, 16, C.byref(need)) == 0 and need.value == 0  # few tokens need none
    assert fn(4000, 8, 16, C.byref(need)) == 0 and need.value > 0
    assert fn(4, 8, 16, None) == NULL and fn(4, 0, 16, C.byref(need)) == EMPTY and fn(2 ** 31, 8, 16, C.byref(need)) == TOO_LARGE
    base = dict(ids=0x1000, grad=0x2000, out=0x3000, workspace=0x4000, workspace_bytes=need.value, tokens=4000, vocab=8, dim=16, padding_id=-1, ids_64=0,
                grad_dtype=BF16, out_dtype=F32, scale=1.0)
    assert _refused("eri_embedding_grad", None) == NULL
    for code, change in [(NULL, dict(ids=0)), (NULL, dict(grad=0)), (NULL, dict(out=0)), (NULL, dict(workspace=0)), (ALIGN, dict(ids=0x1002)),
                         (ALIGN, dict(grad=0x2001)), (ALIGN, dict(out=0x3002)), (ALIGN, dict(workspace=0x4008)), (EMPTY, dict(vocab=0)), (EMPTY, dict(dim=0)),
                         (DTYPE, dict(grad_dtype=F16)), (DTYPE, dict(out_dtype=F8)), (DTYPE, dict(ids_64=-1)), (ARG, dict(grad_stride=15)),
                         (ARG, dict(out_stride=15)), (ARG, dict(workspace_bytes=need.value - 1)), (TOO_LARGE, dict(tokens=2 ** 31))]:
        assert _refused("eri_embedding_grad", _with(EmbeddingGrad, base, **change)) == code, change


@pytest.mark.parametrize("dim", [1, 7, 40, 64, 100, 256, 257, 768, 1155, 4096, 20000])
def test_the_tables_gradients_workspace_does_for_fewer_tokens(dim):
    """Whoever makes it for the largest batch has enough for a shorter last one."""
    fn, need, most = L.lib().eri_embedding_grad_workspace, C.c_uint64(), 0
    fn.restype, fn.argtypes = C.c_int, [C.c_uint64] * 3 + [C.c_void_p]
    for vocab in (8, 49408):
        most = 0
        for tokens in sorted({t for k in range(24) for t in range(max(0, 2 ** k - 40), 2 ** k + 41)} | set(range(0, 40000, 7)) | {9000, 2 ** 31 - 1}):
            assert fn(tokens, vocab, dim, C.byref(need)) == 0
            assert need.value >= most, (tokens, need.value, most)
            most = need.value


def test_refusals_of_dropout():
    base = dict(x=0x1000, y=0x2000, rows=4, cols=16, dtype_tag=F32)
    assert _refused("eri_dropout", None) == NULL
    for code, change in [(NULL, dict(x=0)), (NULL, dict(y=0)), (ALIGN, dict(x=0x1002)), (ALIGN, dict(y=0x2001)), (ALIGN, dict(offset_ptr=0x1004)),
                         (DTYPE, dict(dtype_tag=F16)), (ARG, dict(p=-0.1)), (ARG, dict(p=1.001)), (ARG, dict(p=float("nan"))), (ARG, dict(x_stride=15)),
                         (ARG, dict(y_stride=1)), (TOO_LARGE, dict(rows=2 ** 31)), (TOO_LARGE, dict(cols=2 ** 40 + 1))]:
        assert _refused("eri_dropout", _with(Dropout, base, **change)) == code, change
    assert _refused("eri_dropout", _with(Dropout, base, rows=0, x=0, y=0)) == 0
    assert _refused("eri_dropout", _with(Dropout, base, cols=0, x=0, y=0)) == 0


def test_refusals_of_the_norm():
    base = dict(x=0x1000, residual=0x2000, weight=0x3000, y=0x4000, h=0x5000, rstd=0x6000, scales=0x7000, rows=4, cols=16, eps=1e-6, x_dtype=BF16,
                residual_dtype=F32, weight_dtype=BF16, y_dtype=F8, scale_group=128)
    assert _refused("eri_rms_norm", None) == NULL
    for code, change in [(NULL, dict(x=0)), (NULL, dict(y=0)), (NULL, dict(scales=0)), (ALIGN, dict(x=0x1001)), (ALIGN, dict(residual=0x2002)),
                         (ALIGN, dict(weight=0x3001)), (ALIGN, dict(h=0x5002)), (ALIGN, dict(rstd=0x6002)), (ALIGN, dict(scales=0x7001)),
                         (ALIGN, dict(y=0x4001, y_dtype=BF16, scale_group=0)), (EMPTY, dict(cols=0)), (DTYPE, dict(x_dtype=F16)), (DTYPE, dict(x_dtype=F8)),
                         (DTYPE, dict(residual_dtype=F16)), (DTYPE, dict(weight_dtype=3)), (DTYPE, dict(y_dtype=F16, scale_group=0)), (ARG, dict(scale_group=64)),
                         (ARG, dict(y_dtype=F32)), (ARG, dict(eps=-1e-6)), (ARG, dict(eps=float("nan"))), (ARG, dict(p=2.0)), (ARG, dict(x_stride=15)),
                         (ARG, dict(h_stride=15)), (TOO_LARGE, dict(rows=2 ** 31)), (TOO_LARGE, dict(cols=2 ** 31))]:
        assert _refused("eri_rms_norm", _with(Norm, base, **change)) == code, change
    assert _refused("eri_rms_norm", _with(Norm, base, rows=0, x=0, y=0)) == 0


def test_refusals_of_the_norms_gradient():
    base = dict(grad=0x1000, h=0x2000, rstd=0x3000, weight=0x4000, grad_h=0x5000, grad_x=0x6000, grad_residual=0x7000, grad_weight=0, rows=4, cols=16,
                grad_dtype=BF16, h_dtype=F32, x_dtype=BF16, weight_dtype=BF16, grad_weight_dtype=BF16)
    assert _refused("eri_rms_norm_grad", None) == NULL
    for code, change in [(NULL, dict(grad=0)), (NULL, dict(h=0)), (NULL, dict(rstd=0)), (ALIGN, dict(grad=0x1001)), (ALIGN, dict(h=0x2002)),
                         (ALIGN, dict(rstd=0x3002)), (ALIGN, dict(weight=0x4001)), (ALIGN, dict(grad_h=0x5002)), (ALIGN, dict(grad_x=0x6001)),
                         (ALIGN, dict(grad_residual=0x7002)), (EMPTY, dict(cols=0)), (DTYPE, dict(grad_dtype=F8)), (DTYPE, dict(h_dtype=F16)),
                         (DTYPE, dict(x_dtype=F16)), (DTYPE, dict(weight_dtype=F8)), (DTYPE, dict(grad_weight=0x8000, grad_weight_dtype=F8)), (ARG, dict(p=-1)),
                         (ARG, dict(grad_stride=15)), (ARG, dict(grad_residual_stride=15)), (TOO_LARGE, dict(rows=2 ** 31))]:
        assert _refused("eri_rms_norm_grad", _with(NormGrad, base, **change)) == code, change


def test_the_python_calls_refuse_host_tensors_and_other_types():
    x, ids = torch.zeros(4, 8), torch.zeros(4, dtype=torch.long)
    for call in [lambda: layers.dropout(x, 0.1, 1), lambda: layers.rms_norm(x), lambda: layers.embedding(ids, x),
                 lambda: layers.embedding_grad(ids, x, 8), lambda: layers.rms_norm_grad(x, x, x[:, 0])]:
        with pytest.raises(ValueError, match="take device tensors"):
            call()
    with pytest.raises(TypeError):
        layers.dropout([1.0], 0.1, 1)
    with pytest.raises(TypeError):
        _layers_face.dropout(x)


def _calls(x, ids):
    """Each call, with x wherever a tensor of floats may stand."""
    w, q = x[0], x[:, 0]
    return [lambda: layers.dropout(x, 0.1, 1), lambda: layers.rms_norm(x), lambda: layers.rms_norm(x, w, residual=x), lambda: layers.embedding(ids, x),
            lambda: layers.embedding_grad(ids, x, 8), lambda: layers.rms_norm_grad(x, x, q)]


def test_forward_mode_tangents_are_refused():
    """They would be lost without a word: torch reads a result without a tangent as one that does not change."""
    from torch.autograd import forward_ad as fa
    x, t, ids = torch.zeros(4, 8), torch.ones(4, 8), torch.zeros(4, dtype=torch.long)
    with fa.dual_level():
        d = fa.make_dual(x, t)
        for call in _calls(d, ids):
            with pytest.raises(ValueError, match="forward-mode tangent"):
                call()
        for call in _calls(fa.make_dual(x.clone().requires_grad_(), t), ids):  # beside a gradient that is recorded
            with pytest.raises(ValueError, match="forward-mode tangent"):
                call()
        for call in _calls(fa.unpack_dual(d).primal, ids):
            with pytest.raises(ValueError, match="take device tensors"):
                call()
    with pytest.raises(ValueError, match="no plain tensor|forward-mode tangent"):
        torch.func.jvp(lambda x: layers.dropout(x, 0.1, 1), (x,), (t,))


def test_tracers_are_refused():
    """What they record is the making of the outputs; the program would return memory that nobody wrote."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    x, ids = torch.zeros(4, 8), torch.zeros(4, dtype=torch.long)
    for k, call in enumerate(_calls(x, ids)):
        for trace in (lambda f: torch.jit.trace(f, (x, ids)), lambda f: make_fx(f)(x, ids), lambda f: make_fx(f, tracing_mode="fake")(x, ids)):
            with pytest.raises(ValueError, match="cannot be traced"):
                trace(lambda a, b: _calls(a, b)[k]())
        with FakeTensorMode(), pytest.raises(ValueError, match="cannot be traced"):
            call()
        with pytest.raises(ValueError, match="take device tensors"):  # and not what comes after them
            call()


def _words(got):
    return ["%08x" % int(w) for w in got[0]]


def test_the_oracles_generator_gives_the_published_vectors():
    """The three vectors that its authors distribute with the generator."""
    one = lambda c: np.array([c], np.uint64)  # noqa: E731
    full = 2 ** 64 - 1
    assert _words(of.philox(one(0), 0, 0)) == ["6627e8d5", "e169c58d", "bc57ac4c", "9b00dbd8"]
    assert _words(of.philox(one(full), full, full)) == ["408f276d", "41c83b0e", "a20bc7c6", "6d5451fd"]
    assert _words(of.philox(one(0x85A308D3243F6A88), 0x299F31D0A4093822, 0x0370734413198A2E)) == ["d16cfe09", "94fdcceb", "5001e420", "24126ea1"]


@pytest.mark.parametrize("p", [0.1, 0.5])
def test_the_oracle_keeps_the_share_and_the_mean(p):
    k = of.kept((1000, 257), p, 7, 3)
    n = k.numel()
    assert abs((k == 0).double().mean().item() - p) < 5 * (p * (1 - p) / n) ** 0.5  # five standard deviations
    assert not torch.equal(k, of.kept((1000, 257), p, 7, 4)) and not torch.equal(k, of.kept((1000, 257), p, 8, 3))
    assert torch.equal(k.reshape(-1)[:4000], of.kept((4000,), p, 7, 3))  # an element's place decides, not the shape


@pytest.mark.parametrize("p", [0.0, 0.3])
@pytest.mark.parametrize("residual", [False, True])
def test_the_oracles_gradients_are_the_differences_of_its_forward(p, residual):
    g = torch.Generator().manual_seed(5)
    new = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x, w, r, gy, gh = new(3, 11), new(11), new(3, 11) if residual else None, new(3, 11), new(3, 11)
    dirs = [new(3, 11), new(3, 11), new(11)]

    def loss(t):
        y, h, _ = of.rms_norm(x + t * dirs[0], w + t * dirs[2], 1e-3, r + t * dirs[1] if residual else None, p, 9, 2)
        return (y * gy).sum() + (h * gh).sum()
    _, h, rstd = of.rms_norm(x, w, 1e-3, r, p, 9, 2)
    dx, dr, dw, _, _ = of.rms_norm_grad(gy, h, rstd, w, gh, p, 9, 2)
    want = (dx * dirs[0]).sum() + ((dr * dirs[1]).sum() if residual else 0) + (dw * dirs[2]).sum()
    t = 1e-5  # the difference's own error is of the order t^2
    assert abs((loss(t) - loss(-t)) / (2 * t) - want) < 1e-7 * (1 + abs(want))
