"""The losses' host side without a GPU: exported symbols, refusals of the C functions with their codes, workspaces, the Python calls'
refusals, and the oracle's gradients against differences."""
import ctypes as C
import math
import os
import re

import pytest
import torch

import oracle_c as oc
from eridiffusion_amd import _lib as L
from eridiffusion_amd import losses
from oracle import losses_f64 as of
from test_layers_host import ALIGN, ARG, BF16, DTYPE, EMPTY, F16, F32, F8, NULL, TOO_LARGE, _refused, _struct, _with

ROOT = oc.ROOT

Logprobs = _struct("logits:p ids:p logprob:p entropy:p stats:p top:p top_ids:p workspace:p workspace_bytes:u rows:u vocab:u logits_stride:u temperature:f "
                   "ids_64:i dtype_tag:i top_n:i")
LogprobsGrad = _struct("logits:p ids:p stats:p grad:p grad_entropy:p entropy:p out:p rows:u vocab:u logits_stride:u out_stride:u temperature:f ids_64:i "
                       "dtype_tag:i out_dtype:i")
Distill = _struct("logits:p ids:p teacher:p loss:p stats:p workspace:p workspace_bytes:u rows:u vocab:u logits_stride:u ids_stride:u teacher_stride:u "
                  "temperature:f ids_64:i dtype_tag:i teacher_dtype:i k:i rest:i")
DistillGrad = _struct("logits:p ids:p teacher:p stats:p grad:p out:p rows:u vocab:u logits_stride:u ids_stride:u teacher_stride:u out_stride:u temperature:f "
                      "ids_64:i dtype_tag:i teacher_dtype:i out_dtype:i k:i")


def _header():
    return open(os.path.join(ROOT, "include", "eri_losses.h")).read()


def _rust():
    return open(os.path.join(ROOT, "eridiffusion_amd", "rust", "eri_losses_sys.rs")).read()


def _declared():
    return set(re.findall(r"^int (eri_[a-z0-9_]+)\s*\(", _header(), re.M))


def test_library_exports_every_declared_symbol_and_rust_declares_them():
    lib = L.lib()
    assert len(_declared()) == 6
    for name in _declared():
        assert hasattr(lib, name), name
    assert set(re.findall(r"pub fn (eri_[a-z0-9_]+)\s*\(", _rust())) == _declared()


@pytest.mark.parametrize("kind,name", [(Logprobs, "EriTokenLogprobs"), (LogprobsGrad, "EriTokenLogprobsGrad"), (Distill, "EriDistillTop"),
                                       (DistillGrad, "EriDistillTopGrad")])
def test_structs_of_these_tests_and_of_rust_have_the_headers_fields(kind, name):
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), re.sub(r"/\*.*?\*/", "", _header(), flags=re.S), re.S).group(1)
    fields = [n.strip().lstrip("*") for line in body.split(";") if line.strip() for n in re.sub(r"^\s*(const )?\w+ ", "", line.strip()).split(",")]
    assert fields == [f for f, _ in kind._fields_]
    assert re.findall(r"pub (\w+):", re.search(r"pub struct %s \{(.*?)\}" % name, _rust(), re.S).group(1)) == fields


def _sized(call, *sizes):
    fn, need = getattr(L.lib(), call), C.c_uint64()
    fn.restype, fn.argtypes = C.c_int, [C.c_uint64] * 2 + ([C.c_int32] if len(sizes) == 3 else []) + [C.c_void_p]
    assert fn(*sizes, None) == NULL
    rc = fn(*sizes, C.byref(need))
    return rc or need.value


def test_refusals_of_the_scores():
    base = dict(logits=0x1000, ids=0x2000, logprob=0x3000, entropy=0x4000, stats=0x5000, top=0x6000, top_ids=0x7000, workspace=0x8000, workspace_bytes=1 << 30,
                rows=4, vocab=100000, temperature=1.0, ids_64=1, dtype_tag=BF16, top_n=20)
    assert _refused("eri_token_logprobs", None) == NULL
    need = _sized("eri_token_logprobs_workspace", 4, 100000, 20)
    for code, change in [(NULL, dict(logits=0)), (NULL, dict(stats=0)), (NULL, dict(ids=0)), (NULL, dict(logprob=0)), (NULL, dict(top=0)), (NULL, dict(top_ids=0)),
                         (NULL, dict(workspace=0)), (ALIGN, dict(logits=0x1001)), (ALIGN, dict(ids=0x2004)), (ALIGN, dict(ids=0x2002, ids_64=0)),
                         (ALIGN, dict(logprob=0x3002)), (ALIGN, dict(entropy=0x4001)), (ALIGN, dict(stats=0x5002)), (ALIGN, dict(top=0x6002)),
                         (ALIGN, dict(top_ids=0x7004)), (ALIGN, dict(workspace=0x8008)), (EMPTY, dict(vocab=0, top_n=0)), (DTYPE, dict(dtype_tag=F16)),
                         (DTYPE, dict(dtype_tag=F8)), (DTYPE, dict(ids_64=2)), (ARG, dict(logits_stride=99999)), (ARG, dict(logits_stride=2 ** 41)),
                         (ARG, dict(temperature=0.0)), (ARG, dict(temperature=-1.0)), (ARG, dict(temperature=math.nan)), (ARG, dict(temperature=math.inf)),
                         (ARG, dict(temperature=9e-5)), (ARG, dict(top_n=65)), (ARG, dict(top_n=-1)), (ARG, dict(vocab=19)), (ARG, dict(workspace_bytes=need - 1)),
                         (TOO_LARGE, dict(rows=2 ** 31)), (TOO_LARGE, dict(vocab=2 ** 31))]:
        assert _refused("eri_token_logprobs", _with(Logprobs, base, **change)) == code, change
    assert _refused("eri_token_logprobs", _with(Logprobs, base, rows=0, logits=0, ids=0, logprob=0, stats=0, top=0, workspace=0)) == 0  # nothing to do
    assert _sized("eri_token_logprobs_workspace", 4, 0, 0) == EMPTY and _sized("eri_token_logprobs_workspace", 2 ** 31, 8, 0) == TOO_LARGE
    assert _sized("eri_token_logprobs_workspace", 4, 8, 9) == ARG and _sized("eri_token_logprobs_workspace", 4, 800, 65) == ARG
    assert _sized("eri_token_logprobs_workspace", 0, 100000, 20) == 0


def test_refusals_of_the_scores_gradient():
    base = dict(logits=0x1000, ids=0x2000, stats=0x3000, grad=0x4000, grad_entropy=0x5000, entropy=0x6000, out=0x7000, rows=4, vocab=16, temperature=1.0,
                ids_64=1, dtype_tag=BF16, out_dtype=F32)
    assert _refused("eri_token_logprobs_grad", None) == NULL
    for code, change in [(NULL, dict(logits=0)), (NULL, dict(stats=0)), (NULL, dict(out=0)), (NULL, dict(ids=0)), (NULL, dict(grad=0)), (NULL, dict(entropy=0)),
                         (NULL, dict(grad_entropy=0)), (NULL, dict(grad=0, ids=0, grad_entropy=0, entropy=0)), (ALIGN, dict(logits=0x1001)), (ALIGN, dict(out=0x7002)),
                         (ALIGN, dict(ids=0x2004)), (ALIGN, dict(stats=0x3002)), (ALIGN, dict(grad=0x4002)), (ALIGN, dict(grad_entropy=0x5002)),
                         (ALIGN, dict(entropy=0x6002)), (EMPTY, dict(vocab=0)), (DTYPE, dict(dtype_tag=F16)), (DTYPE, dict(out_dtype=F8)), (DTYPE, dict(ids_64=-1)),
                         (ARG, dict(logits_stride=15)), (ARG, dict(out_stride=15)), (ARG, dict(temperature=2e4)), (TOO_LARGE, dict(rows=2 ** 31)),
                         (TOO_LARGE, dict(vocab=2 ** 31))]:
        assert _refused("eri_token_logprobs_grad", _with(LogprobsGrad, base, **change)) == code, change
    assert _refused("eri_token_logprobs_grad", _with(LogprobsGrad, base, rows=0, logits=0, out=0)) == 0


def test_refusals_of_the_distillation():
    base = dict(logits=0x1000, ids=0x2000, teacher=0x3000, loss=0x4000, stats=0x5000, workspace=0x6000, workspace_bytes=1 << 30, rows=4, vocab=100000,
                temperature=1.0, ids_64=1, dtype_tag=BF16, teacher_dtype=F32, k=20, rest=1)
    assert _refused("eri_distill_top", None) == NULL
    need = _sized("eri_distill_top_workspace", 4, 100000)
    for code, change in [(NULL, dict(logits=0)), (NULL, dict(ids=0)), (NULL, dict(teacher=0)), (NULL, dict(loss=0)), (NULL, dict(stats=0)), (NULL, dict(workspace=0)),
                         (ALIGN, dict(logits=0x1001)), (ALIGN, dict(ids=0x2004)), (ALIGN, dict(teacher=0x3002)), (ALIGN, dict(loss=0x4002)), (ALIGN, dict(stats=0x5002)),
                         (ALIGN, dict(workspace=0x6004)), (EMPTY, dict(vocab=0)), (DTYPE, dict(dtype_tag=F16)), (DTYPE, dict(teacher_dtype=F16)), (DTYPE, dict(ids_64=2)),
                         (ARG, dict(k=0)), (ARG, dict(k=65)), (ARG, dict(k=-1)), (ARG, dict(rest=2)), (ARG, dict(logits_stride=1)), (ARG, dict(ids_stride=19)),
                         (ARG, dict(teacher_stride=19)), (ARG, dict(temperature=0.0)), (ARG, dict(workspace_bytes=need - 1)), (TOO_LARGE, dict(rows=2 ** 31))]:
        assert _refused("eri_distill_top", _with(Distill, base, **change)) == code, change
    assert _refused("eri_distill_top", _with(Distill, base, rows=0, logits=0, ids=0, teacher=0, loss=0, stats=0, workspace=0)) == 0
    assert _sized("eri_distill_top_workspace", 4, 0) == EMPTY and _sized("eri_distill_top_workspace", 4, 2 ** 31) == TOO_LARGE


def test_refusals_of_the_distillations_gradient():
    base = dict(logits=0x1000, ids=0x2000, teacher=0x3000, stats=0x4000, grad=0x5000, out=0x6000, rows=4, vocab=16, temperature=1.0, ids_64=0, dtype_tag=F32,
                teacher_dtype=BF16, out_dtype=BF16, k=64)
    assert _refused("eri_distill_top_grad", None) == NULL
    for code, change in [(NULL, dict(logits=0)), (NULL, dict(ids=0)), (NULL, dict(teacher=0)), (NULL, dict(stats=0)), (NULL, dict(grad=0)), (NULL, dict(out=0)),
                         (ALIGN, dict(logits=0x1002)), (ALIGN, dict(ids=0x2002)), (ALIGN, dict(teacher=0x3001)), (ALIGN, dict(stats=0x4002)), (ALIGN, dict(grad=0x5001)),
                         (ALIGN, dict(out=0x6001)), (EMPTY, dict(vocab=0)), (DTYPE, dict(dtype_tag=F8)), (DTYPE, dict(teacher_dtype=F8)), (DTYPE, dict(out_dtype=F16)),
                         (ARG, dict(k=0)), (ARG, dict(k=65)), (ARG, dict(out_stride=15)), (ARG, dict(ids_stride=63)), (ARG, dict(temperature=math.nan)),
                         (TOO_LARGE, dict(vocab=2 ** 31))]:
        assert _refused("eri_distill_top_grad", _with(DistillGrad, base, **change)) == code, change
    assert _refused("eri_distill_top_grad", _with(DistillGrad, base, rows=0, logits=0, ids=0, teacher=0, stats=0, grad=0, out=0)) == 0


@pytest.mark.parametrize("vocab", [1, 100, 2048, 4096, 8192, 10007, 128000, 2 ** 31 - 1])
def test_the_workspaces_do_for_fewer_rows_and_alternatives(vocab):
    """Whoever makes them for the largest batch has enough for a shorter last one."""
    rows = sorted(set(range(1, 3000, 7)) | {2 ** k + d for k in range(31) for d in (-1, 0, 1) if 0 < 2 ** k + d < 2 ** 31})
    before = None
    for top in (0, 1, min(20, vocab), min(64, vocab)):
        sizes = [_sized("eri_token_logprobs_workspace", r, vocab, top) for r in rows]
        assert sizes == sorted(sizes)
        assert before is None or all(a <= b for a, b in zip(before, sizes))
        before = sizes
    sizes = [_sized("eri_distill_top_workspace", r, vocab) for r in rows]
    assert sizes == sorted(sizes)


def _calls(x):
    """Each call, with x wherever a tensor of floats may stand."""
    ids, one = torch.zeros(4, dtype=torch.long), torch.zeros(4)
    few, part = torch.zeros(4, 3, dtype=torch.long), x[:, :3]
    return [lambda: losses.token_logprobs(x, ids), lambda: losses.token_logprobs(x, top=2), lambda: losses.token_logprobs_grad(x, ids, one, one),
            lambda: losses.distill_top(x, few, part), lambda: losses.distill_top_grad(x, few, part, one, one)]


def test_the_python_calls_refuse_host_tensors_tangents_and_tracers():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.autograd import forward_ad as fa
    from torch.fx.experimental.proxy_tensor import make_fx
    x = torch.zeros(4, 8)
    for k, call in enumerate(_calls(x)):
        with pytest.raises(ValueError, match="take device tensors"):
            call()
        for trace in (lambda f: torch.jit.trace(f, (x,)), lambda f: make_fx(f)(x)):
            with pytest.raises(ValueError, match="cannot be traced"):
                trace(lambda a: _calls(a)[k]())
        with FakeTensorMode(), pytest.raises(ValueError, match="cannot be traced"):
            call()
    with fa.dual_level():
        for call in _calls(fa.make_dual(x, torch.ones(4, 8))):
            with pytest.raises(ValueError, match="forward-mode tangent"):
                call()
    with pytest.raises(TypeError):
        losses.token_logprobs([1.0], None)


def _differences(loss, x, dx, seed):
    d = torch.randn(x.shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)
    h = 1e-5  # the difference's own error is of the order h^2
    want = (loss(x + h * d) - loss(x - h * d)) / (2 * h)
    got = (dx * d).sum()
    assert abs(got - want) < 1e-7 * (1 + abs(want)), (got, want)


@pytest.mark.parametrize("temperature", [1.0, 0.5, 3.0])
def test_the_oracles_gradients_are_the_differences_of_its_forward(temperature):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(6, 11, generator=g, dtype=torch.float64) * 2
    ids, w, wh = torch.tensor([0, 5, -100, 10, 11, 3]), torch.randn(6, generator=g), torch.randn(6, generator=g)

    def scores(z):
        one, h = of.token_logprobs(z, ids, temperature)[:2]
        return (one * w + h * wh).sum()
    _differences(scores, x, of.token_logprobs_grad(x, ids, w, wh, temperature)[0], 1)
    few = torch.tensor([[0, 4, 7], [1, 1, 2], [-1, 3, 12], [5, 6, 8], [9, 10, 0], [2, 2, 2]])  # doubles, and some that name no token
    teacher = torch.randn(6, 3, generator=g, dtype=torch.float64) - 1.5
    teacher[3, 1], teacher[4] = -math.inf, -math.inf
    teacher[5] = 2.0  # probabilities over 1
    for rest in (False, True):
        dx = of.distill_top(x, few, teacher, temperature, rest)[2]
        _differences(lambda z: (of.distill_top(z, few, teacher, temperature, rest)[0] * w).sum(), x, dx * w[:, None], 2)


def test_the_oracles_distillation_is_the_divergence_over_its_classes():
    g = torch.Generator().manual_seed(4)
    x = torch.randn(5, 9, generator=g, dtype=torch.float64)
    full = torch.log_softmax(torch.randn(5, 9, generator=g, dtype=torch.float64), 1)
    value, ids = full.topk(4, 1)
    logp = torch.log_softmax(x, 1)
    q, p = value.exp(), logp.gather(1, ids).exp()
    classes = lambda a: torch.cat((a, 1 - a.sum(1, keepdim=True)), 1)  # noqa: E731
    want = (classes(q) * (classes(q).log() - classes(p).log())).sum(1)
    assert torch.allclose(of.distill_top(x, ids, value, 1.0, True)[0], want, rtol=1e-12)
    r = q / q.sum(1, keepdim=True)
    assert torch.allclose(of.distill_top(x, ids, value, 1.0, False)[0], (r * (r.log() - p.log())).sum(1), rtol=1e-12)
    # all tokens: the whole divergence, with or without a rest
    every = torch.arange(9).expand(5, 9)
    whole = (full.exp() * (full - logp)).sum(1)
    for rest in (False, True):
        assert torch.allclose(of.distill_top(x, every, full, 1.0, rest)[0], whole, rtol=1e-10)
