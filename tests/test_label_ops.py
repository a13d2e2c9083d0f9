"""CPU: the label operators refuse what they do not take, in Python and at the C ABI, before anything is launched."""
import ctypes as C

import pytest
import torch

import object_nerf_amd as A
from object_nerf_amd import _lib


def _distill_args(**kw):
    a = _lib.DistillArgs()
    base = dict(n=2, v=8, k=2, student=64, student_stride=8, student_type=0, teacher_type=0, teacher=64, teacher_stride=2, index=64,
                index_stride=2, index_bytes=4, temperature=1.0, loss=64, upstream=None, upstream_stride=1, grad=None, grad_stride=8)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [dict(n=-1), dict(n=1 << 31), dict(v=0), dict(k=0), dict(k=1025), dict(student_type=3), dict(student_type=-1),
                                 dict(teacher_type=7), dict(index_bytes=2), dict(temperature=0.0), dict(temperature=-1.0),
                                 dict(temperature=float("nan")), dict(temperature=float("inf")), dict(student_stride=-8),
                                 dict(student=None), dict(teacher=None), dict(index=None), dict(loss=None), dict(grad=64),
                                 dict(grad=64, upstream=64, grad_stride=7)])
def test_distill_refuses_at_the_c_abi(bad):
    l = _lib.lib()
    assert l.objnerf_distill_top(C.byref(_distill_args(**bad)), None) < 0
    assert b"distill_top" in l.objnerf_last_error()


def test_distill_c_abi_takes_no_rows_and_no_arguments():
    l = _lib.lib()
    assert l.objnerf_distill_top(C.byref(_distill_args(n=0)), None) == 0
    assert l.objnerf_distill_top(None, None) < 0


def _sample_args(**kw):
    a = _lib.SampleArgs()
    base = dict(n=2, v=8, type=1, logits=64, logits_stride=8, u=64, u_stride=1, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, labels=64)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [dict(n=-1), dict(n=1 << 31), dict(v=0), dict(type=3), dict(logits_stride=-1), dict(temperature=-0.5),
                                 dict(temperature=float("nan")), dict(temperature=float("inf")), dict(top_k=-1), dict(top_p=-0.1),
                                 dict(top_p=float("nan")), dict(min_p=1.5), dict(min_p=-0.1), dict(min_p=float("nan")),
                                 dict(logits=None), dict(u=None), dict(labels=None)])
def test_sample_refuses_at_the_c_abi(bad):
    l = _lib.lib()
    assert l.objnerf_sample_logits(C.byref(_sample_args(**bad)), None) < 0
    assert b"sample_logits" in l.objnerf_last_error()


def test_sample_c_abi_takes_no_rows_and_no_arguments():
    l = _lib.lib()
    assert l.objnerf_sample_logits(C.byref(_sample_args(n=0)), None) == 0
    assert l.objnerf_sample_logits(None, None) < 0


def test_python_refusals_without_a_gpu():
    z, t, i, u = torch.zeros(3, 8), torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3)
    with pytest.raises(RuntimeError, match="GPU"):
        A.distill_top_logits(z, t, i)
    with pytest.raises(RuntimeError, match="GPU"):
        A.distill_top_logits_grad(z, t, i, u)
    with pytest.raises(RuntimeError, match="GPU"):
        A.sample_logits(z, u)
    with pytest.raises(TypeError):
        A.distill_top_logits(z.double(), t, i)
    with pytest.raises(TypeError):
        A.sample_logits(z.long(), u)
    with pytest.raises(TypeError):
        A.sample_logits([1.0, 2.0], u)
    with pytest.raises(TypeError):
        A.distill_top_logits_grad(z, t, i, 1.0)
    with pytest.raises(ValueError):
        A.distill_top_logits(z[0], t, i)
    with pytest.raises(ValueError):
        A.sample_logits(z[None], u)
