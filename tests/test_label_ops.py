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


def _quantize_args(**kw):
    a = _lib.Fp8QuantizeArgs()
    base = dict(rows=4, cols=130, x=64, x_stride=130, type=1, block_rows=1, values=64, scales=64, values_t=None, scales_t=None, column_sums=None, workspace=None)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(cols=-1), dict(rows=1 << 31), dict(rows=1 << 30, cols=1 << 20), dict(type=3), dict(block_rows=2), dict(x_stride=-1),
                                 dict(values=None), dict(scales=None), dict(values=None, scales=None), dict(values_t=64), dict(scales_t=64), dict(column_sums=64),
                                 dict(values=72), dict(scales=66), dict(values_t=72, scales_t=64), dict(x=None), dict(rows=0, column_sums=64, workspace=64)])
def test_quantize_refuses_at_the_c_abi(bad):
    l = _lib.lib()
    assert l.objnerf_fp8_quantize(C.byref(_quantize_args(**bad)), None) < 0
    assert b"fp8_quantize" in l.objnerf_last_error()


def _gemm_args(**kw):
    a = _lib.GemmFp8Args()
    base = dict(M=4, N=8, K=256, a_type=3, a_cols=0, a=64, a_stride=256, a_scale=64, a_scale_stride=4, b=64, b_stride=256, b_scale=64, b_scale_stride=4, bias=None, leaky=0, c_type=1,
                c=64, c_stride=8)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [dict(M=-1), dict(N=-1), dict(K=-128), dict(K=200), dict(M=1 << 31), dict(M=(1 << 31) - 1, N=(1 << 31) - 1, c_stride=1 << 31), dict(c_type=4),
                                 dict(a_stride=128), dict(b_stride=250), dict(b_stride=260), dict(c_stride=7), dict(a_scale_stride=2), dict(b_scale_stride=5), dict(K=640, a_stride=640, b_stride=640),
                                 dict(a=72), dict(b_scale=65), dict(a=None), dict(b=None), dict(a_scale=None), dict(b_scale=None), dict(c=None), dict(a_type=4), dict(a_type=-1), dict(a_type=1, a_cols=128),
                                 dict(a_type=1, a_cols=257), dict(a_type=1, a_cols=256, a_stride=-1)])
def test_gemm_refuses_at_the_c_abi(bad):
    l = _lib.lib()
    assert l.objnerf_gemm_fp8(C.byref(_gemm_args(**bad)), None) < 0
    assert b"gemm_fp8" in l.objnerf_last_error()


def test_gemm_refuses_a_sum_of_nothing_over_too_many_tiles():
    l = _lib.lib()
    assert l.objnerf_gemm_fp8(C.byref(_gemm_args(M=(1 << 31) - 1, N=1, K=0)), None) < 0
    assert b"2^22 tiles" in l.objnerf_last_error()


def test_fp8_c_abi_takes_nothing_to_do():
    l = _lib.lib()
    assert l.objnerf_fp8_quantize(C.byref(_quantize_args(rows=0)), None) == 0 and l.objnerf_fp8_quantize(None, None) < 0
    assert l.objnerf_gemm_fp8(C.byref(_gemm_args(M=0)), None) == 0 and l.objnerf_gemm_fp8(None, None) < 0
    assert l.objnerf_fp8_quantize_workspace_floats(129, 7) == 14 and l.objnerf_fp8_quantize_workspace_floats(0, 7) == 0


def test_fp8_python_refusals_without_a_gpu():
    x = torch.zeros(3, 8)
    for call in (lambda: A.quantize_fp8(x), lambda: A.linear_fp8(x, x)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    with pytest.raises(RuntimeError, match="GPU"):
        q = A.Fp8Matrix(torch.zeros(3, 128, dtype=torch.float8_e4m3fn), torch.zeros(3, 4, dtype=torch.uint8), 8)
        A.matmul_fp8(q, q)
    with pytest.raises(TypeError):
        A.matmul_fp8(x, x)
