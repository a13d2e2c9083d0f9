"""Label operators: what a label field over the rays forms its logits with, learns from and answers with.

  distill_top_logits        loss of rows of student logits against a teacher's top logits (a 2-D segmenter of which only the largest
                            values per pixel are stored), differentiable; distill_top_logits_grad: loss and gradient in one pass
  sample_logits             one label per row at a given random number, behind temperature / top-k / top-p / min-p -- to logits what
                            `sample_pdf` is to a ray's weights; its int64 labels are the `instance_ids` that `CodeLibrary` takes

Rows are (N, V) on the GPU in float32, bfloat16 or float16 with any row stride; a last dimension that is not contiguous is copied.
Python here checks arguments, allocates results and enqueues on the current stream of the tensors' device; nothing synchronises, and
a call can be captured in a graph.  Arguments of a wrong type raise TypeError, of a wrong value or shape ValueError, CPU tensors and
failing launches RuntimeError.
"""
import ctypes as C

import torch

from . import _lib

__all__ = ["distill_top_logits", "distill_top_logits_grad", "sample_logits"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}      # OBJNERF_TYPE_*
MAX_SLOTS = 1024


def _rows(t, name, types=_TYPES):
    """t as a 2-D GPU tensor whose rows are contiguous"""
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a tensor, got %s" % (name, type(t).__name__))
    if t.dim() != 2:
        raise ValueError("%s must have two dimensions, got shape %s" % (name, tuple(t.shape)))
    if t.dtype not in types:
        raise TypeError("%s: dtype %s is not supported" % (name, t.dtype))
    if not t.is_cuda:
        _lib.require_cuda(t, name)
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _column(t, name, n, device, dtype=torch.float32):
    """t as a contiguous (n,) GPU tensor of `dtype`"""
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError("%s must have shape (%d,), got %s" % (name, n, tuple(t.shape)))
    if t.device != device:
        raise ValueError("%s must be on %s, got %s" % (name, device, t.device))
    if t.is_floating_point() != dtype.is_floating_point or t.dtype == torch.bool or t.is_complex():
        raise TypeError("%s: dtype %s is not supported" % (name, t.dtype))
    return (t if t.dtype == dtype else t.to(dtype)).contiguous()


def _call(fn, args, device, what):
    """enqueues `fn` on the current stream of `device`"""
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _call(fn, args, device, what)
    rc = fn(C.byref(args), C.c_void_p(torch.cuda.current_stream().cuda_stream))
    if rc:
        _lib.check(rc, what)


# ---- distillation ----

def _distill_args(student, teacher, index, temperature):
    student = _rows(student, "student")
    teacher = _rows(teacher, "teacher")
    index = _rows(index, "index", (torch.int32, torch.int64))
    if teacher.requires_grad:
        raise ValueError("teacher must not require a gradient: the teacher is a constant (detach it)")
    n, v = student.shape
    if teacher.shape != index.shape or teacher.shape[0] != n:
        raise ValueError("teacher and index must have one shape (%d, k), got %s and %s" % (n, tuple(teacher.shape), tuple(index.shape)))
    k = teacher.shape[1]
    if v < 1 or not 1 <= k <= MAX_SLOTS:
        raise ValueError("distill_top_logits needs at least one label and 1 to %d slots, got %d and %d" % (MAX_SLOTS, v, k))
    if teacher.device != student.device or index.device != student.device:
        raise ValueError("student, teacher and index must be on one device")
    temperature = float(temperature)
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError("temperature must be positive and finite, got %r" % temperature)
    a = _lib.DistillArgs()
    a.n, a.v, a.k = n, v, k
    a.student, a.student_stride, a.student_type = student.data_ptr(), student.stride(0), _TYPES[student.dtype]
    a.teacher, a.teacher_stride, a.teacher_type = teacher.data_ptr(), teacher.stride(0), _TYPES[teacher.dtype]
    a.index, a.index_stride, a.index_bytes = index.data_ptr(), index.stride(0), index.element_size()
    a.temperature = temperature
    return a, (student, teacher, index)       # the tensors whose memory the arguments point to: kept until the call is enqueued


def _run_distill(a, keep, want_loss, upstream):
    student = keep[0]
    loss = grad = None
    if want_loss:
        loss = torch.empty(a.n, dtype=torch.float32, device=student.device)
        a.loss = loss.data_ptr()
    if upstream is not None:
        grad = torch.empty(a.n, a.v, dtype=student.dtype, device=student.device)
        a.upstream, a.upstream_stride = upstream.data_ptr(), (upstream.stride(0) if upstream.dim() else 0)
        a.grad, a.grad_stride = grad.data_ptr(), a.v
    if a.n:
        _call(_lib.lib().objnerf_distill_top, a, student.device, "distill_top")
    return loss, grad


class _DistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, student, teacher, index, temperature):
        a, keep = _distill_args(student, teacher, index, temperature)
        ctx.save_for_backward(student, teacher, index)
        ctx.temperature = temperature
        return _run_distill(a, keep, True, None)[0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_loss):
        a, keep = _distill_args(*ctx.saved_tensors, ctx.temperature)
        return _run_distill(a, keep, False, d_loss if d_loss.dtype == torch.float32 else d_loss.float())[1], None, None, None


def distill_top_logits(student, teacher, index, temperature=1.0):
    """The distillation loss of every row, (N,) float32: KL(p || q) with p = softmax(teacher / T) over the row's filled slots and
    q = softmax(student / T) over all V labels.

    student (N, V); teacher (N, k) logits or log-probabilities, k <= 1024; index (N, k) int32 or int64, the labels that the
    teacher's values belong to.  A slot whose index lies outside [0, V) or whose value is -inf is empty; a row without a filled slot
    has loss 0 and gradient 0.  An index may occur more than once (its shares add).  Differentiable with respect to `student`
    alone; the usual factor T^2 is the caller's.  The backward pass reads the student's row again instead of keeping a copy."""
    if torch.is_grad_enabled() and isinstance(student, torch.Tensor) and student.requires_grad:
        return _DistillFn.apply(student, teacher, index, temperature)
    return _run_distill(*_distill_args(student, teacher, index, temperature), True, None)[0]


def distill_top_logits_grad(student, teacher, index, upstream, temperature=1.0):
    """(loss, grad) of distill_top_logits in one pass over the student's rows, for a loop that knows the gradient of its losses
    beforehand: `upstream` (N,) is d total / d loss_n (1 / N for a mean), grad = d total / d student in the student's type
    (`logits.backward(grad)` goes on from there)."""
    if not isinstance(upstream, torch.Tensor):
        raise TypeError("upstream must be a tensor, got %s" % type(upstream).__name__)
    a, keep = _distill_args(student, teacher, index, temperature)
    return _run_distill(a, keep, True, _column(upstream.detach(), "upstream", a.n, keep[0].device))


# ---- drawing a label ----

def sample_logits(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One label per row, (N,) int64, drawn at the random numbers u (N,) in [0, 1).

    Weights are exp(logits / temperature) (up to a factor).  The labels in order -- falling logits, equal ones by rising index -- are
    cut to the first `top_k` (0: all), of those to the shortest prefix whose share of their weight reaches `top_p` (1: all; at
    least one label stays), of those to the ones with at least `min_p` times the largest weight (0: all).  The label is the
    first, in that order, whose running sum of weight exceeds u times their total.  temperature 0 and top_k 1 give the first
    of the order.  NaN counts as -inf; a row of nothing but -inf gives -1.

    Each setting is a number or an (N,) tensor on the logits' device, one value per row.  Runs give equal labels for equal inputs."""
    logits = _rows(logits, "logits")
    n, v = logits.shape
    dev = logits.device
    if v < 1:
        raise ValueError("sample_logits needs at least one label")
    if not isinstance(u, torch.Tensor):
        raise TypeError("u must be a tensor, got %s" % type(u).__name__)
    u = _column(u, "u", n, dev)
    a = _lib.SampleArgs()
    a.n, a.v, a.type = n, v, _TYPES[logits.dtype]
    a.logits, a.logits_stride, a.u, a.u_stride = logits.data_ptr(), logits.stride(0), u.data_ptr(), 1
    keep = []
    if isinstance(temperature, torch.Tensor):
        keep.append(_column(temperature, "temperature", n, dev))
        a.temperature_rows = keep[-1].data_ptr()
    else:
        if not 0.0 <= temperature < 1e300:
            raise ValueError("temperature must be >= 0 and finite, got %r" % (temperature,))
        a.temperature = temperature
    if isinstance(top_k, torch.Tensor):
        keep.append(_column(top_k, "top_k", n, dev, torch.int32))
        a.top_k_rows = keep[-1].data_ptr()
    else:
        if not 0 <= top_k < 1 << 31:
            raise ValueError("top_k must be >= 0, got %r" % (top_k,))
        a.top_k = top_k
    if isinstance(top_p, torch.Tensor):
        keep.append(_column(top_p, "top_p", n, dev))
        a.top_p_rows = keep[-1].data_ptr()
    else:
        if not top_p >= 0.0:
            raise ValueError("top_p must be >= 0, got %r" % (top_p,))
        a.top_p = top_p
    if isinstance(min_p, torch.Tensor):
        keep.append(_column(min_p, "min_p", n, dev))
        a.min_p_rows = keep[-1].data_ptr()
    else:
        if not 0.0 <= min_p <= 1.0:
            raise ValueError("min_p must lie in [0, 1], got %r" % (min_p,))
        a.min_p = min_p
    labels = torch.empty(n, dtype=torch.int64, device=dev)
    a.labels = labels.data_ptr()
    if n:
        _call(_lib.lib().objnerf_sample_logits, a, dev, "sample_logits")
    return labels
