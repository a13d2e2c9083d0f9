"""Label operators: what a label field over the rays forms its logits with, learns from and answers with.

  linear_fp8                x @ weight.T + bias in 8-bit floating point with a scale for each block of 128, differentiable;
                            quantize_fp8 / matmul_fp8: its two halves, for weights that are laid out once.  The fp32 product of the
                            layer-wise training path (objnerf_gemm) at a quarter of its bytes
  distill_top_logits        loss of rows of student logits against a teacher's top logits (a 2-D segmenter of which only the largest
                            values per pixel are stored), differentiable; distill_top_logits_grad: loss and gradient in one pass
  sample_logits             one label per row at a given random number, behind temperature / top-k / top-p / min-p -- to logits what
                            `sample_pdf` is to a ray's weights; its int64 labels are the `instance_ids` that `CodeLibrary` takes, except
                            the -1 of a row with nothing to draw, which a table lookup on the GPU takes as out of range

Rows are (N, V) on the GPU in float32, bfloat16 or float16 with any row stride; a last dimension that is not contiguous is copied.
Python here checks arguments, allocates results and enqueues on the current stream of the tensors' device; nothing synchronises, and
a call can be captured in a graph.  Arguments of a wrong type raise TypeError, of a wrong value or shape ValueError, CPU tensors and
failing launches RuntimeError.  Differentiable is meant of backward passes, once: a tensor with a forward-mode tangent raises
NotImplementedError.  What records torch operations to run them again without Python (torch.jit.trace, make_fx) sees none of the
kernels and is refused with a RuntimeError.
"""
import ctypes as C
import operator
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _lib

__all__ = ["Fp8Matrix", "quantize_fp8", "matmul_fp8", "linear_fp8", "distill_top_logits", "distill_top_logits_grad", "sample_logits"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}      # OBJNERF_TYPE_*
MAX_SLOTS = 1024
MAX_SUM = 1 << 26                      # terms of a product's sums
MAX_INT = (1 << 31) - 1                # rows, and labels of the distillation
MAX_LABELS = 1 << 19                   # of a row that a label is drawn from


_tracing, _modes, _mode, _PROXY = torch._C._is_tracing, torch._C._len_torch_dispatch_stack, torch._C._get_dispatch_mode, torch._C._TorchDispatchModeKey.PROXY


def _refuse_recording():
    """a recorded program would hold the allocation of the results and no kernel.  Once a call (0.2 us)"""
    if _tracing() or (_modes() and _mode(_PROXY) is not None):
        raise RuntimeError("the label operators cannot be recorded by torch.jit.trace or make_fx: the kernels would be missing")


def _refuse_tangents(*tensors):
    """forward-mode derivatives go past `requires_grad`: the result would come without one"""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if isinstance(t, torch.Tensor) and t.is_floating_point() and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError("the label operators have no forward-mode derivative")


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
    if types is _TYPES and t.is_neg():                # a view that stands for minus its memory (the imaginary part of a conjugate)
        t = t.resolve_neg()
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _column(t, name, n, device, dtype=torch.float32):
    """t as a contiguous (n,) GPU tensor of `dtype`"""
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError("%s must have shape (%d,), got %s" % (name, n, tuple(t.shape)))
    if t.device != device:
        raise ValueError("%s must be on %s, got %s" % (name, device, t.device))
    if t.is_floating_point() != dtype.is_floating_point or t.dtype == torch.bool or t.is_complex():
        raise TypeError("%s: dtype %s is not supported" % (name, t.dtype))
    if t.dtype != dtype:
        t = t.to(dtype)
    return (t.resolve_neg() if t.is_neg() else t).contiguous()


def _call(fn, args, device, what):
    """enqueues `fn` on the current stream of `device`"""
    index = device.index
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            return _call(fn, args, device, what)
    rc = fn(C.byref(args), torch._C._cuda_getCurrentRawStream(index))      # (torch.cuda.current_stream() costs 2.7 us)
    if rc:
        _lib.check(rc, what)


# ---- products in 8-bit floating point ----

BLOCK = 128


class Fp8Matrix(NamedTuple):
    """A matrix (R, cols) in e4m3 with a power-of-two scale for each block of 128 columns of a row.

    data (R, C') float8_e4m3fn, C' = cols filled up to a multiple of 128 with zeros; scale (R, B') uint8, B' = C' / 128 filled up to a
    multiple of 4: element [r, c] stands for data[r, c] * 2 ** (scale[r, c // 128] - 127), scale in [1, 247] (what numbers of fp32 need; fp32
    results of larger scales can overflow)."""
    data: torch.Tensor
    scale: torch.Tensor
    cols: int


def _up(n, step):
    return -(-n // step) * step


def _empty_fp8(rows, cols, device):
    width = _up(cols, BLOCK)
    return Fp8Matrix(torch.empty(rows, width, dtype=torch.float8_e4m3fn, device=device),
                     torch.empty(rows, _up(width // BLOCK, 4), dtype=torch.uint8, device=device), cols)


def _quantize(x, block_rows, rows=True, columns=False, sums=False):
    """(x by rows, x by columns, column sums) of a 2-D GPU tensor with contiguous rows, each where asked for, in one pass over x"""
    r, c = x.shape
    q = _empty_fp8(r, c, x.device) if rows else None
    t = _empty_fp8(c, r, x.device) if columns else None
    total = None
    work = None
    if sums:
        work = torch.empty(_up(r, BLOCK) // BLOCK * c, dtype=torch.float32, device=x.device)
        total = torch.empty(c, dtype=torch.float32, device=x.device)
    a = _lib.Fp8QuantizeArgs(r, c, x.data_ptr(), x.stride(0), _TYPES[x.dtype], block_rows, *((q.data.data_ptr(), q.scale.data_ptr()) if rows else (None, None)),
                             *((t.data.data_ptr(), t.scale.data_ptr()) if columns else (None, None)), *((total.data_ptr(), work.data_ptr()) if sums else (None, None)))
    if r and c:
        _call(_lib.lib().objnerf_fp8_quantize, a, x.device, "fp8_quantize")
    return q, t, total


def _product(a, b, bias, leaky, out_dtype):
    """(M, N) of an Fp8Matrix, or a matrix that the product rounds on its way, and an Fp8Matrix over the same columns"""
    raw = not isinstance(a, Fp8Matrix)
    data = a if raw else a.data
    if b.cols > MAX_SUM:
        raise ValueError("a product over more than 2^26 columns is not supported, got %d" % b.cols)
    m, n, k, dev = data.shape[0], b.data.shape[0], b.data.shape[1], data.device
    out = torch.empty(m, n, dtype=out_dtype, device=dev)
    if not (m and n):
        return out
    lib = _lib.lib()
    a_type, c_type = (_TYPES[data.dtype] if raw else 3), _TYPES[out_dtype]
    floats = lib.objnerf_gemm_fp8_workspace_floats(m, n, k, a_type, c_type)
    work = torch.empty(floats, dtype=torch.float32, device=dev) if floats else None
    g = _lib.GemmFp8Args(m, n, k, a_type, 0, data.data_ptr(), data.stride(0), None if raw else a.scale.data_ptr(), 0 if raw else a.scale.stride(0), b.cols,
                         b.data.data_ptr(), b.data.stride(0), b.scale.data_ptr(), b.scale.stride(0), None if bias is None else bias.data_ptr(),
                         int(leaky), c_type, out.data_ptr(), n, None if work is None else work.data_ptr())
    _call(lib.objnerf_gemm_fp8, g, dev, "gemm_fp8")
    return out


def _rounded_product(x, w, bias, out_dtype):
    """x rounded and multiplied.  One kernel where a row of x is read by one tile of columns (307,200 x 128 x 256: 62 us against 79 us with
    x rounded first), where x is a tile itself (16 x 4096 x 4096: 15 against 20) or the product no more than a launch (2,048 x 512 x
    256: 11 against 16); x rounded first where it is read more often (307,200 x 256 x 256: 107 against 111, 64 x 4096 x 4096: 21
    against 25; rounding inside hides none of its loads behind the products, as built)."""
    m, k, n = x.shape[0], x.shape[1], w.data.shape[0]
    if k and (n <= 128 or m <= 32 or (k <= 1024 and _up(m, BLOCK) * _up(n, BLOCK) <= 256 * BLOCK * BLOCK)):
        return _product(x, w, bias, False, out_dtype)
    return _product(_quantize(x, 1)[0], w, bias, False, out_dtype)


def _checked_fp8(x, name):
    if not isinstance(x, Fp8Matrix):
        raise TypeError("%s must be an Fp8Matrix (quantize_fp8), got %s" % (name, type(x).__name__))
    d, s = x.data, x.scale
    if d.dtype != torch.float8_e4m3fn or s.dtype != torch.uint8:
        raise TypeError("%s: data must be float8_e4m3fn and scale uint8, got %s and %s" % (name, d.dtype, s.dtype))
    width = _up(x.cols, BLOCK)
    if d.dim() != 2 or s.dim() != 2 or d.shape[1] != width or tuple(s.shape) != (d.shape[0], _up(width // BLOCK, 4)):
        raise ValueError("%s: data %s and scale %s do not hold %d columns in blocks of 128" % (name, tuple(d.shape), tuple(s.shape), x.cols))
    if not d.is_cuda:
        _lib.require_cuda(d, name)
    if s.device != d.device:
        raise ValueError("%s: data and scale must be on one device" % name)
    if not (d.is_contiguous() and s.is_contiguous()) or d.data_ptr() % 16 or s.data_ptr() % 4:
        raise ValueError("%s: data and scale must be contiguous and aligned to 16 and 4 bytes" % name)
    return x


def _checked_bias(bias, n, device):
    if bias is None:
        return None
    if not isinstance(bias, torch.Tensor):
        raise TypeError("bias must be a tensor, got %s" % type(bias).__name__)
    return _column(bias.detach(), "bias", n, device)


def quantize_fp8(x, block_rows=1, transpose=False):
    """x (R, C) rounded to an Fp8Matrix: blocks of 128 columns of one row (block_rows 1: activations, gradients) or of 128 rows
    (block_rows 128: weights).  A block's scale is the smallest power of two with max|block| / scale <= 448, so dividing by it is exact and
    an element is rounded once, to nearest even; infinities and NaN become NaN and set no scale.  `transpose` rounds x.T -- its blocks run
    along x's rows -- without forming it."""
    _refuse_recording()
    if block_rows not in (1, BLOCK):
        raise ValueError("block_rows must be 1 or 128, got %r" % (block_rows,))
    q, t, _ = _quantize(_rows(x, "x").detach(), block_rows, not transpose, transpose)
    return t if transpose else q


def matmul_fp8(a, b, bias=None, activation=None, out_dtype=torch.bfloat16):
    """a @ b.T (+ bias) of two Fp8Matrix (M, K) and (N, K) in out_dtype (float32, bfloat16 or float16).

    float32: fp32 sums.  bfloat16, float16: the 8-bit matrix instruction, at twice the rate.  It drops what lies more than 13 bits under the
    largest of eight products on the way into the fp32 sum, 1.5e-5 of the result's norm for normal numbers: less than a rounding for
    results of the usual size, but an element whose terms cancel can be off by more than its own rounding.  Take float32 where that
    counts.  The result is rounded once.  activation: None or "leaky_relu" (slope 0.01, the reference's layers).  Not differentiable
    (linear_fp8 is)."""
    _refuse_recording()
    _checked_fp8(a, "a")
    _checked_fp8(b, "b")
    if a.cols != b.cols:
        raise ValueError("a and b must have the same columns, got %d and %d" % (a.cols, b.cols))
    if a.data.device != b.data.device:
        raise ValueError("a and b must be on one device")
    if activation not in (None, "leaky_relu"):
        raise ValueError("activation must be None or 'leaky_relu', got %r" % (activation,))
    if out_dtype not in _TYPES:
        raise TypeError("out_dtype: %s is not supported" % (out_dtype,))
    _refuse_tangents(bias)
    if bias is not None and isinstance(bias, torch.Tensor) and bias.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("matmul_fp8 is inference-only: use linear_fp8 where a gradient is needed")
    return _product(a, b, _checked_bias(bias, b.data.shape[0], a.data.device), activation is not None, out_dtype)


class _LinearFp8Fn(torch.autograd.Function):
    """y = X8 W8^T + b; dX = dY8 W8, dW = (dY^T)8 (X^T)8, db = column sums of dY.  Kept for the backward pass: both transposed operands in
    their 8-bit form, written by the launches that round the forward's."""

    @staticmethod
    def forward(ctx, x, weight, bias, out_dtype):
        need_x, need_w, _, _ = ctx.needs_input_grad
        xq, xt, _ = _quantize(x, 1, True, need_w)
        wq, wt, _ = _quantize(weight, BLOCK, True, need_x)
        ctx.save_for_backward(*((xt.data, xt.scale) if need_w else (None, None)), *((wt.data, wt.scale) if need_x else (None, None)))
        ctx.types = x.dtype, weight.dtype, None if bias is None else bias.dtype
        ctx.sizes = x.shape[0], weight.shape[0], x.shape[1]
        return _product(xq, wq, _checked_bias(bias, weight.shape[0], x.device), False, out_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        _refuse_tangents(dy)
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        xt, sxt, wt, swt = ctx.saved_tensors
        m, n, k = ctx.sizes
        if dy.dtype not in _TYPES:
            dy = dy.float()
        dy = _rows(dy, "the gradient of y")
        if m == 0:
            db = torch.zeros(n, dtype=torch.float32, device=dy.device) if need_b else None
            dq, dt, _ = _quantize(dy, 1, need_x, need_w)
        else:
            dq, dt, db = _quantize(dy, 1, need_x or not need_w, need_w, need_b)
        dx = _product(dq, Fp8Matrix(wt, swt, n), None, False, ctx.types[0]) if need_x else None
        dw = _product(dt, Fp8Matrix(xt, sxt, m), None, False, ctx.types[1]) if need_w else None
        return dx, dw, None if db is None else db.to(ctx.types[2]), None


def linear_fp8(x, weight, bias=None, out_dtype=None):
    """x @ weight.T + bias, both factors rounded to 8-bit floating point with a scale for each block of 128 (x: 128 columns of a row,
    weight: 128 x 128), (M, N) in out_dtype (default: x's type).

    x (M, K); weight (N, K), K <= 2^26, a tensor -- rounded in every call, so that what an optimizer wrote is what counts -- or the Fp8Matrix that
    quantize_fp8(weight, block_rows=128) laid out once, for inference; bias (N,).  Sizes need not be multiples of anything.  With a tensor
    as weight it is differentiable: dX and dW are products of the same kind, of the gradient rounded along their own sums, in x's and
    weight's types (of at most 2^26 rows of x, of weight); the bias gradient is an fp32 sum.

    Results and gradients in float32 are fp32 sums; in bfloat16 and float16 they are those of the 8-bit matrix instruction (matmul_fp8)."""
    _refuse_recording()
    x = _rows(x, "x")
    _refuse_tangents(x, weight, bias)
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in _TYPES:
        raise TypeError("out_dtype: %s is not supported" % (out_dtype,))
    recording = torch.is_grad_enabled()
    if isinstance(weight, Fp8Matrix):
        _checked_fp8(weight, "weight")
        if weight.cols != x.shape[1] or weight.data.device != x.device:
            raise ValueError("x %s on %s does not fit a weight of %d columns on %s" % (tuple(x.shape), x.device, weight.cols, weight.data.device))
        if recording and (x.requires_grad or (isinstance(bias, torch.Tensor) and bias.requires_grad)):
            raise NotImplementedError("linear_fp8 with an Fp8Matrix is inference-only: pass the weight as a tensor where a gradient is needed")
        return _rounded_product(x, weight, _checked_bias(bias, weight.data.shape[0], x.device), out_dtype)
    weight = _rows(weight, "weight")
    if weight.shape[1] != x.shape[1] or weight.device != x.device:
        raise ValueError("x %s on %s does not fit weight %s on %s" % (tuple(x.shape), x.device, tuple(weight.shape), weight.device))
    if bias is not None:
        _checked_bias(bias, weight.shape[0], x.device)
    if recording and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        if (weight.requires_grad and x.shape[0] > MAX_SUM) or (x.requires_grad and weight.shape[0] > MAX_SUM):
            raise ValueError("a gradient that sums over more than 2^26 rows is not supported: x %s, weight %s" % (tuple(x.shape), tuple(weight.shape)))
        return _LinearFp8Fn.apply(x, weight, bias, out_dtype)
    return _rounded_product(x, _quantize(weight, BLOCK)[0], _checked_bias(bias, weight.shape[0], x.device), out_dtype)


# ---- distillation ----

def _distill_args(student, teacher, index, temperature):
    _refuse_recording()
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
    if n > MAX_INT or v > MAX_INT:
        raise ValueError("student must have fewer than 2^31 rows and labels, got %s" % (tuple(student.shape),))
    a = _lib.DistillArgs(n, v, k, student.data_ptr(), student.stride(0), _TYPES[student.dtype], _TYPES[teacher.dtype], teacher.data_ptr(), teacher.stride(0),
                         index.data_ptr(), index.stride(0), index.element_size(), 0, temperature)
    return a, (student, teacher, index)       # the tensors whose memory the arguments point to: kept until the call is enqueued


def _run_distill(a, keep, want_loss, upstream):
    student = keep[0]
    n, v = student.shape                      # (not a.n, a.v: torch.compile takes a structure's fields for their descriptors)
    loss = grad = None
    if want_loss:
        loss = torch.empty(n, dtype=torch.float32, device=student.device)
        a.loss = loss.data_ptr()
    if upstream is not None:
        grad = torch.empty(n, v, dtype=student.dtype, device=student.device)
        a.upstream, a.upstream_stride = upstream.data_ptr(), (upstream.stride(0) if upstream.dim() else 0)
        a.grad, a.grad_stride = grad.data_ptr(), v
    if n:
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
        _refuse_tangents(d_loss)
        if d_loss.dtype != torch.float32 or d_loss.is_neg():
            d_loss = d_loss.float().resolve_neg()
        a, keep = _distill_args(*ctx.saved_tensors, ctx.temperature)
        return _run_distill(a, keep, False, d_loss)[1], None, None, None


def distill_top_logits(student, teacher, index, temperature=1.0):
    """The distillation loss of every row, (N,) float32: KL(p || q) with p = softmax(teacher / T) over the row's filled slots and
    q = softmax(student / T) over all V labels.

    student (N, V); teacher (N, k) logits or log-probabilities, k <= 1024; index (N, k) int32 or int64, the labels that the
    teacher's values belong to.  A slot whose index lies outside [0, V) or whose value is -inf is empty; a row without a filled slot
    has loss 0 and gradient 0; otherwise NaN or +inf in the row, or nothing but -inf among the student's values, gives a loss of NaN, a
    label ruled out by the student (-inf) under a filled slot a loss of +inf.  An index may occur more than once (its shares add).  Differentiable with respect to `student`
    alone; the usual factor T^2 is the caller's.  The backward pass reads the student's row again instead of keeping a copy."""
    _refuse_tangents(student, teacher)
    if torch.is_grad_enabled() and isinstance(student, torch.Tensor) and student.requires_grad:
        return _DistillFn.apply(student, teacher, index, temperature)
    return _run_distill(*_distill_args(student, teacher, index, temperature), True, None)[0]


def distill_top_logits_grad(student, teacher, index, upstream, temperature=1.0):
    """(loss, grad) of distill_top_logits in one pass over the student's rows, for a loop that knows the gradient of its losses
    beforehand: `upstream` (N,) is d total / d loss_n (1 / N for a mean), grad = d total / d student in the student's type
    (`logits.backward(grad)` goes on from there)."""
    if not isinstance(upstream, torch.Tensor):
        raise TypeError("upstream must be a tensor, got %s" % type(upstream).__name__)
    _refuse_tangents(student, teacher, upstream)
    a, keep = _distill_args(student, teacher, index, temperature)
    return _run_distill(a, keep, True, _column(upstream.detach(), "upstream", keep[0].shape[0], keep[0].device))


# ---- drawing a label ----

def sample_logits(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One label per row, (N,) int64, drawn from logits (N, V), V <= 2^19, at the random numbers u (N,) in [0, 1).

    Weights are exp(logits / temperature) (up to a factor).  The labels in order -- falling logits, equal ones by rising index -- are
    cut to the first `top_k` (0: all), of those to the shortest prefix whose share of their weight reaches `top_p` (1: all; at
    least one label stays), of those to the ones with at least `min_p` times the largest weight (0: all).  The label is the
    first, in that order, whose running sum of weight exceeds u times their total.  temperature 0 and top_k 1 give the first
    of the order.  NaN counts as -inf; a row of nothing but -inf gives -1, which is no index: clamp it, and keep `labels >= 0`, before
    a table lookup.

    Each setting is a number or an (N,) tensor on the logits' device, one value per row, held as float32 (top_k: int32), as u is.  Runs
    give equal labels for equal inputs."""
    _refuse_recording()
    logits = _rows(logits, "logits")
    n, v = logits.shape
    dev = logits.device
    if not 1 <= v <= MAX_LABELS or n > MAX_INT:
        raise ValueError("sample_logits takes fewer than 2^31 rows of 1 to 2^19 labels, got %s" % (tuple(logits.shape),))
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
        a.temperature = temperature = float(temperature)
        if not 0.0 <= temperature < 1e300:
            raise ValueError("temperature must be >= 0 and finite, got %r" % temperature)
    if isinstance(top_k, torch.Tensor):
        if top_k.dtype == torch.uint64:                      # (2^63 and more count as -1: all)
            top_k = top_k.to(torch.int64)
        if top_k.dtype == torch.int64:
            top_k = top_k.clamp(-1, 2 ** 31 - 1)             # (the conversion would drop the upper half)
        keep.append(_column(top_k, "top_k", n, dev, torch.int32))
        a.top_k_rows = keep[-1].data_ptr()
    else:
        a.top_k = top_k = operator.index(top_k)
        if not 0 <= top_k < 1 << 31:
            raise ValueError("top_k must be >= 0, got %r" % top_k)
    if isinstance(top_p, torch.Tensor):
        keep.append(_column(top_p, "top_p", n, dev))
        a.top_p_rows = keep[-1].data_ptr()
    else:
        a.top_p = top_p = float(top_p)
        if not top_p >= 0.0:
            raise ValueError("top_p must be >= 0, got %r" % top_p)
    if isinstance(min_p, torch.Tensor):
        keep.append(_column(min_p, "min_p", n, dev))
        a.min_p_rows = keep[-1].data_ptr()
    else:
        a.min_p = min_p = float(min_p)
        if not 0.0 <= min_p <= 1.0:
            raise ValueError("min_p must lie in [0, 1], got %r" % min_p)
    labels = torch.empty(n, dtype=torch.int64, device=dev)
    a.labels = labels.data_ptr()
    lib = _lib.lib()
    room = lib.objnerf_sample_logits_workspace_bytes(n, v, a.type) if v > 512 else 0
    if room:
        work = torch.empty(room, dtype=torch.uint8, device=dev)
        a.workspace = work.data_ptr()
    if n:
        _call(lib.objnerf_sample_logits, a, dev, "sample_logits")
    return labels
