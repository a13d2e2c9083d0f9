// label_loss.hip -- distillation of a teacher's top logits into rows of label logits: the loss of every row and its gradient.
//
//   p = softmax(t / T) over the row's k slots whose index lies in [0, v),  q = softmax(z / T) over the row's v logits
//   loss = sum_j p_j (log p_j - log q_{i_j})
//   dz_v = (g / T) (q_v - sum_{j : i_j = v} p_j)
//
// With m = max z, s = sum exp((z - m) / T), a_j = (t_j - max t) / T, A = sum exp(a_j), b_j = (z_{i_j} - m) / T:
//   loss = (1 / A) sum_j exp(a_j) (a_j - b_j) + log s - log A          (differences first: no large terms cancel)
//
// Bound by memory: z is read once for (m, s) and, where the gradient is asked for, once more while dz is written.  The statistics
// are fp32, the sums in a fixed order (bit-reproducible).  The gradient's k special columns are not looked up while the row is
// written: the whole row is written as if p were 0, and behind a barrier the slots' own threads write their columns again.  The
// first slot of an index owns its column and adds the shares of later slots with the same index in their order.
#include "host_api.h"
#include "label_ops.h"

namespace objnerf {
namespace {

constexpr int kMaxSlots = 1024;                 // slots of a row: their indices and weights are kept in LDS

struct DistillP {
  long n;
  int v, k;
  const void* z; long ldz;
  const void* t; int t_type; long ldt;
  const void* idx; int idx_bytes; long ldi;
  float c;                                      // log2(e) / T: exp((z - m) / T) = exp2((z - m) c)
  float inv_t;
  float* loss;
  const float* up; long ldu;
  void* dz; long ldd;
};

// one v_exp_f32 (1 ulp; results under 2^-126 are 0)
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// slot j of a row: its column, or -1 where the slot is empty
__device__ __forceinline__ int slot_column(const DistillP& p, long row, int j) {
  if (p.idx_bytes == 4) {
    const int i = static_cast<const int32_t*>(p.idx)[row * p.ldi + j];
    return i >= 0 && i < p.v ? i : -1;
  }
  const long i = static_cast<const int64_t*>(p.idx)[row * p.ldi + j];
  return i >= 0 && i < p.v ? (int)i : -1;
}

template <int THREADS, class OP>
__device__ __forceinline__ float block_reduce(float v, float* tmp) {
  v = lanes_reduce<64, OP>(v);
  if constexpr (THREADS > 64) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();                            // tmp's last readers are done
    if ((threadIdx.x & 63) == 0) tmp[wave] = v;
    __syncthreads();
    v = tmp[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) v = OP::f(v, tmp[w]);
  }
  return v;
}

// One workgroup per row.  The row is read in 16-byte pieces, four in flight per thread.
template <class E, int THREADS>
__global__ void __launch_bounds__(THREADS) distill_row_kernel(DistillP p) {
  __shared__ float tmp[THREADS / 64], tmp2[THREADS / 64];
  __shared__ int slot_i[kMaxSlots];
  __shared__ float slot_e[kMaxSlots];
  const long row = blockIdx.x;
  const int tid = threadIdx.x;
  const char* z = static_cast<const char*>(p.z) + row * p.ldz * E::kBytes;
  const int pieces = p.v / E::kVec;
  constexpr float kInf = __builtin_inff();

  // running maximum and sum
  float m = -kInf, s = 0.f;
  for (int q = tid; q < pieces; q += THREADS * 4) {
    u32x4 r[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) r[u] = load16(z, (long)min(q + u * THREADS, pieces - 1) * 16);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (q + u * THREADS >= pieces) break;
      float x[E::kVec];
      E::unpack(r[u], x);
      float mx = x[0];
#pragma unroll
      for (int i = 1; i < E::kVec; ++i) mx = fmaxf(mx, x[i]);
      if (mx > m) { s *= fast_exp2((m - mx) * p.c); m = mx; }
      // a part of nothing but -inf adds nothing; NaN gets through either way
#pragma unroll
      for (int i = 0; i < E::kVec; ++i) s += x[i] == -kInf ? 0.f : fast_exp2((x[i] - m) * p.c);
    }
  }
  for (int i = pieces * E::kVec + tid; i < p.v; i += THREADS) {
    const float x = E::load(z, i);
    if (x > m) { s *= fast_exp2((m - x) * p.c); m = x; }
    s += x == -kInf ? 0.f : fast_exp2((x - m) * p.c);
  }
  {
    const float mm = block_reduce<THREADS, OpMax>(m, tmp);
    s = m == mm ? s : s * fast_exp2((m - mm) * p.c);
    s = m == -kInf && !(s != s) ? 0.f : s;
    m = mm;
    s = block_reduce<THREADS, OpSum>(s, tmp2);
    if (m == -kInf) s = __builtin_nanf("");     // a row of nothing but -inf has no softmax
  }

  // the teacher's slots
  float tm = -kInf, some = 0.f;
  for (int j = tid; j < p.k; j += THREADS) {
    const int i = slot_column(p, row, j);
    const float t = i >= 0 ? load_any(p.t, row * p.ldt + j, p.t_type) : -kInf;
    slot_i[j] = i >= 0 && t != -kInf ? i : -1;  // a slot of -inf weighs nothing: empty
    slot_e[j] = t;
    if (slot_i[j] >= 0) { tm = fmaxf(tm, t); some = 1.f; }
  }
  tm = block_reduce<THREADS, OpMax>(tm, tmp);
  some = block_reduce<THREADS, OpMax>(some, tmp2);
  float A = 0.f, W = 0.f;
  for (int j = tid; j < p.k; j += THREADS) {
    const int i = slot_i[j];
    float e = 0.f;
    if (i >= 0) {
      const float a = (slot_e[j] - tm) * p.inv_t;
      e = expf(a);
      const float b = (E::load(z, i) - m) * p.inv_t;
      A += e;
      if (e != 0.f) W += e * (a - b);
    }
    slot_e[j] = e;
  }
  A = block_reduce<THREADS, OpSum>(A, tmp);
  W = block_reduce<THREADS, OpSum>(W, tmp2);
  if (p.loss && tid == 0) p.loss[row] = some > 0.f ? W / A + (logf(s) - logf(A)) : 0.f;
  if (!p.dz) return;

  char* dz = static_cast<char*>(p.dz) + row * p.ldd * E::kBytes;
  const float g = some > 0.f ? p.up[row * p.ldu] * p.inv_t : 0.f, coef = g / s;
  if (!(some > 0.f)) {
    const u32x4 zero = {0, 0, 0, 0};
    for (int q = tid; q < pieces; q += THREADS) store16(dz, (long)q * 16, zero);
    for (int i = pieces * E::kVec + tid; i < p.v; i += THREADS) E::store(dz, i, 0.f);
    return;
  }
  for (int q = tid; q < pieces; q += THREADS * 4) {
    u32x4 r[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) r[u] = load16(z, (long)min(q + u * THREADS, pieces - 1) * 16);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (q + u * THREADS >= pieces) break;
      float x[E::kVec];
      E::unpack(r[u], x);
#pragma unroll
      for (int i = 0; i < E::kVec; ++i) x[i] = coef * fast_exp2((x[i] - m) * p.c);
      store16(dz, (long)(q + u * THREADS) * 16, E::pack(x));
    }
  }
  for (int i = pieces * E::kVec + tid; i < p.v; i += THREADS) E::store(dz, i, coef * fast_exp2((E::load(z, i) - m) * p.c));
  __syncthreads();                              // the row stands: the slots' columns are written over it
  for (int j = tid; j < p.k; j += THREADS) {
    const int i = slot_i[j];
    if (i < 0) continue;
    float share = 0.f;
    bool first = true;
    for (int l = 0; l < p.k; ++l)
      if (slot_i[l] == i) {
        if (l < j) first = false;
        share += slot_e[l];
      }
    if (first) E::store(dz, i, g * (fast_exp2((E::load(z, i) - m) * p.c) / s - share / A));
  }
}

template <class E>
int launch_distill(const DistillP& p, hipStream_t s) {
  hipLaunchKernelGGL((distill_row_kernel<E, 256>), dim3((unsigned)p.n), dim3(256), 0, s, p);
  return check_launch("distill_top");
}

}  // namespace
}  // namespace objnerf

using namespace objnerf;

extern "C" int objnerf_distill_top(const objnerf_distill_args* a, void* stream) {
  if (!a) return set_error(-1, "distill_top: no arguments");
  if (a->n < 0 || a->n > INT32_MAX || a->v < 1 || a->k < 1 || a->k > kMaxSlots)
    return set_error(-1, "distill_top: bad sizes (n < 2^31, v >= 1, 1 <= k <= 1024)");
  if (!label_type_ok(a->student_type) || !label_type_ok(a->teacher_type) || (a->index_bytes != 4 && a->index_bytes != 8))
    return set_error(-1, "distill_top: unknown element type");
  if (!(a->temperature >= 1e-30) || !(a->temperature <= 1e30)) return set_error(-1, "distill_top: the temperature must lie in [1e-30, 1e30]");
  if (a->student_stride < 0 || a->teacher_stride < 0 || a->index_stride < 0 || a->upstream_stride < 0 || (a->grad && a->grad_stride < a->v))
    return set_error(-1, "distill_top: bad strides");
  if (a->n == 0) return 0;
  if (!a->student || !a->teacher || !a->index || (!a->loss && !a->grad) || (a->grad && !a->upstream))
    return set_error(-1, "distill_top: a needed buffer is missing");
  DistillP p;
  p.n = a->n; p.v = a->v; p.k = a->k;
  p.z = a->student; p.ldz = a->student_stride;
  p.t = a->teacher; p.t_type = a->teacher_type; p.ldt = a->teacher_stride;
  p.idx = a->index; p.idx_bytes = a->index_bytes; p.ldi = a->index_stride;
  p.c = (float)(1.4426950408889634 / a->temperature);
  p.inv_t = (float)(1.0 / a->temperature);
  p.loss = a->loss; p.up = a->upstream; p.ldu = a->upstream_stride; p.dz = a->grad; p.ldd = a->grad_stride;
  hipStream_t s = (hipStream_t)stream;
  return a->student_type == OBJNERF_TYPE_F32 ? launch_distill<ElemF32>(p, s)
         : a->student_type == OBJNERF_TYPE_BF16 ? launch_distill<ElemBf16>(p, s) : launch_distill<ElemF16>(p, s);
}
