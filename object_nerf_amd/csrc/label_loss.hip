// label_loss.hip -- distillation of a teacher's top logits into rows of label logits: the loss of every row and its gradient.
//
//   p = softmax(t / T) over the row's k slots whose index lies in [0, v),  q = softmax(z / T) over the row's v logits
//   loss = sum_j p_j (log p_j - log q_{i_j})
//   dz_v = (g / T) (q_v - sum_{j : i_j = v} p_j)
//
// With m = max z, s = sum exp((z - m) / T), a_j = (t_j - max t) / T, A = sum exp(a_j), b_j = (z_{i_j} - m) / T:
//   loss = (1 / A) sum_j exp(a_j) (a_j - b_j) + log s - log A          (differences first: no large terms cancel)
// A student's value of the type's lowest number under a slot makes a term as large as fp32 holds, which its weight or the mean may
// bring back: the differences are taken at 2^-12 of their size, and T < 1 divides the weight.
//
// Bound by memory, short rows by the vector units (307,200 x 64: 0.90 busy): a row up to 256 KB is read once and stays in registers
// until dz is written (longer ones are read twice).  The statistics are fp32, the sums in a fixed order (bit-reproducible).  Measured:
// loss of 307,200 x 64 fp32 24 us = 3.6 TB/s, loss and gradient of 1,023 x 30,011 fp16 29 us = 4.2 TB/s and of 2,048 x 32,768 bf16 61 us =
// 4.4 TB/s (a copy of this card: 4.96).  The gradient's k special columns are not looked up while the row is written: the whole row is
// written as if p were 0, and behind a barrier the slots' own threads write their columns again.  The first slot of an index owns its
// column and adds the shares of later slots with the same index in their order.
#include "host_api.h"
#include "label_ops.h"
#include <type_traits>

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

// exp(a_j) (a_j - b_j) / 2^12 of a slot with weight e.  What the student rules out costs +inf whatever weight is left in fp32.
constexpr float kTermScale = 0x1p-12f;
__device__ __forceinline__ float slot_term(const DistillP& p, float e, float t, float tm, float z, float m) {
  if (z == -__builtin_inff()) return __builtin_inff();
  const float d = (t * kTermScale - tm * kTermScale) - (z * kTermScale - m * kTermScale);
  return p.inv_t <= 1.f ? e * (d * p.inv_t) : e * p.inv_t * d;
}

// Reduction over the LANES threads that hold a row: within a wave, or over a workgroup through LDS (tmp: one float per wave, its own
// for every call between two barriers of the caller).
template <int LANES, class OP>
__device__ __forceinline__ float row_reduce(float v, float* tmp) {
  if constexpr (LANES <= 64) {
    return lanes_reduce<LANES, OP>(v);
  } else {
    v = lanes_reduce<64, OP>(v);
    if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
    __syncthreads();
    v = tmp[0];
#pragma unroll
    for (int w = 1; w < LANES / 64; ++w) v = OP::f(v, tmp[w]);
    return v;
  }
}

// LANES threads per row (a row of 16 lanes, a wave, a workgroup).  PIECES > 0: the row stays in registers as it was read, LANES x PIECES
// pieces of 16 bytes, and memory sees it once; 0: it is read again in each pass.
template <class E, int LANES, int PIECES>
__global__ void __launch_bounds__(LANES < 256 ? 256 : LANES, LANES < 1024 ? 6 : 4) distill_kernel(DistillP p) {
  constexpr int kThreads = LANES < 256 ? 256 : LANES;
  constexpr bool kGroups = LANES <= 64;                          // several rows per workgroup: one slot per thread at most
  constexpr float kInf = __builtin_inff();
  __shared__ float tmp[6][kThreads / 64];
  __shared__ __align__(16) int slot_i[kGroups ? kThreads : kMaxSlots];
  __shared__ float slot_e[kGroups ? kThreads : kMaxSlots];
  const int t = kGroups ? threadIdx.x & (LANES - 1) : threadIdx.x;
  const long at = kGroups ? workgroup() * (kThreads / LANES) + threadIdx.x / LANES : workgroup();
  if (!kGroups && at >= p.n) return;
  const bool live = !kGroups || at < p.n;
  const long row = live ? at : p.n - 1;
  int* const my_i = slot_i + (kGroups ? threadIdx.x - t : 0);
  float* const my_e = slot_e + (kGroups ? threadIdx.x - t : 0);
  const char* z = static_cast<const char*>(p.z) + row * p.ldz * E::kBytes;
  const int pieces = p.v / E::kVec, tail = p.v - pieces * E::kVec;

  // asked for first: the row, then this thread's slot -- its index, the teacher's value of a filled slot, the student's value under it,
  // each behind the one before (and, as loads are counted in order, behind the row)
  u32x4 r[PIECES > 0 ? PIECES : 1];
  if constexpr (PIECES > 0)
#pragma unroll
    for (int c = 0; c < PIECES; ++c)
      if (t + c * LANES < pieces) r[c] = load16(z, (long)(t + c * LANES) * 16);
  const float last = t < tail ? E::load(z, (long)pieces * E::kVec + t) : -kInf;
  int i0 = t < p.k ? slot_column(p, row, t) : -1;
  const float t0 = i0 >= 0 ? load_any(p.t, row * p.ldt + t, p.t_type) : -kInf;
  if (t0 == -kInf) i0 = -1;                                      // a slot of -inf weighs nothing: empty
  const float z0 = i0 >= 0 ? E::load(z, i0) : 0.f;

  // largest of the row, of its teacher's values; is there a slot at all
  float m = last, s = 0.f;
  if constexpr (PIECES > 0) {
#pragma unroll
    for (int c = 0; c < PIECES; ++c)
      if (t + c * LANES < pieces) {
        float x[E::kVec];
        E::unpack(r[c], x);
#pragma unroll
        for (int i = 0; i < E::kVec; ++i) m = fmaxf(m, x[i]);
      }
  } else {
    // running maximum and sum, four pieces in flight
    for (int q = t; q < pieces; q += LANES * 4) {
      u32x4 f[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) f[u] = load16(z, (long)min(q + u * LANES, pieces - 1) * 16);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (q + u * LANES >= pieces) break;
        float x[E::kVec];
        E::unpack(f[u], x);
        float mx = x[0];
#pragma unroll
        for (int i = 1; i < E::kVec; ++i) mx = fmaxf(mx, x[i]);
        if (mx > m) { s *= fast_exp2((m - mx) * p.c); m = mx; }
        // a part of nothing but -inf adds nothing; NaN gets through either way
#pragma unroll
        for (int i = 0; i < E::kVec; ++i) s += x[i] == -kInf ? 0.f : fast_exp2((x[i] - m) * p.c);
      }
    }
    if (t < tail && last != -kInf) s += fast_exp2((last - m) * p.c);
  }
  float tm = t0, some = i0 >= 0 ? 1.f : 0.f;
  if constexpr (!kGroups) {
    if (t < p.k) { my_i[t] = i0; my_e[t] = t0; }
    if (t < (p.k + 3) / 4 * 4 - p.k) my_i[p.k + t] = -1;
    for (int j = t + LANES; j < p.k; j += LANES) {
      int i = slot_column(p, row, j);
      const float v = i >= 0 ? load_any(p.t, row * p.ldt + j, p.t_type) : -kInf;
      if (v == -kInf) i = -1;
      my_i[j] = i;
      my_e[j] = v;
      tm = fmaxf(tm, v);
      if (i >= 0) some = 1.f;
    }
  }
  const float own = m;
  m = row_reduce<LANES, OpMax>(m, tmp[0]);
  tm = row_reduce<LANES, OpMax>(tm, tmp[1]);
  some = row_reduce<LANES, OpMax>(some, tmp[2]);

  if constexpr (PIECES > 0) {
    float part[2] = {t < tail ? fast_exp2((last - m) * p.c) : 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < PIECES; ++c)
      if (t + c * LANES < pieces) {
        float x[E::kVec];
        E::unpack(r[c], x);
#pragma unroll
        for (int i = 0; i < E::kVec; ++i) part[i & 1] += fast_exp2((x[i] - m) * p.c);
      }
    s = part[0] + part[1];
  } else {
    // (own == -inf: this thread saw nothing else, s is 0 or NaN)
    if (own != m && own != -kInf) s *= fast_exp2((own - m) * p.c);
  }
  float A = 0.f, W = 0.f;                                        // sum of exp(a_j), and of exp(a_j) (a_j - b_j) / 2^12
  if (i0 >= 0) {
    const float e = expf((t0 - tm) * p.inv_t);
    A = e;
    W = slot_term(p, e, t0, tm, z0, m);
    my_e[t] = e;
  }
  if constexpr (kGroups) my_i[t] = i0;
  if constexpr (!kGroups)
    for (int j = t + LANES; j < p.k; j += LANES) {
      const int i = my_i[j];
      if (i < 0) continue;
      const float e = expf((my_e[j] - tm) * p.inv_t);
      A += e;
      W += slot_term(p, e, my_e[j], tm, E::load(z, i), m);
      my_e[j] = e;
    }
  s = row_reduce<LANES, OpSum>(s, tmp[3]);
  A = row_reduce<LANES, OpSum>(A, tmp[4]);
  W = row_reduce<LANES, OpSum>(W, tmp[5]);
  if (m == -kInf) s = __builtin_nanf("");                        // a row of nothing but -inf has no softmax
  if (p.loss && live && t == 0) p.loss[row] = some > 0.f ? W / A * (1.f / kTermScale) + (logf(s) - logf(A)) : 0.f;
  if (!p.dz) return;

  char* dz = static_cast<char*>(p.dz) + row * p.ldd * E::kBytes;
  const bool filled = some > 0.f;
  const float g = filled ? p.up[row * p.ldu] * p.inv_t : 0.f, coef = filled ? g / s : 0.f;
  if (live) {
    auto piece = [&](int q, u32x4 f) {
      u32x4 o = {0, 0, 0, 0};
      if (filled) {
        float x[E::kVec];
        E::unpack(f, x);
#pragma unroll
        for (int i = 0; i < E::kVec; ++i) x[i] = coef * fast_exp2((x[i] - m) * p.c);
        o = E::pack(x);
      }
      store16(dz, (long)q * 16, o);
    };
    if constexpr (PIECES > 0) {
#pragma unroll
      for (int c = 0; c < PIECES; ++c)
        if (t + c * LANES < pieces) piece(t + c * LANES, r[c]);
    } else {
      for (int q = t; q < pieces; q += LANES * 4) {
        u32x4 f[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) f[u] = load16(z, (long)min(q + u * LANES, pieces - 1) * 16);
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (q + u * LANES < pieces) piece(q + u * LANES, f[u]);
      }
    }
    if (t < tail) E::store(dz, (long)pieces * E::kVec + t, filled ? coef * fast_exp2((last - m) * p.c) : 0.f);
  }
  __syncthreads();                                               // the row stands: the slots' columns are written over it
  if (!live) return;
  for (int j = t; j < p.k; j += LANES) {
    const int i = my_i[j];
    if (i < 0) continue;
    float share = 0.f;
    bool first = true;
#pragma unroll 4
    for (int l = 0; l < p.k; l += 4) {                           // (behind the last slot: -1)
      const int4 o = *reinterpret_cast<const int4*>(my_i + l);
      const int same[4] = {o.x == i, o.y == i, o.z == i, o.w == i};
      if (same[0] | same[1] | same[2] | same[3])
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (same[q]) {
            if (l + q < j) first = false;
            share += my_e[l + q];
          }
    }
    const float zi = j == t ? z0 : E::load(z, i);
    if (first) E::store(dz, i, g * (fast_exp2((zi - m) * p.c) / s - share / A));
  }
}

// Threads per row: the fewest that hold it in registers at a few pieces each, and its slots at one each where rows share a workgroup.
// Loss and gradient in one pass, against the next wider form: 307200 x 64 fp32 16 lanes 42 us, a wave 155; 16384 x 1024 a wave 28, 256
// threads 37; 2048 x 8192 256 threads 25, 1,024 43; 2048 x 16384 512 threads 47, 1,024 60; read again in each pass instead of held:
// 2048 x 8192 39, 1024 x 65536 fp32 144 instead of 133, 512 x 131072 bf16 64 instead of 68, 16 x 131072 bf16 24 instead of 23.
template <class E>
int launch_distill(const DistillP& p, hipStream_t s) {
  const int pieces = p.v / E::kVec;
  auto run = [&](auto lanes, auto held) {
    constexpr int L = decltype(lanes)::value, P = decltype(held)::value;
    constexpr int threads = L < 256 ? 256 : L;
    hipLaunchKernelGGL((distill_kernel<E, L, P>), grid_of((p.n + threads / L - 1) / (threads / L)), dim3(threads), 0, s, p);
  };
  using std::integral_constant;
#define OBJ_ROWS(L, P) run(integral_constant<int, L>{}, integral_constant<int, P>{})
  if (p.k <= 16 && pieces <= 16) OBJ_ROWS(16, 1);
  else if (p.k <= 16 && pieces <= 32) OBJ_ROWS(16, 2);
  else if (p.k <= 16 && pieces <= 64) OBJ_ROWS(16, 4);
  else if (p.k <= 64 && pieces <= 64) OBJ_ROWS(64, 1);
  else if (p.k <= 64 && pieces <= 128) OBJ_ROWS(64, 2);
  else if (p.k <= 64 && pieces <= 256) OBJ_ROWS(64, 4);
  else if (pieces <= 1024) OBJ_ROWS(256, 4);
  else if (pieces <= 2048) OBJ_ROWS(256, 8);
  else if (pieces <= 4096) OBJ_ROWS(512, 8);
  else if (pieces <= 8192) OBJ_ROWS(1024, 8);
  else if (pieces <= 16384) OBJ_ROWS(1024, 16);
  else OBJ_ROWS(1024, 0);
#undef OBJ_ROWS
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
