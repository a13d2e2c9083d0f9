// label_sample.hip -- one label drawn from every row of logits at a given random number, behind the usual filters.
//
//   w_v  = exp((z_v - max z) / T)
//   the labels in order: falling z, equal ones by rising index
//   kept = the first top_k of them; of those the shortest prefix whose share of their weight reaches top_p; of those the ones
//          with w >= min_p.  Each of the three is a prefix of the order, so their meeting is one
//   label = the first of the order whose running sum is over u * (sum of the kept)
//
// Nothing is sorted.  A label's place is its 64-bit key: the logit's bits, ordered as integers, over the index's complement, so
// that keys are all different and equal logits go by the index.  Weights are held as integers, round(w 2^shift) with shift + log2 v
// <= 62: integer sums are exact and need no order, so histograms filled by atomics give the same bits in every run, and every
// question -- the place of the top_k-th, of the top_p border, of u -- is "which label does this count or this weight fall on".
// `find` answers it: a histogram over the row (first in equal steps of the logit, then of the key), the bin in which the running
// sum crosses, and again inside that bin until its members fit a list of kList, where each counts the better ones.
//
// An absolute error of 2^-shift per weight (2^-45 at 131,072 labels, 2^-52 below 1,025) moves a border by far less than a random
// number of 24 bits can resolve.  NaN counts as -inf; a row of nothing but -inf draws -1.
#include "host_api.h"
#include "label_ops.h"

namespace objnerf {
namespace {

constexpr int kBins = 1024, kList = 512;

struct SampleP {
  long n;
  int v;
  const void* z; long ldz;
  const float* u; long ldu;
  const float* t; double t0;              // per row, or one number where the pointer is null
  const int32_t* top_k; int top_k0;
  const float* top_p; double top_p0;
  const float* min_p; double min_p0;
  int shift;
  int64_t* out;
};

__device__ __forceinline__ unsigned order_bits(float z) {
  z = (z != z) ? -__builtin_inff() : z + 0.f;                    // NaN as -inf; -0 as +0
  const unsigned b = __float_as_uint(z);
  return b ^ ((int)b < 0 ? 0xffffffffu : 0x80000000u);
}
constexpr unsigned kNothing = 0x007fffffu;                       // order_bits(-inf)
__device__ __forceinline__ float value_of(unsigned k) { return __uint_as_float(k ^ ((int)k < 0 ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ uint64_t key_of(unsigned bits, int index) { return ((uint64_t)bits << 32) | (0xffffffffu - (unsigned)index); }

struct Found { uint64_t key, upto; };     // the label's key; weight of the order up to it, itself included

template <int THREADS>
struct Shared {
  unsigned count[kBins];
  uint64_t mass[kBins];
  uint64_t list_key[kList], list_mass[kList];
  uint64_t red[THREADS / 64];
  uint64_t part_m[THREADS / 64];
  unsigned part_c[THREADS / 64];
  unsigned listed;
  int bin;
  unsigned base_c, in_bin;
  uint64_t base_m;
  Found found;
};

template <int THREADS, class OP, class T>
__device__ __forceinline__ T block_all(T v, Shared<THREADS>& sh) {
  v = lanes_reduce<64, OP>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x >> 6] = (uint64_t)v;
  __syncthreads();
  T r = (T)sh.red[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) r = OP::f(r, (T)sh.red[w]);
  return r;
}
struct OpMax64 { template <class T> static __device__ __forceinline__ T f(T a, T b) { return a > b ? a : b; } };
struct OpMin64 { template <class T> static __device__ __forceinline__ T f(T a, T b) { return a < b ? a : b; } };

// The row as this workgroup holds it: each(f) calls f(order bits, index) for the labels of this thread
template <class E, int THREADS>
struct RowInMemory {
  const char* z;
  int v;
  template <class F> __device__ __forceinline__ void each(F f) const {
    const int pieces = v / E::kVec;
    for (int q = threadIdx.x; q < pieces; q += THREADS) {
      float x[E::kVec];
      E::unpack(load16(z, (long)q * 16), x);
#pragma unroll
      for (int i = 0; i < E::kVec; ++i) f(order_bits(x[i]), q * E::kVec + i);
    }
    for (int i = pieces * E::kVec + threadIdx.x; i < v; i += THREADS) f(order_bits(E::load(z, i)), i);
  }
};

struct Weight {
  double zmax, inv_t, one;                // one = 2^shift
  __device__ __forceinline__ uint64_t of(unsigned bits) const {
    const float z = value_of(bits);
    const double d = (double)z - zmax;                           // +inf - +inf: the largest itself
    return (double)z == zmax ? (uint64_t)one : (uint64_t)__double2ull_rn(exp(d * inv_t) * one);
  }
};

// The label on which position `want` falls, by count (COUNT: the want-th of the order, from 0) or by weight (the first whose running
// sum is over `want`), among the labels with low <= key <= high, `members` of them.  The histogram in sh.count / sh.mass is that
// of the whole range in steps of (zmax - z) * step where `ready`.
template <bool COUNT, int THREADS, class ROW>
__device__ Found find(const ROW& row, const Weight& w, uint64_t low, uint64_t high, unsigned members, uint64_t want, float step, Shared<THREADS>& sh) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  unsigned base_c = 0;
  uint64_t base_m = 0;
  const float top = (float)w.zmax;
  bool by_value = step > 0.f;
  int bits = 0;
  for (int round = 0; members > (unsigned)kList && round < 10; ++round) {     // 64 bits of key, at least 9 a round
    if (!by_value) {                                             // the members' own range, in equal steps of the key
      uint64_t lo = ~0ull, hi = 0;
      row.each([&](unsigned b, int i) {
        const uint64_t k = key_of(b, i);
        if (k >= low && k <= high) { lo = k < lo ? k : lo; hi = k > hi ? k : hi; }
      });
      low = block_all<THREADS, OpMin64>(lo, sh);
      high = block_all<THREADS, OpMax64>(hi, sh);
      const uint64_t span = high - low;
      bits = 0;
      while ((span >> bits) >= (uint64_t)kBins) ++bits;
    }
    auto bin_of = [&](unsigned b, uint64_t k) {
      return by_value ? (int)fminf((top - value_of(b)) * step, (float)(kBins - 1)) : (int)((high - k) >> bits);
    };
    for (int i = tid; i < kBins; i += THREADS) { sh.count[i] = 0; sh.mass[i] = 0; }
    __syncthreads();
    row.each([&](unsigned b, int i) {
      const uint64_t k = key_of(b, i);
      if (k < low || k > high) return;
      const int at = bin_of(b, k);
      atomicAdd(&sh.count[at], 1u);
      if (!COUNT) atomicAdd((unsigned long long*)&sh.mass[at], (unsigned long long)w.of(b));
    });
    __syncthreads();
    // the bin in which the running sum crosses `want`
    constexpr int PER = kBins / THREADS;
    unsigned c = 0;
    uint64_t m = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) { c += sh.count[tid * PER + i]; m += sh.mass[tid * PER + i]; }
    unsigned ci = c;
    uint64_t mi = m;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const unsigned cu = __shfl_up(ci, o);
      const uint64_t mu = ((uint64_t)__shfl_up((unsigned)(mi >> 32), o) << 32) | __shfl_up((unsigned)mi, o);
      if (lane >= o) { ci += cu; mi += mu; }
    }
    if (lane == 63) { sh.part_c[wave] = ci; sh.part_m[wave] = mi; }
    __syncthreads();
    unsigned cb = base_c + ci - c;
    uint64_t mb = base_m + mi - m;
    for (int x = 0; x < wave; ++x) { cb += sh.part_c[x]; mb += sh.part_m[x]; }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const unsigned cc = sh.count[tid * PER + i];
      const uint64_t mm = sh.mass[tid * PER + i];
      if (COUNT ? (cb <= want && want < (uint64_t)cb + cc) : (mb <= want && want < mb + mm)) {
        sh.bin = tid * PER + i;
        sh.base_c = cb;
        sh.base_m = mb;
        sh.in_bin = cc;
      }
      cb += cc;
      mb += mm;
    }
    __syncthreads();
    const int bin = sh.bin;
    base_c = sh.base_c;
    base_m = sh.base_m;
    members = sh.in_bin;
    // the bin's own range of keys
    uint64_t lo = ~0ull, hi = 0;
    row.each([&](unsigned b, int i) {
      const uint64_t k = key_of(b, i);
      if (k < low || k > high || bin_of(b, k) != bin) return;
      lo = k < lo ? k : lo;
      hi = k > hi ? k : hi;
    });
    low = block_all<THREADS, OpMin64>(lo, sh);
    high = block_all<THREADS, OpMax64>(hi, sh);
    by_value = false;
  }
  __syncthreads();
  if (tid == 0) sh.listed = 0;
  __syncthreads();
  row.each([&](unsigned b, int i) {
    const uint64_t k = key_of(b, i);
    if (k < low || k > high) return;
    const unsigned at = atomicAdd(&sh.listed, 1u);
    if (at < (unsigned)kList) {
      sh.list_key[at] = k;
      sh.list_mass[at] = COUNT ? 0 : w.of(b);
    }
  });
  __syncthreads();
  const int n = (int)min(sh.listed, (unsigned)kList);
  for (int e = tid; e < n; e += THREADS) {
    const uint64_t k = sh.list_key[e];
    uint64_t before = COUNT ? base_c : base_m;
    for (int l = 0; l < n; ++l)
      if (sh.list_key[l] > k) before += COUNT ? 1 : sh.list_mass[l];
    const uint64_t upto = before + (COUNT ? 1 : sh.list_mass[e]);
    if (before <= want && want < upto) sh.found = Found{k, upto};
  }
  __syncthreads();
  return sh.found;
}

template <class E, int THREADS>
__global__ void __launch_bounds__(THREADS) sample_row_kernel(SampleP p) {
  __shared__ Shared<THREADS> sh;
  const long r = blockIdx.x;
  const RowInMemory<E, THREADS> row{static_cast<const char*>(p.z) + r * p.ldz * E::kBytes, p.v};
  const double t = p.t ? (double)p.t[r] : p.t0;
  const int top_k = p.top_k ? p.top_k[r] : p.top_k0;         // <= 0: off
  const double top_p = p.top_p ? (double)p.top_p[r] : p.top_p0, min_p = p.min_p ? (double)p.min_p[r] : p.min_p0;
  const float u = p.u[r * p.ldu];

  uint64_t best = 0;
  unsigned lowest = 0xffffffffu, some = 0;
  row.each([&](unsigned b, int i) {
    if (b == kNothing) return;
    const uint64_t k = key_of(b, i);
    best = k > best ? k : best;
    lowest = b < lowest ? b : lowest;
    ++some;
  });
  best = block_all<THREADS, OpMax64>(best, sh);
  lowest = block_all<THREADS, OpMin64>(lowest, sh);
  some = block_all<THREADS, OpSum>(some, sh);
  if (some == 0 || !(t > 0.0) || top_k == 1) {                   // nothing to draw; or one label alone
    if (threadIdx.x == 0) p.out[r] = some == 0 ? -1 : (int64_t)(0xffffffffu - (unsigned)best);
    return;
  }
  Weight w;
  w.zmax = (double)value_of((unsigned)(best >> 32));
  w.inv_t = 1.0 / t;
  w.one = ldexp(1.0, p.shift);
  const float reach = (float)w.zmax - fmaxf(value_of(lowest), -1e30f);
  const float step = reach > 0.f && reach < 1e30f ? (float)(kBins - 1) / reach : 0.f;
  uint64_t low = key_of(kNothing + 1, 0x7fffffff);
  if (top_k > 0 && (unsigned)top_k < some) {
    low = find<true, THREADS>(row, w, low, best, some, (uint64_t)(top_k - 1), step, sh).key;
    some = (unsigned)top_k;
  }
  uint64_t all = 0, strong = 0;
  const double border = min_p > 0.0 ? fmax(-log(min_p), 0.0) : __builtin_inf();     // the strongest label always stays
  row.each([&](unsigned b, int i) {
    if (key_of(b, i) < low) return;
    const uint64_t m = w.of(b);
    all += m;
    const double d = w.zmax - (double)value_of(b);
    if (!(d * w.inv_t > border)) strong += m;
  });
  all = block_all<THREADS, OpSum>(all, sh);
  strong = block_all<THREADS, OpSum>(strong, sh);
  uint64_t kept = all;
  if (top_p < 1.0) {
    const double want = ceil(top_p * (double)all);
    const uint64_t position = want >= 1.0 ? (uint64_t)want - 1 : 0;
    kept = find<false, THREADS>(row, w, low, best, some, position < all ? position : all - 1, step, sh).upto;
  }
  kept = strong < kept ? strong : kept;
  const double want = floor((double)u * (double)kept);
  uint64_t position = want >= 1.0 ? (want < (double)kept ? (uint64_t)want : kept - 1) : 0;
  if (position >= kept) position = kept - 1;
  const Found f = find<false, THREADS>(row, w, low, best, some, position, step, sh);
  if (threadIdx.x == 0) p.out[r] = (int64_t)(0xffffffffu - (unsigned)f.key);
}

template <class E>
int launch_sample(const SampleP& p, hipStream_t s) {
  hipLaunchKernelGGL((sample_row_kernel<E, 256>), dim3((unsigned)p.n), dim3(256), 0, s, p);
  return check_launch("sample_logits");
}

}  // namespace
}  // namespace objnerf

using namespace objnerf;

extern "C" int objnerf_sample_logits(const objnerf_sample_args* a, void* stream) {
  if (!a) return set_error(-1, "sample_logits: no arguments");
  if (a->n < 0 || a->n > INT32_MAX || a->v < 1) return set_error(-1, "sample_logits: bad sizes (n < 2^31, v >= 1)");
  if (!label_type_ok(a->type)) return set_error(-1, "sample_logits: unknown element type");
  if (a->logits_stride < 0 || a->u_stride < 0) return set_error(-1, "sample_logits: bad strides");
  if (!a->temperature_rows && !(a->temperature >= 0.0 && a->temperature < 1e300)) return set_error(-1, "sample_logits: the temperature must be >= 0 and finite");
  if (!a->top_k_rows && a->top_k < 0) return set_error(-1, "sample_logits: top_k must be >= 0");
  if (!a->top_p_rows && !(a->top_p >= 0.0)) return set_error(-1, "sample_logits: top_p must be >= 0");
  if (!a->min_p_rows && !(a->min_p >= 0.0 && a->min_p <= 1.0)) return set_error(-1, "sample_logits: min_p must lie in [0, 1]");
  if (a->n == 0) return 0;
  if (!a->logits || !a->u || !a->labels) return set_error(-1, "sample_logits: a needed buffer is missing");
  SampleP p;
  p.n = a->n; p.v = a->v;
  p.z = a->logits; p.ldz = a->logits_stride;
  p.u = a->u; p.ldu = a->u_stride;
  p.t = a->temperature_rows; p.t0 = a->temperature;
  p.top_k = a->top_k_rows; p.top_k0 = (int)(a->top_k < a->v ? a->top_k : 0);
  p.top_p = a->top_p_rows; p.top_p0 = a->top_p;
  p.min_p = a->min_p_rows; p.min_p0 = a->min_p;
  int log_v = 0;
  while ((1ll << log_v) < (long long)a->v) ++log_v;
  p.shift = 62 - log_v < 52 ? 62 - log_v : 52;
  p.out = a->labels;
  hipStream_t s = (hipStream_t)stream;
  return a->type == OBJNERF_TYPE_F32 ? launch_sample<ElemF32>(p, s)
         : a->type == OBJNERF_TYPE_BF16 ? launch_sample<ElemBf16>(p, s) : launch_sample<ElemF16>(p, s);
}
