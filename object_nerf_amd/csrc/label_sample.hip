// label_sample.hip -- one label drawn from every row of logits at a given random number, behind the usual filters.
//
//   w_v  = exp((z_v - max z) / T)
//   the labels in order: falling z, equal ones by rising index
//   kept = the first top_k of them; of those the shortest prefix whose share of their weight reaches top_p; of those the ones
//          with w >= min_p.  Each of the three is a prefix of the order, so their meeting is one
//   label = the first of the order whose running sum is over u * (sum of the kept)
//
// A label's place is its 64-bit key: the logit's bits, ordered as integers, over the index's complement, so that keys are all different
// and equal logits go by the index.  Weights are held as integers, round(w 2^shift) with shift + log2 v <= 62: integer sums are exact
// and need no order, so sums formed by atomics give the same bits in every run.  An absolute error of 2^-shift per weight (2^-45 at
// 131,072 labels, 2^-51 below 2,049) moves a border by far less than a random number of 24 bits can resolve.
//
// Rows of up to 512 labels are sorted in the registers of 16 or 64 lanes, and every question -- which are the top_k, where does the
// running sum pass top_p, where u -- is then a prefix sum away.  Longer rows are not sorted: with a small top_k the candidates are
// picked out by a bound (the top_k-th largest of the threads' own maxima), else each question is answered by a histogram in equal
// steps of the logit and by looking into the one bin in which the running sum crosses.
//
// NaN counts as -inf; a row of nothing but -inf draws -1.
#include "host_api.h"
#include "label_ops.h"
#include <type_traits>

namespace objnerf {
namespace {

constexpr int kBins = 2048, kList = 512, kPrune = 128;

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
struct Settings {
  double t, top_p, min_p;
  int top_k;                              // <= 0: off
  float u;
};
__device__ __forceinline__ Settings settings_of(const SampleP& p, long r) {
  Settings s;
  s.t = p.t ? (double)p.t[r] : p.t0;
  s.top_k = p.top_k ? p.top_k[r] : p.top_k0;
  s.top_p = p.top_p ? (double)p.top_p[r] : p.top_p0;
  s.min_p = p.min_p ? (double)p.min_p[r] : p.min_p0;
  s.u = p.u[r * p.ldu];
  return s;
}

__device__ __forceinline__ unsigned order_bits(float z) {
  z = (z != z) ? -__builtin_inff() : z + 0.f;                    // NaN as -inf; -0 as +0
  const unsigned b = __float_as_uint(z);
  return b ^ ((int)b < 0 ? 0xffffffffu : 0x80000000u);
}
constexpr unsigned kNothing = 0x007fffffu;                       // order_bits(-inf)
__device__ __forceinline__ float value_of(unsigned k) { return __uint_as_float(k ^ ((int)k < 0 ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ uint64_t key_of(unsigned bits, int index) { return ((uint64_t)bits << 32) | (0xffffffffu - (unsigned)index); }

// round(exp((z - zmax) / T) 2^shift).  exp as 2^(n / 32) of a table of 32 doubles in LDS (two banks each: no conflicts) times a
// polynomial on |r| <= 1/64, relative error 2^-48; the rounding to a whole number is the addition of 2^52.  17 instructions where the
// library's exp and conversion take about 60.
struct Weight {
  double zmax, c;                         // c = log2(e) / T
  int shift;
  const double* table;                    // 2^(i / 32)
  __device__ __forceinline__ uint64_t of(unsigned bits) const {
    const double z = (double)value_of(bits);
    const double t = fmax((z - zmax) * c, -2000.0);
    const double n = rint(t * 32.0);
    const double r = fma(n, -1.0 / 32.0, t);
    double p = fma(r, 1.33335581464284434e-3, 9.61812910762847716e-3);
    p = fma(r, p, 5.55041086648215800e-2);
    p = fma(r, p, 2.40226506959100712e-1);
    p = fma(r, p, 6.93147180559945309e-1);
    p = fma(r, p, 1.0);
    const int i = (int)n;
    const double w = ldexp(p * table[i & 31], (i >> 5) + shift) + 4503599627370496.0;
    const uint64_t whole = (uint64_t)__double_as_longlong(w) & 0xfffffffffffffull;
    return z == zmax ? 1ull << shift : whole;                    // also where both are +inf
  }
};
__device__ __forceinline__ void fill_table(double* table) {
  if (threadIdx.x < 32) table[threadIdx.x] = exp2((double)threadIdx.x * (1.0 / 32.0));
}

// positions in the running sum: the one on which the top_p border falls (its label is the last one kept), and u's
__device__ __forceinline__ uint64_t border_of(double top_p, uint64_t all) {
  const double want = ceil(top_p * (double)all);
  const uint64_t at = want >= 1.0 ? (uint64_t)want - 1 : 0;
  return at < all ? at : all - 1;
}
__device__ __forceinline__ uint64_t position_of(float u, uint64_t kept) {
  const double want = floor((double)u * (double)kept);
  const uint64_t at = want >= 1.0 ? (want < (double)kept ? (uint64_t)want : kept - 1) : 0;
  return at < kept ? at : kept - 1;
}
// -log2(min_p): what a label may lie below the largest in units of log2(e) / T; the strongest label always stays
__device__ __forceinline__ double reach_of(double min_p) { return min_p > 0.0 ? fmax(-log2(min_p), 0.0) : __builtin_inf(); }
__device__ __forceinline__ bool is_strong(const Weight& w, unsigned bits, double reach) {
  return !((w.zmax - (double)value_of(bits)) * w.c > reach);
}

// ---- rows of up to LANES x PER labels: a sorting network in registers ----
// The key as a double, so that a comparison is one instruction: sign 0, exponent field in [0x400, 0x5ff] (never NaN), order bits, then
// the complement of the index; nothing to draw: 0.0.
constexpr uint64_t kKeyBase = 0x4000000000000000ull;
constexpr unsigned kIndexMask = 0x1fffffffu;
__device__ __forceinline__ double sort_key(float z, int index) {
  const unsigned b = order_bits(z);
  return b == kNothing ? 0.0 : __longlong_as_double((long long)(kKeyBase | ((uint64_t)b << 29) | (kIndexMask - (unsigned)index)));
}
__device__ __forceinline__ unsigned sorted_bits(double k) { return (unsigned)((uint64_t)__double_as_longlong(k) >> 29); }
__device__ __forceinline__ int sorted_index(double k) { return (int)(kIndexMask - ((unsigned)(uint64_t)__double_as_longlong(k) & kIndexMask)); }

template <int MASK> __device__ __forceinline__ unsigned lane_xor(unsigned v) {
  if constexpr (MASK == 1) return dpp_u32<0xB1>(v);
  else if constexpr (MASK == 2) return dpp_u32<0x4E>(v);
  else if constexpr (MASK == 3) return dpp_u32<0x1B>(v);
  else if constexpr (MASK == 4) return dpp_u32<0x1B>(dpp_u32<0x141>(v));         // xor 7, xor 3
  else if constexpr (MASK == 7) return dpp_u32<0x141>(v);
  else if constexpr (MASK == 8) return dpp_u32<0x128>(v);                        // row_ror:8
  else if constexpr (MASK == 15) return dpp_u32<0x140>(v);
  else {
    static_assert(MASK == 16 || MASK == 31 || MASK == 32 || MASK == 63, "a step of the network");
    if constexpr (MASK == 31) v = dpp_u32<0x140>(v);
    if constexpr (MASK == 63) v = lane_xor<31>(v);
    unsigned a, b;
    rows_of<(MASK >= 32)>(v, a, b);                              // a: the lower row's, b: the upper row's, in both
    const bool upper = threadIdx.x & (MASK >= 32 ? 32 : 16);
    return upper ? a : b;
  }
}
template <int MASK> __device__ __forceinline__ double lane_xor(double v) {
  const uint64_t x = (uint64_t)__double_as_longlong(v);
  return __longlong_as_double((long long)(((uint64_t)lane_xor<MASK>((unsigned)(x >> 32)) << 32) | lane_xor<MASK>((unsigned)x)));
}
__device__ __forceinline__ void order_pair(double& a, double& b) {
  const double hi = fmax(a, b), lo = fmin(a, b);
  a = hi;
  b = lo;
}
// one step across lanes: the lower lane keeps the larger.  MIRROR: the partner's registers in reverse order
template <int MASK, int PER, bool MIRROR> __device__ __forceinline__ void lane_exchange(double (&x)[PER]) {
  constexpr int top = MASK >= 32 ? 32 : MASK >= 16 ? 16 : MASK >= 8 ? 8 : MASK >= 4 ? 4 : MASK >= 2 ? 2 : 1;
  const bool upper = threadIdx.x & top;
  double y[PER];
#pragma unroll
  for (int r = 0; r < PER; ++r) y[r] = lane_xor<MASK>(x[r]);
#pragma unroll
  for (int r = 0; r < PER; ++r) {
    const double o = y[MIRROR ? PER - 1 - r : r];
    x[r] = (x[r] > o) != upper ? x[r] : o;
  }
}
// merges of register pairs at distances D, D / 2, .. 1
template <int PER, int D> __device__ __forceinline__ void register_steps(double (&x)[PER]) {
  if constexpr (D >= 1) {
#pragma unroll
    for (int r = 0; r < PER; ++r)
      if (!(r & D)) order_pair(x[r], x[r | D]);
    register_steps<PER, D / 2>(x);
  }
}
template <int PER, int K> __device__ __forceinline__ void register_sort(double (&x)[PER]) {
  if constexpr (K <= PER) {
#pragma unroll
    for (int r = 0; r < PER; ++r)
      if (!(r & (K / 2))) order_pair(x[r], x[r ^ (K - 1)]);
    register_steps<PER, K / 4>(x);
    register_sort<PER, K * 2>(x);
  }
}
template <int PER, int D> __device__ __forceinline__ void lane_steps(double (&x)[PER]) {
  if constexpr (D >= 1) {
    lane_exchange<D, PER, false>(x);
    lane_steps<PER, D / 2>(x);
  }
}
template <int LANES, int PER, int K> __device__ __forceinline__ void lane_sort(double (&x)[PER]) {     // K lanes hold a sorted run afterwards
  if constexpr (K <= LANES) {
    lane_exchange<K - 1, PER, true>(x);
    lane_steps<PER, K / 4>(x);
    register_steps<PER, PER / 2>(x);
    lane_sort<LANES, PER, K * 2>(x);
  }
}
template <int CTRL, int ROWS> __device__ __forceinline__ uint64_t shifted_in(uint64_t v) {
  const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)v, CTRL, ROWS, 0xf, true);
  const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(v >> 32), CTRL, ROWS, 0xf, true);
  return ((uint64_t)hi << 32) | lo;
}
// inclusive prefix sum over the lanes of a row
template <int LANES> __device__ __forceinline__ uint64_t lanes_scan(uint64_t v) {
  v += shifted_in<0x111, 0xf>(v);
  v += shifted_in<0x112, 0xf>(v);
  v += shifted_in<0x114, 0xf>(v);
  v += shifted_in<0x118, 0xf>(v);
  if constexpr (LANES == 64) {
    v += shifted_in<0x142, 0xa>(v);                              // row_bcast:15 into rows 1 and 3
    v += shifted_in<0x143, 0xc>(v);                              // row_bcast:31 into rows 2 and 3
  }
  return v;
}

template <class E, int LANES, int PER>
__global__ void __launch_bounds__(256) sample_sorted_kernel(SampleP p) {
  __shared__ double table[32];
  fill_table(table);
  __syncthreads();
  const int t = threadIdx.x & (LANES - 1);
  const long at = (long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const long r = at < p.n ? at : p.n - 1;
  const char* z = static_cast<const char*>(p.z) + r * p.ldz * E::kBytes;
  const Settings set = settings_of(p, r);
  double x[PER];
  if constexpr (PER * E::kBytes >= 16) {
    if (t * PER + PER <= p.v) {
#pragma unroll
      for (int h = 0; h < PER / E::kVec; ++h) {
        float f[E::kVec];
        E::unpack(load16(z, ((long)t * PER + h * E::kVec) * E::kBytes), f);
#pragma unroll
        for (int i = 0; i < E::kVec; ++i) x[h * E::kVec + i] = sort_key(f[i], t * PER + h * E::kVec + i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) x[i] = t * PER + i < p.v ? sort_key(E::load(z, t * PER + i), t * PER + i) : 0.0;
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) x[i] = t * PER + i < p.v ? sort_key(E::load(z, t * PER + i), t * PER + i) : 0.0;
  }
  register_sort<PER, 2>(x);
  lane_sort<LANES, PER, 2>(x);

  // the largest, in every lane of the row
  const uint64_t own = (uint64_t)__double_as_longlong(x[0]);
  const uint64_t first = ((uint64_t)(unsigned)__shfl((int)(own >> 32), 0, LANES) << 32) | (unsigned)__shfl((int)(unsigned)own, 0, LANES);
  const bool some = first != 0;
  Weight w;
  w.zmax = (double)value_of((unsigned)(first >> 29));
  w.c = 1.4426950408889634 / set.t;
  w.shift = p.shift;
  w.table = table;
  const double reach = reach_of(set.min_p);
  uint64_t run[PER], sum = 0;
  unsigned strong = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const bool in = x[i] != 0.0 && (set.top_k <= 0 || t * PER + i < set.top_k);
    const unsigned b = sorted_bits(x[i]);
    sum += in ? w.of(b) : 0;
    run[i] = sum;
    if (in && is_strong(w, b, reach)) strong |= 1u << i;
  }
  const uint64_t before = lanes_scan<LANES>(sum) - sum;
  const uint64_t all = lanes_reduce<LANES, OpSum>(sum);
  const uint64_t border = set.top_p < 1.0 ? border_of(set.top_p, all) : ~0ull;
  uint64_t kept = 0;                                             // running sum of the last label that every filter keeps
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint64_t ahead = before + (i ? run[i - 1] : 0);
    if ((strong >> i & 1) && ahead <= border) kept = before + run[i];
  }
  kept = lanes_reduce<LANES, OpMax>(kept);
  const uint64_t want = position_of(set.u, kept);
  if (at >= p.n) return;
  if (!some || !(set.t > 0.0)) {                                 // nothing to draw; or the first alone
    if (t == 0) p.out[r] = some ? sorted_index(x[0]) : -1;
    return;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint64_t ahead = before + (i ? run[i - 1] : 0);
    if (ahead <= want && want < before + run[i]) p.out[r] = sorted_index(x[i]);
  }
}

// ---- longer rows: a workgroup each ----

struct Found { uint64_t key, upto; };     // the label's key; weight of the order up to it, itself included

template <int THREADS>
struct Shared {
  unsigned count[kBins];
  uint64_t mass[kBins];
  uint64_t list_key[kList], list_mass[kList];
  double table[32];
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

// The row: each(f) calls f(order bits, index) for the labels of this thread, four pieces of 16 bytes in flight.  It is read again in
// every pass: the first comes from memory, the others from the L2 it left the row in.
template <class E, int THREADS>
struct RowInMemory {
  const char* z;
  int v;
  template <class F> __device__ __forceinline__ void each(F f) const {
    const int pieces = v / E::kVec;
    for (int q = threadIdx.x; q < pieces; q += THREADS * 4) {
      u32x4 r[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) r[u] = load16(z, (long)min(q + u * THREADS, pieces - 1) * 16);
#pragma unroll 1
      for (int u = 0; u < 4; ++u) {
        const int at = q + u * THREADS;
        if (at >= pieces) break;
        float x[E::kVec];
        const u32x4 now = u == 0 ? r[0] : u == 1 ? r[1] : u == 2 ? r[2] : r[3];
        E::unpack(now, x);
#pragma unroll
        for (int i = 0; i < E::kVec; ++i) f(order_bits(x[i]), at * E::kVec + i);
      }
    }
    const int i = pieces * E::kVec + threadIdx.x;
    if (i < v) f(order_bits(E::load(z, i)), i);
  }
};

// A histogram of the labels with low <= key <= high: by equal steps of the value (step > 0) or of the key (2^bits).
struct Steps {
  uint64_t low, high;
  float top, step;
  int bits;
  __device__ __forceinline__ bool has(uint64_t k) const { return k >= low && k <= high; }
  __device__ __forceinline__ int bin(unsigned b, uint64_t k) const {
    return step > 0.f ? (int)fminf((top - value_of(b)) * step, (float)(kBins - 1)) : (int)((high - k) >> bits);
  }
};

// steps of the value over `span` below the largest; 0 (steps of the key) where there is no such span
__device__ __forceinline__ float step_of(float span) {
  const float step = span > 0.f && span < 1e30f ? (float)(kBins - 1) / span : 0.f;
  return step < 1e30f ? step : 0.f;
}

template <bool COUNT, int THREADS, class ROW>
__device__ __forceinline__ void histogram(const ROW& row, const Weight& w, const Steps& st, Shared<THREADS>& sh) {
  for (int i = threadIdx.x; i < kBins; i += THREADS) { sh.count[i] = 0; sh.mass[i] = 0; }
  __syncthreads();
  row.each([&](unsigned b, int i) {
    const uint64_t k = key_of(b, i);
    if (!st.has(k)) return;
    const uint64_t m = COUNT ? 1 : w.of(b);
    if (m == 0) return;                                          // no position can fall on it
    const int at = st.bin(b, k);
    atomicAdd(&sh.count[at], 1u);
    if (!COUNT) atomicAdd((unsigned long long*)&sh.mass[at], (unsigned long long)m);
  });
  __syncthreads();
}

// The label on which position `want` falls, by count (COUNT: the want-th of the order, from 0) or by weight (the first whose running sum
// is over `want`; labels of no weight are left out), among the labels of `st`, at most `members`.  `ready`: the histogram is that of `st`
// (and still is afterwards).
template <bool COUNT, int THREADS, class ROW>
__device__ Found find(const ROW& row, const Weight& w, Steps st, unsigned members, uint64_t want, bool& ready, Shared<THREADS>& sh) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  unsigned base_c = 0;
  uint64_t base_m = 0;
  int bin = -1;                                                  // -1: all of st
  for (int round = 0; members > (unsigned)kList && round < 10; ++round) {      // 64 bits of key, at least 10 a round
    if (bin >= 0) {                                              // the bin's own range of keys, in equal steps of the key
      uint64_t lo = ~0ull, hi = 0;
      row.each([&](unsigned b, int i) {
        const uint64_t k = key_of(b, i);
        if (!st.has(k) || st.bin(b, k) != bin) return;
        lo = k < lo ? k : lo;
        hi = k > hi ? k : hi;
      });
      st.low = block_all<THREADS, OpMin>(lo, sh);
      st.high = block_all<THREADS, OpMax>(hi, sh);
      st.step = 0.f;
    }
    if (!ready || bin >= 0) {
      ready = bin < 0;
      const uint64_t span = st.high - st.low;
      st.bits = 0;
      while ((span >> st.bits) >= (uint64_t)kBins) ++st.bits;
      histogram<COUNT, THREADS>(row, w, st, sh);
    }
    // the bin in which the running sum crosses `want`
    constexpr int PER = kBins / THREADS;
    unsigned c = 0;
    uint64_t m = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) { c += sh.count[tid * PER + i]; m += sh.mass[tid * PER + i]; }
    const uint64_t mi = lanes_scan<64>(m);
    const unsigned ci = (unsigned)lanes_scan<64>((uint64_t)c);
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
    bin = sh.bin;
    base_c = sh.base_c;
    base_m = sh.base_m;
    members = sh.in_bin;
  }
  __syncthreads();
  if (tid == 0) sh.listed = 0;
  __syncthreads();
  row.each([&](unsigned b, int i) {
    const uint64_t k = key_of(b, i);
    if (!st.has(k) || (bin >= 0 && st.bin(b, k) != bin)) return;
    const uint64_t m = COUNT ? 1 : w.of(b);
    if (m == 0) return;
    const unsigned at = atomicAdd(&sh.listed, 1u);
    if (at < (unsigned)kList) {
      sh.list_key[at] = k;
      sh.list_mass[at] = m;
    }
  });
  __syncthreads();
  const int n = (int)min(sh.listed, (unsigned)kList);
  for (int e = tid; e < n; e += THREADS) {
    const uint64_t k = sh.list_key[e];
    uint64_t before = COUNT ? base_c : base_m;
    for (int l = 0; l < n; ++l)
      if (sh.list_key[l] > k) before += sh.list_mass[l];
    const uint64_t upto = before + sh.list_mass[e];
    if (before <= want && want < upto) sh.found = Found{k, upto};
  }
  __syncthreads();
  return sh.found;
}

// The whole draw among the n labels of the list, of which the top_k count.
template <int THREADS>
__device__ __forceinline__ void draw_from_list(const Weight& w, const Settings& set, int n, int64_t* out, Shared<THREADS>& sh) {
  const int tid = threadIdx.x;
  static_assert(kList <= 2 * THREADS, "two labels per thread");
  uint64_t key[2], own[2], before[2];
  uint64_t sum = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int e = tid + h * THREADS;
    key[h] = e < n ? sh.list_key[e] : 0;
    unsigned rank = 0;
    if (e < n)
      for (int l = 0; l < n; ++l) rank += sh.list_key[l] > key[h];
    own[h] = e < n && rank < (unsigned)set.top_k ? sh.list_mass[e] : 0;
    if (own[h] == 0) key[h] = 0;
    sum += own[h];
  }
  const uint64_t all = block_all<THREADS, OpSum>(sum, sh);
  const uint64_t border = set.top_p < 1.0 ? border_of(set.top_p, all) : ~0ull;
  const double reach = reach_of(set.min_p);
  uint64_t kept = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    before[h] = 0;
    if (key[h] == 0) continue;
    for (int l = 0; l < n; ++l)
      if (sh.list_key[l] > key[h]) before[h] += sh.list_mass[l];
    if (before[h] <= border && is_strong(w, (unsigned)(key[h] >> 32), reach)) kept = max(kept, before[h] + own[h]);
  }
  kept = block_all<THREADS, OpMax>(kept, sh);
  const uint64_t want = position_of(set.u, kept);
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (key[h] && before[h] <= want && want < before[h] + own[h]) *out = (int64_t)(0xffffffffu - (unsigned)key[h]);
}

template <class E, int THREADS>
__global__ void __launch_bounds__(THREADS) sample_row_kernel(SampleP p) {
  __shared__ Shared<THREADS> sh;
  const long r = blockIdx.x;
  const RowInMemory<E, THREADS> row{static_cast<const char*>(p.z) + r * p.ldz * E::kBytes, p.v};
  const Settings set = settings_of(p, r);
  fill_table(sh.table);

  uint64_t best = 0;
  unsigned lowest = 0xffffffffu, some = 0;
  row.each([&](unsigned b, int i) {
    if (b == kNothing) return;
    const uint64_t k = key_of(b, i);
    best = k > best ? k : best;
    lowest = b < lowest ? b : lowest;
    ++some;
  });
  const uint64_t mine = best;
  best = block_all<THREADS, OpMax>(best, sh);
  if (best == 0 || !(set.t > 0.0) || set.top_k == 1) {           // nothing to draw; or the first alone
    if (threadIdx.x == 0) p.out[r] = best == 0 ? -1 : (int64_t)(0xffffffffu - (unsigned)best);
    return;
  }
  some = block_all<THREADS, OpSum>(some, sh);
  Weight w;
  w.zmax = (double)value_of((unsigned)(best >> 32));
  w.c = 1.4426950408889634 / set.t;
  w.shift = p.shift;
  w.table = sh.table;
  Steps st;
  st.low = key_of(kNothing + 1, 0x7fffffff);
  st.high = best;
  st.bits = 0;

  if (set.top_k > 0 && (unsigned)set.top_k < some && set.top_k <= kPrune) {
    // a label under the top_k-th largest of 256 groups' maxima has top_k better ones: it is out
    constexpr int kGroups = 256, kGroup = THREADS / kGroups;
    static_assert(kGroup == 1 || kGroup == 4, "a thread or a quad");
    uint64_t* maxima = sh.mass;
    uint64_t group = mine;
    if constexpr (kGroup == 4) {
      group = max(group, lane_step<0xB1>(group));
      group = max(group, lane_step<0x4E>(group));
    }
    if (threadIdx.x % kGroup == 0) maxima[threadIdx.x / kGroup] = group;
    if (threadIdx.x == 0) { sh.listed = 0; sh.found.key = 0; }
    __syncthreads();
    if (threadIdx.x < kGroups) {
      const uint64_t me = maxima[threadIdx.x];
      int better = 0;
#pragma unroll 8
      for (int l = 0; l < kGroups; ++l) better += maxima[l] > me;
      if (me && better == set.top_k - 1) sh.found.key = me;
    }
    __syncthreads();
    const uint64_t bound = max(sh.found.key, st.low);            // fewer groups with a label than top_k: no bound
    row.each([&](unsigned b, int i) {
      const uint64_t k = key_of(b, i);
      if (k < bound) return;
      const unsigned at = atomicAdd(&sh.listed, 1u);
      if (at < (unsigned)kList) {
        sh.list_key[at] = k;
        sh.list_mass[at] = w.of(b);
      }
    });
    __syncthreads();
    if (sh.listed <= (unsigned)kList) {
      draw_from_list<THREADS>(w, set, (int)sh.listed, p.out + r, sh);
      return;
    }
    __syncthreads();                                             // sh.listed has been read
  }
  lowest = block_all<THREADS, OpMin>(lowest, sh);
  const float top = (float)w.zmax;
  const float reach = top - fmaxf(value_of(lowest), -1e30f);
  st.top = top;
  if (set.top_k > 0 && (unsigned)set.top_k < some) {
    st.step = step_of(reach);
    bool ready = false;
    st.low = find<true, THREADS>(row, w, st, some, (uint64_t)(set.top_k - 1), ready, sh).key;
    some = (unsigned)set.top_k;
  }
  // weights more than 2^-52 below the largest are 0 as integers: the steps are spent above that
  st.step = step_of(fminf(reach, (float)(52.0 / w.c)));
  const uint64_t range = st.high - st.low;
  while ((range >> st.bits) >= (uint64_t)kBins) ++st.bits;
  const double weak = reach_of(set.min_p);
  histogram<false, THREADS>(row, w, st, sh);
  bool ready = true;
  uint64_t all = 0, strong = 0;
  for (int i = threadIdx.x; i < kBins; i += THREADS) all += sh.mass[i];
  all = block_all<THREADS, OpSum>(all, sh);
  uint64_t kept = all;
  if (weak < __builtin_inf()) {
    row.each([&](unsigned b, int i) {
      if (st.has(key_of(b, i)) && is_strong(w, b, weak)) strong += w.of(b);
    });
    kept = block_all<THREADS, OpSum>(strong, sh);
  }
  if (set.top_p < 1.0) {
    const uint64_t upto = find<false, THREADS>(row, w, st, some, border_of(set.top_p, all), ready, sh).upto;
    kept = upto < kept ? upto : kept;
  }
  const Found f = find<false, THREADS>(row, w, st, some, position_of(set.u, kept), ready, sh);
  if (threadIdx.x == 0) p.out[r] = (int64_t)(0xffffffffu - (unsigned)f.key);
}

// Up to 512 labels: the sorting network (16 lanes where 8 labels each are enough).  Above: a workgroup per row, of 1,024 threads for
// long rows and where there are too few rows to fill the card with smaller ones.
template <class E>
int launch_sample(const SampleP& p, hipStream_t s) {
  auto sorted = [&](auto lanes, auto per) {
    constexpr int L = decltype(lanes)::value, P = decltype(per)::value;
    hipLaunchKernelGGL((sample_sorted_kernel<E, L, P>), dim3((unsigned)((p.n + 256 / L - 1) / (256 / L))), dim3(256), 0, s, p);
  };
  using std::integral_constant;
#define OBJ_SORTED(L, P) sorted(integral_constant<int, L>{}, integral_constant<int, P>{})
  if (p.v <= 16) OBJ_SORTED(16, 1);
  else if (p.v <= 32) OBJ_SORTED(16, 2);
  else if (p.v <= 64) OBJ_SORTED(16, 4);
  else if (p.v <= 128) OBJ_SORTED(16, 8);
  else if (p.v <= 256) OBJ_SORTED(64, 4);
  else if (p.v <= 512) OBJ_SORTED(64, 8);
  else if (p.v <= 16384 && p.n > 512) hipLaunchKernelGGL((sample_row_kernel<E, 256>), dim3((unsigned)p.n), dim3(256), 0, s, p);
  else hipLaunchKernelGGL((sample_row_kernel<E, 1024>), dim3((unsigned)p.n), dim3(1024), 0, s, p);
#undef OBJ_SORTED
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
  p.shift = 62 - log_v < 51 ? 62 - log_v : 51;
  p.out = a->labels;
  hipStream_t s = (hipStream_t)stream;
  return a->type == OBJNERF_TYPE_F32 ? launch_sample<ElemF32>(p, s)
         : a->type == OBJNERF_TYPE_BF16 ? launch_sample<ElemBf16>(p, s) : launch_sample<ElemF16>(p, s);
}
