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
// and need no order, so sums formed by atomics give the same bits in every run.  A weight is off by half of 2^-shift at most, and weights
// under that become 0, so the sum over a row of a strong label and a flat weak rest can lack v 2^-(shift + 1), about v^2 2^-63 of the
// largest weight: 2^-29 at 131,072 labels, 2^-25 at 2^19.  That is half of what a random number of 24 bits resolves, and kMaxLabels: at
// 2^22 labels it would be 2^-19, at 2^30 an eighth of the weight.
//
// Rows of up to 512 labels are sorted in the registers of 16 or 64 lanes, and every question -- which are the top_k, where does the
// running sum pass top_p, where u -- is then a prefix sum away.  Longer rows are not sorted: with a small top_k the candidates are
// picked out by a bound (the top_k-th largest of the threads' own maxima), else each question is answered by a histogram in equal
// steps of the logit and by looking into the one bin in which the running sum crosses.
//
// Measured: 307,200 x 64 fp32 58 us (79 MB: 1.4 TB/s), bound by the vector units (about 550 instructions per four rows: 130 of them the
// network, 100 the weights); 2,048 x 32,768 bf16 with top_k 50 53 us = 2.5 TB/s, bound by the chain of passes of a row; 257 x 30,011
// fp16 39 us and one row of 131,072 32 us in four kernels, bound by latencies.
//
// NaN counts as -inf; a row of nothing but -inf draws -1.
#include "host_api.h"
#include "label_ops.h"
#include <type_traits>

namespace objnerf {
namespace {

constexpr int kList = 512, kPrune = 128;
constexpr int kMaxLabels = 1 << 19;       // of a row: see the error of the sums above
constexpr int64_t kOpen = -2;             // between two kernels of a call: this row is still to be drawn

struct SampleP {
  long n;
  int v;
  const void* z; long ldz;
  const float* u; long ldu;
  const float* t; double c0;              // per row, or one number where the pointer is null: log2(e) / T, 0 for the first of the order
  const int32_t* top_k; int top_k0;
  const float* top_p; double top_p0;
  const float* min_p; double reach0;      // -log2(min_p)
  int shift;
  int64_t* out;
};
struct Settings {
  double c;                               // log2(e) / T; 0: the first of the order
  double reach;                           // how far a label may lie below the largest, in (logit c): -log2(min_p); the strongest always stays
  double top_p;
  int top_k;                              // <= 0: off
  float u;
};
__host__ __device__ __forceinline__ double scale_of(double t) {    // 0: the first of the order
  return t > 0.0 ? fmin(fmax(1.4426950408889634 / t, 1e-300), 1e300) : 0.0;
}
__host__ __device__ __forceinline__ double reach_of(double min_p) { return min_p > 0.0 ? fmax(-log2(min_p), 0.0) : __builtin_inf(); }
__device__ __forceinline__ Settings settings_of(const SampleP& p, long r) {
  Settings s;
  s.c = p.t ? scale_of((double)p.t[r]) : p.c0;
  s.top_k = p.top_k ? p.top_k[r] : p.top_k0;
  s.top_p = p.top_p ? (double)p.top_p[r] : p.top_p0;
  s.reach = p.min_p ? reach_of((double)p.min_p[r]) : p.reach0;
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
  __device__ __forceinline__ uint64_t of(float logit) const {
    const double z = (double)logit;
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
__constant__ const double kTable[32] = {
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
    1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002,
};
__device__ __forceinline__ void fill_table(double* table) {
  if (threadIdx.x < 32) table[threadIdx.x] = kTable[threadIdx.x];
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
__device__ __forceinline__ bool is_strong(const Weight& w, float logit, double reach) { return !((w.zmax - (double)logit) * w.c > reach); }

// ---- rows of up to LANES x PER labels: a sorting network in registers ----
// On the order bits alone: weights of equal logits are equal, so the running sums do not ask which of them comes first.  Position
// t PER + i of the order is register i of lane t.

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
__device__ __forceinline__ void order_pair(unsigned& a, unsigned& b) {
  const unsigned hi = max(a, b), lo = min(a, b);
  a = hi;
  b = lo;
}
// one step across lanes: the lower lane keeps the larger -- the median of both and all ones, or 0.  MIRROR: the partner's registers in
// reverse order
template <int MASK, int PER, bool MIRROR> __device__ __forceinline__ void lane_exchange(unsigned (&x)[PER]) {
  constexpr int top = MASK >= 32 ? 32 : MASK >= 16 ? 16 : MASK >= 8 ? 8 : MASK >= 4 ? 4 : MASK >= 2 ? 2 : 1;
  const unsigned third = threadIdx.x & top ? 0u : ~0u;
  unsigned y[PER];
#pragma unroll
  for (int r = 0; r < PER; ++r) y[r] = lane_xor<MASK>(x[r]);
#pragma unroll
  for (int r = 0; r < PER; ++r) {
    const unsigned o = y[MIRROR ? PER - 1 - r : r];
    x[r] = max(min(x[r], o), min(max(x[r], o), third));
  }
}
// merges of register pairs at distances D, D / 2, .. 1
template <int PER, int D> __device__ __forceinline__ void register_steps(unsigned (&x)[PER]) {
  if constexpr (D >= 1) {
#pragma unroll
    for (int r = 0; r < PER; ++r)
      if (!(r & D)) order_pair(x[r], x[r | D]);
    register_steps<PER, D / 2>(x);
  }
}
template <int PER, int K> __device__ __forceinline__ void register_sort(unsigned (&x)[PER]) {
  if constexpr (K <= PER) {
#pragma unroll
    for (int r = 0; r < PER; ++r)
      if (!(r & (K / 2))) order_pair(x[r], x[r ^ (K - 1)]);
    register_steps<PER, K / 4>(x);
    register_sort<PER, K * 2>(x);
  }
}
template <int PER, int D> __device__ __forceinline__ void lane_steps(unsigned (&x)[PER]) {
  if constexpr (D >= 1) {
    lane_exchange<D, PER, false>(x);
    lane_steps<PER, D / 2>(x);
  }
}
template <int LANES, int PER, int K> __device__ __forceinline__ void lane_sort(unsigned (&x)[PER]) {     // K lanes hold a sorted run afterwards
  if constexpr (K <= LANES) {
    lane_exchange<K - 1, PER, true>(x);
    lane_steps<PER, K / 4>(x);
    register_steps<PER, PER / 2>(x);
    lane_sort<LANES, PER, K * 2>(x);
  }
}
template <int CTRL, int ROWS> __device__ __forceinline__ uint64_t shifted_in(uint64_t v) {
  if constexpr (ROWS == 0xf) {                                   // lanes without a source get 0
    return ((uint64_t)dpp_u32<CTRL>((unsigned)(v >> 32)) << 32) | dpp_u32<CTRL>((unsigned)v);
  } else {
    const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)v, CTRL, ROWS, 0xf, true);
    const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(v >> 32), CTRL, ROWS, 0xf, true);
    return ((uint64_t)hi << 32) | lo;
  }
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
  const long at = workgroup() * (256 / LANES) + threadIdx.x / LANES;
  const long r = at < p.n ? at : p.n - 1;
  const char* z = static_cast<const char*>(p.z) + r * p.ldz * E::kBytes;
  const Settings set = settings_of(p, r);
  unsigned own[PER], x[PER];                                     // as they lie in the row; in order
  if (PER * E::kBytes >= 16 && t * PER + PER <= p.v) {
#pragma unroll
    for (int h = 0; h < PER / E::kVec; ++h) {
      float f[E::kVec];
      E::unpack(load16(z, ((long)t * PER + h * E::kVec) * E::kBytes), f);
#pragma unroll
      for (int i = 0; i < E::kVec; ++i) own[h * E::kVec + i] = order_bits(f[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) own[i] = t * PER + i < p.v ? order_bits(E::load(z, t * PER + i)) : kNothing;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) x[i] = own[i];
  register_sort<PER, 2>(x);
  lane_sort<LANES, PER, 2>(x);

  const unsigned top = lanes_reduce<LANES, OpMax>(x[0]);
  const Weight w{(double)value_of(top), set.c, p.shift, table};
  uint64_t run[PER], sum = 0;
  unsigned strong = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const bool in = x[i] != kNothing && (set.top_k <= 0 || t * PER + i < set.top_k);
    const float logit = value_of(x[i]);
    sum += in ? w.of(logit) : 0;
    run[i] = sum;
    if (in && is_strong(w, logit, set.reach)) strong |= 1u << i;
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
  unsigned hit = 0, place = 0;                                   // the logit on which `want` falls, and its place in the order
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint64_t ahead = before + (i ? run[i - 1] : 0);
    if (ahead <= want && want < before + run[i]) { hit = x[i]; place = (unsigned)(t * PER + i); }
  }
  hit = lanes_reduce<LANES, OpMax>(hit);
  place = lanes_reduce<LANES, OpMax>(place);
  if (set.c == 0.0) { hit = top; place = 0; }                    // the first alone
  // of the labels with this logit, the one with as many in front of it, by index, as `place` has in the order
  unsigned better = 0, equal = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    better += x[i] > hit;
    equal += own[i] == hit;
  }
  const unsigned nth = place - lanes_reduce<LANES, OpSum>(better);
  unsigned seen = (unsigned)lanes_scan<LANES>((uint64_t)equal) - equal;
  if (at >= p.n) return;
  if (top == kNothing) {
    if (t == 0) p.out[r] = -1;
    return;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (own[i] == hit) {
      if (seen == nth) p.out[r] = t * PER + i;
      ++seen;
    }
}

// ---- longer rows: a workgroup each ----

struct Found { uint64_t key, upto; };     // the label's key; weight of the order up to it, itself included
struct __align__(16) Entry { uint64_t key, mass; };

template <int THREADS>
struct Shared {
  static constexpr int kBins = 8 * THREADS;
  unsigned count[kBins];
  uint64_t mass[kBins];
  Entry list[kList];
  double table[32];
  uint64_t red[THREADS / 64];
  uint64_t part_m[THREADS / 64];
  unsigned part_c[THREADS / 64];
  unsigned listed, bound;
  int bin;
  unsigned base_c, in_bin;
  uint64_t base_m;
  Found found;
};

template <int THREADS, class OP, class T, class SH>
__device__ __forceinline__ T block_all(T v, SH& sh) {
  v = lanes_reduce<64, OP>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x >> 6] = (uint64_t)v;
  __syncthreads();
  T r = (T)sh.red[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) r = OP::f(r, (T)sh.red[w]);
  return r;
}

// The row, or a part of it: each(f) calls f(logit, index) for the labels of this thread, four pieces of 16 bytes in flight.  It is read
// again in every pass: the first comes from memory, the others from the caches it left the row in.
template <class E, int THREADS>
struct RowInMemory {
  const char* z;
  int v;
  int from = 0, to = -1;                  // in pieces; -1: to the row's end
  template <class F> __device__ __forceinline__ void each(F f) const {
    const int pieces = v / E::kVec, end = to < 0 ? pieces : to;
    for (int q = from + threadIdx.x; q < end; q += THREADS * 4) {
      u32x4 r[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) r[u] = load16(z, (long)min(q + u * THREADS, end - 1) * 16);
#pragma unroll 1
      for (int u = 0; u < 4; ++u) {
        const int at = q + u * THREADS;
        if (at >= end) break;
        float x[E::kVec];
        E::unpack(r[0], x);
        r[0] = r[1];
        r[1] = r[2];
        r[2] = r[3];
#pragma unroll
        for (int i = 0; i < E::kVec; ++i) f(x[i], at * E::kVec + i);
      }
    }
    const int i = pieces * E::kVec + threadIdx.x;
    if (to < 0 && i < v) f(E::load(z, i), i);
  }
};

// Steps of a histogram over the labels with low <= key <= high: equal steps of the value (step > 0) or of the key (2^bits).
struct Steps {
  uint64_t low, high;
  float top, step;
  int bits, last;                         // last: the last bin's number
  __device__ __forceinline__ bool has(unsigned b, int i) const {
    const unsigned lo = (unsigned)(low >> 32);
    if (b - lo > (unsigned)(high >> 32) - lo) return false;      // 32 bits decide all but the ends
    const uint64_t k = key_of(b, i);
    return k >= low && k <= high;
  }
  __device__ __forceinline__ int bin(float x, uint64_t k) const {
    return step > 0.f ? (int)fminf((top - x) * step, (float)last) : (int)((high - k) >> bits);
  }
  __device__ __forceinline__ void fit_bits() {
    const uint64_t span = high - low;
    bits = 0;
    while ((span >> bits) > (uint64_t)last) ++bits;
  }
  // steps of the value over `span` below the largest; 0 (steps of the key) where there is no such span
  __device__ __forceinline__ void fit_step(float span) {
    step = span > 0.f && span < 1e30f ? (float)last / span : 0.f;
    if (!(step < 1e30f)) step = 0.f;
  }
};

// also returns this thread's share of the weight of the strong labels
template <bool COUNT, int THREADS, class ROW>
__device__ __forceinline__ uint64_t histogram(const ROW& row, const Weight& w, const Steps& st, double reach, Shared<THREADS>& sh) {
  for (int i = threadIdx.x; i < Shared<THREADS>::kBins; i += THREADS) { sh.count[i] = 0; sh.mass[i] = 0; }
  __syncthreads();
  uint64_t strong = 0;
  row.each([&](float x, int i) {
    const unsigned b = order_bits(x);
    if (!st.has(b, i)) return;
    const uint64_t m = COUNT ? 1 : w.of(x);
    if (m == 0) return;                                          // no position can fall on it
    const int at = st.bin(x, key_of(b, i));
    atomicAdd(&sh.count[at], 1u);
    if (!COUNT) {
      atomicAdd((unsigned long long*)&sh.mass[at], (unsigned long long)m);
      if (is_strong(w, x, reach)) strong += m;
    }
  });
  __syncthreads();
  return strong;
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
      row.each([&](float x, int i) {
        const unsigned b = order_bits(x);
        const uint64_t k = key_of(b, i);
        if (!st.has(b, i) || st.bin(x, k) != bin) return;
        lo = k < lo ? k : lo;
        hi = k > hi ? k : hi;
      });
      st.low = block_all<THREADS, OpMin>(lo, sh);
      st.high = block_all<THREADS, OpMax>(hi, sh);
      st.step = 0.f;
    }
    if (!ready || bin >= 0) {
      ready = bin < 0;
      st.fit_bits();
      histogram<COUNT, THREADS>(row, w, st, 0.0, sh);
    }
    // the bin in which the running sum crosses `want`
    constexpr int PER = Shared<THREADS>::kBins / THREADS;
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
  row.each([&](float x, int i) {
    const unsigned b = order_bits(x);
    const uint64_t k = key_of(b, i);
    if (!st.has(b, i) || (bin >= 0 && st.bin(x, k) != bin)) return;
    const uint64_t m = COUNT ? 1 : w.of(x);
    if (m == 0) return;
    const unsigned at = atomicAdd(&sh.listed, 1u);
    if (at < (unsigned)kList) sh.list[at] = Entry{k, m};
  });
  __syncthreads();
  const int n = (int)min(sh.listed, (unsigned)kList);
  for (int e = tid; e < n; e += THREADS) {
    const Entry me = sh.list[e];
    uint64_t before = COUNT ? base_c : base_m;
#pragma unroll 8
    for (int l = 0; l < n; ++l) {
      const Entry o = sh.list[l];
      before += o.key > me.key ? o.mass : 0;
    }
    if (before <= want && want < before + me.mass) sh.found = Found{me.key, before + me.mass};
  }
  __syncthreads();
  return sh.found;
}

// weights of the list's labels (here and not where they are found: every lane has one to work on)
template <int THREADS, class SH> __device__ __forceinline__ void weigh_list(const Weight& w, int n, SH& sh) {
  for (int e = threadIdx.x; e < n; e += THREADS) sh.list[e].mass = w.of(value_of((unsigned)(sh.list[e].key >> 32)));
  __syncthreads();
}

// The whole draw among the n labels of the list, of which the top_k count.
template <int THREADS, class SH>
__device__ __forceinline__ void draw_from_list(const Weight& w, const Settings& set, int n, int64_t* out, SH& sh) {
  const int tid = threadIdx.x;
  constexpr int H = kList / THREADS > 0 ? kList / THREADS : 1;     // labels per thread
  uint64_t key[H], own[H], before[H];
  uint64_t sum = 0;
#pragma unroll
  for (int h = 0; h < H; ++h) {
    const int e = tid + h * THREADS;
    key[h] = e < n ? sh.list[e].key : 0;
    unsigned rank = 0;
    before[h] = 0;
    if (e < n)
#pragma unroll 8
      for (int l = 0; l < n; ++l) {
        const Entry o = sh.list[l];
        const bool better = o.key > key[h];
        rank += better;
        before[h] += better ? o.mass : 0;
      }
    own[h] = e < n && rank < (unsigned)set.top_k ? sh.list[e].mass : 0;
    if (own[h] == 0) key[h] = 0;
    sum += own[h];
  }
  const uint64_t all = block_all<THREADS, OpSum>(sum, sh);
  const uint64_t border = set.top_p < 1.0 ? border_of(set.top_p, all) : ~0ull;
  uint64_t kept = 0;
#pragma unroll
  for (int h = 0; h < H; ++h)
    if (key[h] && before[h] <= border && is_strong(w, value_of((unsigned)(key[h] >> 32)), set.reach)) kept = max(kept, before[h] + own[h]);
  kept = block_all<THREADS, OpMax>(kept, sh);
  const uint64_t want = position_of(set.u, kept);
#pragma unroll
  for (int h = 0; h < H; ++h)
    if (key[h] && before[h] <= want && want < before[h] + own[h]) *out = (int64_t)(0xffffffffu - (unsigned)key[h]);
}

__device__ __forceinline__ Weight weight_of(const SampleP& p, const Settings& set, unsigned top, const double* table) {
  return Weight{(double)value_of(top), set.c, p.shift, table};
}
// All labels of a row whose largest has order bits `top`, in steps down to where a weight is 0 as an integer, or to the least label that
// counts as one (-1e30: what lies lower masks) where that is known.
__device__ __forceinline__ float span_of(const Weight& w) { return (float)((w.shift + 1) / w.c); }
__device__ __forceinline__ float least_of(float least, float x) { return x > -1e30f ? fminf(least, x) : least; }
template <int THREADS> __device__ __forceinline__ Steps all_steps(const Weight& w, unsigned top, float least) {
  Steps st;
  st.last = Shared<THREADS>::kBins - 1;
  st.low = key_of(kNothing + 1, 0x7fffffff);
  st.high = key_of(top, 0);
  st.top = (float)w.zmax;
  st.fit_step(fminf(span_of(w), st.top - least));
  st.fit_bits();
  return st;
}
__device__ __forceinline__ bool is_single(const Settings& set) { return set.c == 0.0 || set.top_k == 1; }

// What the histogram says of a row: with a top_k that cuts, the labels of bins 0 .. last_k are the candidates; else the border of
// top_p lies in bin_p and u's position in one of bins low_u .. high_u.  Afterwards sh.mass holds the weight in front of each bin, and
// sh.list is free.
struct Places {
  uint64_t all, strong;
  int last_k, bin_p, low_u, high_u;
};
template <int THREADS>
__device__ Places places_of(const uint64_t* mass, const unsigned* counts, uint64_t strong, const Settings& set, Shared<THREADS>& sh) {
  constexpr int PER = Shared<THREADS>::kBins / THREADS;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint64_t m[PER], sum = 0;
  unsigned c[PER], count = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    m[i] = mass[tid * PER + i];
    c[i] = counts[tid * PER + i];
    sum += m[i];
    count += c[i];
  }
  const uint64_t mi = lanes_scan<64>(sum);
  const unsigned ci = (unsigned)lanes_scan<64>((uint64_t)count);
  if (lane == 63) { sh.part_m[wave] = mi; sh.part_c[wave] = ci; }
  int* const found = reinterpret_cast<int*>(&sh.list[0]);        // last_k, bin_p, low_u, high_u
  uint64_t* const border_bin = &sh.list[1].key;                  // weight in front of bin_p, and with it
  if (tid == 0) found[0] = -1;
  __syncthreads();                                               // (and mass / counts have been read, where they are sh's)
  uint64_t before = mi - sum, all = 0;
  unsigned before_c = ci - count;
  for (int x = 0; x < THREADS / 64; ++x) {
    if (x < wave) { before += sh.part_m[x]; before_c += sh.part_c[x]; }
    all += sh.part_m[x];
  }
  Places pl;
  pl.all = all;
  pl.strong = strong;
  const bool cut = set.top_p < 1.0;
  const uint64_t border = cut ? border_of(set.top_p, all) : all - 1;
  uint64_t mb = before;
  unsigned cb = before_c;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (set.top_k > 0 && cb < (unsigned)set.top_k && (unsigned)set.top_k <= cb + c[i]) found[0] = tid * PER + i;
    if (mb <= border && border < mb + m[i]) { found[1] = tid * PER + i; border_bin[0] = mb; border_bin[1] = mb + m[i]; }
    sh.mass[tid * PER + i] = mb;
    mb += m[i];
    cb += c[i];
  }
  __syncthreads();
  pl.last_k = found[0];
  pl.bin_p = cut ? found[1] : -1;
  const uint64_t least = cut ? border_bin[0] + 1 : all, most = cut ? border_bin[1] : all;
  const uint64_t low = position_of(set.u, min(least, pl.strong)), high = position_of(set.u, min(most, pl.strong));
  mb = before;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (mb <= low && low < mb + m[i]) found[2] = tid * PER + i;
    if (mb <= high && high < mb + m[i]) found[3] = tid * PER + i;
    mb += m[i];
  }
  __syncthreads();
  pl.low_u = found[2];
  pl.high_u = found[3];
  __syncthreads();
  return pl;
}

// The draw from the list of all labels of the bins that `pl` names, n <= kList of them.  In front of a label stand the better ones of
// the list, and what lies in front of its bin less the listed bins there.
template <int THREADS>
__device__ __forceinline__ void finish_from_list(const Settings& set, const Steps& st, const Places& pl, int n, int64_t* out, Shared<THREADS>& sh) {
  const int tid = threadIdx.x;
  constexpr int H = kList / THREADS > 0 ? kList / THREADS : 1;
  Entry me[H];
  uint64_t ahead[H];
  int bin[H];
#pragma unroll
  for (int h = 0; h < H; ++h) {
    const int e = tid + h * THREADS;
    bin[h] = -1;
    ahead[h] = 0;
    me[h] = Entry{0, 0};
    if (e >= n) continue;
    me[h] = sh.list[e];
    const int at = st.bin(value_of((unsigned)(me[h].key >> 32)), me[h].key);
    bin[h] = at;
    ahead[h] = sh.mass[at];
    if (at > pl.low_u) ahead[h] -= sh.mass[min(at, pl.high_u + 1)] - sh.mass[pl.low_u];
    if (pl.bin_p >= 0 && pl.bin_p < at && (pl.bin_p < pl.low_u || pl.bin_p > pl.high_u)) ahead[h] -= sh.mass[pl.bin_p + 1] - sh.mass[pl.bin_p];
#pragma unroll 8
    for (int l = 0; l < n; ++l) {
      const Entry o = sh.list[l];
      ahead[h] += o.key > me[h].key ? o.mass : 0;
    }
  }
  uint64_t kept = pl.strong;
  if (pl.bin_p >= 0) {
    const uint64_t border = border_of(set.top_p, pl.all);
#pragma unroll
    for (int h = 0; h < H; ++h)
      if (bin[h] == pl.bin_p && ahead[h] <= border && border < ahead[h] + me[h].mass) sh.base_m = ahead[h] + me[h].mass;
    __syncthreads();
    kept = min(kept, sh.base_m);
  }
  const uint64_t want = position_of(set.u, kept);
#pragma unroll
  for (int h = 0; h < H; ++h)
    if (bin[h] >= 0 && ahead[h] <= want && want < ahead[h] + me[h].mass) *out = (int64_t)(0xffffffffu - (unsigned)me[h].key);
}

// Rows of which a few labels at most are kept (top_k <= kPrune).  A label under the top_k-th largest of 256 groups' maxima has top_k better
// ones: it is out, and about top_k labels are left.  False where more are left than the list takes (equal logits in masses).
template <int THREADS, class ROW, class SH>
__device__ __forceinline__ bool draw_top(const ROW& row, const Weight& w, const Settings& set, unsigned mine, unsigned* maxima, int64_t* out, SH& sh) {
  constexpr int kGroups = 256, kGroup = THREADS / kGroups;
  static_assert(kGroup == 1 || kGroup == 2 || kGroup == 4, "a thread, a pair or a quad");
  const int tid = threadIdx.x;
  unsigned group = mine;
  if constexpr (kGroup >= 2) group = max(group, lane_step<0xB1>(group));
  if constexpr (kGroup == 4) group = max(group, lane_step<0x4E>(group));
  if (tid % kGroup == 0) maxima[tid / kGroup] = group;
  if (tid == 0) { sh.listed = 0; sh.bound = kNothing; }
  __syncthreads();
  if (tid < kGroups) {
    const unsigned me = maxima[tid];
    int better = 0, equal = 0;
#pragma unroll 4
    for (int l = 0; l < kGroups / 4; ++l) {
      const u32x4 o = reinterpret_cast<const u32x4*>(maxima)[l];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        better += o[i] > me;
        equal += o[i] == me;
      }
    }
    if (better < set.top_k && set.top_k <= better + equal) sh.bound = me;        // (equal ones write the same)
  }
  __syncthreads();
  const float bound = value_of(sh.bound);                        // -inf: fewer groups with a label than top_k
  row.each([&](float x, int i) {
    if (!(x >= bound) || x == -__builtin_inff()) return;
    const unsigned at = atomicAdd(&sh.listed, 1u);
    if (at < (unsigned)kList) sh.list[at] = Entry{key_of(order_bits(x), i), 0};
  });
  __syncthreads();
  const unsigned n = sh.listed;
  __syncthreads();                                               // everybody has read it
  if (n > (unsigned)kList) return false;
  weigh_list<THREADS>(w, (int)n, sh);
  draw_from_list<THREADS>(w, set, (int)n, out, sh);
  return true;
}

template <class E, int THREADS>
__device__ void draw_row(const SampleP& p, long r, bool rest, Shared<THREADS>& sh) {
  const RowInMemory<E, THREADS> row{static_cast<const char*>(p.z) + r * p.ldz * E::kBytes, p.v};
  const Settings set = settings_of(p, r);
  fill_table(sh.table);

  float most = -__builtin_inff();
  row.each([&](float x, int) { most = fmaxf(most, x); });
  const unsigned mine = order_bits(most), top = block_all<THREADS, OpMax>(mine, sh);
  if (top == kNothing) {
    if (threadIdx.x == 0) p.out[r] = -1;
    return;
  }
  if (is_single(set)) {
    unsigned at = 0xffffffffu;
    row.each([&](float x, int i) {
      if (order_bits(x) == top) at = min(at, (unsigned)i);
    });
    at = block_all<THREADS, OpMin>(at, sh);
    if (threadIdx.x == 0) p.out[r] = at;
    return;
  }
  const Weight w = weight_of(p, set, top, sh.table);
  Steps st = all_steps<THREADS>(w, top, -__builtin_inff());
  unsigned members = (unsigned)p.v;

  if (set.top_k > 0 && set.top_k < p.v) {
    if (set.top_k <= kPrune && !rest && draw_top<THREADS>(row, w, set, mine, sh.count, p.out + r, sh)) return;
    unsigned some = 0;
    float least = (float)w.zmax;
    row.each([&](float x, int) {
      if (!(x > -__builtin_inff())) return;
      ++some;
      least = fminf(least, x);
    });
    some = block_all<THREADS, OpSum>(some, sh);
    least = value_of(block_all<THREADS, OpMin>(order_bits(least), sh));
    members = some;
    if ((unsigned)set.top_k < some) {
      Steps by = st;
      by.fit_step((float)w.zmax - fmaxf(least, -1e30f));
      bool ready = false;
      st.low = find<true, THREADS>(row, w, by, some, (uint64_t)(set.top_k - 1), ready, sh).key;
      st.fit_bits();
      members = (unsigned)set.top_k;
    }
  }
  if (span_of(w) > 64.f) {                                       // a high temperature: steps of the labels' own range
    float least = (float)w.zmax;
    row.each([&](float x, int) { least = least_of(least, x); });
    const uint64_t low = st.low;
    st = all_steps<THREADS>(w, top, value_of(block_all<THREADS, OpMin>(order_bits(least), sh)));
    st.low = low;
    st.fit_bits();
  }
  const uint64_t strong = block_all<THREADS, OpSum>(histogram<false, THREADS>(row, w, st, set.reach, sh), sh);
  Places pl = places_of<THREADS>(sh.mass, sh.count, strong, set, sh);
  if (threadIdx.x == 0) sh.listed = 0;
  __syncthreads();
  row.each([&](float x, int i) {
    const unsigned b = order_bits(x);
    if (!st.has(b, i)) return;
    const uint64_t k = key_of(b, i);
    const int bin = st.bin(x, k);
    if ((bin < pl.low_u || bin > pl.high_u) && bin != pl.bin_p) return;
    const unsigned at = atomicAdd(&sh.listed, 1u);
    if (at < (unsigned)kList) sh.list[at] = Entry{k, 0};
  });
  __syncthreads();
  if (sh.listed <= (unsigned)kList) {
    weigh_list<THREADS>(w, (int)sh.listed, sh);
    finish_from_list<THREADS>(set, st, pl, (int)sh.listed, p.out + r, sh);
    return;
  }
  __syncthreads();
  bool ready = false;
  uint64_t kept = pl.strong;
  if (set.top_p < 1.0) kept = min(kept, find<false, THREADS>(row, w, st, members, border_of(set.top_p, pl.all), ready, sh).upto);
  const Found f = find<false, THREADS>(row, w, st, members, position_of(set.u, kept), ready, sh);
  if (threadIdx.x == 0) p.out[r] = (int64_t)(0xffffffffu - (unsigned)f.key);
}

template <class E, int THREADS>
__global__ void __launch_bounds__(THREADS, 4) sample_row_kernel(SampleP p, bool rest) {
  __shared__ Shared<THREADS> sh;
  const long r = workgroup();
  if (r >= p.n || (rest && p.out[r] != kOpen)) return;           // sample_top_kernel has drawn it
  draw_row<E, THREADS>(p, r, rest, sh);
}

// Such rows in a kernel of their own: two light passes and a list, many rows at a time on a CU.  Rows of other settings, and rows with
// more left than the list takes, are marked for sample_row_kernel.
template <class E>
__global__ void __launch_bounds__(256, 6) sample_top_kernel(SampleP p) {
  __shared__ struct {
    __align__(16) unsigned maxima[256];
    Entry list[kList];
    double table[32];
    uint64_t red[4];
    unsigned listed, bound;
  } sh;
  const long r = workgroup();
  if (r >= p.n) return;
  Settings set = settings_of(p, r);
  if (is_single(set)) set.top_k = 1;
  if (set.top_k < 1 || set.top_k > kPrune) {
    if (threadIdx.x == 0) p.out[r] = kOpen;
    return;
  }
  const RowInMemory<E, 256> row{static_cast<const char*>(p.z) + r * p.ldz * E::kBytes, p.v};
  fill_table(sh.table);
  float most = -__builtin_inff();
  row.each([&](float x, int) { most = fmaxf(most, x); });
  const unsigned mine = order_bits(most), top = block_all<256, OpMax>(mine, sh);
  if (top == kNothing) {
    if (threadIdx.x == 0) p.out[r] = -1;
    return;
  }
  const Weight w = weight_of(p, set, top, sh.table);
  if (!draw_top<256>(row, w, set, mine, sh.maxima, p.out + r, sh) && threadIdx.x == 0) p.out[r] = kOpen;
}

// ---- few long rows: a row's passes spread over several workgroups, one kernel per pass ----
// 1: maxima of the parts.  2: the histogram of weights relative to the largest (integer atomics: the same bits in any order), and the
// sum of the strong ones.  3: from the histogram, which bins the answers lie in; their labels into a list.  4: one workgroup per row
// looks up the answers in the list.  Where the list overflows (equal logits in masses, a temperature of extremes) it draws the row
// by itself.
constexpr int kSplitThreads = 512, kSplitList = 4096, kSplitBins = Shared<kSplitThreads>::kBins;
struct SplitRow {
  uint64_t mass[kSplitBins];
  uint64_t strong;
  uint64_t list[kSplitList];
  unsigned count[kSplitBins];
  unsigned listed, first;                 // first: the lowest index of the largest logit, where one label alone is kept
};
struct SplitP {
  SplitRow* rows;
  unsigned* top;                          // (n, parts): order bits of the parts' largest, and the least
  float* least;
  int parts, per;                         // pieces of 16 bytes per part
};
template <class E> __device__ __forceinline__ RowInMemory<E, kSplitThreads> part_of(const SampleP& p, const SplitP& sp, long r) {
  const int part = blockIdx.x, pieces = p.v / E::kVec;
  RowInMemory<E, kSplitThreads> row{static_cast<const char*>(p.z) + r * p.ldz * E::kBytes, p.v};
  row.from = min(part * sp.per, pieces);
  row.to = part == sp.parts - 1 ? -1 : min((part + 1) * sp.per, pieces);
  return row;
}
__device__ __forceinline__ unsigned top_of(const SplitP& sp, long r) {       // by every wave for itself
  unsigned top = 0;
  for (int i = threadIdx.x & 63; i < sp.parts; i += 64) top = max(top, sp.top[r * sp.parts + i]);
  return lanes_reduce<64, OpMax>(top);
}
__device__ __forceinline__ float least_label(const SplitP& sp, long r) {
  float least = __builtin_inff();
  for (int i = threadIdx.x & 63; i < sp.parts; i += 64) least = fminf(least, sp.least[r * sp.parts + i]);
  return -lanes_reduce<64, OpMax>(-least);
}
// labels of a list that lie in one bin of `st`
struct RowInList {
  const uint64_t* keys;
  int n, bin;
  Steps st;
  template <class F> __device__ __forceinline__ void each(F f) const {
    for (int e = threadIdx.x; e < n; e += kSplitThreads) {
      const uint64_t k = keys[e];
      const float x = value_of((unsigned)(k >> 32));
      if (st.bin(x, k) == bin) f(x, (int)(0xffffffffu - (unsigned)k));
    }
  }
};

template <class E>
__global__ void __launch_bounds__(kSplitThreads, 4) split_best_kernel(SampleP p, SplitP sp) {
  __shared__ float red[2][kSplitThreads / 64];
  const long r = blockIdx.y;
  float most = -__builtin_inff(), least = __builtin_inff();
  part_of<E>(p, sp, r).each([&](float x, int) {
    most = fmaxf(most, x);
    least = least_of(least, x);
  });
  most = lanes_reduce<64, OpMax>(most);
  least = -lanes_reduce<64, OpMax>(-least);
  if ((threadIdx.x & 63) == 0) { red[0][threadIdx.x >> 6] = most; red[1][threadIdx.x >> 6] = least; }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kSplitThreads / 64; ++i) { most = fmaxf(most, red[0][i]); least = fminf(least, red[1][i]); }
    sp.top[r * sp.parts + blockIdx.x] = order_bits(most);
    sp.least[r * sp.parts + blockIdx.x] = least;
  }
  SplitRow& sr = sp.rows[r];                                     // cleared for the kernels behind this one
  for (int i = blockIdx.x * kSplitThreads + threadIdx.x; i < kSplitBins; i += sp.parts * kSplitThreads) {
    sr.mass[i] = 0;
    sr.count[i] = 0;
    if (i == 0) { sr.strong = 0; sr.listed = 0; sr.first = 0xffffffffu; }
  }
}

template <class E>
__global__ void __launch_bounds__(kSplitThreads, 4) split_histogram_kernel(SampleP p, SplitP sp) {
  __shared__ Shared<kSplitThreads> sh;
  const long r = blockIdx.y;
  const Settings set = settings_of(p, r);
  const unsigned top = top_of(sp, r);
  SplitRow& sr = sp.rows[r];
  const auto row = part_of<E>(p, sp, r);
  if (top == kNothing) return;
  if (is_single(set)) {
    row.each([&](float x, int i) {
      if (order_bits(x) == top) atomicMin(&sr.first, (unsigned)i);
    });
    return;
  }
  fill_table(sh.table);
  const Weight w = weight_of(p, set, top, sh.table);
  uint64_t strong = histogram<false, kSplitThreads>(row, w, all_steps<kSplitThreads>(w, top, least_label(sp, r)), set.reach, sh);
  for (int i = threadIdx.x; i < kSplitBins; i += kSplitThreads)
    if (sh.count[i]) {
      atomicAdd(&sr.count[i], sh.count[i]);
      atomicAdd((unsigned long long*)&sr.mass[i], (unsigned long long)sh.mass[i]);
    }
  strong = block_all<kSplitThreads, OpSum>(strong, sh);
  if (threadIdx.x == 0 && strong) atomicAdd((unsigned long long*)&sr.strong, (unsigned long long)strong);
}

template <class E>
__global__ void __launch_bounds__(kSplitThreads, 4) split_collect_kernel(SampleP p, SplitP sp) {
  __shared__ Shared<kSplitThreads> sh;
  const long r = blockIdx.y;
  const Settings set = settings_of(p, r);
  const unsigned top = top_of(sp, r);
  if (top == kNothing || is_single(set)) return;
  const Weight w = weight_of(p, set, top, sh.table);             // (no weight is formed: the table stays empty)
  const Steps st = all_steps<kSplitThreads>(w, top, least_label(sp, r));
  SplitRow& sr = sp.rows[r];
  const Places pl = places_of<kSplitThreads>(sr.mass, sr.count, sr.strong, set, sh);
  const int from = pl.last_k >= 0 ? 0 : pl.low_u, to = pl.last_k >= 0 ? pl.last_k : pl.high_u, also = pl.last_k >= 0 ? -1 : pl.bin_p;
  part_of<E>(p, sp, r).each([&](float x, int i) {
    if (!(x > -__builtin_inff())) return;
    const unsigned b = order_bits(x);
    const uint64_t k = key_of(b, i);
    const int bin = st.bin(x, k);
    if ((bin < from || bin > to) && bin != also) return;
    const unsigned at = atomicAdd(&sr.listed, 1u);
    if (at < (unsigned)kSplitList) sr.list[at] = k;
  });
}

template <class E>
__global__ void __launch_bounds__(kSplitThreads, 4) split_draw_kernel(SampleP p, SplitP sp) {
  __shared__ Shared<kSplitThreads> sh;
  const long r = blockIdx.x;
  const int tid = threadIdx.x;
  const Settings set = settings_of(p, r);
  const unsigned top = top_of(sp, r);
  const SplitRow& sr = sp.rows[r];
  if (top == kNothing || is_single(set)) {
    if (tid == 0) p.out[r] = top == kNothing ? -1 : (int64_t)sr.first;
    return;
  }
  const int n = (int)min(sr.listed, (unsigned)kSplitList);
  fill_table(sh.table);
  const Weight w = weight_of(p, set, top, sh.table);
  const Steps st = all_steps<kSplitThreads>(w, top, least_label(sp, r));
  const Places pl = places_of<kSplitThreads>(sr.mass, sr.count, sr.strong, set, sh);
  if (sr.listed > (unsigned)(pl.last_k >= 0 ? kList : kSplitList)) {
    __syncthreads();
    draw_row<E, kSplitThreads>(p, r, false, sh);
    return;
  }
  if (n <= kList) {
    for (int e = tid; e < n; e += kSplitThreads) {
      const uint64_t k = sr.list[e];
      sh.list[e] = Entry{k, w.of(value_of((unsigned)(k >> 32)))};
    }
    __syncthreads();
    if (pl.last_k >= 0) draw_from_list<kSplitThreads>(w, set, n, p.out + r, sh);
    else finish_from_list<kSplitThreads>(set, st, pl, n, p.out + r, sh);
    return;
  }
  // the label of one bin on which a position falls
  auto look_up = [&](int bin, uint64_t front, uint64_t want) {
    const RowInList row{sr.list, n, bin, st};
    Steps in = st;
    in.step = 0.f;
    uint64_t lo = ~0ull, hi = 0;
    row.each([&](float x, int i) {
      const uint64_t k = key_of(order_bits(x), i);
      lo = min(lo, k);
      hi = max(hi, k);
    });
    in.low = block_all<kSplitThreads, OpMin>(lo, sh);
    in.high = block_all<kSplitThreads, OpMax>(hi, sh);
    bool ready = false;
    Found f = find<false, kSplitThreads>(row, w, in, (unsigned)n, want - front, ready, sh);
    f.upto += front;
    return f;
  };
  // what stands in front of the bins that matter; find has its own use for sh.mass
  uint64_t kept = pl.strong;
  const uint64_t front_p = pl.bin_p >= 0 ? sh.mass[pl.bin_p] : 0;
  const int bins_u = pl.high_u - pl.low_u;
  uint64_t front_u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) front_u[i] = sh.mass[min(pl.low_u + i, kSplitBins - 1)];
  const bool near = bins_u < 4;                                  // u's position moves over a few bins at most; else search again
  __syncthreads();
  if (pl.bin_p >= 0) kept = min(kept, look_up(pl.bin_p, front_p, border_of(set.top_p, pl.all)).upto);
  const uint64_t want = position_of(set.u, kept);
  int bin = pl.low_u;
  uint64_t front = front_u[0];
  if (near) {
#pragma unroll
    for (int i = 1; i < 4; ++i)
      if (i <= bins_u && front_u[i] <= want) { bin = pl.low_u + i; front = front_u[i]; }
  } else {
    front = 0;
    for (int i = 0; i <= pl.high_u; ++i) {
      const uint64_t m = sr.mass[i];
      if (front + m > want) { bin = i; break; }
      front += m;
    }
  }
  const Found f = look_up(bin, front, want);
  if (tid == 0) p.out[r] = (int64_t)(0xffffffffu - (unsigned)f.key);
}

struct SplitPlan { int parts, per; };
// A row is spread over several workgroups where its own passes take longer than the four kernels and the rows' turns in them: 1,024
// workgroups in all, of at least 4,096 labels each.  bf16, one workgroup of 512 threads to a row against spread: 1 x 131072 117 against
// 32 us, 1 x 32768 36 / 28, 64 x 131072 124 / 90, 128 x 131072 128 / 114, but 4 x 16384 24 / 28, 32 x 32768 36 / 39, 64 x 32768 37 / 48,
// 256 x 131072 134 / 174.  With a small top_k a row costs an eighth of that by itself: 1 x 131072 26 / 29, 16 x 131072 27 / 47.
inline SplitPlan split_plan(long n, int v, int vec, bool small_k) {
  const int pieces = v / vec;
  const long most = n > 0 ? 1024 / n : 0, parts = most < v / 4096 ? most : v / 4096;
  if (parts < 2 || v < (24576 + 768 * n) * (small_k ? 8 : 1)) return SplitPlan{1, pieces};
  const int per = (int)((pieces + parts - 1) / parts);
  return SplitPlan{(pieces + per - 1) / per, per};
}
inline int64_t split_bytes(long n, const SplitPlan& plan) {
  return plan.parts < 2 ? 0 : n * (int64_t)sizeof(SplitRow) + n * plan.parts * 8;
}

// Up to 512 labels: the sorting network, in the 16 lanes of a row of the vector unit, whose steps are all within it (65536 x 128 28 us
// against 53 with 64 lanes), 64 lanes for 512 labels, and for 256 where that many rows do not fill the card (65536 x 256 82 us with 64
// lanes, 52 with 16; 2048 x 256 5.4 and 7.6).  Above: a workgroup per row, or several (32768 x 512 75 us sorted, 314 in workgroups).
template <class E>
int launch_sample(const SampleP& p, void* workspace, hipStream_t s) {
  auto sorted = [&](auto lanes, auto per) {
    constexpr int L = decltype(lanes)::value, P = decltype(per)::value;
    hipLaunchKernelGGL((sample_sorted_kernel<E, L, P>), grid_of((p.n + 256 / L - 1) / (256 / L)), dim3(256), 0, s, p);
  };
  using std::integral_constant;
#define OBJ_SORTED(L, P) sorted(integral_constant<int, L>{}, integral_constant<int, P>{})
  if (p.v <= 16) OBJ_SORTED(16, 1);
  else if (p.v <= 32) OBJ_SORTED(16, 2);
  else if (p.v <= 64) OBJ_SORTED(16, 4);
  else if (p.v <= 128) OBJ_SORTED(16, 8);
  else if (p.v <= 256 && p.n > 4096) OBJ_SORTED(16, 16);
  else if (p.v <= 256) OBJ_SORTED(64, 4);
  else if (p.v <= 512) OBJ_SORTED(64, 8);
  else {
    const bool small_k = p.top_k0 >= 1 && p.top_k0 <= kPrune && !p.top_k;
    const SplitPlan plan = split_plan(p.n, p.v, E::kVec, small_k);
    if (plan.parts > 1) {
      SplitP sp;
      sp.rows = static_cast<SplitRow*>(workspace);
      sp.top = reinterpret_cast<unsigned*>(sp.rows + p.n);
      sp.least = reinterpret_cast<float*>(sp.top + p.n * plan.parts);
      sp.parts = plan.parts;
      sp.per = plan.per;
      const dim3 grid((unsigned)plan.parts, (unsigned)p.n), block(kSplitThreads);
      hipLaunchKernelGGL((split_best_kernel<E>), grid, block, 0, s, p, sp);
      hipLaunchKernelGGL((split_histogram_kernel<E>), grid, block, 0, s, p, sp);
      hipLaunchKernelGGL((split_collect_kernel<E>), grid, block, 0, s, p, sp);
      hipLaunchKernelGGL((split_draw_kernel<E>), dim3((unsigned)p.n), block, 0, s, p, sp);
    } else {
      // a kernel for small top_k pays where rows wait for a place on the card (2048 rows of 32768 bf16, top_k 50: 74 -> 55 us, 768: 35 ->
      // 28); where all are on it at once, a second kernel only follows the first (512: 22 and 22, 257 of 30011: 18 -> 20)
      const bool light = p.n > 512 && (p.t || p.top_k || p.c0 == 0.0 || small_k);
      const dim3 grid = grid_of(p.n);
      if (light) hipLaunchKernelGGL((sample_top_kernel<E>), grid, dim3(256), 0, s, p);
      // 512 threads where all rows are on the card at once (512 x 8192 22.6 us against 24.0 with 256 threads, 200 x 32768 42 / 65, 512 x
      // 131072 196 / 253), 256 where rows wait for places or are short (1024 x 8192 33 / 42, 2048 x 32768 178 / 193, 200 x 2048 11.7 / 13.1)
      if (p.v <= 4096 || p.n > 512) hipLaunchKernelGGL((sample_row_kernel<E, 256>), grid, dim3(256), 0, s, p, light);
      else hipLaunchKernelGGL((sample_row_kernel<E, 512>), grid, dim3(512), 0, s, p, light);
    }
  }
#undef OBJ_SORTED
  return check_launch("sample_logits");
}

}  // namespace
}  // namespace objnerf

using namespace objnerf;

extern "C" int64_t objnerf_sample_logits_workspace_bytes(int64_t n, int32_t v, int type) {
  if (n <= 0 || v <= 512 || v > kMaxLabels || !label_type_ok(type)) return 0;
  return split_bytes(n, split_plan(n, v, 16 / label_type_bytes(type), false));
}

extern "C" int objnerf_sample_logits(const objnerf_sample_args* a, void* stream) {
  if (!a) return set_error(-1, "sample_logits: no arguments");
  if (a->n < 0 || a->n > INT32_MAX || a->v < 1 || a->v > kMaxLabels) return set_error(-1, "sample_logits: bad sizes (n < 2^31, 1 <= v <= 2^19)");
  if (!label_type_ok(a->type)) return set_error(-1, "sample_logits: unknown element type");
  if (a->logits_stride < 0 || a->u_stride < 0) return set_error(-1, "sample_logits: bad strides");
  if (!a->temperature_rows && !(a->temperature >= 0.0 && a->temperature < 1e300)) return set_error(-1, "sample_logits: the temperature must be >= 0 and finite");
  if (!a->top_k_rows && a->top_k < 0) return set_error(-1, "sample_logits: top_k must be >= 0");
  if (!a->top_p_rows && !(a->top_p >= 0.0)) return set_error(-1, "sample_logits: top_p must be >= 0");
  if (!a->min_p_rows && !(a->min_p >= 0.0 && a->min_p <= 1.0)) return set_error(-1, "sample_logits: min_p must lie in [0, 1]");
  if (a->n == 0) return 0;
  if (!a->logits || !a->u || !a->labels) return set_error(-1, "sample_logits: a needed buffer is missing");
  if (objnerf_sample_logits_workspace_bytes(a->n, a->v, a->type) && (!a->workspace || (uintptr_t)a->workspace & 7))
    return set_error(-1, "sample_logits: a workspace (8-byte aligned) is needed");
  SampleP p;
  p.n = a->n; p.v = a->v;
  p.z = a->logits; p.ldz = a->logits_stride;
  p.u = a->u; p.ldu = a->u_stride;
  p.t = a->temperature_rows; p.c0 = scale_of(a->temperature);
  p.top_k = a->top_k_rows; p.top_k0 = (int)(a->top_k < a->v ? a->top_k : 0);
  p.top_p = a->top_p_rows; p.top_p0 = a->top_p;
  p.min_p = a->min_p_rows; p.reach0 = reach_of(a->min_p);
  int log_v = 0;
  while ((1ll << log_v) < (long long)a->v) ++log_v;
  p.shift = 62 - log_v < 51 ? 62 - log_v : 51;
  p.out = a->labels;
  hipStream_t s = (hipStream_t)stream;
  return a->type == OBJNERF_TYPE_F32 ? launch_sample<ElemF32>(p, a->workspace, s)
         : a->type == OBJNERF_TYPE_BF16 ? launch_sample<ElemBf16>(p, a->workspace, s) : launch_sample<ElemF16>(p, a->workspace, s);
}
