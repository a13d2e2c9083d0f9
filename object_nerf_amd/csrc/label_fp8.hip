// label_fp8.hip -- products in 8-bit floating point (OCP e4m3) with a scale for each block of 128, and the rounding to that form.
//
//   Q(x): blocks of 128 consecutive columns of a row (or of 128 x 128); scale s = the smallest power of two with
//         max|block| / s <= 448, held as the byte 127 + log2 s; element = e4m3(x / s), to nearest even
//   C[m][n] = sum_k a[m][k] b[n][k] (+ bias[n]) (LeakyReLU)
//
// Measured (copy of this card 4.96 TB/s, fp8 product of the library at 8192 x 8192 x 8192 2.77 PFLOP/s): rounding 307,200 x 256 bf16 by
// rows 46 us = 5.1 TB/s, 16,383 x 2,056 in both forms 33 us = 4.1 TB/s; product 8192 x 8192 x 8192 480 us = 2.29 PFLOP/s, x 4096
// 239-259 us = 2.1-2.3 PFLOP/s, 4096 x 4096 x 4096 64 us = 2.15 PFLOP/s and 120 with fp32 results = 1.14, 2,056 x 520 x 16,384 with fp32
// results 53-56 us = 0.64 PFLOP/s; four rows against 32,768 x 256 (8.4 MB of weights) 4-6 us.  What bounds it: large products waits, for
// fragments read just in front of their products and for a block's copies (the matrix pipe is busy 0.46 of the time); sums of a few blocks
// the launch-to-store latency of a tile; hidden layers over a frame the write path.  Columns that are no multiple of 8 read a row's last
// ones an element after the other.
//
// The scale is a power of two on purpose.  Dividing by it is exact, so an element is rounded once and the byte form has one meaning;
// a factor up to 2 of the range it gives away costs no precision (a floating-point format's step does not depend on where in its
// range a value lies, down to its subnormals at 2^-15 of the block's largest).  And it is the form that the matrix instruction itself
// takes: v_mfma_scale_f32_16x16x128_f8f6f4 multiplies a block of 128 by both scales on its way into the fp32 accumulator, so a
// block costs no instruction besides its product.
//
// That instruction adds eight products at a time on a common exponent and drops what lies more than 13 bits under the largest of
// them, before the sum reaches the fp32 accumulator (measured; the older v_mfma_f32_16x16x32_fp8_fp8 does the same): a product of
// 128 normal numbers comes out 1.5e-5 off, relative to its norm.  Behind it a 16-bit result rounds by 1.7e-3 (bf16) or 2.1e-4 (fp16), so
// C in 16 bits takes it.  C in fp32 does not: its operands are widened to bf16 in registers (exact: 4 bits and a power of two, down to
// kLeastWide) and multiplied by the bf16 instruction at half the rate, which keeps fp32 sums (1.2e-8).
//
// Layout: values (R, C') with C' = C filled up to whole blocks with zeros; scales (R, B') bytes, one per row and block, B' = the
// number of blocks filled up to a multiple of 4 (with 127): one aligned dword holds four blocks' scales, the instruction's op_sel
// picks the byte.  Blocks of 128 x 128 repeat their scale in 128 rows: a 128th of the values' bytes buys one form for all.
#include "host_api.h"
#include "device_math.h"
#include "label_ops.h"
#include <type_traits>

namespace objnerf {
namespace {

constexpr int kBlock = 128;
using i32x8 = __attribute__((ext_vector_type(8))) int;

// largest finite |x| of a block -> its scale byte
__device__ __forceinline__ unsigned scale_byte(float largest) {
  const unsigned b = __float_as_uint(largest);
  const int e = (int)(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);      // 448 = 1.75 * 2^8
  return b == 0 ? 127u : (unsigned)max(e, 1);
}
__device__ __forceinline__ float inverse_scale(unsigned byte) { return __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < __builtin_inff() ? a : 0.f;                         // NaN and infinities set no scale (and become NaN)
}
__device__ __forceinline__ unsigned fp8x4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

// eight consecutive columns of a row as they lie in memory; what lies behind its end is 0
template <class E> struct Eight {
  static constexpr int kPieces = 8 / E::kVec;
  u32x4 r[kPieces];
  __device__ __forceinline__ void load(const char* row, long c, long cols) {
    if (c + 8 <= cols) {
#pragma unroll
      for (int h = 0; h < kPieces; ++h) r[h] = load16(row, (c + h * E::kVec) * E::kBytes);
    } else {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = c + i < cols ? E::load(row, c + i) : 0.f;
#pragma unroll
      for (int h = 0; h < kPieces; ++h) r[h] = E::pack(x + h * E::kVec);
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int h = 0; h < kPieces; ++h) r[h] = u32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ void values(float* x) const {
#pragma unroll
    for (int h = 0; h < kPieces; ++h) E::unpack(r[h], x + h * E::kVec);
  }
};

struct QuantP {
  long rows, cols;
  const void* x; long ldx;
  uint8_t* q; uint8_t* scale;             // rows
  uint8_t* qt; uint8_t* scale_t;          // columns as rows
  float* part;                            // (row blocks, cols): column sums of 128 rows
};
__host__ __device__ __forceinline__ long blocks_of(long n) { return (n + kBlock - 1) / kBlock; }
__host__ __device__ __forceinline__ long scale_stride(long n) { return (blocks_of(n) + 3) / 4 * 4; }

// Blocks of one row: 16 lanes each.  Streams x once and writes half of it (or a quarter) back.
template <class E>
__global__ void __launch_bounds__(256) quantize_rows_kernel(QuantP p) {
  const long kb = blocks_of(p.cols), sb = scale_stride(p.cols);
  const long block = workgroup() * 16 + (threadIdx.x >> 4);
  const int l = threadIdx.x & 15;
  const bool in = block < p.rows * kb;
  const long row = in ? block / kb : 0, b = in ? block - row * kb : 0;
  const char* xr = static_cast<const char*>(p.x) + row * p.ldx * E::kBytes;
  Eight<E> held;
  held.load(xr, b * kBlock + l * 8, p.cols);
  float x[8];
  held.values(x);
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = fmaxf(a, finite_abs(x[i]));
  a = lanes_reduce<16, OpMax>(a);
  if (!in) return;
  const unsigned byte = scale_byte(a);
  const float inv = inverse_scale(byte);
  uint2 o;
  o.x = fp8x4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
  o.y = fp8x4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
  *reinterpret_cast<uint2*>(p.q + row * kb * kBlock + b * kBlock + l * 8) = o;
  if (l == 0) p.scale[row * sb + b] = (uint8_t)byte;
  if (b == kb - 1 && l > 0 && b + l < sb) p.scale[row * sb + b + l] = 127;
}

// A 128 x 128 tile: blocks of 128 x 128, the transposed form, both forms at once, and the column sums.  Thread (g, l): rows 8 g .. 8 g + 7,
// columns 8 l .. 8 l + 7, held as they were read.  A row of the transposed tile is 144 bytes of LDS.
constexpr int kPitch = 144;
template <class E, bool ROWS, bool TRANS, bool SQUARE>
__global__ void __launch_bounds__(256, 4) quantize_tile_kernel(QuantP p) {
  __shared__ float per_thread[16][kBlock];
  __shared__ unsigned col_byte[kBlock];
  __shared__ __align__(16) uint8_t tile[TRANS ? kBlock * kPitch : 16];
  const long kb = blocks_of(p.cols), sb = scale_stride(p.cols), mb = blocks_of(p.rows), sbt = scale_stride(p.rows);
  const long bc = workgroup() % kb, br = workgroup() / kb;
  if (br >= mb) return;
  const int g = threadIdx.x >> 4, l = threadIdx.x & 15;
  const long r0 = br * kBlock + g * 8, c0 = bc * kBlock + l * 8;
  Eight<E> held[8];
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    if (r0 + s < p.rows) held[s].load(static_cast<const char*>(p.x) + (r0 + s) * p.ldx * E::kBytes, c0, p.cols);
    else held[s].clear();
  }
  // one pass over the rows: largest of each row (16 lanes), of each column (16 threads), column sums (8 rows in order, then 16 threads)
  float column[8], sum[8];
  unsigned row_byte[8], square_byte = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) { column[i] = 0.f; sum[i] = 0.f; }
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    float x[8], a = 0.f;
    held[s].values(x);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float v = finite_abs(x[i]);
      a = fmaxf(a, v);
      column[i] = fmaxf(column[i], v);
      sum[i] = s == 0 ? x[i] : sum[i] + x[i];
    }
    if (ROWS && !SQUARE) row_byte[s] = scale_byte(lanes_reduce<16, OpMax>(a));
  }
  if (TRANS || SQUARE) {
#pragma unroll
    for (int i = 0; i < 8; ++i) per_thread[g][l * 8 + i] = column[i];
    __syncthreads();
    if (threadIdx.x < kBlock) {
      float a = 0.f;
#pragma unroll
      for (int s = 0; s < 16; ++s) a = fmaxf(a, per_thread[s][threadIdx.x]);
      col_byte[threadIdx.x] = SQUARE ? __float_as_uint(a) : scale_byte(a);
    }
    __syncthreads();
    if (SQUARE) {
      unsigned a = max(col_byte[threadIdx.x & 63], col_byte[64 + (threadIdx.x & 63)]);      // non-negative floats order as their bits
      square_byte = scale_byte(__uint_as_float(lanes_reduce<64, OpMax>(a)));
    }
  }
  if (p.part) {
    if (TRANS || SQUARE) __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) per_thread[g][l * 8 + i] = sum[i];
    __syncthreads();
    const long col = bc * kBlock + threadIdx.x;
    if (threadIdx.x < kBlock && col < p.cols) {
      float a = per_thread[0][threadIdx.x];
#pragma unroll
      for (int s = 1; s < 16; ++s) a += per_thread[s][threadIdx.x];
      p.part[br * p.cols + col] = a;
    }
  }
  if (ROWS) {
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const unsigned byte = SQUARE ? square_byte : row_byte[s];
      const float inv = inverse_scale(byte);
      const long row = r0 + s;
      if (row < p.rows) {
        float x[8];
        held[s].values(x);
        uint2 o;
        o.x = fp8x4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
        o.y = fp8x4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
        *reinterpret_cast<uint2*>(p.q + row * kb * kBlock + c0) = o;
        if (l == 0) p.scale[row * sb + bc] = (uint8_t)byte;
        if (bc == kb - 1 && l > 0 && bc + l < sb) p.scale[row * sb + bc + l] = 127;
      }
    }
  }
  if (TRANS) {
    // four rows at a time: four bytes of each of the eight columns
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      float x[4][8];
#pragma unroll
      for (int s = 0; s < 4; ++s) held[q * 4 + s].values(x[s]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float inv = inverse_scale(SQUARE ? square_byte : col_byte[l * 8 + i]);
        *reinterpret_cast<unsigned*>(&tile[(l * 8 + i) * kPitch + g * 8 + q * 4]) = fp8x4(x[0][i] * inv, x[1][i] * inv, x[2][i] * inv, x[3][i] * inv);
      }
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int piece = s * 256 + threadIdx.x, c = piece >> 3, at = (piece & 7) * 16;
      const long col = bc * kBlock + c;
      if (col < p.cols) *reinterpret_cast<u32x4*>(p.qt + col * mb * kBlock + br * kBlock + at) = *reinterpret_cast<const u32x4*>(&tile[c * kPitch + at]);
    }
    const long col = bc * kBlock + threadIdx.x;
    if (threadIdx.x < kBlock && col < p.cols) {
      p.scale_t[col * sbt + br] = (uint8_t)(SQUARE ? square_byte : col_byte[threadIdx.x]);
      if (br == mb - 1)
        for (long e = mb; e < sbt; ++e) p.scale_t[col * sbt + e] = 127;
    }
  }
}

// column sums from the tiles' partial sums: 16 threads per column, each a run of row blocks in order, joined in order
__global__ void __launch_bounds__(256) join_sums_kernel(const float* __restrict__ part, long blocks, long cols, float* __restrict__ sum) {
  __shared__ float s[16][16];
  const int l = threadIdx.x & 15, g = threadIdx.x >> 4;
  const long col = workgroup() * 16 + l;
  const long per = (blocks + 15) / 16;
  float a = 0.f;
  if (col < cols)
    for (long b = g * per; b < min((g + 1) * per, blocks); ++b) a += part[b * cols + col];
  s[g][l] = a;
  __syncthreads();
  if (g == 0 && col < cols) {
#pragma unroll
    for (int i = 1; i < 16; ++i) a += s[i][l];
    sum[col] = a;
  }
}

template <class E>
int launch_quantize(const QuantP& p, bool square, float* sum, hipStream_t s) {
  const long tiles = blocks_of(p.rows) * blocks_of(p.cols);
  if (!square && !p.qt && !p.part) {
    hipLaunchKernelGGL((quantize_rows_kernel<E>), grid_of((p.rows * blocks_of(p.cols) + 15) / 16), dim3(256), 0, s, p);
  } else {
    const dim3 grid = grid_of(tiles);
    if (square) {
      if (p.q && p.qt) hipLaunchKernelGGL((quantize_tile_kernel<E, true, true, true>), grid, dim3(256), 0, s, p);
      else if (p.q) hipLaunchKernelGGL((quantize_tile_kernel<E, true, false, true>), grid, dim3(256), 0, s, p);
      else hipLaunchKernelGGL((quantize_tile_kernel<E, false, true, true>), grid, dim3(256), 0, s, p);
    } else {
      if (p.q && p.qt) hipLaunchKernelGGL((quantize_tile_kernel<E, true, true, false>), grid, dim3(256), 0, s, p);
      else if (p.q) hipLaunchKernelGGL((quantize_tile_kernel<E, true, false, false>), grid, dim3(256), 0, s, p);
      else hipLaunchKernelGGL((quantize_tile_kernel<E, false, true, false>), grid, dim3(256), 0, s, p);
    }
  }
  if (sum) hipLaunchKernelGGL(join_sums_kernel, grid_of((p.cols + 15) / 16), dim3(256), 0, s, p.part, blocks_of(p.rows), p.cols, sum);
  return check_launch("fp8_quantize");
}

// ---- the product ----

struct GemmP {
  long M, N, K;                            // K: whole blocks
  const uint8_t* a; long lda; const uint8_t* sa; long ldsa;      // a not yet rounded: elements (M, cols), lda in elements, no sa
  long cols;
  const uint8_t* b; long ldb; const uint8_t* sb; long ldsb;
  const float* bias;
  int leaky;
  void* c; long ldc;
  float* partial;                          // (splits, M, N) sums of a run of blocks each, or null
  long blocks_per_split;
};

using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
typedef __attribute__((address_space(3))) uint8_t lds_byte;
typedef const __attribute__((address_space(1))) uint8_t global_byte;

// 8 elements (two dwords) times their block's scale: exact where the last bit of e4m3's smallest, 2^-9 of the scale, is not under bf16's
// smallest number, 2^-133: for scale bytes from kLeastWide on
constexpr int kLeastWide = 3;
__device__ __forceinline__ bf16x8 widened(int lo, int hi, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ float scale_of(unsigned byte) { return __uint_as_float(byte << 23); }
__device__ __forceinline__ float finished(float v, const GemmP& p, float bias) {
  v += bias;
  return p.leaky ? fmaxf(v, 0.01f * v) : v;
}

// Where piece c of a row lies in LDS: at c ^ piece_key(row).  Rows are 32 banks apart, so that 16 rows of a fragment need their eight pairs
// on eight different pieces; and the hardware serves a 16-byte read not in runs of 16 lanes but, e.g., lanes 0-3, 12-15 and 20-27
// together: rows 0-3 and 12-15 of piece c with rows 4-11 of piece c + 2.  Keys 0 2 | 1 3 5 7 | 4 6 keep both apart.
__device__ __forceinline__ int piece_key(int row) { return 0x64753120 >> ((row >> 1 & 7) * 4) & 7; }

// Four neighbouring columns of one row of C.
template <class E> __device__ __forceinline__ void write4(char* c, f32x4 v) {
  if (E::kBytes == 4) {
    *reinterpret_cast<u32x4e*>(c) = u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
  } else {
    float x[8] = {v[0], v[1], v[2], v[3], 0.f, 0.f, 0.f, 0.f};
    const u32x4 o = E::pack(x);
    typedef unsigned u32x2e __attribute__((ext_vector_type(2), aligned(2)));
    *reinterpret_cast<u32x2e*>(c) = u32x2e{o[0], o[1]};
  }
}
template <class E> __device__ __forceinline__ void store4(const GemmP& p, long m, long n, f32x4 v) {
  char* c = static_cast<char*>(p.c) + (m * p.ldc + n) * E::kBytes;
  if (n + 4 <= p.N) {
    write4<E>(c, v);
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (n + r < p.N) E::store(c, r, v[r]);
  }
}

// Which BM x BN of C is number `at` of a launch's tiles.  Workgroups go round the 8 XCDs (and a workgroup's tiles are a multiple of 8
// apart): each XCD takes one run of tiles, in panels of 8 tile rows, so that its L2 serves neighbours.
template <int BM, int BN> __device__ __forceinline__ long tiles_of(const GemmP& p) { return (p.M + BM - 1) / BM * ((p.N + BN - 1) / BN); }
template <int BM, int BN> __device__ __forceinline__ void tile_of(const GemmP& p, long at, long& m0, long& n0) {
  const long mt = (p.M + BM - 1) / BM, nt = (p.N + BN - 1) / BN, tiles = mt * nt;
  const long xcd = at % 8, per = tiles / 8, more = tiles % 8;
  const long tile = xcd * per + min(xcd, more) + at / 8;
  const long panel = tile / (8 * nt), rows = min(mt - panel * 8, 8l), in = tile - panel * 8 * nt;
  m0 = (panel * 8 + in % rows) * BM;
  n0 = in / rows * BN;
}

// The copies of a workgroup's rows from memory straight into LDS.  A step is one block of 128: BM + BN rows of 128 bytes into one of two
// slots.  The 16-byte pieces of a row are permuted (piece_key) on the addresses the lanes read from, since LDS is filled in order.  Scales:
// a dword of each row, four steps' worth, into two slots of their own; a wave copies those of 64 rows.  Which slot is the caller's count.
template <int BM, int BN, int WAVES, bool RAW> struct Copies {
  static constexpr int kScaleRows = (BM + BN + 63) / 64 * 64, kScaleCopies = (kScaleRows / 64 + WAVES - 1) / WAVES;
  static constexpr int kSlot = (BM + BN) * kBlock, kBytes = 2 * kSlot + 2 * kScaleRows * 4;
  static constexpr int RA = RAW ? 0 : BM / WAVES / 8, RB = BN / WAVES / 8;
  static_assert((RAW || BM % (8 * WAVES) == 0) && BN % (8 * WAVES) == 0, "whole groups of 8 rows per wave");
  const uint8_t *abase, *bbase, *sbase[kScaleCopies];
  unsigned aoff[RA + 1], boff[RB];
  lds_byte* lds;
  __device__ __forceinline__ void aim(const GemmP& p, long m0, long n0, long first) {
    const int lane = threadIdx.x & 63, wave = uni((int)(threadIdx.x >> 6));
    // this lane's part: row lane / 8 of every 8, piece lane % 8 of LDS
    const long arow = min(m0 + wave * RA * 8, p.M - 1), brow = min(n0 + wave * RB * 8, p.N - 1);
    abase = RAW ? nullptr : p.a + arow * p.lda + first * kBlock;
    bbase = p.b + brow * p.ldb + first * kBlock;
#pragma unroll
    for (int c = 0; c < RA; ++c) {
      const int r = wave * RA * 8 + c * 8 + lane / 8;
      aoff[c] = (unsigned)((min(m0 + r, p.M - 1) - arow) * p.lda) + (((lane & 7) ^ piece_key(r)) << 4);
    }
#pragma unroll
    for (int c = 0; c < RB; ++c) {
      const int r = wave * RB * 8 + c * 8 + lane / 8;
      boff[c] = (unsigned)((min(n0 + r, p.N - 1) - brow) * p.ldb) + (((lane & 7) ^ piece_key(r)) << 4);
    }
#pragma unroll
    for (int c = 0; c < kScaleCopies; ++c) {
      const int r = (c * WAVES + wave) * 64 + lane;
      sbase[c] = r < BM && !RAW ? p.sa + min(m0 + r, p.M - 1) * p.ldsa : p.sb + max(min(n0 + r - BM, p.N - 1), 0l) * p.ldsb;
    }
  }
  __device__ __forceinline__ void rows(long step, int to) const {
    const int wave = uni((int)(threadIdx.x >> 6));
    lds_byte* slot = lds + to * kSlot + wave * RA * 1024;
    const uint8_t* from = abase + step * kBlock;
#pragma unroll
    for (int c = 0; c < RA; ++c)
      __builtin_amdgcn_global_load_lds((global_byte*)(from + aoff[c]), (__attribute__((address_space(3))) void*)(slot + c * 1024), 16, 0, 0);
    slot = lds + to * kSlot + BM * kBlock + wave * RB * 1024;
    from = bbase + step * kBlock;
#pragma unroll
    for (int c = 0; c < RB; ++c)
      __builtin_amdgcn_global_load_lds((global_byte*)(from + boff[c]), (__attribute__((address_space(3))) void*)(slot + c * 1024), 16, 0, 0);
  }
  // (a's rows where it is rounded here: their dwords are another wave's stores, the copy starts behind them)
  __device__ __forceinline__ void scales(long group, int to) const {
    const int wave = uni((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
#pragma unroll
    for (int c = 0; c < kScaleCopies; ++c) {
      const int from = (c * WAVES + wave) * 64;
      if (from >= kScaleRows || (RAW && from + 64 <= BM)) continue;
      if (RAW && from < BM && from + lane < BM) continue;        // lanes of a's rows copy nothing: their places stay as they are
      __builtin_amdgcn_global_load_lds((global_byte*)(sbase[c] + group * 4), (__attribute__((address_space(3))) void*)(lds + 2 * kSlot + (to * kScaleRows + from) * 4), 4, 0, 0);
    }
  }
  // scale byte of row 0 of the tile for a block; rows are 4 bytes apart, b's rows behind a's
  __device__ __forceinline__ lds_byte* scale_at(long block, int slot) const { return lds + 2 * kSlot + slot * kScaleRows * 4 + (int)(block & 3); }
};
// a's rows of a step where they are rounded on their way into LDS: 16 lanes per row and block, held in registers from the load to the
// store.  The load is not hidden by the step in between: as built, the step's products stand behind the wait for it.
template <class A, int BM, int THREADS, class COPY> struct RawRows {
  static constexpr int kPasses = BM * 16 / THREADS;
  Eight<A> held[kPasses];
  __device__ __forceinline__ void load(const GemmP& p, long m0, long block) {
    const int l = threadIdx.x & 15, g = threadIdx.x >> 4;
#pragma unroll
    for (int s = 0; s < kPasses; ++s)
      held[s].load(reinterpret_cast<const char*>(p.a) + min(m0 + s * (THREADS / 16) + g, p.M - 1) * p.lda * A::kBytes, block * kBlock + l * 8, p.cols);
  }
  __device__ __forceinline__ void store(const COPY& copy, int slot, lds_byte* scale) const {
    const int l = threadIdx.x & 15, g = threadIdx.x >> 4;
    lds_byte* const rows = copy.lds + slot * COPY::kSlot;
#pragma unroll
    for (int s = 0; s < kPasses; ++s) {
      float x[8];
      held[s].values(x);
      float largest = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) largest = fmaxf(largest, finite_abs(x[i]));
      const unsigned byte = scale_byte(lanes_reduce<16, OpMax>(largest));
      const float inv = inverse_scale(byte);
      typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
      const u32x2 o = {fp8x4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv), fp8x4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv)};
      const int r = s * (THREADS / 16) + g;
      *(__attribute__((address_space(3))) u32x2*)(rows + r * kBlock + (((l >> 1) ^ piece_key(r)) << 4) + (l & 1) * 8) = o;
      if (l == 0) scale[r * 4] = (uint8_t)byte;
    }
  }
};
struct NoRaw {
  template <class... T> __device__ __forceinline__ void load(T...) {}
  template <class... T> __device__ __forceinline__ void store(T...) const {}
};

// a lane's 32 bytes of a fragment: row i of the 16 rows at `rows`, the h-th run of 32 of the block
__device__ __forceinline__ i32x8 fragment(const lds_byte* rows, int i, int h) {
  const int key = piece_key(i);
  const u32x4 lo = *(const __attribute__((address_space(3))) u32x4*)(rows + i * kBlock + ((h * 2 ^ key) << 4));
  const u32x4 hi = *(const __attribute__((address_space(3))) u32x4*)(rows + i * kBlock + (((h * 2 + 1) ^ key) << 4));
  return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}
__device__ __forceinline__ f32x4 mfma8(i32x8 b, i32x8 a, f32x4 c, int sb, int sa) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, c, 0, 0, 0, sb, 0, sa);
}

// A wave's TM x TN tiles of 16 x 16 to memory, 16 rows at a time through 16 x (16 TN + 4) floats of LDS that are the wave's own (it serves
// a wave's accesses in order: no barrier), so that neighbouring lanes store neighbouring 16 bytes of a row.
template <class E, int TM, int TN>
__device__ __forceinline__ void write_tile(const GemmP& p, long m0, long n0, lds_byte* area, const f32x4 (&acc)[TM][TN]) {
  typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
  constexpr int kPitch = TN * 16 + 4, kLanes = TN * 16 / E::kVec, kRows = 64 / kLanes;       // lanes per row, rows at once
  const int lane = threadIdx.x & 63, i = lane & 15, h = lane >> 4, c = lane % kLanes * E::kVec;
  const long n = n0 + c;
  const int have = (int)min(max(p.N - n, 0l), (long)E::kVec);    // columns of this lane that exist
  float bias[E::kVec];
#pragma unroll
  for (int e = 0; e < E::kVec; ++e) bias[e] = p.bias && e < have ? p.bias[n + e] : 0.f;
#pragma unroll
  for (int u = 0; u < TM; ++u) {
#pragma unroll
    for (int t = 0; t < TN; ++t) *(lds_f32x4*)(area + (i * kPitch + t * 16 + h * 4) * 4) = acc[u][t];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 1
    for (int r = lane / kLanes; r < 16; r += kRows) {
      const long m = m0 + u * 16 + r;
      if (m >= p.M || have == 0) continue;
      float x[E::kVec];
#pragma unroll
      for (int q = 0; q < E::kVec / 4; ++q) {
        const f32x4 v = *(const lds_f32x4*)(area + (r * kPitch + c + q * 4) * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[q * 4 + e] = v[e];
      }
      if (p.partial) {
        float* o = p.partial + ((long)blockIdx.y * p.M + m) * p.N + n;
        if (have == E::kVec) {
#pragma unroll
          for (int q = 0; q < E::kVec / 4; ++q) store16(o, q * 16, u32x4{__float_as_uint(x[q * 4]), __float_as_uint(x[q * 4 + 1]), __float_as_uint(x[q * 4 + 2]), __float_as_uint(x[q * 4 + 3])});
        } else {
#pragma unroll 1
          for (int e = 0; e < have; ++e) o[e] = *(const __attribute__((address_space(3))) float*)(area + (r * kPitch + c + e) * 4);
        }
        continue;
      }
#pragma unroll
      for (int e = 0; e < E::kVec; ++e) x[e] = finished(x[e], p, bias[e]);
      char* o = static_cast<char*>(p.c) + (m * p.ldc + n) * E::kBytes;
      if (have == E::kVec) store16(o, 0, E::pack(x));
      else
#pragma unroll
        for (int e = 0; e < E::kVec; ++e)
          if (e < have) E::store(o, e, x[e]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// A wave's tiles once more where some block's scale was under kLeastWide: the products without scales, and both exponents added to every
// block's sums.  Straight from memory, a tile after the other: it is rare (an operand's block with nothing over 2^-116), and as code behind
// the loop it costs the loop one minimum per scale: nothing measurable at 4096 x 4096 x 4096 (120 us), 3 % where a is fp32 rounded inside
// (307200 x 128 x 256: 110 to 114 us, registers).
template <class A> struct AgainRow {                               // a lane's 32 elements of a block of a's row, and its scale
  u32x4 f[2];
  int scale;
  __device__ __forceinline__ void load(const GemmP& p, long row, long block, int h) {
    if constexpr (std::is_same<A, void>::value) {
      const u32x4* const from = reinterpret_cast<const u32x4*>(p.a + row * p.lda + block * kBlock + h * 32);
      f[0] = from[0];
      f[1] = from[1];
      scale = p.sa[row * p.ldsa + block];
    } else {
      const char* const from = reinterpret_cast<const char*>(p.a) + row * p.lda * A::kBytes;
      const long c = block * kBlock + h * 32;
      Eight<A> held;
      float largest = 0.f, x[8];
#pragma unroll 1
      for (int e = 0; e < 32; ++e) largest = fmaxf(largest, finite_abs(c + e < p.cols ? A::load(from, c + e) : 0.f));
      largest = join_rows<OpMax, true>(join_rows<OpMax, false>(largest));      // the four lanes of a row
      scale = (int)scale_byte(largest);
      const float inv = inverse_scale(scale);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        held.load(from, c + e * 8, p.cols);
        held.values(x);
        f[e >> 1][(e & 1) * 2] = fp8x4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
        f[e >> 1][(e & 1) * 2 + 1] = fp8x4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
};
template <class A, int TM, int TN>
__device__ __forceinline__ void sum_again(const GemmP& p, long m0, long n0, long first, long steps, f32x4 (&acc)[TM][TN]) {
#pragma unroll
  for (int u = 0; u < TM; ++u)
#pragma unroll
    for (int t = 0; t < TN; ++t) {
      f32x4 total = {};
#pragma unroll 1
      for (long block = first; block < first + steps; ++block) {
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));                             // no address is held from block to block or through the loops around
        const int i = lane & 15, h = lane >> 4;
        AgainRow<A> a;
        a.load(p, min(m0 + u * 16 + i, p.M - 1), block, h);
        const u32x4* const at = reinterpret_cast<const u32x4*>(p.b + min(n0 + t * 16 + i, p.N - 1) * p.ldb + block * kBlock + h * 32);
        const u32x4 fb[2] = {at[0], at[1]};
        f32x4 sum = {};
#pragma unroll
        for (int q = 0; q < 4; ++q)
          sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widened(fb[q >> 1][(q & 1) * 2], fb[q >> 1][(q & 1) * 2 + 1], 1.f),
                                                        widened(a.f[q >> 1][(q & 1) * 2], a.f[q >> 1][(q & 1) * 2 + 1], 1.f), sum, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) total[r] += __builtin_amdgcn_ldexpf(sum[r], a.scale + p.sb[min(n0 + t * 16 + h * 4 + r, p.N - 1) * p.ldsb + block] - 254);
      }
      acc[u][t] = total;
      __builtin_amdgcn_sched_barrier(0);
    }
}

// Before a barrier behind which other waves read what this one's copies bring: the copies count as loads from memory, and nothing in the
// barrier itself waits for them.
__device__ __forceinline__ void copies_landed() { __builtin_amdgcn_s_waitcnt(0x0f70); }      // vmcnt 0; the other counters stay

// BM x BN of C per workgroup of WM x WN waves, rows copied one step ahead, one barrier a step.  The instruction's "A" is b's rows and its
// "B" a's: a lane's four results are four neighbouring columns of one row of C.  In the widened form the four instructions of a
// block take 8 bytes of every lane's 32 each: another order of the same sum.
template <class E, class A, bool WIDE, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(WM * WN * 64, 2) gemm_fp8_kernel(GemmP p) {
  constexpr bool kRaw = !std::is_same<A, void>::value, kRun = BM < 256;      // (256 x 256: no registers to spare for a next tile)
  using Copy = Copies<BM, BN, WM * WN, kRaw>;
  using Raw = typename std::conditional<kRaw, RawRows<typename std::conditional<kRaw, A, ElemF32>::type, BM, WM * WN * 64, Copy>, NoRaw>::type;
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
  __shared__ __align__(16) uint8_t ring[Copy::kBytes];
  static_assert(WM * WN * 16 * (TN * 16 + 4) * 4 <= Copy::kSlot, "the waves' areas of write_tile fit into a slot");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, h = lane >> 4;
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
  const long first = blockIdx.y * p.blocks_per_split, steps = min(p.blocks_per_split, p.K / kBlock - first);
  long at = blockIdx.x, m0, n0;
  tile_of<BM, BN>(p, at, m0, n0);
  Copy copy;
  copy.lds = (lds_byte*)ring;
  copy.aim(p, m0, n0, first);
  Raw raw;
  int slot = 0, scale_slot = 0;
  if (steps > 0) {
    raw.load(p, m0, first);
    copy.rows(0, 0);
    copy.scales(first >> 2, 0);
    raw.store(copy, 0, copy.scale_at(first, 0));
  }
  // a workgroup's tiles one after the other: the next one's first rows are asked for before this one's results are written, and have
  // arrived before the first of them is stored (write_tile's loads of the bias are counted behind them)
  for (bool more = true; more;) {
    f32x4 acc[TM][TN] = {};
    int least = kLeastWide;                                        // scale byte of this lane's rows, where C is fp32
    const long m = m0, n = n0;
    at += gridDim.x;
    more = kRun && at < tiles_of<BM, BN>(p);
    for (long step = 0; step < steps; ++step) {
      copies_landed();
      __syncthreads();                                             // the step's rows have landed; the other slot has been read
      const lds_byte* const rows_a = copy.lds + slot * Copy::kSlot + wm * kBlock;
      const lds_byte* const rows_b = copy.lds + slot * Copy::kSlot + (BM + wn) * kBlock;
      const lds_byte* const scale_a = copy.scale_at(first + step, scale_slot) + (wm + i) * 4;
      const lds_byte* const scale_b = copy.scale_at(first + step, scale_slot) + (BM + wn + i) * 4;
      const bool last = step + 1 == steps;
      const long block = last ? first : first + step + 1;          // the next one, of this tile or of the next
      slot ^= 1;
      if (!last || more) {
        if (last) {
          tile_of<BM, BN>(p, at, m0, n0);
          copy.aim(p, m0, n0, first);
        }
        raw.load(p, m0, block);
        copy.rows(block - first, slot);
        if (last || (block & 3) == 0) {
          scale_slot ^= 1;
          copy.scales(block >> 2, scale_slot);
        }
      }
      i32x8 fa[TM];
      int sa[TM];
#pragma unroll
      for (int t = 0; t < TM; ++t) sa[t] = scale_a[t * 64];
#pragma unroll
      for (int t = 0; t < TM; ++t) fa[t] = fragment(rows_a + t * 16 * kBlock, i, h);
      if constexpr (WIDE) {
        i32x8 fb[TN];
#pragma unroll
        for (int t = 0; t < TN; ++t) fb[t] = fragment(rows_b + t * 16 * kBlock, i, h);
#pragma unroll
        for (int t = 0; t < TM; ++t) least = min(least, sa[t]);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          bf16x8 xa[TM];
#pragma unroll
          for (int t = 0; t < TM; ++t) xa[t] = widened(fa[t][2 * q], fa[t][2 * q + 1], scale_of(sa[t]));
#pragma unroll
          for (int t = 0; t < TN; ++t) {
            const int sb = scale_b[t * 64];
            if (q == 3) least = min(least, sb);
            const bf16x8 xb = widened(fb[t][2 * q], fb[t][2 * q + 1], scale_of(sb));
#pragma unroll
            for (int u = 0; u < TM; ++u) acc[u][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xb, xa[u], acc[u][t], 0, 0, 0);
          }
        }
      } else {
#pragma unroll
        for (int t = 0; t < TN; ++t) {
          const i32x8 fb = fragment(rows_b + t * 16 * kBlock, i, h);
          const int sb = scale_b[t * 64];
#pragma unroll
          for (int u = 0; u < TM; ++u) acc[u][t] = mfma8(fb, fa[u], acc[u][t], sb, sa[u]);
        }
      }
      if (!last || more) raw.store(copy, slot, copy.scale_at(block, scale_slot));
    }
    if constexpr (WIDE)
      if (__any(least < kLeastWide)) sum_again<A, TM, TN>(p, m + wm, n + wn, first, steps, acc);
    // the slot that has just been read serves the results; the other one's copies are under way: a barrier that waits for none of them
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    write_tile<E, TM, TN>(p, m + wm, n + wn, copy.lds + (slot ^ 1) * Copy::kSlot + wave * 16 * (TN * 16 + 4) * 4, acc);
  }
}

// C from the partial sums of the splits, in their order
template <class E>
__global__ void __launch_bounds__(256) join_splits_kernel(GemmP p, int splits) {
  const long groups = (p.N + 3) / 4, at = (long)blockIdx.x * 256 + threadIdx.x;
  if (at >= p.M * groups) return;
  const long m = at / groups, n = (at - m * groups) * 4;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  const bool whole = n + 4 <= p.N;
  for (int s = 0; s < splits; s += 4) {
    f32x4 o[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float* at_s = p.partial + ((long)min(s + u, splits - 1) * p.M + m) * p.N + n;
      if (whole) {
        __builtin_memcpy(&o[u], at_s, 16);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) o[u][r] = n + r < p.N ? at_s[r] : 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (s + u < splits) v += o[u];
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = finished(v[r], p, p.bias && n + r < p.N ? p.bias[n + r] : 0.f);
  store4<E>(p, m, n, v);
}

// Tile and split of a product.  Up to 32 rows: 32 x 128 per workgroup.  Else 256 x 256, one workgroup per CU, or 128 x 128, two per CU.  A
// round of the larger takes as long as 1.8 of the smaller (four times the work at 1.1 times the rate, against twice), a last round of the
// smaller with one tile per CU 0.6; the larger is taken where its rounds take less and the sum has four blocks at least: 8192 x 8192 x
// 4096 245-259 us against 267, 8192 x 8192 x 512 58 against 60, 4096 x 4096 x 1024 25 against 27, but 16383 x 2056 x 640 49 against 39,
// 16383 x 520 x 2176 36 against 33, 16384 x 512 x 2048 34 against 23, 307200 x 256 x 256 59 against 55.
// The sum is split where a workgroup's share of the blocks (0.64 us each, 1.06 for fp32, half for 32 rows) and the joining kernel (2.3 us
// and 0.55 us per MB of partial sums) take less than the whole: 2056 x 520 x 16384 40 us against 84 in one, 512 x 512 x 4096 14 / 25, 128 x
// 128 x 8192 11 / 44, 16 x 4096 x 4096 8.5 / 13.3, but 1000 x 1000 x 1000 in two 13.8 / 10.3, 1000 x 1000 x 2048 in four 19 / 15.5.
struct Plan { int bm, bn, splits; long blocks; };
inline Plan plan_of(long M, long N, long K, bool wide, bool raw) {
  const long blocks = K / kBlock;
  const long big = (((M + 255) / 256) * ((N + 255) / 256) + 255) / 256, small = ((M + 127) / 128) * ((N + 127) / 128), over = small % 512;
  const long rounds10 = small / 512 * 10 + (over == 0 ? 0 : over <= 256 ? 6 : 10);
  if (!wide && !raw && blocks >= 4 && big * 18 < rounds10) return Plan{256, 256, 1, blocks};
  const int bm = M <= 32 ? 32 : 128;
  const long tiles = ((M + bm - 1) / bm) * ((N + 127) / 128);
  long most = tiles ? 512 / tiles : 1;                           // two workgroups per CU
  most = most < blocks / 4 ? most : blocks / 4;                  // of at least four blocks each
  const double block = (wide ? 1.06 : 0.64) * (bm == 32 ? 0.5 : 1.0), join = 2.2e-6 * M * N;
  Plan best{bm, 128, 1, blocks};
  double cost = block * blocks;
  for (long s = 2; s <= most; s = s < most && s * 2 > most ? most : s * 2) {
    const long per = (blocks + s - 1) / s, splits = (blocks + per - 1) / per;
    const double c = block * per + 2.3 + join * splits;
    if (c < cost) {
      cost = c;
      best = Plan{bm, 128, (int)splits, per};
    }
  }
  return best;
}

template <class E, class A>
int launch_gemm_fp8(GemmP p, float* workspace, hipStream_t s) {
  constexpr bool wide = E::kBytes == 4, raw = !std::is_same<A, void>::value;
  const Plan plan = plan_of(p.M, p.N, p.K, wide, raw);
  p.blocks_per_split = plan.blocks;
  p.partial = plan.splits > 1 ? workspace : nullptr;
  // as many workgroups as the card holds at once, each with every so manieth tile (a multiple of 8 apart)
  const long tiles = ((p.M + plan.bm - 1) / plan.bm) * ((p.N + plan.bn - 1) / plan.bn);
  const long places = plan.bm == 256 || p.K == 0 ? tiles : plan.bm == 128 ? 512 : 768;
  const dim3 grid((unsigned)(tiles < places ? tiles : places), (unsigned)plan.splits);
  if (plan.bm == 256) {
    if constexpr (!wide && !raw) hipLaunchKernelGGL((gemm_fp8_kernel<E, A, false, 256, 256, 2, 4>), grid, dim3(512), 0, s, p);
  } else if (plan.bm == 32) {
    hipLaunchKernelGGL((gemm_fp8_kernel<E, A, wide, 32, 128, 1, 4>), grid, dim3(256), 0, s, p);
  } else {
    hipLaunchKernelGGL((gemm_fp8_kernel<E, A, wide, 128, 128, 2, 2>), grid, dim3(256), 0, s, p);
  }
  if (plan.splits > 1)
    hipLaunchKernelGGL((join_splits_kernel<E>), dim3((unsigned)((p.M * ((p.N + 3) / 4) + 255) / 256)), dim3(256), 0, s, p, plan.splits);
  return check_launch("gemm_fp8");
}
template <class E> int launch_gemm_of(int a_type, const GemmP& p, float* workspace, hipStream_t s) {
  return a_type == OBJNERF_TYPE_FP8 ? launch_gemm_fp8<E, void>(p, workspace, s) : a_type == OBJNERF_TYPE_F32 ? launch_gemm_fp8<E, ElemF32>(p, workspace, s)
         : a_type == OBJNERF_TYPE_BF16 ? launch_gemm_fp8<E, ElemBf16>(p, workspace, s) : launch_gemm_fp8<E, ElemF16>(p, workspace, s);
}

constexpr int64_t kMaxSize = 1ll << 31, kMaxK = 1ll << 26;     // 32 rows of kMaxK bytes: 32-bit offsets in a wave's copies

}  // namespace
}  // namespace objnerf

using namespace objnerf;

extern "C" {

int64_t objnerf_fp8_quantize_workspace_floats(int64_t rows, int64_t cols) { return rows > 0 && cols > 0 ? blocks_of(rows) * cols : 0; }

int objnerf_fp8_quantize(const objnerf_fp8_quantize_args* a, void* stream) {
  if (!a) return set_error(-1, "fp8_quantize: no arguments");
  if (a->rows < 0 || a->cols < 0 || a->rows >= kMaxSize || a->cols >= kMaxSize || (a->rows && a->cols > (1ll << 40) / a->rows))
    return set_error(-1, "fp8_quantize: bad sizes (rows, cols < 2^31, rows * cols <= 2^40)");
  if (!label_type_ok(a->type)) return set_error(-1, "fp8_quantize: unknown element type");
  if (a->block_rows != 1 && a->block_rows != kBlock) return set_error(-1, "fp8_quantize: blocks have 1 or 128 rows");
  if (a->x_stride < 0) return set_error(-1, "fp8_quantize: bad stride");
  if ((!a->values) != (!a->scales) || (!a->values_t) != (!a->scales_t) || (!a->values && !a->values_t))
    return set_error(-1, "fp8_quantize: values and scales belong together, and one form at least is asked for");
  if (a->column_sums && !a->workspace) return set_error(-1, "fp8_quantize: column sums need a workspace");
  if (((uintptr_t)a->values | (uintptr_t)a->values_t) & 15 || ((uintptr_t)a->scales | (uintptr_t)a->scales_t) & 3)
    return set_error(-1, "fp8_quantize: values must be 16-byte, scales 4-byte aligned");
  if (a->rows == 0 || a->cols == 0) return a->column_sums && a->cols ? set_error(-1, "fp8_quantize: column sums of no rows") : 0;
  if (!a->x) return set_error(-1, "fp8_quantize: a needed buffer is missing");
  QuantP p;
  p.rows = a->rows; p.cols = a->cols; p.x = a->x; p.ldx = a->x_stride;
  p.q = a->values; p.scale = a->scales; p.qt = a->values_t; p.scale_t = a->scales_t;
  p.part = a->column_sums ? a->workspace : nullptr;
  hipStream_t s = (hipStream_t)stream;
  const bool square = a->block_rows == kBlock;
  return a->type == OBJNERF_TYPE_F32 ? launch_quantize<ElemF32>(p, square, a->column_sums, s)
         : a->type == OBJNERF_TYPE_BF16 ? launch_quantize<ElemBf16>(p, square, a->column_sums, s)
                                        : launch_quantize<ElemF16>(p, square, a->column_sums, s);
}

int64_t objnerf_gemm_fp8_workspace_floats(int64_t M, int64_t N, int64_t K, int a_type, int c_type) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const Plan plan = plan_of(M, N, K, c_type == OBJNERF_TYPE_F32, a_type != OBJNERF_TYPE_FP8);
  return plan.splits > 1 ? plan.splits * M * N : 0;
}

int objnerf_gemm_fp8(const objnerf_gemm_fp8_args* a, void* stream) {
  if (!a) return set_error(-1, "gemm_fp8: no arguments");
  if (a->M < 0 || a->N < 0 || a->K < 0 || a->M >= kMaxSize || a->N >= kMaxSize || a->K > kMaxK || a->K % kBlock)
    return set_error(-1, "gemm_fp8: bad sizes (M, N < 2^31, K <= 2^26, K a multiple of 128)");
  const bool raw = a->a_type != OBJNERF_TYPE_FP8;
  if (!label_type_ok(a->c_type) || (raw && !label_type_ok(a->a_type))) return set_error(-1, "gemm_fp8: unknown element type");
  if (raw && (a->a_cols <= a->K - kBlock || a->a_cols > a->K)) return set_error(-1, "gemm_fp8: K is a_cols filled up to whole blocks");
  if (a->K && ((raw ? a->a_stride < 0 : a->a_stride < a->K || a->a_stride % 16 || a->a_stride > kMaxK) || a->b_stride < a->K || a->b_stride % 16 || a->b_stride > kMaxK))
    return set_error(-1, "gemm_fp8: bad strides (8-bit operands: multiples of 16, at least K, at most 2^26)");
  if (a->c_stride < a->N) return set_error(-1, "gemm_fp8: bad strides (c: at least N)");
  const int64_t nb = a->K / kBlock;
  if (a->K && ((!raw && (a->a_scale_stride < nb || a->a_scale_stride % 4)) || a->b_scale_stride < nb || a->b_scale_stride % 4))
    return set_error(-1, "gemm_fp8: bad scale strides (multiples of 4, at least K / 128)");
  if (((raw ? 0 : (uintptr_t)a->a) | (uintptr_t)a->b) & 15 || ((raw ? 0 : (uintptr_t)a->a_scale) | (uintptr_t)a->b_scale) & 3)
    return set_error(-1, "gemm_fp8: 8-bit operands must be 16-byte, scales 4-byte aligned");
  if (a->M == 0 || a->N == 0) return 0;
  if (((a->M + 31) / 32) > (1 << 30) / ((a->N + 127) / 128)) return set_error(-1, "gemm_fp8: more than 2^30 tiles");
  if (a->K == 0 && ((a->M + 31) / 32) * ((a->N + 127) / 128) >= 1 << 22) return set_error(-1, "gemm_fp8: a sum of nothing over more than 2^22 tiles");
  if (!a->c || (a->K && (!a->a || !a->b || (!raw && !a->a_scale) || !a->b_scale))) return set_error(-1, "gemm_fp8: a needed buffer is missing");
  if (objnerf_gemm_fp8_workspace_floats(a->M, a->N, a->K, a->a_type, a->c_type) && !a->workspace) return set_error(-1, "gemm_fp8: a workspace is needed");
  GemmP p;
  p.M = a->M; p.N = a->N; p.K = a->K;
  p.a = static_cast<const uint8_t*>(a->a); p.lda = a->a_stride; p.sa = a->a_scale; p.ldsa = a->a_scale_stride; p.cols = a->a_cols;
  p.b = a->b; p.ldb = a->b_stride; p.sb = a->b_scale; p.ldsb = a->b_scale_stride;
  p.bias = a->bias; p.leaky = a->leaky;
  p.c = a->c; p.ldc = a->c_stride;
  p.partial = nullptr; p.blocks_per_split = 0;
  hipStream_t s = (hipStream_t)stream;
  return a->c_type == OBJNERF_TYPE_F32 ? launch_gemm_of<ElemF32>(a->a_type, p, a->workspace, s)
         : a->c_type == OBJNERF_TYPE_BF16 ? launch_gemm_of<ElemBf16>(a->a_type, p, a->workspace, s) : launch_gemm_of<ElemF16>(a->a_type, p, a->workspace, s);
}

}  // extern "C"
