// label_fp8.hip -- products in 8-bit floating point (OCP e4m3) with a scale for each block of 128, and the rounding to that form.
//
//   Q(x): blocks of 128 consecutive columns of a row (or of 128 x 128); scale s = the smallest power of two with
//         max|block| / s <= 448, held as the byte 127 + log2 s; element = e4m3(x / s), to nearest even
//   C[m][n] = sum_k a[m][k] b[n][k] (+ bias[n]) (LeakyReLU)
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
// C in 16 bits takes it.  C in fp32 does not: its operands are widened to bf16 in registers (exact: 4 bits and a power of two) and
// multiplied by the bf16 instruction at half the rate, which keeps fp32 sums (1.2e-8).
//
// Layout: values (R, C') with C' = C filled up to whole blocks with zeros; scales (R, B') bytes, one per row and block, B' = the
// number of blocks filled up to a multiple of 4 (with 127): one aligned dword holds four blocks' scales, the instruction's op_sel
// picks the byte.  Blocks of 128 x 128 repeat their scale in 128 rows: a 128th of the values' bytes buys one form for all.
#include "host_api.h"
#include "label_ops.h"

namespace objnerf {
namespace {

constexpr int kBlock = 128;
using i32x8 = __attribute__((ext_vector_type(8))) int;
using f32x4 = __attribute__((ext_vector_type(4))) float;

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

// eight consecutive columns of a row; what lies behind its end is 0
template <class E>
__device__ __forceinline__ void load8(const char* row, long c, long cols, float* x) {
  if (c + 8 <= cols) {
#pragma unroll
    for (int h = 0; h < 8 / E::kVec; ++h) E::unpack(load16(row, (c + h * E::kVec) * E::kBytes), x + h * E::kVec);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = c + i < cols ? E::load(row, c + i) : 0.f;
  }
}

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
  const long block = (long)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int l = threadIdx.x & 15;
  const bool in = block < p.rows * kb;
  const long row = in ? block / kb : 0, b = in ? block - row * kb : 0;
  const char* xr = static_cast<const char*>(p.x) + row * p.ldx * E::kBytes;
  float x[8];
  load8<E>(xr, b * kBlock + l * 8, p.cols, x);
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
// columns 8 l .. 8 l + 7, so that a column's eight bytes of a thread are one 8-byte LDS write of the transposed tile.
constexpr int kPitch = 144;
template <class E, bool ROWS, bool TRANS, bool SQUARE>
__global__ void __launch_bounds__(256) quantize_tile_kernel(QuantP p) {
  __shared__ float col_max[16][kBlock];
  __shared__ unsigned col_byte[kBlock];
  __shared__ __align__(16) uint8_t tile[TRANS ? kBlock * kPitch : 16];
  const long kb = blocks_of(p.cols), sb = scale_stride(p.cols), mb = blocks_of(p.rows), sbt = scale_stride(p.rows);
  const long bc = blockIdx.x % kb, br = blockIdx.x / kb;
  const int g = threadIdx.x >> 4, l = threadIdx.x & 15;
  const long r0 = br * kBlock + g * 8, c0 = bc * kBlock + l * 8;
  float x[8][8];
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    if (r0 + s < p.rows) load8<E>(static_cast<const char*>(p.x) + (r0 + s) * p.ldx * E::kBytes, c0, p.cols, x[s]);
    else
#pragma unroll
      for (int i = 0; i < 8; ++i) x[s][i] = 0.f;
  }
  unsigned square_byte = 0;
  if (TRANS || SQUARE) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float a = 0.f;
#pragma unroll
      for (int s = 0; s < 8; ++s) a = fmaxf(a, finite_abs(x[s][i]));
      col_max[g][l * 8 + i] = a;
    }
    __syncthreads();
    if (threadIdx.x < kBlock) {
      float a = 0.f;
#pragma unroll
      for (int s = 0; s < 16; ++s) a = fmaxf(a, col_max[s][threadIdx.x]);
      col_byte[threadIdx.x] = SQUARE ? __float_as_uint(a) : scale_byte(a);
    }
    __syncthreads();
    if (SQUARE) {
      unsigned a = max(col_byte[threadIdx.x & 63], col_byte[64 + (threadIdx.x & 63)]);      // non-negative floats order as their bits
      square_byte = scale_byte(__uint_as_float(lanes_reduce<64, OpMax>(a)));
    }
  }
  if (ROWS) {
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      unsigned byte = square_byte;
      if (!SQUARE) {
        float a = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) a = fmaxf(a, finite_abs(x[s][i]));
        byte = scale_byte(lanes_reduce<16, OpMax>(a));
      }
      const float inv = inverse_scale(byte);
      const long row = r0 + s;
      if (row < p.rows) {
        uint2 o;
        o.x = fp8x4(x[s][0] * inv, x[s][1] * inv, x[s][2] * inv, x[s][3] * inv);
        o.y = fp8x4(x[s][4] * inv, x[s][5] * inv, x[s][6] * inv, x[s][7] * inv);
        *reinterpret_cast<uint2*>(p.q + row * kb * kBlock + c0) = o;
        if (l == 0) p.scale[row * sb + bc] = (uint8_t)byte;
        if (bc == kb - 1 && l > 0 && bc + l < sb) p.scale[row * sb + bc + l] = 127;
      }
    }
  }
  if (TRANS) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float inv = inverse_scale(SQUARE ? square_byte : col_byte[l * 8 + i]);
      uint2 o;
      o.x = fp8x4(x[0][i] * inv, x[1][i] * inv, x[2][i] * inv, x[3][i] * inv);
      o.y = fp8x4(x[4][i] * inv, x[5][i] * inv, x[6][i] * inv, x[7][i] * inv);
      *reinterpret_cast<uint2*>(&tile[(l * 8 + i) * kPitch + g * 8]) = o;
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
  if (p.part) {                                                  // sums of 8 rows in order, then of 16 threads in order
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float a = x[0][i];
#pragma unroll
      for (int s = 1; s < 8; ++s) a += x[s][i];
      col_max[g][l * 8 + i] = a;
    }
    __syncthreads();
    const long col = bc * kBlock + threadIdx.x;
    if (threadIdx.x < kBlock && col < p.cols) {
      float a = col_max[0][threadIdx.x];
#pragma unroll
      for (int s = 1; s < 16; ++s) a += col_max[s][threadIdx.x];
      p.part[br * p.cols + col] = a;
    }
  }
}

// column sums from the tiles' partial sums: 16 threads per column, each a run of row blocks in order, joined in order
__global__ void __launch_bounds__(256) join_sums_kernel(const float* __restrict__ part, long blocks, long cols, float* __restrict__ sum) {
  __shared__ float s[16][16];
  const int l = threadIdx.x & 15, g = threadIdx.x >> 4;
  const long col = (long)blockIdx.x * 16 + l;
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
    hipLaunchKernelGGL((quantize_rows_kernel<E>), dim3((unsigned)((p.rows * blocks_of(p.cols) + 15) / 16)), dim3(256), 0, s, p);
  } else {
    const dim3 grid((unsigned)tiles);
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
  if (sum) hipLaunchKernelGGL(join_sums_kernel, dim3((unsigned)((p.cols + 15) / 16)), dim3(256), 0, s, p.part, blocks_of(p.rows), p.cols, sum);
  return check_launch("fp8_quantize");
}

// ---- the product ----

struct GemmP {
  long M, N, K;                            // K: whole blocks
  const uint8_t* a; long lda; const uint8_t* sa; long ldsa;
  const uint8_t* b; long ldb; const uint8_t* sb; long ldsb;
  const float* bias;
  int leaky;
  void* c; long ldc;
};

using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;

__device__ __forceinline__ i32x8 fragment(const uint8_t* p) {
  const u32x4 lo = *reinterpret_cast<const u32x4*>(p), hi = *reinterpret_cast<const u32x4*>(p + 16);
  return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}
// 8 elements times their block's scale: exact (4 bits, and bf16 has fp32's exponents)
__device__ __forceinline__ bf16x8 widened(const uint8_t* p, float scale) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v.x, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v.x, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v.y, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v.y, scale, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ float scale_of(unsigned byte) { return __uint_as_float(byte << 23); }
template <int SEL> __device__ __forceinline__ f32x4 mfma(i32x8 a, i32x8 b, f32x4 c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, SEL, sa, SEL, sb);
}

// A workgroup of four waves per 64 x 64 of C, a wave per 16 rows of C; fragments straight from memory.  The instruction's "A" is b's rows
// and its "B" a's, so that a lane's four results are four neighbouring columns of one row of C.
template <class E, bool WIDE>
__global__ void __launch_bounds__(256) gemm_fp8_kernel(GemmP p) {
  const long nb = (p.N + 63) / 64;
  const long m0 = (blockIdx.x / nb) * 64 + (threadIdx.x >> 6) * 16, n0 = (blockIdx.x % nb) * 64;
  const int lane = threadIdx.x & 63, i = lane & 15, h = lane >> 4;
  const long m = min(m0 + i, p.M - 1);
  f32x4 acc[4] = {};
  for (long k = 0; k < p.K; k += kBlock) {
    const unsigned sa = p.sa[m * p.ldsa + k / kBlock];
    if constexpr (WIDE) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const bf16x8 fa = widened(p.a + m * p.lda + k + q * 32 + h * 8, scale_of(sa));
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const long n = min(n0 + t * 16 + i, p.N - 1);
          const bf16x8 fb = widened(p.b + n * p.ldb + k + q * 32 + h * 8, scale_of(p.sb[n * p.ldsb + k / kBlock]));
          acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb, fa, acc[t], 0, 0, 0);
        }
      }
    } else {
      const i32x8 fa = fragment(p.a + m * p.lda + k + h * 32);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const long n = min(n0 + t * 16 + i, p.N - 1);
        acc[t] = mfma<0>(fragment(p.b + n * p.ldb + k + h * 32), fa, acc[t], (int)p.sb[n * p.ldsb + k / kBlock], (int)sa);
      }
    }
  }
  if (m0 + i >= p.M) return;
  char* c = static_cast<char*>(p.c) + (m0 + i) * p.ldc * E::kBytes;
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const long n = n0 + t * 16 + h * 4 + r;
      if (n >= p.N) continue;
      float v = acc[t][r] + (p.bias ? p.bias[n] : 0.f);
      if (p.leaky) v = fmaxf(v, 0.01f * v);
      E::store(c, n, v);
    }
}

template <class E>
int launch_gemm_fp8(const GemmP& p, hipStream_t s) {
  const long tiles = ((p.M + 63) / 64) * ((p.N + 63) / 64);
  hipLaunchKernelGGL((gemm_fp8_kernel<E, E::kBytes == 4>), dim3((unsigned)tiles), dim3(256), 0, s, p);
  return check_launch("gemm_fp8");
}

constexpr int64_t kMaxSize = 1ll << 31;

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

int objnerf_gemm_fp8(const objnerf_gemm_fp8_args* a, void* stream) {
  if (!a) return set_error(-1, "gemm_fp8: no arguments");
  if (a->M < 0 || a->N < 0 || a->K < 0 || a->M >= kMaxSize || a->N >= kMaxSize || a->K >= kMaxSize || a->K % kBlock)
    return set_error(-1, "gemm_fp8: bad sizes (M, N, K < 2^31, K a multiple of 128)");
  if (!label_type_ok(a->c_type)) return set_error(-1, "gemm_fp8: unknown element type");
  if ((a->K && (a->a_stride < a->K || a->b_stride < a->K || a->a_stride % 16 || a->b_stride % 16)) || a->c_stride < a->N)
    return set_error(-1, "gemm_fp8: bad strides (operands: multiples of 16, at least K)");
  const int64_t nb = a->K / kBlock;
  if (a->K && (a->a_scale_stride < nb || a->b_scale_stride < nb || a->a_scale_stride % 4 || a->b_scale_stride % 4))
    return set_error(-1, "gemm_fp8: bad scale strides (multiples of 4, at least K / 128)");
  if (((uintptr_t)a->a | (uintptr_t)a->b) & 15 || ((uintptr_t)a->a_scale | (uintptr_t)a->b_scale) & 3)
    return set_error(-1, "gemm_fp8: operands must be 16-byte, scales 4-byte aligned");
  if (a->M == 0 || a->N == 0) return 0;
  if (((a->M + 63) / 64) > INT32_MAX / ((a->N + 63) / 64)) return set_error(-1, "gemm_fp8: more than 2^31 tiles");
  if (!a->c || (a->K && (!a->a || !a->b || !a->a_scale || !a->b_scale))) return set_error(-1, "gemm_fp8: a needed buffer is missing");
  GemmP p;
  p.M = a->M; p.N = a->N; p.K = a->K;
  p.a = a->a; p.lda = a->a_stride; p.sa = a->a_scale; p.ldsa = a->a_scale_stride;
  p.b = a->b; p.ldb = a->b_stride; p.sb = a->b_scale; p.ldsb = a->b_scale_stride;
  p.bias = a->bias; p.leaky = a->leaky;
  p.c = a->c; p.ldc = a->c_stride;
  hipStream_t s = (hipStream_t)stream;
  return a->c_type == OBJNERF_TYPE_F32 ? launch_gemm_fp8<ElemF32>(p, s)
         : a->c_type == OBJNERF_TYPE_BF16 ? launch_gemm_fp8<ElemBf16>(p, s) : launch_gemm_fp8<ElemF16>(p, s);
}

}  // extern "C"
