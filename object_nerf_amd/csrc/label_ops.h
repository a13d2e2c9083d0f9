// label_ops.h -- what the label operators (label_loss.hip, label_sample.hip, label_fp8.hip) share: the element types of a row of
// logits, 16-byte pieces of it, and reductions over the lanes that hold a row.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>
#include "../../include/objnerf_hip.h"

namespace objnerf {

// A launch holds fewer than 2^32 threads in each dimension: workgroups past 2^20 go into the second one (at most 2^11 of them, for 2^31
// rows).  The last line of workgroups is not full: a kernel returns, or writes nothing, for a number behind the end.
constexpr int kGridLine = 20;
inline dim3 grid_of(long workgroups) {
  const long lines = ((workgroups - 1) >> kGridLine) + 1;
  return dim3((unsigned)(lines > 1 ? 1l << kGridLine : workgroups), (unsigned)lines);
}
__device__ __forceinline__ long workgroup() { return ((long)blockIdx.y << kGridLine) + blockIdx.x; }

using u32x4 = __attribute__((ext_vector_type(4))) unsigned;
// rows of 2-byte elements start at any even address: gfx950 takes a 16-byte global access at any element's address
typedef u32x4 u32x4e __attribute__((aligned(2)));
using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
using f16x2 = __attribute__((ext_vector_type(2))) _Float16;
using f32v2 = __attribute__((ext_vector_type(2))) float;

struct ElemF32 {
  static constexpr int kBytes = 4, kVec = 4;
  static __device__ __forceinline__ void unpack(u32x4 r, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(r[i]);
  }
  static __device__ __forceinline__ u32x4 pack(const float* x) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(x[i]);
    return r;
  }
  static __device__ __forceinline__ float load(const void* p, long i) { return static_cast<const float*>(p)[i]; }
  static __device__ __forceinline__ void store(void* p, long i, float v) { static_cast<float*>(p)[i] = v; }
};
struct ElemBf16 {
  static constexpr int kBytes = 2, kVec = 8;
  static __device__ __forceinline__ void unpack(u32x4 r, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(r[i] << 16); x[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u); }
  }
  static __device__ __forceinline__ u32x4 pack(const float* x) {       // one rounding, to nearest even
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(unsigned, __builtin_convertvector((f32v2){x[2 * i], x[2 * i + 1]}, bf16x2));
    return r;
  }
  static __device__ __forceinline__ float load(const void* p, long i) { return __uint_as_float((unsigned)static_cast<const uint16_t*>(p)[i] << 16); }
  static __device__ __forceinline__ void store(void* p, long i, float v) { static_cast<__bf16*>(p)[i] = (__bf16)v; }
};
struct ElemF16 {
  static constexpr int kBytes = 2, kVec = 8;
  static __device__ __forceinline__ void unpack(u32x4 r, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned w = r[i];            // a copy: __builtin_bit_cast of a vector's element takes element 0 on this compiler
      const f16x2 h = __builtin_bit_cast(f16x2, w);
      x[2 * i] = (float)h[0];
      x[2 * i + 1] = (float)h[1];
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float* x) {       // one rounding, to nearest even
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(unsigned, __builtin_convertvector((f32v2){x[2 * i], x[2 * i + 1]}, f16x2));
    return r;
  }
  static __device__ __forceinline__ float load(const void* p, long i) { return (float)static_cast<const _Float16*>(p)[i]; }
  static __device__ __forceinline__ void store(void* p, long i, float v) { static_cast<_Float16*>(p)[i] = (_Float16)v; }
};

__device__ __forceinline__ u32x4 load16(const void* p, long byte) { return *reinterpret_cast<const u32x4e*>(static_cast<const char*>(p) + byte); }
__device__ __forceinline__ void store16(void* p, long byte, u32x4 v) { *reinterpret_cast<u32x4e*>(static_cast<char*>(p) + byte) = v; }

// an element of a small side tensor whose type is known at run time only (OBJNERF_TYPE_*)
__device__ __forceinline__ float load_any(const void* p, long i, int type) {
  return type == OBJNERF_TYPE_F32 ? ElemF32::load(p, i) : type == OBJNERF_TYPE_BF16 ? ElemBf16::load(p, i) : ElemF16::load(p, i);
}

// ---- reductions over 16 or 64 lanes, every lane getting the same bits: DPP / row-swap steps, each of which adds the two halves of
// a symmetric exchange (a + b and b + a round alike) ----
struct OpSum { template <class T> static __device__ __forceinline__ T f(T a, T b) { return a + b; } };
struct OpMax {
  static __device__ __forceinline__ float f(float a, float b) { return fmaxf(a, b); }
  template <class T> static __device__ __forceinline__ T f(T a, T b) { return a > b ? a : b; }
};
struct OpMin { template <class T> static __device__ __forceinline__ T f(T a, T b) { return a < b ? a : b; } };

template <int CTRL> __device__ __forceinline__ unsigned dpp_u32(unsigned v) {
  return (unsigned)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);
}
// CTRL of the steps inside a row of 16: lanes xor 1, xor 2 (quad_perm), then quads (half mirror), then halves (mirror)
template <int CTRL> __device__ __forceinline__ float lane_step(float v) { return __uint_as_float(dpp_u32<CTRL>(__float_as_uint(v))); }
template <int CTRL> __device__ __forceinline__ unsigned lane_step(unsigned v) { return dpp_u32<CTRL>(v); }
template <int CTRL> __device__ __forceinline__ uint64_t lane_step(uint64_t v) {
  return ((uint64_t)dpp_u32<CTRL>((unsigned)(v >> 32)) << 32) | dpp_u32<CTRL>((unsigned)v);
}
// the two rows (ROW32 false: neighbouring rows of 16; true: halves of 32) that a step joins, one in each result, for every lane
template <bool ROW32> __device__ __forceinline__ void rows_of(unsigned v, unsigned& a, unsigned& b) {
  const auto r = ROW32 ? __builtin_amdgcn_permlane32_swap(v, v, false, false) : __builtin_amdgcn_permlane16_swap(v, v, false, false);
  a = r[0];
  b = r[1];
}
template <class OP, bool ROW32> __device__ __forceinline__ float join_rows(float v) {
  unsigned a, b;
  rows_of<ROW32>(__float_as_uint(v), a, b);
  return OP::f(__uint_as_float(a), __uint_as_float(b));
}
template <class OP, bool ROW32> __device__ __forceinline__ unsigned join_rows(unsigned v) {
  unsigned a, b;
  rows_of<ROW32>(v, a, b);
  return OP::f(a, b);
}
template <class OP, bool ROW32> __device__ __forceinline__ uint64_t join_rows(uint64_t v) {
  unsigned a, b, c, d;
  rows_of<ROW32>((unsigned)v, a, b);
  rows_of<ROW32>((unsigned)(v >> 32), c, d);
  return OP::f(((uint64_t)c << 32) | a, ((uint64_t)d << 32) | b);
}
template <int G, class OP, class T> __device__ __forceinline__ T lanes_reduce(T v) {
  static_assert(G == 16 || G == 64, "a row of a wave or the wave");
  v = OP::f(v, lane_step<0xB1>(v));
  v = OP::f(v, lane_step<0x4E>(v));
  v = OP::f(v, lane_step<0x141>(v));
  v = OP::f(v, lane_step<0x140>(v));
  if constexpr (G == 64) {
    v = join_rows<OP, false>(v);
    v = join_rows<OP, true>(v);
  }
  return v;
}

// ---- argument checks that the entry points share ----
inline bool label_type_ok(int type) { return type == OBJNERF_TYPE_F32 || type == OBJNERF_TYPE_BF16 || type == OBJNERF_TYPE_F16; }
inline int label_type_bytes(int type) { return type == OBJNERF_TYPE_F32 ? 4 : 2; }

}  // namespace objnerf
