// Rows of a decoder's tensors in any of the three element types (sa_norm.hip, sa_embed.hip, sa_xent*.hip).

#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "sa_host.h"

namespace {

using namespace sa_host;

typedef __bf16 bf16_t;

constexpr int64_t LAUNCH_BLOCKS = 1 << 20;   // workgroups of a launch whose kernel strides over the rest

inline int64_t lm_elem_size(int dtype) { return dtype == SA_DTYPE_F32 ? 4 : dtype == SA_DTYPE_BF16 || dtype == SA_DTYPE_F16 ? 2 : 0; }

__device__ __forceinline__ float from16(uint32_t bits, int dtype) {
  return dtype == SA_DTYPE_BF16 ? __uint_as_float(bits << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}
__device__ __forceinline__ uint16_t to16(float x, int dtype) {   // round to nearest even
  return dtype == SA_DTYPE_BF16 ? __builtin_bit_cast(uint16_t, (bf16_t)x) : __builtin_bit_cast(uint16_t, (_Float16)x);
}

// Four elements of a row as a lane loads them, before they are needed as numbers. VEC: four neighbours from element e on
// (a 16- or 8-byte load); else elements e, e + gap, e + 2 gap, e + 3 gap, one load each, those from `width` on zero. The type is
// the same for the whole launch, so the branches on it are scalar, and a caller that fetches all it needs before it reads
// any has the loads in flight together.
struct Quad {
  uint32_t d[4];
};
template <bool VEC>
__device__ __forceinline__ Quad fetch(const void* row, int dtype, int e, int gap, int width) {
  Quad q;
#pragma unroll
  for (int j = 0; j < 4; ++j) q.d[j] = 0u;
  if constexpr (VEC) {
    if (e >= width) return q;
    if (dtype == SA_DTYPE_F32) {
      const uint4 v = *reinterpret_cast<const uint4*>((const float*)row + e);
      q.d[0] = v.x, q.d[1] = v.y, q.d[2] = v.z, q.d[3] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>((const uint16_t*)row + e);
      q.d[0] = v.x, q.d[1] = v.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = e + j * gap;
      if (i < width) q.d[j] = dtype == SA_DTYPE_F32 ? ((const uint32_t*)row)[i] : ((const uint16_t*)row)[i];
    }
  }
  return q;
}
template <bool VEC>
__device__ __forceinline__ void numbers(const Quad& q, int dtype, float (&x)[4]) {
  if (dtype == SA_DTYPE_F32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(q.d[j]);
  } else if constexpr (VEC) {
    if (dtype == SA_DTYPE_BF16) {
      x[0] = __uint_as_float(q.d[0] << 16), x[1] = __uint_as_float(q.d[0] & 0xffff0000u);
      x[2] = __uint_as_float(q.d[1] << 16), x[3] = __uint_as_float(q.d[1] & 0xffff0000u);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = from16((q.d[j >> 1] >> (16 * (j & 1))) & 0xffffu, SA_DTYPE_F16);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = from16(q.d[j], dtype);
  }
}
template <bool VEC>
__device__ __forceinline__ void put(void* row, int dtype, int e, int gap, int width, const float (&x)[4]) {
  if constexpr (VEC) {
    if (e >= width) return;
    if (dtype == SA_DTYPE_F32) {
      *reinterpret_cast<float4*>((float*)row + e) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
      uint2 v;
      v.x = to16(x[0], dtype) | ((uint32_t)to16(x[1], dtype) << 16);
      v.y = to16(x[2], dtype) | ((uint32_t)to16(x[3], dtype) << 16);
      *reinterpret_cast<uint2*>((uint16_t*)row + e) = v;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = e + j * gap;
      if (i >= width) continue;
      if (dtype == SA_DTYPE_F32) ((float*)row)[i] = x[j];
      else ((uint16_t*)row)[i] = to16(x[j], dtype);
    }
  }
}
// the number that storing x in `dtype` leaves
__device__ __forceinline__ float stored(float x, int dtype) { return dtype == SA_DTYPE_F32 ? x : from16(to16(x, dtype), dtype); }

__device__ __forceinline__ const void* row_of(const void* p, int64_t row, int64_t ld, int dtype) {
  return (const char*)p + row * ld * (dtype == SA_DTYPE_F32 ? 4 : 2);
}
__device__ __forceinline__ void* row_of(void* p, int64_t row, int64_t ld, int dtype) {
  return (char*)p + row * ld * (dtype == SA_DTYPE_F32 ? 4 : 2);
}

// Whether rows at p, ld elements apart, can be read and written four elements at a time (the width: a multiple of 4).
inline bool quads_ok(const void* p, int64_t ld, int dtype) {
  return !p || ((uintptr_t)p % (4 * lm_elem_size(dtype)) == 0 && ld % 4 == 0);
}

}  // namespace
