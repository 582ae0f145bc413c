// Device helpers that the paged cache's kernels share (jma_paged.hip, jma_paged_prefill.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "jma_kernels.h"

namespace jma {
namespace {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef float float2_t __attribute__((ext_vector_type(2)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));

#define JMA_INL __attribute__((always_inline))

// Raises an error in the context's error word, in host memory: one byte per kind.
constexpr int kErrNonFinite = 0, kErrBadPage = 2;
__device__ __forceinline__ void report(int* err, int kind) {
  __hip_atomic_store((uint8_t*)err + kind, (uint8_t)1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

// x0*c - x1*s and x0*s + x1*c, every product and sum rounded on its own.
__device__ __forceinline__ void rotate_pair(float& x0, float& x1, float c, float s) {
#pragma clang fp contract(off)
  const float y0 = x0 * c - x1 * s, y1 = x0 * s + x1 * c;
  x0 = y0;
  x1 = y1;
}

// 1 / rms of a head in LDS, its sum of squares in order (TensorOps.rmsNorm); value: the norm without a
// weight (Gemma4Math.normalizeWithoutWeight).
template <int D>
__device__ __forceinline__ float head_scale(const float* x, float eps, bool value) {
#pragma clang fp contract(off)
  float ss = 0.0f;
#pragma unroll 4
  for (int e = 0; e < D; e += 4) {
    const float4_t v = *(const float4_t*)(x + e);
#pragma unroll
    for (int i = 0; i < 4; ++i) ss = ss + v[i] * v[i];
  }
  const double mean = (double)(ss / (float)D + eps);
  return value ? (float)(1.0 / sqrt(mean)) : 1.0f / (float)sqrt(mean);
}

// Pair j of a head in LDS, rotated with the factors of its position (RoPE row `at`).
__device__ __forceinline__ void rotate_in(float* x, uint32_t j, const PagedRotation& r, uint64_t at) {
  const uint32_t e0 = r.neox ? j : 2 * j, e1 = r.neox ? j + r.pairs : 2 * j + 1;
  float x0 = x[e0], x1 = x[e1];
  rotate_pair(x0, x1, r.cos_t[at * r.pairs + j], r.sin_t[at * r.pairs + j]);
  x[e0] = x0;
  x[e1] = x1;
}

// The query heads (rows 0 .. heads - 1 of s) of one token, and where `with_kv` its key and value of one kv
// head (rows kv0, kv0 + 1), normalised and rotated in LDS by the whole workgroup. Ends with a barrier.
template <int D, int kStride>
__device__ __forceinline__ void prepare_token(float* s, float* s_scale, uint32_t heads, uint32_t kv0, bool with_kv,
                                              const PagedRotation& r, uint32_t pos, uint32_t threads) {
  __syncthreads();
  const uint32_t tid = threadIdx.x, rows = heads + (with_kv ? 2u : 0u);
  auto row_of = [&](uint32_t i) JMA_INL { return i < heads ? i : kv0 + i - heads; };
  if (r.q_norm_w != nullptr || r.k_norm_w != nullptr || r.v_norm != 0) {
#pragma clang fp contract(off)
    if (tid < rows) {
      const bool value = tid == heads + 1;
      if (tid < heads ? r.q_norm_w != nullptr : value ? r.v_norm != 0 : r.k_norm_w != nullptr)
        s_scale[tid] = head_scale<D>(s + row_of(tid) * kStride, r.norm_eps, value);
    }
    __syncthreads();
    for (uint32_t i = tid; i < rows * D; i += threads) {
      const uint32_t row = i / D, e = i % D;
      const bool value = row == heads + 1;
      const float* w = row < heads ? r.q_norm_w : r.k_norm_w;
      if (value ? r.v_norm == 0 : w == nullptr) continue;
      float* x = s + row_of(row) * kStride + e;
      const float y = *x * s_scale[row];
      *x = value ? y : y * w[e];
    }
    __syncthreads();
  }
  if (r.cos_t != nullptr) {
    for (uint32_t i = tid; i < (heads + (with_kv ? 1u : 0u)) * r.pairs; i += threads)
      rotate_in(s + row_of(i / r.pairs) * kStride, i % r.pairs, r, pos);
    __syncthreads();
  }
}

__device__ __forceinline__ void swap16(float x, float& a, float& b) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  a = __uint_as_float(r[0]);
  b = __uint_as_float(r[1]);
}
__device__ __forceinline__ void swap32(float x, float& a, float& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  a = __uint_as_float(r[0]);
  b = __uint_as_float(r[1]);
}
// Over the two halves of a wave, which hold the same column of a 32-column product.
__device__ __forceinline__ float max_halves(float x) {
  float a, b;
  swap32(x, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float sum_halves(float x) {
  float a, b;
  swap32(x, a, b);
  return a + b;
}
// Over the four 16-lane groups, which hold the same column of a 16-column product.
__device__ __forceinline__ float max_groups(float x) {
  float a, b;
  swap16(x, a, b);
  return max_halves(fmaxf(a, b));
}
__device__ __forceinline__ float sum_groups(float x) {
  float a, b;
  swap16(x, a, b);
  return sum_halves(a + b);
}

// Partial states move between workgroups with 16-byte device-coherent accesses (sc1).
constexpr int kCoherent = 16;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t part_rsrc(float* p) {
  return __builtin_amdgcn_make_buffer_rsrc(p, 0, 0x7FFFFFF0, 0x00020000);
}
__device__ __forceinline__ void store_part(__amdgpu_buffer_rsrc_t rs, uint32_t at, const float4_t& x) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(uint4_t, x), rs, at, 0, kCoherent);
}
__device__ __forceinline__ float4_t load_part(__amdgpu_buffer_rsrc_t rs, uint32_t at) {
  return __builtin_bit_cast(float4_t, __builtin_amdgcn_raw_buffer_load_b128(rs, at, 0, kCoherent));
}

// The hi and lo f16 halves of x: x = hi + lo to 2^-22.
__device__ __forceinline__ void halves(float x, _Float16& hi, _Float16& lo) {
  hi = (_Float16)x;
  lo = (_Float16)(x - (float)hi);
}

// x minus the low (high) half of h, in one instruction.
__device__ __forceinline__ float minus_low(float x, half2_t h) {
  float y;
  asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[0,0,0] op_sel_hi:[1,0,0]" : "=v"(y) : "v"(h), "v"(x));
  return y;
}
__device__ __forceinline__ float minus_high(float x, half2_t h) {
  float y;
  asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(y) : "v"(h), "v"(x));
  return y;
}

// Nonzero where one of the halves is infinite or no number.
__device__ __forceinline__ uint32_t not_finite(const half8_t& x) {
  const uint4_t w = __builtin_bit_cast(uint4_t, x);
  uint32_t odd = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) odd |= ((w[i] & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
  return odd;
}
__device__ __forceinline__ uint32_t not_finite(const float4_t& x) {
  uint32_t odd = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) odd |= (__float_as_uint(x[i]) & 0x7F800000u) == 0x7F800000u ? 1u : 0u;
  return odd;
}
// Sets them to zero, and `is` to one in their place and zero elsewhere.
template <typename V>
__device__ __forceinline__ void split_finite(V& x, V& is) {
  constexpr int kN = sizeof(V) / sizeof(x[0]);
#pragma unroll
  for (int e = 0; e < kN; ++e) {
    const bool odd = !(fabsf((float)x[e]) < INFINITY);
    is[e] = odd ? 1.0f : 0.0f;
    x[e] = odd ? 0.0f : (float)x[e];
  }
}

}  // namespace
}  // namespace jma
