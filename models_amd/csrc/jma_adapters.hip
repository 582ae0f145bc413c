// gfx950 kernels of low-rank adapters beside a shared projection: out = base + scale B (A x), each run
// of rows with an adapter of its own.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "jma_kernels.h"

namespace jma {
namespace {

typedef float float4_t __attribute__((ext_vector_type(4)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));

#define JMA_INL __attribute__((always_inline))

// Rows of a run that share a workgroup's weight loads.
constexpr uint32_t kRowBlock = 8;

// Eight weights, widened exactly.
template <uint32_t kType>
__device__ __forceinline__ void load8(const void* p, uint64_t at, float (&w)[8]) {
  if constexpr (kType == kAdapterF32) {
    const float4_t x = *(const float4_t*)((const float*)p + at), y = *(const float4_t*)((const float*)p + at + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = x[e], w[4 + e] = y[e];
  } else if constexpr (kType == kAdapterF16) {
    typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
    const half8_t x = *(const half8_t*)((const _Float16*)p + at);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = (float)x[e];
  } else {
    const uint4_t x = *(const uint4_t*)((const uint16_t*)p + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[2 * e] = __uint_as_float(x[e] << 16);
      w[2 * e + 1] = __uint_as_float(x[e] & 0xFFFF0000u);
    }
  }
}

// Workgroup = (piece of the columns, block of a run's rows, run): A x over that piece, for every rank.
// A wave takes a rank at a time, its lanes eight columns each; sums are 32-bit, in a fixed tree.
template <uint32_t kType>
__global__ __launch_bounds__(256) void adapter_down_kernel(const AdapterArgs a) {
  const AdapterRun run = a.run[blockIdx.z];
  const uint32_t r0 = blockIdx.y * kRowBlock;
  if (run.rank16 == 0 || r0 >= run.rows) return;
  const uint32_t rows = min(kRowBlock, run.rows - r0);
  const uint32_t c0 = blockIdx.x * a.cols_per_split, c1 = min(c0 + a.cols_per_split, a.cols);
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float* x = a.x + (uint64_t)(run.row0 + r0) * a.cols;
  for (uint32_t r = wave; r < run.rank16; r += 4) {
    float sum[kRowBlock] = {};
    for (uint32_t c = c0 + 8 * lane; c < c1; c += 512) {
      float w[8];
      load8<kType>(a.a, run.a_at + (uint64_t)r * a.cols + c, w);
#pragma unroll
      for (uint32_t i = 0; i < kRowBlock; ++i) {
        if (i >= rows) continue;
        const float4_t u = *(const float4_t*)(x + (uint64_t)i * a.cols + c), v = *(const float4_t*)(x + (uint64_t)i * a.cols + c + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sum[i] = fmaf(w[e], u[e], sum[i]);
          sum[i] = fmaf(w[4 + e], v[e], sum[i]);
        }
      }
    }
#pragma unroll
    for (uint32_t i = 0; i < kRowBlock; ++i) {
      if (i >= rows) continue;
#pragma unroll
      for (int m = 32; m >= 1; m /= 2) sum[i] += __shfl_xor(sum[i], m);
      if (lane == 0) a.down[((uint64_t)(run.row0 + r0 + i) * a.splits + blockIdx.x) * a.max_rank16 + r] = sum[i];
    }
  }
}

// Workgroup = (256 outputs, block of a run's rows, run): base + scale B (A x), the pieces of A x summed
// in order.
template <uint32_t kType>
__global__ __launch_bounds__(256) void adapter_up_kernel(const AdapterArgs a) {
  const AdapterRun run = a.run[blockIdx.z];
  const uint32_t r0 = blockIdx.y * kRowBlock;
  if (r0 >= run.rows) return;
  const uint32_t rows = min(kRowBlock, run.rows - r0);
  __shared__ __attribute__((aligned(16))) float s_down[kRowBlock][kMaxRank];
  for (uint32_t i = threadIdx.x; i < rows * run.rank16; i += 256) {
    const uint32_t row = i / run.rank16, r = i % run.rank16;
    const float* p = a.down + (uint64_t)(run.row0 + r0 + row) * a.splits * a.max_rank16 + r;
    float sum = 0.0f;
    for (uint32_t s = 0; s < a.splits; ++s) sum += p[(uint64_t)s * a.max_rank16];
    s_down[row][r] = sum * run.scale;
  }
  __syncthreads();
  const uint32_t o = blockIdx.x * 256 + threadIdx.x;
  if (o >= a.outs) return;
  float sum[kRowBlock];
  const uint64_t at = (uint64_t)(run.row0 + r0) * a.outs + o;
#pragma unroll
  for (uint32_t i = 0; i < kRowBlock; ++i) sum[i] = 0.0f;
  for (uint32_t r = 0; r < run.rank16; r += 8) {
    float w[8];
    load8<kType>(a.b, run.b_at + (uint64_t)o * run.rank16 + r, w);
#pragma unroll
    for (uint32_t i = 0; i < kRowBlock; ++i)
      if (i < rows)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[i] = fmaf(w[e], s_down[i][r + e], sum[i]);
  }
#pragma unroll
  for (uint32_t i = 0; i < kRowBlock; ++i)
    if (i < rows) a.out[at + (uint64_t)i * a.outs] = (a.base ? a.base[at + (uint64_t)i * a.outs] : 0.0f) + sum[i];
}

// An adapter's weights into their stored form, the ranks behind its own zero.
template <typename T>
__global__ __launch_bounds__(256) void adapter_load_kernel(const AdapterLoadArgs a) {
  const uint32_t r16 = adapter_rank16(a.rank);
  const uint64_t na = (uint64_t)r16 * a.cols, nb = (uint64_t)a.outs * r16;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < na + nb; i += (uint64_t)gridDim.x * 256) {
    if (i < na) {
      ((T*)a.a_to)[i] = i / a.cols < a.rank ? ((const T*)a.a)[i] : (T)0;
    } else {
      const uint64_t j = i - na, o = j / r16, r = j % r16;
      ((T*)a.b_to)[j] = r < a.rank ? ((const T*)a.b)[o * a.rank + r] : (T)0;
    }
  }
}

}  // namespace

hipError_t launch_adapter_load(const AdapterLoadArgs& a, hipStream_t stream) {
  if (a.dtype == kAdapterF32) adapter_load_kernel<uint32_t><<<256, 256, 0, stream>>>(a);
  else adapter_load_kernel<uint16_t><<<256, 256, 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t launch_adapter_apply(const AdapterArgs& a, hipStream_t stream) {
  const uint32_t blocks = (a.max_rows + kRowBlock - 1) / kRowBlock;
  const dim3 down(a.splits, blocks, a.runs), up((a.outs + 255) / 256, blocks, a.runs);
  auto go = [&](auto type) {
    constexpr uint32_t kType = decltype(type)::value;
    adapter_down_kernel<kType><<<down, 256, 0, stream>>>(a);
    adapter_up_kernel<kType><<<up, 256, 0, stream>>>(a);
    return hipGetLastError();
  };
  if (a.dtype == kAdapterF32) return go(std::integral_constant<uint32_t, kAdapterF32>{});
  if (a.dtype == kAdapterF16) return go(std::integral_constant<uint32_t, kAdapterF16>{});
  return go(std::integral_constant<uint32_t, kAdapterBF16>{});
}

}  // namespace jma
