// gfx950 kernels of low-rank adapters beside a shared projection: out = base + scale B (A x), each run
// of rows with an adapter of its own.
//
//   adapter_few_kernel    runs of few rows, one launch: every workgroup forms all of A x for its rows
//   adapter_down_kernel   longer runs: A x on the matrix cores, split over the columns
//   adapter_up_kernel     base + scale B (A x) on the matrix cores
//
// Inputs, sums and outputs are 32-bit and weights exact, so the result is that of 32-bit arithmetic for
// every weight type (f16 weights of longer runs: inputs to 2^-22, below); sums are formed in a fixed order.
// A weight that is no finite number may make NaN of what 32-bit arithmetic makes infinite.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "jma_kernels.h"

namespace jma {
namespace {

typedef float float4_t __attribute__((ext_vector_type(4)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));
typedef uint32_t uint2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf8_t __attribute__((ext_vector_type(8)));

#define JMA_INL __attribute__((always_inline))

// N (4 or 8) weights as they are stored, and widened.
template <uint32_t kType, int N>
struct Raw {
  static constexpr int kWords = kType == kAdapterF32 ? N : N / 2;
  typedef uint32_t words_t __attribute__((ext_vector_type(kWords)));
  words_t w;
  __device__ __forceinline__ void load(const void* p, uint64_t at) {
    const char* q = (const char*)p + at * adapter_elem(kType);
    if constexpr (kWords == 8) {
      const uint4_t x = *(const uint4_t*)q, y = *(const uint4_t*)(q + 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = x[i], w[4 + i] = y[i];
    } else {
      w = *(const words_t*)q;
    }
  }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (kType == kAdapterF32) return __uint_as_float(w[i]);
    else if constexpr (kType == kAdapterBF16) return __uint_as_float(i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)(i & 1 ? w[i / 2] >> 16 : w[i / 2]));
  }
};

// The run that a block of rows belongs to: a grid of the runs' blocks one after another, none empty, so that
// workgroups spread evenly (three runs of 500 to 900 rows, a grid of the longest's blocks for each: some
// compute units got two workgroups, others none, 29 us for the first product instead of 18, in f32 products).
__device__ __forceinline__ const AdapterRun& run_of(const AdapterArgs& a, uint32_t block) {
  uint32_t lo = 0, hi = a.runs;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (a.run[mid].block0 <= block) lo = mid;
    else hi = mid;
  }
  return a.run[lo];
}

template <int kCtrl>
__device__ __forceinline__ float moved(float x) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), kCtrl, 0xF, 0xF, false));
}
// Sum over the wave's 64 lanes; every lane gets the same bits.
__device__ __forceinline__ float wave_sum(float x) {
  x += moved<0x128>(x);  // row_ror by 8, 4, 2, 1
  x += moved<0x124>(x);
  x += moved<0x122>(x);
  x += moved<0x121>(x);
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ uint32_t max_groups(uint32_t x) {  // over the lanes of a column of a 16-column product
  auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = max(r[0], r[1]);
  r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return max(r[0], r[1]);
}

// acc += W x over 64 columns: lane (g, c) holds columns 8g .. 8g+7 of either 32, of row c of x and of row
// c of each 16-row tile of W, whose stored type the matrix instructions take. f16: x is carried as two halves
// (x = hi + lo to 2^-22, or to 2^-39 of the 64 columns' largest), scaled by a power of two that puts that into
// [2^13, 2^14); bf16: as three pieces of 8 bits, exactly; f32, and where an x is no finite number: one f32
// product of four columns after another. 64 columns of 64 ranks: 1.8 us a pair of waves in f32, 0.2 in halves.
template <uint32_t kType, int kN>
__device__ __forceinline__ void products(const float (&x)[2][8], const Raw<kType, 8> (&w)[2][kN], float4_t (&acc)[kN]) {
  if constexpr (kType != kAdapterF32) {
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) bits = max(bits, __float_as_uint(x[i][e]) & 0x7FFFFFFFu);
    bits = max_groups(bits);
    if (__ballot(bits >= 0x7F800000u) == 0) {
      if constexpr (kType == kAdapterF16) {
        const int ex = max(bits != 0 ? __builtin_amdgcn_frexp_expf(__uint_as_float(bits)) : 0, -100);
        float4_t sum[kN] = {};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          half8_t hi, lo;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float y = __builtin_amdgcn_ldexpf(x[i][e], 14 - ex);
            hi[e] = (_Float16)y;
            lo[e] = (_Float16)(y - (float)hi[e]);
          }
#pragma unroll
          for (int n = 0; n < kN; ++n) sum[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, w[i][n].w), lo, sum[n], 0, 0, 0);
#pragma unroll
          for (int n = 0; n < kN; ++n) sum[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, w[i][n].w), hi, sum[n], 0, 0, 0);
        }
        const float factor = __builtin_amdgcn_ldexpf(1.0f, ex - 14);
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n][e] = fmaf(sum[n][e], factor, acc[n][e]);
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float rest[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) rest[e] = x[i][e];
#pragma unroll
          for (int piece = 0; piece < 3; ++piece) {
            uint4_t top;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
              const uint32_t a = __float_as_uint(rest[e]), b = __float_as_uint(rest[e + 1]);
              top[e / 2] = __builtin_amdgcn_perm(b, a, 0x07060302u);  // their upper halves
              rest[e] -= __uint_as_float(a & 0xFFFF0000u);
              rest[e + 1] -= __uint_as_float(b & 0xFFFF0000u);
            }
#pragma unroll
            for (int n = 0; n < kN; ++n)
              acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8_t, w[i][n].w), __builtin_bit_cast(bf8_t, top), acc[n], 0, 0, 0);
          }
        }
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int n = 0; n < kN; ++n) acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[i][n][e], x[i][e], acc[n], 0, 0, 0);
}

// Workgroup = (512 outputs, block of kRows rows, run). Every workgroup forms all of A x for its rows: A
// comes from the L2 for all but the first, and a second launch, which would have to wait for the first,
// costs more than reading it again (2048 columns and outputs: one row of rank 16 9.1 us as two launches,
// 5.5 as one; 64 rows of 40 adapters of ranks 8 to 64 24.7 and 11.0). A wave takes two ranks at a time, its lanes
// eight columns each of every 512; then a thread takes an output.
template <uint32_t kType, int kRows>
__global__ __launch_bounds__(512) void adapter_few_kernel(const AdapterArgs a) {
  const AdapterRun run = a.run[blockIdx.z];
  const uint32_t r0 = blockIdx.y * kRows;
  if (r0 >= run.rows) return;
  const uint32_t rows = min((uint32_t)kRows, run.rows - r0);
  extern __shared__ __attribute__((aligned(16))) float s_x[];  // [kRows][cols]
  __shared__ __attribute__((aligned(16))) float s_down[kRows][kMaxRank];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t o = blockIdx.x * kFewOuts + threadIdx.x;
  const uint64_t at = (uint64_t)(run.row0 + r0) * a.outs + o;
  if (run.rank16 != 0) {
    const float* x = a.x + (uint64_t)(run.row0 + r0) * a.cols;
    for (uint32_t i = threadIdx.x; i < rows * (a.cols / 4); i += 512) *(float4_t*)&s_x[4 * i] = *(const float4_t*)(x + 4 * i);
    __syncthreads();
    for (uint32_t r = 2 * wave; r < run.rank16; r += 16) {
      float sum[2][kRows] = {};
      auto take = [&](const Raw<kType, 8>& w0, const Raw<kType, 8>& w1, uint32_t c) JMA_INL {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          if (i > 0 && (uint32_t)i >= rows) continue;
          const float4_t u = *(const float4_t*)&s_x[i * a.cols + c], v = *(const float4_t*)&s_x[i * a.cols + c + 4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            sum[0][i] = fmaf(w0[e], u[e], sum[0][i]);
            sum[1][i] = fmaf(w1[e], u[e], sum[1][i]);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            sum[0][i] = fmaf(w0[4 + e], v[e], sum[0][i]);
            sum[1][i] = fmaf(w1[4 + e], v[e], sum[1][i]);
          }
        }
      };
      const uint64_t row = run.a_at + (uint64_t)r * a.cols;
      uint32_t c = 8 * lane;
      for (; c + 3 * 512 < a.cols; c += 4 * 512) {  // eight loads in flight
        Raw<kType, 8> w0[4], w1[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w0[i].load(a.a, row + c + 512 * i);
          w1[i].load(a.a, row + a.cols + c + 512 * i);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) take(w0[i], w1[i], c + 512 * i);
      }
      for (; c < a.cols; c += 512) {
        Raw<kType, 8> w0, w1;
        w0.load(a.a, row + c);
        w1.load(a.a, row + a.cols + c);
        take(w0, w1, c);
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const float d0 = wave_sum(sum[0][i]), d1 = wave_sum(sum[1][i]);
        if (lane == 0) {
          s_down[i][r] = d0 * run.scale;
          s_down[i][r + 1] = d1 * run.scale;
        }
      }
    }
    __syncthreads();
  }
  if (o >= a.outs) return;
  float sum[kRows] = {};
  for (uint32_t r = 0; r < run.rank16; r += 16) {
    Raw<kType, 8> w0, w1;
    w0.load(a.b, run.b_at + adapter_b_index(o, r, a.outs));
    w1.load(a.b, run.b_at + adapter_b_index(o, r + 8, a.outs));
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sum[i] = fmaf(w0[e], s_down[i][r + e], sum[i]);
        sum[i] = fmaf(w1[e], s_down[i][r + 8 + e], sum[i]);
      }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i)
    if ((uint32_t)i < rows) a.out[at + (uint64_t)i * a.outs] = (a.base ? a.base[at + (uint64_t)i * a.outs] : 0.0f) + sum[i];
}

// Workgroup = (piece of the columns, 16 rows of a run): A x over that piece. Its eight waves take an
// eighth of the piece each and meet in LDS, so that few pieces, which the second launch has to sum, fill
// the device. Lane (g, c) holds eight neighbouring columns 8g .. 8g+7 of its row of either operand per 32, so
// both are read in wide loads, two steps of 64 ahead; ranks are taken 64 at a time, which is all of them for
// most adapters. 2000 rows by 4096 columns, ranks 48 and 64: 17 us for 33 MB of x and, out of the L2s, 64 MB of A,
// which every workgroup reads: four steps a wave do not hide the loads' latency. Workgroups of 32 rows
// read half of A and spill (22 us).
template <uint32_t kType>
__global__ __launch_bounds__(512) void adapter_down_kernel(const AdapterArgs a) {
  static_assert(kDownRows == kUpRows, "the runs' blocks are those of both products");
  const AdapterRun run = run_of(a, blockIdx.y);
  const uint32_t r0 = (blockIdx.y - run.block0) * kDownRows;
  if (run.rank16 == 0) return;
  const uint32_t rows = min(kDownRows, run.rows - r0);
  const uint32_t lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t c0 = blockIdx.x * a.cols_per_split, c1 = min(c0 + a.cols_per_split, a.cols);
  const uint32_t eighth = ((c1 - c0 + 7) / 8 + 31) / 32 * 32;
  const uint32_t w0 = min(c0 + wave * eighth, c1), w1 = min(w0 + eighth, c1);
  __shared__ __attribute__((aligned(16))) float s_part[8][4][64][4];  // [wave][rank tile][lane]
  // Rows behind the run's last repeat it; their columns of the product are not stored.
  const float* x = a.x + (uint64_t)(run.row0 + r0 + min(c16, rows - 1)) * a.cols;
  // `tiles` tiles of 16 ranks from rank0 on. (Known when compiled: a load under a branch would be waited for
  // where the branch ends.)
  auto take = [&](uint32_t rank0, auto count) JMA_INL {
    constexpr int kTiles = decltype(count)::value;
    struct Operands {  // two steps
      float4_t v[2][2];
      Raw<kType, 8> w[2][kTiles];
    };
    const uint64_t wrow = run.a_at + (uint64_t)(rank0 + c16) * a.cols;
    float4_t acc[kTiles] = {};
    // Columns past the piece's end read its first ones and count as zero.
    auto load = [&](Operands& y, uint32_t c) JMA_INL {
#pragma unroll
      for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t at = c + 32 * i + 8 * g < w1 ? c + 32 * i + 8 * g : c0;
        y.v[i][0] = *(const float4_t*)(x + at);
        y.v[i][1] = *(const float4_t*)(x + at + 4);
#pragma unroll
        for (int n = 0; n < kTiles; ++n) y.w[i][n].load(a.a, wrow + (uint64_t)16 * n * a.cols + at);
      }
    };
    auto step = [&](Operands& y, uint32_t c) JMA_INL {
      float v[2][8];
#pragma unroll
      for (uint32_t i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = y.v[i][e / 4][e % 4];
      if (c + 64 > w1) {
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
          const bool in = c + 32 * i + 8 * g < w1;
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] = in ? v[i][e] : 0.0f;
#pragma unroll
          for (int n = 0; n < kTiles; ++n)
#pragma unroll
            for (int e = 0; e < Raw<kType, 8>::kWords; ++e) y.w[i][n].w[e] = in ? y.w[i][n].w[e] : 0u;
        }
      }
      products<kType, kTiles>(v, y.w, acc);
    };
    Operands ya, yb;
    if (w0 < w1) {
      load(ya, w0);
      for (uint32_t c = w0;; c += 128) {
        load(yb, c + 64);
        step(ya, c);
        if (c + 64 >= w1) break;
        load(ya, c + 128);
        step(yb, c + 64);
        if (c + 128 >= w1) break;
      }
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < kTiles; ++n) *(float4_t*)s_part[wave][n][lane] = acc[n];
    __syncthreads();
    // Lane (g, c) of a tile holds ranks 4g .. 4g+3 of row c.
    if (threadIdx.x < kTiles * 64) {
      const uint32_t l = threadIdx.x % 64, n = threadIdx.x / 64, row = l & 15;
      float4_t sum = *(const float4_t*)s_part[0][n][l];
#pragma unroll
      for (int w = 1; w < 8; ++w) sum += *(const float4_t*)s_part[w][n][l];
      if (row < rows)
        *(float4_t*)&a.down[((uint64_t)(run.row0 + r0 + row) * a.splits + blockIdx.x) * a.max_rank16 + rank0 + 16 * n + 4 * (l >> 4)] = sum;
    }
  };
  for (uint32_t rank0 = 0; rank0 < run.rank16; rank0 += 64) {
    const uint32_t tiles = min(4u, (run.rank16 - rank0) / 16);
    if (tiles == 4) take(rank0, std::integral_constant<int, 4>{});
    else if (tiles == 3) take(rank0, std::integral_constant<int, 3>{});
    else if (tiles == 2) take(rank0, std::integral_constant<int, 2>{});
    else take(rank0, std::integral_constant<int, 1>{});
  }
}

// Workgroup = (128 outputs, 16 rows of a run): base + scale B (A x), the pieces of A x summed in order
// into LDS first. A wave takes 32 outputs; a product leaves lane (g, c) four neighbouring outputs of row c,
// which go through LDS, so that base is read (before all else) and out written in whole rows of 512 bytes.
// Bound by those, in rounds of six workgroups a compute unit (2000 rows by 4096 outputs: 17 us, 3.9 TB/s; in
// f32 products 20; tiles of 32 rows, whose registers leave fewer workgroups resident, 24).
template <uint32_t kType>
__global__ __launch_bounds__(256) void adapter_up_kernel(const AdapterArgs a) {
  const AdapterRun run = run_of(a, blockIdx.y);
  const uint32_t r0 = (blockIdx.y - run.block0) * kUpRows;
  const uint32_t rows = min(kUpRows, run.rows - r0);
  const uint32_t lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15, wave = threadIdx.x >> 6;
  const uint32_t o0 = blockIdx.x * kUpOuts;
  constexpr int kDownStride = 64 + 4, kOutStride = kUpOuts + 4;
  __shared__ __attribute__((aligned(16))) float s_mem[kUpRows * kOutStride];  // A x, then the outputs
  const bool wide = a.outs % 4 == 0;
  // This thread's pieces of four outputs.
  constexpr int kPieces = kUpRows * kUpOuts / 4 / 256;
  const uint32_t o = o0 + 4 * (threadIdx.x % (kUpOuts / 4)), row_of = threadIdx.x / (kUpOuts / 4);
  constexpr uint32_t kRowStep = 256 / (kUpOuts / 4);
  float4_t base[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    base[i] = float4_t{0.f, 0.f, 0.f, 0.f};
    const uint32_t row = row_of + kRowStep * i;
    if (a.base == nullptr || row >= rows || o >= a.outs) continue;
    const float* p = a.base + (uint64_t)(run.row0 + r0 + row) * a.outs + o;
    if (wide) base[i] = *(const float4_t*)p;
    else
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e)
        if (o + e < a.outs) base[i][e] = p[e];
  }
  static_assert(kUpRows == 16, "one tile of rows");
  float4_t acc[2] = {};  // [output tile]
  for (uint32_t rank0 = 0; rank0 < run.rank16; rank0 += 64) {
    const uint32_t ranks = min(64u, run.rank16 - rank0);
    Raw<kType, 8> w[2][2];
#pragma unroll
    for (uint32_t k = 0; k < 2; ++k)
#pragma unroll
      for (int n = 0; n < 2; ++n)
        w[k][n].load(a.b, run.b_at + adapter_b_index(min(o0 + 32 * wave + 16 * n + c16, a.outs - 1), rank0 + min(32 * k + 8 * g, ranks - 8), a.outs));
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < kUpRows * (ranks / 4); i += 256) {
      const uint32_t row = i / (ranks / 4), r = 4 * (i % (ranks / 4));
      float4_t sum = {0.f, 0.f, 0.f, 0.f};
      if (row < rows) {
        const float* p = a.down + (uint64_t)(run.row0 + r0 + row) * a.splits * a.max_rank16 + rank0 + r;
        for (uint32_t s = 0; s < a.splits; ++s) sum += *(const float4_t*)(p + (uint64_t)s * a.max_rank16);
      }
      *(float4_t*)&s_mem[row * kDownStride + r] = sum * run.scale;
    }
    __syncthreads();
    float d[2][8];
#pragma unroll
    for (uint32_t k = 0; k < 2; ++k) {
      const bool in = 32 * k + 8 * g < ranks;
      const float* p = &s_mem[c16 * kDownStride + (in ? 32 * k + 8 * g : 0)];
      const float4_t d0 = *(const float4_t*)p, d1 = *(const float4_t*)(p + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) d[k][e] = in ? d0[e] : 0.0f, d[k][4 + e] = in ? d1[e] : 0.0f;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < Raw<kType, 8>::kWords; ++e) w[k][n].w[e] = in ? w[k][n].w[e] : 0u;
    }
    products<kType, 2>(d, w, acc);
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < 2; ++n) *(float4_t*)&s_mem[c16 * kOutStride + 32 * wave + 16 * n + 4 * g] = acc[n];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const uint32_t row = row_of + kRowStep * i;
    if (row >= rows || o >= a.outs) continue;
    float* p = a.out + (uint64_t)(run.row0 + r0 + row) * a.outs + o;
    const float4_t y = base[i] + *(const float4_t*)&s_mem[row * kOutStride + (o - o0)];
    if (wide) *(float4_t*)p = y;
    else
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e)
        if (o + e < a.outs) p[e] = y[e];
  }
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
      const uint64_t j = i - na, o = j / r16;
      const uint32_t r = (uint32_t)(j % r16);
      ((T*)a.b_to)[adapter_b_index(o, r, a.outs)] = r < a.rank ? ((const T*)a.b)[o * a.rank + r] : (T)0;
    }
  }
}

template <typename F>
hipError_t by_type(uint32_t dtype, F&& f) {
  if (dtype == kAdapterF32) return f(std::integral_constant<uint32_t, kAdapterF32>{});
  if (dtype == kAdapterF16) return f(std::integral_constant<uint32_t, kAdapterF16>{});
  return f(std::integral_constant<uint32_t, kAdapterBF16>{});
}

}  // namespace

hipError_t launch_adapter_load(const AdapterLoadArgs& a, hipStream_t stream) {
  if (a.dtype == kAdapterF32) adapter_load_kernel<uint32_t><<<256, 256, 0, stream>>>(a);
  else adapter_load_kernel<uint16_t><<<256, 256, 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t launch_adapter_few(const AdapterArgs& a, hipStream_t stream) {
  const dim3 grid((a.outs + kFewOuts - 1) / kFewOuts, (a.max_rows + a.row_block - 1) / a.row_block, a.runs);
  const uint32_t lds = a.row_block * a.cols * 4;
  return by_type(a.dtype, [&](auto type) {
    constexpr uint32_t kType = decltype(type)::value;
    if (a.row_block == 1) adapter_few_kernel<kType, 1><<<grid, 512, lds, stream>>>(a);
    else if (a.row_block == 2) adapter_few_kernel<kType, 2><<<grid, 512, lds, stream>>>(a);
    else adapter_few_kernel<kType, 4><<<grid, 512, lds, stream>>>(a);
    return hipGetLastError();
  });
}

hipError_t launch_adapter_long(const AdapterArgs& a, hipStream_t stream) {
  const dim3 down(a.splits, a.blocks), up((a.outs + kUpOuts - 1) / kUpOuts, a.blocks);
  return by_type(a.dtype, [&](auto type) {
    constexpr uint32_t kType = decltype(type)::value;
    if (a.max_rank16) adapter_down_kernel<kType><<<down, 512, 0, stream>>>(a);
    adapter_up_kernel<kType><<<up, 256, 0, stream>>>(a);
    return hipGetLastError();
  });
}

}  // namespace jma
