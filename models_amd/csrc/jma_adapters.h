// Arguments and layout of the low-rank adapter kernels (jma_adapters.hip), shared with the host runtime
// (jma_runtime_adapters.inc) and the CPU checks (tests/paged_check.cpp). Plain C++: no HIP types.
#pragma once

#include <stdint.h>

#include <algorithm>

#include "jma_plan.h"

namespace jma {

constexpr uint32_t kMaxRuns = 128;      // runs of rows one launch takes in its kernel arguments
constexpr uint32_t kMaxRank = 256;
constexpr uint32_t kNoAdapter = 0xFFFFFFFFu;
constexpr uint32_t kAdapterF32 = 0, kAdapterF16 = 1, kAdapterBF16 = 2;

JMA_HD uint32_t adapter_elem(uint32_t dtype) { return dtype == kAdapterF32 ? 4u : 2u; }
// Ranks are stored rounded up to 16 with zeros: A [rank16][cols], B [outs][rank16].
JMA_HD uint32_t adapter_rank16(uint32_t rank) { return (rank + 15u) & ~15u; }

// `rows` rows from row0 on, adapter at element offset `at` of the weights (rank16 0: none).
struct AdapterRun {
  uint32_t rows, row0, rank16;
  float scale;
  uint64_t a_at, b_at;
};

struct AdapterArgs {
  const void* a;       // the adapters' A and B weights
  const void* b;
  const float* x;      // [rows][cols]
  const float* base;   // [rows][outs], may be out; null: zero
  float* out;
  float* down;         // scratch [rows][splits][max_rank16]
  uint32_t dtype, cols, outs, max_rank16, splits, cols_per_split, max_rows, runs;
  AdapterRun run[kMaxRuns - 32];
};
constexpr uint32_t kRunsPerLaunch = kMaxRuns - 32;
static_assert(sizeof(AdapterArgs) <= 4096, "kernel arguments exceed their limit");

struct AdapterLoadArgs {
  const void* a;  // [rank][cols]
  const void* b;  // [outs][rank]
  void* a_to;     // [rank16][cols]
  void* b_to;     // [outs][rank16]
  uint32_t dtype, rank, cols, outs;
};

// Columns one workgroup of the first product takes: at least 256, at most 8 pieces a row.
inline uint32_t adapter_splits(uint32_t cols) { return std::max(1u, std::min(8u, cols / 256)); }

}  // namespace jma
