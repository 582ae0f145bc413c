// Arguments and layout of the low-rank adapter kernels (jma_adapters.hip), shared with the host runtime
// (jma_runtime_adapters.inc) and the CPU checks (tests/hostsim/launch_stubs.cpp). Plain C++: no HIP types.
#pragma once

#include <stdint.h>

#include <algorithm>

#include "jma_plan.h"

namespace jma {

constexpr uint32_t kMaxRank = 256;
constexpr uint32_t kNoAdapter = 0xFFFFFFFFu;
constexpr uint32_t kAdapterF32 = 0, kAdapterF16 = 1, kAdapterBF16 = 2;

JMA_HD uint32_t adapter_elem(uint32_t dtype) { return dtype == kAdapterF32 ? 4u : 2u; }
// Ranks are stored rounded up to 16 with zeros: A [rank16][cols], and B, whose products read eight ranks
// of neighbouring outputs, [rank16 / 8][outs][8].
JMA_HD uint32_t adapter_rank16(uint32_t rank) { return (rank + 15u) & ~15u; }
JMA_HD uint64_t adapter_b_index(uint64_t out, uint32_t r, uint32_t outs) {
  return ((uint64_t)(r / 8) * outs + out) * 8 + r % 8;
}

// `rows` rows from row0 on, adapter at element offsets a_at, b_at of the weights (rank16 0: none).
struct AdapterRun {
  uint32_t rows, row0, rank16;
  uint32_t block0;  // blocks of kUpRows rows of the launch's runs before this one
  float scale;
  uint64_t a_at, b_at;
};
constexpr uint32_t kMaxRuns = 96;  // runs of rows one launch takes in its kernel arguments

struct AdapterArgs {
  const void* a;       // the adapters' A and B weights
  const void* b;
  const float* x;      // [rows][cols]
  const float* base;   // [rows][outs], may be out; null: zero
  float* out;
  float* down;         // scratch [rows][splits][max_rank16] of the two-launch form
  uint32_t dtype, cols, outs, max_rank16;
  uint32_t splits, cols_per_split;  // pieces of the columns in the two-launch form
  uint32_t row_block;               // rows of one workgroup in the one-launch form
  uint32_t max_rows, runs, blocks;  // blocks: of kUpRows rows, of all runs
  AdapterRun run[kMaxRuns];
};
static_assert(sizeof(AdapterArgs) <= 4096, "kernel arguments exceed their limit");

struct AdapterLoadArgs {
  const void* a;  // [rank][cols]
  const void* b;  // [outs][rank]
  void* a_to;
  void* b_to;
  uint32_t dtype, rank, cols, outs;
};

// Outputs of a workgroup of the one-launch form, and the LDS floats its input rows may take.
constexpr uint32_t kFewOuts = 512, kFewFloats = 14336;
// Rows one workgroup takes in the one-launch form (0: the columns do not fit).
JMA_HD uint32_t adapter_few_rows(uint32_t cols) {
  const uint32_t fit = kFewFloats / cols;
  return fit < 4u ? fit : 4u;
}
// Rows and outputs of a workgroup's tile in the two-launch form.
constexpr uint32_t kDownRows = 16, kUpRows = 16, kUpOuts = 128;
// Pieces of the columns: as many as keep the first product's workgroups (one a compute unit) in one round,
// at least 512 columns each. row_blocks: of kDownRows rows.
inline uint32_t adapter_splits(uint32_t cols, uint64_t row_blocks, uint32_t cus) {
  const uint64_t want = cus / std::max<uint64_t>(row_blocks, 1);
  return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>({want, 16ull, std::max(1u, cols / 512)}));
}

}  // namespace jma
