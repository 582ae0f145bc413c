// Arguments, layout and launch planning of the paged-cache kernels (jma_paged.hip), shared with the
// host runtime (jma_runtime_paged.inc) and the CPU checks (tests/hostsim/launch_stubs.cpp). Plain C++: no HIP
// types, so it also builds with g++ alone.
#pragma once

#include <stdint.h>

#include <algorithm>

#include "jma_plan.h"

namespace jma {

// Chunks of new tokens that one launch takes in its kernel arguments (more are split into several).
constexpr uint32_t kMaxChunks = 128;
// Slots of a storage tile, the unit a page is made of.
constexpr uint32_t kTileSlots = 32;
// Entries of a selected-page list that name no page.
constexpr uint32_t kNoPage = 0xFFFFFFFFu;

// One layer's pages. A page holds 2^page_log2 slots (32 to 256) of every kv head:
//   K       [page][kv head][slots / 32][d / W][32][W]  (panels of 64 bytes a row: W = 32 f16, 16 f32)
//   V       [page][kv head][slots / 32][d][32]         (values transposed, slots in order)
//   bounds  [page][kv head][2][d]                      (smallest, largest key element of the filled slots)
// A panel is what one matrix-core operand load reads (16 rows x 64 bytes) in one place; the
// transposed values are the other product's operand. Slot p % slots of page table[p / slots] of its
// sequence holds position p.
struct PagedView {
  void* k;
  void* v;
  void* bounds;           // null: the cache keeps none
  const uint32_t* table;  // [sequences][table_stride]
  uint32_t table_stride, pages, page_log2, hkv;
};

JMA_HD uint64_t paged_head_elems(uint32_t page_log2, uint32_t d) { return (uint64_t)d << page_log2; }
// Element of the layer's K (or V) storage where kv head `h`'s part of page `page` starts.
JMA_HD uint64_t paged_base(uint32_t page, uint32_t hkv, uint32_t h, uint32_t page_log2, uint32_t d) {
  return ((uint64_t)page * hkv + h) * paged_head_elems(page_log2, d);
}
JMA_HD uint32_t paged_k_index(uint32_t slot, uint32_t e, uint32_t d, bool f16) {
  const uint32_t w = f16 ? 32u : 16u;
  return (slot / kTileSlots) * kTileSlots * d + (e / w) * (kTileSlots * w) + (slot % kTileSlots) * w + e % w;
}
JMA_HD uint32_t paged_v_index(uint32_t slot, uint32_t e, uint32_t d) {
  return (slot / kTileSlots) * kTileSlots * d + e * kTileSlots + slot % kTileSlots;
}

// `rows` new tokens of sequence `seq` at positions start .. start + rows - 1; row0: their first row of
// the launch's q, k, v and out. An attention launch cuts the chunk's blocks of query rows into up to
// nsplit splits, whose states are items part0 + (block of the chunk) * nsplit + split.
struct PagedChunk {
  uint32_t seq, start, rows, row0, nsplit, part0;
  uint32_t block0;  // 16-column attention: blocks of rows of the launch's chunks before this one
};

// What new rows are made with: QK-norm, then RoPE.
struct PagedRotation {
  const float* cos_t;  // [max_positions][pairs]; null: no RoPE
  const float* sin_t;
  const float* q_norm_w;  // [d]; null: no norm of that side
  const float* k_norm_w;
  float norm_eps;
  uint32_t v_norm;  // 1: values are normalised without a weight
  uint32_t pairs, neox;
};

// Rows that a workgroup of the append kernel takes: an aligned run of slots. Of long heads fewer, whose rows
// and RoPE factors are then all in registers at once (heads of 256, 1000 rows: 12.3 us with 32 rows, 6 with 16).
JMA_HD constexpr uint32_t paged_append_rows(uint32_t d) { return d >= 128 ? 16 : 32; }
struct PagedAppendArgs {
  PagedView kv;
  const float* q;  // [rows][num_heads * d]; null: no query is rotated
  const float* k;  // [rows][hkv * d]
  const float* v;
  float* q_out;
  PagedRotation rot;
  uint32_t num_heads;
  uint32_t max_tiles;  // runs of slots (paged_append_rows) of the chunk with the most (the grid's x)
  uint32_t max_pages;  // pages of the chunk with the most (the bounds kernel's x)
  uint32_t chunks;
  PagedChunk c[kMaxChunks];
};

struct PagedAttendArgs {
  PagedView kv;
  const float* q;        // [rows][num_heads * d], rotated, or raw with k_new
  float* out;            // [rows][num_heads * d]
  const float* k_new;    // chunks of one row: raw keys and values [rows][hkv * d] that the launch appends; null:
  const float* v_new;    // the rows are appended already
  PagedRotation rot;
  int* err;
  float* part;           // [item][16][d + 4] partial states (acc, m, l) of split blocks
  uint32_t* tickets;     // [unit], zero between launches
  const uint32_t* pages; // selected pages [rows][hkv][budget], ascending, kNoPage behind; null: every page
  float scale;           // score scale x log2(e)
  uint32_t num_heads, group, window, budget;
  uint32_t head_groups;  // groups of at most 16 (prefill: 32) query heads of a kv head
  uint32_t rows_per_block;  // query rows of one workgroup
  uint32_t rows_per_stripe, heads_per_stripe;  // prefill: query rows and heads of a wave's 32 columns
  uint32_t max_blocks;   // row blocks of the chunk with the most
  uint32_t blocks;       // and of all chunks (16-column attention)
  uint32_t tiles_per_split, max_splits;
  uint32_t chunks;
  PagedChunk c[kMaxChunks];
};
static_assert(sizeof(PagedAttendArgs) <= 4096 && sizeof(PagedAppendArgs) <= 4096,
              "kernel arguments exceed their limit");

// Pages one workgroup of the selection scores.
constexpr uint32_t kSelectPages = 64;

struct PagedSelectArgs {
  PagedView kv;
  const float* q;      // rotated, or raw with `raw`
  PagedRotation rot;
  uint32_t raw;
  uint32_t* pages;     // out: [rows][hkv][budget]
  float* keys;         // scratch [block][row of the block][paged_row_keys]: scores in 32 bits, and behind them,
                       // where those are needed, in 64, as ordered integers
  float* maxima;       // scratch [block][max_wgs][4]: largest bound of a wave's pages
  uint32_t* tickets;   // [block], zero between launches; block = (chunk, row block, kv head)
  uint32_t num_heads, group, top, first, last, budget;
  uint32_t rows_per_block, max_blocks;  // query rows of a workgroup; row blocks of the chunk with the most
  uint32_t key_stride, max_wgs;  // pages of the row furthest back; workgroups a block may have
  uint32_t chunks;
  PagedChunk c[kMaxChunks];
};
static_assert(sizeof(PagedSelectArgs) <= 4096, "kernel arguments exceed their limit");

// Table entries written by one launch.
constexpr uint32_t kTableWrites = 448;
struct PagedTableArgs {
  uint32_t* table;
  uint32_t count;
  uint32_t at[kTableWrites], page[kTableWrites];
};
static_assert(sizeof(PagedTableArgs) <= 4096, "kernel arguments exceed their limit");

// Floats of one row's scores: 32 bits a page, to an even number, and 64 a page.
JMA_HD uint64_t paged_row_keys(uint32_t pages) { return ((pages + 1) & ~1u) + (uint64_t)2 * pages; }
// Query rows of a selection workgroup: its matrix product has 16 columns.
JMA_HD uint32_t select_rows(uint32_t group) { return group >= 16 ? 1u : 16u / group; }
// Floats of a group's queries that the selection kernel stages where it takes them raw.
constexpr uint32_t kSelectFloats = 8192;

inline bool paged_supported(uint32_t d) { return d == 32 || d == 64 || d == 128 || d == 256; }

// Waves of an attention workgroup, and the slots one wave takes at a step.
constexpr int paged_waves(int d) { return d >= 128 ? 4 : 8; }
JMA_HD uint32_t paged_step(bool f16) { return f16 ? 32u : 16u; }

// The steps (of paged_step slots) that a block of query rows at positions pos0 .. pos1 reads: all
// positions that any of its rows sees, or (budget > 0) the steps of its row's selected pages.
JMA_HD void paged_range(uint32_t pos0, uint32_t pos1, uint32_t window, uint32_t budget, uint32_t page_log2,
                        uint32_t step, uint32_t& t0, uint32_t& t1) {
  if (budget) {
    const uint32_t seen = (pos1 >> page_log2) + 1;
    t0 = 0;
    t1 = (budget < seen ? budget : seen) * ((1u << page_log2) / step);
  } else {
    t0 = first_visible(pos0, window) / step;
    t1 = pos1 / step + 1;
  }
}

// Split plan of one attention launch: every workgroup streams tiles_per_split steps, at least one a
// wave, raised until the launch is near `target` workgroups and no block needs more than kMaxSplits
// splits. Fills the chunks' nsplit and part0.
struct PagedPlan {
  uint32_t tiles_per_split = 0, max_splits = 1, max_blocks = 0, blocks = 0, rows_per_block = 1, head_groups = 1;
  uint64_t part_bytes = 0, ticket_bytes = 0;
};
inline PagedPlan plan_paged(PagedChunk* c, uint32_t chunks, uint32_t group, uint32_t hkv, uint32_t d, bool f16,
                            uint32_t window, uint32_t page_log2, uint32_t budget, uint32_t target) {
  PagedPlan p;
  const uint32_t step = paged_step(f16), waves = (uint32_t)paged_waves((int)d);
  p.head_groups = (group + kHeadSlots - 1) / kHeadSlots;
  p.rows_per_block = budget ? 1u : std::max(1u, (uint32_t)kHeadSlots / group);
  const uint64_t per = (uint64_t)hkv * p.head_groups;
  auto each = [&](uint32_t i, auto&& f) {  // the steps of every block of chunk i
    for (uint32_t r0 = 0; r0 < c[i].rows; r0 += p.rows_per_block) {
      uint32_t t0, t1;
      paged_range(c[i].start + r0, c[i].start + std::min(r0 + p.rows_per_block, c[i].rows) - 1, window, budget,
                  page_log2, step, t0, t1);
      f(t1 - t0);
    }
  };
  uint64_t total = 0;
  uint32_t longest = 1;
  for (uint32_t i = 0; i < chunks; ++i) {
    each(i, [&](uint32_t n) {
      total += n * per;
      longest = std::max(longest, n);
    });
    const uint32_t blocks = (c[i].rows + p.rows_per_block - 1) / p.rows_per_block;
    p.max_blocks = std::max(p.max_blocks, blocks);
    c[i].block0 = p.blocks;
    p.blocks += blocks;
  }
  uint64_t tps = std::max<uint64_t>(waves, (total + target - 1) / std::max(target, 1u));
  tps = std::max<uint64_t>(tps, (longest + kMaxSplits - 1) / kMaxSplits);
  p.tiles_per_split = (uint32_t)tps;
  uint64_t items = 0;
  for (uint32_t i = 0; i < chunks; ++i) {
    uint32_t most = 1;
    each(i, [&](uint32_t n) { most = std::max(most, (uint32_t)((n + tps - 1) / tps)); });
    c[i].nsplit = most;
    c[i].part0 = (uint32_t)items;
    if (most > 1) items += (uint64_t)((c[i].rows + p.rows_per_block - 1) / p.rows_per_block) * per * most;
    p.max_splits = std::max(p.max_splits, most);
  }
  if (p.max_splits > 1) {
    p.part_bytes = items * kHeadSlots * (d + 4) * 4;
    p.ticket_bytes = (uint64_t)p.blocks * per * 4;
  }
  return p;
}

// The prefill kernel: waves of a workgroup (32 columns each), storage tiles of a step, and floats of one
// workgroup's partial state: [wave][d / 8 words of O^T, then (m, l)][64 lanes] float4.
constexpr int kPrefillWaves = 4;
JMA_HD constexpr int paged_prefill_tiles(int d) { return d >= 256 ? 1 : 2; }
// Waves of one SIMD: what the registers of a wave (q and O^T of 32 columns) leave room for.
JMA_HD constexpr int paged_prefill_waves_per_simd(int d) { return d >= 256 ? 1 : d >= 128 ? 2 : d >= 64 ? 3 : 4; }
JMA_HD constexpr uint32_t paged_prefill_item(int d) { return (uint32_t)(kPrefillWaves * (d / 8 + 1) * 64 * 4); }

// Plan of one prefill launch: blocks are split only where there are too few to fill `target` places, into
// as many equal parts as fill them, of at least 4 tiles (1000 rows in a window of 512, heads of 256: 32 us, of at
// least 8 tiles 36).
inline PagedPlan plan_paged_prefill(PagedChunk* c, uint32_t chunks, uint32_t rows_per_block, uint32_t head_groups,
                                    uint32_t hkv, uint32_t d, uint32_t window, uint32_t target) {
  PagedPlan p;
  p.rows_per_block = rows_per_block;
  p.head_groups = head_groups;
  const uint64_t per = (uint64_t)hkv * head_groups;
  uint64_t units = 0;
  uint32_t longest = 1;
  auto each = [&](uint32_t i, auto&& f) {
    for (uint32_t r0 = 0; r0 < c[i].rows; r0 += rows_per_block) {
      uint32_t t0, t1;
      paged_range(c[i].start + r0, c[i].start + std::min(r0 + rows_per_block, c[i].rows) - 1, window, 0, 0, kTileSlots, t0, t1);
      f(t1 - t0);
    }
  };
  for (uint32_t i = 0; i < chunks; ++i) {
    each(i, [&](uint32_t n) { longest = std::max(longest, n); });
    const uint32_t blocks = (c[i].rows + rows_per_block - 1) / rows_per_block;
    p.max_blocks = std::max(p.max_blocks, blocks);
    units += blocks * per;
  }
  const uint32_t ways = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(kMaxSplits, target / std::max<uint64_t>(units, 1)));
  p.tiles_per_split = std::max(4u, (longest + ways - 1) / ways);
  p.tiles_per_split = (p.tiles_per_split + 1) / 2 * 2;
  uint64_t items = 0;
  for (uint32_t i = 0; i < chunks; ++i) {
    uint32_t most = 1;
    each(i, [&](uint32_t n) { most = std::max(most, (n + p.tiles_per_split - 1) / p.tiles_per_split); });
    c[i].nsplit = most;
    c[i].part0 = (uint32_t)items;
    if (most > 1) items += (uint64_t)((c[i].rows + rows_per_block - 1) / rows_per_block) * per * most;
    p.max_splits = std::max(p.max_splits, most);
  }
  if (p.max_splits > 1) {
    p.part_bytes = items * paged_prefill_item((int)d) * 4;
  }
  return p;
}

}  // namespace jma
