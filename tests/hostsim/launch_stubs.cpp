// The kernel side of libjmodels_attn for the host simulation (tests/hostsim/hip_sim.cpp): every
// launch function of models_amd/csrc/jma_kernels.h, with the runtime's own arguments, names the
// device ranges its kernel reads or writes (the extents follow the kernels' indexing: the layer
// region of the cache for each row's sequence, the partial buffers by the plan's item count, the
// row tables' largest position for the RoPE tables, every projection matrix's weights, outputs
// and addends) and hands them to the simulation, which checks them against the live allocations
// when the launch executes (for a captured launch: at every graph replay). No kernel runs.
#include <hip/hip_runtime.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <functional>
#include <string>
#include <vector>

#include "jma_kernels.h"

namespace jma {
namespace {

struct Range {
  const void* p;
  size_t bytes;
  std::string what;
};

struct Launch {
  std::vector<Range> ranges;
};

void check_all(void* arg) {
  for (const Range& r : ((Launch*)arg)->ranges) hipsim_check_range(r.p, r.bytes, r.what.c_str());
}

void drop(void* arg) { delete (Launch*)arg; }

hipError_t submit(hipStream_t stream, const char* kernel, Launch* l) {
  for (Range& r : l->ranges) r.what = std::string(kernel) + ": " + r.what;
  return hipsim_launch(stream, kernel, check_all, l, drop);
}

void add(Launch* l, const void* p, size_t bytes, const char* what) {
  if (p != nullptr && bytes > 0) l->ranges.push_back({p, bytes, what});
}

uint32_t row_seq(const RowList& r, uint32_t i) { return r.contiguous ? r.seq0 : r.seq[i]; }
uint32_t row_pos(const RowList& r, uint32_t i) { return r.contiguous ? r.start + i : r.pos[i]; }

uint32_t max_pos(const RowList& r) {
  uint32_t m = 0;
  for (uint32_t i = 0; i < r.count; ++i) m = std::max(m, row_pos(r, i));
  return m;
}

// The layer region (all kv heads, every slot) of each row's sequence, K and V.
void add_cache(Launch* l, const KvView& kv, const RowList& rows, uint32_t hkv, uint32_t dk,
               uint32_t dv, size_t es) {
  for (uint32_t i = 0; i < rows.count; ++i) {
    const uint64_t s = row_seq(rows, i);
    add(l, (const char*)kv.k + (s * kv.seq_stride_k + kv.layer_off_k) * es, (size_t)hkv * kv.cap * dk * es, "K cache");
    add(l, (const char*)kv.v + (s * kv.seq_stride_v + kv.layer_off_v) * es, (size_t)hkv * kv.cap * dv * es, "V cache");
  }
}

}  // namespace

hipError_t fixed_scratch_reset(const FixedScratch& s, hipStream_t) {
  memset(s.counters, 0, s.counters_bytes);
  memset(s.part_f, 0xFF, s.part_f_bytes);
  return hipSuccess;
}

hipError_t fixed_scratch(int device, hipStream_t stream, FixedScratch* out) {
  // The product's sizes (a file-scope device array there; one allocation kept to the end here).
  static FixedScratch s;
  static bool ready = false;
  if (device != 0) return hipErrorInvalidDevice;
  if (!ready) {
    const size_t c = size_t(64) << 10, f = size_t(16) << 20, acc = size_t(16) << 20,
                 ml = size_t(1) << 20, q = size_t(8) << 20;
    unsigned char* base = nullptr;
    hipError_t e = hipMalloc((void**)&base, c + f + acc + ml + q);
    if (e != hipSuccess) return e;
    s.counters = (uint32_t*)base;
    s.counters_bytes = c;
    s.part_f = (float*)(base + c);
    s.part_f_bytes = f;
    s.part_acc = (float*)(base + c + f);
    s.part_acc_bytes = acc;
    s.part_ml = (float*)(base + c + f + acc);
    s.part_ml_bytes = ml;
    s.qrot = (float*)(base + c + f + acc + ml);
    s.qrot_bytes = q;
    e = fixed_scratch_reset(s, stream);
    if (e != hipSuccess) return e;
    ready = true;
  }
  *out = s;
  return hipSuccess;
}

hipError_t launch_append(const AppendArgs& a, bool f16, hipStream_t stream) {
  Launch* l = new Launch();
  const size_t n = a.rows.count;
  add(l, a.q, n * a.num_heads * a.dk * 4, "q");
  add(l, a.k, n * a.num_kv_heads * a.dk * 4, "k");
  add(l, a.v, n * a.num_kv_heads * a.dv * 4, "v");
  add(l, a.q_out, n * a.num_heads * a.dk * 4, "rotated q");
  add(l, a.cos_t, ((size_t)max_pos(a.rows) + 1) * a.pairs * 4, "cos table");
  add(l, a.sin_t, ((size_t)max_pos(a.rows) + 1) * a.pairs * 4, "sin table");
  add(l, a.q_norm_w, (size_t)a.dk * 4, "q norm");
  add(l, a.k_norm_w, (size_t)a.dk * 4, "k norm");
  add_cache(l, a.kv, a.rows, a.num_kv_heads, a.dk, a.dv, f16 ? 2 : 4);
  return submit(stream, "rope_append_kernel", l);
}

hipError_t launch_decode(const DecodeArgs& a, bool f16, int dk, int dv, hipStream_t stream) {
  if (!decode_supported(f16, dk, dv)) return hipErrorInvalidValue;
  if (a.total_items == 0) return hipSuccess;
  Launch* l = new Launch();
  const size_t n = a.rows.count, es = f16 ? 2 : 4;
  add(l, a.q, n * a.num_heads * dk * 4, "q");
  add(l, a.out, n * a.num_heads * dv * 4, "out");
  add(l, a.k_new, n * a.num_kv_heads * dk * 4, "new k rows");
  add(l, a.v_new, n * a.num_kv_heads * dv * 4, "new v rows");
  add(l, a.cos_t, ((size_t)max_pos(a.rows) + 1) * a.pairs * 4, "cos table");
  add(l, a.sin_t, ((size_t)max_pos(a.rows) + 1) * a.pairs * 4, "sin table");
  add(l, a.q_norm_w, (size_t)dk * 4, "q norm");
  add(l, a.k_norm_w, (size_t)dk * 4, "k norm");
  add(l, a.err, 4, "error word");
  const size_t dvs = (size_t)dv / std::max<uint32_t>(a.slices, 1);
  if (a.counters != nullptr) {
    add(l, a.part_f, (size_t)a.total_items * kHeadSlots * (dvs + 4) * 4, "fused partials");
    add(l, a.counters, n * a.num_kv_heads * a.hgroups * 4, "arrival tickets");
  } else if (a.max_splits > 1) {
    const size_t items = a.total_items / std::max<uint32_t>(a.slices, 1);
    add(l, a.part_acc, items * kHeadSlots * dv * 4, "split partials");
    add(l, a.part_ml, items * kHeadSlots * 2 * 4, "split maxima");
  }
  add_cache(l, a.kv, a.rows, a.num_kv_heads, dk, dv, es);
  if (a.k_base != nullptr) {
    add(l, a.k_base, (size_t)a.num_kv_heads * a.kv.cap * dk * es, "K base");
    add(l, a.v_base, (size_t)a.num_kv_heads * a.kv.cap * dv * es, "V base");
  }
  return submit(stream, "decode_kernel", l);
}

hipError_t launch_reduce(const DecodeArgs& a, int dv, hipStream_t stream) {
  Launch* l = new Launch();
  const size_t items = a.total_items / std::max<uint32_t>(a.slices, 1);
  add(l, a.part_acc, items * kHeadSlots * dv * 4, "split partials");
  add(l, a.part_ml, items * kHeadSlots * 2 * 4, "split maxima");
  add(l, a.out, (size_t)a.rows.count * a.num_heads * dv * 4, "out");
  add(l, a.err, 4, "error word");
  return submit(stream, "reduce_kernel", l);
}

hipError_t launch_prefill(const PrefillArgs& a, int dk, int dv, hipStream_t stream) {
  if (!prefill_supported(dk, dv)) return hipErrorInvalidValue;
  Launch* l = new Launch();
  add(l, a.q, (size_t)a.n * a.num_heads * dk * 4, "q");
  add(l, a.out, (size_t)a.n * a.num_heads * dv * 4, "out");
  add(l, a.err, 4, "error word");
  RowList one{};
  one.count = 1;
  one.contiguous = 1;
  one.seq0 = a.seq;
  add_cache(l, a.kv, one, a.num_kv_heads, dk, dv, 2);
  if (a.split_blocks > 0) {
    const size_t S = (size_t)prefill_stripes(dk);
    const size_t pairs = (size_t)a.split_blocks * a.head_groups * a.num_kv_heads;
    add(l, a.part, pairs * 2 * (S * ((dk / 8) * 64 + 32) + S * kPrefillKvGroups) * 16, "split partials");
    add(l, a.tickets, pairs * 4, "split tickets");
  }
  return submit(stream, "prefill_kernel", l);
}

hipError_t launch_prefill_slice(const PrefillArgs& a, bool f16, int dk, int dv, hipStream_t stream) {
  if (!prefill_slice_supported(f16, dk, dv)) return hipErrorInvalidValue;
  Launch* l = new Launch();
  add(l, a.q, (size_t)a.n * a.num_heads * dk * 4, "q");
  add(l, a.out, (size_t)a.n * a.num_heads * dv * 4, "out");
  add(l, a.err, 4, "error word");
  RowList one{};
  one.count = 1;
  one.contiguous = 1;
  one.seq0 = a.seq;
  add_cache(l, a.kv, one, a.num_kv_heads, dk, dv, f16 ? 2 : 4);
  if (a.split_blocks > 0) {
    const size_t splits = (size_t)a.split_blocks * a.head_groups * a.num_kv_heads;
    const size_t half = f16 ? 4 * kPairPartWords * 64 * 16 : (size_t)slice_waves(dk) * slice_state_words(dk) * 64 * 16;
    add(l, a.part, splits * 2 * half, "split states");
    add(l, a.tickets, splits * 4, "pair split tickets");
  }
  return submit(stream, "prefill_slice_kernel", l);
}

namespace {
void add_matrices(Launch* l, const QMatArgs& a, uint32_t fmt) {
  add(l, a.x, (size_t)a.batch * a.cols * 4, "activations");
  for (uint32_t i = 0; i < a.count; ++i) {
    const QMatrix& m = a.m[i];
    add(l, m.w, (size_t)m.rows * a.blocks * qmat_block_bytes(fmt), "weights");
    add(l, m.out, (size_t)a.batch * m.rows * 4, "output");
    if (a.addend_mode == 1) add(l, m.addend, (size_t)m.rows * 4, "bias");
    if (a.addend_mode == 2) add(l, m.addend, (size_t)a.batch * m.rows * 4, "residual");
  }
}
}  // namespace

hipError_t launch_qmatvec(const QMatArgs& a, uint32_t fmt, uint32_t, hipStream_t stream) {
  Launch* l = new Launch();
  add_matrices(l, a, fmt);
  return submit(stream, "qmatvec_kernel", l);
}

hipError_t launch_q8_0_quant(const float* x, uint32_t batch, uint32_t cols, void* act, void* scales,
                             hipStream_t stream) {
  Launch* l = new Launch();
  const size_t rows = (size_t)qact_tiles(batch) * 32;
  add(l, x, (size_t)batch * cols * 4, "activations");
  add(l, act, rows * cols * 2, "quantized activations");
  add(l, scales, rows * (cols / 32) * 2, "activation scales");
  return submit(stream, "q8_0_quant_kernel", l);
}

hipError_t launch_qgemm(const QMatArgs& a, uint32_t fmt, uint32_t, uint32_t, const void* act,
                        const void* act_scale, hipStream_t stream) {
  Launch* l = new Launch();
  const size_t rows = (size_t)qact_tiles(a.batch) * 32;
  add_matrices(l, a, fmt);
  add(l, act, rows * a.cols * 2, "quantized activations");
  add(l, act_scale, rows * a.blocks * 2, "activation scales");
  return submit(stream, "qgemm_kernel", l);
}

hipError_t launch_q8_k_quant(const float* x, uint32_t batch, uint32_t cols, void* act, void* classes,
                             void* sums, void* scales, hipStream_t stream) {
  Launch* l = new Launch();
  const size_t rows = (size_t)qact_tiles(batch) * 32;
  add(l, x, (size_t)batch * cols * 4, "activations");
  if (!act && !classes) hipsim_fail("quantized activations in neither order");
  if (act) add(l, act, rows * cols * 2, "quantized activations");
  if (classes) add(l, classes, rows * cols * 2, "quantized activations in class order");
  if (act) add(l, sums, rows * (cols / 16) * 2, "activation sums");
  add(l, scales, rows * (cols / 256) * 4, "activation scales");
  return submit(stream, "q8_k_quant_kernel", l);
}

hipError_t launch_qkgemm(const QMatArgs& a, uint32_t fmt, uint32_t, uint32_t, const void* act,
                         const void* sums, const void* scales, hipStream_t stream) {
  Launch* l = new Launch();
  const size_t rows = (size_t)qact_tiles(a.batch) * 32;
  add_matrices(l, a, fmt);
  add(l, act, rows * a.cols * 2, "quantized activations");
  if (fmt != 3) add(l, sums, rows * (a.cols / 16) * 2, "activation sums");
  add(l, scales, rows * a.blocks * 4, "activation scales");
  return submit(stream, "qkgemm_kernel", l);
}

// ---------------------------------------------------------------- paged cache and adapters
//
// What these kernels touch depends on the page tables, which the simulated table launches write: the
// checks read them when the launch executes, as the kernels do.

namespace {

hipError_t run(hipStream_t stream, const char* kernel, std::function<void()> f) {
  auto* fn = new std::function<void()>(std::move(f));
  return hipsim_launch(stream, kernel, [](void* p) { (*(std::function<void()>*)p)(); }, fn,
                       [](void* p) { delete (std::function<void()>*)p; });
}

void check(const void* p, uint64_t bytes, const char* what) {
  if (bytes) hipsim_check_range(p, bytes, what);
}

// Pages [from, to] of a sequence's list: in the pool, their K, V and bounds of every kv head.
void check_pages(const PagedView& kv, uint32_t seq, uint32_t from, uint32_t to, uint32_t d, size_t es) {
  const uint32_t* t = kv.table + (uint64_t)seq * kv.table_stride;
  check(t + from, (to - from + 1) * 4ull, "page table");
  if (to >= kv.table_stride) hipsim_fail("page table row too short");
  for (uint32_t i = from; i <= to; ++i) {
    if (t[i] >= kv.pages) hipsim_fail("page number out of the pool");
    const uint64_t n = kv.hkv * paged_head_elems(kv.page_log2, d);
    check((const char*)kv.k + t[i] * n * es, n * es, "page keys");
    check((const char*)kv.v + t[i] * n * es, n * es, "page values");
    if (kv.bounds) check((const char*)kv.bounds + (uint64_t)t[i] * kv.hkv * 2 * d * es, kv.hkv * 2 * d * es, "page bounds");
  }
}

void check_rotation(const PagedRotation& r, uint64_t position) {
  if (r.cos_t == nullptr) return;
  check(r.cos_t, (position + 1) * r.pairs * 4, "rope cos");
  check(r.sin_t, (position + 1) * r.pairs * 4, "rope sin");
}

void check_grid(uint64_t x, uint64_t y, uint64_t z) {
  if (x == 0 || y == 0 || z == 0 || x > 0x7FFFFFFFu || y > 65535 || z > 65535) hipsim_fail("grid out of range");
}

}  // namespace

hipError_t launch_paged_table(const PagedTableArgs& a, hipStream_t stream) {
  return run(stream, "paged_table_kernel", [a] {
    if (a.count > kTableWrites) hipsim_fail("too many table writes");
    for (uint32_t i = 0; i < a.count; ++i) {
      check(a.table + a.at[i], 4, "page table");
      a.table[a.at[i]] = a.page[i];
    }
  });
}

hipError_t launch_paged_append(const PagedAppendArgs& a, bool f16, uint32_t d, hipStream_t stream) {
  return run(stream, "paged_append_kernel", [a, f16, d] {
    const size_t es = f16 ? 2 : 4;
    check_grid(a.max_tiles, a.num_heads + 2 * a.kv.hkv, a.chunks);
    if ((a.q_out == nullptr) != (a.num_heads == 0)) hipsim_fail("query heads without a place for them");
    for (uint32_t i = 0; i < a.chunks; ++i) {
      const PagedChunk& c = a.c[i];
      const uint32_t last = c.start + c.rows - 1;
      if (last / paged_append_rows(d) - c.start / paged_append_rows(d) >= a.max_tiles) hipsim_fail("chunk of more tiles than the grid");
      if ((last >> a.kv.page_log2) - (c.start >> a.kv.page_log2) >= a.max_pages) hipsim_fail("chunk of more pages than the grid");
      const uint64_t qd = (uint64_t)a.num_heads * d, kd = (uint64_t)a.kv.hkv * d;
      if (a.q_out) {
        check(a.q + c.row0 * qd, c.rows * qd * 4, "q");
        check(a.q_out + c.row0 * qd, c.rows * qd * 4, "rotated q");
      }
      check(a.k + c.row0 * kd, c.rows * kd * 4, "k");
      check(a.v + c.row0 * kd, c.rows * kd * 4, "v");
      check_rotation(a.rot, last);
      check_pages(a.kv, c.seq, c.start >> a.kv.page_log2, last >> a.kv.page_log2, d, es);
    }
  });
}

hipError_t launch_paged_select(const PagedSelectArgs& a, bool f16, uint32_t d, hipStream_t stream) {
  return run(stream, "paged_select_kernel", [a, f16, d] {
    check_grid(a.max_wgs, (uint64_t)a.max_blocks * a.kv.hkv, a.chunks);
    const uint64_t blocks = (uint64_t)a.chunks * a.max_blocks * a.kv.hkv;
    check(a.keys, blocks * a.rows_per_block * paged_row_keys(a.key_stride) * 4, "page scores");
    check(a.maxima, blocks * a.max_wgs * 16, "largest bounds");
    check(a.tickets, blocks * 4, "tickets");
    for (uint64_t i = 0; i < blocks; ++i)
      if (a.tickets[i] != 0) hipsim_fail("a ticket is not zero");
    for (uint32_t i = 0; i < a.chunks; ++i) {
      const PagedChunk& c = a.c[i];
      const uint32_t last = (c.start + c.rows - 1) >> a.kv.page_log2;
      if ((c.rows + a.rows_per_block - 1) / a.rows_per_block > a.max_blocks || last >= a.key_stride) hipsim_fail("chunk past the launch's sizes");
      if (a.raw) check_rotation(a.rot, c.start + c.rows - 1);
      if (a.raw && (c.rows != 1 || a.group * (d + 4) > kSelectFloats)) hipsim_fail("raw queries past the kernel's room");
      check(a.q + (uint64_t)c.row0 * a.num_heads * d, (uint64_t)c.rows * a.num_heads * d * 4, "q");
      check(a.pages + (uint64_t)c.row0 * a.kv.hkv * a.budget, (uint64_t)c.rows * a.kv.hkv * a.budget * 4, "selected pages");
      check_pages(a.kv, c.seq, 0, last, d, f16 ? 2 : 4);
    }
  });
}

hipError_t launch_paged_attend(const PagedAttendArgs& a, bool f16, uint32_t d, hipStream_t stream) {
  return run(stream, "paged_attend_kernel", [a, f16, d] {
    const uint64_t units = (uint64_t)a.blocks * a.kv.hkv * a.head_groups;
    check_grid(a.max_splits, units, 1);
    if (a.max_splits > 1) {
      check(a.tickets, units * 4, "tickets");
      for (uint64_t i = 0; i < units; ++i)
        if (a.tickets[i] != 0) hipsim_fail("a ticket is not zero");
    }
    uint32_t before = 0;
    for (uint32_t i = 0; i < a.chunks; ++i) {
      const PagedChunk& c = a.c[i];
      if (c.block0 != before) hipsim_fail("chunks' blocks are not one after another");
      before += (c.rows + a.rows_per_block - 1) / a.rows_per_block;
      if (before > a.blocks || (a.max_blocks == 1 && c.rows > a.rows_per_block)) hipsim_fail("chunk past the grid");
      const uint64_t qd = (uint64_t)a.num_heads * d;
      check(a.q + c.row0 * qd, c.rows * qd * 4, "q");
      check(a.out + c.row0 * qd, c.rows * qd * 4, "out");
      if (a.k_new) {
        if (c.rows != 1) hipsim_fail("a fused launch with a chunk of more than one row");
        check(a.k_new + (uint64_t)c.row0 * a.kv.hkv * d, (uint64_t)a.kv.hkv * d * 4, "new k");
        check(a.v_new + (uint64_t)c.row0 * a.kv.hkv * d, (uint64_t)a.kv.hkv * d * 4, "new v");
        check_rotation(a.rot, c.start);
      }
      if (a.pages) check(a.pages + (uint64_t)c.row0 * a.kv.hkv * a.budget, (uint64_t)c.rows * a.kv.hkv * a.budget * 4, "selected pages");
      const uint32_t blocks = (c.rows + a.rows_per_block - 1) / a.rows_per_block;
      if (blocks > a.max_blocks) hipsim_fail("chunk of more blocks than the grid");
      for (uint32_t b = 0; b < blocks; ++b) {
        const uint32_t r0 = b * a.rows_per_block, r1 = std::min(r0 + a.rows_per_block, c.rows) - 1;
        uint32_t t0, t1;
        paged_range(c.start + r0, c.start + r1, a.window, a.pages ? a.budget : 0, a.kv.page_log2, paged_step(f16), t0, t1);
        const uint32_t ns = (t1 - t0 + a.tiles_per_split - 1) / a.tiles_per_split;
        if (ns > c.nsplit || ns > a.max_splits) hipsim_fail("block of more splits than planned");
      }
      if (c.nsplit > 1)
        check(a.part + (uint64_t)c.part0 * kHeadSlots * (d + 4),
              (uint64_t)blocks * a.kv.hkv * a.head_groups * c.nsplit * kHeadSlots * (d + 4) * 4, "split states");
      check_pages(a.kv, c.seq, first_visible(c.start, a.window) >> a.kv.page_log2, (c.start + c.rows - 1) >> a.kv.page_log2,
                  d, f16 ? 2 : 4);
    }
  });
}

hipError_t launch_paged_prefill(const PagedAttendArgs& a, uint32_t d, hipStream_t stream) {
  return run(stream, "paged_prefill_kernel", [a, d] {
    const uint64_t units = (uint64_t)a.max_blocks * a.kv.hkv * a.head_groups;
    check_grid(a.max_splits, units, a.chunks);
    if (a.pages || a.rows_per_block != kPrefillWaves * a.rows_per_stripe || a.rows_per_stripe * a.heads_per_stripe > 32 ||
        a.heads_per_stripe * a.head_groups < a.group)
      hipsim_fail("stripes do not cover the heads");
    for (uint32_t i = 0; i < a.chunks; ++i) {
      const PagedChunk& c = a.c[i];
      const uint64_t qd = (uint64_t)a.num_heads * d;
      check(a.q + c.row0 * qd, c.rows * qd * 4, "q");
      check(a.out + c.row0 * qd, c.rows * qd * 4, "out");
      const uint32_t blocks = (c.rows + a.rows_per_block - 1) / a.rows_per_block;
      if (blocks > a.max_blocks) hipsim_fail("chunk of more blocks than the grid");
      for (uint32_t b = 0; b < blocks; ++b) {
        const uint32_t r0 = b * a.rows_per_block, r1 = std::min(r0 + a.rows_per_block, c.rows) - 1;
        uint32_t t0, t1;
        paged_range(c.start + r0, c.start + r1, a.window, 0, a.kv.page_log2, kTileSlots, t0, t1);
        const uint32_t ns = (t1 - t0 + a.tiles_per_split - 1) / a.tiles_per_split;
        if (ns > c.nsplit || ns > a.max_splits) hipsim_fail("block of more splits than planned");
      }
      const uint64_t item = paged_prefill_item((int)d) * 4ull;
      if (c.nsplit > 1)
        check((const char*)a.part + c.part0 * item, (uint64_t)blocks * a.kv.hkv * a.head_groups * c.nsplit * item, "split states");
      check_pages(a.kv, c.seq, first_visible(c.start, a.window) >> a.kv.page_log2, (c.start + c.rows - 1) >> a.kv.page_log2, d, 2);
    }
  });
}

hipError_t launch_adapter_load(const AdapterLoadArgs& a, hipStream_t stream) {
  return run(stream, "adapter_load_kernel", [a] {
    const uint64_t e = adapter_elem(a.dtype), r16 = adapter_rank16(a.rank);
    check(a.a, a.rank * (uint64_t)a.cols * e, "A");
    check(a.b, a.rank * (uint64_t)a.outs * e, "B");
    check(a.a_to, r16 * a.cols * e, "stored A");
    check(a.b_to, r16 * a.outs * e, "stored B");
  });
}

namespace {
void check_runs(const AdapterArgs& a, bool scratch) {
  const uint64_t e = adapter_elem(a.dtype);
  if (a.runs > kMaxRuns) hipsim_fail("too many runs");
  for (uint32_t i = 0; i < a.runs; ++i) {
    const AdapterRun& r = a.run[i];
    if (r.rows > a.max_rows) hipsim_fail("run past the launch's sizes");
    check(a.x + (uint64_t)r.row0 * a.cols, (uint64_t)r.rows * a.cols * 4, "input");
    if (a.base) check(a.base + (uint64_t)r.row0 * a.outs, (uint64_t)r.rows * a.outs * 4, "base");
    check(a.out + (uint64_t)r.row0 * a.outs, (uint64_t)r.rows * a.outs * 4, "output");
    if (r.rank16 == 0) continue;
    if (scratch) {
      if (r.rank16 > a.max_rank16) hipsim_fail("run of more ranks than the scratch");
      check(a.down + (uint64_t)r.row0 * a.splits * a.max_rank16, (uint64_t)r.rows * a.splits * a.max_rank16 * 4, "products");
    }
    check((const char*)a.a + r.a_at * e, (uint64_t)r.rank16 * a.cols * e, "stored A");
    check((const char*)a.b + r.b_at * e, (uint64_t)r.rank16 * a.outs * e, "stored B");
  }
}
}  // namespace

hipError_t launch_adapter_few(const AdapterArgs& a, hipStream_t stream) {
  return run(stream, "adapter_few_kernel", [a] {
    check_grid((a.outs + kFewOuts - 1) / kFewOuts, (a.max_rows + a.row_block - 1) / a.row_block, a.runs);
    if (a.row_block != 1 && a.row_block != 2 && a.row_block != 4) hipsim_fail("unknown row block");
    if ((uint64_t)a.row_block * a.cols > kFewFloats) hipsim_fail("rows do not fit the LDS");
    check_runs(a, false);
  });
}

hipError_t launch_adapter_long(const AdapterArgs& a, hipStream_t stream) {
  return run(stream, "adapter_long_kernels", [a] {
    check_grid(a.splits, a.blocks, 1);
    check_grid((a.outs + kUpOuts - 1) / kUpOuts, a.blocks, 1);
    uint32_t blocks = 0;
    for (uint32_t i = 0; i < a.runs; ++i) {
      if (a.run[i].block0 != blocks) hipsim_fail("runs' blocks are not one after another");
      blocks += (a.run[i].rows + kUpRows - 1) / kUpRows;
    }
    if (blocks != a.blocks) hipsim_fail("blocks of the runs");
    if ((uint64_t)a.splits * a.cols_per_split < a.cols || (uint64_t)(a.splits - 1) * a.cols_per_split >= a.cols)
      hipsim_fail("pieces do not cover the columns");
    check_runs(a, true);
  });
}

}  // namespace jma
