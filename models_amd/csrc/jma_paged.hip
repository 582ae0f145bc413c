// gfx950 kernels of the paged KV cache:
//
//   paged_append_kernel   QK-norm and RoPE of new tokens, K/V stored into their sessions' pages
//   paged_bounds_kernel   smallest and largest key elements of the pages that were written
//   paged_select_kernel   the pages whose bounds promise the largest scores, per row and kv head
//   paged_attend_kernel   causal attention over a session's pages, or over its selected ones
//
// Semantics follow the contiguous cache's kernels (jma_kernels.hip): pairs and rotation of
// TensorOps.rope/ropeNeox (backend-java/src/main/java/com/integrallis/models/backend/purejava/ops/
// TensorOps.java:1336-1390, 1474-1486), head norms of :50-58 and gemma4/Gemma4Math.java:38-55,
// attention of llama/LlamaForwardPass.java:1543-1670.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "jma_paged_device.h"

namespace jma {
namespace {

// ================================================================ append

// Workgroup = (storage tile of 32 slots that a chunk writes to, head of q, k or v, chunk). The rows'
// parts of that head go through LDS: one thread a row forms a head's norm sum in the reference's
// order, pairs are rotated in place, and keys and values are stored in the page's layout. Bound by
// latency for single tokens and by the bytes of q, k and v for prompts.
template <typename KV, int D>
__global__ __launch_bounds__(256) void paged_append_kernel(const PagedAppendArgs a) {
  const PagedChunk c = a.c[blockIdx.z];
  if (c.rows == 0) return;
  const uint32_t tile = c.start / kTileSlots + blockIdx.x;
  const uint32_t p0 = max(c.start, tile * kTileSlots), p1 = min(c.start + c.rows, (tile + 1) * kTileSlots);
  if (p0 >= p1) return;
  const uint32_t n = p1 - p0;
  const uint32_t hkv = a.kv.hkv;
  uint32_t item = blockIdx.y;  // q heads, then k heads, then v heads
  const bool is_q = item < a.num_heads;
  if (!is_q) item -= a.num_heads;
  const bool is_k = !is_q && item < hkv;
  const uint32_t head = is_q || is_k ? item : item - hkv;
  const uint32_t heads = is_q ? a.num_heads : hkv;
  const float* src = is_q ? a.q : is_k ? a.k : a.v;
  const uint64_t row0 = (uint64_t)c.row0 + (p0 - c.start);
  src += (row0 * heads + head) * D;

  constexpr int kStride = D + 4;
  __shared__ __attribute__((aligned(16))) float s_x[kTileSlots][kStride];
  __shared__ float s_scale[kTileSlots];
  for (uint32_t i = threadIdx.x; i < n * (D / 4); i += 256) {
    const uint32_t r = i / (D / 4), e = 4 * (i % (D / 4));
    *(float4_t*)&s_x[r][e] = *(const float4_t*)(src + (uint64_t)r * heads * D + e);
  }
  __syncthreads();
  const float* w = is_q ? a.rot.q_norm_w : is_k ? a.rot.k_norm_w : nullptr;
  const bool v_norm = !is_q && !is_k && a.rot.v_norm != 0;
  if (w != nullptr || v_norm) {
#pragma clang fp contract(off)
    if (threadIdx.x < n) s_scale[threadIdx.x] = head_scale<D>(s_x[threadIdx.x], a.rot.norm_eps, v_norm);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n * D; i += 256) {
      const uint32_t r = i / D, e = i % D;
      float x = s_x[r][e] * s_scale[r];
      if (!v_norm) x = x * w[e];
      s_x[r][e] = x;
    }
    __syncthreads();
  }
  if ((is_q || is_k) && a.rot.cos_t != nullptr) {
    for (uint32_t i = threadIdx.x; i < n * a.rot.pairs; i += 256)
      rotate_in(s_x[i / a.rot.pairs], i % a.rot.pairs, a.rot, p0 + i / a.rot.pairs);
    __syncthreads();
  }
  if (is_q) {
    float* dst = a.q_out + (row0 * heads + head) * D;
    for (uint32_t i = threadIdx.x; i < n * (D / 4); i += 256) {
      const uint32_t r = i / (D / 4), e = 4 * (i % (D / 4));
      *(float4_t*)(dst + (uint64_t)r * heads * D + e) = *(const float4_t*)&s_x[r][e];
    }
    return;
  }
  const uint32_t slots = 1u << a.kv.page_log2;
  const uint32_t page = a.kv.table[(uint64_t)c.seq * a.kv.table_stride + (p0 >> a.kv.page_log2)];
  const uint64_t base = paged_base(page, hkv, head, a.kv.page_log2, D);
  const uint32_t slot0 = p0 & (slots - 1);  // the rows' slots are one run inside the tile
  constexpr bool kF16 = std::is_same<KV, _Float16>::value;
  if (is_k) {
    KV* dst = (KV*)a.kv.k + base;
    constexpr uint32_t kW = kF16 ? 8 : 4;  // elements of 16 bytes
    for (uint32_t i = threadIdx.x; i < n * (D / kW); i += 256) {
      // Rows vary fastest: consecutive threads fill consecutive 64-byte rows of a panel.
      const uint32_t q = i % (4 * n), panel = i / (4 * n);
      const uint32_t r = q / 4, e = panel * (4 * kW) + (q % 4) * kW;
      typedef KV kv16_t __attribute__((ext_vector_type(kW)));
      kv16_t y;
#pragma unroll
      for (uint32_t t = 0; t < kW; ++t) y[t] = (KV)s_x[r][e + t];
      *(kv16_t*)(dst + paged_k_index(slot0 + r, e, D, kF16)) = y;
    }
  } else {
    KV* dst = (KV*)a.kv.v + base + (slot0 / kTileSlots) * kTileSlots * D;
    const uint32_t at = slot0 % kTileSlots;
    if (n == kTileSlots) {
      constexpr uint32_t kW = kF16 ? 8 : 4;
      for (uint32_t i = threadIdx.x; i < kTileSlots / kW * D; i += 256) {
        const uint32_t e = i / (kTileSlots / kW), r = (i % (kTileSlots / kW)) * kW;
        typedef KV kv16_t __attribute__((ext_vector_type(kW)));
        kv16_t y;
#pragma unroll
        for (uint32_t t = 0; t < kW; ++t) y[t] = (KV)s_x[r + t][e];
        *(kv16_t*)(dst + e * kTileSlots + r) = y;
      }
    } else {
      for (uint32_t i = threadIdx.x; i < n * D; i += 256) {
        const uint32_t e = i / n, r = i % n;
        dst[e * kTileSlots + at + r] = (KV)s_x[r][e];
      }
    }
  }
}

// The smallest and the largest of a page's key elements of one kv head, over its first `filled` slots, by a
// workgroup of kThreads. Exact, whatever the order: no sums. A NaN key element is left out of them.
// fresh: the last of these slots' keys in LDS (null: stored like the others). s_red: 2 * kThreads * 16
// bytes / sizeof(KV) floats.
template <typename KV, int D, uint32_t kThreads>
__device__ __forceinline__ void page_bounds(const PagedView& kv, uint32_t page, uint32_t head, uint32_t filled,
                                            const float* fresh, float* s_red) {
  const KV* src = (const KV*)kv.k + paged_base(page, kv.hkv, head, kv.page_log2, D);
  constexpr bool kF16 = std::is_same<KV, _Float16>::value;
  constexpr uint32_t kW = kF16 ? 8 : 4, kPieces = D / kW, kLanes = kThreads / kPieces;
  typedef KV kv16_t __attribute__((ext_vector_type(kW)));
  const uint32_t piece = threadIdx.x % kPieces, lane = threadIdx.x / kPieces;
  float lo[kW], hi[kW];
#pragma unroll
  for (uint32_t t = 0; t < kW; ++t) lo[t] = INFINITY, hi[t] = -INFINITY;
  const uint32_t stored = filled - (fresh ? 1u : 0u);
#pragma unroll 4
  for (uint32_t s = lane; s < stored; s += kLanes) {
    const kv16_t x = *(const kv16_t*)(src + paged_k_index(s, piece * kW, D, kF16));
#pragma unroll
    for (uint32_t t = 0; t < kW; ++t) {
      lo[t] = fminf(lo[t], (float)x[t]);
      hi[t] = fmaxf(hi[t], (float)x[t]);
    }
  }
  float* s_lo = s_red;
  float* s_hi = s_red + kLanes * D;
#pragma unroll
  for (uint32_t t = 0; t < kW; ++t) {
    s_lo[lane * D + piece * kW + t] = lo[t];
    s_hi[lane * D + piece * kW + t] = hi[t];
  }
  __syncthreads();
  KV* dst = (KV*)kv.bounds + ((uint64_t)page * kv.hkv + head) * 2 * D;
  for (uint32_t i = threadIdx.x; i < 2 * D; i += kThreads) {
    const uint32_t e = i % D;
    float x = i < D ? s_lo[e] : s_hi[e];
    for (uint32_t l = 1; l < kLanes; ++l) x = i < D ? fminf(x, s_lo[l * D + e]) : fmaxf(x, s_hi[l * D + e]);
    if (fresh) {
      const float y = (float)(KV)fresh[e];
      x = i < D ? fminf(x, y) : fmaxf(x, y);
    }
    dst[i] = (KV)x;
  }
}

// Workgroup = (page that a chunk wrote to, kv head, chunk).
template <typename KV, int D>
__global__ __launch_bounds__(256) void paged_bounds_kernel(const PagedAppendArgs a) {
  const PagedChunk c = a.c[blockIdx.z];
  if (c.rows == 0) return;
  const uint32_t number = (c.start >> a.kv.page_log2) + blockIdx.x, end = c.start + c.rows;
  if (number > (end - 1) >> a.kv.page_log2) return;
  __shared__ float s_red[2 * 256 * 16 / sizeof(KV)];
  page_bounds<KV, D, 256>(a.kv, a.kv.table[(uint64_t)c.seq * a.kv.table_stride + number], blockIdx.y,
                          min(end - (number << a.kv.page_log2), 1u << a.kv.page_log2), nullptr, s_red);
}

__global__ __launch_bounds__(512) void paged_table_kernel(const PagedTableArgs a) {
  if (threadIdx.x < a.count) a.table[a.at[threadIdx.x]] = a.page[threadIdx.x];
}

// ================================================================ page selection

// A score as an integer of the same order. A score that is no number (an infinite key element
// against a zero of the query) counts as the largest, so that attention meets the page and says so.
__device__ __forceinline__ uint64_t ordered(double x) {
  if (x != x) return 0xFFFFFFFFFFFFFFFFull;
  const uint64_t b = (uint64_t)__double_as_longlong(x == 0.0 ? 0.0 : x);
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

// Sum over the 16 lanes of a row, in vector ALU exchanges; every lane gets the same bits.
template <int kCtrl>
__device__ __forceinline__ double row_moved(double x) {
  const uint64_t b = (uint64_t)__double_as_longlong(x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)b, kCtrl, 0xF, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(b >> 32), kCtrl, 0xF, 0xF, false);
  return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
__device__ __forceinline__ double row_sum(double x) {
  x += row_moved<0x128>(x);  // row_ror by 8, 4, 2, 1
  x += row_moved<0x124>(x);
  x += row_moved<0x122>(x);
  x += row_moved<0x121>(x);
  return x;
}

// The pages of one (row, kv head), ascending: the first `first`, the last `last` and the `top` others of
// the largest keys, of equal ones the lowest. The key of the last page taken is narrowed by eight
// bits a pass, from the highest bit in which any two keys differ, until every key that shares the bits
// found so far is taken (two or three passes: the keys are spread). n > first + last + top.
template <uint32_t kPickRounds>
__device__ __forceinline__ void pick_pages(const uint64_t* keys, uint32_t n, uint32_t top, uint32_t first, uint32_t last,
                                           uint32_t* out) {
  __shared__ uint32_t s_hist[256], s_found[3], s_any[4][2], s_sum[4];
  __shared__ uint32_t s_count[64];
  constexpr uint32_t kPickPages = 256 * kPickRounds;  // keys the workgroup holds in registers
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint64_t k[kPickRounds];
  auto candidate = [&](uint32_t p) JMA_INL { return p >= first && p + last < n; };
  auto load = [&](uint32_t base) JMA_INL {
#pragma unroll
    for (uint32_t i = 0; i < kPickRounds; ++i) {
      // Unconditional, so that all are in flight together: those of no candidate are not looked at.
      const uint32_t p = min(base + 256 * i + tid, n - last - 1);
      k[i] = __hip_atomic_load(&keys[p], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  };
  auto each = [&](auto&& f) JMA_INL {  // f(round's first page) over the keys, re-read where they are too many
    for (uint32_t base = 0; base < n; base += kPickPages) {
      if (n > kPickPages) load(base);
      f(base);
    }
  };
  load(0);

  // The bits in which the keys differ from the first one's.
  const uint64_t reference = __hip_atomic_load(&keys[first], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  uint64_t differ = 0;
  each([&](uint32_t base) JMA_INL {
#pragma unroll
    for (uint32_t i = 0; i < kPickRounds; ++i)
      if (candidate(base + 256 * i + tid)) differ |= k[i] ^ reference;
  });
  uint32_t lo = (uint32_t)differ, hi = (uint32_t)(differ >> 32);
#pragma unroll
  for (int m = 1; m < 64; m *= 2) {
    lo |= __shfl_xor(lo, m);
    hi |= __shfl_xor(hi, m);
  }
  if (lane == 0) s_any[wave][0] = lo, s_any[wave][1] = hi;
  __syncthreads();
  differ = (uint64_t)(s_any[0][1] | s_any[1][1] | s_any[2][1] | s_any[3][1]) << 32 | (s_any[0][0] | s_any[1][0] | s_any[2][0] | s_any[3][0]);
  int shift = differ == 0 ? 0 : max(0, 64 - __clzll((long long)differ) - 8);
  uint64_t prefix = shift + 8 >= 64 ? 0 : reference >> (shift + 8);  // bits found so far
  uint32_t need = top;
  bool all = top == 0 || differ == 0;
  if (differ == 0) prefix = reference;
  const bool tie = differ == 0;  // one key throughout: the lowest pages
  for (; !all; shift = max(0, shift - 8)) {
    s_hist[tid] = 0;
    __syncthreads();
    each([&](uint32_t base) JMA_INL {
#pragma unroll
      for (uint32_t i = 0; i < kPickRounds; ++i)
        if (candidate(base + 256 * i + tid) && (shift + 8 >= 64 || k[i] >> (shift + 8) == prefix))
          atomicAdd(&s_hist[(k[i] >> shift) & 255], 1u);
    });
    __syncthreads();
    // How many keys are in bin `tid` and above.
    const uint32_t mine = s_hist[tid];
    uint32_t above = mine;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
      const uint32_t x = __shfl_down(above, m);
      if (lane + m < 64) above += x;
    }
    if (lane == 0) s_sum[wave] = above;
    __syncthreads();
    for (uint32_t w = wave + 1; w < 4; ++w) above += s_sum[w];
    if (above >= need && above - mine < need) {
      s_found[0] = tid;
      s_found[1] = need - (above - mine);
      s_found[2] = mine;
    }
    __syncthreads();
    prefix = prefix << 8 | s_found[0];
    need = s_found[1];
    all = need == s_found[2] || shift == 0;
    if (all) break;
    if (shift < 8) {  // the last pass takes the bits that are left
      const int left = shift;
      s_hist[tid] = 0;
      __syncthreads();
      each([&](uint32_t base) JMA_INL {
#pragma unroll
        for (uint32_t i = 0; i < kPickRounds; ++i)
          if (candidate(base + 256 * i + tid) && k[i] >> left == prefix) atomicAdd(&s_hist[k[i] & ((1u << left) - 1)], 1u);
      });
      __syncthreads();
      const uint32_t bin = s_hist[tid];
      uint32_t up = bin;
#pragma unroll
      for (int m = 1; m < 64; m *= 2) {
        const uint32_t x = __shfl_down(up, m);
        if (lane + m < 64) up += x;
      }
      if (lane == 0) s_sum[wave] = up;
      __syncthreads();
      for (uint32_t w = wave + 1; w < 4; ++w) up += s_sum[w];
      if (up >= need && up - bin < need) {
        s_found[0] = tid;
        s_found[1] = need - (up - bin);
        s_found[2] = bin;
      }
      __syncthreads();
      prefix = prefix << left | s_found[0];
      need = s_found[1];
      shift = 0;
      break;
    }
  }
  // Taken: keys above the last one's bits, and of those that share them the lowest `need` pages (all of
  // them unless keys are equal).
  uint32_t taken = 0, equal = 0;  // before this round of kPickPages pages
  each([&](uint32_t base) JMA_INL {
    uint32_t flags = 0, ties = 0;
#pragma unroll
    for (uint32_t i = 0; i < kPickRounds; ++i) {
      const uint32_t p = base + 256 * i + tid;
      const uint64_t x = tie ? k[i] : k[i] >> shift;
      const bool c = candidate(p), eq = c && top != 0 && x == prefix;
      if (p < n && (!c || (top != 0 && x > prefix))) flags |= 1u << i;
      if (eq) ties |= 1u << i;
    }
    // Ranks of the equal keys, in page order.
    auto ranks = [&](uint32_t set, uint32_t before, uint32_t* total) JMA_INL {
      __syncthreads();
#pragma unroll
      for (uint32_t i = 0; i < kPickRounds; ++i) {
        const uint64_t b = __ballot((set >> i) & 1);
        if (lane == 0) s_count[4 * i + wave] = __popcll(b);
      }
      __syncthreads();
      if (wave == 0) {
        const uint32_t mine = lane < 4 * kPickRounds ? s_count[lane] : 0;
        uint32_t sum = mine;
#pragma unroll
        for (int m = 1; m < 64; m *= 2) {
          const uint32_t x = __shfl_up(sum, m);
          if (lane >= (uint32_t)m) sum += x;
        }
        s_count[lane] = sum - mine;
        if (lane == 63) s_sum[0] = sum;
      }
      __syncthreads();
      *total = before + s_sum[0];
      return before;
    };
    auto rank = [&](uint32_t set, uint32_t i, uint32_t before) JMA_INL {
      const uint64_t b = __ballot((set >> i) & 1);
      return before + s_count[4 * i + wave] + (uint32_t)__popcll(b & ((1ull << lane) - 1));
    };
    uint32_t next;
    const uint32_t before_eq = ranks(ties, equal, &next);
#pragma unroll
    for (uint32_t i = 0; i < kPickRounds; ++i) {
      const uint32_t r = rank(ties, i, before_eq);
      if (((ties >> i) & 1) && r < need) flags |= 1u << i;
    }
    equal = next;
    const uint32_t before = ranks(flags, taken, &next);
#pragma unroll
    for (uint32_t i = 0; i < kPickRounds; ++i) {
      const uint32_t r = rank(flags, i, before);
      if ((flags >> i) & 1) out[r] = base + 256 * i + tid;
    }
    taken = next;
  });
}

// Workgroup = (64 pages, row x kv head, chunk). Scores: for a page with bounds lo, hi and each query
// head of the group, sum_d max(q_d lo_d, q_d hi_d), which no key of the page exceeds; the page's score
// is the largest of the heads'. The sums are formed in 64 bits, where the products are exact, so that
// which of two nearly equal pages is taken does not depend on the order of a sum. 16 lanes take a page,
// four pages each, whose table entries and bounds are all in flight before the first is used: the
// kernel's time is those two memory round trips and the pick's, not its arithmetic (64 pages, 4 heads of
// 128: 1 us). The last workgroup of a (row, kv head) to finish picks the pages.
template <typename KV, int D>
__global__ __launch_bounds__(256) void paged_select_kernel(const PagedSelectArgs a) {
  const PagedChunk c = a.c[blockIdx.z];
  const uint32_t hkv = a.kv.hkv, kvh = blockIdx.y % hkv, r = blockIdx.y / hkv;
  if (r >= c.rows) return;
  const uint32_t pos = c.start + r, row = c.row0 + r;
  const uint32_t n = (pos >> a.kv.page_log2) + 1;
  const uint32_t first_page = blockIdx.x * kSelectPages;
  if (first_page >= n) return;
  const uint32_t wgs = (n + kSelectPages - 1) / kSelectPages;
  uint32_t* out = a.pages + ((uint64_t)row * hkv + kvh) * a.budget;
  if (n <= a.budget) {  // every page
    if (blockIdx.x == 0)
      for (uint32_t i = threadIdx.x; i < a.budget; i += 256) out[i] = i < n ? i : kNoPage;
    return;
  }
  const uint64_t slot = ((uint64_t)blockIdx.z * a.max_rows + r) * hkv + kvh;
  uint64_t* keys = a.keys + slot * a.key_stride;
  extern __shared__ __attribute__((aligned(16))) float s_queries[];  // raw: [group][D + 4]
  __shared__ float s_scale[kSelectFloats / 32];

  constexpr int kE = D / 16, kP = kSelectPages / 16;
  typedef KV kve_t __attribute__((ext_vector_type(kE)));
  const uint32_t lane16 = threadIdx.x % 16, own = threadIdx.x / 16;
  const uint32_t* table = a.kv.table + (uint64_t)c.seq * a.kv.table_stride;
  uint32_t page[kP];
#pragma unroll
  for (int i = 0; i < kP; ++i) page[i] = table[min(first_page + 16 * i + own, n - 1)];
  kve_t lo[kP], hi[kP];
#pragma unroll
  for (int i = 0; i < kP; ++i) {
    const KV* b = (const KV*)a.kv.bounds + ((uint64_t)page[i] * hkv + kvh) * 2 * D + lane16 * kE;
    lo[i] = *(const kve_t*)b;
    hi[i] = *(const kve_t*)(b + D);
  }
  const float* q = a.q + ((uint64_t)row * a.num_heads + kvh * a.group) * D;
  if (a.raw) {
    for (uint32_t i = threadIdx.x; i < a.group * (D / 4); i += 256)
      *(float4_t*)&s_queries[i / (D / 4) * (D + 4) + 4 * (i % (D / 4))] = *(const float4_t*)(q + 4 * i);
    prepare_token<D, D + 4>(s_queries, s_scale, a.group, 0, false, a.rot, pos, 256);
  }
  double best[kP];
  bool odd[kP];
#pragma unroll
  for (int i = 0; i < kP; ++i) best[i] = -INFINITY, odd[i] = false;
  for (uint32_t h = 0; h < a.group; ++h) {
    float x[kE];
#pragma unroll
    for (int e = 0; e < kE; ++e) x[e] = a.raw ? s_queries[h * (D + 4) + lane16 * kE + e] : q[(uint64_t)h * D + lane16 * kE + e];
#pragma unroll
    for (int i = 0; i < kP; ++i) {
      double s = 0.0;
#pragma unroll
      for (int e = 0; e < kE; ++e) s = fma((double)x[e], (double)(float)(x[e] >= 0.0f ? hi[i][e] : lo[i][e]), s);
      s = row_sum(s);
      odd[i] = odd[i] || s != s;
      best[i] = s > best[i] ? s : best[i];
    }
  }
#pragma unroll
  for (int i = 0; i < kP; ++i) {
    const uint32_t p = first_page + 16 * i + own;
    if (lane16 == 0 && p < n)
      __hip_atomic_store(&keys[p], odd[i] ? 0xFFFFFFFFFFFFFFFFull : ordered(best[i]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  // The keys are acknowledged (visible device-wide) before the ticket is taken.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (wgs > 1) {
    __shared__ uint32_t s_last;
    if (threadIdx.x == 0)
      s_last = __hip_atomic_fetch_add(&a.tickets[slot], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (s_last + 1 != wgs) return;
    if (threadIdx.x == 0) __hip_atomic_store(&a.tickets[slot], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (n <= 1024) pick_pages<4>(keys, n, a.top, a.first, a.last, out);
  else pick_pages<16>(keys, n, a.top, a.first, a.last, out);
}

// ================================================================ attention

// One step's K and V of one lane, in matrix-core operand order (below).
template <typename KV, int D>
struct Step;

template <int D>
struct Step<_Float16, D> {
  half8_t k[2][D / 32], v[D / 16];
  __device__ __forceinline__ void load_k(const _Float16* kt, uint32_t, int c16, int g) {
    const uint32_t slot = 8 * (c16 >> 2) + (c16 & 3);
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int c = 0; c < D / 32; ++c) k[b][c] = *(const half8_t*)(kt + c * 1024 + (slot + 4 * b) * 32 + 8 * g);
  }
  __device__ __forceinline__ void load_v(const _Float16* vt, uint32_t, int c16, int g) {
#pragma unroll
    for (int n = 0; n < D / 16; ++n) v[n] = *(const half8_t*)(vt + (16 * n + c16) * 32 + 8 * g);
  }
  // Slot r of the step replaced by the key (value) in LDS.
  __device__ __forceinline__ void patch_k(const float* x, uint32_t r, int c16, int g) {
    const uint32_t slot = 8 * (c16 >> 2) + (c16 & 3);
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) k[b][c][e] = slot + 4 * b == r ? (_Float16)x[32 * c + 8 * g + e] : k[b][c][e];
  }
  __device__ __forceinline__ void patch_v(const float* x, uint32_t r, int c16, int g) {
#pragma unroll
    for (int n = 0; n < D / 16; ++n) {
      const _Float16 y = (_Float16)x[16 * n + c16];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[n][e] = r == (uint32_t)(8 * g + e) ? y : v[n][e];
    }
  }
};
template <int D>
struct Step<float, D> {
  float4_t k[D / 16], v[D / 16];
  __device__ __forceinline__ void load_k(const float* kt, uint32_t half, int c16, int g) {
#pragma unroll
    for (int c = 0; c < D / 16; ++c) k[c] = *(const float4_t*)(kt + c * 512 + (16 * half + c16) * 16 + 4 * g);
  }
  __device__ __forceinline__ void load_v(const float* vt, uint32_t half, int c16, int g) {
#pragma unroll
    for (int n = 0; n < D / 16; ++n) v[n] = *(const float4_t*)(vt + (16 * n + c16) * 32 + 16 * half + 4 * g);
  }
  __device__ __forceinline__ void patch_k(const float* x, uint32_t r, int c16, int g) {
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) k[c][e] = (uint32_t)c16 == r ? x[16 * c + 4 * g + e] : k[c][e];
  }
  __device__ __forceinline__ void patch_v(const float* x, uint32_t r, int c16, int g) {
#pragma unroll
    for (int n = 0; n < D / 16; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[n][e] = r == (uint32_t)(4 * g + e) ? x[16 * n + c16] : v[n][e];
  }
};

// The new token of a chunk of one row, stored by a workgroup of its own: K, V, and the bounds of their page.
template <typename KV, int D, uint32_t kThreads>
__device__ __forceinline__ void store_token(const PagedView& kv, const PagedChunk& ch, uint32_t kvh, const float* key,
                                            const float* value, float* s_red) {
  constexpr bool kF16 = std::is_same<KV, _Float16>::value;
  const uint32_t page = kv.table[(uint64_t)ch.seq * kv.table_stride + (ch.start >> kv.page_log2)];
  const uint32_t slot = ch.start & ((1u << kv.page_log2) - 1);
  const uint64_t base = paged_base(page, kv.hkv, kvh, kv.page_log2, D);
  for (uint32_t e = threadIdx.x; e < D; e += kThreads) {
    ((KV*)kv.k)[base + paged_k_index(slot, e, D, kF16)] = (KV)key[e];
    ((KV*)kv.v)[base + paged_v_index(slot, e, D)] = (KV)value[e];
  }
  if (kv.bounds != nullptr) page_bounds<KV, D, kThreads>(kv, page, kvh, slot + 1, key, s_red);
}

// Workgroup = (split, kv head x head group x block of query rows, chunk): 16 matrix-core columns =
// (query row, query head) pairs that share every K/V load; its waves stride over the split's steps
// of 32 slots (f16) or 16 (f32), each with the running maximum and sum of its own softmax.
//
// S = K Q^T on 16-slot blocks leaves lane (g, c) scores of column c. f16: row i of block b is slot
// 8 (i / 4) + 4 b + i % 4, so that the lane's eight scores are slots 8g .. 8g+7, in order, and are
// the B operand of O^T = V^T P as they stand. f32: four slots 4g .. 4g+3 of a 16-slot half, one
// 16x16x4 product each.
//
// f16 operands carry q and p as hi + lo halves (x = hi + lo to 2^-22), two products each, so that
// the result is that of 32-bit arithmetic. Each column's q is scaled by a power of two that puts its
// largest element in [2^13, 2^14), which costs nothing (the score's factor undoes it) and keeps both
// halves far from f16's ends; p is formed as 2^(s - m + 6) for the same reason.
//
// kFused: the chunks are one token each, whose q, k and v come raw: every workgroup normalises and rotates
// its queries, the one of the last split also the token's key, which it puts in place of the stored slot,
// and one more workgroup per kv head (split = their count) stores the token, so that nobody waits for it.
//
// Positions a column does not see are masked after the product. A value that is no finite number, in a
// step that a column sees in part, reaches all of the wave's columns (0 x inf is no 0); a wave with such an
// output does its steps again, with those values taken out of the product and what they make of the
// columns that see them (NaN) put in.
template <typename KV, int D, bool kSelected, bool kFused>
__global__ __launch_bounds__(64 * paged_waves(D)) __attribute__((amdgpu_waves_per_eu(D <= 64 ? 4 : D == 128 ? 2 : 1)))
void paged_attend_kernel(const PagedAttendArgs a) {
  constexpr bool kF16 = std::is_same<KV, _Float16>::value;
  constexpr int kW = paged_waves(D), kNs = kF16 ? 8 : 4, kNv = D / 16;
  constexpr uint32_t kStep = kF16 ? 32 : 16, kThreads = 64 * kW;
  constexpr int kQStride = D + 4, kHStride = D + 8;
  // At heads of 256 a step's K and V take half the registers: only the next step's K is loaded ahead, and
  // the queries' halves stay in LDS.
  constexpr bool kWide = D >= 256;
  __shared__ __attribute__((aligned(16))) float s_q[(kFused ? 18 : 16) * kQStride];
  __shared__ __attribute__((aligned(16))) _Float16 s_qh[kWide && kF16 ? 2 * 16 * kHStride : 8];
  // The waves' states; a storing workgroup's bounds (page_bounds) before.
  constexpr int kAccFloats = kW * 16 * D, kRedFloats = kFused ? 2 * kThreads * 16 / sizeof(KV) : 0;
  __shared__ __attribute__((aligned(16))) float s_acc_mem[kAccFloats > kRedFloats ? kAccFloats : kRedFloats];
  float (*s_acc)[16][D] = (float (*)[16][D])s_acc_mem;
  __shared__ float s_ml[kW][16][2];
  __shared__ float s_scale[18];
  __shared__ uint32_t s_ticket;

  const PagedChunk ch = a.c[blockIdx.z];
  const uint32_t hkv = a.kv.hkv, R = a.rows_per_block;
  const uint32_t kvh = blockIdx.y % hkv, rest = blockIdx.y / hkv;
  const uint32_t hg = rest % a.head_groups, row0 = rest / a.head_groups * R;
  if (row0 >= ch.rows) return;
  const uint32_t rows = min(R, ch.rows - row0), heads = min(16u, a.group - 16 * hg);
  const uint32_t pos0 = ch.start + row0, pos1 = pos0 + rows - 1;

  uint32_t t0, t1;
  const uint32_t page_log2 = a.kv.page_log2;
  const uint32_t steps_log2 = page_log2 - (kF16 ? 5 : 4);  // steps of a page
  paged_range(pos0, pos1, a.window, kSelected ? a.budget : 0u, page_log2, kStep, t0, t1);
  // A fused launch's lists end with the token's own page: its steps behind the token are left out, and the
  // token is in the last split.
  if (kSelected && kFused) t1 -= (1u << steps_log2) - 1 - (pos0 & ((1u << page_log2) - 1)) / kStep;
  const uint32_t ns = (t1 - t0 + a.tiles_per_split - 1) / a.tiles_per_split, split = blockIdx.x;
  if (split >= ns + (kFused && hg == 0 ? 1u : 0u)) return;
  const bool stores = kFused && split == ns;  // the workgroup that appends the token
  t0 += split * a.tiles_per_split;
  t1 = min(t1, t0 + a.tiles_per_split);

  const int lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // This lane's column; one past the block's (row, head) pairs holds zeros and is never stored.
  const uint32_t col_row = c16 / heads;
  const uint32_t cpos = pos0 + min(col_row, rows - 1), cfirst = first_visible(cpos, a.window);
  const uint64_t qrow = (uint64_t)ch.row0 + row0;

  // The page of each of this wave's next 64 steps is held by the lane of that number: its logical
  // number and where it is.
  const uint32_t* table = a.kv.table + (uint64_t)ch.seq * a.kv.table_stride;
  const uint32_t* list = kSelected ? a.pages + ((qrow * hkv) + kvh) * a.budget : nullptr;
  // A list made by the caller may hold anything: numbers past the row's position, or not ascending, are
  // reported and left out.
  auto listed = [&](uint32_t i) JMA_INL -> uint32_t {
    const uint32_t n = list[i], before = i == 0 ? 0u : list[i - 1];
    if (n == kNoPage) return n;
    if (n <= cpos >> page_log2 && (i == 0 || before < n)) return n;
    report(a.err, kErrBadPage);
    return kNoPage;
  };
  uint32_t my_page = 0, my_number = 0;
  auto fetch_pages = [&](uint32_t t) JMA_INL {
    const uint32_t mine = t + lane * kW;
    my_page = kNoPage;
    if (mine < t1) {
      my_number = kSelected ? listed(mine >> steps_log2) : mine >> steps_log2;
      if (!kSelected || my_number != kNoPage) my_page = table[my_number];
    }
  };
  const KV* kbase = (const KV*)a.kv.k;
  const KV* vbase = (const KV*)a.kv.v;
  // Where step t, on `page`, is stored: its K (the V storage has the same shape).
  auto place = [&](uint32_t t, uint32_t page) JMA_INL {
    const uint32_t in = t & ((1u << steps_log2) - 1), tile = kF16 ? in : in >> 1;
    return paged_base(page, hkv, kvh, page_log2, D) + tile * kTileSlots * D;
  };
  struct Place {
    uint64_t at;
    uint32_t p0;  // the step's first position, kNoPage: the step has no page
  };
  // Step t, the i-th since fetch_pages.
  auto placed = [&](uint32_t t, uint32_t i) JMA_INL {
    const uint32_t page = __builtin_amdgcn_readlane(my_page, i), number = __builtin_amdgcn_readlane(my_number, i);
    Place x;
    x.p0 = page < a.kv.pages ? (number << page_log2) + (t & ((1u << steps_log2) - 1)) * kStep : kNoPage;
    x.at = place(t, page < a.kv.pages ? page : 0u);
    return x;
  };

  uint32_t t = t0 + wave;
  if (!stores && t < t1) fetch_pages(t);

  // q of the block's columns, in LDS; the token's key and value behind them where they are needed.
  const bool with_kv = kFused && split + 1 >= ns;
  const float* q = a.q + (qrow * a.num_heads + kvh * a.group + 16 * hg) * D;
  for (uint32_t i = threadIdx.x; i < 16 * (D / 4); i += kThreads) {
    const uint32_t c = i / (D / 4), e = 4 * (i % (D / 4)), r = c / heads, h = c % heads;
    float4_t x = {0.f, 0.f, 0.f, 0.f};
    if (r < rows) x = *(const float4_t*)(q + ((uint64_t)r * a.num_heads + h) * D + e);
    *(float4_t*)&s_q[c * kQStride + e] = x;
  }
  if (with_kv && threadIdx.x < 2 * (D / 4)) {
    const uint32_t i = threadIdx.x / (D / 4), e = 4 * (threadIdx.x % (D / 4));
    *(float4_t*)&s_q[(16 + i) * kQStride + e] = *(const float4_t*)((i == 0 ? a.k_new : a.v_new) + (qrow * hkv + kvh) * D + e);
  }

  Step<KV, D> xa, xb;
  Place pa = {0, kNoPage}, pb = {0, kNoPage};
  uint32_t i = 0;
  if (!stores && t < t1) {
    pa = placed(t, 0);
    const uint32_t half = t & 1;
    xa.load_k(kbase + pa.at, half, c16, g);
    if (!kWide) xa.load_v(vbase + pa.at, half, c16, g);
  }
  if constexpr (kFused) prepare_token<D, kQStride>(s_q, s_scale, heads, 16, with_kv, a.rot, pos0, kThreads);
  const float* new_k = s_q + 16 * kQStride;
  const float* new_v = s_q + 17 * kQStride;
  if (stores) {
    __syncthreads();
    store_token<KV, D, kThreads>(a.kv, ch, kvh, new_k, new_v, s_acc_mem);
    return;
  }
  const uint32_t new_p0 = kFused ? pos0 / kStep * kStep : kNoPage - 1, new_r = pos0 % kStep;
  __syncthreads();

  // Q operand and the factor of each column's scores.
  half8_t qhi[kF16 && !kWide ? D / 32 : 1], qlo[kF16 && !kWide ? D / 32 : 1];
  float4_t qf[kF16 ? 1 : D / 16];
  float factor = a.scale;
  if constexpr (kF16) {
    float top = 0.0f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const float4_t x0 = *(const float4_t*)&s_q[c16 * kQStride + 32 * c + 8 * g], x1 = *(const float4_t*)&s_q[c16 * kQStride + 32 * c + 8 * g + 4];
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, fmaxf(fabsf(x0[e]), fabsf(x1[e])));
    }
    top = max_groups(top);
    int ex = 0;  // top in [2^(ex-1), 2^ex)
    if (top > 0.0f && top < INFINITY) ex = __builtin_amdgcn_frexp_expf(top);
    ex = max(ex, -100);
    factor = __builtin_amdgcn_ldexpf(a.scale, ex - 14);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      if (kWide && c % kW != wave) continue;
      const float4_t x0 = *(const float4_t*)&s_q[c16 * kQStride + 32 * c + 8 * g], x1 = *(const float4_t*)&s_q[c16 * kQStride + 32 * c + 8 * g + 4];
      half8_t yh, yl;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        _Float16 hi, lo;
        halves(__builtin_amdgcn_ldexpf(e < 4 ? x0[e & 3] : x1[e & 3], 14 - ex), hi, lo);
        yh[e] = hi;
        yl[e] = lo;
      }
      if constexpr (kWide) {
        *(half8_t*)&s_qh[c16 * kHStride + 32 * c + 8 * g] = yh;
        *(half8_t*)&s_qh[(16 + c16) * kHStride + 32 * c + 8 * g] = yl;
      } else {
        qhi[c] = yh;
        qlo[c] = yl;
      }
    }
    if constexpr (kWide) __syncthreads();
  } else {
#pragma unroll
    for (int c = 0; c < D / 16; ++c) qf[c] = *(const float4_t*)&s_q[c16 * kQStride + 16 * c + 4 * g];
  }

  float m = -INFINITY, l = 0.0f;  // of this lane's slots, maximum in log2 units shared by the column
  float4_t acc[kNv];
#pragma unroll
  for (int n = 0; n < kNv; ++n) acc[n] = float4_t{0.f, 0.f, 0.f, 0.f};

  // Scores of the step at p0; the products are left to step().
  auto scores = [&](const Step<KV, D>& x, float (&sc)[kNs]) JMA_INL {
    float4_t s[kF16 ? 2 : 1] = {};
    if constexpr (kF16) {
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        const half8_t hi = kWide ? *(const half8_t*)&s_qh[c16 * kHStride + 32 * c + 8 * g] : qhi[kWide ? 0 : c];
        const half8_t lo = kWide ? *(const half8_t*)&s_qh[(16 + c16) * kHStride + 32 * c + 8 * g] : qlo[kWide ? 0 : c];
#pragma unroll
        for (int b = 0; b < 2; ++b) s[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.k[b][c], lo, s[b], 0, 0, 0);
#pragma unroll
        for (int b = 0; b < 2; ++b) s[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.k[b][c], hi, s[b], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int c = 0; c < D / 16; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.k[c][e], qf[c][e], s[0], 0, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < kNs; ++e) sc[e] = s[e >> 2][e & 3];
  };
  auto step = [&](Step<KV, D>& x, uint32_t p0, float (&sc)[kNs], auto robust) JMA_INL {
    if (p0 + kStep - 1 > pos0 || p0 < first_visible(pos1, a.window)) {
#pragma unroll
      for (int e = 0; e < kNs; ++e) {
        const uint32_t p = p0 + kNs * g + e;
        sc[e] = p >= cfirst && p <= cpos ? sc[e] : -INFINITY;
      }
    }
    float tmax = sc[0];
#pragma unroll
    for (int e = 1; e < kNs; ++e) tmax = fmaxf(tmax, sc[e]);
    tmax = max_groups(tmax) * factor;
    // The running maximum rises only by more than 2^8: most steps rescale nothing.
    const bool up = m == -INFINITY ? tmax > -INFINITY : tmax > m + 8.0f;
    if (__ballot(up) != 0) {
      const float mn = up ? tmax : m;
      const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int n = 0; n < kNv; ++n) acc[n] *= alpha;
    }
    const float shift = (kF16 ? 6.0f : 0.0f) - (m == -INFINITY ? 0.0f : m);
    float pr[kNs];
#pragma unroll
    for (int e = 0; e < kNs; ++e) {
      pr[e] = __builtin_amdgcn_exp2f(fmaf(sc[e], factor, shift));
      l += pr[e];
    }
    half8_t ph, pl;
    if constexpr (kF16) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        _Float16 hi, lo;
        halves(pr[e], hi, lo);
        ph[e] = hi;
        pl[e] = lo;
      }
    }
    auto product = [&](const auto& v, float4_t o) JMA_INL {
      if constexpr (kF16) {
        o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl, o, 0, 0, 0);
        o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph, o, 0, 0, 0);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) o = __builtin_amdgcn_mfma_f32_16x16x4f32(v[e], pr[e], o, 0, 0, 0);
      }
      return o;
    };
    if constexpr (decltype(robust)::value) {
      std::conditional_t<kF16, half8_t, float4_t> sees;
#pragma unroll
      for (int e = 0; e < kNs; ++e) {
        const uint32_t p = p0 + kNs * g + e;
        sees[e] = p >= cfirst && p <= cpos ? 1.0f : 0.0f;
      }
#pragma unroll
      for (int n = 0; n < kNv; ++n) {
        auto is = x.v[n];
        split_finite(x.v[n], is);
        float4_t found = {0.f, 0.f, 0.f, 0.f};
        if constexpr (kF16) {
          found = __builtin_amdgcn_mfma_f32_16x16x32_f16(is, sees, found, 0, 0, 0);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) found = __builtin_amdgcn_mfma_f32_16x16x4f32(is[e], sees[e], found, 0, 0, 0);
        }
        acc[n] = product(x.v[n], acc[n]);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][e] = found[e] > 0.0f ? NAN : acc[n][e];
      }
    } else {
#pragma unroll
      for (int n = 0; n < kNv; ++n) acc[n] = product(x.v[n], acc[n]);
    }
  };
  // Step x at p; the next one, y, is loaded meanwhile.
  auto half_loop = [&](Step<KV, D>& x, const Place& px, Step<KV, D>& y, Place& py) JMA_INL {
    const uint32_t tn = t + kW;
    if (!kWide && tn < t1) {
      if (++i == 64) {
        fetch_pages(tn);
        i = 0;
      }
      py = placed(tn, i);
      y.load_k(kbase + py.at, tn & 1, c16, g);
      y.load_v(vbase + py.at, tn & 1, c16, g);
    }
    float sc[kNs];
    const uint32_t p0 = px.p0;
    if (kWide) x.load_v(vbase + px.at, t & 1, c16, g);
    if (kFused && p0 == new_p0) {
      x.patch_k(new_k, new_r, c16, g);
      x.patch_v(new_v, new_r, c16, g);
    }
    scores(x, sc);
    if (kWide && tn < t1) {
      if (++i == 64) {
        fetch_pages(tn);
        i = 0;
      }
      py = placed(tn, i);
      x.load_k(kbase + py.at, tn & 1, c16, g);
    }
    if (p0 != kNoPage) step(x, p0, sc, std::false_type{});
    t = tn;
  };
  const uint32_t t_first = t;
  if constexpr (kWide) {
    while (t < t1) {
      Place next = {0, kNoPage};
      half_loop(xa, pa, xa, next);
      pa = next;
    }
  } else {
    while (t < t1) {
      half_loop(xa, pa, xb, pb);
      if (t >= t1) break;
      half_loop(xb, pb, xa, pa);
    }
  }

  float odd = 0.0f;
#pragma unroll
  for (int n = 0; n < kNv; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) odd = fmaf(acc[n][e], 0.0f, odd);
  if (__ballot(odd != 0.0f) != 0) {
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int n = 0; n < kNv; ++n) acc[n] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (t = t_first; t < t1; t += kW) {
      const uint32_t number = __builtin_amdgcn_readfirstlane(kSelected ? listed(t >> steps_log2) : t >> steps_log2);
      if (number == kNoPage) continue;
      const uint32_t page = __builtin_amdgcn_readfirstlane(table[number]);
      if (page >= a.kv.pages) continue;
      const uint32_t p0 = (number << page_log2) + (t & ((1u << steps_log2) - 1)) * kStep;
      const uint64_t at = place(t, page);
      xa.load_k(kbase + at, t & 1, c16, g);
      xa.load_v(vbase + at, t & 1, c16, g);
      if (kFused && p0 == new_p0) {
        xa.patch_k(new_k, new_r, c16, g);
        xa.patch_v(new_v, new_r, c16, g);
      }
      float sc[kNs];
      scores(xa, sc);
      step(xa, p0, sc, std::true_type{});
    }
  }

  // The waves' states meet in LDS.
  l = sum_groups(l);
#pragma unroll
  for (int n = 0; n < kNv; ++n)
    *(float4_t*)&s_acc[wave][c16][16 * n + 4 * g] = acc[n];
  if (g == 0) {
    s_ml[wave][c16][0] = m;
    s_ml[wave][c16][1] = l;
  }
  __syncthreads();

  const uint32_t cols = rows * heads;
  const uint64_t unit = (uint64_t)blockIdx.z * gridDim.y + blockIdx.y;
  float* part = a.part + (ch.part0 + (uint64_t)blockIdx.y * ch.nsplit) * (16 * (D + 4));  // this block's states
  const __amdgpu_buffer_rsrc_t rs = part_rsrc(part);
  float* out = a.out + (qrow * a.num_heads + kvh * a.group + 16 * hg) * D;
  auto finish = [&](uint32_t c, uint32_t e, const float4_t& o, float sum) JMA_INL {
    const uint32_t r = c / heads, h = c % heads;
    if (e == 0 && !(sum > 0.0f && sum < INFINITY)) report(a.err, kErrNonFinite);
    *(float4_t*)(out + ((uint64_t)r * a.num_heads + h) * D + e) = o * (sum > 0.0f ? 1.0f / sum : sum);
  };
  for (uint32_t k = threadIdx.x; k < cols * (D / 4); k += kThreads) {
    const uint32_t c = k / (D / 4), e = 4 * (k % (D / 4));
    float M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int w = 0; w < kW; ++w) M = fmaxf(M, s_ml[w][c][0]);
    float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      const float wm = s_ml[w][c][0], f = wm == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(wm - M);
      L = fmaf(s_ml[w][c][1], f, L);
      const float4_t x = *(const float4_t*)&s_acc[w][c][e];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = fmaf(x[j], f, o[j]);
    }
    if (ns == 1) {
      finish(c, e, o, L);
    } else {
      const uint32_t at = ((split * 16 + c) * (D + 4) + e) * 4;
      store_part(rs, at, o);
      if (e == 0) store_part(rs, at + D * 4, float4_t{M, L, 0.f, 0.f});
    }
  }
  if (ns == 1) return;
  // The states are acknowledged (visible device-wide) before the ticket is taken; the last workgroup
  // of the unit joins them in split order, whichever it is.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) s_ticket = __hip_atomic_fetch_add(&a.tickets[unit], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (s_ticket + 1 != ns) return;
  if (threadIdx.x == 0) __hip_atomic_store(&a.tickets[unit], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // Two round trips: every split's (m, l), and its share of O, eight splits' words in flight.
  float (*s_all)[16][2] = (float (*)[16][2])s_acc_mem;  // [split][column]
  for (uint32_t k = threadIdx.x; k < ns * 16; k += kThreads) {
    const float4_t ml = load_part(rs, ((k / 16 * 16 + min(k % 16, cols - 1)) * (D + 4) + D) * 4);
    s_all[k / 16][k % 16][0] = ml[0];
    s_all[k / 16][k % 16][1] = ml[1];
  }
  __syncthreads();
  for (uint32_t k = threadIdx.x; k < cols * (D / 4); k += kThreads) {
    const uint32_t c = k / (D / 4), e = 4 * (k % (D / 4));
    float M = -INFINITY, L = 0.0f;
    float4_t o = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t s0 = 0; s0 < ns; s0 += 8) {
      float4_t x[8];
#pragma unroll
      for (uint32_t i8 = 0; i8 < 8; ++i8) x[i8] = load_part(rs, ((min(s0 + i8, ns - 1) * 16 + c) * (D + 4) + e) * 4);
      if (s0 == 0)
        for (uint32_t s = 0; s < ns; ++s) M = fmaxf(M, s_all[s][c][0]);
#pragma unroll
      for (uint32_t i8 = 0; i8 < 8; ++i8) {
        if (s0 + i8 >= ns) break;
        const float ms = s_all[s0 + i8][c][0], f = ms == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ms - M);
        L = fmaf(s_all[s0 + i8][c][1], f, L);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = fmaf(x[i8][j], f, o[j]);
      }
    }
    finish(c, e, o, L);
  }
}

template <typename F>
hipError_t by_shape(bool f16, uint32_t d, F&& f) {
  switch (d) {
    case 32: return f16 ? f((_Float16)0, std::integral_constant<int, 32>{}) : f(0.0f, std::integral_constant<int, 32>{});
    case 64: return f16 ? f((_Float16)0, std::integral_constant<int, 64>{}) : f(0.0f, std::integral_constant<int, 64>{});
    case 128: return f16 ? f((_Float16)0, std::integral_constant<int, 128>{}) : f(0.0f, std::integral_constant<int, 128>{});
    case 256: return f16 ? f((_Float16)0, std::integral_constant<int, 256>{}) : f(0.0f, std::integral_constant<int, 256>{});
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t launch_paged_table(const PagedTableArgs& a, hipStream_t stream) {
  paged_table_kernel<<<1, 512, 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t launch_paged_append(const PagedAppendArgs& a, bool f16, uint32_t d, hipStream_t stream) {
  return by_shape(f16, d, [&](auto kv, auto dim) {
    using KV = decltype(kv);
    constexpr int D = decltype(dim)::value;
    const uint32_t heads = (a.q_out ? a.num_heads : 0) + 2 * a.kv.hkv;
    paged_append_kernel<KV, D><<<dim3(a.max_tiles, heads, a.chunks), 256, 0, stream>>>(a);
    if (a.kv.bounds != nullptr)
      paged_bounds_kernel<KV, D><<<dim3(a.max_pages, a.kv.hkv, a.chunks), 256, 0, stream>>>(a);
    return hipGetLastError();
  });
}

hipError_t launch_paged_select(const PagedSelectArgs& a, bool f16, uint32_t d, uint32_t max_pages, hipStream_t stream) {
  return by_shape(f16, d, [&](auto kv, auto dim) {
    using KV = decltype(kv);
    constexpr int D = decltype(dim)::value;
    const uint32_t wgs = (max_pages + kSelectPages - 1) / kSelectPages;
    const uint32_t lds = a.raw ? a.group * (D + 4) * 4 : 0;
    paged_select_kernel<KV, D><<<dim3(wgs, a.max_rows * a.kv.hkv, a.chunks), 256, lds, stream>>>(a);
    return hipGetLastError();
  });
}

hipError_t launch_paged_attend(const PagedAttendArgs& a, bool f16, uint32_t d, hipStream_t stream) {
  return by_shape(f16, d, [&](auto kv, auto dim) {
    using KV = decltype(kv);
    constexpr int D = decltype(dim)::value;
    const bool fused = a.k_new != nullptr;
    const dim3 grid(a.max_splits + (fused ? 1 : 0), a.max_blocks * a.kv.hkv * a.head_groups, a.chunks);
    constexpr uint32_t kThreads = 64 * paged_waves(D);
    if (fused && a.pages != nullptr) paged_attend_kernel<KV, D, true, true><<<grid, kThreads, 0, stream>>>(a);
    else if (fused) paged_attend_kernel<KV, D, false, true><<<grid, kThreads, 0, stream>>>(a);
    else if (a.pages != nullptr) paged_attend_kernel<KV, D, true, false><<<grid, kThreads, 0, stream>>>(a);
    else paged_attend_kernel<KV, D, false, false><<<grid, kThreads, 0, stream>>>(a);
    return hipGetLastError();
  });
}

}  // namespace jma
