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
  const float* w = is_q ? a.q_norm_w : is_k ? a.k_norm_w : nullptr;
  const bool v_norm = !is_q && !is_k && a.v_norm != 0;
  if (w != nullptr || v_norm) {
#pragma clang fp contract(off)
    if (threadIdx.x < n) {
      const float* x = s_x[threadIdx.x];
      float ss = 0.0f;
#pragma unroll 4
      for (int e = 0; e < D; e += 4) {
        const float4_t v = *(const float4_t*)(x + e);
#pragma unroll
        for (int i = 0; i < 4; ++i) ss = ss + v[i] * v[i];
      }
      const double mean = (double)(ss / (float)D + a.norm_eps);
      s_scale[threadIdx.x] = v_norm ? (float)(1.0 / sqrt(mean)) : 1.0f / (float)sqrt(mean);
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n * D; i += 256) {
      const uint32_t r = i / D, e = i % D;
      float x = s_x[r][e] * s_scale[r];
      if (!v_norm) x = x * w[e];
      s_x[r][e] = x;
    }
    __syncthreads();
  }
  if ((is_q || is_k) && a.cos_t != nullptr) {
    for (uint32_t i = threadIdx.x; i < n * a.pairs; i += 256) {
      const uint32_t r = i / a.pairs, j = i % a.pairs;
      const uint64_t at = (uint64_t)(p0 + r) * a.pairs + j;
      const uint32_t e0 = a.neox ? j : 2 * j, e1 = a.neox ? j + a.pairs : 2 * j + 1;
      float x0 = s_x[r][e0], x1 = s_x[r][e1];
      rotate_pair(x0, x1, a.cos_t[at], a.sin_t[at]);
      s_x[r][e0] = x0;
      s_x[r][e1] = x1;
    }
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

// Workgroup = (page that a chunk wrote to, kv head, chunk): the smallest and the largest of the page's
// key elements, over all of its filled slots (those before the chunk's end). Exact, whatever the
// order: no sums. A NaN key element is left out of them.
template <typename KV, int D>
__global__ __launch_bounds__(256) void paged_bounds_kernel(const PagedAppendArgs a) {
  const PagedChunk c = a.c[blockIdx.z];
  if (c.rows == 0) return;
  const uint32_t number = (c.start >> a.kv.page_log2) + blockIdx.x, end = c.start + c.rows;
  if (number > (end - 1) >> a.kv.page_log2) return;
  const uint32_t filled = min(end - (number << a.kv.page_log2), 1u << a.kv.page_log2);
  const uint32_t page = a.kv.table[(uint64_t)c.seq * a.kv.table_stride + number];
  const uint32_t head = blockIdx.y;
  const KV* src = (const KV*)a.kv.k + paged_base(page, a.kv.hkv, head, a.kv.page_log2, D);
  constexpr bool kF16 = std::is_same<KV, _Float16>::value;
  constexpr uint32_t kW = kF16 ? 8 : 4, kPieces = D / kW, kLanes = 256 / kPieces;
  typedef KV kv16_t __attribute__((ext_vector_type(kW)));
  const uint32_t piece = threadIdx.x % kPieces, lane = threadIdx.x / kPieces;
  float lo[kW], hi[kW];
#pragma unroll
  for (uint32_t t = 0; t < kW; ++t) lo[t] = INFINITY, hi[t] = -INFINITY;
  for (uint32_t s = lane; s < filled; s += kLanes) {
    const kv16_t x = *(const kv16_t*)(src + paged_k_index(s, piece * kW, D, kF16));
#pragma unroll
    for (uint32_t t = 0; t < kW; ++t) {
      lo[t] = fminf(lo[t], (float)x[t]);
      hi[t] = fmaxf(hi[t], (float)x[t]);
    }
  }
  __shared__ float s_lo[kLanes][D], s_hi[kLanes][D];
#pragma unroll
  for (uint32_t t = 0; t < kW; ++t) {
    s_lo[lane][piece * kW + t] = lo[t];
    s_hi[lane][piece * kW + t] = hi[t];
  }
  __syncthreads();
  KV* dst = (KV*)a.kv.bounds + ((uint64_t)page * a.kv.hkv + head) * 2 * D;
  for (uint32_t i = threadIdx.x; i < 2 * D; i += 256) {
    const uint32_t e = i % D;
    float x = i < D ? s_lo[0][e] : s_hi[0][e];
    for (uint32_t l = 1; l < kLanes; ++l) x = i < D ? fminf(x, s_lo[l][e]) : fmaxf(x, s_hi[l][e]);
    dst[i] = (KV)x;
  }
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

constexpr uint32_t kPickRounds = 16, kPickPages = 256 * kPickRounds;  // keys a workgroup holds in registers

// The pages of one (row, kv head), ascending: the first `first`, the last `last` and the `top` others of
// the largest keys, of equal ones the lowest. The key of the last page taken is narrowed by eight
// bits a pass, from the highest bit in which any two keys differ, until every key that shares the bits
// found so far is taken (two or three passes: the keys are spread). n > first + last + top.
__device__ __forceinline__ void pick_pages(const uint64_t* keys, uint32_t n, uint32_t top, uint32_t first, uint32_t last,
                                           uint32_t* out) {
  __shared__ uint32_t s_hist[256], s_found[3], s_any[4][2], s_sum[4];
  __shared__ uint32_t s_count[4 * kPickRounds];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint64_t k[kPickRounds];
  auto candidate = [&](uint32_t p) JMA_INL { return p >= first && p + last < n; };
  auto load = [&](uint32_t base) JMA_INL {
#pragma unroll
    for (uint32_t i = 0; i < kPickRounds; ++i) {
      const uint32_t p = base + 256 * i + tid;
      k[i] = 0;
      if (base + 256 * i < n && candidate(p)) k[i] = __hip_atomic_load(&keys[p], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
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
        const uint32_t mine = s_count[lane];
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
  const float* q = a.q + ((uint64_t)row * a.num_heads + kvh * a.group) * D + lane16 * kE;
  double best[kP];
  bool odd[kP];
#pragma unroll
  for (int i = 0; i < kP; ++i) best[i] = -INFINITY, odd[i] = false;
  for (uint32_t h = 0; h < a.group; ++h) {
    float x[kE];
#pragma unroll
    for (int e = 0; e < kE; ++e) x[e] = q[(uint64_t)h * D + e];
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
  pick_pages(keys, n, a.top, a.first, a.last, out);
}

// ================================================================ attention

// One step's K and V of one lane, in matrix-core operand order (below).
template <typename KV, int D>
struct Step;

template <int D>
struct Step<_Float16, D> {
  half8_t k[2][D / 32], v[D / 16];
  __device__ __forceinline__ void load(const _Float16* kt, const _Float16* vt, uint32_t, int c16, int g) {
    const uint32_t slot = 8 * (c16 >> 2) + (c16 & 3);
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int c = 0; c < D / 32; ++c) k[b][c] = *(const half8_t*)(kt + c * 1024 + (slot + 4 * b) * 32 + 8 * g);
#pragma unroll
    for (int n = 0; n < D / 16; ++n) v[n] = *(const half8_t*)(vt + (16 * n + c16) * 32 + 8 * g);
  }
};
template <int D>
struct Step<float, D> {
  float4_t k[D / 16], v[D / 16];
  __device__ __forceinline__ void load(const float* kt, const float* vt, uint32_t half, int c16, int g) {
#pragma unroll
    for (int c = 0; c < D / 16; ++c) k[c] = *(const float4_t*)(kt + c * 512 + (16 * half + c16) * 16 + 4 * g);
#pragma unroll
    for (int n = 0; n < D / 16; ++n) v[n] = *(const float4_t*)(vt + (16 * n + c16) * 32 + 16 * half + 4 * g);
  }
};

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
// Positions a column does not see are masked after the product, and values that are no finite number
// in a step that is masked in part reach only the columns that see them (0 x inf is no 0), as NaN.
template <typename KV, int D, bool kSelected>
__global__ __launch_bounds__(64 * paged_waves(D)) void paged_attend_kernel(const PagedAttendArgs a) {
  constexpr bool kF16 = std::is_same<KV, _Float16>::value;
  constexpr int kW = paged_waves(D), kNs = kF16 ? 8 : 4, kNv = D / 16;
  constexpr uint32_t kStep = kF16 ? 32 : 16;
  constexpr int kQStride = D + 4;
  __shared__ __attribute__((aligned(16))) float s_q[16][kQStride];
  __shared__ __attribute__((aligned(16))) float s_acc[kW][16][D];
  __shared__ float s_ml[kW][16][2];
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
  const uint32_t ns = (t1 - t0 + a.tiles_per_split - 1) / a.tiles_per_split, split = blockIdx.x;
  if (split >= ns) return;
  t0 += split * a.tiles_per_split;
  t1 = min(t1, t0 + a.tiles_per_split);

  const int lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // This lane's column; one past the block's (row, head) pairs holds zeros and is never stored.
  const uint32_t col_row = c16 / heads;
  const uint32_t cpos = pos0 + min(col_row, rows - 1), cfirst = first_visible(cpos, a.window);
  const uint64_t qrow = (uint64_t)ch.row0 + row0;

  // q of the block's columns, in LDS.
  const float* q = a.q + (qrow * a.num_heads + kvh * a.group + 16 * hg) * D;
  for (uint32_t i = threadIdx.x; i < 16 * (D / 4); i += 64 * kW) {
    const uint32_t c = i / (D / 4), e = 4 * (i % (D / 4)), r = c / heads, h = c % heads;
    float4_t x = {0.f, 0.f, 0.f, 0.f};
    if (r < rows) x = *(const float4_t*)(q + ((uint64_t)r * a.num_heads + h) * D + e);
    *(float4_t*)&s_q[c][e] = x;
  }

  // The page of each of this wave's next 64 steps is held by the lane of that number: its logical
  // number and where it is.
  const uint32_t* table = a.kv.table + (uint64_t)ch.seq * a.kv.table_stride;
  const uint32_t* list = kSelected ? a.pages + ((qrow * hkv) + kvh) * a.budget : nullptr;
  uint32_t my_page = 0, my_number = 0;
  auto fetch_pages = [&](uint32_t t) JMA_INL {
    const uint32_t mine = t + lane * kW;
    my_page = kNoPage;
    if (mine < t1) {
      if (kSelected) {
        const uint32_t i = mine >> steps_log2;
        my_number = list[i];
        // A list made by the caller may hold anything: numbers past the row's position, or not
        // ascending, are reported and left out.
        if (my_number != kNoPage) {
          const bool ok = my_number <= cpos >> page_log2 && (i == 0 || list[i - 1] < my_number);
          if (!ok) report(a.err, kErrBadPage);
          if (ok) my_page = table[my_number];
        }
      } else {
        my_number = mine >> steps_log2;
        my_page = table[my_number];
      }
    }
  };
  const KV* kbase = (const KV*)a.kv.k;
  const KV* vbase = (const KV*)a.kv.v;
  // Loads step t (the i-th since fetch_pages) and returns its first position, or kNoPage.
  auto load = [&](Step<KV, D>& x, uint32_t t, uint32_t i) JMA_INL -> uint32_t {
    const uint32_t page = __builtin_amdgcn_readlane(my_page, i);
    const uint32_t number = __builtin_amdgcn_readlane(my_number, i);
    if (page >= a.kv.pages) return kNoPage;
    const uint32_t in = t & ((1u << steps_log2) - 1), tile = kF16 ? in : in >> 1;
    const uint64_t at = paged_base(page, hkv, kvh, page_log2, D) + tile * kTileSlots * D;
    x.load(kbase + at, vbase + at, in & 1, c16, g);
    return (number << page_log2) + in * kStep;
  };

  uint32_t t = t0 + wave;
  Step<KV, D> cur, nxt;
  uint32_t p_cur = kNoPage, p_nxt = kNoPage, i = 0;
  if (t < t1) {
    fetch_pages(t);
    p_cur = load(cur, t, 0);
  }
  __syncthreads();

  // Q operand and the factor of each column's scores.
  half8_t qhi[kF16 ? D / 32 : 1], qlo[kF16 ? D / 32 : 1];
  float4_t qf[kF16 ? 1 : D / 16];
  float factor = a.scale;
  if constexpr (kF16) {
    float top = 0.0f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const float4_t x0 = *(const float4_t*)&s_q[c16][32 * c + 8 * g], x1 = *(const float4_t*)&s_q[c16][32 * c + 8 * g + 4];
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
      const float4_t x0 = *(const float4_t*)&s_q[c16][32 * c + 8 * g], x1 = *(const float4_t*)&s_q[c16][32 * c + 8 * g + 4];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = __builtin_amdgcn_ldexpf(e < 4 ? x0[e & 3] : x1[e & 3], 14 - ex);
        qhi[c][e] = (_Float16)x;
        qlo[c][e] = (_Float16)(x - (float)qhi[c][e]);
      }
    }
  } else {
#pragma unroll
    for (int c = 0; c < D / 16; ++c) qf[c] = *(const float4_t*)&s_q[c16][16 * c + 4 * g];
  }

  float m = -INFINITY, l = 0.0f;  // of this lane's slots, maximum in log2 units shared by the column
  float4_t acc[kNv];
#pragma unroll
  for (int n = 0; n < kNv; ++n) acc[n] = float4_t{0.f, 0.f, 0.f, 0.f};

  auto step = [&](const Step<KV, D>& x, uint32_t p0) JMA_INL {
    float4_t s[kF16 ? 2 : 1];
#pragma unroll
    for (int b = 0; b < (kF16 ? 2 : 1); ++b) {
      s[b] = float4_t{0.f, 0.f, 0.f, 0.f};
      if constexpr (kF16) {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) s[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.k[b][c], qlo[c], s[b], 0, 0, 0);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) s[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x.k[b][c], qhi[c], s[b], 0, 0, 0);
      } else {
#pragma unroll
        for (int c = 0; c < D / 16; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.k[c][e], qf[c][e], s[b], 0, 0, 0);
      }
    }
    const bool whole = p0 + kStep - 1 <= pos0 && p0 >= first_visible(pos1, a.window);
    float sc[kNs];
#pragma unroll
    for (int e = 0; e < kNs; ++e) {
      sc[e] = s[e >> 2][e & 3];
      if (!whole) {
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
    const float shift = kF16 ? 6.0f - (m == -INFINITY ? 0.0f : m) : (m == -INFINITY ? 0.0f : -m);
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
        ph[e] = (_Float16)pr[e];
        pl[e] = (_Float16)(pr[e] - (float)ph[e]);
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
    if (!whole) {
      // Values here that are no finite number are left out of the product, and what they make of the
      // columns that see them is added: a second product counts, for each output, the ones its column sees.
      uint32_t odd = 0;
#pragma unroll
      for (int n = 0; n < kNv; ++n) odd |= not_finite(x.v[n]);
      if (__ballot(odd != 0) != 0) {
        std::conditional_t<kF16, half8_t, float4_t> sees;
#pragma unroll
        for (int e = 0; e < kNs; ++e) {
          const uint32_t p = p0 + kNs * g + e;
          sees[e] = p >= cfirst && p <= cpos ? 1.0f : 0.0f;
        }
#pragma unroll
        for (int n = 0; n < kNv; ++n) {
          auto v = x.v[n], is = x.v[n];
          split_finite(v, is);
          float4_t count = {0.f, 0.f, 0.f, 0.f};
          if constexpr (kF16) {
            count = __builtin_amdgcn_mfma_f32_16x16x32_f16(is, sees, count, 0, 0, 0);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) count = __builtin_amdgcn_mfma_f32_16x16x4f32(is[e], sees[e], count, 0, 0, 0);
          }
          acc[n] = product(v, acc[n]);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n][e] = count[e] > 0.0f ? NAN : acc[n][e];
        }
        return;
      }
    }
#pragma unroll
    for (int n = 0; n < kNv; ++n) acc[n] = product(x.v[n], acc[n]);
  };

  while (t < t1) {
    const uint32_t tn = t + kW;
    if (tn < t1) {
      if (++i == 64) {
        fetch_pages(tn);
        i = 0;
      }
      p_nxt = load(nxt, tn, i);
    }
    if (p_cur != kNoPage) step(cur, p_cur);
    cur = nxt;
    p_cur = p_nxt;
    t = tn;
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
  for (uint32_t k = threadIdx.x; k < cols * (D / 4); k += 64 * kW) {
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
  float (*s_all)[16][2] = (float (*)[16][2])s_acc;  // [split][column]
  for (uint32_t k = threadIdx.x; k < ns * 16; k += 64 * kW) {
    const float4_t ml = load_part(rs, ((k / 16 * 16 + min(k % 16, cols - 1)) * (D + 4) + D) * 4);
    s_all[k / 16][k % 16][0] = ml[0];
    s_all[k / 16][k % 16][1] = ml[1];
  }
  __syncthreads();
  for (uint32_t k = threadIdx.x; k < cols * (D / 4); k += 64 * kW) {
    const uint32_t c = k / (D / 4), e = 4 * (k % (D / 4));
    float M = -INFINITY, L = 0.0f;
    float4_t o = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t s0 = 0; s0 < ns; s0 += 8) {
      float4_t x[8];
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) x[i] = load_part(rs, ((min(s0 + i, ns - 1) * 16 + c) * (D + 4) + e) * 4);
      if (s0 == 0)
        for (uint32_t s = 0; s < ns; ++s) M = fmaxf(M, s_all[s][c][0]);
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) {
        if (s0 + i >= ns) break;
        const float ms = s_all[s0 + i][c][0], f = ms == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ms - M);
        L = fmaf(s_all[s0 + i][c][1], f, L);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = fmaf(x[i][j], f, o[j]);
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
    paged_select_kernel<KV, D><<<dim3(wgs, a.max_rows * a.kv.hkv, a.chunks), 256, 0, stream>>>(a);
    return hipGetLastError();
  });
}

hipError_t launch_paged_attend(const PagedAttendArgs& a, bool f16, uint32_t d, hipStream_t stream) {
  return by_shape(f16, d, [&](auto kv, auto dim) {
    using KV = decltype(kv);
    constexpr int D = decltype(dim)::value;
    const dim3 grid(a.max_splits, a.max_blocks * a.kv.hkv * a.head_groups, a.chunks);
    if (a.pages != nullptr) paged_attend_kernel<KV, D, true><<<grid, 64 * paged_waves(D), 0, stream>>>(a);
    else paged_attend_kernel<KV, D, false><<<grid, 64 * paged_waves(D), 0, stream>>>(a);
    return hipGetLastError();
  });
}

}  // namespace jma
