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
// order, pairs are rotated, and keys and values are stored in the page's layout. All that a workgroup reads
// (rows, factors of their positions, norm weight) is in flight before the first is used: one memory round
// trip, which bounds it up to some hundred rows, and the bytes of q, k and v beyond (2048 rows of 32 + 16
// heads of 128: 20 us, 4.5 TB/s; read piece by piece it took 24).
template <typename KV, int D>
__global__ __launch_bounds__(256) void paged_append_kernel(const PagedAppendArgs a) {
  const PagedChunk c = a.c[blockIdx.z];
  if (c.rows == 0) return;
  constexpr uint32_t kT = paged_append_rows(D);
  const uint32_t tile = c.start / kT + blockIdx.x;
  const uint32_t p0 = max(c.start, tile * kT), p1 = min(c.start + c.rows, (tile + 1) * kT);
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
  __shared__ __attribute__((aligned(16))) float s_x[kT][kStride];
  __shared__ float s_scale[kT];
  const uint32_t tid = threadIdx.x;
  constexpr uint32_t kLoads = kT * (D / 4) / 256, kRows = 256 / (D / 4);  // rows of 256 pieces of 16 bytes
  constexpr uint32_t kPairs = kT * (D / 2) / 256, kPairRows = 256 / (D / 2);
  const bool rotates = (is_q || is_k) && a.rot.cos_t != nullptr && a.rot.pairs > 0;
  const float* w = is_q ? a.rot.q_norm_w : is_k ? a.rot.k_norm_w : nullptr;
  const bool v_norm = !is_q && !is_k && a.rot.v_norm != 0;
  float4_t x[kLoads];
  float cs[kPairs], sn[kPairs], weight = 1.0f;
  const uint32_t row = tid / (D / 4), e4 = 4 * (tid % (D / 4)), pair_row = tid / (D / 2), pair = tid % (D / 2);
#pragma unroll
  for (uint32_t i = 0; i < kLoads; ++i)
    if (kRows * i < n) x[i] = *(const float4_t*)(src + (uint64_t)min(row + kRows * i, n - 1) * heads * D + e4);
  if (rotates) {
    const uint64_t at = (uint64_t)p0 * a.rot.pairs + min(pair, a.rot.pairs - 1);
#pragma unroll
    for (uint32_t i = 0; i < kPairs; ++i)
      if (kPairRows * i < n) {
        const uint64_t f = at + (uint64_t)min(pair_row + kPairRows * i, n - 1) * a.rot.pairs;
        cs[i] = a.rot.cos_t[f];
        sn[i] = a.rot.sin_t[f];
      }
  }
  if (w != nullptr) weight = w[tid % D];
#pragma unroll
  for (uint32_t i = 0; i < kLoads; ++i)
    if (row + kRows * i < n) *(float4_t*)&s_x[row + kRows * i][e4] = x[i];
  __syncthreads();
  if (w != nullptr || v_norm) {
#pragma clang fp contract(off)
    if (tid < n) s_scale[tid] = head_scale<D>(s_x[tid], a.rot.norm_eps, v_norm);
    __syncthreads();
    for (uint32_t r = tid / D; r < n; r += 256 / D) {
      float y = s_x[r][tid % D] * s_scale[r];
      if (!v_norm) y = y * weight;
      s_x[r][tid % D] = y;
    }
    __syncthreads();
  }
  if (rotates) {
    const uint32_t e0 = a.rot.neox ? pair : 2 * pair, e1 = a.rot.neox ? pair + a.rot.pairs : 2 * pair + 1;
    if (pair < a.rot.pairs) {
#pragma unroll
      for (uint32_t i = 0; i < kPairs; ++i) {
        const uint32_t r = pair_row + kPairRows * i;
        if (r >= n) break;
        float x0 = s_x[r][e0], x1 = s_x[r][e1];
        rotate_pair(x0, x1, cs[i], sn[i]);
        s_x[r][e0] = x0;
        s_x[r][e1] = x1;
      }
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
    if (n == kT) {
      constexpr uint32_t kW = kF16 ? 8 : 4;
      for (uint32_t i = threadIdx.x; i < kT / kW * D; i += 256) {
        const uint32_t e = i / (kT / kW), r = (i % (kT / kW)) * kW;
        typedef KV kv16_t __attribute__((ext_vector_type(kW)));
        kv16_t y;
#pragma unroll
        for (uint32_t t = 0; t < kW; ++t) y[t] = (KV)s_x[r + t][e];
        *(kv16_t*)(dst + e * kTileSlots + at + r) = y;
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

template <int kCtrl>
__device__ __forceinline__ float row_moved(float x) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(x), kCtrl, 0xF, 0xF, false));
}
__device__ __forceinline__ float max_wave(float x) {
  x = fmaxf(x, row_moved<0x128>(x));
  x = fmaxf(x, row_moved<0x124>(x));
  x = fmaxf(x, row_moved<0x122>(x));
  x = fmaxf(x, row_moved<0x121>(x));
  return max_groups(x);
}

__device__ __forceinline__ uint32_t lanes_below(uint64_t mask, uint32_t lane) {
  return (uint32_t)__popcll(mask & ((1ull << lane) - 1));
}

// What picks a row's pages works on, in LDS: a wave's share.
constexpr uint32_t kHeldScores = 1024, kPickBins = 512, kPickNear = 64;
struct PickSpace {
  uint32_t hist[4][kPickBins];
  float score[4][kHeldScores];
  uint32_t near[4][kPickNear];    // pages whose scores lie too near the border to be told apart in 32 bits
  uint64_t exact[4][kPickNear];
  float least[4], most[4];
  uint32_t odd[4], sure[4], count[4];
};

// 64-bit keys of a row's candidates first <= p < end, at keys[p], read again in every pass.
struct Keys {
  const uint64_t* keys;
  uint32_t first, end, lane;
  template <typename F>
  __device__ __forceinline__ void each(F&& f) {  // f(page, key, whether there is such a candidate)
    for (uint32_t base = first; base < end; base += 256) {
      uint64_t k[4];
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i)  // unconditional, so that all are in flight together
        k[i] = __hip_atomic_load(&keys[min(base + 64 * i + lane, end - 1)], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) f(base + 64 * i + lane, k[i], base + 64 * i + lane < end);
    }
  }
};

// Sum over this lane and the ones before it.
template <int kCtrl, int kRows>
__device__ __forceinline__ uint32_t lane_moved(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kCtrl, kRows, 0xF, false);
}
__device__ __forceinline__ uint32_t sum_up_to(uint32_t x) {
  x += lane_moved<0x111, 0xF>(x);  // row_shr by 1, 2, 4, 8
  x += lane_moved<0x112, 0xF>(x);
  x += lane_moved<0x114, 0xF>(x);
  x += lane_moved<0x118, 0xF>(x);
  x += lane_moved<0x142, 0xA>(x);  // lane 15 of a row to the next, then lane 31 to the upper half
  x += lane_moved<0x143, 0xC>(x);
  return x;
}

// Which of the 64 kPerLane bins of a histogram holds the need-th largest; then need is its rank within the bin.
template <uint32_t kPerLane>
__device__ __forceinline__ void border_bin(const uint32_t* hist, uint32_t lane, uint32_t& need, uint32_t& bin, uint32_t& count) {
  const uint32_t b0 = kPerLane * (63 - lane);  // the highest bins first
  uint32_t c[kPerLane], mine = 0;
#pragma unroll
  for (uint32_t i = 0; i < kPerLane; i += 4) {
    const uint4 x = *(const uint4*)&hist[b0 + i];
    c[i] = x.x, c[i + 1] = x.y, c[i + 2] = x.z, c[i + 3] = x.w;
    mine += x.x + x.y + x.z + x.w;
  }
  const uint32_t upto = sum_up_to(mine);
  const int at = __ffsll((long long)__ballot(upto >= need)) - 1;
  uint32_t left = upto - mine, b = 0, n = 0, rest = 0;
#pragma unroll
  for (int i = (int)kPerLane - 1; i >= 0; --i) {
    const bool here = left < need && left + c[i] >= need;
    b = here ? b0 + i : b;
    n = here ? c[i] : n;
    rest = here ? need - left : rest;
    left += c[i];
  }
  bin = __builtin_amdgcn_readlane(b, at);
  count = __builtin_amdgcn_readlane(n, at);
  need = __builtin_amdgcn_readlane(rest, at);
}

// The n-th largest of 64-bit keys: eight bits a pass, from the highest bit in which any two differ, until all
// keys that share the bits found are among the n largest.
__device__ __forceinline__ uint64_t nth_largest(Keys& keys, uint32_t n, uint32_t* hist) {
  const uint32_t lane = keys.lane;
  const uint64_t reference = __hip_atomic_load(&keys.keys[keys.first], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  uint32_t lo = 0, hi = 0;
  keys.each([&](uint32_t, uint64_t x, bool there) JMA_INL {
    if (!there) return;
    lo |= (uint32_t)(x ^ reference);
    hi |= (uint32_t)((x ^ reference) >> 32);
  });
#pragma unroll
  for (int m = 1; m < 64; m *= 2) {
    lo |= __shfl_xor(lo, m);
    hi |= __shfl_xor(hi, m);
  }
  int shift = hi ? 64 - __clz(hi) : lo ? 32 - __clz(lo) : 0;  // the bits in which keys differ
  if (shift == 0) return reference;
  uint64_t prefix = shift >= 64 ? 0 : reference >> shift;
  uint32_t need = n;
  while (shift > 0) {
    const int bits = min(8, shift), next = shift - bits;
#pragma unroll
    for (int i = 0; i < 4; ++i) hist[64 * i + lane] = 0;
    __builtin_amdgcn_wave_barrier();
    keys.each([&](uint32_t, uint64_t x, bool there) JMA_INL {
      if (there && (shift >= 64 || x >> shift == prefix)) atomicAdd(&hist[(uint32_t)(x >> next) & ((1u << bits) - 1)], 1u);
    });
    __builtin_amdgcn_wave_barrier();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    uint32_t bin, count;
    border_bin<4>(hist, lane, need, bin, count);
    prefix = shift >= 64 ? (uint64_t)bin : prefix << bits | bin;
    shift = next;
    if (need == count) break;
  }
  if (shift == 0) return prefix;
  // All keys with these bits are taken: the smallest of them.
  uint64_t least = ~0ull;
  keys.each([&](uint32_t, uint64_t x, bool there) JMA_INL {
    if (there && x >> shift == prefix) least = x < least ? x : least;
  });
#pragma unroll
  for (int m = 1; m < 64; m *= 2) {
    const uint64_t x = __shfl_xor(least, m);
    least = x < least ? x : least;
  }
  return least;
}

// Workgroup = (64 pages, block of query rows x kv head, chunk). A page with bounds lo, hi scores
// sum_d max(q_d lo_d, q_d hi_d) for a query head, which no key of the page exceeds, and the largest of the
// heads' for a (row, kv head). That is the product of [lo, hi] with [min(q, 0), max(q, 0)]: 16 pages x 16
// columns (rows x heads) a matrix product, in 32 bits (f16 bounds: q as two halves, like the attention's).
//
// Which of two nearly equal pages is taken must not depend on a rounding. The 32-bit scores are off by at
// most eps = (2^-22 + (4 d + 16) 2^-23) |q|_1 max|bound|; with T the border score, pages above T + 2 eps are
// taken and pages below T - 2 eps are not, whatever the exact scores are, and the few between are scored
// again in 64 bits, where the products are exact (two to six of a thousand pages). Where they are more than
// 64, these go by keys of 64 bits in memory; where a score is not finite or out of range, all pages of the row.
//
// A wave takes 16 pages at a time, all their bounds in flight. One token of 32 heads of 64 over 1563 pages:
// 14 us, of which the bounds and their products 2.6, the scores' way to the last workgroup of the block
// to finish and its reading them 3.5, the pick (by its four waves) 5, the start and the lists' stores the
// rest: dependent round trips throughout, no unit busy. 61 rows of 12 heads of 128 over 626 pages (a wave
// picks a row) 25 us; scored in 64 bits throughout it was 45, and 17 for the token. Where all pages score
// the same, and so all are scored again four at a time, it takes 190 and 330 us.
template <typename KV, int D>
__global__ __launch_bounds__(256) void paged_select_kernel(const PagedSelectArgs a) {
  constexpr bool kF16 = std::is_same<KV, _Float16>::value;
  constexpr int kQStride = D + 4;
  const PagedChunk c = a.c[blockIdx.z];
  const uint32_t hkv = a.kv.hkv, kvh = blockIdx.y % hkv, r0 = blockIdx.y / hkv * a.rows_per_block;
  if (r0 >= c.rows) return;
  const uint32_t rows = min(a.rows_per_block, c.rows - r0);
  const uint32_t pos0 = c.start + r0, row0 = c.row0 + r0;
  auto pages_of = [&](uint32_t r) JMA_INL { return ((pos0 + r) >> a.kv.page_log2) + 1; };
  const uint32_t n1 = pages_of(rows - 1);
  if (blockIdx.x * kSelectPages >= n1) return;
  auto list_of = [&](uint32_t r) JMA_INL { return a.pages + ((uint64_t)(row0 + r) * hkv + kvh) * a.budget; };
  if (blockIdx.x == 0)  // rows that see no more pages than they may
    for (uint32_t r = 0; r < rows && pages_of(r) <= a.budget; ++r)
      for (uint32_t i = threadIdx.x; i < a.budget; i += 256) list_of(r)[i] = i < pages_of(r) ? i : kNoPage;
  if (n1 <= a.budget) return;
  const uint32_t wgs = min(gridDim.x, (n1 + kSelectPages - 1) / kSelectPages);
  const uint64_t block = ((uint64_t)blockIdx.z * a.max_blocks + blockIdx.y / hkv) * hkv + kvh;
  float* keys = a.keys + block * a.rows_per_block * paged_row_keys(a.key_stride);
  float* maxima = a.maxima + block * 4 * a.max_wgs;

  extern __shared__ __attribute__((aligned(16))) float s_queries[];  // raw: [group][D + 4]
  union Space {
    struct {
      float q[16 * kQStride], score[kSelectPages][17];
    };
    PickSpace pick;
  };
  __shared__ __attribute__((aligned(16))) Space s_mem;
  __shared__ float s_l1[16], s_scale[kSelectFloats / 32];
  __shared__ uint32_t s_last;
  float* const s_q = s_mem.q;
  PickSpace& space = s_mem.pick;

  const uint32_t tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c16 = lane & 15;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t* table = a.kv.table + (uint64_t)c.seq * a.kv.table_stride;
  auto bounds_of = [&](uint32_t p) JMA_INL { return (const KV*)a.kv.bounds + ((uint64_t)table[p] * hkv + kvh) * 2 * D; };

  const float* q = a.q + ((uint64_t)row0 * a.num_heads + kvh * a.group) * D;
  if (a.raw) {
    for (uint32_t i = tid; i < a.group * (D / 4); i += 256)
      *(float4_t*)&s_queries[i / (D / 4) * kQStride + 4 * (i % (D / 4))] = *(const float4_t*)(q + 4 * i);
    prepare_token<D, kQStride>(s_queries, s_scale, a.group, 0, false, a.rot, pos0, 256);
  }
  auto query = [&](uint32_t r, uint32_t h) JMA_INL -> const float* {
    return a.raw ? s_queries + h * kQStride : q + ((uint64_t)r * a.num_heads + h) * D;
  };
  constexpr int kCh = kF16 ? D / 32 : D / 16;  // operands of a bound
  typedef std::conditional_t<kF16, half8_t, float4_t> operand_t;
  constexpr int kE = kF16 ? 8 : 4;
  float most = 0.0f;
  for (uint32_t h0 = 0; h0 < a.group; h0 += 16) {
    const uint32_t heads = min(16u, a.group - h0);
    __syncthreads();
    for (uint32_t i = tid; i < 16 * (D / 4); i += 256) {
      const uint32_t col = i / (D / 4), e = 4 * (i % (D / 4)), r = col / heads;
      float4_t x = {0.f, 0.f, 0.f, 0.f};
      if (r < rows) x = *(const float4_t*)(query(r, h0 + col % heads) + e);
      *(float4_t*)&s_q[col * kQStride + e] = x;
    }
    __syncthreads();
    float factor = 1.0f, l1 = 0.0f, top = 0.0f;
    int ex = 0;
    const float* mine = s_q + c16 * kQStride + kE * g;
#pragma unroll
    for (int i = 0; i < kCh; ++i)
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        const float x = fabsf(mine[4 * kE * i + e]);
        l1 += x;
        top = fmaxf(top, x);
      }
    l1 = sum_groups(l1);
    l1 = l1 < INFINITY ? l1 : INFINITY;  // also where it is no number
    if (wave == 0 && g == 0) s_l1[c16] = h0 == 0 ? l1 : fmaxf(l1, s_l1[c16]);
    if constexpr (kF16) {
      top = max_groups(top);
      if (top > 0.0f && top < INFINITY) ex = __builtin_amdgcn_frexp_expf(top);
      ex = max(ex, -100);
      factor = __builtin_amdgcn_ldexpf(1.0f, ex - 14);
    }
    // 16 pages at a time.
    for (uint32_t p16 = 16 * (4 * blockIdx.x + wave); p16 < n1; p16 += 64 * wgs) {
      operand_t lo[kCh], hi[kCh];
      const KV* b = bounds_of(min(p16 + c16, n1 - 1)) + kE * g;
#pragma unroll
      for (int i = 0; i < kCh; ++i) {
        lo[i] = *(const operand_t*)(b + 4 * kE * i);
        hi[i] = *(const operand_t*)(b + D + 4 * kE * i);
      }
      // The pages that are taken in any case are not scored; a new token's own may have no bounds yet.
      const bool candidate = p16 + c16 >= a.first && p16 + c16 + a.last < n1;
      float4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kCh; ++i) {
        if constexpr (kF16) {
          half8_t below_h, below_l, above_h, above_l;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float x = __builtin_amdgcn_ldexpf(mine[32 * i + e], 14 - ex);
            _Float16 h, l;
            halves(fminf(x, 0.0f), h, l);
            below_h[e] = h;
            below_l[e] = l;
            halves(fmaxf(x, 0.0f), h, l);
            above_h[e] = h;
            above_l[e] = l;
          }
          s = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo[i], below_l, s, 0, 0, 0);
          s = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi[i], above_l, s, 0, 0, 0);
          s = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo[i], below_h, s, 0, 0, 0);
          s = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi[i], above_h, s, 0, 0, 0);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = mine[16 * i + e];
            s = __builtin_amdgcn_mfma_f32_16x16x4f32(lo[i][e], fminf(x, 0.0f), s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_16x16x4f32(hi[i][e], fmaxf(x, 0.0f), s, 0, 0, 0);
          }
        }
        float here = 0.0f;
#pragma unroll
        for (int e = 0; e < kE; ++e) here = fmaxf(here, fmaxf(fabsf((float)lo[i][e]), fabsf((float)hi[i][e])));
        most = fmaxf(most, candidate ? here : 0.0f);
      }
      // Lane (g, c) holds pages 4g .. 4g + 3 of column c. A score that is not finite stays so.
      float(*score)[17] = s_mem.score + 16 * wave;
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = 0; i < 4; ++i) score[4 * g + i][c16] = s[i] * factor;
      __builtin_amdgcn_wave_barrier();
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (p16 + c16 < n1)
        for (uint32_t r = g; r < rows; r += 4) {
          float best = -INFINITY;
          bool odd = false;
          for (uint32_t h = 0; h < heads; ++h) {
            const float x = score[c16][r * heads + h];
            odd = odd || !(fabsf(x) < INFINITY);
            best = fmaxf(best, x);
          }
          float* key = keys + (uint64_t)r * paged_row_keys(a.key_stride) + p16 + c16;
          if (h0 > 0) {  // this lane's own
            const float x = __hip_atomic_load(key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            odd = odd || x != x;
            best = fmaxf(best, x);
          }
          __hip_atomic_store(key, odd ? NAN : best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
  }
  most = max_wave(most);
  if (lane == 0) __hip_atomic_store(&maxima[4 * blockIdx.x + wave], most, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // The keys are acknowledged (visible device-wide) before the ticket is taken.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (wgs > 1) {
    if (tid == 0) s_last = __hip_atomic_fetch_add(&a.tickets[block], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (s_last + 1 != wgs) return;
    if (tid == 0) __hip_atomic_store(&a.tickets[block], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }

  // Exact score of page p, of the 16 lanes that call with it.
  auto exact = [&](uint32_t r, uint32_t p) JMA_INL -> uint64_t {
    constexpr int kX = D / 16;
    const KV* b = bounds_of(p) + c16 * kX;
    constexpr uint32_t kHeads = D >= 256 ? 2 : 4;  // heads whose elements are read together
    float low[kX], high[kX];
#pragma unroll
    for (int e = 0; e < kX; ++e) low[e] = (float)b[e], high[e] = (float)b[D + e];
    double best = -INFINITY;
    bool odd = false;
    for (uint32_t h0 = 0; h0 < a.group; h0 += kHeads) {
      float x[kHeads][kX];
#pragma unroll
      for (uint32_t i = 0; i < kHeads; ++i) {
        const float* from = query(r, min(h0 + i, a.group - 1)) + c16 * kX;
#pragma unroll
        for (int e = 0; e < kX; ++e) x[i][e] = from[e];
      }
#pragma unroll
      for (uint32_t i = 0; i < kHeads; ++i) {
        double s = 0.0;
#pragma unroll
        for (int e = 0; e < kX; ++e) {
          const double u = (double)x[i][e] * (double)low[e], v = (double)x[i][e] * (double)high[e];  // exact
          s += u > v || u != u ? u : v;
        }
        s = row_sum(s);
        odd = odd || s != s;
        best = s > best ? s : best;
      }
    }
    return odd ? 0xFFFFFFFFFFFFFFFFull : ordered(best);
  };
  // The pages of row r, by a wave of its own, or by all four.
  auto pick = [&](uint32_t r, auto team) JMA_INL {
    constexpr uint32_t kWaves = decltype(team)::value, kBins = kWaves == 1 ? kPickBins : 2 * kPickBins, kZero = kBins / kWaves;
    const uint32_t m = kWaves == 1 ? 0 : wave, w = wave - m;  // which of the team; its first wave, whose share of the LDS it has
    auto meet = [&]() JMA_INL {
      if constexpr (kWaves > 1) {
        __syncthreads();
      } else {
        __builtin_amdgcn_wave_barrier();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
    };
    const uint32_t n = pages_of(r);
    uint32_t* out = list_of(r);
    if (m == 0) {
      for (uint32_t i = lane; i < a.first; i += 64) out[i] = i;
      for (uint32_t i = lane; i < a.last; i += 64) out[a.first + a.top + i] = n - a.last + i;
    }
    if (a.top == 0) return;
    out += a.first;
    float* row_keys = keys + (uint64_t)r * paged_row_keys(a.key_stride);
    // This wave's share of the candidates, kept in LDS where it fits.
    const uint32_t candidates = n - a.last - a.first, share = (candidates + 64 * kWaves - 1) / (64 * kWaves) * 64;
    const uint32_t p0 = a.first + min(m * share, candidates), p1 = a.first + min((m + 1) * share, candidates);
    const bool held = share <= kHeldScores;
    float* mine = space.score[wave];
    uint32_t* hist = space.hist[w];
    float bound = 0.0f;  // the largest of the pages' bounds
    for (uint32_t i = lane; i < 4 * wgs; i += 64) bound = fmaxf(bound, __hip_atomic_load(&maxima[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
#pragma unroll
    for (uint32_t i = 0; i < kZero / 64; ++i) hist[kZero * m + 64 * i + lane] = 0;
    float least = INFINITY, most = -INFINITY;
    bool odd = false;
    for (uint32_t b = p0; b < p1; b += 512) {
      float x[8];
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i)  // unconditional, so that all are in flight together
        x[i] = __hip_atomic_load(&row_keys[min(b + 64 * i + lane, p1 - 1)], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) {  // the last one again does no harm
        odd = odd || x[i] != x[i];
        least = fminf(least, x[i]);
        most = fmaxf(most, x[i]);
        if (held) mine[b - p0 + 64 * i + lane] = x[i];
      }
    }
    auto each = [&](auto&& f) JMA_INL {  // f(page, score, whether there is such a candidate)
      for (uint32_t b = p0; b < p1; b += 256) {
        float x[4];
        if (held) {
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) x[i] = mine[b - p0 + 64 * i + lane];
        } else {
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i)
            x[i] = __hip_atomic_load(&row_keys[min(b + 64 * i + lane, p1 - 1)], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) f(b + 64 * i + lane, x[i], b + 64 * i + lane < p1);
      }
    };
    bound = max_wave(bound);
    least = -max_wave(-least);
    most = max_wave(most);
    uint32_t odds = __ballot(odd) != 0 ? 1 : 0;
    if constexpr (kWaves > 1) {
      if (lane == 0) space.least[wave] = least, space.most[wave] = most, space.odd[wave] = odds;
      meet();
#pragma unroll
      for (uint32_t i = 0; i < kWaves; ++i) {
        least = fminf(least, space.least[i]);
        most = fmaxf(most, space.most[i]);
        odds |= space.odd[i];
      }
    } else {
      meet();
    }
    const uint32_t heads = min(16u, a.group);
    float l1 = 0.0f;
    for (uint32_t h = 0; h < heads; ++h) l1 = fmaxf(l1, s_l1[r * heads + h]);
    if (odds == 0 && l1 == 0.0f) {  // every score is zero
      if (m == 0)
        for (uint32_t i = lane; i < a.top; i += 64) out[i] = a.first + i;
      return;
    }
    const float eps = 1.001f * (0x1p-22f + (4 * D + 16) * 0x1p-23f) * l1 * bound + 0x1p-120f;  // and underflows
    // Everything is scored in 64 bits where a score, or the steps of the histogram, are out of range.
    const bool all = odds != 0 || !(l1 < INFINITY) || !(eps < INFINITY) || !(most - least > 0x1p-90f && most - least < INFINITY);
    float high = INFINITY, low = -INFINITY;  // above: taken; below: not
    if (!all) {
      const float steps = (float)(kBins - 1) / (most - least), step = (most - least) / (float)(kBins - 1);
      each([&](uint32_t, float x, bool there) JMA_INL {
        if (there) atomicAdd(&hist[min((uint32_t)((x - least) * steps), kBins - 1)], 1u);
      });
      meet();
      uint32_t need = a.top, bin, count;
      border_bin<kBins / 64>(hist, lane, need, bin, count);
      high = least + ((float)bin + 1.01f) * step + 2.0f * eps;  // .01: (x - least) * steps is rounded
      low = least + ((float)bin - 0.01f) * step - 2.0f * eps;
    }
    auto above = [&](float x) JMA_INL { return x > high; };
    auto near = [&](float x) JMA_INL { return !(x > high) && !(x < low); };
    uint32_t sure = 0, count = 0;
    if (!all) {
      each([&](uint32_t p, float x, bool there) JMA_INL {
        sure += (uint32_t)__popcll(__ballot(there && above(x)));
        const bool in = there && near(x);
        const uint64_t b = __ballot(in);
        const uint32_t i = count + lanes_below(b, lane);
        if (in && i < kPickNear) space.near[wave][i] = p;
        count += (uint32_t)__popcll(b);
      });
      if constexpr (kWaves > 1)
        if (lane == 0) space.sure[wave] = sure, space.count[wave] = count;
      meet();
    }
    // Of the whole row, and of the waves before this one.
    uint32_t all_sure = sure, all_near = count, near_before = 0, sure_before = 0, start[kWaves + 1] = {};
    if constexpr (kWaves > 1) {
      all_sure = all_near = 0;
#pragma unroll
      for (uint32_t i = 0; i < kWaves; ++i) {
        if (i == m) sure_before = all_sure, near_before = all_near;
        start[i] = all_near;
        all_sure += space.sure[i];
        all_near += space.count[i];
      }
    }
    if (!all && (all_near <= kPickNear || all_sure + all_near == a.top)) {
      uint64_t taken = ~0ull;  // of those near
      if (all_sure + all_near != a.top) {
        for (uint32_t b = 4 * m; b < all_near; b += 4 * kWaves) {
          uint32_t i = min(b + g, all_near - 1), of = w;
          if constexpr (kWaves > 1) {
#pragma unroll
            for (uint32_t k = 1; k < kWaves; ++k)
              if (i >= start[k]) of = k;
            i -= start[0] * (of == 0) + start[1] * (of == 1) + start[2] * (of == 2) + start[3] * (of == 3);
          }
          const uint64_t e = exact(r, space.near[of][i]);
          if (c16 == 0 && b + g < all_near) space.exact[w][b + g] = e;
        }
        meet();
        const uint64_t e = space.exact[w][min(lane, all_near - 1)];
        uint32_t better = 0;
        for (uint32_t i = 0; i < all_near; ++i) {
          const uint64_t x = space.exact[w][i];
          better += x > e || (x == e && i < lane) ? 1u : 0u;
        }
        taken = __ballot(lane < all_near && better < a.top - all_sure);
      }
      uint32_t seen = near_before;
      uint32_t at = sure_before + (taken == ~0ull ? near_before : (uint32_t)__popcll(taken & ((near_before < 64 ? 1ull << near_before : 0ull) - 1)));
      each([&](uint32_t p, float x, bool there) JMA_INL {
        const bool in = there && near(x);
        const uint64_t b = __ballot(in);
        const uint32_t i = seen + lanes_below(b, lane);
        const bool take = (there && above(x)) || (in && (taken == ~0ull || ((taken >> (i & 63)) & 1)));
        seen += (uint32_t)__popcll(b);
        const uint64_t t = __ballot(take);
        if (take) out[at + lanes_below(t, lane)] = p;
        at += (uint32_t)__popcll(t);
      });
      return;
    }
    // Keys of 64 bits for all that are near, behind the scores: four pages of the wave's share at a time.
    uint64_t* wide = (uint64_t*)(row_keys + ((a.key_stride + 1) & ~1u));
    for (uint32_t b = p0; b < p1; b += 64) {
      const float v = __hip_atomic_load(&row_keys[min(b + lane, p1 - 1)], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const bool there = b + lane < p1;
      uint64_t in = __ballot(there && (all || near(v)));
      if (there && !(all || near(v))) __hip_atomic_store(&wide[b + lane], above(v) ? ~0ull : 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      while (in != 0) {
        uint32_t at[4];
        uint32_t found = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          at[i] = in != 0 ? (uint32_t)__ffsll((long long)in) - 1 : at[i > 0 ? i - 1 : 0];
          if (in != 0) ++found, in &= in - 1;
        }
        const uint32_t p = b + (g == 0 ? at[0] : g == 1 ? at[1] : g == 2 ? at[2] : at[3]);
        const uint64_t e = exact(r, p);
        if (c16 == 0 && g < found) __hip_atomic_store(&wide[p], e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    meet();
    if (m != 0) return;
    Keys k{wide, a.first, a.first + candidates, lane};
    const uint64_t border = nth_largest(k, a.top, space.hist[w]);
    uint32_t larger = 0;
    k.each([&](uint32_t, uint64_t x, bool there) JMA_INL { larger += (uint32_t)__popcll(__ballot(there && x > border)); });
    uint32_t at = 0, equal = 0;
    k.each([&](uint32_t p, uint64_t x, bool there) JMA_INL {
      const uint64_t b = __ballot(there && x == border);
      const bool take = there && (x > border || (x == border && equal + lanes_below(b, lane) < a.top - larger));
      equal += (uint32_t)__popcll(b);
      const uint64_t t = __ballot(take);
      if (take) out[at + lanes_below(t, lane)] = p;
      at += (uint32_t)__popcll(t);
    });
  };
  if (rows == 1)
    pick(0, std::integral_constant<uint32_t, 4>{});
  else
    for (uint32_t r = wave; r < rows; r += 4)
      if (pages_of(r) > a.budget) pick(r, std::integral_constant<uint32_t, 1>{});
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

// Workgroup = (split, kv head x head group x block of query rows of a chunk): 16 matrix-core columns =
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
//
// Large batches are bound by the bytes of K and V (64 tokens of 32 + 8 heads of 128, 383 MB: 81 us, 4.7 TB/s,
// where a large copy moves 5.2); one token by the dependent round trips from its table entry to the joined
// splits (32 + 8 heads of 64, 700 positions: 9 us); f32 caches of many rows by f32
// matrix instructions at half their rate, two waves a SIMD being what the registers hold (12 tokens and 200
// rows of 16 + 8 heads of 128: 86 us). Eight waves a workgroup at heads of 128 took 89 us for the batch.
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

  const uint32_t hkv = a.kv.hkv, R = a.rows_per_block;
  const uint32_t block = blockIdx.y / (hkv * a.head_groups);
  uint32_t chunk = block;
  if (!kFused && a.max_blocks > 1) {  // the chunk that this block of rows belongs to
    uint32_t lo = 0, hi = a.chunks;
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (a.c[mid].block0 <= block) lo = mid;
      else hi = mid;
    }
    chunk = lo;
  }
  const PagedChunk ch = a.c[chunk];
  const uint32_t nth = blockIdx.y - ch.block0 * hkv * a.head_groups;  // among the chunk's
  const uint32_t kvh = nth % hkv, rest = nth / hkv;
  const uint32_t hg = rest % a.head_groups, row0 = rest / a.head_groups * R;
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
  const uint32_t unit = blockIdx.y;
  float* part = a.part + (ch.part0 + (uint64_t)nth * ch.nsplit) * (16 * (D + 4));  // this block's states
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

hipError_t launch_paged_select(const PagedSelectArgs& a, bool f16, uint32_t d, hipStream_t stream) {
  return by_shape(f16, d, [&](auto kv, auto dim) {
    using KV = decltype(kv);
    constexpr int D = decltype(dim)::value;
    const uint32_t lds = a.raw ? a.group * (D + 4) * 4 : 0;
    paged_select_kernel<KV, D><<<dim3(a.max_wgs, a.max_blocks * a.kv.hkv, a.chunks), 256, lds, stream>>>(a);
    return hipGetLastError();
  });
}

hipError_t launch_paged_attend(const PagedAttendArgs& a, bool f16, uint32_t d, hipStream_t stream) {
  return by_shape(f16, d, [&](auto kv, auto dim) {
    using KV = decltype(kv);
    constexpr int D = decltype(dim)::value;
    const bool fused = a.k_new != nullptr;
    const dim3 grid(a.max_splits + (fused ? 1 : 0), a.blocks * a.kv.hkv * a.head_groups);
    constexpr uint32_t kThreads = 64 * paged_waves(D);
    if (fused && a.pages != nullptr) paged_attend_kernel<KV, D, true, true><<<grid, kThreads, 0, stream>>>(a);
    else if (fused) paged_attend_kernel<KV, D, false, true><<<grid, kThreads, 0, stream>>>(a);
    else if (a.pages != nullptr) paged_attend_kernel<KV, D, true, false><<<grid, kThreads, 0, stream>>>(a);
    else paged_attend_kernel<KV, D, false, false><<<grid, kThreads, 0, stream>>>(a);
    return hipGetLastError();
  });
}

}  // namespace jma
