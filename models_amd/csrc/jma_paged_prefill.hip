// gfx950 kernel of the paged KV cache for chunks of many rows:
//
//   paged_prefill_kernel        causal attention of a chunk over its sequence's pages, f16 caches
//   paged_prefill_join_kernel   the states of row blocks whose range of positions is split
#include "jma_paged_device.h"

namespace jma {
namespace {

typedef float float16_t __attribute__((ext_vector_type(16)));

// 16 bytes a lane from global memory straight into LDS (lane i's at lds + 16 i).
__device__ __forceinline__ void dma16(const _Float16* base, _Float16* lds, uint32_t voff, uint32_t soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(
      __builtin_amdgcn_make_buffer_rsrc(const_cast<_Float16*>(base), 0, 0x7FFFFFF0, 0x00020000),
      (__attribute__((address_space(3))) void*)lds, 16, voff, soff, 0, 0);
}

// Which slot of a tile row i of the score product is (bits 2 and 3 exchanged), and where 16-byte piece c
// of a 64-byte row r lies in LDS: the eight lanes of one LDS cycle read the same piece of eight rows,
// which the exchange spreads over all banks.
__device__ __forceinline__ uint32_t swap23(uint32_t i) { return (i & ~12u) | ((i & 4u) << 1) | ((i & 8u) >> 1); }
__device__ __forceinline__ uint32_t swz_k(uint32_t slot) { return ((slot >> 1) & 1u) | ((slot >> 2) & 2u); }
__device__ __forceinline__ uint32_t swz_v(uint32_t row) { return (row >> 1) & 3u; }

// Workgroup = (split, kv head x head group x block of query rows, chunk); each of its four waves owns 32
// matrix-core columns = (query row, query head) pairs, and all share the K and V tiles, which
// direct-to-LDS loads bring a step (64 slots; 32 at heads of 256) ahead of their use.
//
// v_mfma_f32_32x32x16_f16, lane l, j = l % 32, h = l / 32: A[i][k]: i = j, k = 8h + e; B[k][c]: c = j,
// k = 8h + e; D[i][c]: c = j, i = 8 (e / 4) + 4h + e % 4. S^T = K Q^T with row i of the product at slot
// swap23(i) leaves a lane the scores of slots 8h .. 8h+7 and 16 + 8h .. 16 + 8h + 7, in order: they are the
// B operand of O^T = V^T P as they stand.
//
// Precision, masks and values that are no number are paged_attend_kernel's: q and p as two f16 halves,
// each column's q scaled by a power of two.
//
// Bound at heads of 128 by the matrix instructions, twice the operands' f16 products: 2048 rows of 32 + 8
// heads over 8049 positions, 236 GFLOP of results, 405 us: 1.16 PFLOP/s of instructions, what a large f16
// product reaches. At heads of 64 by the exponentials and halves of p beside them (two chunks of 301 rows,
// 34 us, a fifth of the matrix rate); short windows by a step's latency (1000 rows of 4 + 1 heads of 256 in
// a window of 512: 20 us for four steps a workgroup).
template <int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(paged_prefill_waves_per_simd(D)))) void paged_prefill_kernel(const PagedAttendArgs a) {
  constexpr int S = kPrefillWaves, T = paged_prefill_tiles(D);
  constexpr int kKS = D / 16, kNb = D / 32, kTile = 32 * D;
  constexpr int kLoads = T * (D / 16) / S;  // 1 KB loads a wave makes of a step's K (and of its V)
  constexpr uint32_t kItem = paged_prefill_item(D);
  __shared__ __attribute__((aligned(16))) _Float16 lx[2 * T * kTile];  // K tiles, then V tiles
  __shared__ __attribute__((aligned(16))) _Float16 ly[2 * T * kTile];

  const PagedChunk ch = a.c[blockIdx.z];
  const uint32_t hkv = a.kv.hkv, R = a.rows_per_stripe, Gz = a.heads_per_stripe;
  const uint32_t kvh = blockIdx.y % hkv, rest = blockIdx.y / hkv;
  const uint32_t hg = rest % a.head_groups, rank = rest / a.head_groups;
  const uint32_t blocks = (ch.rows + S * R - 1) / (S * R);
  if (rank >= blocks) return;
  const uint32_t b_row0 = (blocks - 1 - rank) * S * R;  // the longest ranges first
  const uint32_t b_row1 = min(b_row0 + S * R, ch.rows) - 1;
  uint32_t t0, t1;
  paged_range(ch.start + b_row0, ch.start + b_row1, a.window, 0u, a.kv.page_log2, kTileSlots, t0, t1);
  const uint32_t ns = (t1 - t0 + a.tiles_per_split - 1) / a.tiles_per_split, split = blockIdx.x;
  if (split >= ns) return;
  t0 += split * a.tiles_per_split;
  t1 = min(t1, t0 + a.tiles_per_split);

  const int lane = threadIdx.x & 63, j = lane & 31, h = lane >> 5;
  const int s = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t row0 = min(b_row0 + s * R, ch.rows - 1);  // a stripe behind the chunk repeats its last row
  const bool stripe_ok = b_row0 + s * R < ch.rows;
  const uint32_t rows = min(R, ch.rows - row0), heads = min(Gz, a.group - hg * Gz);
  const uint32_t pos0 = ch.start + row0, pos1 = pos0 + rows - 1;
  const uint32_t first0 = first_visible(pos0, a.window), first1 = first_visible(pos1, a.window);
  // This lane's column; one past the stripe's (row, head) pairs repeats a valid one and is never stored.
  const uint32_t col_row = min((uint32_t)j / heads, rows - 1);
  const bool col_ok = stripe_ok && (uint32_t)j / heads < rows;
  const uint32_t cpos = pos0 + col_row, cfirst = first_visible(cpos, a.window);
  const uint64_t qat = (((uint64_t)ch.row0 + row0 + col_row) * a.num_heads + kvh * a.group + hg * Gz + j % heads) * D;

  // The page of tile base + lane of this split.
  const uint32_t* table = a.kv.table + (uint64_t)ch.seq * a.kv.table_stride;
  const uint32_t tiles_log2 = a.kv.page_log2 - 5;
  uint32_t pages_at = t0;
  uint32_t my_page = table[min(t0 + lane, t1 - 1) >> tiles_log2];
  // This lane's place in a 1 KB piece: 16 rows of 64 bytes, four 16-byte pieces each.
  const uint32_t lrow = lane / 4;
  const uint32_t koff = lrow * 64 + ((lane & 3) ^ swz_k(lrow)) * 16, voff = lrow * 64 + ((lane & 3) ^ swz_v(lrow)) * 16;
  auto stage = [&](uint32_t t, _Float16* lds) JMA_INL {
    const _Float16* kt[T];
    const _Float16* vt[T];
#pragma unroll
    for (int i = 0; i < T; ++i) {
      const uint32_t tile = min(t + i, t1 - 1);  // a tile behind the last is loaded again, and not used
      const uint32_t page = __builtin_amdgcn_readlane(my_page, tile - pages_at);
      const uint64_t at = paged_base(page, hkv, kvh, a.kv.page_log2, D) + (tile & ((1u << tiles_log2) - 1)) * kTile;
      kt[i] = (const _Float16*)a.kv.k + at;
      vt[i] = (const _Float16*)a.kv.v + at;
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint32_t u = s + S * i, tile = T == 1 ? 0 : u / (D / 16), c = u % (D / 16);
      dma16(T == 1 || tile == 0 ? kt[0] : kt[T - 1], lds + 512 * u, koff, 1024 * c);
      dma16(T == 1 || tile == 0 ? vt[0] : vt[T - 1], lds + T * kTile + 512 * u, voff, 1024 * c);
    }
  };
  stage(t0, lx);

  // Q^T operands and the factor of the column's scores.
  half8_t qhi[kKS], qlo[kKS];
  float factor;
  {
    const float* q = a.q + qat + 8 * h;
    float4_t x[kKS][2];
    float top = 0.0f;
#pragma unroll
    for (int ks = 0; ks < kKS; ++ks)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        x[ks][i] = *(const float4_t*)(q + 16 * ks + 4 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(x[ks][i][e]));
      }
    top = max_halves(top);
    int ex = 0;  // top in [2^(ex-1), 2^ex)
    if (top > 0.0f && top < INFINITY) ex = __builtin_amdgcn_frexp_expf(top);
    ex = max(ex, -100);
    factor = __builtin_amdgcn_ldexpf(a.scale, ex - 14);
#pragma unroll
    for (int ks = 0; ks < kKS; ++ks)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        _Float16 hi, lo;
        halves(__builtin_amdgcn_ldexpf(x[ks][e / 4][e % 4], 14 - ex), hi, lo);
        qhi[ks][e] = hi;
        qlo[ks][e] = lo;
      }
  }

  float m = -INFINITY, l = 0.0f;
  float16_t o[kNb];
#pragma unroll
  for (int nb = 0; nb < kNb; ++nb)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[nb][e] = 0.0f;

  const uint32_t kr = swap23(j), kswz = swz_k(kr), vswz = swz_v(j);
  // kN tiles at once, in LDS, or (kRobust) in global memory. kMasked: some column of the workgroup may not
  // see all of them.
  auto tile_step = [&](const _Float16* kt, const _Float16* vt, uint32_t p0, auto count, auto masked, auto robust) JMA_INL {
    constexpr int kN = decltype(count)::value;
    constexpr bool kMasked = decltype(masked)::value, kRobust = decltype(robust)::value;
    static_assert(kN == 1 || !kMasked, "masked tiles one at a time");
    if (kMasked && (p0 > pos1 || p0 + 31 < first0)) return;  // this stripe sees none of it
    float16_t sc[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[i][e] = 0.0f;
    constexpr int kB = kKS * kN < 4 ? kKS : 4 / kN;  // operand reads issued ahead of their products
#pragma unroll
    for (int k0 = 0; k0 < kKS; k0 += kB) {
      half8_t kf[kB][kN];
#pragma unroll
      for (int i = 0; i < kB; ++i)
#pragma unroll
        for (int n = 0; n < kN; ++n) {
          const int ks = k0 + i;
          kf[i][n] = *(const half8_t*)(kt + n * kTile + (ks / 2) * 1024 + kr * 32 + 8 * ((2 * (ks % 2) + h) ^ (kRobust ? 0u : kswz)));
        }
#pragma unroll
      for (int i = 0; i < kB; ++i) {
#pragma unroll
        for (int n = 0; n < kN; ++n) sc[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[i][n], qlo[k0 + i], sc[n], 0, 0, 0);
#pragma unroll
        for (int n = 0; n < kN; ++n) sc[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[i][n], qhi[k0 + i], sc[n], 0, 0, 0);
      }
    }
    const bool whole = !kMasked || (p0 + 31 <= pos0 && p0 >= first1);
    if (kMasked && !whole) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t p = p0 + 16 * (e / 8) + 8 * h + e % 8;
        sc[0][e] = p >= cfirst && p <= cpos ? sc[0][e] : -INFINITY;
      }
    }
    float tmax = sc[0][0];
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int e = 0; e < 16; ++e) tmax = fmaxf(tmax, sc[n][e]);
    tmax = max_halves(tmax) * factor;
    // The running maximum rises only by more than 2^8: most tiles rescale nothing.
    const bool up = m == -INFINITY ? tmax > -INFINITY : tmax > m + 8.0f;
    if (__ballot(up) != 0) {
      const float mn = up ? tmax : m;
      const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int nb = 0; nb < kNb; ++nb) o[nb] *= alpha;
    }
    const float shift = 6.0f - (m == -INFINITY ? 0.0f : m);
    half8_t ph[kN][2], pl[kN][2];
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float x0 = __builtin_amdgcn_exp2f(fmaf(sc[n][e], factor, shift)), x1 = __builtin_amdgcn_exp2f(fmaf(sc[n][e + 1], factor, shift));
        sum[0] += x0;
        sum[1] += x1;
        const half2_t hi = __builtin_convertvector((float2_t{x0, x1}), half2_t);
        const half2_t lo = __builtin_convertvector((float2_t{minus_low(x0, hi), minus_high(x1, hi)}), half2_t);
        ph[n][e / 8][e % 8] = hi[0];
        ph[n][e / 8][e % 8 + 1] = hi[1];
        pl[n][e / 8][e % 8] = lo[0];
        pl[n][e / 8][e % 8 + 1] = lo[1];
      }
    l += sum[0] + sum[1];
    auto value = [&](int n, int nb, int b) JMA_INL {
      return *(const half8_t*)(vt + n * kTile + (32 * nb + j) * 32 + 8 * ((2 * b + h) ^ (kRobust ? 0u : vswz)));
    };
    if constexpr (kRobust) {
      // Values that are no finite number are left out of the product, and what they make of the columns
      // that see them is added: a second product counts, for each output, the ones its column sees.
      half8_t sees[2];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t p = p0 + 16 * (e / 8) + 8 * h + e % 8;
        sees[e / 8][e % 8] = p >= cfirst && p <= cpos ? (_Float16)1.0f : (_Float16)0.0f;
      }
#pragma unroll
      for (int nb = 0; nb < kNb; ++nb) {
        float16_t found;
#pragma unroll
        for (int e = 0; e < 16; ++e) found[e] = 0.0f;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          half8_t v = value(0, nb, b), is;
          split_finite(v, is);
          found = __builtin_amdgcn_mfma_f32_32x32x16_f16(is, sees[b], found, 0, 0, 0);
          o[nb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl[0][b], o[nb], 0, 0, 0);
          o[nb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph[0][b], o[nb], 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) o[nb][e] = found[e] > 0.0f ? NAN : o[nb][e];
      }
      return;
    }
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int nb = 0; nb < kNb; nb += 2) {
        constexpr int kV = kNb < 2 ? 1 : 2;
        half8_t v[kV][2];
#pragma unroll
        for (int i = 0; i < kV; ++i)
#pragma unroll
          for (int b = 0; b < 2; ++b) v[i][b] = value(n, nb + i, b);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
          for (int i = 0; i < kV; ++i) o[nb + i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[i][b], pl[n][b], o[nb + i], 0, 0, 0);
#pragma unroll
          for (int i = 0; i < kV; ++i) o[nb + i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[i][b], ph[n][b], o[nb + i], 0, 0, 0);
        }
      }
  };
  constexpr std::integral_constant<int, 1> kOne{};

  // One barrier a step: behind it every wave's loads of this step have landed (each wave waited for its
  // own) and every wave has done with the array that the next step's loads then overwrite.
  auto step = [&](uint32_t t, _Float16* lds, _Float16* next, auto masked) JMA_INL {
    __builtin_amdgcn_s_waitcnt((0 & 15) | (7 << 4) | (15 << 8));  // vmcnt(0)
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (t + T < t1) {
      if (min(t + 2 * T, t1) > pages_at + 64) {  // the next step's pages
        pages_at = t + T;
        my_page = table[min(pages_at + lane, t1 - 1) >> tiles_log2];
      }
      stage(t + T, next);
    }
    if constexpr (decltype(masked)::value) {
#pragma unroll 1
      for (int i = 0; i < T; ++i)
        if (t + i < t1) tile_step(lds + i * kTile, lds + (T + i) * kTile, 32 * (t + i), kOne, masked, std::false_type{});
    } else {
      tile_step(lds, lds + T * kTile, 32 * t, std::integral_constant<int, T>{}, masked, std::false_type{});
    }
  };
  // Steps whose tiles every column of the workgroup sees whole run in a loop of their own, two at a time.
  const uint32_t whole0 = (first_visible(ch.start + b_row1, a.window) + 31) / 32, whole1 = (ch.start + b_row0 + 1) / 32;
  auto fast = [&](uint32_t t) JMA_INL { return t >= whole0 && t + 2 * T <= min(whole1, t1); };
  for (uint32_t t = t0; t < t1; t += 2 * T) {
    for (; fast(t); t += 2 * T) {
      step(t, lx, ly, std::false_type{});
      step(t + T, ly, lx, std::false_type{});
    }
    if (t >= t1) break;
    step(t, lx, ly, std::true_type{});
    if (t + T < t1) step(t + T, ly, lx, std::true_type{});
  }

  // A value that is no finite number, in a tile that a column sees in part, reaches all of the wave's columns
  // (0 x inf is no 0). A wave with such an output does its tiles again, straight from global memory, and
  // keeps what it finds then.
  float odd = 0.0f;
#pragma unroll
  for (int nb = 0; nb < kNb; ++nb)
#pragma unroll
    for (int e = 0; e < 16; ++e) odd = fmaf(o[nb][e], 0.0f, odd);
  if (__ballot(odd != 0.0f) != 0) {
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int nb = 0; nb < kNb; ++nb)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[nb][e] = 0.0f;
#pragma unroll 1
    for (uint32_t t = t0; t < t1; ++t) {
      const uint32_t page = __builtin_amdgcn_readfirstlane(table[t >> tiles_log2]);
      const uint64_t at = paged_base(page, hkv, kvh, a.kv.page_log2, D) + (t & ((1u << tiles_log2) - 1)) * kTile;
      tile_step((const _Float16*)a.kv.k + at, (const _Float16*)a.kv.v + at, 32 * t, kOne, std::true_type{}, std::true_type{});
    }
  }

  l = sum_halves(l);
  auto finish = [&](auto&& chunk_of, float sum) JMA_INL {
    if (__ballot(col_ok && !(sum > 0.0f && sum < INFINITY)) != 0 && lane == 0) report(a.err, kErrNonFinite);
    const float inv = sum > 0.0f ? 1.0f / sum : sum;
    float* out = a.out + qat + 4 * h;
#pragma unroll
    for (int c = 0; c < D / 8; ++c) {
      const float4_t x = chunk_of(c);
      if (col_ok) *(float4_t*)(out + 8 * c) = x * inv;
    }
  };
  auto mine = [&](int c) JMA_INL {
    return float4_t{o[c / 4][4 * (c % 4)], o[c / 4][4 * (c % 4) + 1], o[c / 4][4 * (c % 4) + 2], o[c / 4][4 * (c % 4) + 3]};
  };
  if (ns == 1) {
    finish(mine, l);
    return;
  }
  // A split block's state, for paged_prefill_join_kernel.
  float4_t* part = (float4_t*)(a.part + (ch.part0 + (uint64_t)blockIdx.y * ch.nsplit + split) * kItem) + s * (D / 8 + 1) * 64 + lane;
#pragma unroll
  for (int c = 0; c < D / 8; ++c) part[64 * c] = mine(c);
  part[64 * (D / 8)] = float4_t{m, l, 0.0f, 0.0f};
}

// Joins the states of split blocks, in split order: workgroup = (four (wave, word of O^T) pairs, block,
// chunk), one word a thread. A launch of its own: a last workgroup that waited for the
// others' states and joined them alone took up to 29 us (1000 rows of 4 + 1 heads of 256), this launch 7.
template <int D>
__global__ __launch_bounds__(256) void paged_prefill_join_kernel(const PagedAttendArgs a) {
  constexpr int S = kPrefillWaves;
  constexpr uint32_t kItem = paged_prefill_item(D);
  const PagedChunk ch = a.c[blockIdx.z];
  const uint32_t hkv = a.kv.hkv, R = a.rows_per_stripe, Gz = a.heads_per_stripe;
  const uint32_t kvh = blockIdx.y % hkv, rest = blockIdx.y / hkv;
  const uint32_t hg = rest % a.head_groups, rank = rest / a.head_groups;
  const uint32_t blocks = (ch.rows + S * R - 1) / (S * R);
  if (rank >= blocks) return;
  const uint32_t b_row0 = (blocks - 1 - rank) * S * R, b_row1 = min(b_row0 + S * R, ch.rows) - 1;
  uint32_t t0, t1;
  paged_range(ch.start + b_row0, ch.start + b_row1, a.window, 0u, a.kv.page_log2, kTileSlots, t0, t1);
  const uint32_t ns = (t1 - t0 + a.tiles_per_split - 1) / a.tiles_per_split;
  if (ns == 1) return;
  const uint32_t lane = threadIdx.x & 63, unit = blockIdx.x * 4 + threadIdx.x / 64;  // (stripe, word)
  const uint32_t s = unit / (D / 8), c = unit % (D / 8), j = lane & 31, h = lane >> 5;
  const uint32_t row0 = b_row0 + s * R, heads = min(Gz, a.group - hg * Gz);
  if (row0 >= ch.rows || j / heads >= min(R, ch.rows - row0)) return;
  const float4_t* part = (const float4_t*)(a.part + (ch.part0 + (uint64_t)blockIdx.y * ch.nsplit) * kItem) + s * (D / 8 + 1) * 64 + lane;
  float m = -INFINITY, l = 0.0f;
  float4_t y = {0.0f, 0.0f, 0.0f, 0.0f};
  for (uint32_t sp0 = 0; sp0 < ns; sp0 += 4) {  // four splits' words in flight
    float4_t ml[4], x[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const float4_t* p = part + (uint64_t)min(sp0 + i, ns - 1) * (kItem / 4);
      ml[i] = p[64 * (D / 8)];
      x[i] = p[64 * c];
    }
    float top = m;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      if (sp0 + i >= ns) ml[i] = float4_t{-INFINITY, 0.0f, 0.0f, 0.0f};
      top = fmaxf(top, ml[i][0]);
    }
    const float back = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
    m = top;
    l *= back;
    y *= back;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      if (ml[i][0] == -INFINITY) continue;  // it saw nothing
      const float f = __builtin_amdgcn_exp2f(ml[i][0] - m);
      l = fmaf(ml[i][1], f, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = fmaf(x[i][e], f, y[e]);
    }
  }
  if (c == 0 && !(l > 0.0f && l < INFINITY)) report(a.err, kErrNonFinite);
  const uint64_t at = (((uint64_t)ch.row0 + row0 + j / heads) * a.num_heads + kvh * a.group + hg * Gz + j % heads) * D;
  *(float4_t*)(a.out + at + 8 * c + 4 * h) = y * (l > 0.0f ? 1.0f / l : l);
}

template <int D>
void launch_prefill(const PagedAttendArgs& a, hipStream_t stream) {
  const uint32_t units = a.max_blocks * a.kv.hkv * a.head_groups;
  paged_prefill_kernel<D><<<dim3(a.max_splits, units, a.chunks), 64 * kPrefillWaves, 0, stream>>>(a);
  if (a.max_splits > 1)
    paged_prefill_join_kernel<D><<<dim3(kPrefillWaves * (D / 8) / 4, units, a.chunks), 256, 0, stream>>>(a);
}

}  // namespace

hipError_t launch_paged_prefill(const PagedAttendArgs& a, uint32_t d, hipStream_t stream) {
  switch (d) {
    case 32: launch_prefill<32>(a, stream); break;
    case 64: launch_prefill<64>(a, stream); break;
    case 128: launch_prefill<128>(a, stream); break;
    case 256: launch_prefill<256>(a, stream); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace jma
