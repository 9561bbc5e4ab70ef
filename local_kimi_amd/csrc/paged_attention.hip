// Causal softmax attention of new rows on a paged cache, for gfx950.

#include <algorithm>

#include "lk_attention_tile.hpp"
#include "lk_paged.h"

namespace lk {
namespace {

// Queries x heads of a block for single tokens: a tile of the 16 x 16 products, or two. Up to
// 32 heads of one key head share a block, so that its keys are read once: 32 heads on
// one, 64 tokens on 2.1 million keys 220 us, 361 as two blocks of 16.
constexpr int kFewRows = 16;
constexpr int kPagedPack = 32;
// Runs that a call's keys are dealt in: four a CU, so that lengths of all kinds even out.
// With 512 / 1024 / 2048, 64 tokens on up to 8192 keys x 8 heads took 225 / 216 / 215 us, 1071
// rows of a mixed step 169 / 165 / 205. Rows of long pieces, bound by their products, take
// runs of twice the length (2048 rows on 16048 keys 539 us in 1024 runs, 523 so). At least
// kMinRun keys: 19 rows on 1119 keys take 18 us, in runs of 128 (nine, so that the join takes four waves
// a row) 28, one token on 16384 23 either way.
constexpr int kFill = 1024;
constexpr int kMinRun = 256;
constexpr int kJoinFew = 4, kJoinMany = 16;  // rows of a block of the join
constexpr int64_t kMaxSequences = 65536;
// From here on a launch of its own counts through the sequences. With it / without it, single tokens x 8
// heads of 128 on up to 512 keys: 64 sequences 29 / 26 us, 128 46 / 46, 255 64 / 71, 512 115 / 150, 1024
// 220 / 367; on up to 128 keys 64 11 / 8, 256 33 / 33, 1024 113 / 168.
constexpr int64_t kPlanSequences = 256;

struct PagedArgs : AttnShape {
  const uint16_t *k, *v;
  Sequences sq;
  PageTable table;
  int64_t k_page, k_row, k_head, v_page, v_row, v_head;
  // where keys can be in runs, else null: their number and tiles, then their rows' sums
  struct SplitTiles* split;
  float* partial;
  uint32_t units;  // of kFewRows rows that `partial` holds
  struct PlanEntry* plan;  // of each sequence, and behind the last; null: every block counts
};

// A tile whose keys are in runs, for the join.
struct SplitTile {
  int64_t row;  // its first
  int rows, pack, runs, units;
  uint32_t unit;
};
struct SplitTiles {
  int count;
  SplitTile tile[kFill];
};

// Rows in pages: a wave stages 16 rows of each tile, which lie in one page. The
// pages of its next 64 tiles are in the lanes of two registers.
template <int DQ, int DV>
struct PagedKeys {
  static constexpr int kKChunks = DQ / 8, kVChunks = DV / 8;
  static constexpr int kKLoads = kAttnKeys * kKChunks / kAttnThreads;
  static constexpr int kVLoads = kAttnKeys * kVChunks / kAttnThreads;
  static_assert(kKLoads * kWave == kPageStep * kKChunks && kVLoads * kWave == kPageStep * kVChunks,
                "a wave's share of a tile");
  const PagedArgs& a;
  const uint16_t *kb, *vb;  // of the first page, this head's
  const int32_t* pages;     // of the sequence
  int lk, wave, lane;
  int first;       // position of the tile that lane 0 has the page of
  int page, row;   // of this wave's rows in tile `lane` from there on; -1: none
  uint32_t lds;
  uint32_t koff[kKLoads], voff[kVLoads];

  __device__ __forceinline__ PagedKeys(const PagedArgs& args, const AttnBlock& b, int sequence,
                                       const uint16_t* stage)
      : a(args) {
    const int hk = b.pack * a.pack / a.group;
    kb = a.k + hk * a.k_head, vb = a.v + hk * a.v_head;
    pages = a.table.pages_of + sequence * a.table.stride;
    lk = static_cast<int>(b.lk);
    lane = threadIdx.x & (kWave - 1);
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    lds = lds_offset(stage);
    first = -kAttnKeys * kWave;
#pragma unroll
    for (int i = 0; i < kKLoads; ++i) {
      const int slot = i * kWave + lane, r = slot / kKChunks;  // the wave's row
      const int c = slot % kKChunks ^ key_swizzle<kKChunks>(r);
      koff[i] = 8 * c < a.d_qk ? static_cast<uint32_t>(r * a.k_row + 8 * c) * 2u : 0xFFFFFFF0u;
    }
#pragma unroll
    for (int i = 0; i < kVLoads; ++i) {
      const int slot = i * kWave + lane, r = slot / kVChunks;
      const int c = slot % kVChunks ^ value_swizzle<kVChunks>(r);
      voff[i] = 8 * c < a.d_v ? static_cast<uint32_t>(r * a.v_row + 8 * c) * 2u : 0xFFFFFFF0u;
    }
    static_assert(key_swizzle<kKChunks>(kPageStep) == 0 && value_swizzle<kVChunks>(kPageStep) == 0,
                  "a wave's rows have the tile's swizzles");
  }

  __device__ __forceinline__ void find_pages(int k0) {
    const int64_t at = static_cast<int64_t>(k0) + kAttnKeys * lane + kPageStep * wave;
    page = -1, row = 0;
    if (at < lk) {  // (so within the table)
      const uint32_t block = static_cast<uint32_t>(at) / static_cast<uint32_t>(a.table.page_rows);
      row = static_cast<int>(at) - static_cast<int>(block) * a.table.page_rows;
      page = pages[block];
      if (page >= a.table.pages) page = -1;
    }
    first = k0;
  }

  // Rows without a page, and those behind the sequence's last, read as zeros.
  // ONCE: past the caches, for keys that one block reads (attend_few).
  template <bool ONCE = false>
  __device__ __forceinline__ void fetch(int64_t at, int buf) {
    const int k0 = static_cast<int>(at);
    if (k0 >= first + kAttnKeys * kWave) find_pages(k0);
    const int j = (k0 - first) / kAttnKeys;
    const int pg = __builtin_amdgcn_readlane(page, j), r0 = __builtin_amdgcn_readlane(row, j);
    const int left = lk - k0 - kPageStep * wave, rows = left < kPageStep ? left : kPageStep;
    const int64_t in = pg < 0 ? 0 : pg;
    const u32x4_t rk = buffer_rsrc(kb + in * a.k_page + r0 * a.k_row,
                                   pg < 0 ? 0 : ((rows - 1) * a.k_row + a.d_qk) * 2);
    const u32x4_t rv = buffer_rsrc(vb + in * a.v_page + r0 * a.v_row,
                                   pg < 0 ? 0 : ((rows - 1) * a.v_row + a.d_v) * 2);
    const uint32_t base = lds + buf * kAttnKeys * (DQ + DV) * 2;
#pragma unroll
    for (int i = 0; i < kKLoads; ++i)
      lds_direct16<ONCE>(rk, base + (wave * kKLoads + i) * kWave * 16, koff[i], 0);
#pragma unroll
    for (int i = 0; i < kVLoads; ++i)
      lds_direct16<ONCE>(rv, base + kAttnKeys * DQ * 2 + (wave * kVLoads + i) * kWave * 16, voff[i], 0);
  }

  __device__ __forceinline__ const uint16_t* value_row(int64_t key) const {
    const int block = static_cast<int>(key) / a.table.page_rows;
    const int64_t pg = pages[block];
    if (pg < 0 || pg >= a.table.pages) return nullptr;
    return vb + pg * a.v_page + (key - static_cast<int64_t>(block) * a.table.page_rows) * a.v_row;
  }
};

template <bool BF16>
__device__ inline f32x4_t mfma16(u32x4_t a, u32x4_t b, f32x4_t c) {
  if constexpr (BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// 16 x 16 x 16: a lane has four of k, 4 (lane / 16) to + 3, as it gets four rows of a product.
template <bool BF16>
__device__ inline f32x4_t mfma16_half(uint2 a, uint2 b, f32x4_t c) {
  if constexpr (BF16) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(i16x4_t, a),
                                                     __builtin_bit_cast(i16x4_t, b), c, 0, 0, 0);
  } else {
    typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4_t, a),
                                                 __builtin_bit_cast(f16x4_t, b), c, 0, 0, 0);
  }
}

// Up to 16 GROUPS rows (queries x heads of one key head) against the run's keys: the four
// waves take 16 keys of each 64, every wave with a maximum and sums of its own and no
// barrier between them, since a wave reads what it staged itself; at the end the four
// are joined. S^T = K Q^T and O^T += V^T P^T as in attend_rows, on 16 x 16 tiles: a
// lane holds four scores of a row, which rounded are its part of the next
// product's operand.
//
// Bound by HBM: two tiles of 64 keys a block, two blocks a CU, keep up to 128 KB a CU on their
// way. 64 tokens on up to 8192 keys x 8 heads of 128 (1.1 GB) take 191 us in all, 5.7 TB/s (7.0 is
// what a kernel that only reads reaches here). Loads go past the caches: 64 tokens on 8192 keys each take
// 346 us, 382 through the caches. Where several blocks read the same keys the caches would serve, and
// the kernel does not look for that: several packs on a key head (64 heads on 1, 64 tokens on 16384
// keys: 195 us, 170 through the caches; 37 on 1, a pack each, on 8192: 1271 and 547) and forks of one
// prompt (64 of one of 8192: 136 and 124).
template <bool BF16, int DQ, int DV, int GROUPS>
__device__ __forceinline__ void attend_few(const PagedArgs& a, const AttnBlock& b,
                                           PagedKeys<DQ, DV>& keys_of, uint16_t* stage,
                                           float* part) {
  constexpr int kQSteps = DQ / 32, kVTiles = DV / 16, kKChunks = DQ / 8, kVChunks = DV / 8;
  constexpr int kStage = kAttnKeys * (DQ + DV);
  constexpr int kLoads = PagedKeys<DQ, DV>::kKLoads + PagedKeys<DQ, DV>::kVLoads;  // of a tile
  constexpr float kLift = BF16 ? 0.f : 6.f;
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int n = lane & 15, g = lane >> 4;
  const int lq = static_cast<int>(b.q.end - b.q.begin), lk = static_cast<int>(b.lk);
  int token[GROUPS];
#pragma unroll
  for (int j = 0; j < GROUPS; ++j) token[j] = (kFewRows * j + n) * a.inv_pack >> 16;
  const int ahead = static_cast<int>(b.ahead);
  const int first_sees = ahead < lk ? ahead : lk - 1;  // the last key that the first query sees
  int sees[GROUPS];                                    // and the lane's
#pragma unroll
  for (int j = 0; j < GROUPS; ++j) sees[j] = token[j] + ahead < lk ? token[j] + ahead : lk - 1;
  const int per = ((lk + b.splits - 1) / b.splits + kAttnKeys - 1) / kAttnKeys * kAttnKeys;
  const int64_t from64 = static_cast<int64_t>(b.split) * per;
  const int from = from64 < lk ? static_cast<int>(from64) : lk;
  const int to = lk - from < per ? lk : from + per;
  u32x4_t qf[GROUPS][kQSteps];
#pragma unroll
  for (int j = 0; j < GROUPS; ++j) {
    const int64_t head = b.pack * a.pack + kFewRows * j + n - token[j] * a.pack;
    const uint16_t* const qp =
        a.q + (b.q.begin + (token[j] < lq ? token[j] : lq - 1)) * a.q_row + head * a.q_head;
#pragma unroll
    for (int i = 0; i < kQSteps; ++i) {
      const int d = 32 * i + 8 * g;
      const u32x4_t z = {0u, 0u, 0u, 0u};
      qf[j][i] = d < a.d_qk ? *reinterpret_cast<const u32x4_t*>(qp + d) : z;
      qf[j][i] = (qf[j][i] & a.q_keep) ^ a.q_flip;
    }
  }
  f32x4_t o[GROUPS][kVTiles];
  float top[GROUPS], sum[GROUPS];
#pragma unroll
  for (int j = 0; j < GROUPS; ++j) {
    top[j] = -INFINITY, sum[j] = 0.f;
#pragma unroll
    for (int t = 0; t < kVTiles; ++t) o[j][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  // where this lane reads in its wave's rows of a tile: K row n, chunks 4 i + g; V row
  // 4 g + lane % 16 / 4, columns 16 t + 4 (lane % 4)
  constexpr int kAddrs = kKChunks % 16 == 0 ? 4 : 2;
  int kaddr[kAddrs];
#pragma unroll
  for (int i = 0; i < kAddrs; ++i)
    kaddr[i] = (kPageStep * wave + n) * DQ + 8 * ((4 * i + g) ^ key_swizzle<kKChunks>(n));
  int vaddr[kVTiles];
#pragma unroll
  for (int t = 0; t < kVTiles; ++t) {
    const int row = 4 * g + n / 4, col = 16 * t + 4 * (lane & 3);
    vaddr[t] = kAttnKeys * DQ + (kPageStep * wave + row) * DV +
               8 * ((col / 8) ^ value_swizzle<kVChunks>(row)) + col % 8;
  }
  bool bad = false;
  if (from < to) keys_of.template fetch<true>(from, 0);
  if (from + kAttnKeys < to) keys_of.template fetch<true>(from + kAttnKeys, 1);
  int buf = 0;
  for (int k0 = from; k0 < to; k0 += kAttnKeys, buf ^= 1) {
    if (k0 + kAttnKeys < to) wait_vmcnt<kLoads>();
    else wait_vmcnt<0>();
    const uint16_t* const tile = stage + buf * kStage;
    const int p0 = k0 + kPageStep * wave;
    u32x4_t kf[kQSteps];
    uint2 vf[kVTiles];
#pragma unroll
    for (int i = 0; i < kQSteps; ++i)
      kf[i] = *reinterpret_cast<const u32x4_t*>(tile + kaddr[i % kAddrs] + 32 * kAddrs * (i / kAddrs));
#pragma unroll
    for (int t = 0; t < kVTiles; ++t) vf[t] = lds_read_transposed(tile + vaddr[t]);
    // once it is all in registers, its place may be filled again
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (k0 + 2 * kAttnKeys < to) keys_of.template fetch<true>(k0 + 2 * kAttnKeys, buf);
    if (p0 < lk) {
      const bool edge = p0 + kPageStep - 1 > first_sees;  // not seen by every query
      if (edge) {
#pragma unroll
        for (int t = 0; t < kVTiles; ++t) {
          const u32x4_t both = {vf[t].x, vf[t].y, 0u, 0u};
          if (__builtin_expect(__any(any_nonfinite<BF16>(both)), 0)) {
            bad = true;
            const u32x4_t kept = finite_only<BF16>(both);
            vf[t] = make_uint2(kept[0], kept[1]);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) {
        f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kQSteps; ++i) s = mfma16<BF16>(kf[i], qf[j][i], s);
        if (edge) {
          const int seen = sees[j] + 1 - p0 - 4 * g;
#pragma unroll
          for (int i = 0; i < 4; ++i) s[i] = i < seen ? s[i] : -INFINITY;
        }
        float most = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
        {
          auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(most), __float_as_uint(most),
                                                    false, false);
          most = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
          x = __builtin_amdgcn_permlane32_swap(__float_as_uint(most), __float_as_uint(most), false,
                                               false);
          most = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])) * a.scale_log2;
        }
        constexpr float kSlack = 8.f;  // as in attend_rows
        const bool moves = most > top[j] + kSlack;
        if (__any(moves)) {
          const float next = moves ? most : top[j];
          const float fade = next == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(top[j] - next);
          top[j] = next;
          sum[j] *= fade;
#pragma unroll
          for (int t = 0; t < kVTiles; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[j][t][i] *= fade;
        }
        const float base = kLift - (top[j] == -INFINITY ? 0.f : top[j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], a.scale_log2, base));
        sum[j] += (s[0] + s[1]) + (s[2] + s[3]);
        const uint2 p = make_uint2(pack2<BF16>(s[0], s[1]), pack2<BF16>(s[2], s[3]));
#pragma unroll
        for (int t = 0; t < kVTiles; ++t) o[j][t] = mfma16_half<BF16>(vf[t], p, o[j][t]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < GROUPS; ++j) {
    auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(sum[j]), __float_as_uint(sum[j]), false, false);
    sum[j] = __uint_as_float(x[0]) + __uint_as_float(x[1]);
    x = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum[j]), __float_as_uint(sum[j]), false, false);
    sum[j] = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  }
  if (__builtin_expect(bad, 0)) {
    // the infinities and NaNs left out above, for the queries that see them
    int left = a.d_v - 4 * g;
#pragma unroll 1
    for (int key = from; key < to; ++key) {
      const int p0 = key / kPageStep * kPageStep;
      if ((p0 - from) / kPageStep % kAttnWaves != wave || p0 + kPageStep - 1 <= first_sees) continue;
      const uint16_t* const row = keys_of.value_row(key);
      if (!row) continue;
      asm volatile("" : "+v"(left));  // (as in attend_rows)
#pragma unroll
      for (int j = 0; j < GROUPS; ++j)
#pragma unroll
        for (int t = 0; t < kVTiles; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int d = 16 * t + i;
            const float x = d < left && key <= sees[j] ? value_of<BF16>(row[4 * g + d]) : 0.f;
            if (!(fabsf(x) < INFINITY)) o[j][t][i] += x;
          }
    }
  }
  // the four waves' sums, through LDS, 16 rows at a time
  constexpr int kRow = DV + 4, kCols = DV / 16;
  float* const sums = reinterpret_cast<float*>(stage);
  float* const tops = sums + kAttnWaves * kFewRows * kRow;  // then the sums of p
  static_assert(kAttnWaves * kFewRows * (kRow + 2) * 4 <= 2 * kStage * 2, "sums in LDS");
#pragma unroll
  for (int j = 0; j < GROUPS; ++j) {
    __syncthreads();
#pragma unroll
    for (int t = 0; t < kVTiles; ++t)
      *reinterpret_cast<f32x4_t*>(sums + (wave * kFewRows + n) * kRow + 16 * t + 4 * g) = o[j][t];
    if (g == 0) {
      tops[wave * kFewRows + n] = top[j];
      tops[(kAttnWaves + wave) * kFewRows + n] = sum[j];
    }
    __syncthreads();
    const int mine = tid / 16, col = tid % 16 * kCols;
    const int row = kFewRows * j + mine, query = row * a.inv_pack >> 16;
    if (query >= lq) continue;
    float all = -INFINITY, total = 0.f, acc[kCols] = {};
#pragma unroll
    for (int w = 0; w < kAttnWaves; ++w) all = fmaxf(all, tops[w * kFewRows + mine]);
#pragma unroll
    for (int w = 0; w < kAttnWaves; ++w) {
      const float t = tops[w * kFewRows + mine];
      const float weight = t == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(t - all);
      total = fmaf(weight, tops[(kAttnWaves + w) * kFewRows + mine], total);
      const float* const from_wave = sums + (w * kFewRows + mine) * kRow + col;
#pragma unroll
      for (int c = 0; c < kCols; ++c) acc[c] = fmaf(weight, from_wave[c], acc[c]);
    }
    if (part) {
#pragma unroll
      for (int c = 0; c < kCols; c += 4)
        *reinterpret_cast<float4*>(part + row * DV + col + c) =
            make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
      if (col == 0) {
        part[kFewRows * GROUPS * DV + row] = all;
        part[kFewRows * GROUPS * (DV + 1) + row] = total;
      }
      continue;
    }
    const float inv = total == 0.f ? 0.f : 1.0f / total;
    const int64_t head = b.pack * a.pack + row - query * a.pack;
    uint16_t* const out = a.out + ((b.q.begin + query) * a.heads + head) * a.d_v + col;
#pragma unroll
    for (int c = 0; c < kCols; c += 4)
      if (col + c < a.d_v)
        *reinterpret_cast<uint2*>(out + c) =
            make_uint2(pack2<BF16>(within_type<BF16>(acc[c] * inv), within_type<BF16>(acc[c + 1] * inv)),
                       pack2<BF16>(within_type<BF16>(acc[c + 2] * inv),
                                   within_type<BF16>(acc[c + 3] * inv)));
  }
}

// ---------------------------------------------------------------------------
// Who does what. A call's work is found on the device, from the lengths as they are:
// sequence s has ceil(n / tokens) tiles of rows (one of up to 16 or 32 rows where its
// new tokens fit) for each pack of heads, and every tile's keys are taken in runs of about
// L keys, L = a kFill-th of all keys that the call's tiles see (twice that for tiles of
// kAttnRows), kMinRun at the least. Each block finds its tile and run by a scan over the
// sequences, 64 at a time, or from paged_plan_kernel's; the rows behind the last sequence come
// after all. A tile in runs is noted for the join.
//
// Blocks: tiles <= packs (rows / tokens + sequences + 1), and runs beyond one a tile <=
// kFill, since L kFill >= all keys. A tile in runs has more than L keys, so there are up to
// kFill of those, with fewer than 2 kFill runs.

struct PagedTile {
  RowRange q;
  int lk, tiles, runs;
  int ahead;  // positions before its first new one, lk at the most
  int units;  // of kFewRows rows that a tile has: 1, 2 or those of kAttnRows
};
constexpr int kManyUnits = kAttnRows / kFewRows;

__device__ inline PagedTile paged_tiles(const PagedArgs& a, int s) {
  PagedTile t{};
  if (s >= a.sq.count) return t;
  t.q = sequence_rows(a.sq, s);
  const int lq = static_cast<int>(t.q.end - t.q.begin);
  if (lq == 0) return t;
  t.lk = static_cast<int>(cached_length(a.table, s));
  t.ahead = static_cast<int>(positions_before(a.table, s, lq));
  t.ahead = t.ahead < t.lk ? t.ahead : t.lk;
  const int64_t rows = static_cast<int64_t>(lq) * a.pack;
  t.units = rows <= kFewRows ? 1 : (rows <= 2 * kFewRows ? 2 : kManyUnits);
  t.tiles = t.units < kManyUnits ? 1 : (lq + a.tokens - 1) / a.tokens;
  t.runs = 1;
  return t;
}

// Keys that a row of the sequence sees, in the mean.
__device__ inline float keys_seen(const PagedTile& t) {
  const float lk = static_cast<float>(t.lk), lq = static_cast<float>(t.q.end - t.q.begin);
  return fmaxf(lk - 0.5f * lq, 0.5f * lk);
}

__device__ inline uint32_t scan_wave(uint32_t v) {
  v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x111, 0xF, 0xF, false));
  v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x112, 0xF, 0xF, false));
  v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x114, 0xF, 0xF, false));
  v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x118, 0xF, 0xF, false));
  v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x142, 0xA, 0xF, false));
  v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x143, 0xC, 0xF, false));
  return v;
}

__device__ inline int from_lane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

struct PagedItem {
  AttnBlock b;
  int sequence;  // -1: there is none of this number
  int units;     // of kFewRows rows: 1, 2 or kManyUnits
  uint32_t unit;  // where its sums go (its runs' begin), in units of kFewRows rows
  uint32_t tile;  // its number among the tiles in runs
};

// Keys of a run, about: tiles of few rows, and of kAttnRows.
struct RunLengths {
  float few, many;
};

__device__ inline RunLengths run_lengths(float work) {
  // (a 1024th more than the mean, for what rounding can lose)
  const float share = work * (1.0009765625f / kFill);
  return {fmaxf(static_cast<float>(kMinRun), ceilf(share)),
          fmaxf(static_cast<float>(kMinRun), ceilf(2.f * share))};
}

__device__ inline float tile_work(const PagedArgs& a, const PagedTile& t) {
  return keys_seen(t) * static_cast<float>(t.tiles) * static_cast<float>(a.packs);
}

__device__ inline int runs_of(const PagedArgs& a, const PagedTile& t, const RunLengths& length) {
  if (!a.partial || t.tiles == 0) return 1;
  const float n = ceilf(keys_seen(t) / (t.units < kManyUnits ? length.few : length.many));
  return n < 2.f ? 1 : (n > static_cast<float>(kWave) ? kWave : static_cast<int>(n));
}

// What comes before a sequence: blocks, units of sums, tiles in runs; and its own runs.
struct PlanEntry {
  uint32_t first, unit, split;
  int runs;
};

// Block `local` of sequence `s`, with what comes before it.
__device__ inline void place_item(const PagedArgs& a, int s, const PagedTile& own, uint32_t local,
                                  const PlanEntry& before, PagedItem& item) {
  const uint32_t packs = a.packs;
  item.units = own.units;
  item.sequence = s;
  item.b.pack = __builtin_amdgcn_readfirstlane(local % packs);
  item.b.split = __builtin_amdgcn_readfirstlane(local / packs % before.runs);
  item.b.splits = before.runs;
  // later tiles see more keys, and are begun first
  const int tile =
      own.tiles - 1 - static_cast<int>(__builtin_amdgcn_readfirstlane(local / packs / before.runs));
  const uint32_t index = tile * packs + item.b.pack, step = own.units;
  const bool few = step < kManyUnits;
  item.unit = before.unit + (index * before.runs + item.b.split) * step;
  item.tile = before.split + index;
  item.b.q = own.q;
  item.b.lk = own.lk;
  item.b.ahead = own.ahead;
  const int64_t lq = own.q.end - own.q.begin;
  item.b.q0 = few ? 0 : static_cast<int64_t>(tile) * a.tokens;
  item.b.last = few || lq - item.b.q0 < a.tokens ? lq : item.b.q0 + a.tokens;
  // (offsets that are not in order can ask for more than there is)
  if (tile < 0 || tile >= own.tiles ||
      (before.runs > 1 && (item.unit >= a.units || a.units - item.unit < step || item.tile >= kFill)))
    item.sequence = -1;
}

// Tile and run of block `number`. A number beyond the last gets the count of tiles in
// runs in `tile`.
__device__ inline PagedItem find_item(const PagedArgs& a, uint32_t number) {
  const int lane = static_cast<int>(threadIdx.x & (kWave - 1));
  PagedItem item{};
  item.sequence = -1;
  const int count = a.sq.count;
  uint32_t before = 0, units_before = 0, split_before = 0;
  if (a.plan) {
    // the last sequence that begins at or before this number, 64 candidates at a time
    int lo = 0, span = count + 1;
    while (span > 1) {
      const int step = (span + kWave - 1) / kWave, off = lane * step, at = lo + (off < span ? off : 0);
      const int n = __popcll(__ballot(off < span && a.plan[at].first <= number));
      const int skip = n > 0 ? (n - 1) * step : 0;
      lo += skip;
      span = span - skip < step ? span - skip : step;
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    const PlanEntry entry = a.plan[lo];
    if (lo < count) {
      const PagedTile own = paged_tiles(a, lo);
      if (number >= entry.first) place_item(a, lo, own, number - entry.first, entry, item);
      return item;
    }
    before = entry.first;
  } else {
    PagedTile own = paged_tiles(a, lane);
    RunLengths length{};
    if (a.partial) {
      float work = tile_work(a, own);
      for (int s = kWave; s < count; s += kWave) work += tile_work(a, paged_tiles(a, s + lane));
      length = run_lengths(over_wave(work, [](float x, float y) { return x + y; }));
    }
    for (int s0 = 0; s0 < count; s0 += kWave) {
      if (s0 > 0) own = paged_tiles(a, s0 + lane);
      own.runs = runs_of(a, own, length);
      const uint32_t tiles = static_cast<uint32_t>(own.tiles) * a.packs, mine = tiles * own.runs;
      const uint32_t split = own.runs > 1 ? tiles : 0u;
      const uint32_t units = split * own.runs * own.units;
      const uint32_t upto = scan_wave(mine), units_upto = scan_wave(units), split_upto = scan_wave(split);
      const uint64_t hit = __ballot(number < before + upto);
      if (hit) {
        const int at = __builtin_ctzll(hit);
        PagedTile t{};
        t.q.begin = from_lane(static_cast<int>(own.q.begin), at);  // (rows are below 2^31)
        t.q.end = from_lane(static_cast<int>(own.q.end), at);
        t.lk = from_lane(own.lk, at);
        t.ahead = from_lane(own.ahead, at);
        t.tiles = from_lane(own.tiles, at);
        t.units = from_lane(own.units, at);
        const PlanEntry entry{before + from_lane(upto - mine, at),
                              units_before + from_lane(units_upto - units, at),
                              split_before + from_lane(split_upto - split, at),
                              from_lane(own.runs, at)};
        place_item(a, s0 + at, t, number - entry.first, entry, item);
        return item;
      }
      before += from_lane(upto, kWave - 1);
      units_before += from_lane(units_upto, kWave - 1);
      split_before += from_lane(split_upto, kWave - 1);
    }
    item.tile = split_before;
  }
  // the rows behind the last sequence
  const uint32_t packs = a.packs, local = number - before, tile = local / packs;
  const RowRange rows = sequence_rows(a.sq, count);
  const int64_t lq = rows.end - rows.begin, q0 = static_cast<int64_t>(tile) * a.tokens;
  if (q0 < lq) {
    item.sequence = count;
    item.b.pack = __builtin_amdgcn_readfirstlane(local % packs);
    item.b.splits = 1;
    item.b.q = rows;
    item.b.q0 = q0;
    item.b.last = lq - q0 < a.tokens ? lq : q0 + a.tokens;
  }
  return item;
}

// The same scan once for all blocks, by a block of its own. (Its runs may differ from those that
// the blocks would find by a rounding of `work`; a call has the one or the others.)
constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / kWave;
__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(PagedArgs a) {
  __shared__ float works[kPlanWaves];
  __shared__ uint32_t sums[3][kPlanWaves];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave, count = a.sq.count;
  RunLengths length{};
  if (a.partial) {
    float work = 0.f;
    for (int s = tid; s < count; s += kPlanThreads) work += tile_work(a, paged_tiles(a, s));
    work = over_wave(work, [](float x, float y) { return x + y; });
    if (lane == 0) works[wave] = work;
    __syncthreads();
    work = 0.f;
    for (int w = 0; w < kPlanWaves; ++w) work += works[w];
    length = run_lengths(work);
  }
  uint32_t before[3] = {0, 0, 0};
  for (int s0 = 0; s0 <= count; s0 += kPlanThreads) {
    const int s = s0 + tid;
    const PagedTile own = paged_tiles(a, s);
    const int runs = runs_of(a, own, length);
    const uint32_t tiles = static_cast<uint32_t>(own.tiles) * a.packs;
    const uint32_t split = runs > 1 ? tiles : 0u;
    const uint32_t mine[3] = {tiles * runs, split * runs * own.units, split};
    uint32_t upto[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      upto[i] = scan_wave(mine[i]);
      if (lane == kWave - 1) sums[i][wave] = upto[i];
    }
    __syncthreads();
    uint32_t at[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      at[i] = before[i] + upto[i] - mine[i];
      for (int w = 0; w < kPlanWaves; ++w) {
        if (w < wave) at[i] += sums[i][w];
        before[i] += sums[i][w];
      }
    }
    if (s <= count) a.plan[s] = PlanEntry{at[0], at[1], at[2], runs};
    if (s == count && a.partial) a.split->count = at[2] < kFill ? static_cast<int>(at[2]) : kFill;
    __syncthreads();
  }
}

template <int DV>
__device__ inline float* sums_of(const PagedArgs& a, uint32_t unit) {
  return a.partial + static_cast<int64_t>(unit) * (kFewRows * (DV + 2));
}

template <bool BF16, int DQ, int DV>
__global__ void __launch_bounds__(kAttnThreads, 2) paged_attend_kernel(PagedArgs a) {
  constexpr int kVTiles = DV / 32;
  __shared__ alignas(16) uint16_t stage[2 * kAttnKeys * (DQ + DV)];
  const PagedItem item = find_item(a, blockIdx.x);
  // (the last number is beyond all tiles)
  if (a.partial && !a.plan && blockIdx.x == gridDim.x - 1 && threadIdx.x == 0)
    a.split->count = item.tile < kFill ? static_cast<int>(item.tile) : kFill;
  if (item.sequence < 0) return;
  const AttnBlock& b = item.b;
  float* part = nullptr;
  if (b.splits > 1) {
    part = sums_of<DV>(a, item.unit);
    if (b.split == 0 && threadIdx.x == 0)
      a.split->tile[item.tile] = SplitTile{b.q.begin + b.q0, static_cast<int>(b.last - b.q0) * a.pack,
                                           b.pack, b.splits, item.units, item.unit};
  }
  if (item.units < kManyUnits && item.sequence < a.sq.count) {
    PagedKeys<DQ, DV> keys(a, b, item.sequence, stage);
    if (item.units == 2) attend_few<BF16, DQ, DV, 2>(a, b, keys, stage, part);
    else attend_few<BF16, DQ, DV, 1>(a, b, keys, stage, part);
    return;
  }
  f32x16_t o[kVTiles];
#pragma unroll
  for (int t = 0; t < kVTiles; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[t][r] = 0.f;
  float top = -INFINITY, sum = 0.f;
  if (item.sequence < a.sq.count) {
    PagedKeys<DQ, DV> keys(a, b, item.sequence, stage);
    attend_rows<BF16, DQ, DV>(a, b, keys, stage, o, top, sum);
  }
  if (part) store_sums<DV>(a, b, part, o, top, sum);
  else store_rows<BF16, DQ, DV>(a, b, stage, o, sum);
}

// Output row of a tile from its joined sums: a lane two columns (one of 64).
template <bool BF16, int DV>
__device__ inline void store_joined(const PagedArgs& a, const SplitTile& tile, int row,
                                    const float (&acc)[DV / 64], float total) {
  const int lane = threadIdx.x & (kWave - 1), token = row * a.inv_pack >> 16;
  const float inv = total == 0.f ? 0.f : 1.0f / total;
  uint16_t* const out = a.out + ((tile.row + token) * a.heads + tile.pack * a.pack + row -
                                 token * a.pack) * static_cast<int64_t>(a.d_v);
  if constexpr (DV == 128) {
    if (2 * lane < a.d_v)
      *reinterpret_cast<uint32_t*>(out + 2 * lane) =
          pack2<BF16>(within_type<BF16>(acc[0] * inv), within_type<BF16>(acc[1] * inv));
  } else {
    if (lane < a.d_v)
      out[lane] = static_cast<uint16_t>(pack2<BF16>(within_type<BF16>(acc[0] * inv), 0.f));
  }
}

// ROWS rows of a tile in runs: weights 2^(top - largest top) of the runs, a lane each,
// then the runs from `begin` on, RUNS of them, a lane its columns. Rows that do not
// exist read the first's. Every load is on its way before the first is used.
template <int DV, int ROWS, int RUNS>
__device__ inline void join_rows(const float* sums, int size, int most, int runs, int begin,
                                 const int (&row)[ROWS], float (&acc)[ROWS][DV / 64],
                                 float (&total)[ROWS]) {
  constexpr int kCols = DV / 64;
  const int lane = threadIdx.x & (kWave - 1);
  const float* const tops = sums + (lane < runs ? lane : 0) * size + most * DV;
  float weight[ROWS], x[ROWS][RUNS][kCols];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    weight[r] = lane < runs ? tops[row[r]] : -INFINITY;
    total[r] = lane < runs ? tops[most + row[r]] : 0.f;
#pragma unroll
    for (int i = 0; i < RUNS; ++i)
#pragma unroll
      for (int c = 0; c < kCols; ++c)
        x[r][i][c] = sums[(begin + i < runs ? begin + i : 0) * size + row[r] * DV + kCols * lane + c];
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const float top = over_wave(weight[r], [](float x, float y) { return fmaxf(x, y); });
    weight[r] = weight[r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(weight[r] - top);
    total[r] = over_wave(total[r] * weight[r], [](float x, float y) { return x + y; });
#pragma unroll
    for (int c = 0; c < kCols; ++c) acc[r][c] = 0.f;
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
      const float w = __uint_as_float(
          __builtin_amdgcn_readlane(__float_as_uint(weight[r]), (begin + i) & (kWave - 1)));
#pragma unroll
      for (int c = 0; c < kCols; ++c)
        acc[r][c] = begin + i < runs ? fmaf(w, x[r][i][c], acc[r][c]) : acc[r][c];
    }
  }
}

// The runs of a tile joined, in their order: a block takes a quarter of a tile of 16 or 32
// rows, 16 rows of one of 128. Up to kJoinRuns runs a wave joins a row by itself, two at a time; more are dealt
// over the four waves, whose sums then meet in LDS.
// Bound by latency: the tile, then one trip to memory for each turn of the loop.
constexpr int kJoinRuns = 8;
template <bool BF16, int DV>
__global__ void __launch_bounds__(kAttnThreads) paged_join_kernel(PagedArgs a, int parts) {
  constexpr int kCols = DV / 64, kShare = kWave / kAttnWaves;  // runs of a wave
  __shared__ float shared[kAttnWaves][kAttnWaves][DV];
  const int index = static_cast<int>(blockIdx.x) / parts;
  if (index >= a.split->count) return;
  const SplitTile tile = a.split->tile[index];
  // (offsets that are not in order can leave tiles unnoted, so that this is what the workspace held:
  // whatever that is, nothing outside the tensors)
  if (tile.runs < 2 || tile.runs > kWave || tile.pack < 0 || tile.pack >= a.packs || tile.row < 0 ||
      tile.units < 1 || tile.units > kManyUnits || tile.rows < 0 ||
      tile.rows > tile.units * kFewRows || tile.row > a.sq.rows ||
      (a.sq.rows - tile.row) * a.pack < tile.rows ||
      tile.unit >= a.units || a.units - tile.unit < static_cast<uint32_t>(tile.runs * tile.units))
    return;
  const int lane = threadIdx.x & (kWave - 1), runs = tile.runs;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int most = tile.units * kFewRows, size = most * (DV + 2);
  // the rows that exist are the first ones: tokens of `pack` heads
  const int step = tile.units < kManyUnits ? kJoinFew * tile.units : kJoinMany;
  const int begin = static_cast<int>(blockIdx.x) % parts * step;
  const int end = begin + step < tile.rows ? begin + step : tile.rows;
  if (begin >= end) return;
  const float* const sums = sums_of<DV>(a, tile.unit);
  if (runs <= kJoinRuns) {
    for (int row0 = begin + wave; row0 < end; row0 += 2 * kAttnWaves) {
      const bool two = row0 + kAttnWaves < end;
      const int row[2] = {row0, two ? row0 + kAttnWaves : row0};
      float acc[2][kCols], total[2];
      join_rows<DV, 2, kJoinRuns>(sums, size, most, runs, 0, row, acc, total);
      store_joined<BF16, DV>(a, tile, row[0], acc[0], total[0]);
      if (two) store_joined<BF16, DV>(a, tile, row[1], acc[1], total[1]);
    }
    return;
  }
  for (int row0 = begin; row0 < end; row0 += kAttnWaves) {
    int row[kAttnWaves];
#pragma unroll
    for (int r = 0; r < kAttnWaves; ++r) row[r] = row0 + r < end ? row0 + r : row0;
    float acc[kAttnWaves][kCols], total[kAttnWaves];
    join_rows<DV, kAttnWaves, kShare>(sums, size, most, runs, wave * kShare, row, acc, total);
    if (row0 > begin) __syncthreads();
#pragma unroll
    for (int r = 0; r < kAttnWaves; ++r)
#pragma unroll
      for (int c = 0; c < kCols; ++c) shared[wave][r][kCols * lane + c] = acc[r][c];
    __syncthreads();
    if (row0 + wave < end) {
      float all[kCols] = {}, sum = total[0];
#pragma unroll
      for (int r = 1; r < kAttnWaves; ++r) sum = wave == r ? total[r] : sum;
#pragma unroll
      for (int w = 0; w < kAttnWaves; ++w)
#pragma unroll
        for (int c = 0; c < kCols; ++c) all[c] += shared[w][wave][kCols * lane + c];
      store_joined<BF16, DV>(a, tile, row0 + wave, all, sum);
    }
  }
}

constexpr int64_t kSplitBytes = (sizeof(SplitTiles) + 255) / 256 * 256;

// The most units that a tile of the call can have.
int most_units(int64_t rows, int64_t sequences, bool packed, int pack) {
  const int64_t most = (packed ? rows : rows / sequences) * pack;
  return most <= kFewRows ? 1 : (most <= 2 * kFewRows ? 2 : kManyUnits);
}

int64_t paged_units(int64_t rows, int64_t sequences, bool packed, int64_t capacity, int pack) {
  if (capacity <= kMinRun) return 0;  // no tile has more keys than one run
  return int64_t{2} * kFill * most_units(rows, sequences, packed, pack);
}

int64_t plan_bytes(int64_t sequences) {
  if (sequences < kPlanSequences) return 0;
  return ((sequences + 1) * static_cast<int64_t>(sizeof(PlanEntry)) + 255) / 256 * 256;
}

template <bool BF16>
int launch_paged(const PagedArgs& a, hipStream_t s) {
  constexpr const char* kName = "lk_attention_paged";
  const int64_t tiles_most = a.packs * (a.sq.rows / a.tokens + a.sq.count + 1);
  const int64_t blocks = tiles_most + (a.partial ? kFill + 1 : 0);
  LK_REQUIRE(grid_fits(blocks, kAttnThreads), "too many query rows and heads for one call");
  const bool few = most_units(a.sq.rows, a.sq.count, a.sq.cu != nullptr, a.pack) < kManyUnits;
  const int parts = few ? kFewRows / kJoinFew : kAttnRows / kJoinMany;
  const int64_t tiles = std::min<int64_t>(kFill, tiles_most);
  if (a.plan) {
    paged_plan_kernel<<<1, kPlanThreads, 0, s>>>(a);
    if (const int st = check_launch(kName)) return st;
  }
  const dim3 grid(static_cast<unsigned>(blocks)), join(static_cast<unsigned>(tiles * parts));
#define LK_PAGED(Q, V)                                                   \
  if (a.d_qk <= Q && a.d_v <= V) {                                       \
    paged_attend_kernel<BF16, Q, V><<<grid, kAttnThreads, 0, s>>>(a);    \
    if (a.partial) {                                                     \
      if (const int st = check_launch(kName)) return st;                 \
      paged_join_kernel<BF16, V><<<join, kAttnThreads, 0, s>>>(a, parts); \
    }                                                                    \
    return check_launch(kName);                                          \
  }
  LK_PAGED(64, 64)
  LK_PAGED(128, 128)
  LK_PAGED(192, 128)
#undef LK_PAGED
  return fail_arg("attention head dimensions too large");
}

}  // namespace
}  // namespace lk

using namespace lk;

extern "C" {

int64_t lk_attention_paged_workspace(int64_t rows, int64_t sequences, int64_t capacity,
                                     int64_t heads, int64_t kv_heads, int64_t d_qk, int64_t d_v,
                                     int packed) {
  if (rows < 0 || sequences <= 0 || capacity < 0 || heads <= 0 || kv_heads <= 0 ||
      heads % kv_heads || d_qk <= 0 || d_v <= 0 || d_qk > kAttnMaxQk || d_v > kAttnMaxV)
    return -1;
  const int64_t dv = d_qk <= 64 && d_v <= 64 ? 64 : 128;
  const int64_t units = paged_units(rows, sequences, packed != 0, capacity, attention_pack(heads, kv_heads, kPagedPack));
  return plan_bytes(sequences) + (units == 0 ? 0 : kSplitBytes + units * kFewRows * (dv + 2) * 4);
}

int lk_attention_paged(const void* q, const void* k_pages, const void* v_pages, void* out,
                       const int32_t* page_table, const int32_t* lengths, const int32_t* cu,
                       int64_t sequences, int64_t rows, int64_t heads, int64_t kv_heads,
                       int64_t d_qk, int64_t d_v, int64_t q_row_stride, int64_t q_head_stride,
                       int64_t pages, int64_t page_rows, int64_t table_width,
                       int64_t table_stride, int64_t k_page, int64_t k_page_row,
                       int64_t k_page_head, int64_t v_page, int64_t v_page_row,
                       int64_t v_page_head, float scale, int dtype, void* workspace,
                       int64_t workspace_bytes, void* stream) {
  LK_REQUIRE(rows >= 0 && rows < (int64_t{1} << 31), "rows must be in 0 .. 2^31 - 1");
  LK_REQUIRE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && heads <= 65535,
             "attention heads must be a positive multiple of the key heads");
  LK_REQUIRE(d_qk > 0 && d_qk % 8 == 0 && d_qk <= kAttnMaxQk,
             "attention d_qk must be a multiple of 8 up to %d, got %lld", kAttnMaxQk,
             (long long)d_qk);
  LK_REQUIRE(d_v > 0 && d_v % 8 == 0 && d_v <= kAttnMaxV,
             "attention d_v must be a multiple of 8 up to %d, got %lld", kAttnMaxV,
             (long long)d_v);
  LK_REQUIRE(dtype == LK_DTYPE_F16 || dtype == LK_DTYPE_BF16,
             "attention tensors must be fp16 or bf16");
  LK_REQUIRE(q_row_stride >= 0 && q_head_stride >= 0 && q_row_stride % 8 == 0 &&
                 q_head_stride % 8 == 0,
             "strides must be multiples of 8 elements, not negative");
  if (const int st = check_pages(sequences, rows, cu != nullptr, pages, page_rows, table_width,
                                 table_stride, {k_page, k_page_row, k_page_head, v_page, v_page_row,
                                                v_page_head}))
    return st;
  LK_REQUIRE(k_page_row < (int64_t{1} << 24) && v_page_row < (int64_t{1} << 24),
             "page row strides must be below 2^24 elements");
  LK_REQUIRE(sequences <= kMaxSequences, "attention takes up to %lld sequences a call",
             (long long)kMaxSequences);
  const float scale_log2 = fabsf(scale) * 1.4426950408889634f;
  LK_REQUIRE(scale_log2 < INFINITY, "the attention scale must be finite, below 2^127");
  if (rows == 0) return LK_OK;
  LK_REQUIRE(q && out && lengths && (table_width == 0 || page_table) &&
                 (pages == 0 || (k_pages && v_pages)),
             "null pointer argument");
  for (const void* p : {q, k_pages, v_pages, static_cast<const void*>(out)})
    LK_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0,
               "attention tensors must start on a 16-byte boundary");
  const int pack = attention_pack(heads, kv_heads, kPagedPack);
  const int64_t need = lk_attention_paged_workspace(rows, sequences, table_width * page_rows, heads,
                                                    kv_heads, d_qk, d_v, cu != nullptr);
  LK_REQUIRE(need == 0 || (workspace && workspace_bytes >= need),
             "attention workspace too small: %lld bytes, %lld needed", (long long)workspace_bytes,
             (long long)need);
  LK_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
             "attention workspace must be 16-byte aligned");
  PagedArgs a{};
  a.q = static_cast<const uint16_t*>(q), a.out = static_cast<uint16_t*>(out);
  a.k = static_cast<const uint16_t*>(k_pages), a.v = static_cast<const uint16_t*>(v_pages);
  a.sq = Sequences{cu, rows, rows / sequences, static_cast<int>(sequences)};
  a.table = PageTable{page_table, lengths, table_stride, pages, static_cast<int>(table_width),
                      static_cast<int>(page_rows)};
  a.q_row = q_row_stride, a.q_head = q_head_stride;
  a.k_page = k_page, a.k_row = k_page_row, a.k_head = k_page_head;
  a.v_page = v_page, a.v_row = v_page_row, a.v_head = v_page_head;
  a.heads = static_cast<int>(heads), a.group = static_cast<int>(heads / kv_heads);
  a.d_qk = static_cast<int>(d_qk), a.d_v = static_cast<int>(d_v);
  a.pack = pack, a.inv_pack = 65536 / pack + 1, a.tokens = kAttnRows / pack;
  a.packs = static_cast<int>(heads) / pack;
  a.units = static_cast<uint32_t>(paged_units(rows, sequences, cu != nullptr, table_width * page_rows, pack));
  // the plan, the tiles in runs, their sums
  char* at = static_cast<char*>(workspace);
  if (plan_bytes(sequences)) a.plan = reinterpret_cast<PlanEntry*>(at);
  at += plan_bytes(sequences);
  if (a.units) {
    a.split = reinterpret_cast<SplitTiles*>(at);
    a.partial = reinterpret_cast<float*>(at + kSplitBytes);
  }
  a.scale_log2 = scale == 0.f ? 1.f : scale_log2;
  a.q_keep = scale == 0.f ? 0u : 0xFFFFFFFFu, a.q_flip = scale < 0.f ? 0x80008000u : 0u;
  const hipStream_t s = as_stream(stream);
  return dtype == LK_DTYPE_BF16 ? launch_paged<true>(a, s) : launch_paged<false>(a, s);
}

}  // extern "C"
