// Causal softmax attention of new rows on a paged cache, for gfx950.

#include "lk_attention_tile.hpp"
#include "lk_paged.h"

namespace lk {
namespace {

constexpr int kFewRows = 16;  // queries x heads of a block for single tokens
constexpr int kFill = 512;    // blocks that fill the chip: two a CU
constexpr int kMinRun = 256;  // keys of a run, at the least
constexpr int kJoinRows = 2;  // of a wave of the join
constexpr int kJoinBlockRows = kAttnWaves * kJoinRows;
constexpr int64_t kMaxSequences = 65536;

struct PagedArgs : AttnShape {
  const uint16_t *k, *v;
  Sequences sq;
  PageTable table;
  int64_t k_page, k_row, k_head, v_page, v_row, v_head;
  float* partial;  // sums of rows whose keys are in runs; null where none can be
  uint32_t units;  // of kFewRows rows that it holds
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
      lds_direct16(rk, base + (wave * kKLoads + i) * kWave * 16, koff[i], 0);
#pragma unroll
    for (int i = 0; i < kVLoads; ++i)
      lds_direct16(rv, base + kAttnKeys * DQ * 2 + (wave * kVLoads + i) * kWave * 16, voff[i], 0);
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

// Up to 16 rows (queries x heads of one key head) against the run's keys: the four
// waves take 16 keys of each 64, every wave with a maximum and sums of its own and no
// barrier between them, since a wave reads what it staged itself; at the end the four
// are joined. S^T = K Q^T and O^T += V^T P^T as in attend_rows, on 16 x 16 tiles: a
// lane holds four scores of a row, which rounded are its part of the next
// product's operand.
template <bool BF16, int DQ, int DV>
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
  const int token = n * a.inv_pack >> 16;
  const int ahead = lk - lq;  // query i sees the keys up to ahead + i
  const int per = ((lk + b.splits - 1) / b.splits + kAttnKeys - 1) / kAttnKeys * kAttnKeys;
  const int64_t from64 = static_cast<int64_t>(b.split) * per;
  const int from = from64 < lk ? static_cast<int>(from64) : lk;
  const int to = lk - from < per ? lk : from + per;
  u32x4_t qf[kQSteps];
  {
    const int64_t head = b.pack * a.pack + n - token * a.pack;
    const uint16_t* const qp =
        a.q + (b.q.begin + (token < lq ? token : lq - 1)) * a.q_row + head * a.q_head;
#pragma unroll
    for (int i = 0; i < kQSteps; ++i) {
      const int d = 32 * i + 8 * g;
      const u32x4_t z = {0u, 0u, 0u, 0u};
      qf[i] = d < a.d_qk ? *reinterpret_cast<const u32x4_t*>(qp + d) : z;
      qf[i] = (qf[i] & a.q_keep) ^ a.q_flip;
    }
  }
  f32x4_t o[kVTiles];
#pragma unroll
  for (int t = 0; t < kVTiles; ++t) o[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, sum = 0.f;
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
  if (from < to) keys_of.fetch(from, 0);
  if (from + kAttnKeys < to) keys_of.fetch(from + kAttnKeys, 1);
  int buf = 0;
  for (int k0 = from; k0 < to; k0 += kAttnKeys, buf ^= 1) {
    if (k0 + kAttnKeys < to) wait_vmcnt<kLoads>();
    else wait_vmcnt<0>();
    const uint16_t* const tile = stage + buf * kStage;
    const int p0 = k0 + kPageStep * wave;
    if (p0 < lk) {
      u32x4_t kf[kQSteps];
#pragma unroll
      for (int i = 0; i < kQSteps; ++i)
        kf[i] = *reinterpret_cast<const u32x4_t*>(tile + kaddr[i % kAddrs] +
                                                  32 * kAddrs * (i / kAddrs));
      uint2 vf[kVTiles];
#pragma unroll
      for (int t = 0; t < kVTiles; ++t) vf[t] = lds_read_transposed(tile + vaddr[t]);
      f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kQSteps; ++i) s = mfma16<BF16>(kf[i], qf[i], s);
      const bool edge = p0 + kPageStep - 1 > ahead;  // not seen by every query
      if (edge) {
        const int seen = token + ahead + 1 - p0 - 4 * g;
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
      const bool moves = most > top + kSlack;
      if (__any(moves)) {
        const float next = moves ? most : top;
        const float fade = next == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(top - next);
        top = next;
        sum *= fade;
#pragma unroll
        for (int t = 0; t < kVTiles; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[t][i] *= fade;
      }
      const float base = kLift - (top == -INFINITY ? 0.f : top);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], a.scale_log2, base));
      sum += (s[0] + s[1]) + (s[2] + s[3]);
      const uint2 p = make_uint2(pack2<BF16>(s[0], s[1]), pack2<BF16>(s[2], s[3]));
#pragma unroll
      for (int t = 0; t < kVTiles; ++t) {
        if (edge) {
          const u32x4_t both = {vf[t].x, vf[t].y, 0u, 0u};
          if (__builtin_expect(__any(any_nonfinite<BF16>(both)), 0)) {
            bad = true;
            const u32x4_t kept = finite_only<BF16>(both);
            vf[t] = make_uint2(kept[0], kept[1]);
          }
        }
        o[t] = mfma16_half<BF16>(vf[t], p, o[t]);
      }
    }
    // what was read above is in registers: its place may be filled again
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (k0 + 2 * kAttnKeys < to) keys_of.fetch(k0 + 2 * kAttnKeys, buf);
  }
  {
    auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
    sum = __uint_as_float(x[0]) + __uint_as_float(x[1]);
    x = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
    sum = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  }
  if (__builtin_expect(bad, 0)) {
    // the infinities and NaNs left out above, for the queries that see them
#pragma unroll 1
    for (int key = from; key < to; ++key) {
      const int p0 = key / kPageStep * kPageStep;
      if ((p0 - from) / kPageStep % kAttnWaves != wave || p0 + kPageStep - 1 <= ahead) continue;
      const uint16_t* const row = keys_of.value_row(key);
      if (!row) continue;
#pragma unroll
      for (int t = 0; t < kVTiles; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = 16 * t + 4 * g + i;
          const float x = d < a.d_v && key <= token + ahead ? value_of<BF16>(row[d]) : 0.f;
          if (!(fabsf(x) < INFINITY)) o[t][i] += x;
        }
    }
  }
  // the four waves' sums, through LDS
  constexpr int kRow = DV + 4, kCols = DV / 16;
  float* const sums = reinterpret_cast<float*>(stage);
  float* const tops = sums + kAttnWaves * kFewRows * kRow;  // then the sums of p
  static_assert(kAttnWaves * kFewRows * (kRow + 2) * 4 <= 2 * kStage * 2, "sums in LDS");
  __syncthreads();
#pragma unroll
  for (int t = 0; t < kVTiles; ++t)
    *reinterpret_cast<f32x4_t*>(sums + (wave * kFewRows + n) * kRow + 16 * t + 4 * g) = o[t];
  if (g == 0) {
    tops[wave * kFewRows + n] = top;
    tops[(kAttnWaves + wave) * kFewRows + n] = sum;
  }
  __syncthreads();
  const int row = tid / 16, col = tid % 16 * kCols, query = row * a.inv_pack >> 16;
  if (query >= lq) return;
  float all = -INFINITY, total = 0.f, acc[kCols] = {};
#pragma unroll
  for (int w = 0; w < kAttnWaves; ++w) all = fmaxf(all, tops[w * kFewRows + row]);
#pragma unroll
  for (int w = 0; w < kAttnWaves; ++w) {
    const float t = tops[w * kFewRows + row];
    const float weight = t == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(t - all);
    total = fmaf(weight, tops[(kAttnWaves + w) * kFewRows + row], total);
    const float* const from_wave = sums + (w * kFewRows + row) * kRow + col;
    // (a wave that saw nothing has zeros; one whose weight is 0 may have none)
#pragma unroll
    for (int c = 0; c < kCols; ++c) acc[c] = fmaf(weight, from_wave[c], acc[c]);
  }
  if (part) {
#pragma unroll
    for (int c = 0; c < kCols; c += 4)
      *reinterpret_cast<float4*>(part + row * DV + col + c) =
          make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
    if (col == 0) {
      part[kFewRows * DV + row] = all;
      part[kFewRows * (DV + 1) + row] = total;
    }
    return;
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

// ---------------------------------------------------------------------------
// Who does what. A call's work is found on the device, from the lengths as they are:
// sequence s has ceil(n / tokens) tiles of rows (one of up to 16 rows where its new
// tokens fit) for each pack of heads, and every tile's keys are taken in runs of about
// L keys, L = what two blocks a CU would have each if all keys of the call were dealt
// evenly, kMinRun at the least. Each block finds its tile and run by a scan over the
// sequences, 64 at a time. The rows behind the last sequence are one sequence more,
// without keys.
//
// Blocks: tiles <= packs (rows / tokens + sequences + 1), and runs beyond one a tile <=
// kFill, since L kFill >= all keys. A tile in runs has more than L keys, so there are up to
// kFill of those, with fewer than 2 kFill runs.

struct PagedTile {
  RowRange q;
  int sequence, lk, tiles, runs;
  bool few;
};

__device__ inline PagedTile paged_tiles(const PagedArgs& a, int s) {
  PagedTile t{};
  t.sequence = s;
  if (s > a.sq.count) return t;
  t.q = sequence_rows(a.sq, s);
  const int lq = static_cast<int>(t.q.end - t.q.begin);
  if (lq == 0) return t;
  t.lk = s < a.sq.count ? static_cast<int>(cached_length(a.table, s)) : 0;
  t.few = lq * a.pack <= kFewRows && s < a.sq.count;
  t.tiles = t.few ? 1 : (lq + a.tokens - 1) / a.tokens;
  t.runs = 1;
  return t;
}

// Keys that a row of the sequence sees, in the mean. (Here and in find_item nothing is
// contracted: the join has to come to the very numbers that the blocks came to.)
__device__ inline float keys_seen(const PagedTile& t) {
#pragma clang fp contract(off)
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
  bool few;
  uint32_t unit;  // where its sums go (its runs' begin), in units of kFewRows rows
};

// Tile and run of block `number`, or (JOIN) the tile in runs of this number.
template <bool JOIN>
__device__ inline PagedItem find_item(const PagedArgs& a, uint32_t number) {
#pragma clang fp contract(off)
  const int lane = static_cast<int>(threadIdx.x & (kWave - 1));
  PagedItem item{};
  item.sequence = -1;
  const int entries = a.sq.count + 1;
  PagedTile own = paged_tiles(a, lane);
  float run = 0.f;
  if (a.partial) {
    float work = keys_seen(own) * static_cast<float>(own.tiles) * static_cast<float>(a.packs);
    for (int s = kWave; s < entries; s += kWave) {
      const PagedTile t = paged_tiles(a, s + lane);
      work += keys_seen(t) * static_cast<float>(t.tiles) * static_cast<float>(a.packs);
    }
    work = over_wave(work, [](float x, float y) { return x + y; });
    // (a 1024th more than the mean, for what rounding can lose)
    run = fmaxf(static_cast<float>(kMinRun), ceilf(work * (1.0009765625f / kFill)));
  }
  uint32_t before = 0, units_before = 0;
  for (int s0 = 0; s0 < entries; s0 += kWave) {
    if (s0 > 0) own = paged_tiles(a, s0 + lane);
    if (a.partial && own.tiles > 0) {
      const float n = ceilf(keys_seen(own) / run);
      own.runs = n < 2.f ? 1 : (n > static_cast<float>(kWave) ? kWave : static_cast<int>(n));
    }
    const uint32_t rows = static_cast<uint32_t>(own.tiles * a.packs);
    const uint32_t split = own.runs > 1 ? rows : 0u;
    const uint32_t units = split * own.runs * (own.few ? 1u : kAttnRows / kFewRows);
    const uint32_t mine = JOIN ? split : rows * own.runs;
    const uint32_t upto = scan_wave(mine), units_upto = scan_wave(units);
    const uint64_t hit = __ballot(number < before + upto);
    if (hit) {
      const int at = __builtin_ctzll(hit);
      const uint32_t local = number - (before + from_lane(upto - mine, at));
      const int tiles = from_lane(own.tiles, at), runs = from_lane(own.runs, at);
      item.few = from_lane(own.few, at) != 0;
      item.sequence = s0 + at;
      const uint32_t packs = a.packs;
      const uint32_t step = JOIN ? local / packs : local / packs / runs;
      item.b.pack = __builtin_amdgcn_readfirstlane(local % packs);
      item.b.split = JOIN ? 0 : __builtin_amdgcn_readfirstlane(local / packs % runs);
      item.b.splits = runs;
      // later tiles see more keys, and are begun first
      const int tile = tiles - 1 - static_cast<int>(__builtin_amdgcn_readfirstlane(step));
      item.unit = units_before + from_lane(units_upto - units, at) +
                  ((tile * packs + item.b.pack) * runs + item.b.split) *
                      (item.few ? 1u : kAttnRows / kFewRows);
      item.b.q = sequence_rows(a.sq, item.sequence);
      item.b.lk = from_lane(own.lk, at);
      const int64_t lq = item.b.q.end - item.b.q.begin;
      item.b.q0 = item.few ? 0 : static_cast<int64_t>(tile) * a.tokens;
      item.b.last = item.few || lq - item.b.q0 < a.tokens ? lq : item.b.q0 + a.tokens;
      // (offsets that are not in order can ask for more than there is)
      const uint32_t need = (JOIN ? runs : 1) * (item.few ? 1u : kAttnRows / kFewRows);
      if (tile < 0 || tile >= tiles ||
          (runs > 1 && (item.unit >= a.units || a.units - item.unit < need)))
        item.sequence = -1;
      return item;
    }
    before += from_lane(upto, kWave - 1);
    units_before += from_lane(units_upto, kWave - 1);
  }
  return item;
}

template <int DV>
__device__ inline float* sums_of(const PagedArgs& a, uint32_t unit) {
  return a.partial + static_cast<int64_t>(unit) * (kFewRows * (DV + 2));
}

template <bool BF16, int DQ, int DV>
__global__ void __launch_bounds__(kAttnThreads, 2) paged_attend_kernel(PagedArgs a) {
  constexpr int kVTiles = DV / 32;
  __shared__ alignas(16) uint16_t stage[2 * kAttnKeys * (DQ + DV)];
  const PagedItem item = find_item<false>(a, blockIdx.x);
  if (item.sequence < 0) return;
  const AttnBlock& b = item.b;
  float* const part = b.splits > 1 ? sums_of<DV>(a, item.unit) : nullptr;
  if (item.few) {
    PagedKeys<DQ, DV> keys(a, b, item.sequence, stage);
    attend_few<BF16, DQ, DV>(a, b, keys, stage, part);
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

// The runs of a tile joined, as in attention.hip: a wave takes two rows, a lane a run's
// maxima and sums of them, then columns.
template <bool BF16, int DV>
__global__ void __launch_bounds__(kAttnThreads) paged_join_kernel(PagedArgs a, int parts) {
  constexpr int kCols = DV / 64, kRuns = 4;
  const PagedItem item = find_item<true>(a, blockIdx.x / parts);
  if (item.sequence < 0) return;
  const AttnBlock& b = item.b;
  const int lane = threadIdx.x & (kWave - 1), runs = b.splits;
  const int row0 = (blockIdx.x % parts * kAttnWaves + threadIdx.x / kWave) * kJoinRows;
  const int most = item.few ? kFewRows : kAttnRows, size = most * (DV + 2);
  auto exists = [&](int row) {
    return row < most && b.q0 + (row * a.inv_pack >> 16) < b.last && (row * a.inv_pack >> 16) < a.tokens;
  };
  if (!exists(row0)) return;
  const float* const sums = sums_of<DV>(a, item.unit);
  const float* const tops = sums + (lane < runs ? lane : 0) * size + most * DV;
  float weight[kJoinRows], total[kJoinRows], acc[kJoinRows][kCols] = {};
  int from[kJoinRows];  // rows that do not exist read the first
#pragma unroll
  for (int r = 0; r < kJoinRows; ++r) {
    from[r] = exists(row0 + r) ? row0 + r : row0;
    weight[r] = lane < runs ? tops[from[r]] : -INFINITY;
    total[r] = lane < runs ? tops[most + from[r]] : 0.f;
  }
#pragma unroll
  for (int r = 0; r < kJoinRows; ++r) {
    const float top = over_wave(weight[r], [](float x, float y) { return fmaxf(x, y); });
    weight[r] = weight[r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(weight[r] - top);
    total[r] = over_wave(total[r] * weight[r], [](float x, float y) { return x + y; });
  }
  for (int i0 = 0; i0 < runs; i0 += kRuns) {
    float x[kJoinRows][kRuns][kCols];
#pragma unroll
    for (int r = 0; r < kJoinRows; ++r)
#pragma unroll
      for (int i = 0; i < kRuns; ++i)
#pragma unroll
        for (int c = 0; c < kCols; ++c)
          x[r][i][c] = sums[(i0 + i < runs ? i0 + i : i0) * size + from[r] * DV + kCols * lane + c];
#pragma unroll
    for (int r = 0; r < kJoinRows; ++r)
#pragma unroll
      for (int i = 0; i < kRuns; ++i) {
        const float w = __uint_as_float(
            __builtin_amdgcn_readlane(__float_as_uint(weight[r]), (i0 + i) & (kWave - 1)));
#pragma unroll
        for (int c = 0; c < kCols; ++c)
          acc[r][c] = i0 + i < runs ? fmaf(w, x[r][i][c], acc[r][c]) : acc[r][c];
      }
  }
#pragma unroll
  for (int r = 0; r < kJoinRows; ++r) {
    const int row = row0 + r;
    if (!exists(row)) return;
    const int token = row * a.inv_pack >> 16;
    const float inv = total[r] == 0.f ? 0.f : 1.0f / total[r];
    uint16_t* const out = a.out + ((b.q.begin + b.q0 + token) * a.heads +
                                   static_cast<int64_t>(b.pack) * a.pack + row - token * a.pack) * a.d_v;
    if constexpr (DV == 128) {
      if (2 * lane < a.d_v)
        *reinterpret_cast<uint32_t*>(out + 2 * lane) =
            pack2<BF16>(within_type<BF16>(acc[r][0] * inv), within_type<BF16>(acc[r][1] * inv));
    } else {
      if (lane < a.d_v)
        out[lane] = static_cast<uint16_t>(pack2<BF16>(within_type<BF16>(acc[r][0] * inv), 0.f));
    }
  }
}

// Whether every sequence of a call of so many rows has few.
bool all_few(int64_t rows, int pack) { return rows * pack <= kFewRows; }

int64_t paged_units(int64_t rows, int64_t capacity, int pack) {
  if (capacity <= kMinRun) return 0;  // no tile has more keys than one run
  return int64_t{2} * kFill * (all_few(rows, pack) ? 1 : kAttnRows / kFewRows);
}

template <bool BF16>
int launch_paged(const PagedArgs& a, hipStream_t s) {
  constexpr const char* kName = "lk_attention_paged";
  const int64_t blocks = a.packs * (a.sq.rows / a.tokens + a.sq.count + 1) + (a.partial ? kFill : 0);
  LK_REQUIRE(grid_fits(blocks, kAttnThreads), "too many query rows and heads for one call");
  const int parts = (all_few(a.sq.rows, a.pack) ? kFewRows : kAttnRows) / kJoinBlockRows;
  const dim3 grid(static_cast<unsigned>(blocks)), join(static_cast<unsigned>(kFill * parts));
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
                                     int64_t heads, int64_t kv_heads, int64_t d_qk, int64_t d_v) {
  if (rows < 0 || sequences <= 0 || capacity < 0 || heads <= 0 || kv_heads <= 0 ||
      heads % kv_heads || d_qk <= 0 || d_v <= 0 || d_qk > kAttnMaxQk || d_v > kAttnMaxV)
    return -1;
  const int64_t dv = d_qk <= 64 && d_v <= 64 ? 64 : 128;
  return paged_units(rows, capacity, attention_pack(heads, kv_heads)) * kFewRows * (dv + 2) * 4;
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
  const int pack = attention_pack(heads, kv_heads);
  const int64_t need = lk_attention_paged_workspace(rows, sequences, table_width * page_rows, heads,
                                                    kv_heads, d_qk, d_v);
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
  a.units = static_cast<uint32_t>(paged_units(rows, table_width * page_rows, pack));
  a.partial = need ? static_cast<float*>(workspace) : nullptr;
  a.scale_log2 = scale == 0.f ? 1.f : scale_log2;
  a.q_keep = scale == 0.f ? 0u : 0xFFFFFFFFu, a.q_flip = scale < 0.f ? 0x80008000u : 0u;
  const hipStream_t s = as_stream(stream);
  return dtype == LK_DTYPE_BF16 ? launch_paged<true>(a, s) : launch_paged<false>(a, s);
}

}  // extern "C"
