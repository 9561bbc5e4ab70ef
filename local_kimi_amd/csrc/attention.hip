// Causal softmax attention over packed prompts, for gfx950.

#include "lk_attention.h"
#include "lk_attention_tile.hpp"

namespace lk {
namespace {

constexpr int kJoinRows = 2;  // of a wave of the join
constexpr int kJoinBlocks = kAttnRows / (kAttnWaves * kJoinRows);

struct AttnArgs : AttnShape {
  const uint16_t *k, *v;
  Sequences sq, sk;
  int64_t k_row, k_head, v_row, v_head;
  int64_t tiles;
  int splits;       // runs of each block's keys
  float* partial;   // more than one run: their sums, else null
};

// A tile of queries, and the rows of its sequence.
struct AttnTile {
  SequenceTile at;
  RowRange q, k;
};

// From the last one back: a sequence's later tiles see more keys, and are begun first.
__device__ inline AttnTile attention_tile(const AttnArgs& a, int64_t rank) {
  AttnTile t;
  t.at = find_sequence_tile(a.sq, a.tiles - 1 - rank, a.tokens);
  const int from = t.at.sequence < 0 ? 0 : t.at.sequence;
  t.q = sequence_rows(a.sq, from);
  t.k = sequence_rows(a.sk, from);
  return t;
}

// A block's rows against its sequence's keys (attend_rows), to the output or, in runs,
// to the workspace.
//
// Two stages of 64 keys are up to 80 KB of LDS, so two blocks share a CU and one's
// products run beside the other's softmax. Long prompts are bound by the matrix
// unit and VALU together (53% and 31% of the cycles, at the 1.77 GHz that the card
// runs at meanwhile): 8192 tokens x 32 heads of 192/128 take 690 to 705 us, 975 to 996
// TFLOP/s, where a bf16 8192^3 library product reaches 1139. Short calls are bound by latency.
template <bool BF16, int DQ, int DV>
__global__ void __launch_bounds__(kAttnThreads, 2) attention_kernel(AttnArgs a) {
  constexpr int kVTiles = DV / 32;
  __shared__ alignas(16) uint16_t stage[2 * kAttnKeys * (DQ + DV)];
  const int pack = static_cast<int>(blockIdx.x % a.packs);
  const int64_t item = blockIdx.x / a.packs;
  const int split = static_cast<int>(item % a.splits);
  const AttnTile tile = attention_tile(a, item / a.splits);
  const SequenceTile at = tile.at;
  if (at.sequence < 0) return;
  const int64_t lq = tile.q.end - tile.q.begin;
  const int64_t q0 = at.tile * a.tokens;
  if (q0 >= lq) return;
  const int64_t last = q0 + a.tokens < lq ? q0 + a.tokens : lq;  // the block's, exclusive
  const int64_t lk = tile.k.end - tile.k.begin;
  const AttnBlock b{tile.q, lk, lk - (tile.q.end - tile.q.begin), q0, last, pack, split, a.splits};
  f32x16_t o[kVTiles];
#pragma unroll
  for (int t = 0; t < kVTiles; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[t][r] = 0.f;
  float top = -INFINITY;  // (scaled) maximum that p is taken against
  float sum = 0.f;
  if (at.sequence < a.sq.count) {
    const int hk = pack * a.pack / a.group;
    DenseKeys<DQ, DV> keys(a.k + tile.k.begin * a.k_row + hk * a.k_head,
                           a.v + tile.k.begin * a.v_row + hk * a.v_head, a.k_row, a.v_row, b.lk, a,
                           stage);
    attend_rows<BF16, DQ, DV>(a, b, keys, stage, o, top, sum);
  }
  if (a.partial) {
    store_sums<DV>(a, b, a.partial + ((item / a.splits * a.packs + pack) * a.splits + split) *
                                         (kAttnRows * (DV + 2)), o, top, sum);
    return;
  }
  store_rows<BF16, DQ, DV>(a, b, stage, o, sum);
}

// The runs of a block's keys joined: a wave takes kJoinRows rows, a lane a run's
// maxima and sums of them, then columns. Weights 2^(top - largest top) in fp32, the
// runs in order. Bound by latency, a chain of five loads: with one row a wave there
// were more rounds of them (777 queries x 32 heads in two runs: 151 us with the runs
// themselves, 146 with two rows or four), with four a single query waited for
// rows that it does not have (1 x 16384 keys: 24 us, 26 with four).
template <bool BF16, int DV>
__global__ void __launch_bounds__(kAttnThreads) attention_join_kernel(AttnArgs a) {
  const int64_t block = blockIdx.x / kJoinBlocks;
  const AttnTile tile = attention_tile(a, block / a.packs);
  if (tile.at.sequence < 0) return;
  constexpr int kRun = kAttnRows * (DV + 2), kCols = DV / 64, kRuns = 4;
  const int lane = threadIdx.x & (kWave - 1);
  const int row0 = (blockIdx.x % kJoinBlocks * kAttnWaves + threadIdx.x / kWave) * kJoinRows;
  const int64_t q0 = tile.q.begin + tile.at.tile * a.tokens;
  const int64_t head0 = block % a.packs * a.pack;
  auto exists = [&](int row) {
    const int token = row * a.inv_pack >> 16;
    return token < a.tokens && q0 + token < tile.q.end;
  };
  if (!exists(row0)) return;
  const float* const parts = a.partial + block * a.splits * kRun;
  const float* const tops = parts + (lane < a.splits ? lane : 0) * kRun + kAttnRows * DV;
  float weight[kJoinRows], total[kJoinRows], acc[kJoinRows][kCols] = {};
  int from[kJoinRows];  // rows that do not exist read the first
#pragma unroll
  for (int r = 0; r < kJoinRows; ++r) {
    from[r] = exists(row0 + r) ? row0 + r : row0;
    weight[r] = lane < a.splits ? tops[from[r]] : -INFINITY;
    total[r] = lane < a.splits ? tops[kAttnRows + from[r]] : 0.f;
  }
#pragma unroll
  for (int r = 0; r < kJoinRows; ++r) {
    const float top = over_wave(weight[r], [](float x, float y) { return fmaxf(x, y); });
    weight[r] = weight[r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(weight[r] - top);
    total[r] = over_wave(total[r] * weight[r], [](float x, float y) { return x + y; });
  }
  for (int i0 = 0; i0 < a.splits; i0 += kRuns) {
    float x[kJoinRows][kRuns][kCols];
#pragma unroll
    for (int r = 0; r < kJoinRows; ++r)
#pragma unroll
      for (int i = 0; i < kRuns; ++i)
#pragma unroll
        for (int c = 0; c < kCols; ++c)
          x[r][i][c] = parts[(i0 + i < a.splits ? i0 + i : i0) * kRun + from[r] * DV + kCols * lane + c];
#pragma unroll
    for (int r = 0; r < kJoinRows; ++r)
#pragma unroll
      for (int i = 0; i < kRuns; ++i) {
        const float w = __uint_as_float(
            __builtin_amdgcn_readlane(__float_as_uint(weight[r]), (i0 + i) & (kWave - 1)));
#pragma unroll
        for (int c = 0; c < kCols; ++c)
          acc[r][c] = i0 + i < a.splits ? fmaf(w, x[r][i][c], acc[r][c]) : acc[r][c];
      }
  }
#pragma unroll
  for (int r = 0; r < kJoinRows; ++r) {
    if (!exists(row0 + r)) return;
    const int token = (row0 + r) * a.inv_pack >> 16;
    const float inv = total[r] == 0.f ? 0.f : 1.0f / total[r];
    uint16_t* const out =
        a.out + ((q0 + token) * a.heads + head0 + row0 + r - token * a.pack) * a.d_v;
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

// Runs of each block's keys. A block alone on a CU leaves its matrix unit idle
// through every softmax, and a call with fewer blocks than CUs leaves CUs idle: where
// there are fewer than two blocks a CU, long key ranges are taken in runs, until
// there are, of kAttnRun keys at least in the mean (the runs' sums are written and read
// again). Counts are estimates from the call's sizes: the lengths are on the device. A
// sequence far longer than the mean is in fewer runs than it could be, a shorter one in
// shorter runs: 64 queries x 8 heads, one on 16384 keys and 63 on 16, take 337 us, the
// one alone 25.
// With one run / by this rule, bf16 heads of 128: one query x 16384 keys x 8 heads
// 329 / 21 us, 512 x 4096 x 32 93 / 58, 4096 x 4096 x 4 91 / 44, 16 x 800 x 32 23 / 18.
// 1024 queries x 1024 keys x 32 took 30 in one and 40 in two runs (of 256 keys).
constexpr int kAttnFill = 512;
constexpr int kAttnRun = 384;
int attention_splits(int64_t rows_q, int64_t rows_k, int64_t sequences, int64_t heads, int pack) {
  const int64_t blocks = (rows_q / (kAttnRows / pack) + sequences) * (heads / pack);
  const int64_t want = (kAttnFill + blocks - 1) / blocks;
  const int64_t seen = (rows_k - rows_q / 2) / sequences;  // keys of a query, about
  const int64_t n = want < seen / kAttnRun ? want : seen / kAttnRun;
  return n < 1 ? 1 : (n > kWave ? kWave : static_cast<int>(n));  // the join has a lane for each
}

template <bool BF16>
int launch_attention(const AttnArgs& a, hipStream_t s) {
  const int64_t items = a.tiles * a.packs, blocks = items * a.splits;
  LK_REQUIRE(grid_fits(blocks, kAttnThreads) &&
                 (!a.partial || grid_fits(items * kJoinBlocks, kAttnThreads)),
             "too many query rows and heads for one call");
  const dim3 grid(static_cast<unsigned>(blocks)), join(static_cast<unsigned>(items * kJoinBlocks));
#define LK_ATTENTION(Q, V)                                          \
  if (a.d_qk <= Q && a.d_v <= V) {                                  \
    attention_kernel<BF16, Q, V><<<grid, kAttnThreads, 0, s>>>(a);  \
    if (a.partial) {                                                \
      if (const int st = check_launch("lk_attention_prefill")) return st; \
      attention_join_kernel<BF16, V><<<join, kAttnThreads, 0, s>>>(a); \
    }                                                               \
    return check_launch("lk_attention_prefill");                    \
  }
  LK_ATTENTION(64, 64)
  LK_ATTENTION(128, 128)
  LK_ATTENTION(192, 128)
#undef LK_ATTENTION
  return fail_arg("attention head dimensions too large");
}

}  // namespace
}  // namespace lk

using namespace lk;

extern "C" {

int64_t lk_attention_prefill_workspace(int64_t rows_q, int64_t rows_k, int64_t sequences,
                                       int64_t heads, int64_t kv_heads, int64_t d_qk,
                                       int64_t d_v) {
  if (rows_q < 0 || rows_k < 0 || sequences <= 0 || heads <= 0 || kv_heads <= 0 ||
      heads % kv_heads || d_qk <= 0 || d_v <= 0 || d_qk > kAttnMaxQk || d_v > kAttnMaxV)
    return -1;
  const int pack = attention_pack(heads, kv_heads);
  const int64_t splits = attention_splits(rows_q, rows_k, sequences, heads, pack);
  if (splits == 1) return 0;
  const int64_t dv = d_qk <= 64 && d_v <= 64 ? 64 : 128;
  const int64_t tiles = sequence_tiles(rows_q, sequences, kAttnRows / pack);
  return tiles * (heads / pack) * splits * kAttnRows * (dv + 2) * 4;
}

int lk_attention_prefill(const void* q, const void* k, const void* v, void* out,
                         const int32_t* cu_q, const int32_t* cu_k, int64_t sequences,
                         int64_t rows_q, int64_t rows_k, int64_t heads, int64_t kv_heads,
                         int64_t d_qk, int64_t d_v, int64_t q_row_stride, int64_t q_head_stride,
                         int64_t k_row_stride, int64_t k_head_stride, int64_t v_row_stride,
                         int64_t v_head_stride, float scale, int dtype, void* workspace,
                         int64_t workspace_bytes, void* stream) {
  LK_REQUIRE(sequences > 0 && rows_q >= 0 && rows_k >= 0, "attention needs sequences, and rows >= 0");
  LK_REQUIRE(rows_q < (int64_t{1} << 31) && rows_k < (int64_t{1} << 31) &&
                 sequences < (int64_t{1} << 24),
             "too many rows or sequences");
  LK_REQUIRE((cu_q || rows_q % sequences == 0) && (cu_k || rows_k % sequences == 0),
             "without offsets the rows must divide into equal sequences");
  LK_REQUIRE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && heads <= 65535,
             "attention heads must be a positive multiple of the key heads");
  LK_REQUIRE(d_qk > 0 && d_qk % 8 == 0 && d_qk <= kAttnMaxQk,
             "attention d_qk must be a multiple of 8 up to %d, got %lld", kAttnMaxQk,
             (long long)d_qk);
  LK_REQUIRE(d_v > 0 && d_v % 8 == 0 && d_v <= kAttnMaxV,
             "attention d_v must be a multiple of 8 up to %d, got %lld", kAttnMaxV, (long long)d_v);
  LK_REQUIRE(dtype == LK_DTYPE_F16 || dtype == LK_DTYPE_BF16,
             "attention tensors must be fp16 or bf16");
  LK_REQUIRE(q_row_stride % 8 == 0 && q_head_stride % 8 == 0 && k_row_stride % 8 == 0 &&
                 k_head_stride % 8 == 0 && v_row_stride % 8 == 0 && v_head_stride % 8 == 0,
             "attention strides must be multiples of 8 elements");
  LK_REQUIRE(q_row_stride >= 0 && q_head_stride >= 0 && k_row_stride >= 0 && k_head_stride >= 0 &&
                 v_row_stride >= 0 && v_head_stride >= 0,
             "attention strides must not be negative");
  LK_REQUIRE(k_row_stride < (int64_t{1} << 24) && v_row_stride < (int64_t{1} << 24),
             "attention row strides must be below 2^24 elements");
  const float scale_log2 = fabsf(scale) * 1.4426950408889634f;
  LK_REQUIRE(scale_log2 < INFINITY, "the attention scale must be finite, below 2^127");
  if (rows_q == 0) return LK_OK;
  LK_REQUIRE(q && out && (rows_k == 0 || (k && v)), "null pointer argument");
  for (const void* p : {q, k, v, static_cast<const void*>(out)})
    LK_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0,
               "attention tensors must start on a 16-byte boundary");
  const int64_t need =
      lk_attention_prefill_workspace(rows_q, rows_k, sequences, heads, kv_heads, d_qk, d_v);
  LK_REQUIRE(need == 0 || (workspace && workspace_bytes >= need),
             "attention workspace too small: %lld bytes, %lld needed", (long long)workspace_bytes,
             (long long)need);
  LK_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
             "attention workspace must be 16-byte aligned");
  const int n = static_cast<int>(sequences), pack = attention_pack(heads, kv_heads);
  AttnArgs a{};
  a.q = static_cast<const uint16_t*>(q), a.out = static_cast<uint16_t*>(out);
  a.k = static_cast<const uint16_t*>(k), a.v = static_cast<const uint16_t*>(v);
  a.sq = Sequences{cu_q, rows_q, rows_q / sequences, n};
  a.sk = Sequences{cu_k, rows_k, rows_k / sequences, n};
  a.heads = static_cast<int>(heads), a.group = static_cast<int>(heads / kv_heads);
  a.d_qk = static_cast<int>(d_qk), a.d_v = static_cast<int>(d_v);
  a.pack = pack, a.inv_pack = 65536 / pack + 1, a.tokens = kAttnRows / pack;
  a.packs = static_cast<int>(heads) / pack;
  a.q_row = q_row_stride, a.q_head = q_head_stride, a.k_row = k_row_stride;
  a.k_head = k_head_stride, a.v_row = v_row_stride, a.v_head = v_head_stride;
  a.tiles = sequence_tiles(rows_q, sequences, a.tokens);
  a.splits = attention_splits(rows_q, rows_k, sequences, heads, pack);
  a.partial = need ? static_cast<float*>(workspace) : nullptr;
  a.scale_log2 = scale == 0.f ? 1.f : scale_log2;
  a.q_keep = scale == 0.f ? 0u : 0xFFFFFFFFu, a.q_flip = scale < 0.f ? 0x80008000u : 0u;
  const hipStream_t s = as_stream(stream);
  return dtype == LK_DTYPE_BF16 ? launch_attention<true>(a, s) : launch_attention<false>(a, s);
}

}  // extern "C"
