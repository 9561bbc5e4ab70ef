// Causal softmax attention over packed prompts, for gfx950.

#include "lk_attention.h"
#include "lk_gemm.hpp"
#include "lk_pages.hpp"

namespace lk {
namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));

constexpr int kAttnThreads = 256;
constexpr int kAttnWaves = kAttnThreads / kWave;
constexpr int kAttnRows = 32 * kAttnWaves;  // queries x heads of a block
constexpr int kAttnKeys = 64;                  // per pass of the loop
constexpr int kJoinRows = 2;  // of a wave of the join
constexpr int kJoinBlocks = kAttnRows / (kAttnWaves * kJoinRows);
constexpr int kAttnMaxQk = 192;
constexpr int kAttnMaxV = 128;

struct AttnArgs {
  const uint16_t *q, *k, *v;
  uint16_t* out;
  Sequences sq, sk;
  int heads, group, d_qk, d_v;
  // A block's rows: `tokens` queries of `pack` heads that share a key head, row r
  // query r / pack (r inv_pack >> 16), head r % pack. Blocks for a query: `packs`.
  int pack, inv_pack, tokens, packs;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  int64_t tiles;
  int splits;       // runs of each block's keys
  float* partial;   // more than one run: their sums, else null
  float scale_log2;  // |scale| * log2(e), 1 where scale is 0
  uint32_t q_keep, q_flip;  // bits of q kept (none where scale is 0), flipped (signs, scale < 0)
};

template <bool BF16>
__device__ inline f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
  if constexpr (BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// A finite mean of V's values, within the type: p is rounded before its product and
// not in the sum that divides it, so that a mean of 65504 can come out as much as
// 2^-11 above it, where fp16 has infinity from 2^-12 on. (bf16 ends where fp32 does.)
template <bool BF16>
__device__ inline float within_type(float x) {
  if constexpr (BF16) return x;
  else return fabsf(x) < INFINITY ? fminf(fmaxf(x, -65504.f), 65504.f) : x;
}

// Whether any of the eight values is an infinity or a NaN (exponent all ones:
// one more carries into the sign's place).
template <bool BF16>
__device__ inline bool any_nonfinite(u32x4_t x) {
  constexpr uint32_t kExp = BF16 ? 0x7F807F80u : 0x7C007C00u, kOne = BF16 ? 0x00800080u : 0x04000400u;
  uint32_t hit = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) hit |= (x[i] & kExp) + kOne;
  return (hit & 0x80008000u) != 0;
}

// The eight values with those set to zero.
template <bool BF16>
__device__ inline u32x4_t finite_only(u32x4_t x) {
  constexpr uint32_t kExp = BF16 ? 0x7F807F80u : 0x7C007C00u, kOne = BF16 ? 0x00800080u : 0x04000400u;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] &= ~((((x[i] & kExp) + kOne) >> 15 & 0x00010001u) * 0xFFFFu);
  return x;
}

// Staging. A tile of K (V) in LDS is kAttnKeys rows of C 16-byte chunks, filled
// by direct loads (a wave-wide load fills 1 KB in slot order), row r's chunk c
// in slot r C + (c ^ swizzle(r)). A matrix row's chunks are read by 16 or 32 lanes
// with consecutive rows at once, so the swizzle spreads 16 consecutive rows over
// all 16-byte columns of the 64 banks; rows shorter than 256 bytes share one
// pass over the banks with their neighbours, and longer ones than 256 start at
// either half of them, hence the row's upper bits there.
template <int C>
__host__ __device__ constexpr int key_swizzle(int r) {
  return C % 16 == 0 ? r & 15 : (r >> 1) & 7;
}
// V is read down its columns (four rows of 32 bytes by 16 lanes, twice that by a
// half-wave): four consecutive rows go to four quarters of the banks.
template <int C>
__host__ __device__ constexpr int value_swizzle(int r) {
  return C % 16 == 0 ? (r & 3) << 2 : ((r >> 1) & 1) << 2;
}

typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4_t lds_i16x4_t;

// Four rows of 16 columns, by 16 lanes: lane l gives the address of row l / 4,
// columns 4 (l % 4) to + 3, and gets column l of the four rows.
__device__ inline uint2 lds_read_transposed(const uint16_t* p) {
  const i16x4_t v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (lds_i16x4_t*)(const __attribute__((address_space(3))) uint16_t*)(p));
  return __builtin_bit_cast(uint2, v);
}

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

// o_i = sum_j p_ij v_j / sum_j p_ij, p_ij = 2^(s_ij - top_i), in one pass over the
// keys: s in units of log2, top_i the running maximum, what is summed scaled down
// where it moves.
//
// Block = 128 rows (queries x heads of one key head), a wave 32 of them. Scores
// are computed transposed, S^T = K Q^T (32x32 MFMA tiles, keys down, queries
// across), so a lane holds one query's scores in its registers: the softmax needs
// one exchange between the half-waves per 64 keys, the running maximum and sum are
// a scalar per lane, and the score registers, rounded, are the B operand of
// O^T += V^T P^T as they stand. That rounding of p to the inputs' type is the one
// before the output's: the products need it, the sums of p are of the unrounded.
//
// Two stages of 64 keys are up to 80 KB of LDS, so two blocks share a CU and one's
// products run beside the other's softmax. Long prompts are bound by the matrix
// unit and VALU together (53% and 31% of the cycles, at the 1.77 GHz that the card
// runs at meanwhile): 8192 tokens x 32 heads of 192/128 take 690 to 705 us, 975 to 996
// TFLOP/s, where a bf16 8192^3 library product reaches 1139. Short calls are bound by latency.
template <bool BF16, int DQ, int DV>
__global__ void __launch_bounds__(kAttnThreads, 2) attention_kernel(AttnArgs a) {
  constexpr int kQSteps = DQ / 16;
  constexpr int kVTiles = DV / 32;
  constexpr int kKChunks = DQ / 8, kVChunks = DV / 8;
  constexpr int kKLoads = kAttnKeys * kKChunks / kAttnThreads;
  constexpr int kVLoads = kAttnKeys * kVChunks / kAttnThreads;
  constexpr int kStage = kAttnKeys * (DQ + DV);  // values of one stage
  // p is stored as 2^kLift times itself: fp16 keeps 2^-24 at the least
  constexpr float kLift = BF16 ? 0.f : 6.f;
  __shared__ alignas(16) uint16_t stage[2 * kStage];
  const int pack = static_cast<int>(blockIdx.x % a.packs);
  const int64_t item = blockIdx.x / a.packs;
  const int split = static_cast<int>(item % a.splits);
  const AttnTile tile = attention_tile(a, item / a.splits);
  const SequenceTile at = tile.at;
  if (at.sequence < 0) return;
  const RowRange rq = tile.q;
  const int64_t lq = rq.end - rq.begin;
  const int64_t q0 = at.tile * a.tokens;
  if (q0 >= lq) return;
  const int64_t last = q0 + a.tokens < lq ? q0 + a.tokens : lq;  // the block's, exclusive
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int n = lane & 31, half = lane >> 5;
  const int64_t qw = q0 + (wave * 32 * a.inv_pack >> 16);  // the wave's first query
  const int row = wave * 32 + n, token = row * a.inv_pack >> 16;
  const int64_t qi = q0 + token;  // the lane's, of this head
  const int h = pack * a.pack + row - token * a.pack;
  f32x16_t o[kVTiles];
#pragma unroll
  for (int t = 0; t < kVTiles; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[t][r] = 0.f;
  float top = -INFINITY;  // (scaled) maximum that p is taken against
  float sum = 0.f;
  if (at.sequence < a.sq.count) {
    const RowRange rk = tile.k;
    const int64_t lk = rk.end - rk.begin;
    const int64_t ahead = lk - lq;
    // keys seen by the block's last query, and by the wave's
    const int64_t all = last + ahead < 0 ? 0 : last + ahead;
    // this block's run of them, and the wave's end of it
    const int64_t per = ((all + a.splits - 1) / a.splits + kAttnKeys - 1) / kAttnKeys * kAttnKeys;
    const int64_t from = split * per < all ? split * per : all;
    const int64_t keys = from + per < all ? from + per : all;
    const int64_t end_wave = q0 + ((wave * 32 + 31) * a.inv_pack >> 16) + 1 + ahead;
    const int64_t keys_wave = end_wave < keys ? end_wave : keys;
    const int hk = pack * a.pack / a.group;
    const uint16_t* const kb = a.k + rk.begin * a.k_row + hk * a.k_head;
    const uint16_t* const vb = a.v + rk.begin * a.v_row + hk * a.v_head;
    u32x4_t qf[kQSteps];
    {
      const uint16_t* const qp = a.q + (rq.begin + (qi < lq ? qi : lq - 1)) * a.q_row + h * a.q_head;
#pragma unroll
      for (int i = 0; i < kQSteps; ++i) {
        const int d = 16 * i + 8 * half;
        const u32x4_t z = {0u, 0u, 0u, 0u};
        qf[i] = d < a.d_qk ? *reinterpret_cast<const u32x4_t*>(qp + d) : z;
        qf[i] = (qf[i] & a.q_keep) ^ a.q_flip;
      }
    }
    // byte offsets of this lane's chunks from a tile's first row
    uint32_t koff[kKLoads], voff[kVLoads];
#pragma unroll
    for (int i = 0; i < kKLoads; ++i) {
      const int slot = (wave * kKLoads + i) * kWave + lane, r = slot / kKChunks;
      const int c = slot % kKChunks ^ key_swizzle<kKChunks>(r);
      koff[i] = 8 * c < a.d_qk ? static_cast<uint32_t>(r * a.k_row + 8 * c) * 2u : 0xFFFFFFF0u;
    }
#pragma unroll
    for (int i = 0; i < kVLoads; ++i) {
      const int slot = (wave * kVLoads + i) * kWave + lane, r = slot / kVChunks;
      const int c = slot % kVChunks ^ value_swizzle<kVChunks>(r);
      voff[i] = 8 * c < a.d_v ? static_cast<uint32_t>(r * a.v_row + 8 * c) * 2u : 0xFFFFFFF0u;
    }
    const uint32_t lds = lds_offset(stage);
    auto fetch = [&](int64_t k0, int buf) {
      // rows behind the sequence's last read as zeros
      const int64_t rows = lk - k0 < kAttnKeys ? lk - k0 : kAttnKeys;
      const u32x4_t rk_ = buffer_rsrc(kb + k0 * a.k_row, ((rows - 1) * a.k_row + a.d_qk) * 2);
      const u32x4_t rv_ = buffer_rsrc(vb + k0 * a.v_row, ((rows - 1) * a.v_row + a.d_v) * 2);
      const uint32_t base = lds + buf * kStage * 2;
#pragma unroll
      for (int i = 0; i < kKLoads; ++i)
        lds_direct16(rk_, base + (wave * kKLoads + i) * kWave * 16, koff[i], 0);
#pragma unroll
      for (int i = 0; i < kVLoads; ++i)
        lds_direct16(rv_, base + kAttnKeys * DQ * 2 + (wave * kVLoads + i) * kWave * 16, voff[i], 0);
    };
    // where this lane reads, in values from the start of a tile: K row n (and n +
    // 32), chunks 2 i + half (the swizzle takes a chunk's low bits alone, so the
    // reads of later chunks are those of the first at a fixed distance)
    constexpr int kAddrs = kKChunks % 16 == 0 ? 8 : 4;
    int kaddr[kAddrs];
#pragma unroll
    for (int i = 0; i < kAddrs; ++i)
      kaddr[i] = n * DQ + 8 * ((2 * i + half) ^ key_swizzle<kKChunks>(n));
    static_assert(key_swizzle<kKChunks>(32) == 0 && value_swizzle<kVChunks>(8) == 0, "row steps");
    // V rows 4 half + lane % 16 / 4 (and + 8), columns 16 (lane / 16 % 2) + 4 (lane % 4)
    int vaddr[2][kVTiles];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int vt = 0; vt < kVTiles; ++vt) {
        const int row = 8 * x + 4 * half + (lane & 15) / 4;
        const int col = 32 * vt + 16 * (lane / 16 & 1) + 4 * (lane & 3);
        vaddr[x][vt] = row * DV + 8 * ((col / 8) ^ value_swizzle<kVChunks>(row)) + col % 8;
      }

    if (from < keys) fetch(from, 0);
    wait_vmcnt<0>();
    __syncthreads();
    int buf = 0;
    bool bad = false;  // V has an infinity or a NaN in a tile that not every query sees
    for (int64_t k0 = from; k0 < keys; k0 += kAttnKeys, buf ^= 1) {
      if (k0 + kAttnKeys < keys) fetch(k0 + kAttnKeys, buf ^ 1);
      if (k0 < keys_wave && qw < lq) {
        const uint16_t* const lk_ = stage + buf * kStage;
        const uint16_t* const lv = lk_ + kAttnKeys * DQ;
        f32x16_t s[2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[t][r] = 0.f;
        // K two steps ahead of its use: read one pair at a time as the matrix
        // unit wants them, each pair of products waited for LDS
        u32x4_t kf[3][2];
        auto read_k = [&](int i) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
            kf[i % 3][t] = *reinterpret_cast<const u32x4_t*>(
                lk_ + kaddr[i % kAddrs] + 8 * (2 * kAddrs) * (i / kAddrs) + 32 * t * DQ);
        };
        read_k(0);
        read_k(1);
#pragma unroll
        for (int i = 0; i < kQSteps; ++i) {
          if (i + 2 < kQSteps) read_k(i + 2);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int t = 0; t < 2; ++t) s[t] = mfma32<BF16>(kf[i % 3][t], qf[i], s[t]);
        }
        // the first V rows, on their way through the softmax
        u32x4_t vf[2][kVTiles];
        auto read_v = [&](int i) {
#pragma unroll
          for (int vt = 0; vt < kVTiles; ++vt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const uint2 v = lds_read_transposed(lv + vaddr[x][vt] + 16 * i * DV);
              vf[i & 1][vt][2 * x] = v.x;
              vf[i & 1][vt][2 * x + 1] = v.y;
            }
        };
        read_v(0);
        __builtin_amdgcn_sched_barrier(0);
        // register r of tile t: key k0 + 32 t + 8 (r / 4) + 4 half + r % 4. What a
        // query does not see is left out of its maximum and gets p = 0, which
        // an infinity or a NaN in V would turn into one of its own: such values
        // are taken out of the product there and added at the end, for the
        // queries that see them.
        const bool edge = k0 + kAttnKeys - 1 > qw + ahead;  // a query does not see all of them
        if (edge) {
          // keys of this tile that the lane's query sees, from its first register on
          const int seen =
              static_cast<int>(qi + ahead - k0 < kAttnKeys ? qi + ahead - k0 + 1 : kAttnKeys) - 4 * half;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              s[t][r] = 32 * t + 8 * (r / 4) + r % 4 < seen ? s[t][r] : -INFINITY;
        }
        float most = s[0][0];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) most = fmaxf(most, s[t][r]);
        {
          const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(most),
                                                          __float_as_uint(most), false, false);
          most = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])) * a.scale_log2;
        }
        // a query's maximum only moves when it has grown by more than 2^kSlack: p
        // stays below that, and most passes leave the accumulators alone. Each query
        // decides for itself, though the wave branches together: the others' keys
        // may be ones that it does not see.
        constexpr float kSlack = 8.f;
        const bool moves = most > top + kSlack;  // (any at all from -infinity)
        if (__any(moves)) {
          const float next = moves ? most : top;
          const float fade = next == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(top - next);
          top = next;
          sum *= fade;
#pragma unroll
          for (int t = 0; t < kVTiles; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[t][r] *= fade;
        }
        const float base = kLift - (top == -INFINITY ? 0.f : top);
        float part[2] = {0.f, 0.f};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            s[t][r] = __builtin_amdgcn_exp2f(fmaf(s[t][r], a.scale_log2, base));
            part[t] += s[t][r];
          }
        sum += part[0] + part[1];
        // k-slots of MFMA step i: keys 16 i + 4 half + {0..3} and + 8
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int t = i / 2, r = 8 * (i & 1);
          const u32x4_t p = {pack2<BF16>(s[t][r], s[t][r + 1]), pack2<BF16>(s[t][r + 2], s[t][r + 3]),
                             pack2<BF16>(s[t][r + 4], s[t][r + 5]),
                             pack2<BF16>(s[t][r + 6], s[t][r + 7])};
          if (i < 3) read_v(i + 1);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int vt = 0; vt < kVTiles; ++vt) {
            if (edge && __builtin_expect(__any(any_nonfinite<BF16>(vf[i & 1][vt])), 0)) {
              bad = true;
              vf[i & 1][vt] = finite_only<BF16>(vf[i & 1][vt]);
            }
            o[vt] = mfma32<BF16>(vf[i & 1][vt], p, o[vt]);
          }
        }
      }
      wait_vmcnt<0>();  // the next tile has landed
      __syncthreads();
    }
    sum += __shfl_xor(sum, 32);
    if (__builtin_expect(bad, 0)) {
      // the infinities and NaNs left out above, for the queries that see them
      int64_t key = qw + ahead + 1 < 0 ? 0 : (qw + ahead + 1) / kAttnKeys * kAttnKeys;
      key = key < from ? from : key;
#pragma unroll 1
      for (; key < keys_wave; ++key) {
        const uint16_t* const row = vb + key * a.v_row;
#pragma unroll
        for (int t = 0; t < kVTiles; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int d = 32 * t + 8 * (r / 4) + 4 * half + r % 4;
            const float x = d < a.d_v && key <= qi + ahead ? value_of<BF16>(row[d]) : 0.f;
            if (!(fabsf(x) < INFINITY)) o[t][r] += x;
          }
      }
    }
  }
  if (a.partial) {
    // the run's sums as they are, with what they are taken against
    float* const part = a.partial + ((item / a.splits * a.packs + pack) * a.splits + split) *
                                        (kAttnRows * (DV + 2));
    if (qi >= last) return;
#pragma unroll
    for (int t = 0; t < kVTiles; ++t)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *reinterpret_cast<float4*>(part + row * DV + 32 * t + 8 * (r / 4) + 4 * half) =
            make_float4(o[t][r], o[t][r + 1], o[t][r + 2], o[t][r + 3]);
    if (half == 0) {
      part[kAttnRows * DV + row] = top;
      part[kAttnRows * (DV + 1) + row] = sum;
    }
    return;
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  // whole rows through the wave's share of LDS (every wave has left the loop)
  constexpr int kOutStride = DV + 8;
  static_assert(kAttnWaves * 32 * kOutStride <= 2 * kStage, "output tile in LDS");
  uint16_t* const rows = stage + wave * 32 * kOutStride;
#pragma unroll
  for (int t = 0; t < kVTiles; ++t)
#pragma unroll
    for (int r = 0; r < 16; r += 4)
      *reinterpret_cast<uint2*>(rows + n * kOutStride + 32 * t + 8 * (r / 4) + 4 * half) =
          make_uint2(pack2<BF16>(within_type<BF16>(o[t][r] * inv), within_type<BF16>(o[t][r + 1] * inv)),
                     pack2<BF16>(within_type<BF16>(o[t][r + 2] * inv),
                                 within_type<BF16>(o[t][r + 3] * inv)));
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 32 * kVChunks / kWave; ++i) {
    const int slot = i * kWave + lane, r = slot / kVChunks, d = slot % kVChunks * 8;
    const int to = wave * 32 + r, q = to * a.inv_pack >> 16;
    const int64_t head = pack * a.pack + to - q * a.pack;
    if (q0 + q < last && d < a.d_v)
      *reinterpret_cast<u32x4_t*>(a.out + ((rq.begin + q0 + q) * a.heads + head) * a.d_v + d) =
          *reinterpret_cast<const u32x4_t*>(rows + r * kOutStride + d);
  }
}

// A sum (or maximum) over the wave's lanes, in every lane.
template <typename Op>
__device__ inline float over_wave(float v, Op op) {
  v = op(v, dpp_f32<kQuadXor1>(v));
  v = op(v, dpp_f32<kQuadXor2>(v));
  v = op(v, dpp_f32<kRowHalfMirror>(v));
  v = op(v, dpp_f32<kRowMirror>(v));
  auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = op(__uint_as_float(x[0]), __uint_as_float(x[1]));
  x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(x[0]), __uint_as_float(x[1]));
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

// Heads of a block: as many as divide those of a key head, up to 16, so that a
// key is read once for all of them and a few queries fill more of a block's rows
// (one query x 16384 keys, 32 heads on 8: 48 us with a head a block, 24 with four;
// 2 x 2048 queries 92 and 90). Up to 16, 112 of the 128 rows are in use at least.
constexpr int kAttnPack = 16;
int attention_pack(int64_t heads, int64_t kv_heads) {
  int pack = 1;
  for (int p = 2; p <= kAttnPack; ++p)
    if (heads / kv_heads % p == 0) pack = p;
  return pack;
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
  const AttnArgs a{static_cast<const uint16_t*>(q),
                   static_cast<const uint16_t*>(k),
                   static_cast<const uint16_t*>(v),
                   static_cast<uint16_t*>(out),
                   Sequences{cu_q, rows_q, rows_q / sequences, n},
                   Sequences{cu_k, rows_k, rows_k / sequences, n},
                   static_cast<int>(heads),
                   static_cast<int>(heads / kv_heads),
                   static_cast<int>(d_qk),
                   static_cast<int>(d_v),
                   pack,
                   65536 / pack + 1,
                   kAttnRows / pack,
                   static_cast<int>(heads) / pack,
                   q_row_stride, q_head_stride, k_row_stride, k_head_stride, v_row_stride,
                   v_head_stride,
                   sequence_tiles(rows_q, sequences, kAttnRows / pack),
                   attention_splits(rows_q, rows_k, sequences, heads, pack),
                   need ? static_cast<float*>(workspace) : nullptr,
                   scale == 0.f ? 1.f : scale_log2,
                   scale == 0.f ? 0u : 0xFFFFFFFFu,
                   scale < 0.f ? 0x80008000u : 0u};
  const hipStream_t s = as_stream(stream);
  return dtype == LK_DTYPE_BF16 ? launch_attention<true>(a, s) : launch_attention<false>(a, s);
}

}  // extern "C"
