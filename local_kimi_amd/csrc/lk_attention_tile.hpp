// Causal attention of a block of query rows over tiles of 64 keys: the part that
// attention.hip (dense keys) and paged_attention.hip (pages) share.
#pragma once

#include "lk_gemm.hpp"
#include "lk_pages.hpp"

namespace lk {

typedef float f32x16_t __attribute__((ext_vector_type(16)));

constexpr int kAttnThreads = 256;
constexpr int kAttnWaves = kAttnThreads / kWave;
constexpr int kAttnRows = 32 * kAttnWaves;  // queries x heads of a block
constexpr int kAttnKeys = 64;                  // per pass of the loop
constexpr int kAttnMaxQk = 192;
constexpr int kAttnMaxV = 128;

struct AttnShape {
  const uint16_t* q;
  uint16_t* out;
  int heads, group, d_qk, d_v;
  // A block's rows: `tokens` queries of `pack` heads that share a key head, row r
  // query r / pack (r inv_pack >> 16), head r % pack. Blocks for a query: `packs`.
  int pack, inv_pack, tokens, packs;
  int64_t q_row, q_head;
  float scale_log2;  // |scale| * log2(e), 1 where scale is 0
  uint32_t q_keep, q_flip;  // bits of q kept (none where scale is 0), flipped (signs, scale < 0)
};

// A block's share: rows q0 to last - 1 of the sequence's queries, run `split` of
// `splits` of the keys that they see.
struct AttnBlock {
  RowRange q;  // rows of the sequence
  int64_t lk;  // its keys
  int64_t ahead;  // query i sees those up to ahead + i (lk - lq, or more: all of them at lk)
  int64_t q0, last;
  int pack, split, splits;
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

// Heads of a block: as many as divide those of a key head, up to 16, so that a
// key is read once for all of them and a few queries fill more of a block's rows
// (one query x 16384 keys, 32 heads on 8: 48 us with a head a block, 24 with four;
// 2 x 2048 queries 92 and 90). Up to 16, 112 of the 128 rows are in use at least.
constexpr int kAttnPack = 16;
inline int attention_pack(int64_t heads, int64_t kv_heads, int most = kAttnPack) {
  int pack = 1;
  for (int p = 2; p <= most; ++p)
    if (heads / kv_heads % p == 0) pack = p;
  return pack;
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

// Rows of K and V that lie a fixed step apart: a tile's chunks by direct loads, this
// lane's at fixed offsets from the tile's first row.
template <int DQ, int DV>
struct DenseKeys {
  static constexpr int kKChunks = DQ / 8, kVChunks = DV / 8;
  static constexpr int kKLoads = kAttnKeys * kKChunks / kAttnThreads;
  static constexpr int kVLoads = kAttnKeys * kVChunks / kAttnThreads;
  const uint16_t *kb, *vb;  // of the sequence's first row, this head's
  int64_t k_row, v_row, lk;
  int d_qk, d_v, wave;
  uint32_t lds;
  uint32_t koff[kKLoads], voff[kVLoads];

  __device__ __forceinline__ DenseKeys(const uint16_t* k, const uint16_t* v, int64_t k_step, int64_t v_step,
                       int64_t rows, const AttnShape& a, const uint16_t* stage)
      : kb(k), vb(v), k_row(k_step), v_row(v_step), lk(rows), d_qk(a.d_qk), d_v(a.d_v) {
    const int lane = threadIdx.x & (kWave - 1);
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    lds = lds_offset(stage);
#pragma unroll
    for (int i = 0; i < kKLoads; ++i) {
      const int slot = (wave * kKLoads + i) * kWave + lane, r = slot / kKChunks;
      const int c = slot % kKChunks ^ key_swizzle<kKChunks>(r);
      koff[i] = 8 * c < d_qk ? static_cast<uint32_t>(r * k_row + 8 * c) * 2u : 0xFFFFFFF0u;
    }
#pragma unroll
    for (int i = 0; i < kVLoads; ++i) {
      const int slot = (wave * kVLoads + i) * kWave + lane, r = slot / kVChunks;
      const int c = slot % kVChunks ^ value_swizzle<kVChunks>(r);
      voff[i] = 8 * c < d_v ? static_cast<uint32_t>(r * v_row + 8 * c) * 2u : 0xFFFFFFF0u;
    }
  }

  __device__ __forceinline__ void fetch(int64_t k0, int buf) {
    // rows behind the sequence's last read as zeros
    const int64_t rows = lk - k0 < kAttnKeys ? lk - k0 : kAttnKeys;
    const u32x4_t rk_ = buffer_rsrc(kb + k0 * k_row, ((rows - 1) * k_row + d_qk) * 2);
    const u32x4_t rv_ = buffer_rsrc(vb + k0 * v_row, ((rows - 1) * v_row + d_v) * 2);
    const uint32_t base = lds + buf * kAttnKeys * (DQ + DV) * 2;
#pragma unroll
    for (int i = 0; i < kKLoads; ++i)
      lds_direct16(rk_, base + (wave * kKLoads + i) * kWave * 16, koff[i], 0);
#pragma unroll
    for (int i = 0; i < kVLoads; ++i)
      lds_direct16(rv_, base + kAttnKeys * DQ * 2 + (wave * kVLoads + i) * kWave * 16, voff[i], 0);
  }

  __device__ __forceinline__ const uint16_t* value_row(int64_t key) const { return vb + key * v_row; }
};

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
// Returns with every wave's reads of `stage` done. o holds the sums of p v (a lane its
// query's, register r of tile t dimension 32 t + 8 (r / 4) + 4 (lane / 32) + r % 4), sum
// those of p, both scaled by 2^-top (o and sum by 2^kLift more in fp16).
template <bool BF16, int DQ, int DV, class Keys>
__device__ __forceinline__ void attend_rows(const AttnShape& a, const AttnBlock& b, Keys& keys_of,
                                   uint16_t* stage, f32x16_t (&o)[DV / 32], float& top, float& sum) {
  constexpr int kQSteps = DQ / 16;
  constexpr int kVTiles = DV / 32;
  constexpr int kKChunks = DQ / 8, kVChunks = DV / 8;
  constexpr int kStage = kAttnKeys * (DQ + DV);  // values of one stage
  // p is stored as 2^kLift times itself: fp16 keeps 2^-24 at the least
  constexpr float kLift = BF16 ? 0.f : 6.f;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int n = lane & 31, half = lane >> 5;
  const int64_t lq = b.q.end - b.q.begin, lk = b.lk, q0 = b.q0, last = b.last;
  const int64_t qw = q0 + (wave * 32 * a.inv_pack >> 16);  // the wave's first query
  const int row = wave * 32 + n, token = row * a.inv_pack >> 16;
  const int64_t qi = q0 + token;  // the lane's, of this head
  const int h = b.pack * a.pack + row - token * a.pack;
  const int64_t ahead = b.ahead;
  // the last key that the lane's query sees, and the wave's first
  const int sees = static_cast<int>(qi + ahead < lk ? qi + ahead : lk - 1);
  const int first_sees = static_cast<int>(qw + ahead < lk ? qw + ahead : lk - 1);
  // keys seen by the block's last query, and by the wave's
  const int64_t most_seen = last + ahead < lk ? last + ahead : lk;
  const int64_t all = most_seen < 0 ? 0 : most_seen;
  // this block's run of them, and the wave's end of it
  const int64_t per = ((all + b.splits - 1) / b.splits + kAttnKeys - 1) / kAttnKeys * kAttnKeys;
  const int64_t from = b.split * per < all ? b.split * per : all;
  const int64_t keys = from + per < all ? from + per : all;
  const int64_t end_wave = q0 + ((wave * 32 + 31) * a.inv_pack >> 16) + 1 + ahead;
  const int64_t keys_wave = end_wave < keys ? end_wave : keys;
  u32x4_t qf[kQSteps];
  {
    const uint16_t* const qp = a.q + (b.q.begin + (qi < lq ? qi : lq - 1)) * a.q_row + h * a.q_head;
#pragma unroll
    for (int i = 0; i < kQSteps; ++i) {
      const int d = 16 * i + 8 * half;
      const u32x4_t z = {0u, 0u, 0u, 0u};
      qf[i] = d < a.d_qk ? *reinterpret_cast<const u32x4_t*>(qp + d) : z;
      qf[i] = (qf[i] & a.q_keep) ^ a.q_flip;
    }
  }
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

  if (from < keys) keys_of.fetch(from, 0);
  wait_vmcnt<0>();
  __syncthreads();
  int buf = 0;
  bool bad = false;  // V has an infinity or a NaN in a tile that not every query sees
  for (int64_t k0 = from; k0 < keys; k0 += kAttnKeys, buf ^= 1) {
    if (k0 + kAttnKeys < keys) keys_of.fetch(k0 + kAttnKeys, buf ^ 1);
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
      const bool edge = k0 + kAttnKeys - 1 > first_sees;  // a query does not see all of them
      if (edge) {
        // keys of this tile that the lane's query sees, from its first register on
        const int left = sees - static_cast<int>(k0);
        const int seen = (left < kAttnKeys ? left + 1 : kAttnKeys) - 4 * half;
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
    int64_t key = first_sees < 0 ? 0 : (first_sees + int64_t{1}) / kAttnKeys * kAttnKeys;
    key = key < from ? from : key;
    int left = a.d_v - 4 * half;
#pragma unroll 1
    for (; key < keys_wave; ++key) {
      const uint16_t* const row = keys_of.value_row(key);
      if (!row) continue;
      asm volatile("" : "+v"(left));  // (64 comparisons kept over the loop would not fit)
#pragma unroll
      for (int t = 0; t < kVTiles; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int d = 32 * t + 8 * (r / 4) + r % 4;
          const float x = d < left && key <= sees ? value_of<BF16>(row[4 * half + d]) : 0.f;
          if (!(fabsf(x) < INFINITY)) o[t][r] += x;
        }
    }
  }
}

// A run's sums as they are, with what they are taken against.
template <int DV>
__device__ __forceinline__ void store_sums(const AttnShape& a, const AttnBlock& b, float* part,
                                  const f32x16_t (&o)[DV / 32], float top, float sum) {
  const int lane = threadIdx.x & (kWave - 1), n = lane & 31, half = lane >> 5;
  const int row = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) * 32 + n;
  if (b.q0 + (row * a.inv_pack >> 16) >= b.last) return;
#pragma unroll
  for (int t = 0; t < DV / 32; ++t)
#pragma unroll
    for (int r = 0; r < 16; r += 4)
      *reinterpret_cast<float4*>(part + row * DV + 32 * t + 8 * (r / 4) + 4 * half) =
          make_float4(o[t][r], o[t][r + 1], o[t][r + 2], o[t][r + 3]);
  if (half == 0) {
    part[kAttnRows * DV + row] = top;
    part[kAttnRows * (DV + 1) + row] = sum;
  }
}

// The rows themselves, whole ones through the wave's share of LDS (every wave has left
// attend_rows).
template <bool BF16, int DQ, int DV>
__device__ __forceinline__ void store_rows(const AttnShape& a, const AttnBlock& b, uint16_t* stage,
                                  const f32x16_t (&o)[DV / 32], float sum) {
  constexpr int kVTiles = DV / 32, kVChunks = DV / 8, kStage = kAttnKeys * (DQ + DV);
  const int lane = threadIdx.x & (kWave - 1), n = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
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
    const int64_t head = b.pack * a.pack + to - q * a.pack;
    if (b.q0 + q < b.last && d < a.d_v)
      *reinterpret_cast<u32x4_t*>(a.out + ((b.q.begin + b.q0 + q) * a.heads + head) * a.d_v + d) =
          *reinterpret_cast<const u32x4_t*>(rows + r * kOutStride + d);
  }
}

}  // namespace lk
