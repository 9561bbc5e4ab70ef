// Causal softmax attention over packed prompts, for gfx950.

#include "lk_attention.h"
#include "lk_common.hpp"
#include "lk_sequences.hpp"

namespace lk {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

constexpr int kAttnThreads = 256;
constexpr int kAttnWaves = kAttnThreads / kWave;
constexpr int kAttnQueries = 32 * kAttnWaves;  // per block
constexpr int kAttnKeys = 64;                  // per pass of the loop
constexpr int kAttnMaxQk = 192;
constexpr int kAttnMaxV = 128;

struct AttnArgs {
  const uint16_t *q, *k, *v;
  uint16_t* out;
  Sequences sq, sk;
  int heads, group, d_qk, d_v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  int64_t tiles;
  float scale_log2;  // scale * log2(e)
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

template <bool BF16>
__device__ inline uint32_t pack2(float a, float b) {
  if constexpr (BF16) {
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, v2{static_cast<__bf16>(a), static_cast<__bf16>(b)});
  } else {
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, v2{static_cast<_Float16>(a), static_cast<_Float16>(b)});
  }
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

// o += V^T P^T for 16 keys of which a query may not see some, where V holds an
// infinity or a NaN: p = 0 would not silence it, so each key's product is
// taken alone and dropped where the key is not seen. Rare and slow.
template <bool BF16>
__device__ __attribute__((noinline)) f32x16_t mfma_seen(u32x4_t v, u32x4_t p, f32x16_t o, int half,
                                                        int first, int seen) {
  for (int slot = 0; slot < 16; ++slot) {
    const int j = slot & 7, owner = slot >> 3;
    const uint32_t mask = half != owner ? 0u : (j & 1 ? 0xFFFF0000u : 0xFFFFu);
    u32x4_t v1, p1;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      v1[w] = w == j / 2 ? v[w] & mask : 0u;
      p1[w] = w == j / 2 ? p[w] & mask : 0u;
    }
    f32x16_t part;
#pragma unroll
    for (int r = 0; r < 16; ++r) part[r] = 0.f;
    part = mfma32<BF16>(v1, p1, part);
    const int key = first + 8 * (j / 4) + 4 * owner + j % 4;
#pragma unroll
    for (int r = 0; r < 16; ++r) o[r] = key < seen ? o[r] + part[r] : o[r];
  }
  return o;
}

// Block = 128 queries of one head, a wave 32 of them. Scores are computed
// transposed, S^T = K Q^T (32x32 MFMA tiles, keys down, queries across), so a
// lane holds one query's scores in its registers: the softmax needs one
// exchange between the half-waves per 64 keys, the running maximum and sum are
// a scalar per lane, and the score registers, rounded, are the B operand of
// O^T += V^T P^T as they stand.
template <bool BF16, int DQ, int DV>
__global__ void __launch_bounds__(kAttnThreads) attention_kernel(AttnArgs a) {
  constexpr int kQSteps = DQ / 16;
  constexpr int kVTiles = DV / 32;
  constexpr int kKStride = DQ + 8;
  constexpr int kVStride = kAttnKeys + 8;
  __shared__ alignas(16) uint16_t lk_[kAttnKeys * kKStride];
  __shared__ alignas(16) uint16_t lvt[DV * kVStride];
  const int64_t number = blockIdx.x % a.tiles;
  const int h = static_cast<int>(blockIdx.x / a.tiles);
  const SequenceTile at = find_sequence_tile(a.sq, number, kAttnQueries);
  const RowRange rq = sequence_rows(a.sq, at.sequence);
  const int64_t lq = rq.end - rq.begin;
  const int64_t q0 = at.tile * kAttnQueries;
  if (q0 >= lq) return;
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid & (kWave - 1);
  const int n = lane & 31, half = lane >> 5;
  const int64_t qi = q0 + wave * 32 + n;  // the lane's query
  uint16_t* const orow = a.out + ((rq.begin + qi) * a.heads + h) * a.d_v;
  f32x16_t o[kVTiles];
#pragma unroll
  for (int t = 0; t < kVTiles; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[t][r] = 0.f;
  float m = -INFINITY, sum = 0.f;

  if (at.sequence < a.sq.count) {
    const RowRange rk = sequence_rows(a.sk, at.sequence);
    const int64_t lk = rk.end - rk.begin;
    const int64_t ahead = lk - lq;
    // keys seen by the block's last query
    const int64_t last = q0 + kAttnQueries < lq ? q0 + kAttnQueries : lq;
    const int64_t keys = last + ahead < 0 ? 0 : last + ahead;
    const int hk = h / a.group;
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
      }
    }
    for (int64_t k0 = 0; k0 < keys; k0 += kAttnKeys) {
      __syncthreads();
      for (int c = tid; c < kAttnKeys * (DQ / 8); c += kAttnThreads) {
        const int r = c / (DQ / 8), d = c % (DQ / 8) * 8;
        const u32x4_t z = {0u, 0u, 0u, 0u};
        *reinterpret_cast<u32x4_t*>(lk_ + r * kKStride + d) =
            k0 + r < lk && d < a.d_qk
                ? *reinterpret_cast<const u32x4_t*>(kb + (k0 + r) * a.k_row + d)
                : z;
      }
      for (int c = tid; c < kAttnKeys * (DV / 8); c += kAttnThreads) {
        const int r = c / (DV / 8), d = c % (DV / 8) * 8;
        u32x4_t x = {0u, 0u, 0u, 0u};
        if (k0 + r < lk && d < a.d_v)
          x = *reinterpret_cast<const u32x4_t*>(vb + (k0 + r) * a.v_row + d);
#pragma unroll
        for (int j = 0; j < 8; ++j) lvt[(d + j) * kVStride + r] = static_cast<uint16_t>(x[j / 2] >> (16 * (j & 1)));
      }
      __syncthreads();
      f32x16_t s[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[t][r] = 0.f;
#pragma unroll
        for (int i = 0; i < kQSteps; ++i)
          s[t] = mfma32<BF16>(*reinterpret_cast<const u32x4_t*>(lk_ + (32 * t + n) * kKStride +
                                                               16 * i + 8 * half),
                              qf[i], s[t]);
      }
      // a query of the wave does not see all of these keys
      const bool edge = k0 + kAttnKeys - 1 > q0 + wave * 32 + ahead;
      // register r of tile t: key k0 + 32 t + 8 (r / 4) + 4 half + r % 4
      float top = -INFINITY;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int64_t key = k0 + 32 * t + 8 * (r / 4) + 4 * half + r % 4;
          s[t][r] = key > qi + ahead ? -INFINITY : s[t][r] * a.scale_log2;
          top = fmaxf(top, s[t][r]);
        }
      top = fmaxf(top, __shfl_xor(top, 32));
      const float mn = fmaxf(m, top);
      const float base = mn == -INFINITY ? 0.f : mn;
      const float fade = __builtin_amdgcn_exp2f(m - base);
      m = mn;
      float part = 0.f;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[t][r] = __builtin_amdgcn_exp2f(s[t][r] - base);
          part += s[t][r];
        }
      sum = sum * fade + part;
#pragma unroll
      for (int t = 0; t < kVTiles; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[t][r] *= fade;
      // k-slots of MFMA step i: keys 16 i + 4 half + {0..3} and + 8
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = i / 2, r = 8 * (i & 1);
        const u32x4_t p = {pack2<BF16>(s[t][r], s[t][r + 1]), pack2<BF16>(s[t][r + 2], s[t][r + 3]),
                           pack2<BF16>(s[t][r + 4], s[t][r + 5]),
                           pack2<BF16>(s[t][r + 6], s[t][r + 7])};
#pragma unroll
        for (int vt = 0; vt < kVTiles; ++vt) {
          const uint16_t* const vp = lvt + (32 * vt + n) * kVStride + 16 * i + 4 * half;
          const uint2 lo = *reinterpret_cast<const uint2*>(vp);
          const uint2 hi = *reinterpret_cast<const uint2*>(vp + 8);
          const u32x4_t vf = {lo.x, lo.y, hi.x, hi.y};
          if (__builtin_expect(edge && __any(any_nonfinite<BF16>(vf)), 0))
            o[vt] = mfma_seen<BF16>(vf, p, o[vt], half, 16 * i, static_cast<int>(qi + ahead - k0 + 1));
          else
            o[vt] = mfma32<BF16>(vf, p, o[vt]);
        }
      }
    }
    sum += __shfl_xor(sum, 32);
  }
  if (qi >= lq) return;
  const float inv = sum > 0.f ? 1.0f / sum : (sum == 0.f ? 0.f : sum);
#pragma unroll
  for (int t = 0; t < kVTiles; ++t)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int d = 32 * t + 8 * (r / 4) + 4 * half;
      if (d < a.d_v)
        *reinterpret_cast<uint2*>(orow + d) =
            make_uint2(pack2<BF16>(o[t][r] * inv, o[t][r + 1] * inv),
                       pack2<BF16>(o[t][r + 2] * inv, o[t][r + 3] * inv));
    }
}

template <bool BF16>
int launch_attention(const AttnArgs& a, hipStream_t s) {
  const int64_t blocks = a.tiles * a.heads;
  LK_REQUIRE(blocks < (int64_t{1} << 31), "too many query rows and heads for one call");
  const dim3 grid(static_cast<unsigned>(blocks));
#define LK_ATTENTION(Q, V)                                          \
  if (a.d_qk <= Q && a.d_v <= V) {                                  \
    attention_kernel<BF16, Q, V><<<grid, kAttnThreads, 0, s>>>(a);  \
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
  return 0;
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
  LK_REQUIRE(scale == scale && scale - scale == 0.f, "the attention scale must be finite");
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
  const int n = static_cast<int>(sequences);
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
                   q_row_stride, q_head_stride, k_row_stride, k_head_stride, v_row_stride,
                   v_head_stride,
                   sequence_tiles(rows_q, sequences, kAttnQueries),
                   scale * 1.4426950408889634f};
  const hipStream_t s = as_stream(stream);
  return dtype == LK_DTYPE_BF16 ? launch_attention<true>(a, s) : launch_attention<false>(a, s);
}

}  // extern "C"
