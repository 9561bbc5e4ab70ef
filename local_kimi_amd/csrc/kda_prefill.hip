// Kimi Delta Attention over whole prompts, for gfx950: the width-4 short
// convolutions and the recurrence, each over packed sequences with the state
// carried in and out. The single-token forms are in kda.hip.

#include "lk_common.hpp"
#include "lk_kda.h"
#include "lk_sequences.hpp"

namespace lk {
namespace {

// ---------------------------------------------------------------------------
// storage types

template <int DT>
struct Storage {
  using type = uint16_t;
};
template <>
struct Storage<LK_DTYPE_F32> {
  using type = float;
};

template <int DT>
__device__ inline float to_f32(typename Storage<DT>::type v) {
  if constexpr (DT == LK_DTYPE_F32) return v;
  else if constexpr (DT == LK_DTYPE_BF16) return bf16_to_f32(v);
  else return static_cast<float>(__builtin_bit_cast(_Float16, v));
}

template <int DT>
__device__ inline typename Storage<DT>::type from_f32(float v) {
  if constexpr (DT == LK_DTYPE_F32) return v;
  else if constexpr (DT == LK_DTYPE_BF16) return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v));
  else return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
}

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

// ---------------------------------------------------------------------------
// Short convolutions. y_t = silu(w0 x_{t-3} + w1 x_{t-2} + w2 x_{t-1} + w3 x_t)
// per channel, with x before a sequence's first token from its state; the
// state becomes the last four of (state, tokens).
//
// Bound by HBM: 12 operations on a value that is read and written once (16384
// tokens x 3 x 2304 fp16: 89 us, 5.1 TB/s, as fast as a large copy). A
// thread owns N neighbouring channels (16 bytes) of one convolution and walks
// a tile of kConvTile tokens with the three earlier inputs in registers,
// kConvRows rows' loads in flight; the tile's first three inputs are read again (3
// rows in kConvTile, mostly from a cache). Where rows do not start on 16 bytes, N
// is one: 4096 tokens x 3 x 4095 bf16 48 us, 4096 channels 38, eight times the loads
// and stores of a 16th each, which the caches join. Threads are dealt over the three
// convolutions' channels as one row, so that only a call's last block has idle
// ones. The thread with a sequence's first tile has read the state's values, so
// it is the one that replaces them: the state may be updated in place.
constexpr int kConvThreads = 128;
constexpr int kConvTile = 16;  // 4096 tokens x 3 x 4096 bf16: 40 us at 16, 42 at 32, 46 at 64
constexpr int kConvRows = 8;

struct ConvArgs {
  const void* in[3];
  const void* state[3];
  void* state_out[3];
  const void* weight[3];
  void* out[3];
  Sequences seq;
  int64_t channels;
  int64_t stride;  // elements from an input row to the next
  int column_blocks;
};

template <typename T>
__device__ inline T pick(const T (&v)[3], int i) {
  return i == 0 ? v[0] : (i == 1 ? v[1] : v[2]);
}

template <int DT, int WDT, int N>
__global__ void __launch_bounds__(kConvThreads) conv_prefill_kernel(ConvArgs a) {
  using T = typename Storage<DT>::type;
  using W = typename Storage<WDT>::type;
  using P = Pack<T, N>;
  const int64_t number = blockIdx.x / a.column_blocks;
  const int64_t item = static_cast<int64_t>(blockIdx.x % a.column_blocks) * kConvThreads + threadIdx.x;
  const int64_t chunks = a.channels / N;
  const int conv = item < chunks ? 0 : (item < 2 * chunks ? 1 : 2);
  const int64_t c = (item - conv * chunks) * N;
  const SequenceTile at = find_sequence_tile(a.seq, number, kConvTile);
  if (c >= a.channels || at.sequence < 0) return;
  const RowRange rows = sequence_rows(a.seq, at.sequence);
  const int64_t length = rows.end - rows.begin;
  const int64_t t0 = at.tile * kConvTile;
  const T* const x = static_cast<const T*>(pick(a.in, conv)) + rows.begin * a.stride + c;
  T* const y = static_cast<T*>(pick(a.out, conv)) + rows.begin * a.channels + c;
  const int64_t t1 = t0 + kConvTile < length ? t0 + kConvTile : length;
  if (at.sequence == a.seq.count) {  // behind the last sequence
    P zero;
#pragma unroll
    for (int j = 0; j < N; ++j) zero.v[j] = 0;
    for (int64_t t = t0; t < t1; ++t) *reinterpret_cast<P*>(y + t * a.channels) = zero;
    return;
  }
  if (t0 >= length && at.tile > 0) return;

  // every load of the tile's start first
  P row[kConvRows];
  auto fetch = [&](int64_t t) {
#pragma unroll
    for (int r = 0; r < kConvRows; ++r) {
      const int64_t tr = t + r < t1 ? t + r : t1 - 1;
      row[r] = *reinterpret_cast<const P*>(x + tr * a.stride);
    }
  };
  Pack<W, 4> taps[N];
#pragma unroll
  for (int j = 0; j < N; ++j)
    taps[j] = reinterpret_cast<const Pack<W, 4>*>(pick(a.weight, conv))[c + j];
  if (t0 < t1) fetch(t0);
  float x1[N], x2[N], x3[N];  // the inputs 3, 2 and 1 tokens back
  if (at.tile == 0) {
    const int64_t sc = static_cast<int64_t>(at.sequence) * a.channels + c;
    const auto* const s = static_cast<const Pack<T, 4>*>(pick(a.state, conv)) + sc;
    auto* const so = static_cast<Pack<T, 4>*>(pick(a.state_out, conv)) + sc;
    // entry i of the next state: token length - 4 + i, or entry length + i of
    // this one where that lies before the first token
    P last[4];
    if (length > 0)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        last[i] = *reinterpret_cast<const P*>(x + (length - 4 + i > 0 ? length - 4 + i : 0) * a.stride);
    Pack<T, 4> old[N];
#pragma unroll
    for (int j = 0; j < N; ++j) old[j] = s[j];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      x1[j] = to_f32<DT>(old[j].v[1]);
      x2[j] = to_f32<DT>(old[j].v[2]);
      x3[j] = to_f32<DT>(old[j].v[3]);
      Pack<T, 4> next;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t t = length - 4 + i;
        next.v[i] = t >= 0 ? last[i].v[j]
                           : (t == -4 ? old[j].v[0]
                                      : (t == -3 ? old[j].v[1] : (t == -2 ? old[j].v[2] : old[j].v[3])));
      }
      so[j] = next;
    }
  } else {
    const P a1 = *reinterpret_cast<const P*>(x + (t0 - 3) * a.stride);
    const P a2 = *reinterpret_cast<const P*>(x + (t0 - 2) * a.stride);
    const P a3 = *reinterpret_cast<const P*>(x + (t0 - 1) * a.stride);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      x1[j] = to_f32<DT>(a1.v[j]);
      x2[j] = to_f32<DT>(a2.v[j]);
      x3[j] = to_f32<DT>(a3.v[j]);
    }
  }
  float w[4][N];
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i][j] = to_f32<WDT>(taps[j].v[i]);

  for (int64_t t = t0; t < t1; t += kConvRows) {
    P res[kConvRows];
#pragma unroll
    for (int r = 0; r < kConvRows; ++r) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float now = to_f32<DT>(row[r].v[j]);
        const float acc =
            fmaf(now, w[3][j], fmaf(x3[j], w[2][j], fmaf(x2[j], w[1][j], x1[j] * w[0][j])));
        res[r].v[j] = from_f32<DT>(silu_fast_f32(acc));
        x1[j] = x2[j];
        x2[j] = x3[j];
        x3[j] = now;
      }
    }
    if (t + kConvRows < t1) fetch(t + kConvRows);
#pragma unroll
    for (int r = 0; r < kConvRows; ++r)
      if (t + r < t1) *reinterpret_cast<P*>(y + (t + r) * a.channels) = res[r];
  }
}

// ---------------------------------------------------------------------------
// The recurrence, a step at a time. Per head, with S [d_k, d_v]:
//   S' = e^g S (per key row);  u = v - S'^T k;  S = S' + beta k u^T;
//   o = scale S^T q = scale (S'^T q + beta (k . q) u),
// so one pass over S' gives both sums and a step has one reduction.
//
// A wave holds 4 columns of S: lane l has key rows [RPL * (l % 16), + RPL) of
// column l / 16, sums over the 16 lanes of a DPP row. A block of four waves
// takes 16 columns and stages kSerialTokens steps of q, k, e^g and k . q in
// LDS (one lane of the staging per 16th of a row, as the steps use them) while
// the batch before it runs. Bound by the chain from step to step, in which a wave
// has nothing else to do: six LDS reads, RPL products after one another for each of
// the two sums, four DPP additions, RPL more products. 32 heads take 0.28 us a step at
// d_k = 64, 0.35 at 128 (256 steps 90 us), 0.67 to 0.70 at 256 (256 steps 179 us, 1024
// steps 680).
constexpr int kSerialThreads = 256;
constexpr int kSerialCols = 16;
constexpr int kSerialTokens = 16;

struct ScanArgs {
  const float* state;
  float* state_out;
  const float* q;
  const float* k;
  const void* v;
  const float* decay;
  const float* beta;
  void* out;
  Sequences seq;
  int heads, d_k, d_v;
  float scale;
};

__device__ inline float row16_sum(float v) {
  v += dpp_f32<kQuadXor1>(v);
  v += dpp_f32<kQuadXor2>(v);
  v += dpp_f32<kRowHalfMirror>(v);
  v += dpp_f32<kRowMirror>(v);
  return v;
}

// p[first .. first + RPL) of a row of d_k values, zeros behind it and where the
// row is not ok (p is a row that can be read all the same). No branch: loads under
// one wait for each other.
template <int RPL>
__device__ inline void load_rows(const float* p, int first, int d_k, bool ok, float (&r)[RPL]) {
  if ((d_k & 3) == 0) {
    float4 x[RPL / 4];
#pragma unroll
    for (int i = 0; i < RPL; i += 4)
      x[i / 4] = *reinterpret_cast<const float4*>(p + (first + i < d_k ? first + i : 0));
#pragma unroll
    for (int i = 0; i < RPL; i += 4) {
      const bool in = ok && first + i < d_k;
      r[i] = in ? x[i / 4].x : 0.f;
      r[i + 1] = in ? x[i / 4].y : 0.f;
      r[i + 2] = in ? x[i / 4].z : 0.f;
      r[i + 3] = in ? x[i / 4].w : 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < RPL; ++i) r[i] = p[first + i < d_k ? first + i : 0];
#pragma unroll
    for (int i = 0; i < RPL; ++i) r[i] = ok && first + i < d_k ? r[i] : 0.f;
  }
}

template <int DT, int RPL>
__global__ void __launch_bounds__(kSerialThreads) scan_serial_kernel(ScanArgs a, int col_blocks) {
  using T = typename Storage<DT>::type;
  constexpr int kRow = RPL * 16;
  __shared__ float4 lq[kSerialTokens][kRow / 4], lk_[kSerialTokens][kRow / 4],
      lg[kSerialTokens][kRow / 4];
  __shared__ float lv[kSerialTokens][kSerialCols], lo[kSerialTokens][kSerialCols];
  __shared__ float lbeta[kSerialTokens], lkq[kSerialTokens];
  const int cb = blockIdx.x % col_blocks;
  const int64_t sh = blockIdx.x / col_blocks;
  const int h = static_cast<int>(sh % a.heads);
  const int s = static_cast<int>(sh / a.heads);
  const RowRange rows = sequence_rows(a.seq, s);
  const int tid = threadIdx.x, l = tid & 15;
  const int col = tid >> 4;  // of the block: wave * 4 + lane / 16; in staging: the token
  const int c = cb * kSerialCols + col;
  if (s == a.seq.count) {  // rows behind the last sequence
    for (int64_t t = rows.begin + col; t < rows.end; t += 16)
      if (cb * kSerialCols + l < a.d_v)
        static_cast<T*>(a.out)[(t * a.heads + h) * a.d_v + cb * kSerialCols + l] = 0;
    return;
  }
  float st[RPL];
  const int64_t sbase = sh * a.d_k * a.d_v;
#pragma unroll
  for (int i = 0; i < RPL; ++i) {
    const int r = l * RPL + i;
    st[i] = r < a.d_k && c < a.d_v ? a.state[sbase + static_cast<int64_t>(r) * a.d_v + c] : 0.f;
  }

  float fq[RPL], fk[RPL], fg[RPL], fv = 0.f, fb = 0.f;
  auto fetch = [&](int64_t t0) {  // thread: rows of lane l of token t0 + col
    const int64_t t = t0 + col;
    const bool ok = t < rows.end;
    const int64_t at = ((ok ? t : rows.begin) * a.heads + h) * a.d_k;
    load_rows<RPL>(a.q + at, l * RPL, a.d_k, ok, fq);
    load_rows<RPL>(a.k + at, l * RPL, a.d_k, ok, fk);
    load_rows<RPL>(a.decay + at, l * RPL, a.d_k, ok, fg);
    const int vc = cb * kSerialCols + l;
    const int64_t th = (ok ? t : rows.begin) * a.heads + h;
    fv = to_f32<DT>(static_cast<const T*>(a.v)[th * a.d_v + (vc < a.d_v ? vc : 0)]);
    fb = a.beta[th];
    fv = ok && vc < a.d_v ? fv : 0.f;
    fb = ok ? fb : 0.f;
  };
  if (rows.begin < rows.end) fetch(rows.begin);
  for (int64_t t0 = rows.begin; t0 < rows.end; t0 += kSerialTokens) {
    float kq = 0.f;
#pragma unroll
    for (int i = 0; i < RPL; ++i) kq = fmaf(fk[i], fq[i], kq);
    kq = row16_sum(kq);
    __syncthreads();  // the batch before has been used
#pragma unroll
    for (int i = 0; i < RPL; i += 4) {
      const int at = (i / 4) * 16 + l;  // 16 lanes of 16 bytes side by side
      lq[col][at] = make_float4(fq[i], fq[i + 1], fq[i + 2], fq[i + 3]);
      lk_[col][at] = make_float4(fk[i], fk[i + 1], fk[i + 2], fk[i + 3]);
      lg[col][at] = make_float4(expf(fg[i]), expf(fg[i + 1]), expf(fg[i + 2]), expf(fg[i + 3]));
    }
    lv[col][l] = fv;
    if (l == 0) {
      lbeta[col] = fb;
      lkq[col] = kq;
    }
    __syncthreads();
    const int steps = static_cast<int>(rows.end - t0 < kSerialTokens ? rows.end - t0 : kSerialTokens);
    if (t0 + kSerialTokens < rows.end) fetch(t0 + kSerialTokens);
    for (int i = 0; i < steps; ++i) {
      float pred = 0.f, sq = 0.f;
      float kk[RPL];
#pragma unroll
      for (int j = 0; j < RPL; j += 4) {
        const float4 g = lg[i][(j / 4) * 16 + l], k = lk_[i][(j / 4) * 16 + l],
                     q = lq[i][(j / 4) * 16 + l];
        const float gv[4] = {g.x, g.y, g.z, g.w}, kv[4] = {k.x, k.y, k.z, k.w},
                    qv[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          st[j + m] *= gv[m];
          kk[j + m] = kv[m];
          pred = fmaf(st[j + m], kv[m], pred);
          sq = fmaf(st[j + m], qv[m], sq);
        }
      }
      pred = row16_sum(pred);
      sq = row16_sum(sq);
      const float bu = lbeta[i] * (lv[i][col] - pred);
#pragma unroll
      for (int j = 0; j < RPL; ++j) st[j] = fmaf(kk[j], bu, st[j]);
      if (l == 0) lo[i][col] = a.scale * fmaf(lkq[i], bu, sq);
    }
    __syncthreads();
    const int oc = cb * kSerialCols + l;
    if (col < steps && oc < a.d_v)
      static_cast<T*>(a.out)[((t0 + col) * a.heads + h) * a.d_v + oc] = from_f32<DT>(lo[col][l]);
  }
#pragma unroll
  for (int i = 0; i < RPL; ++i) {
    const int r = l * RPL + i;
    if (r < a.d_k && c < a.d_v) a.state_out[sbase + static_cast<int64_t>(r) * a.d_v + c] = st[i];
  }
}

// ---------------------------------------------------------------------------
// The recurrence in chunks of 32 steps. Within a chunk with the state S before
// it, D_i the product of e^g over its steps up to i (per key row) and D_(j,i] that
// of the steps behind j up to i,
//   A_ij = beta_j sum_d k_i k_j D_(j,i]   (j < i)
//   P_ij = scale beta_j sum_d q_i k_j D_(j,i]   (j <= i)
//   (I + A) [W | U0] = [k D | v]
//   U = U0 - W S,   o = scale (q D) S + P U,   S = D_31 S + (beta k D_(.,31])^T U,
// which is the step form with its corrections u solved for together. Only the
// last line follows from chunk to chunk, so one launch computes W, U0, P and the
// scaled rows of every chunk (chunk_prepare_kernel) and another takes the
// states through them (chunk_scan_kernel). State, sums and everything that leaves
// the second launch are fp32; what multiplies there, W, Q, K, S and U, goes in as
// sums of two fp16 (22 bits, with powers of two beside them: see Scale), since an
// fp32 matrix instruction takes 8 times the time of four fp16 products.
//
// Decays are multiplied up, never divided or taken as differences of sums: every
// product of e^g <= 1 stays in [0, 1] with a relative error of 2^-24 a factor,
// whatever the decays (a sum of logs of 100 would carry 2^-17 of error into its
// exponential, a quotient of products overflows where a channel fades within
// the chunk). A and P then cost a product of every channel for every pair of
// steps in VALU work, so they and W, U0 are computed for halves a, b of 16 steps
// (120 + 136 pairs each) and the halves joined by matrix products: with
// M = W_b (beta k D)_a^T over a's decays to its end,
//   W_b <- W_b D_a - M W_a,  U0_b <- U0_b - M U0_a,  P_ba = (scale q D)_b (beta k D)_a^T,
//   (q D)_b <- (q D)_b D_a,  (beta k D)_a <- (beta k D)_a D_b.
// The scan is bound by the way from one chunk's state to the next (products, a
// barrier, an exchange through LDS, 1.2 us), hence not 16 steps a chunk: 8192 tokens
// x 32 heads took 707 us in chunks of 16, 605 in chunks of 32 (of then).
//
// Records. A chunk and head has one record in the workspace, its parts in the
// order in which the second launch's lanes load them (16 bytes a lane, 1 KB a
// wave): with m = lane % 16, g = lane / 16, r = 0..3, half h
//   W, Q (scale q D):    [h][p][hi, lo][lane][i] = row 16 h + m, channel 32 p + c(i)
//   K (beta k D_(.,31]): [t][hi, lo][lane][i] = channel 16 t + m, step c(i)
//                        (i = 0..7, c(i) = 16 (i / 4) + 4 g + i % 4)
//   D (D_31):            [channel]
//   P:                   [aa, ba, bb][lane][r] = row m, column 4 g + r of that block
//   the inverse scales of W's rows, Q's rows (both by kRowsUp) and K's tiles
//   U0:                  [h][tile t][lane][r] = value column 16 t + m, step 16 h + 4 g + r
// These are A operands for B operands that are the accumulators of an earlier
// product as they stand: lane (m, g) of a 16 x 16 result holds column m, rows 4 g + r,
// and two such tiles, split, serve as 32 rows of a product over 32.
constexpr int kHalf = 16;
constexpr int kChunk = 2 * kHalf;
constexpr int kPrepareThreads = 512;  // four waves a half
constexpr int kPass = 128;            // value columns solved at a time

typedef float f32x4_t __attribute__((ext_vector_type(4)));

struct ChunkArgs {
  float* records;
  int64_t first, count;  // chunk numbers of this window
  int64_t record;        // floats of one record
  int v_tiles;           // 16-column tiles of d_v
};

template <int NW>
struct ChunkLayout {  // float offsets of a record's parts; 32 NW channels, 2 NW tiles
  static constexpr int kChannels = 32 * NW;
  static constexpr int kTiles = 2 * NW;
  static constexpr int kW = 0, kQ = kChannels * kChunk, kK = 2 * kChannels * kChunk,
                       kD = 3 * kChannels * kChunk, kP = kD + kChannels, kS = kP + 3 * 256,
                       kU = kS + 2 * kChunk + 16;
};

typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// Eight fp32 values as the sums of two fp16 each, hi + lo, of 2^k times them.
struct Split {
  f16x8_t hi, lo;
};
// 2^k that brings the largest magnitude to [2^14, 2^15), as fp32 (at most 2^126),
// and its inverse. A value down to 2^-16 of the largest keeps 22 bits, a smaller one
// 2^-39 of the largest.
struct Scale {
  float up, down;
};
// Of the products with W and Q, what takes the state's scale back takes the rows' 2^14
// back as well, and the rows' inverse scales are kept 2^14 times as large: between the
// two the sums are at most 64 times the state's largest value, not 2^21 times.
constexpr float kRowsDown = 0x1p-14f, kRowsUp = 0x1p14f;
__device__ inline Scale scale_for(float largest) {
  const uint32_t e = __float_as_uint(largest) & 0x7F800000u;
  const uint32_t up = e < (15u << 23) ? 253u << 23 : (268u << 23) - e;
  return {__uint_as_float(up), __uint_as_float((254u << 23) - up)};
}
// (v - v == 0 would not do: of a product it is contracted to its rounding error)
__device__ inline bool is_finite(float v) { return fabsf(v) < INFINITY; }
__device__ inline float finite_abs(float v) { return is_finite(v) ? fabsf(v) : 0.f; }
__device__ inline Split split8(const float (&v)[8], float up) {
  Split s;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {  // (two at a time: packed conversions)
    const f32x2_t x = {v[i] * up, v[i + 1] * up};
    const f16x2_t hi = __builtin_convertvector(x, f16x2_t);
    s.hi[i] = hi[0];
    s.hi[i + 1] = hi[1];
    s.lo[i] = static_cast<_Float16>(fmaf(v[i], up, -static_cast<float>(hi[0])));
    s.lo[i + 1] = static_cast<_Float16>(fmaf(v[i + 1], up, -static_cast<float>(hi[1])));
  }
  return s;
}
// a . b over 32 (four products: the smallest is 2^-22 of the largest)
__device__ inline f32x4_t mfma_split(const Split& a, const Split& b, f32x4_t c) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.lo, b.lo, c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.lo, b.hi, c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.hi, b.lo, c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.hi, b.hi, c, 0, 0, 0);
}
// the largest over the four lanes 16 apart of values >= 0, whose bits order as they do
__device__ inline float column_max(float v) {
  auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const uint32_t m = x[0] > x[1] ? x[0] : x[1];
  x = __builtin_amdgcn_permlane16_swap(m, m, false, false);
  return __uint_as_float(x[0] > x[1] ? x[0] : x[1]);
}

// Sums of four values of each lane over the wave's four 16-lane rows: row g is left
// with that of value (g & 1) + 2 (g >> 1), by two exchanges that each halve what a
// lane still holds.
__device__ inline float rows_reduce(const float (&v)[4]) {
  float h[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]),
                                                    __float_as_uint(v[i + 2]), false, false);
    h[i] = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  }
  const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(h[0]), __float_as_uint(h[1]),
                                                  false, false);
  return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}

// `at` again, as a value that is known only once x is: keeps the LDS reads at it
// below x's computation. (The compiler otherwise moves the reads of all unrolled
// rows to the front: 420 registers, one wave on a SIMD.)
__device__ inline int after(int at, float x) {
  asm volatile("" : "+v"(at) : "v"(x));
  return at;
}

__device__ inline f32x4_t lds4(const float* p) { return *reinterpret_cast<const f32x4_t*>(p); }

// Block = one chunk and head; two share a CU (80 KB of LDS each) and cover each
// other's loads and barriers. 3840 records of 32 steps x 128 x 128 take 141 us, 370 MB
// read and written. No one thing bounds it: of 164 us (traced) 30 went without A and
// P, 27 with a third of the stores, none without the solve, and none with the next
// chunk's loads under way or with half the LDS reads of A and P.
template <int DT, int NW>
__global__ void __launch_bounds__(kPrepareThreads, 4) chunk_prepare_kernel(ScanArgs a, ChunkArgs c) {
  using T = typename Storage<DT>::type;
  using L = ChunkLayout<NW>;
  constexpr int RT = NW / 2;
  constexpr int kStride = L::kChannels + 4;  // rows 16 bytes apart in the banks
  constexpr int kVStride = kPass + 4;
  // rows of q, k, e^g; then of scale q D, beta k D, W
  __shared__ alignas(16) float sq[kChunk][kStride], sk[kChunk][kStride], sg[kChunk][kStride];
  __shared__ alignas(16) union {
    float part[2][2][4][kHalf * kHalf];  // the waves' sums for A and P of each half
    float u[kChunk][kVStride];           // U0 of one pass
  } sx;
  __shared__ alignas(16) float sa[2][kHalf][kHalf];
  __shared__ f32x4_t sm[8][kWave];  // the waves' sums for M and P_ba
  __shared__ alignas(16) float sd[2][L::kChannels];
  __shared__ float sb[kChunk];
  __shared__ float sl[2][2][NW][kHalf];  // largest of W, Q rows over 32 channels each
  const int h = static_cast<int>(blockIdx.x % a.heads);
  const int64_t local = blockIdx.x / a.heads;
  const SequenceTile at = find_sequence_tile(a.seq, c.first + local, kChunk);
  if (at.sequence < 0 || at.sequence == a.seq.count) return;
  const RowRange rows = sequence_rows(a.seq, at.sequence);
  const int64_t t0 = rows.begin + at.tile * kChunk;
  if (t0 >= rows.end) return;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), l = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int half = wave >> 2, in_half = tid & 255, w4 = wave & 3;

  // this thread's value column of the first pass (the upper threads of a half)
  float x[kHalf];
  auto load_values = [&](int vc) {
    const int from = vc >= 0 && vc < a.d_v ? vc : 0;
    const int64_t th = t0 + kHalf * half;
#pragma unroll
    for (int i = 0; i < kHalf; ++i) {
      const int64_t t = th + i < rows.end ? th + i : t0;
      x[i] = to_f32<DT>(static_cast<const T*>(a.v)[(t * a.heads + h) * a.d_v + from]);
    }
#pragma unroll
    for (int i = 0; i < kHalf; ++i) x[i] = th + i < rows.end && from == vc ? x[i] : 0.f;
  };
  load_values(in_half - kPass);
  {  // steps behind the sequence's end: no decay, no key, no query
    const int row = tid >> 4;
    const int64_t t = t0 + row;
    const bool ok = t < rows.end;
    const int64_t base = ((ok ? t : t0) * a.heads + h) * a.d_k;
    float qs[RT][4], ks[RT][4], gs[RT][4];
    const float beta = a.beta[(ok ? t : t0) * a.heads + h];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int d = 4 * (l + 16 * i);
      load_rows<4>(a.q + base, d, a.d_k, ok, qs[i]);
      load_rows<4>(a.k + base, d, a.d_k, ok, ks[i]);
      load_rows<4>(a.decay + base, d, a.d_k, ok, gs[i]);
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int d = 4 * (l + 16 * i);
      float(&q)[4] = qs[i], (&k)[4] = ks[i], (&e)[4] = gs[i];
#pragma unroll
      for (int y = 0; y < 4; ++y) e[y] = expf(e[y]);
      *reinterpret_cast<float4*>(&sq[row][d]) = make_float4(q[0], q[1], q[2], q[3]);
      *reinterpret_cast<float4*>(&sk[row][d]) = make_float4(k[0], k[1], k[2], k[3]);
      *reinterpret_cast<float4*>(&sg[row][d]) = make_float4(e[0], e[1], e[2], e[3]);
    }
    if (l == 0) sb[row] = ok ? beta : 0.f;
  }
  __syncthreads();

  // A and P of a half: lane (j, g) of wave w has key j against every row i >= j,
  // over a 16th of the channels; its product of decays runs along with i. Rows
  // i < j are dropped below.
  {
    const float beta = sb[kHalf * half + l];
    const int d0 = w4 * 16 * RT + g * 4 * RT;
    f32x4_t f[RT];
#pragma unroll 1
    for (int i0 = 0; i0 < kHalf; i0 += 4) {  // four rows at a time
      float kk[4] = {0.f, 0.f, 0.f, 0.f}, qk[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int y = 0; y < RT; ++y) {
        const int d = d0 + 4 * y;
        const f32x4_t own = lds4(&sk[kHalf * half + l][d]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = kHalf * half + i0 + i;
          const f32x4_t e = lds4(&sg[row][d]), k = lds4(&sk[row][d]), q = lds4(&sq[row][d]);
          const bool first = i0 + i <= l;
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            f[y][z] = first ? own[z] * beta : f[y][z] * e[z];
            kk[i] = fmaf(k[z], f[y][z], kk[i]);
            qk[i] = fmaf(q[z], f[y][z], qk[i]);
          }
        }
      }
      const int i = i0 + (g & 1) + 2 * (g >> 1);
      sx.part[half][0][w4][i * kHalf + l] = rows_reduce(kk);
      sx.part[half][1][w4][i * kHalf + l] = rows_reduce(qk);
    }
  }
  __syncthreads();
  float* const rec = c.records + (local * a.heads + h) * c.record;
  {
    const int i = in_half >> 4;
    const auto& kk = sx.part[half][0];
    const auto& qk = sx.part[half][1];
    const float as = (kk[0][in_half] + kk[1][in_half]) + (kk[2][in_half] + kk[3][in_half]);
    const float ps = (qk[0][in_half] + qk[1][in_half]) + (qk[2][in_half] + qk[3][in_half]);
    sa[half][i][l] = l < i ? as : 0.f;
    rec[L::kP + 512 * half + (i + 16 * (l >> 2)) * 4 + (l & 3)] = l <= i ? a.scale * ps : 0.f;
  }
  __syncthreads();

  // columns of [W | U0] of a half: one thread solves a column, row by row
  auto solve = [&]() {
#pragma unroll
    for (int i = 1; i < kHalf; ++i) {
      const int from = i < 4 ? 0 : after(0, x[i - 4]);  // three rows of A ahead
#pragma unroll
      for (int j = 0; j < i; j += 4) {
        const f32x4_t r = lds4(&sa[half][i][4 * from + j]);
#pragma unroll
        for (int y = 0; y < 4; ++y)
          if (j + y < i) x[i] = fmaf(-r[y], x[j + y], x[i]);
      }
    }
  };
  const int row0 = kHalf * half;
  if (in_half < L::kChannels) {
    const int col = in_half;  // read and replaced by this thread alone
    float left = 1.f, kept[kHalf];
#pragma unroll
    for (int j = kHalf - 1; j >= 0; --j) {
      kept[j] = sb[row0 + j] * sk[row0 + j][col] * left;
      left *= sg[row0 + j][col];
    }
    float keep = 1.f;
#pragma unroll
    for (int i = 0; i < kHalf; ++i) {
      keep *= sg[row0 + i][col];
      x[i] = sk[row0 + i][col] * keep;
      sq[row0 + i][col] *= a.scale * keep;
      sk[row0 + i][col] = kept[i];
    }
    sd[half][col] = keep;
    solve();
#pragma unroll
    for (int i = 0; i < kHalf; ++i) sg[row0 + i][col] = x[i];
  } else if (in_half >= kPass) {
    solve();
#pragma unroll
    for (int i = 0; i < kHalf; ++i) sx.u[row0 + i][in_half - kPass] = x[i];
  }
  __syncthreads();

  // M (waves 0 to 3) and P_ba (4 to 7), a quarter of the channels each; both
  // transposed: lane (row of b, g), register r = step 4 g + r of a
  {
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int y = 0; y < RT; ++y) {
      const int d = 16 * (w4 * RT + y) + 4 * g;
      const f32x4_t ka = lds4(&sk[l][d]);
      const f32x4_t rb = half ? lds4(&sq[kHalf + l][d]) : lds4(&sg[kHalf + l][d]);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(ka[r], rb[r], acc, 0, 0, 0);
    }
    sm[wave][lane] = acc;
  }
  __syncthreads();
  const f32x4_t mt = (sm[0][lane] + sm[1][lane]) + (sm[2][lane] + sm[3][lane]);
  auto put = [&](int off, f32x4_t v) { *reinterpret_cast<f32x4_t*>(rec + off + 4 * lane) = v; };
  if (wave == 4) put(L::kP + 256, (sm[4][lane] + sm[5][lane]) + (sm[6][lane] + sm[7][lane]));
  auto put_split = [&](int off, const Split& v) {
    *reinterpret_cast<f16x8_t*>(rec + off + 4 * lane) = v.hi;
    *reinterpret_cast<f16x8_t*>(rec + off + 256 + 4 * lane) = v.lo;
  };
  // W and Q of half b, channels 32 p to + 31, by wave 2 p + b
  float wv[8], qv[8];
  const int p = wave >> 1, b = wave & 1;
  if (p < NW) {
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int t = 2 * p + y, d = 16 * t + 4 * g;
      f32x4_t w = lds4(&sg[kHalf * b + l][d]), q = lds4(&sq[kHalf * b + l][d]);
      if (b) {
        const f32x4_t da = lds4(&sd[0][d]);
        f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc = __builtin_amdgcn_mfma_f32_16x16x4f32(sg[4 * g + r][16 * t + l], mt[r], acc, 0, 0, 0);
        w = w * da - acc;
        q *= da;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        wv[4 * y + r] = w[r];
        qv[4 * y + r] = q[r];
      }
    }
    float mw = 0.f, mq = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      mw = fmaxf(mw, finite_abs(wv[i]));
      mq = fmaxf(mq, finite_abs(qv[i]));
    }
    mw = column_max(mw);
    mq = column_max(mq);
    if (g == 0) {
      sl[0][b][p][l] = mw;
      sl[1][b][p][l] = mq;
    }
  }
  if (wave < L::kTiles) {
    const int ch = 16 * wave + l;
    const float db = sd[1][ch];
    float kv[8], most = 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      kv[r] = sk[4 * g + r][ch] * db;
      kv[4 + r] = sk[kHalf + 4 * g + r][ch];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) most = fmaxf(most, finite_abs(kv[i]));
#pragma unroll
    for (int i = 1; i < kWave; i <<= 1) most = fmaxf(most, __shfl_xor(most, i));
    const Scale sc = scale_for(most);
    put_split(L::kK + 512 * wave, split8(kv, sc.up));
    if (lane == 0) rec[L::kS + 2 * kChunk + wave] = sc.down;
    if (l == 0)
      *reinterpret_cast<f32x4_t*>(rec + L::kD + 16 * wave + 4 * g) =
          lds4(&sd[0][16 * wave + 4 * g]) * lds4(&sd[1][16 * wave + 4 * g]);
  }
  __syncthreads();
  if (p < NW) {  // a row has one scale over all channels
    float mw = sl[0][b][0][l], mq = sl[1][b][0][l];
#pragma unroll
    for (int y = 1; y < NW; ++y) {
      mw = fmaxf(mw, sl[0][b][y][l]);
      mq = fmaxf(mq, sl[1][b][y][l]);
    }
    const Scale w = scale_for(mw), q = scale_for(mq);
    put_split(L::kW + 512 * (b * NW + p), split8(wv, w.up));
    put_split(L::kQ + 512 * (b * NW + p), split8(qv, q.up));
    if (p == 0 && g == 0) {
      rec[L::kS + kHalf * b + l] = w.down * kRowsUp;
      rec[L::kS + kChunk + kHalf * b + l] = q.down * kRowsUp;
    }
  }
  for (int first = 0;;) {
    const int ct = first / 16 + wave;
    if (ct < c.v_tiles) {
      f32x4_t ua, ub, acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        ua[r] = sx.u[4 * g + r][16 * wave + l];
        ub[r] = sx.u[kHalf + 4 * g + r][16 * wave + l];
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(mt[r], ua[r], acc, 0, 0, 0);
      }
      put(L::kU + 256 * ct, ua);
      put(L::kU + 256 * (c.v_tiles + ct), ub - acc);
    }
    first += kPass;
    if (first >= 16 * c.v_tiles) break;
    __syncthreads();
    if (in_half >= kPass) {
      load_values(first + in_half - kPass);
      solve();
#pragma unroll
      for (int i = 0; i < kHalf; ++i) sx.u[row0 + i][in_half - kPass] = x[i];
    }
    __syncthreads();
  }
}

// Block = one sequence's and head's 16 CT value columns, through the chunks of the
// window. Each of NW waves keeps 32 key rows of the state as accumulators; the
// sums over all rows (W S - U0, Q S) meet in LDS, in wave order, with one barrier a
// chunk: W S before it, Q S behind it, where it covers the wait for the other
// waves' sums. Two more waves for each 16 columns, one for each half, do what is
// off the path from one state to the next: they bring U0 and the decays, and
// add up, complete (P U) and store the outputs, a chunk later.
//
// One prompt is bound by that path: 1.2 us a chunk for 32 heads of 128 x 128, where
// the matrix unit is busy for a sixth of the time and VALU for a third. So are many
// prompts, though their chunks are independent: with the records on their way a block's
// registers (204 a lane, 246 for two tiles) leave room for no second block on its CU,
// which could use the waits (4096 tokens of 11 prompts: 180 us, the longest prompt's
// chunks 41). 48 of a record's 68 KB
// are loaded as operands by the blocks of each 16 columns. The waves meet at the
// barrier, so their loads come at the same time: they are put between the
// products that follow it (in one place they held the waves up for 500 cycles of
// 1900), two chunks ahead, and without a branch (the last record again at the
// end), so that a wait leaves the younger ones in flight.
template <int DT, int NW, int CT>
__global__ void __launch_bounds__((NW + 2 * CT) * kWave)
chunk_scan_kernel(ScanArgs a, ChunkArgs c) {
  using T = typename Storage<DT>::type;
  using L = ChunkLayout<NW>;
  constexpr int kScanWaves = NW + 2 * CT;
  constexpr int kU0 = NW, kQS = NW + 1, kU = 2 * NW + 1;
  // of the last two chunks and each half: the waves' W S, - U0, the waves' Q S, - U;
  // D; what the rows of W and the tiles of K are scaled by
  __shared__ f32x4_t parts[2][CT][2][2 * NW + 2][kWave];
  __shared__ f32x4_t decay[2][L::kTiles * 4], w_down[2][2][4];
  __shared__ float k_down[2][L::kTiles];
  // the column tiles of a head, which read the same records, lie 8 blocks apart:
  // on one XCD, whose cache then holds a record for all of them
  const int64_t span = 8 * ((c.v_tiles + CT - 1) / CT), at = blockIdx.x % span;
  const int64_t sh = blockIdx.x / span * 8 + at % 8;
  const int ct = static_cast<int>(at / 8) * CT;  // the first of the block's tiles
  const int h = static_cast<int>(sh % a.heads);
  const int s = static_cast<int>(sh / a.heads);
  if (s > a.seq.count) return;
  const RowRange rows = sequence_rows(a.seq, s);
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int m = lane & 15, g = lane >> 4;
  if (s == a.seq.count) {  // rows behind the last sequence
    if (c.first == 0)
      for (int64_t t = rows.begin + (tid >> 4); t < rows.end; t += kScanWaves * 4)
        for (int x = 0; x < CT; ++x) {
          const int col = (ct + x) * 16 + m;
          if (col < a.d_v) static_cast<T*>(a.out)[(t * a.heads + h) * a.d_v + col] = 0;
        }
    return;
  }
  // the sequence's chunk numbers, at least one, and those of the window
  const int64_t number = rows.begin / kChunk + s;
  const int64_t chunks = (rows.end - rows.begin + kChunk - 1) / kChunk;
  const int64_t end_all = number + (chunks > 0 ? chunks : 1);
  const int64_t lo = number > c.first ? number : c.first;
  const int64_t hi = end_all < c.first + c.count ? end_all : c.first + c.count;
  if (lo >= hi) return;
  const int steps = chunks > 0 ? static_cast<int>(hi - lo) : 0;
  const int64_t stride = static_cast<int64_t>(a.heads) * c.record * 4;  // bytes from record to record
  const char* const first =
      reinterpret_cast<const char*>(c.records + ((lo - c.first) * a.heads + h) * c.record);
  const char* const last = first + (hi - lo - 1) * stride;
  // a record's parts at 32-bit byte offsets behind a scalar base
  const char* ahead = first;
  auto part_at = [&](uint32_t off) { return *reinterpret_cast<const f32x4_t*>(ahead + off); };
  auto advance = [&]() { ahead = ahead < last ? ahead + stride : last; };

  if (wave >= NW) {
    if (steps == 0) return;
    const int half = (wave - NW) & 1, tile = (wave - NW) >> 1;  // of the block
    const int vt = ct + tile < c.v_tiles ? ct + tile : ct;      // (no such tile: no column of it)
    const int col = (ct + tile) * 16 + m;
    const uint32_t values = static_cast<uint32_t>((L::kU + ((half * c.v_tiles + vt) * 64 + lane) * 4) * 4);
    const uint32_t planes = static_cast<uint32_t>((L::kP + 4 * lane) * 4);
    const uint32_t decays = static_cast<uint32_t>((L::kD + lane % (L::kChannels / 2) * 2) * 4);
    const uint32_t w_scales = static_cast<uint32_t>((L::kS + kHalf * half + m) * 4);
    const uint32_t q_scales = static_cast<uint32_t>((L::kS + kChunk + kHalf * half + 4 * g) * 4);
    const uint32_t k_scales = static_cast<uint32_t>((L::kS + 2 * kChunk + lane % L::kTiles) * 4);
    struct Record {
      f32x4_t u, p, pba, q_down;
      float2 d;
      float w_down, k_down;
    };
    auto fetch = [&](Record& f) {
      f.u = part_at(values);
      f.p = part_at(planes + 2048 * half);
      f.pba = part_at(planes + 1024);
      f.q_down = part_at(q_scales);
      f.d = *reinterpret_cast<const float2*>(ahead + decays);
      f.w_down = *reinterpret_cast<const float*>(ahead + w_scales);
      f.k_down = *reinterpret_cast<const float*>(ahead + k_scales);
      advance();
    };
    auto hand_over = [&](int i, const Record& f) {
      parts[i & 1][tile][half][kU0][lane] = -f.u;
      if (tile > 0) return;
      if (lane < kHalf) reinterpret_cast<float*>(w_down[i & 1][half])[lane] = f.w_down;
      if (half == 0) {
        if (lane < L::kChannels / 2) reinterpret_cast<float2*>(decay[i & 1])[lane] = f.d;
      } else if (lane < L::kTiles) {
        k_down[i & 1][lane] = f.k_down;
      }
    };
    // rows behind the sequence, columns behind the last and chunks not begun go
    // past the buffer's end: stores without a branch. Behind a branch the
    // compiler has to take them for not issued, and its waits for a record's
    // loads then wait for the stores as well (0.06 us a chunk).
    const int64_t row_values = static_cast<int64_t>(a.heads) * a.d_v;
    const int64_t row0 = rows.begin + (lo - number) * kChunk + kHalf * half;
    T* out = static_cast<T*>(a.out) + row0 * row_values + h * a.d_v;
    int64_t left = rows.end - row0;
    int off[4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
      off[r] = col < a.d_v
                   ? static_cast<int>(((4 * g + r) * row_values + col) * static_cast<int>(sizeof(T)))
                   : static_cast<int>(0x80000000u);
    const char* rec = first;
    // a chunk's outputs: begun behind the barrier of the next one, stored behind
    // the one after that, so that no barrier waits for their products
    auto begin = [&](int i, const f32x4_t& p, const f32x4_t& pba, const f32x4_t& q_down,
                     f32x4_t& u) {
      const f32x4_t(*const part)[kWave] = parts[i & 1][tile][half];
      u = -part[kU][lane];
      f32x4_t o = part[kQS][lane] + part[kQS + 1][lane];
      if constexpr (NW == 4) o += part[kQS + 2][lane] + part[kQS + 3][lane];
      o *= q_down;
      if (half) {
        const f32x4_t ua = -parts[i & 1][tile][0][kU][lane];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          o = __builtin_amdgcn_mfma_f32_16x16x4f32(pba[r], ua[r], o, 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
        o = __builtin_amdgcn_mfma_f32_16x16x4f32(p[r], is_finite(u[r]) ? u[r] : 0.f, o, 0, 0, 0);
      return o;
    };
    auto store = [&](f32x4_t o, f32x4_t u, bool begun) {
      const bool fine = is_finite(u[0]) && is_finite(u[1]) && is_finite(u[2]) && is_finite(u[3]);
      if (__builtin_expect(begun && !__all(fine), 0)) {
        // infinities and NaNs, which P's zeros would hand to the steps before
        // their own: left out of P U, and taken one by one by the steps
        // from theirs on
        const float* const p = reinterpret_cast<const float*>(rec) + L::kP + 512 * half;
#pragma unroll 1
        for (int j = 0; j < kHalf; ++j) {
          const float mine = (j & 2) ? ((j & 1) ? u[3] : u[2]) : ((j & 1) ? u[1] : u[0]);
          const float uj = __shfl(mine, m + 16 * (j >> 2));
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float pij = p[((4 * g + r) + 16 * (j >> 2)) * 4 + (j & 3)];
            if (j <= 4 * g + r && !is_finite(uj)) o[r] = fmaf(pij, uj, o[r]);
          }
        }
      }
      const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(out, 0, 0x7FFFFFFF, 0x00020000);
      const int live = begun ? (left < kHalf ? static_cast<int>(left) : kHalf) : 0;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at_r = 4 * g + r < live ? off[r] : static_cast<int>(0x80000000u);
        if constexpr (DT == LK_DTYPE_F32)
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(o[r]), rsrc, at_r, 0, 0);
        else
          __builtin_amdgcn_raw_buffer_store_b16(from_f32<DT>(o[r]), rsrc, at_r, 0, 0);
      }
      if (begun) {
        out += kChunk * row_values;
        left -= kChunk;
        rec += stride;
      }
    };
    // records three in turn, each until its outputs are begun (a copy of one on
    // its way would wait for it)
    Record f0, f1, f2;
    f32x4_t p = {0.f, 0.f, 0.f, 0.f}, pba = p, q_down = p, o = p, u = p;
    fetch(f0);
    fetch(f1);
    auto turn = [&](int i, const Record& f, Record& next) {
      hand_over(i, f);
      fetch(next);
      __syncthreads();
      store(o, u, i > 1);
      o = begin(i - 1, p, pba, q_down, u);  // (of nothing for i = 0)
      p = f.p;
      pba = f.pba;
      q_down = f.q_down;
    };
    int i = 0;
    for (; i + 3 <= steps; i += 3) {
      turn(i, f0, f2);
      turn(i + 1, f1, f0);
      turn(i + 2, f2, f1);
    }
    if (i < steps) turn(i, f0, f2);
    if (i + 1 < steps) turn(i + 1, f1, f0);
    __syncthreads();
    store(o, u, steps > 1);
    o = begin(steps - 1, p, pba, q_down, u);
    store(o, u, true);
    return;
  }

  // the state's rows 32 wave + 16 t + 4 g + r, and as the operand of the next chunk
  const float* const src = lo == number ? a.state : a.state_out;
  const int64_t sbase = sh * a.d_k * a.d_v;
  f32x4_t st[CT][2];
#pragma unroll
  for (int x = 0; x < CT; ++x)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 32 * wave + 16 * t + 4 * g + r, col = (ct + x) * 16 + m;
        st[x][t][r] =
            row < a.d_k && col < a.d_v ? src[sbase + static_cast<int64_t>(row) * a.d_v + col] : 0.f;
      }
  // both tiles (halves) of a column as an operand with one scale
  auto split_column = [&](const f32x4_t& v0, const f32x4_t& v1, Split& out) {
    const float v[8] = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(v[i]));
    const Scale sc = scale_for(column_max(most));
    out = split8(v, sc.up);
    return sc.down;
  };
  Split ss[CT];
  float s_down[CT];
#pragma unroll
  for (int x = 0; x < CT; ++x) s_down[x] = kRowsDown * split_column(st[x][0], st[x][1], ss[x]);
  struct Record {
    Split w[2], q[2], k[2];  // [half], [half], [tile]
  };
  // 2 KB a fragment; W and Q: half NW + wave, K: tile 2 wave + t
  const int w_at = (512 * wave + 4 * lane) * 4, k_at = (1024 * wave + 4 * lane) * 4;
  constexpr int kHalfBytes = 2048 * NW;
  auto split_at = [&](int at, int part) {  // (buffer loads: no 64-bit address for each)
    const auto rec = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(ahead), 0, 0x7FFFFFFF, 0x00020000);
    return Split{__builtin_bit_cast(f16x8_t, __builtin_amdgcn_raw_buffer_load_b128(rec, at, part, 0)),
                 __builtin_bit_cast(f16x8_t, __builtin_amdgcn_raw_buffer_load_b128(rec, at + 1024, part, 0))};
  };
  auto w_of = [&](int b) { return split_at(w_at, L::kW * 4 + kHalfBytes * b); };
  auto q_of = [&](int b) { return split_at(w_at, L::kQ * 4 + kHalfBytes * b); };
  auto k_of = [&](int t) { return split_at(k_at + 2048 * t, L::kK * 4); };
  auto fetch = [&](Record& f) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      f.w[x] = w_of(x);
      f.q[x] = q_of(x);
      f.k[x] = k_of(x);
    }
    advance();
  };
  auto step = [&](int i, const Record& f, Record& next) {
    f32x4_t(*const part)[2][2 * NW + 2][kWave] = parts[i & 1];
    const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < CT; ++x)
#pragma unroll
      for (int b = 0; b < 2; ++b)
        part[x][b][wave][lane] = mfma_split(f.w[b], ss[x], zero) * s_down[x];
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);  // Q S is not to be moved up
    f32x4_t down[2], d[2], y[CT][2], u[CT][2];
    float kd[2], u_down[CT];
    Split us[CT];
#pragma unroll
    for (int x = 0; x < CT; ++x) {
      f32x4_t xs[2][NW + 1];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int w = 0; w < NW + 1; ++w) xs[b][w] = part[x][b][w][lane];
      if (x == 0)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          down[b] = w_down[i & 1][b][g];
          d[b] = decay[i & 1][(2 * wave + b) * 4 + g];
          kd[b] = k_down[i & 1][2 * wave + b];
        }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        y[x][b] = mfma_split(f.q[b], ss[x], zero);
        if (x == 0) next.w[b] = w_of(b);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        f32x4_t sum = xs[b][0] + xs[b][1];
        if constexpr (NW == 4) sum += xs[b][2] + xs[b][3];
        u[x][b] = sum * down[b] + xs[b][kU0];  // - U
      }
      u_down[x] = split_column(u[x][0], u[x][1], us[x]);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x4_t acc[CT];
#pragma unroll
      for (int x = 0; x < CT; ++x) acc[x] = mfma_split(f.k[t], us[x], zero);
#pragma unroll
      for (int x = 0; x < CT; ++x) st[x][t] *= d[t];  // beside those products
      next.q[t] = q_of(t);
      next.k[t] = k_of(t);
#pragma unroll
      for (int x = 0; x < CT; ++x) part[x][t][kQS + wave][lane] = y[x][t] * s_down[x];
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int x = 0; x < CT; ++x) {
        const float down_x = -(kd[t] * u_down[x]);
#pragma unroll
        for (int r = 0; r < 4; ++r) st[x][t][r] = fmaf(acc[x][r], down_x, st[x][t][r]);
      }
    }
    advance();
    if (wave < 2)
#pragma unroll
      for (int x = 0; x < CT; ++x) part[x][wave][kU][lane] = wave == 0 ? u[x][0] : u[x][1];
#pragma unroll
    for (int x = 0; x < CT; ++x) s_down[x] = kRowsDown * split_column(st[x][0], st[x][1], ss[x]);
  };
  if (steps > 0) {
    Record f0, f1, f2;  // in turn
    fetch(f0);
    fetch(f1);
    int i = 0;
    for (; i + 3 <= steps; i += 3) {
      step(i, f0, f2);
      step(i + 1, f1, f0);
      step(i + 2, f2, f1);
    }
    if (i < steps) step(i, f0, f2);
    if (i + 1 < steps) step(i + 1, f1, f0);
    __syncthreads();  // the last chunk's Q S and U, for the other waves
  }
#pragma unroll
  for (int x = 0; x < CT; ++x)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 32 * wave + 16 * t + 4 * g + r, col = (ct + x) * 16 + m;
        if (row < a.d_k && col < a.d_v)
          a.state_out[sbase + static_cast<int64_t>(row) * a.d_v + col] = st[x][t][r];
      }
}

bool known_dtype(int d) { return d == LK_DTYPE_F32 || d == LK_DTYPE_F16 || d == LK_DTYPE_BF16; }
bool aligned(const void* p, int64_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(bytes) == 0;
}

int check_sequences(const int32_t* cu, int64_t sequences, int64_t tokens) {
  LK_REQUIRE(sequences > 0 && tokens >= 0, "a prompt call needs sequences, and tokens >= 0");
  LK_REQUIRE(tokens < (int64_t{1} << 31) && sequences < (int64_t{1} << 24),
             "too many tokens or sequences");
  LK_REQUIRE(cu || tokens % sequences == 0,
             "without offsets the tokens must divide into equal sequences");
  return LK_OK;
}

template <int DT, int WDT>
int launch_conv(const ConvArgs& a, bool wide, hipStream_t s) {
  constexpr int kWide = DT == LK_DTYPE_F32 ? 4 : 8;  // 16 bytes
  ConvArgs b = a;
  const int64_t items = 3 * (a.channels / (wide ? kWide : 1));
  const int64_t blocks = (items + kConvThreads - 1) / kConvThreads;
  const int64_t tiles = sequence_tiles(a.seq.rows, a.seq.count, kConvTile);
  LK_REQUIRE(grid_fits(blocks * tiles, kConvThreads), "too many tokens and channels for one call");
  b.column_blocks = static_cast<int>(blocks);
  const dim3 grid(static_cast<unsigned>(blocks * tiles));
  if (wide)
    conv_prefill_kernel<DT, WDT, kWide><<<grid, kConvThreads, 0, s>>>(b);
  else
    conv_prefill_kernel<DT, WDT, 1><<<grid, kConvThreads, 0, s>>>(b);
  return check_launch("lk_kda_short_conv_prefill");
}

template <int DT>
int launch_conv_weights(const ConvArgs& a, int weight_dtype, bool wide, hipStream_t s) {
  if (weight_dtype == LK_DTYPE_F32) return launch_conv<DT, LK_DTYPE_F32>(a, wide, s);
  if (weight_dtype == LK_DTYPE_F16) return launch_conv<DT, LK_DTYPE_F16>(a, wide, s);
  return launch_conv<DT, LK_DTYPE_BF16>(a, wide, s);
}

template <int DT>
int launch_serial(const ScanArgs& a, hipStream_t s) {
  const int64_t col_blocks = (a.d_v + kSerialCols - 1) / kSerialCols;
  const int64_t blocks = (a.seq.count + 1) * static_cast<int64_t>(a.heads) * col_blocks;
  LK_REQUIRE(grid_fits(blocks, kSerialThreads), "too many sequences x heads for one call");
  const dim3 grid(static_cast<unsigned>(blocks));
  const int cb = static_cast<int>(col_blocks);
  if (a.d_k <= 64)
    scan_serial_kernel<DT, 4><<<grid, kSerialThreads, 0, s>>>(a, cb);
  else if (a.d_k <= 128)
    scan_serial_kernel<DT, 8><<<grid, kSerialThreads, 0, s>>>(a, cb);
  else
    scan_serial_kernel<DT, 16><<<grid, kSerialThreads, 0, s>>>(a, cb);
  return check_launch("lk_kda_prefill");
}

// Floats of a chunk's and head's record.
int64_t chunk_record(int64_t d_k, int64_t d_v) {
  const int64_t channels = d_k <= 64 ? 64 : 128;
  return channels * (3 * kChunk + 1) + 3 * 256 + 2 * kChunk + 16 + (d_v + 15) / 16 * 16 * kChunk;
}

// From this many 16-column tiles of a call on (four for each CU, which holds one
// block), a block takes two: half the blocks load the same records. With one / with two
// tiles a block, us a call: 32 heads of 128 x 128, equal prompts, 4096 tokens in all,
// 256 tiles 298 / 337, 512 304 / 274, 1024 310 / 278, 2048 324 / 295, 4096 358 / 305;
// prompts of 512 tokens, 256 tiles 46 / 52, 512 75 / 68, 768 107 / 106, 1024 146 / 132,
// 4096 651 / 567. 16 heads of 64 x 64, prompts of 512 tokens, 1024 tiles 135 / 142, 2048
// 302 / 312. (Half as many tiles would do at d_k = 128; at 64 one is better.)
constexpr int64_t kTwoTiles = 1024;

// Chunks of one window: the records of a window are written by one launch and
// read by the next, partly from the 256 MB cache in front of HBM. Smaller windows
// leave more of them there, but begin and end more launches: 32, 64 and 128 MB
// were slower for 8192 tokens x 32 heads. It bounds the workspace as well.
constexpr int64_t kWindowBytes = int64_t{256} << 20;
int64_t chunk_window(int64_t chunks, int64_t heads, int64_t record) {
  const int64_t most = kWindowBytes / (heads * record * 4);
  const int64_t w = most < 1 ? 1 : most;
  return w < chunks ? w : chunks;
}

int64_t chunk_bytes(int64_t sequences, int64_t tokens, int64_t heads, int64_t d_k, int64_t d_v) {
  const int64_t record = chunk_record(d_k, d_v);
  return chunk_window(sequence_tiles(tokens, sequences, kChunk), heads, record) * heads * record * 4;
}

bool takes_chunks(int64_t sequences, int64_t tokens, int64_t heads, int64_t d_k, int64_t d_v) {
  const int choice = path_choice(kKnobKdaPrefill);
  // (a chunk's outputs are stored at 31-bit byte offsets. Beyond d_k = 128 there are
  // no chunks: prepare's rows of q, k and e^g alone would take 100 of a CU's 160 KB of
  // LDS at 256.) Chunks from 48 tokens a sequence on: 32 heads of 128 x 128 took, in
  // steps / in chunks, for one sequence of 32 tokens 15 / 18 us, of 48 20 / 19, of 128
  // 48 / 22; 16 heads of 64 x 64 for 16 sequences of 32 tokens 19 / 23. The tokens a
  // sequence are the call's mean, since the lengths are on the device; that takes the
  // slower form for 32 sequences of 32 tokens (150 / 127) and where one prompt is
  // among many short sequences: 1000 tokens beside 32 single ones 396 / 176, 2048
  // beside 64 880 / 390. The knob is for those.
  if (d_k > 128 || tokens == 0 || choice == 1 || heads * d_v >= (int64_t{1} << 24)) return false;
  return choice == 2 || tokens >= 48 * sequences;
}

template <int DT, int NW>
int launch_chunks(const ScanArgs& a, float* records, hipStream_t s) {
  ChunkArgs c;
  c.records = records;
  c.record = chunk_record(a.d_k, a.d_v);
  c.v_tiles = (a.d_v + 15) / 16;
  const int64_t chunks = sequence_tiles(a.seq.rows, a.seq.count, kChunk);
  const int64_t window = chunk_window(chunks, a.heads, c.record);
  const int64_t pairs = (a.seq.count + 1) * static_cast<int64_t>(a.heads);
  const bool two = c.v_tiles > 1 && a.seq.count * static_cast<int64_t>(a.heads) * c.v_tiles >= kTwoTiles;
  const int64_t scans = (pairs + 7) / 8 * 8 * (two ? (c.v_tiles + 1) / 2 : c.v_tiles);
  LK_REQUIRE(grid_fits(window * a.heads, kPrepareThreads) &&
                 grid_fits(scans, (NW + (two ? 4 : 2)) * kWave),
             "too many sequences x heads for one call");
  for (c.first = 0; c.first < chunks; c.first += window) {
    c.count = window < chunks - c.first ? window : chunks - c.first;
    chunk_prepare_kernel<DT, NW>
        <<<static_cast<unsigned>(c.count * a.heads), kPrepareThreads, 0, s>>>(a, c);
    if (const int st = check_launch("lk_kda_prefill")) return st;
    if (two)
      chunk_scan_kernel<DT, NW, 2><<<static_cast<unsigned>(scans), (NW + 4) * kWave, 0, s>>>(a, c);
    else
      chunk_scan_kernel<DT, NW, 1><<<static_cast<unsigned>(scans), (NW + 2) * kWave, 0, s>>>(a, c);
    if (const int st = check_launch("lk_kda_prefill")) return st;
  }
  return LK_OK;
}

template <int DT>
int launch_scan(const ScanArgs& a, bool chunks, void* workspace, hipStream_t s) {
  if (!chunks) return launch_serial<DT>(a, s);
  float* const records = static_cast<float*>(workspace);
  return a.d_k <= 64 ? launch_chunks<DT, 2>(a, records, s) : launch_chunks<DT, 4>(a, records, s);
}

}  // namespace
}  // namespace lk

using namespace lk;

extern "C" {

int lk_kda_short_conv_prefill(const void* q_in, const void* k_in, const void* v_in,
                              const void* q_state, const void* k_state, const void* v_state,
                              void* q_state_out, void* k_state_out, void* v_state_out,
                              const void* q_weight, const void* k_weight, const void* v_weight,
                              void* q_out, void* k_out, void* v_out, const int32_t* cu_seqlens,
                              int64_t sequences, int64_t tokens, int64_t channels,
                              int64_t row_stride, int value_dtype, int weight_dtype,
                              void* stream) {
  if (const int st = check_sequences(cu_seqlens, sequences, tokens)) return st;
  LK_REQUIRE(channels > 0 && channels < (int64_t{1} << 31), "short convolutions need channels");
  LK_REQUIRE(row_stride >= channels, "the row stride must hold a row");
  LK_REQUIRE(known_dtype(value_dtype) && known_dtype(weight_dtype), "unknown dtype code");
  LK_REQUIRE((tokens == 0 || (q_in && k_in && v_in && q_out && k_out && v_out)) && q_state &&
                 k_state && v_state && q_state_out && k_state_out && v_state_out && q_weight &&
                 k_weight && v_weight,
             "null pointer argument");
  const int size = value_dtype == LK_DTYPE_F32 ? 4 : 2;
  for (const void* p : {q_state, k_state, v_state, static_cast<const void*>(q_state_out),
                        static_cast<const void*>(k_state_out),
                        static_cast<const void*>(v_state_out)})
    LK_REQUIRE(aligned(p, 4 * size), "convolution states must be aligned to a channel's entries");
  for (const void* p : {q_weight, k_weight, v_weight})
    LK_REQUIRE(aligned(p, weight_dtype == LK_DTYPE_F32 ? 16 : 8),
               "convolution weights must be aligned to a channel's entries");
  bool wide = channels * size % 16 == 0 && row_stride * size % 16 == 0;
  for (const void* p : {q_in, k_in, v_in, static_cast<const void*>(q_out),
                        static_cast<const void*>(k_out), static_cast<const void*>(v_out)})
    wide = wide && aligned(p, 16);
  const ConvArgs a{{q_in, k_in, v_in},
                   {q_state, k_state, v_state},
                   {q_state_out, k_state_out, v_state_out},
                   {q_weight, k_weight, v_weight},
                   {q_out, k_out, v_out},
                   Sequences{cu_seqlens, tokens, tokens / sequences, static_cast<int>(sequences)},
                   channels,
                   row_stride,
                   0};
  const hipStream_t s = as_stream(stream);
  if (value_dtype == LK_DTYPE_F32) return launch_conv_weights<LK_DTYPE_F32>(a, weight_dtype, wide, s);
  if (value_dtype == LK_DTYPE_F16) return launch_conv_weights<LK_DTYPE_F16>(a, weight_dtype, wide, s);
  return launch_conv_weights<LK_DTYPE_BF16>(a, weight_dtype, wide, s);
}

int64_t lk_kda_prefill_workspace(int64_t sequences, int64_t tokens, int64_t heads, int64_t d_k,
                                 int64_t d_v) {
  if (sequences <= 0 || tokens < 0 || heads <= 0 || d_k <= 0 || d_v <= 0 || d_k > 256) return -1;
  if (!takes_chunks(sequences, tokens, heads, d_k, d_v)) return 0;
  return chunk_bytes(sequences, tokens, heads, d_k, d_v);
}

int lk_kda_prefill(const float* state, float* state_out, const float* q, const float* k,
                   const void* v, const float* decay, const float* beta, void* out,
                   const int32_t* cu_seqlens, int64_t sequences, int64_t tokens, int64_t heads,
                   int64_t d_k, int64_t d_v, float scale, int value_dtype, void* workspace,
                   int64_t workspace_bytes, void* stream) {
  if (const int st = check_sequences(cu_seqlens, sequences, tokens)) return st;
  LK_REQUIRE(heads > 0 && d_k > 0 && d_v > 0, "KDA prefill dimensions must be nonzero");
  LK_REQUIRE(heads <= 65535 && d_v <= (int64_t{1} << 20), "KDA prefill: too many heads or values");
  LK_REQUIRE(d_k <= 256, "KDA prefill supports d_k up to 256, got %lld", (long long)d_k);
  LK_REQUIRE(known_dtype(value_dtype), "unknown dtype code");
  LK_REQUIRE(state && state_out && (tokens == 0 || (q && k && v && decay && beta && out)),
             "null pointer argument");
  for (const void* p : {static_cast<const void*>(state), static_cast<const void*>(state_out),
                        static_cast<const void*>(q), static_cast<const void*>(k), v,
                        static_cast<const void*>(decay), static_cast<const void*>(out)})
    LK_REQUIRE(aligned(p, 16), "KDA prefill tensors must start on a 16-byte boundary");
  // the choice is read once: the knob may change in the middle of a call
  const bool chunks = takes_chunks(sequences, tokens, heads, d_k, d_v);
  const int64_t need = chunks ? chunk_bytes(sequences, tokens, heads, d_k, d_v) : 0;
  LK_REQUIRE(need == 0 || (workspace && workspace_bytes >= need),
             "KDA prefill workspace too small: %lld bytes, %lld needed",
             (long long)workspace_bytes, (long long)need);
  const ScanArgs a{state, state_out, q, k, v, decay, beta, out,
                   Sequences{cu_seqlens, tokens, tokens / sequences, static_cast<int>(sequences)},
                   static_cast<int>(heads), static_cast<int>(d_k), static_cast<int>(d_v), scale};
  LK_REQUIRE(aligned(workspace, 16), "KDA prefill workspace must be 16-byte aligned");
  const hipStream_t s = as_stream(stream);
  if (value_dtype == LK_DTYPE_F32) return launch_scan<LK_DTYPE_F32>(a, chunks, workspace, s);
  if (value_dtype == LK_DTYPE_F16) return launch_scan<LK_DTYPE_F16>(a, chunks, workspace, s);
  return launch_scan<LK_DTYPE_BF16>(a, chunks, workspace, s);
}

}  // extern "C"
