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
// Bound by HBM: 12 operations on a value that is read and written once. A
// thread owns N neighbouring channels (16 bytes) of one convolution and walks
// a tile of kConvTile tokens with the three earlier inputs in registers, eight
// rows' loads in flight; the tile's first three inputs are read again (3 rows
// in kConvTile, mostly from a cache). The thread with a sequence's first tile
// has read the state's values, so it is the one that replaces them: the state
// may be updated in place.
constexpr int kConvThreads = 256;
constexpr int kConvTile = 32;
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
  int weight_dtype;
};

template <typename T>
__device__ inline T pick(const T (&v)[3], int i) {
  return i == 0 ? v[0] : (i == 1 ? v[1] : v[2]);
}

__device__ inline float load_weight(const void* p, int64_t i, int dt) {
  if (dt == LK_DTYPE_F32) return static_cast<const float*>(p)[i];
  const uint16_t b = static_cast<const uint16_t*>(p)[i];
  return dt == LK_DTYPE_BF16 ? bf16_to_f32(b) : to_f32<LK_DTYPE_F16>(b);
}

template <int DT, int N>
__global__ void __launch_bounds__(kConvThreads) conv_prefill_kernel(ConvArgs a) {
  using T = typename Storage<DT>::type;
  using P = Pack<T, N>;
  const int64_t number = blockIdx.x / a.column_blocks;
  const int cb = blockIdx.x % a.column_blocks;
  const int conv = blockIdx.y;
  const int64_t c = (static_cast<int64_t>(cb) * kConvThreads + threadIdx.x) * N;
  if (c >= a.channels) return;
  const SequenceTile at = find_sequence_tile(a.seq, number, kConvTile);
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

  float w[4][N];
  {
    const void* const wp = pick(a.weight, conv);
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i][j] = load_weight(wp, (c + j) * 4 + i, a.weight_dtype);
  }
  float x1[N], x2[N], x3[N];  // the inputs 3, 2 and 1 tokens back
  if (at.tile == 0) {
    const int64_t sc = (static_cast<int64_t>(at.sequence) * a.channels + c) * 4;
    const T* const s = static_cast<const T*>(pick(a.state, conv)) + sc;
    T* const so = static_cast<T*>(pick(a.state_out, conv)) + sc;
    T old[N][4];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const Pack<T, 4> p = *reinterpret_cast<const Pack<T, 4>*>(s + 4 * j);
#pragma unroll
      for (int i = 0; i < 4; ++i) old[j][i] = p.v[i];
      x1[j] = to_f32<DT>(old[j][1]);
      x2[j] = to_f32<DT>(old[j][2]);
      x3[j] = to_f32<DT>(old[j][3]);
    }
    // entry i of the next state: token length - 4 + i, or entry length + i of
    // this one where that lies before the first token
    P last[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t t = length - 4 + i;
      if (t >= 0) {
        last[i] = *reinterpret_cast<const P*>(x + t * a.stride);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
          last[i].v[j] = t == -4 ? old[j][0] : (t == -3 ? old[j][1] : (t == -2 ? old[j][2] : old[j][3]));
      }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      Pack<T, 4> p;
#pragma unroll
      for (int i = 0; i < 4; ++i) p.v[i] = last[i].v[j];
      *reinterpret_cast<Pack<T, 4>*>(so + 4 * j) = p;
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

  for (int64_t t = t0; t < t1; t += kConvRows) {
    P row[kConvRows];
#pragma unroll
    for (int r = 0; r < kConvRows; ++r) {
      const int64_t tr = t + r < t1 ? t + r : t1 - 1;
      row[r] = *reinterpret_cast<const P*>(x + tr * a.stride);
    }
#pragma unroll
    for (int r = 0; r < kConvRows; ++r) {
      P res;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float now = to_f32<DT>(row[r].v[j]);
        const float acc =
            fmaf(now, w[3][j], fmaf(x3[j], w[2][j], fmaf(x2[j], w[1][j], x1[j] * w[0][j])));
        res.v[j] = from_f32<DT>(silu_fast_f32(acc));
        x1[j] = x2[j];
        x2[j] = x3[j];
        x3[j] = now;
      }
      if (t + r < t1) *reinterpret_cast<P*>(y + (t + r) * a.channels) = res;
    }
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
// the batch before it runs.
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

template <int RPL>
__device__ inline void load_rows(const float* p, int first, int d_k, bool ok, float (&r)[RPL]) {
  if ((d_k & 3) == 0) {
#pragma unroll
    for (int i = 0; i < RPL; i += 4) {
      const bool in = ok && first + i < d_k;
      const float4 x = in ? *reinterpret_cast<const float4*>(p + first + i)
                          : make_float4(0.f, 0.f, 0.f, 0.f);
      r[i] = x.x;
      r[i + 1] = x.y;
      r[i + 2] = x.z;
      r[i + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < RPL; ++i) r[i] = ok && first + i < d_k ? p[first + i] : 0.f;
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
    fv = ok && vc < a.d_v
             ? to_f32<DT>(static_cast<const T*>(a.v)[(t * a.heads + h) * a.d_v + vc])
             : 0.f;
    fb = ok ? a.beta[t * a.heads + h] : 0.f;
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

template <int DT>
int launch_conv(const ConvArgs& a, bool wide, hipStream_t s) {
  constexpr int kWide = DT == LK_DTYPE_F32 ? 4 : 8;  // 16 bytes
  ConvArgs b = a;
  const int64_t per = kConvThreads * (wide ? kWide : 1);
  const int64_t blocks = (a.channels + per - 1) / per;
  const int64_t tiles = sequence_tiles(a.seq.rows, a.seq.count, kConvTile);
  LK_REQUIRE(blocks * tiles < (int64_t{1} << 31), "too many tokens and channels for one call");
  b.column_blocks = static_cast<int>(blocks);
  const dim3 grid(static_cast<unsigned>(blocks * tiles), 3);
  if (wide)
    conv_prefill_kernel<DT, kWide><<<grid, kConvThreads, 0, s>>>(b);
  else
    conv_prefill_kernel<DT, 1><<<grid, kConvThreads, 0, s>>>(b);
  return check_launch("lk_kda_short_conv_prefill");
}

template <int DT>
int launch_serial(const ScanArgs& a, hipStream_t s) {
  const int64_t col_blocks = (a.d_v + kSerialCols - 1) / kSerialCols;
  const int64_t blocks = (a.seq.count + 1) * static_cast<int64_t>(a.heads) * col_blocks;
  LK_REQUIRE(blocks < (int64_t{1} << 31), "too many sequences x heads for one call");
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
                   0,
                   weight_dtype};
  const hipStream_t s = as_stream(stream);
  if (value_dtype == LK_DTYPE_F32) return launch_conv<LK_DTYPE_F32>(a, wide, s);
  if (value_dtype == LK_DTYPE_F16) return launch_conv<LK_DTYPE_F16>(a, wide, s);
  return launch_conv<LK_DTYPE_BF16>(a, wide, s);
}

int64_t lk_kda_prefill_workspace(int64_t sequences, int64_t tokens, int64_t heads, int64_t d_k,
                                 int64_t d_v) {
  if (sequences <= 0 || tokens < 0 || heads <= 0 || d_k <= 0 || d_v <= 0 || d_k > 256) return -1;
  return 0;
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
  const int64_t need = lk_kda_prefill_workspace(sequences, tokens, heads, d_k, d_v);
  LK_REQUIRE(need == 0 || (workspace && workspace_bytes >= need),
             "KDA prefill workspace too small: %lld bytes, %lld needed",
             (long long)workspace_bytes, (long long)need);
  const ScanArgs a{state, state_out, q, k, v, decay, beta, out,
                   Sequences{cu_seqlens, tokens, tokens / sequences, static_cast<int>(sequences)},
                   static_cast<int>(heads), static_cast<int>(d_k), static_cast<int>(d_v), scale};
  const hipStream_t s = as_stream(stream);
  if (value_dtype == LK_DTYPE_F32) return launch_serial<LK_DTYPE_F32>(a, s);
  if (value_dtype == LK_DTYPE_F16) return launch_serial<LK_DTYPE_F16>(a, s);
  return launch_serial<LK_DTYPE_BF16>(a, s);
}

}  // extern "C"
