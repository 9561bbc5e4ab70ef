// The paged cache of full attention layers, for gfx950: norms and rotation of new
// queries and keys, their write to the pages, copies of pages.

#include <algorithm>
#include <new>

#include "lk_common.hpp"
#include "lk_paged.h"
#include "lk_pages.hpp"

namespace lk {
namespace {

// ---------------------------------------------------------------------------
// Head norms, rotation, append

constexpr int kHeadThreads = 256;
constexpr int kHeadMaxDim = 256;

struct HeadArgs {
  const void *q, *k, *v, *q_weight, *k_weight;
  const float* cos_sin;
  const void* positions;
  void *q_out, *k_out, *v_out;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  int64_t k_page, k_page_row, k_page_head, v_page, v_page_row, v_page_head;
  PageTable table;
  Sequences sq;
  int64_t table_rows;
  int heads, kv_heads, d, d_v, rotary, offset;
  int slots, parts;  // of a token: heads of q, k (and v); blocks
  float eps;
  int interleaved, positions_64, weight_dtype;
};

template <int DT>
struct Four;  // four neighbouring values as stored
template <>
struct Four<LK_DTYPE_F32> {
  float4 v;
};
template <>
struct Four<LK_DTYPE_F16> {
  uint2 v;
};
template <>
struct Four<LK_DTYPE_BF16> {
  uint2 v;
};

template <int DT>
__device__ inline void unpack4(const Four<DT>& x, float (&f)[4]) {
  if constexpr (DT == LK_DTYPE_F32) {
    f[0] = x.v.x, f[1] = x.v.y, f[2] = x.v.z, f[3] = x.v.w;
  } else {
    const uint32_t w[4] = {x.v.x & 0xFFFFu, x.v.x >> 16, x.v.y & 0xFFFFu, x.v.y >> 16};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = value_of<DT == LK_DTYPE_BF16>(w[i]);
  }
}

template <int DT>
__device__ inline Four<DT> pack4(const float (&f)[4]) {
  if constexpr (DT == LK_DTYPE_F32)
    return {make_float4(f[0], f[1], f[2], f[3])};
  else
    return {make_uint2(pack2<DT == LK_DTYPE_BF16>(f[0], f[1]), pack2<DT == LK_DTYPE_BF16>(f[2], f[3]))};
}

template <int DT>
__device__ inline Four<DT> load4(const void* base, int64_t at) {
  return *reinterpret_cast<const Four<DT>*>(
      static_cast<const char*>(base) + at * static_cast<int64_t>(sizeof(Four<DT>) / 4));
}
template <int DT>
__device__ inline void store4(void* base, int64_t at, const Four<DT>& x) {
  *reinterpret_cast<Four<DT>*>(static_cast<char*>(base) +
                               at * static_cast<int64_t>(sizeof(Four<DT>) / 4)) = x;
}

__device__ inline void weights4(const void* base, int at, int dtype, float (&f)[4]) {
  if (dtype == LK_DTYPE_F32) unpack4(load4<LK_DTYPE_F32>(base, at), f);
  else if (dtype == LK_DTYPE_F16) unpack4(load4<LK_DTYPE_F16>(base, at), f);
  else unpack4(load4<LK_DTYPE_BF16>(base, at), f);
}

template <int LPR>
__device__ inline float lanes_sum(float v) {
  v += dpp_f32<kQuadXor1>(v);
  v += dpp_f32<kQuadXor2>(v);
  v += dpp_f32<kRowHalfMirror>(v);
  if constexpr (LPR >= 16) v += dpp_f32<kRowMirror>(v);
  if constexpr (LPR >= 32) v += __shfl_xor(v, 16);
  return v;
}

// A row (a head of a token) is LPR lanes' (8, 16 or 32), a lane has two groups of
// four of its values: the partners of a rotation, so that nothing is exchanged but
// the sum of squares.
template <int DT, int LPR, bool PAGED>
__global__ void __launch_bounds__(kHeadThreads) head_rope_kernel(HeadArgs a) {
  constexpr int kRows = kHeadThreads / LPR;
  const int64_t t = blockIdx.x / a.parts;
  const int part = static_cast<int>(blockIdx.x % a.parts);
  const int lane = threadIdx.x % LPR;
  int64_t pos = 0;
  bool behind = false, place = false;
  int64_t page = 0;
  int in_page = 0;
  if constexpr (PAGED) {
    const int s = find_sequence(a.sq, t);
    const RowRange rows = sequence_rows(a.sq, s);
    behind = s >= a.sq.count || t < rows.begin || t >= rows.end;
    if (!behind) {
      pos = cached_length(a.table, s) - (rows.end - t);
      if (pos >= 0) {
        const int64_t block = pos / a.table.page_rows;
        in_page = static_cast<int>(pos - block * a.table.page_rows);
        page = a.table.pages_of[s * a.table.stride + block];
        place = page >= 0 && page < a.table.pages;
      }
    }
  } else {
    pos = a.positions_64 ? static_cast<const int64_t*>(a.positions)[t]
                         : static_cast<const int32_t*>(a.positions)[t];
  }
  pos = pos < 0 ? 0 : (pos >= a.table_rows ? a.table_rows - 1 : pos);
  // where this lane's two groups start, and whether they are turned
  int ga, gb, angle = 0;
  bool turned;
  if (a.interleaved) {
    ga = 8 * lane, gb = ga + 4;
    turned = ga >= a.offset && ga < a.offset + a.rotary;
    angle = (ga - a.offset) / 2;
  } else {
    turned = 8 * lane < a.rotary;
    ga = turned ? a.offset + 4 * lane : 8 * lane - a.rotary;
    if (!turned && ga >= a.offset) ga += a.rotary;
    gb = turned ? ga + a.rotary / 2 : ga + 4;
    angle = 4 * lane;
  }
  float c[4] = {1.f, 1.f, 1.f, 1.f}, s[4] = {0.f, 0.f, 0.f, 0.f};
  if (turned) {
    const float* const row = a.cos_sin + pos * a.rotary + angle;
    unpack4(load4<LK_DTYPE_F32>(row, 0), c);
    unpack4(load4<LK_DTYPE_F32>(row, a.rotary / 2), s);
  }
  for (int slot = part * kRows + threadIdx.x / LPR; slot < a.slots; slot += a.parts * kRows) {
    if (PAGED && slot >= a.heads + a.kv_heads) {  // v, as it is
      const int head = slot - a.heads - a.kv_heads;
      if (8 * lane < a.d_v && place) {
        const int64_t from = t * a.v_row + head * a.v_head + 8 * lane;
        const int64_t to = page * a.v_page + in_page * a.v_page_row + head * a.v_page_head + 8 * lane;
        const Four<DT> x = load4<DT>(a.v, from), y = load4<DT>(a.v, from + 4);
        store4(a.v_out, to, x);
        store4(a.v_out, to + 4, y);
      }
      continue;
    }
    const bool is_q = slot < a.heads;
    const int head = is_q ? slot : slot - a.heads;
    const bool mine = 8 * lane < a.d;
    float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
    if (mine) {
      const void* const from = is_q ? a.q : a.k;
      const int64_t at = is_q ? t * a.q_row + head * a.q_head : t * a.k_row + head * a.k_head;
      unpack4(load4<DT>(from, at + ga), x);
      unpack4(load4<DT>(from, at + gb), y);
    }
    const void* const weight = is_q ? a.q_weight : a.k_weight;
    if (weight) {
      float sq = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) sq = fmaf(x[i], x[i], sq);
#pragma unroll
      for (int i = 0; i < 4; ++i) sq = fmaf(y[i], y[i], sq);
      const float r = 1.0f / sqrtf(lanes_sum<LPR>(sq) / static_cast<float>(a.d) + a.eps);
      if (mine) {
        float w[4], u[4];
        weights4(weight, ga, a.weight_dtype, w);
        weights4(weight, gb, a.weight_dtype, u);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = x[i] * r * w[i], y[i] = y[i] * r * u[i];
      }
    }
    if (turned) {
      if (a.interleaved) {
        const float p[4] = {x[0], x[2], y[0], y[2]}, q[4] = {x[1], x[3], y[1], y[3]};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float* const to = i < 2 ? x + 2 * i : y + 2 * (i - 2);
          to[0] = p[i] * c[i] - q[i] * s[i];
          to[1] = q[i] * c[i] + p[i] * s[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = x[i], q = y[i];
          x[i] = p * c[i] - q * s[i];
          y[i] = q * c[i] + p * s[i];
        }
      }
    }
    if (PAGED && behind) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = y[i] = 0.f;
    }
    if (!mine || (PAGED && !is_q && !place)) continue;
    void* const out = is_q ? a.q_out : a.k_out;
    int64_t to = (t * (is_q ? a.heads : a.kv_heads) + head) * a.d;
    if (PAGED && !is_q) to = page * a.k_page + in_page * a.k_page_row + head * a.k_page_head;
    store4(out, to + ga, pack4<DT>(x));
    store4(out, to + gb, pack4<DT>(y));
  }
}

template <int DT, bool PAGED>
int launch_heads(HeadArgs& a, int64_t rows, const char* name, hipStream_t s) {
  const int width = PAGED && a.d_v > a.d ? a.d_v : a.d;
  const int lanes = width <= 64 ? 8 : (width <= 128 ? 16 : 32);
  a.parts = (a.slots + kHeadThreads / lanes - 1) / (kHeadThreads / lanes);
  const int64_t blocks = rows * a.parts;
  LK_REQUIRE(grid_fits(blocks, kHeadThreads), "too many rows and heads for one call");
  const dim3 grid(static_cast<unsigned>(blocks));
  if (lanes == 8) head_rope_kernel<DT, 8, PAGED><<<grid, kHeadThreads, 0, s>>>(a);
  else if (lanes == 16) head_rope_kernel<DT, 16, PAGED><<<grid, kHeadThreads, 0, s>>>(a);
  else head_rope_kernel<DT, 32, PAGED><<<grid, kHeadThreads, 0, s>>>(a);
  return check_launch(name);
}

bool on_16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// What both entry points ask of heads, widths, weights and the table of angles.
int check_heads(int64_t rows, int64_t heads, int64_t kv_heads, int64_t d, int64_t rotary,
                int64_t offset, int64_t table_rows, float eps, const void* q_weight,
                const void* k_weight, bool with_q, const float* cos_sin, int weight_dtype) {
  LK_REQUIRE(rows >= 0 && rows < (int64_t{1} << 31), "rows must be in 0 .. 2^31 - 1");
  LK_REQUIRE(heads >= 0 && kv_heads > 0 && heads <= 65535 && kv_heads <= 65535,
             "heads must be in 1 .. 65535");
  LK_REQUIRE(d > 0 && d % 8 == 0 && d <= kHeadMaxDim,
             "the head dimension must be a multiple of 8 up to %d, got %lld", kHeadMaxDim,
             (long long)d);
  LK_REQUIRE(rotary >= 0 && rotary % 8 == 0 && offset >= 0 && offset % 8 == 0 && rotary <= d &&
                 offset <= d - rotary,
             "the rotated slice must lie within the head, in multiples of 8");
  LK_REQUIRE(rotary == 0 || (cos_sin && on_16(cos_sin) && table_rows > 0),
             "a rotation needs a table of angles on a 16-byte boundary");
  LK_REQUIRE(!with_q || (q_weight == nullptr) == (k_weight == nullptr),
             "both norm weights must be given, or neither");
  LK_REQUIRE(on_16(q_weight) && on_16(k_weight), "norm weights must start on a 16-byte boundary");
  LK_REQUIRE(weight_dtype >= LK_DTYPE_F32 && weight_dtype <= LK_DTYPE_BF16,
             "unknown norm weight dtype %d", weight_dtype);
  LK_REQUIRE(eps >= 0.f, "eps must be non-negative");
  return LK_OK;
}

// ---------------------------------------------------------------------------
// Copies of pages

constexpr int kCopyThreads = 256;
constexpr int kCopyPairs = 192;    // of a launch: the lists travel as its arguments
constexpr int kCopyTensors = 64;   // of a launch

struct CopyArgs {
  char* tensor[kCopyTensors];
  int64_t stride[kCopyTensors];
  int32_t chunks[kCopyTensors];  // of 16 bytes a page
  int32_t src[kCopyPairs], dst[kCopyPairs];
};
static_assert(sizeof(CopyArgs) <= 4096, "kernel arguments");

__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(CopyArgs a) {
  const int z = blockIdx.z, pair = blockIdx.y;
  const uint4* const from = reinterpret_cast<const uint4*>(a.tensor[z] + a.src[pair] * a.stride[z]);
  uint4* const to = reinterpret_cast<uint4*>(a.tensor[z] + a.dst[pair] * a.stride[z]);
  const int i = blockIdx.x * kCopyThreads + threadIdx.x;
  if (i < a.chunks[z]) to[i] = from[i];
}

// A page is written once, and is no other pair's source: what a launch reads it
// does not write.
int check_pairs(const int32_t* src, const int32_t* dst, int64_t pairs, int64_t pages) {
  for (int64_t i = 0; i < pairs; ++i)
    LK_REQUIRE(src[i] >= 0 && src[i] < pages && dst[i] >= 0 && dst[i] < pages,
               "pair %lld copies page %d to %d of a cache of %lld", (long long)i, src[i], dst[i],
               (long long)pages);
  int32_t* const sorted = new (std::nothrow) int32_t[2 * pairs];
  LK_REQUIRE(sorted, "no memory for the list of pages");
  int32_t *const to = sorted, *const from = sorted + pairs;
  int64_t n = 0;
  for (int64_t i = 0; i < pairs; ++i)
    if (src[i] != dst[i]) to[n] = dst[i], from[n++] = src[i];
  std::sort(to, to + n);
  std::sort(from, from + n);
  int32_t twice = -1, both = -1;
  for (int64_t i = 1; i < n; ++i)
    if (to[i] == to[i - 1]) twice = to[i];
  for (int64_t i = 0, j = 0; i < n && j < n;) {
    if (to[i] == from[j]) both = to[i];
    if (to[i] <= from[j]) ++i;
    else ++j;
  }
  delete[] sorted;
  LK_REQUIRE(twice < 0, "page %d is written twice", twice);
  LK_REQUIRE(both < 0, "page %d is both read and written", both);
  return LK_OK;
}

}  // namespace
}  // namespace lk

using namespace lk;

extern "C" {

int lk_qk_norm_rope(const void* q, const void* k, const void* q_weight, const void* k_weight,
                    const float* cos_sin, const void* positions, void* q_out, void* k_out,
                    int64_t rows, int64_t heads, int64_t kv_heads, int64_t d,
                    int64_t q_row_stride, int64_t q_head_stride, int64_t k_row_stride,
                    int64_t k_head_stride, int64_t rotary, int64_t offset, int interleaved,
                    int64_t table_rows, int positions_64, float eps, int dtype, int weight_dtype,
                    void* stream) {
  if (const int st = check_heads(rows, heads, kv_heads, d, rotary, offset, table_rows, eps,
                                 q_weight, k_weight, true, cos_sin, weight_dtype))
    return st;
  LK_REQUIRE(heads > 0, "heads must be in 1 .. 65535");
  for (const int64_t stride : {q_row_stride, q_head_stride, k_row_stride, k_head_stride})
    LK_REQUIRE(stride >= 0 && stride % 8 == 0, "strides must be multiples of 8 elements, not negative");
  LK_REQUIRE(dtype >= LK_DTYPE_F32 && dtype <= LK_DTYPE_BF16, "unknown dtype %d", dtype);
  if (rows == 0) return LK_OK;
  LK_REQUIRE(q && k && q_out && k_out && (positions || rotary == 0), "null pointer argument");
  LK_REQUIRE(on_16(q) && on_16(k) && on_16(q_out) && on_16(k_out),
             "queries and keys must start on a 16-byte boundary");
  HeadArgs a{};
  a.q = q, a.k = k, a.q_weight = q_weight, a.k_weight = k_weight;
  a.cos_sin = cos_sin, a.positions = positions, a.q_out = q_out, a.k_out = k_out;
  a.q_row = q_row_stride, a.q_head = q_head_stride, a.k_row = k_row_stride, a.k_head = k_head_stride;
  a.table_rows = table_rows, a.positions_64 = positions_64 != 0;
  a.heads = static_cast<int>(heads), a.kv_heads = static_cast<int>(kv_heads);
  a.d = static_cast<int>(d), a.rotary = static_cast<int>(rotary), a.offset = static_cast<int>(offset);
  a.slots = a.heads + a.kv_heads;
  a.eps = eps, a.interleaved = interleaved != 0, a.weight_dtype = weight_dtype;
  const hipStream_t s = as_stream(stream);
  constexpr const char* kName = "lk_qk_norm_rope";
  if (dtype == LK_DTYPE_F32) return launch_heads<LK_DTYPE_F32, false>(a, rows, kName, s);
  if (dtype == LK_DTYPE_F16) return launch_heads<LK_DTYPE_F16, false>(a, rows, kName, s);
  return launch_heads<LK_DTYPE_BF16, false>(a, rows, kName, s);
}

int lk_paged_append(const void* q, const void* k, const void* v, const void* q_weight,
                    const void* k_weight, const float* cos_sin, const int32_t* page_table,
                    const int32_t* lengths, const int32_t* cu, void* q_out, void* k_pages,
                    void* v_pages, int64_t sequences, int64_t rows, int64_t heads,
                    int64_t kv_heads, int64_t d_qk, int64_t d_v, int64_t q_row_stride,
                    int64_t q_head_stride, int64_t k_row_stride, int64_t k_head_stride,
                    int64_t v_row_stride, int64_t v_head_stride, int64_t pages, int64_t page_rows,
                    int64_t table_width, int64_t table_stride, int64_t k_page, int64_t k_page_row,
                    int64_t k_page_head, int64_t v_page, int64_t v_page_row, int64_t v_page_head,
                    int64_t rotary, int64_t offset, int interleaved, int64_t table_rows, float eps,
                    int dtype, int weight_dtype, void* stream) {
  if (const int st = check_heads(rows, heads, kv_heads, d_qk, rotary, offset, table_rows, eps,
                                 heads ? q_weight : nullptr, k_weight, heads > 0, cos_sin,
                                 weight_dtype))
    return st;
  LK_REQUIRE(d_v > 0 && d_v % 8 == 0 && d_v <= kHeadMaxDim,
             "the value dimension must be a multiple of 8 up to %d, got %lld", kHeadMaxDim,
             (long long)d_v);
  LK_REQUIRE(dtype == LK_DTYPE_F16 || dtype == LK_DTYPE_BF16, "cached values must be fp16 or bf16");
  for (const int64_t stride : {q_row_stride, q_head_stride, k_row_stride, k_head_stride,
                               v_row_stride, v_head_stride})
    LK_REQUIRE(stride >= 0 && stride % 8 == 0, "strides must be multiples of 8 elements, not negative");
  if (const int st = check_pages(sequences, rows, cu != nullptr, pages, page_rows, table_width,
                                 table_stride, {k_page, k_page_row, k_page_head, v_page, v_page_row,
                                                v_page_head}))
    return st;
  if (rows == 0) return LK_OK;
  LK_REQUIRE(k && v && lengths && (table_width == 0 || page_table) && (pages == 0 || (k_pages && v_pages)) &&
                 (heads == 0 || (q && q_out)),
             "null pointer argument");
  LK_REQUIRE(on_16(k) && on_16(v) && on_16(k_pages) && on_16(v_pages) &&
                 (heads == 0 || (on_16(q) && on_16(q_out))),
             "queries, keys, values and pages must start on a 16-byte boundary");
  HeadArgs a{};
  a.q = q, a.k = k, a.v = v, a.q_weight = q_weight, a.k_weight = k_weight;
  a.cos_sin = cos_sin, a.q_out = q_out, a.k_out = k_pages, a.v_out = v_pages;
  a.q_row = q_row_stride, a.q_head = q_head_stride, a.k_row = k_row_stride, a.k_head = k_head_stride;
  a.v_row = v_row_stride, a.v_head = v_head_stride;
  a.k_page = k_page, a.k_page_row = k_page_row, a.k_page_head = k_page_head;
  a.v_page = v_page, a.v_page_row = v_page_row, a.v_page_head = v_page_head;
  a.table = PageTable{page_table, lengths, table_stride, pages, static_cast<int>(table_width),
                      static_cast<int>(page_rows)};
  a.sq = Sequences{cu, rows, rows / sequences, static_cast<int>(sequences)};
  a.table_rows = table_rows;
  a.heads = static_cast<int>(heads), a.kv_heads = static_cast<int>(kv_heads);
  a.d = static_cast<int>(d_qk), a.d_v = static_cast<int>(d_v);
  a.rotary = static_cast<int>(rotary), a.offset = static_cast<int>(offset);
  a.slots = a.heads + 2 * a.kv_heads;
  a.eps = eps, a.interleaved = interleaved != 0, a.weight_dtype = weight_dtype;
  const hipStream_t s = as_stream(stream);
  constexpr const char* kName = "lk_paged_append";
  if (dtype == LK_DTYPE_F16) return launch_heads<LK_DTYPE_F16, true>(a, rows, kName, s);
  return launch_heads<LK_DTYPE_BF16, true>(a, rows, kName, s);
}

int lk_copy_pages(void* const* tensors, const int64_t* page_strides, const int64_t* page_bytes,
                  int64_t count, const int32_t* src, const int32_t* dst, int64_t pairs,
                  int64_t pages, void* stream) {
  LK_REQUIRE(count >= 0 && pairs >= 0 && pages >= 0 && pages < (int64_t{1} << 31) &&
                 pairs < (int64_t{1} << 31),
             "tensors, pairs and pages must be in 0 .. 2^31 - 1");
  if (count == 0 || pairs == 0) return LK_OK;
  LK_REQUIRE(tensors && page_strides && page_bytes && src && dst, "null pointer argument");
  int64_t most = 0;
  for (int64_t i = 0; i < count; ++i) {
    LK_REQUIRE(tensors[i], "null pointer argument");
    LK_REQUIRE(on_16(tensors[i]) && page_strides[i] % 16 == 0 && page_bytes[i] % 16 == 0,
               "pages must start on 16-byte boundaries and be a multiple of 16 bytes");
    LK_REQUIRE(page_bytes[i] >= 0 && page_bytes[i] <= page_strides[i] &&
                   page_bytes[i] < (int64_t{1} << 31),
               "pages must not overlap, and be below 2^31 bytes");
    most = std::max(most, page_bytes[i]);
  }
  if (const int st = check_pairs(src, dst, pairs, pages)) return st;
  if (most == 0) return LK_OK;
  const hipStream_t s = as_stream(stream);
  for (int64_t z0 = 0; z0 < count; z0 += kCopyTensors)
    for (int64_t p0 = 0; p0 < pairs; p0 += kCopyPairs) {
      CopyArgs a{};
      const int z = static_cast<int>(std::min<int64_t>(kCopyTensors, count - z0));
      const int n = static_cast<int>(std::min<int64_t>(kCopyPairs, pairs - p0));
      for (int i = 0; i < z; ++i) {
        a.tensor[i] = static_cast<char*>(tensors[z0 + i]);
        a.stride[i] = page_strides[z0 + i];
        a.chunks[i] = static_cast<int32_t>(page_bytes[z0 + i] / 16);
      }
      std::copy(src + p0, src + p0 + n, a.src);
      std::copy(dst + p0, dst + p0 + n, a.dst);
      const dim3 grid(static_cast<unsigned>((most / 16 + kCopyThreads - 1) / kCopyThreads),
                      static_cast<unsigned>(n), static_cast<unsigned>(z));
      copy_pages_kernel<<<grid, kCopyThreads, 0, s>>>(a);
      if (const int st = check_launch("lk_copy_pages")) return st;
    }
  return LK_OK;
}

}  // extern "C"
