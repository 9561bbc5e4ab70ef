// Causal softmax attention of new rows on a paged cache, for gfx950.

#include "lk_common.hpp"
#include "lk_paged.h"
#include "lk_pages.hpp"

namespace lk {
namespace {

constexpr int kPagedThreads = 256;
constexpr int kPagedWaves = kPagedThreads / kWave;
constexpr int kPagedMaxQk = 192;
constexpr int kPagedMaxV = 128;

struct PagedArgs {
  const uint16_t *q, *k, *v;
  uint16_t* out;
  Sequences sq;
  PageTable table;
  int64_t q_row, q_head;
  int64_t k_page, k_row, k_head, v_page, v_row, v_head;
  int heads, group, d_qk, d_v;
  float scale_log2;
};

// One wave a row and head: a lane a key of each 64, then a lane two columns.
template <bool BF16>
__global__ void __launch_bounds__(kPagedThreads) paged_rows_kernel(PagedArgs a) {
  __shared__ alignas(16) float query[kPagedWaves][kPagedMaxQk];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kPagedWaves + wave;
  const int64_t t = item / a.heads;
  const int head = static_cast<int>(item - t * a.heads);
  if (t >= a.sq.rows) return;
  float* const qs = query[wave];
  for (int i = lane; i < a.d_qk; i += kWave)
    qs[i] = value_of<BF16>(a.q[t * a.q_row + head * a.q_head + i]);
  const int s = find_sequence(a.sq, t);
  const RowRange rows = sequence_rows(a.sq, s);
  int64_t seen = 0;
  if (s < a.sq.count && t >= rows.begin && t < rows.end)
    seen = cached_length(a.table, s) - (rows.end - t) + 1;
  const int64_t hk = head / a.group;
  float top = -INFINITY, sum = 0.f, acc[2] = {0.f, 0.f};
  for (int64_t k0 = 0; k0 < seen; k0 += kWave) {
    const int64_t key = k0 + lane;
    float score = -INFINITY;
    int64_t page = -1, row = 0;
    if (key < seen) {
      const int64_t block = key / a.table.page_rows;
      row = key - block * a.table.page_rows;
      page = a.table.pages_of[s * a.table.stride + block];
      if (page >= a.table.pages) page = -1;
      float dot = 0.f;
      if (page >= 0) {
        const uint16_t* const kp = a.k + page * a.k_page + row * a.k_row + hk * a.k_head;
        for (int i = 0; i < a.d_qk; ++i) dot = fmaf(value_of<BF16>(kp[i]), qs[i], dot);
      }
      score = dot * a.scale_log2;
    }
    float most = score;
    for (int m = 1; m < kWave; m *= 2) most = fmaxf(most, __shfl_xor(most, m));
    const float next = fmaxf(top, most);
    const float fade = next == -INFINITY ? 1.f : exp2f(top - next);
    top = next;
    const float p = score == -INFINITY ? 0.f : exp2f(score - top);
    sum = sum * fade + p;
    acc[0] *= fade, acc[1] *= fade;
    for (int j = 0; j < kWave && k0 + j < seen; ++j) {
      const float pj = __shfl(p, j);
      const int64_t pg = __shfl(static_cast<int>(page), j), r = __shfl(static_cast<int>(row), j);
      if (pg < 0) continue;
      const uint16_t* const vp = a.v + pg * a.v_page + r * a.v_row + hk * a.v_head;
#pragma unroll
      for (int c = 0; c < 2; ++c)
        if (lane + c * kWave < a.d_v) acc[c] = fmaf(pj, value_of<BF16>(vp[lane + c * kWave]), acc[c]);
    }
  }
  for (int m = 1; m < kWave; m *= 2) sum += __shfl_xor(sum, m);
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
  for (int c = 0; c < 2; ++c)
    if (lane + c * kWave < a.d_v)
      a.out[item * a.d_v + lane + c * kWave] = static_cast<uint16_t>(pack2<BF16>(acc[c] * inv, 0.f));
}

}  // namespace
}  // namespace lk

using namespace lk;

extern "C" {

int64_t lk_attention_paged_workspace(int64_t rows, int64_t sequences, int64_t capacity,
                                     int64_t heads, int64_t kv_heads, int64_t d_qk, int64_t d_v) {
  if (rows < 0 || sequences <= 0 || capacity < 0 || heads <= 0 || kv_heads <= 0 ||
      heads % kv_heads || d_qk <= 0 || d_v <= 0 || d_qk > kPagedMaxQk || d_v > kPagedMaxV)
    return -1;
  return 0;
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
  LK_REQUIRE(d_qk > 0 && d_qk % 8 == 0 && d_qk <= kPagedMaxQk,
             "attention d_qk must be a multiple of 8 up to %d, got %lld", kPagedMaxQk,
             (long long)d_qk);
  LK_REQUIRE(d_v > 0 && d_v % 8 == 0 && d_v <= kPagedMaxV,
             "attention d_v must be a multiple of 8 up to %d, got %lld", kPagedMaxV,
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
  const float scale_log2 = fabsf(scale) * 1.4426950408889634f;
  LK_REQUIRE(scale_log2 < INFINITY, "the attention scale must be finite, below 2^127");
  if (rows == 0) return LK_OK;
  LK_REQUIRE(q && out && lengths && (table_width == 0 || page_table) &&
                 (pages == 0 || (k_pages && v_pages)),
             "null pointer argument");
  for (const void* p : {q, k_pages, v_pages, static_cast<const void*>(out)})
    LK_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0,
               "attention tensors must start on a 16-byte boundary");
  const int64_t blocks = (rows * heads + kPagedWaves - 1) / kPagedWaves;
  LK_REQUIRE(grid_fits(blocks, kPagedThreads), "too many query rows and heads for one call");
  PagedArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k_pages);
  a.v = static_cast<const uint16_t*>(v_pages);
  a.out = static_cast<uint16_t*>(out);
  a.sq = Sequences{cu, rows, rows / sequences, static_cast<int>(sequences)};
  a.table = PageTable{page_table, lengths, table_stride, pages, static_cast<int>(table_width),
                      static_cast<int>(page_rows)};
  a.q_row = q_row_stride, a.q_head = q_head_stride;
  a.k_page = k_page, a.k_row = k_page_row, a.k_head = k_page_head;
  a.v_page = v_page, a.v_row = v_page_row, a.v_head = v_page_head;
  a.heads = static_cast<int>(heads), a.group = static_cast<int>(heads / kv_heads);
  a.d_qk = static_cast<int>(d_qk), a.d_v = static_cast<int>(d_v);
  a.scale_log2 = scale * 1.4426950408889634f;
  const hipStream_t s = as_stream(stream);
  const dim3 grid(static_cast<unsigned>(blocks));
  if (dtype == LK_DTYPE_BF16) paged_rows_kernel<true><<<grid, kPagedThreads, 0, s>>>(a);
  else paged_rows_kernel<false><<<grid, kPagedThreads, 0, s>>>(a);
  return check_launch("lk_attention_paged");
}

}  // extern "C"
