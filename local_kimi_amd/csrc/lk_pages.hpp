// Cached sequences in pages (paged_cache.hip, paged_attention.hip), and the
// conversions of the 16-bit types that the attention kernels share.
#pragma once

#include <initializer_list>

#include "lk_common.hpp"
#include "lk_sequences.hpp"

namespace lk {

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

template <bool BF16>
__device__ inline float value_of(uint32_t x) {
  if constexpr (BF16) return bf16_to_f32(static_cast<uint16_t>(x));
  else return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(x)));
}

struct PageTable {
  const int32_t* pages_of;  // [sequences, width], rows `stride` apart
  const int32_t* lengths;
  int64_t stride, pages;
  int width, page_rows;
};

// The position of the first of sequence s's n new rows (below 0: it has no place), whatever the
// table can name: the last rows of a length beyond it have no place, the others keep theirs.
__device__ inline int64_t positions_before(const PageTable& t, int s, int64_t n) {
  const int64_t length = t.lengths[s];
  return (length < 0 ? 0 : length) - n;
}

// Positions of sequence s, its new ones among them: within what its row of the table can name.
__device__ inline int64_t cached_length(const PageTable& t, int s) {
  const int64_t n = t.lengths[s], most = static_cast<int64_t>(t.width) * t.page_rows;
  return n < 0 ? 0 : (n > most ? most : n);
}

// The sequence of row t, `count` behind the last one; called by whole waves with one
// t. The last s of 0..count that begins at or before t, 64 candidates at a time.
__device__ inline int find_sequence(const Sequences& q, int64_t t) {
  if (!q.cu) return static_cast<int>(t / q.length);
  const int lane = static_cast<int>(threadIdx.x & 63);
  int lo = 0, span = q.count + 1;
  while (span > 1) {
    const int step = (span + 63) / 64, off = lane * step, at = lo + (off < span ? off : 0);
    const int n = __popcll(__ballot(off < span && sequence_begin(q, at) <= t));
    const int skip = n > 0 ? (n - 1) * step : 0;
    lo += skip;
    span = span - skip < step ? span - skip : step;
  }
  return lo;
}

constexpr int kPageStep = 16;  // a page is a multiple of this many rows

// What the entry points that take a cache ask of it.
inline int check_pages(int64_t sequences, int64_t rows, bool offsets, int64_t pages,
                       int64_t page_rows, int64_t table_width, int64_t table_stride,
                       std::initializer_list<int64_t> strides) {
  LK_REQUIRE(sequences > 0 && sequences < (int64_t{1} << 24), "sequences must be in 1 .. 2^24 - 1");
  LK_REQUIRE(offsets || rows % sequences == 0,
             "without offsets the rows must divide into equal sequences");
  LK_REQUIRE(pages >= 0 && pages < (int64_t{1} << 31), "pages must be in 0 .. 2^31 - 1");
  LK_REQUIRE(page_rows > 0 && page_rows % kPageStep == 0 && page_rows <= 65536,
             "page rows must be a multiple of %d up to 65536, got %lld", kPageStep,
             (long long)page_rows);
  LK_REQUIRE(table_width >= 0 && table_width < (int64_t{1} << 31) &&
                 table_width * page_rows <= (int64_t{1} << 30) && table_stride >= table_width,
             "the page table must name up to 2^30 positions a sequence");
  for (const int64_t s : strides)
    LK_REQUIRE(s >= 0 && s % 8 == 0, "page strides must be multiples of 8 elements, not negative");
  return LK_OK;
}

}  // namespace lk
