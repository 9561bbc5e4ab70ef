// Packed sequences of the prompt kernels (kda_prefill.hip, attention.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lk {

// `count` sequences over `rows` rows: row cu[s] to cu[s + 1] - 1 of sequence s,
// or without offsets equal sequences of rows / count. Offsets are read on the
// device and clamped to the rows (a decreasing pair is an empty sequence), so
// no offset leads outside the tensors.
struct Sequences {
  const int32_t* cu;
  int64_t rows;
  int64_t length;  // of equal sequences
  int count;
};

struct RowRange {
  int64_t begin, end;
};

__device__ inline int64_t sequence_begin(const Sequences& q, int s) {
  if (!q.cu) return static_cast<int64_t>(s) * q.length;
  const int64_t at = q.cu[s];
  return at < 0 ? 0 : (at > q.rows ? q.rows : at);
}

// The rows of sequence s; s = count: the rows behind the last one.
__device__ inline RowRange sequence_rows(const Sequences& q, int s) {
  const int64_t begin = sequence_begin(q, s);
  const int64_t end = s < q.count ? sequence_begin(q, s + 1) : q.rows;
  return {begin, end < begin ? begin : end};
}

// Tiles of `tile` rows that never span two sequences, numbered without a table:
// tile t of sequence s has number begin(s) / tile + s + t. A sequence of n rows
// at b needs ceil(n / tile) <= (b + n) / tile - b / tile + 1 numbers, which is
// what lies between its first number and the next one's, so the numbers are
// distinct, every sequence has one at least, and sequence_tiles() bounds them
// from the sizes alone: no offset is read on the host and no launch builds a
// list. The rows behind the last sequence count as one more sequence.
inline int64_t sequence_tiles(int64_t rows, int64_t count, int64_t tile) {
  return rows / tile + count + 1;
}

struct SequenceTile {
  int sequence;
  int64_t tile;
};

__device__ inline SequenceTile find_sequence_tile(const Sequences& q, int64_t number, int tile) {
  int lo = 0, hi = q.count;  // the last s of 0..count with begin(s) / tile + s <= number
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (sequence_begin(q, mid) / tile + mid <= number)
      lo = mid;
    else
      hi = mid - 1;
  }
  // decreasing offsets can name a number before the sequence's first
  const int64_t t = number - (sequence_begin(q, lo) / tile + lo);
  return {lo, t < 0 ? 0 : t};
}

}  // namespace lk
