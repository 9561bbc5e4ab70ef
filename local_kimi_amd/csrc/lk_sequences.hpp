// Packed sequences of the prompt kernels (kda_prefill.hip, attention.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lk {

// `count` sequences over `rows` rows: row cu[s] to cu[s + 1] - 1 of sequence s,
// or without offsets equal sequences of rows / count. Offsets start with 0 and
// do not decrease. They are read on the device and clamped to the rows (a
// decreasing pair is an empty sequence), so that no offset leads outside the
// tensors; what other offsets give is left open.
struct Sequences {
  const int32_t* cu;
  int64_t rows;
  int64_t length;  // of equal sequences
  int count;
};

// Whether a launch takes this many blocks: the threads of a grid are counted in 32 bits.
inline bool grid_fits(int64_t blocks, int64_t threads) {
  return blocks < (int64_t{1} << 31) && blocks * threads < (int64_t{1} << 32);
}

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

// The tile with this number; called by whole waves. The last s of 0..count with
// begin(s) / tile + s <= number, 64 candidates at a time, a lane each (one load's
// latency for up to 63 sequences). Sequence -1 for a number before the found
// one's first, which only offsets that decrease or do not start with 0 give.
__device__ inline SequenceTile find_sequence_tile(const Sequences& q, int64_t number, int tile) {
  const int lane = static_cast<int>(threadIdx.x & 63);
  int lo = 0, span = q.count + 1;
  while (span > 1) {
    const int step = (span + 63) / 64, off = lane * step, at = lo + (off < span ? off : 0);
    const bool before = off < span && sequence_begin(q, at) / tile + at <= number;
    const int n = __popcll(__ballot(before));
    const int skip = n > 0 ? (n - 1) * step : 0;
    lo += skip;
    span = span - skip < step ? span - skip : step;
  }
  const int64_t t = number - (sequence_begin(q, lo) / tile + lo);
  return {t < 0 ? -1 : lo, t};
}

}  // namespace lk
