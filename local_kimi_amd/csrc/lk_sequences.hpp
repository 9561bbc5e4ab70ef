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

// The tile with this number; called by whole waves. The last s of 0..count with
// begin(s) / tile + s <= number, 64 candidates at a time, a lane each (one load's
// latency for up to 63 sequences). Offsets that decrease give some s of that range
// and perhaps a number before its first.
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
  return {lo, t < 0 ? 0 : t};
}

// The same tiles from the longest down: rank 0 is a last tile of the sequence with
// the most, ties go by sequence, and the rows behind the last sequence come at
// the end. A tile whose cost grows with its place in its sequence is best
// started first. For up to 63 sequences, whose rows the wave's lanes hold (`own`
// of lane s: those of sequence s, of lane count: the ones behind the last);
// called by whole waves. Sequence -1 where there are fewer tiles (of fewer than
// sequence_tiles()).
__device__ inline SequenceTile find_longest_tile(const RowRange& own, int count, int64_t rank,
                                                 int tile) {
  const int lane = static_cast<int>(threadIdx.x & 63);
  const int tiles = static_cast<int>((own.end - own.begin + tile - 1) / tile);
  const int mine = lane < count ? tiles : 0;
  int most = mine;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int other = __shfl_xor(most, m);
    most = other > most ? other : most;
  }
  int64_t left = rank;
  for (int t = __builtin_amdgcn_readfirstlane(most) - 1; t >= 0; --t) {
    const uint64_t have = __ballot(mine > t);
    const int n = __popcll(have);
    if (left < n) {
      uint64_t rest = have;
      for (int i = 0; i < static_cast<int>(left); ++i) rest &= rest - 1;
      return {__ffsll(static_cast<unsigned long long>(rest)) - 1, t};
    }
    left -= n;
  }
  const int behind = __builtin_amdgcn_readlane(tiles, count);
  return left < behind ? SequenceTile{count, left} : SequenceTile{-1, 0};
}

// What a lane of the wave holds (rows are below 2^31).
__device__ inline RowRange lane_rows(const RowRange& own, int lane) {
  return {__builtin_amdgcn_readlane(static_cast<int>(own.begin), lane),
          __builtin_amdgcn_readlane(static_cast<int>(own.end), lane)};
}

}  // namespace lk
