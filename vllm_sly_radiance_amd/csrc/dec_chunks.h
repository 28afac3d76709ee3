// The chunks of a batch's sequences: which slot has which rows, whatever the starts hold.
#pragma once
#include "dec_internal.h"

namespace dec {

// Chunk slots: sequence b's begin at starts[b] / 64 + b, so that total / 64 + batch slots hold all.
__device__ __forceinline__ int first_chunk(const Sequences& s, int b) {
  return min(max(s.starts[b], 0), s.total) / kChunk + b;
}

// The sequence that chunk slot c belongs to, the last whose slots begin at it or before (-1 for none), its first
// row and its number of rows.
__device__ __forceinline__ int sequence_of(const Sequences& s, int c, int& first, int& n) {
  const int lane = threadIdx.x & 63;
  int b = -1;
  for (int b0 = 0; b0 < s.batch; b0 += 64) {
    const int start = s.starts[min(b0 + lane, s.batch)];
    const int m = __popcll(__ballot(b0 + lane < s.batch && min(max(start, 0), s.total) / kChunk + b0 + lane <= c));
    b += m;
    if (m < 64 && m) {                  // its start and the next are here
      first = min(max(__builtin_amdgcn_readlane(start, m - 1), 0), s.total);
      n = min(max(__builtin_amdgcn_readlane(start, m), first), s.total) - first;
      return b;
    }
    if (m < 64) break;
  }
  if (b >= 0) rows_of(s, b, first, n);
  return b;
}

// The rows of chunk slot c: m of them from row0 on, all of one sequence; false where no sequence has it. (Where starts go
// back a slot may be taken for a sequence's whose own begin behind it. Rows are in [0, total) there too: those of the
// sequence and ones in front of it.)
__device__ __forceinline__ bool rows_of_chunk(const Sequences& s, int c, size_t& row0, int& m) {
  int first, n;
  const int b = sequence_of(s, c, first, n);
  if (b < 0) return false;
  const int i0 = (c - first / kChunk - b) * kChunk;
  m = min(n - i0, kChunk);
  row0 = (size_t)((long)first + i0);
  return i0 < n;
}

}  // namespace dec
