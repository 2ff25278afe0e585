// Tiles of ragged rows, shared by the kernels that work on CSR-pointed sequences.
#pragma once

#include "common.h"

namespace hy {

// Tile numbers go by sequence without a table of them: sequence e's tiles start at number
// start(e) / T + e.  ceil(len / T) <= end / T - start / T + 1, so they never meet the next
// sequence's, the numbers grow with e, and N / T + S + 2 of them cover everything: a launch
// depends on shapes alone.  e = 0 are the rows before the first sequence and e = S + 1 those
// behind the last (both without keys); a tile number between is a tile without rows.
struct Tile {
  int seq;         // -1: rows of no sequence
  int start, end;  // rows of the tile (of `size` at most); start >= end: none
};

__device__ __forceinline__ int ptr_at(const int* ptr, int S, int N, int e) {  // e in [0, S + 2]
  if (e == 0) return 0;
  if (e == S + 2) return N;
  return min(max(ptr[e - 1], 0), N);
}

__host__ __device__ inline int64_t tile_count(int64_t N, int64_t S, int size) { return N / size + S + 2; }

__device__ __forceinline__ Tile find_tile(const int* ptr, int S, int N, int size, int number) {
  const int lane = lane_id();
  int lo = 0, n = S + 2;
  while (n > 1) {  // the last e with start(e) / size + e <= number, 64 candidates at a time
    const int step = (n + 63) >> 6;
    const int e = lo + lane * step;
    const bool le = lane * step < n && ptr_at(ptr, S, N, min(e, S + 1)) / size + e <= number;
    const int sel = max(__popcll(__ballot(le)) - 1, 0);
    lo += sel * step;
    n = min(step, n - sel * step);
  }
  const int s0 = ptr_at(ptr, S, N, lo), s1 = max(ptr_at(ptr, S, N, lo + 1), s0);
  Tile t;
  t.seq = lo >= 1 && lo <= S ? lo - 1 : -1;
  const int64_t off = number - (s0 / size + lo), at = s0 + off * size;
  t.start = off >= 0 && at < s1 ? (int)at : s1;  // (off < 0: pointers that do not ascend)
  t.end = min(s1 - t.start, size) + t.start;
  t.seq = __builtin_amdgcn_readfirstlane(t.seq);
  t.start = __builtin_amdgcn_readfirstlane(t.start);
  t.end = __builtin_amdgcn_readfirstlane(t.end);
  return t;
}

}  // namespace hy
