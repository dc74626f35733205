// Visibility of sliding-window attention with kept first tokens: position i sees j <= i if i - j < window or j < keep_first;
// window 0: every j <= i. The visible keys are two ranges, [0, kept) and [first, i], that do not overlap.
#pragma once
#include "common.cuh"

struct WindowRange {
  int kept, first;
};

__host__ __device__ __forceinline__ WindowRange window_range(int i, int window, int keep_first) {
  const int first = window > 0 && i >= window ? i - window + 1 : 0;
  return {keep_first < first ? keep_first : first, first};
}

// Sequences that leave their first positions in another slot's cache (null pointers: none does). Nobody shares more than both hold
// before the portion, so nothing that a launch appends is among what it reads as shared.
struct SharedPrefix {
  const int *lead, *shared;
};

// whether the real rows of a portion of T rows at position pos fit the cache
__device__ __forceinline__ bool window_fits(int pos, int count, int T, int Smax) { return pos >= 0 && pos <= Smax - min(count, T); }

// how many positions of sequence b, at position pos, are those of `lead` (which is set to b where there are none)
__device__ __forceinline__ int shared_edge(const SharedPrefix& s, const int* pos_of, int b, int pos, int batch, int& lead) {
  lead = s.lead[b];
  int e = min(s.shared[b], pos);
  if (lead < 0 || lead >= batch) e = 0;
  else e = min(e, pos_of[lead]);
  if (e <= 0) lead = b;
  return max(e, 0);
}
