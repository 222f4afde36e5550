// Index arithmetic of the paged cache, shared by the kernels and by the host
// (where the tests run it).
#pragma once

#include <cstdint>

namespace fa {

// First row of sequence b among the T packed rows, and the first behind it.
// Boundaries are held to [0, T] and to rising order, so that no kernel indexes
// outside the packed tensors whatever the array holds.
struct SeqRows {
  int begin, end;
};
__host__ __device__ __forceinline__ SeqRows seq_rows(const int32_t* cu, int b, int T) {
  SeqRows r;
  if (cu == nullptr) {
    r.begin = b;
    r.end = b + 1;
    return r;
  }
  const int lo = cu[b], hi = cu[b + 1];
  r.begin = lo < 0 ? 0 : (lo > T ? T : lo);
  r.end = hi < r.begin ? r.begin : (hi > T ? T : hi);
  return r;
}

// Sequence that row t belongs to (the last b with cu[b] <= t), or -1.  A search by
// 32 probes at a time: count(lo, step, hi) is the number of the probes lo + step,
// lo + 2 step, ... (32 of them, those below hi) with cu[probe] <= t.
template <typename Count>
__host__ __device__ __forceinline__ int seq_of_row(const int32_t* cu, int B, int t, Count count) {
  if (cu == nullptr) return t < B ? t : -1;
  const int below = cu[0], above = cu[B];
  int lo = 0, hi = B;                 // cu[lo] <= t < cu[hi]
  while (hi - lo > 1) {
    const int step = (hi - lo - 1 + 31) / 32;
    const int n = count(lo, step, hi);
    if (hi - lo > (n + 1) * static_cast<int64_t>(step)) hi = lo + (n + 1) * step;
    lo += n * step;
  }
  return t < below || t >= above ? -1 : lo;
}

// Page of key `place` of a sequence with this table row: -1 where the place lies
// outside the table or the entry outside the cache.
__host__ __device__ __forceinline__ int page_at(const int32_t* row, int place, int page_shift,
                                                int max_pages, int pages) {
  if (place < 0 || (place >> page_shift) >= max_pages) return -1;
  const int page = row[place >> page_shift];
  return page >= 0 && page < pages ? page : -1;
}

// A sequence's length as far as its table goes.
__host__ __device__ __forceinline__ int held_len(int len, int page_shift, int max_pages) {
  const int64_t cap = static_cast<int64_t>(max_pages) << page_shift;
  if (len < 0) return 0;
  return len > cap ? static_cast<int>(cap) : len;
}

}  // namespace fa
