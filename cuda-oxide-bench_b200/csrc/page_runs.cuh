// page_runs.cuh — which entries of a list of page copies (src[i] -> dst[i]) share a
// read.  Plain C++, so that a host program can walk a list as the kernel does.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define GDN_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define GDN_HOST_DEVICE inline
#endif

namespace gdn {

constexpr int kRun = 8;  // copies of one source that are written with one read

// The entry after j in its run (side by side, of one source, up to kRun), -1 at its end.
GDN_HOST_DEVICE int64_t run_next(const int32_t* src, int64_t pairs, int64_t j) {
  return j + 1 < pairs && (j + 1) % kRun && src[j + 1] == src[j] ? j + 1 : -1;
}

// -1: entry i reads nothing; else it reads its source for itself and the rest of its
// run, of which the result is the first entry that has a destination.  A negative
// destination marks an entry that the plan has left out, whose source may lie outside
// the pool: a source is read only if an entry with a destination wants it.
GDN_HOST_DEVICE int64_t run_first(const int32_t* src, const int32_t* dst, int64_t pairs, int64_t i) {
  if (src[i] < 0 || (i % kRun && src[i - 1] == src[i])) return -1;
  int64_t j = i;
  while (j >= 0 && dst[j] < 0) j = run_next(src, pairs, j);
  return j;
}

}  // namespace gdn
