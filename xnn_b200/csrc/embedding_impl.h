// Which table elements the output elements of the lookup take: shared by the kernel (embedding.cu) and a host check of
// every address.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define XNN_EMB_HD __host__ __device__ __forceinline__
#else
#define XNN_EMB_HD inline
#endif

// the table row of entry n, -1 where its id is outside the table
template <typename I>
XNN_EMB_HD int64_t row_of(const I* ids, int64_t n, int64_t V) {
  const int64_t v = (int64_t)ids[n];
  return v >= 0 && v < V ? v : -1;
}

// take(e, v, c) for the W output elements from e0 on, whatever rows of C they are of: element c of table row v, or v = -1
// where the id is outside the table. WHOLE: all W exist; otherwise it ends with the last of the `items` elements, behind
// which there is neither an id nor a row to step to.
template <int W, bool WHOLE, typename I, typename F>
XNN_EMB_HD void walk_elements(uint32_t e0, uint32_t items, uint32_t C, int64_t V, const I* ids, F&& take) {
  uint32_t n = e0 / C, c = e0 - n * C;
  int64_t v = row_of(ids, n, V);
#ifdef __CUDACC__
#pragma unroll
#endif
  for (int e = 0; e < W; ++e) {
    if (WHOLE || e0 + e < items) take(e, v, c);
    if (++c == C && e0 + e + 1 < items) {
      c = 0;
      v = row_of(ids, ++n, V);
    }
  }
}
