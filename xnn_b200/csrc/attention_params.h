// Launch parameters of the structure-attention kernels.
#pragma once
#include <stdint.h>

namespace attn {

// everything a launch needs; rows of q-like tensors are (N, H, D), of k-like ones (N, HK, D), any strides
// but a contiguous last dimension
template <typename T>
struct Params {
  const T *q, *k, *v, *o, *go;       // inputs, forward output, its cotangent
  const T *ca, *cb, *cc;             // cotangents of dq, dk, dv (second derivative)
  int64_t qs, ks, vs, os, gos, cas, cbs, ccs;      // row strides
  int64_t qh, kh, vh, oh, goh, cah, cbh, cch;      // head strides
  const int64_t* ptr;
  const uint8_t* mask;               // 1 where an atom may be attended to, or null
  T *out0, *out1, *out2, *out3;      // contiguous outputs
  T *lse, *delta;                    // (H, N) row statistics
  T *work, *work_k;                  // partial results of split passes: over keys, over queries
  T scale;
  int N, num, H, HK, D, splits, splits_k;
  int min_len, max_len;              // the lengths that this launch takes (others return at once)
  int rest;                          // whether it takes the rows of no structure too
  int compact;                       // only structures of more than 32 atoms, blocks numbered by windows of 32 rows
};

}  // namespace attn
