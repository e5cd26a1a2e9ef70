// Softmax attention over the atoms of each structure of a packed batch, its backward pass and the backward pass of that:
// the formulas, the kernels of short structures on the FP32 / FP64 pipes (attention_tc*.cu and attention_f64.cu hold those of
// the long ones) and the joins of split walks. The matrix of probabilities never leaves the chip.
//
// With S = scale q k^T over the allowed keys of a row's structure (x = S log2 e, so that powers of two
// serve), P = softmax_row(S), O = P V:
//   forward   one pass over the keys with the running maximum m and sum l of each row; the row statistic
//             kept for later is L = m + log2 l, from which P = 2^(x - L) is formed again.
//   backward  D = do.o, dP = do V^T, dS = P (dP - D):  dq = scale dS K, dk = scale dS^T Q, dv = P^T do.
//   second    cotangents A, B, C of dq, dk, dv: T = scale (A K^T + Q B^T), E = do C^T, r = sum_j P T,
//             G = (T - r) (dP - D) + E, c = sum_j P G = sum_j P (T dP + E) - D r, M = P (G - c),
//             q' = scale (M K + dS B), k' = scale (M^T Q + dS^T A), v' = (P (T - r))^T do,
//             do' = P (T - r) V + P C.
// Row-owning blocks write dq, q', do' and key-owning ones dk, dv, k', v': every sum has a fixed order
// and there are no atomics. Statistics and accumulators have the operands' type (32 or 64 bits).
#include "attention.h"
#include "attention_tile.cuh"

namespace attn {
namespace {

template <typename T, int BQ_, int BK_, int DP_, int RI_, int TX_>
struct Cfg {
  static constexpr int BQ = BQ_, BK = BK_, DP = DP_, RI = RI_, TX = TX_;
  static constexpr int RJ = BK / TX, NT = BQ / RI * TX, W = Vec<T>::W;
  static constexpr int LD = DP + W, LDP = BK + W;
};

__device__ __forceinline__ bool allowed(int j, int hi, const uint8_t* mask) {
  return j < hi && (mask == nullptr || mask[j]);
}

// a masked key's gradients are zero whatever its queries hold (0 NaN is NaN)
template <typename T, int N>
__device__ __forceinline__ void hide(T (&a)[N], T (&b)[N], bool hidden) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    a[n] = hidden ? T(0) : a[n];
    b[n] = hidden ? T(0) : b[n];
  }
}

// ------------------------------------------------------------------------------------------ forward
template <typename T, typename C>
__global__ void __launch_bounds__(C::NT) fwd_kernel(const Params<T> p) {
  extern __shared__ __align__(16) char smem_raw[];
  T* sQ = reinterpret_cast<T*>(smem_raw);
  T* sK = sQ + C::BQ * C::LD;
  T* sV = sK + C::BK * C::LD;
  T* sP = sV + C::BK * C::LD;
  Part part;
  if (!find_part<C::BQ>(p, blockIdx.x, part)) return;
  const int h = blockIdx.y, hk = h / (p.H / p.HK);
  const int tx = threadIdx.x % C::TX, i0 = threadIdx.x / C::TX * C::RI;
  const T *gq = p.q + h * p.qh, *gk = p.k + hk * p.kh, *gv = p.v + hk * p.vh;
  const bool vq = vec_ok(p.q, p.qs, p.qh, p.D), vk = vec_ok(p.k, p.ks, p.kh, p.D), vv = vec_ok(p.v, p.vs, p.vh, p.D);
  const int k_lo = part.lo, k_hi = part.keys ? part.hi : part.lo;
  const T c2 = p.scale * log2e<T>();
  T m[C::RI], l[C::RI], acc[C::RI][C::DP / C::TX];
#pragma unroll
  for (int r = 0; r < C::RI; ++r) {
    m[r] = neg_inf<T>();
    l[r] = T(0);
#pragma unroll
    for (int n = 0; n < C::DP / C::TX; ++n) acc[r][n] = T(0);
  }
  if (k_lo < k_hi) load_tile<T, C::BQ, C::DP, C::LD, C::NT>(sQ, gq, p.qs, part.row, part.hi, p.D, vq);
  for (int k0 = k_lo; k0 < k_hi; k0 += C::BK) {
    load_tile<T, C::BK, C::DP, C::LD, C::NT>(sK, gk, p.ks, k0, k_hi, p.D, vk, p.mask);
    load_tile<T, C::BK, C::DP, C::LD, C::NT>(sV, gv, p.vs, k0, k_hi, p.D, vv, p.mask);
    __syncthreads();
    T s[C::RI][C::RJ] = {};
    tile_nt<T, C::RI, C::RJ, C::TX, C::DP, C::LD>(s, sQ, i0, sK, tx);
    bool ok[C::RJ];
#pragma unroll
    for (int c = 0; c < C::RJ; ++c) ok[c] = allowed(k0 + tx + C::TX * c, k_hi, p.mask);
#pragma unroll
    for (int r = 0; r < C::RI; ++r) {
      T top = neg_inf<T>();
#pragma unroll
      for (int c = 0; c < C::RJ; ++c) {
        s[r][c] = ok[c] ? s[r][c] * c2 : neg_inf<T>();
        top = s[r][c] > top ? s[r][c] : top;
      }
      top = row_max<C::TX>(top);
      const T mn = top > m[r] ? top : m[r];
      const T base = mn == neg_inf<T>() ? T(0) : mn;       // a row without a key yet: 2^(-inf - 0) = 0
      const T f = pow2(m[r] - base);
      T sum = T(0);
#pragma unroll
      for (int c = 0; c < C::RJ; ++c) {
        const T e = pow2(s[r][c] - base);
        sum += e;
        sP[(i0 + r) * C::LDP + tx + C::TX * c] = e;
      }
      l[r] = l[r] * f + row_sum<C::TX>(sum);
      m[r] = mn;
#pragma unroll
      for (int n = 0; n < C::DP / C::TX; ++n) acc[r][n] *= f;
    }
    __syncthreads();
    tile_nn<T, C::RI, C::BK, C::TX, C::DP, C::LDP, C::LD>(acc, sP, i0, sV, tx, k_hi - k0);
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < C::RI; ++r) {
    const int row = part.row + i0 + r;
    if (row >= part.hi) continue;
    const bool none = m[r] == neg_inf<T>() && l[r] == T(0);   // NaN scores are not an empty row
    store_row<T, C::DP, C::TX>(p.out0 + ((int64_t)row * p.H + h) * p.D, acc[r], none ? T(0) : T(1) / l[r], p.D, tx);
    if (tx == 0 && p.lse) p.lse[(int64_t)h * p.N + row] = none ? -neg_inf<T>() : m[r] + lg2(l[r]);
  }
}

// Joins the splits of a row, a warp per (row, head): the lanes fetch the splits' statistics at once (at most 32
// splits), then the partial rows, whose loads do not depend on one another.
template <typename T>
__global__ void __launch_bounds__(128) join_kernel(const Params<T> p) {
  const int64_t i = (int64_t)blockIdx.x * 4 + threadIdx.x / 32, rows = (int64_t)p.H * p.N;
  const int lane = threadIdx.x % 32;
  if (i >= rows) return;
  const int h = (int)(i % p.H), row = (int)(i / p.H);
  const T* stats = p.work + p.splits * rows * p.D;
  const int64_t at = (int64_t)h * p.N + row;
  const bool in = lane < p.splits;
  const T mz = in ? stats[lane * rows + at] : neg_inf<T>(), lz = in ? stats[(p.splits + lane) * rows + at] : T(0);
  const T m = row_max<32>(mz), base = m == neg_inf<T>() ? T(0) : m;
  const T f = pow2(mz - base), l = row_sum<32>(in ? f * lz : T(0));
  const bool none = m == neg_inf<T>() && l == T(0);
  for (int d = lane; d - lane < p.D; d += 32) {
    T a = T(0);
#pragma unroll 4
    for (int z = 0; z < p.splits; ++z) {
      const T g = __shfl_sync(0xffffffffu, f, z);
      if (d < p.D) a += g * p.work[(z * rows + at) * p.D + d];
    }
    if (d < p.D) p.out0[((int64_t)row * p.H + h) * p.D + d] = none ? T(0) : a / l;
  }
  if (lane == 0 && p.lse) p.lse[at] = none ? -neg_inf<T>() : m + lg2(l);
}

// out[i] = sum of the splits' partial results in their order, for one result or two whose splits follow each other
template <typename T>
__global__ void __launch_bounds__(256) sum_kernel(int64_t n, int splits, const T* __restrict__ work, T* __restrict__ out0,
                                                  T* __restrict__ out1) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  work += blockIdx.y * splits * n;
  T a = T(0);
#pragma unroll 4
  for (int z = 0; z < splits; ++z) a += work[z * n + i];
  (blockIdx.y ? out1 : out0)[i] = a;
}

// ------------------------------------------------------------------------------------------ backward
// structures of at most BQ atoms: one block holds the whole probability matrix of a head, so that the
// softmax is formed at once (neither the forward output nor its statistics are read) and dq, dk, dv
// come from one launch and one reading of the inputs (4000 structures of 8-31 atoms x 4 heads x 64: 505 us)
template <typename T, typename C>
__global__ void __launch_bounds__(C::NT) bwd_short_kernel(const Params<T> p) {
  static_assert(C::BQ == C::BK, "square tiles");
  extern __shared__ __align__(16) char smem_raw[];
  T* sK = reinterpret_cast<T*>(smem_raw);
  T* sV = sK + C::BQ * C::LD;
  T* sQ = sV + C::BQ * C::LD;
  T* sO = sQ + C::BK * C::LD;
  T* sP = sO + C::BK * C::LD;
  T* sS = sP + C::BQ * C::LDP;
  Part part;
  if (!find_part<C::BQ>(p, blockIdx.x, part)) return;
  const int hk = blockIdx.y, group = p.H / p.HK;
  const int tx = threadIdx.x % C::TX, i0 = threadIdx.x / C::TX * C::RI;
  const T c2 = p.scale * log2e<T>();
  const bool keys = part.keys;
  // a structure longer than the caller's bound on the lengths: its gradients are not formed, say so
  const T good = keys && part.hi - part.lo > C::BQ ? std::numeric_limits<T>::quiet_NaN() : T(1);
  T dk[C::RI][C::DP / C::TX] = {}, dv[C::RI][C::DP / C::TX] = {};
  if (keys) {
    load_tile<T, C::BQ, C::DP, C::LD, C::NT>(sK, p.k + hk * p.kh, p.ks, part.row, part.hi, p.D, vec_ok(p.k, p.ks, p.kh, p.D), p.mask);
    load_tile<T, C::BQ, C::DP, C::LD, C::NT>(sV, p.v + hk * p.vh, p.vs, part.row, part.hi, p.D, vec_ok(p.v, p.vs, p.vh, p.D), p.mask);
  }
  for (int g = 0; g < group; ++g) {
    const int h = hk * group + g;
    T dq[C::RI][C::DP / C::TX] = {};
    if (keys) {
      load_tile<T, C::BK, C::DP, C::LD, C::NT>(sQ, p.q + h * p.qh, p.qs, part.row, part.hi, p.D, vec_ok(p.q, p.qs, p.qh, p.D));
      load_tile<T, C::BK, C::DP, C::LD, C::NT>(sO, p.go + h * p.goh, p.gos, part.row, part.hi, p.D, vec_ok(p.go, p.gos, p.goh, p.D));
      __syncthreads();
      T s[C::RI][C::RJ] = {}, dp[C::RI][C::RJ] = {};
      tile_nt<T, C::RI, C::RJ, C::TX, C::DP, C::LD>(s, sQ, i0, sK, tx);
      tile_nt<T, C::RI, C::RJ, C::TX, C::DP, C::LD>(dp, sO, i0, sV, tx);
      bool ok[C::RJ];
#pragma unroll
      for (int c = 0; c < C::RJ; ++c) ok[c] = allowed(part.row + tx + C::TX * c, part.hi, p.mask);
#pragma unroll
      for (int r = 0; r < C::RI; ++r) {
        T top = neg_inf<T>();
#pragma unroll
        for (int c = 0; c < C::RJ; ++c) {
          s[r][c] = ok[c] ? s[r][c] * c2 : neg_inf<T>();
          top = s[r][c] > top ? s[r][c] : top;
        }
        top = row_max<C::TX>(top);
        const T base = top == neg_inf<T>() ? T(0) : top;
        T sum = T(0);
#pragma unroll
        for (int c = 0; c < C::RJ; ++c) { s[r][c] = pow2(s[r][c] - base); sum += s[r][c]; }
        sum = row_sum<C::TX>(sum);
        const T inv = (top == neg_inf<T>() && sum == T(0)) || part.row + i0 + r >= part.hi ? T(0) : T(1) / sum;
        T D = T(0);
#pragma unroll
        for (int c = 0; c < C::RJ; ++c) {
          s[r][c] = ok[c] ? s[r][c] * inv : T(0);
          dp[r][c] = ok[c] ? dp[r][c] : T(0);
          D += s[r][c] * dp[r][c];
        }
        D = row_sum<C::TX>(D);
#pragma unroll
        for (int c = 0; c < C::RJ; ++c) {
          sP[(i0 + r) * C::LDP + tx + C::TX * c] = s[r][c];
          sS[(i0 + r) * C::LDP + tx + C::TX * c] = s[r][c] * (dp[r][c] - D);
        }
      }
      __syncthreads();
      tile_nn<T, C::RI, C::BK, C::TX, C::DP, C::LDP, C::LD>(dq, sS, i0, sK, tx, part.hi - part.row);
      tile_tn<T, C::RI, C::BK, C::TX, C::DP, C::LDP, C::LD>(dk, sS, i0, sQ, tx, part.hi - part.row);
      tile_tn<T, C::RI, C::BK, C::TX, C::DP, C::LDP, C::LD>(dv, sP, i0, sO, tx, part.hi - part.row);
      __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < C::RI; ++r) {
      const int row = part.row + i0 + r;
      if (row < part.hi) store_row<T, C::DP, C::TX>(p.out0 + ((int64_t)row * p.H + h) * p.D, dq[r], p.scale * good, p.D, tx);
    }
  }
#pragma unroll
  for (int r = 0; r < C::RI; ++r) {
    const int row = part.row + i0 + r;
    if (row >= part.hi) continue;
    hide(dk[r], dv[r], p.mask != nullptr && !p.mask[row]);
    const int64_t at = ((int64_t)row * p.HK + hk) * p.D;
    store_row<T, C::DP, C::TX>(p.out1 + at, dk[r], p.scale * good, p.D, tx);
    store_row<T, C::DP, C::TX>(p.out2 + at, dv[r], good, p.D, tx);
  }
}

// ------------------------------------------------------------------------------------------ second derivative
// Structures of at most BQ atoms, as in bwd_short_kernel: 12 products on a structure instead of the 22 of separate walks
// for do', q' and the keys, no statistics from memory. Four tiles of shared memory serve seven operands: q, k, A, B for the
// scores, do, v, C in place of the first three for the products with them, then q, k, A again (from L2), which keeps four
// blocks of 128 threads an SM at 64 columns. 64 structures of 9-30 atoms x 4 heads x 64: 25 us (80 in separate walks), 4000:
// 1.22 ms (3.91).
template <typename T, typename C>
__global__ void __launch_bounds__(C::NT) second_short_kernel(const Params<T> p) {
  static_assert(C::BQ == C::BK, "square tiles");
  extern __shared__ __align__(16) char smem_raw[];
  T* s0 = reinterpret_cast<T*>(smem_raw);
  T* s1 = s0 + C::BQ * C::LD;
  T* s2 = s1 + C::BQ * C::LD;
  T* sB = s2 + C::BQ * C::LD;
  T* sP = sB + C::BQ * C::LD;                            // P, P (T - r), M, P (dP - D)
  T* sT = sP + C::BQ * C::LDP;
  T* sM = sT + C::BQ * C::LDP;
  T* sS = sM + C::BQ * C::LDP;
  Part part;
  if (!find_part<C::BQ>(p, blockIdx.x, part)) return;
  const int hk = blockIdx.y, group = p.H / p.HK, used = part.hi - part.row;
  const int tx = threadIdx.x % C::TX, i0 = threadIdx.x / C::TX * C::RI;
  const T c2 = p.scale * log2e<T>();
  const bool keys = part.keys;
  const T good = keys && part.hi - part.lo > C::BQ ? std::numeric_limits<T>::quiet_NaN() : T(1);
  T dk[C::RI][C::DP / C::TX] = {}, dv[C::RI][C::DP / C::TX] = {};
  const auto tile = [&](T* to, const T* g, int64_t rs, int64_t hs, int head, const uint8_t* mask) {
    load_tile<T, C::BQ, C::DP, C::LD, C::NT>(to, g + head * hs, rs, part.row, part.hi, p.D, vec_ok(g, rs, hs, p.D), mask);
  };
  if (keys) tile(sB, p.cb, p.cbs, p.cbh, hk, p.mask);
  for (int g = 0; g < group; ++g) {
    const int h = hk * group + g;
    T dq[C::RI][C::DP / C::TX] = {}, dout[C::RI][C::DP / C::TX] = {};
    if (keys) {
      tile(s0, p.q, p.qs, p.qh, h, nullptr);
      tile(s1, p.k, p.ks, p.kh, hk, p.mask);
      tile(s2, p.ca, p.cas, p.cah, h, nullptr);
      __syncthreads();
      T s[C::RI][C::RJ] = {}, t[C::RI][C::RJ] = {}, dp[C::RI][C::RJ] = {}, e[C::RI][C::RJ] = {};
      tile_nt<T, C::RI, C::RJ, C::TX, C::DP, C::LD>(s, s0, i0, s1, tx);
      tile_nt<T, C::RI, C::RJ, C::TX, C::DP, C::LD>(t, s2, i0, s1, tx);
      tile_nt<T, C::RI, C::RJ, C::TX, C::DP, C::LD>(t, s0, i0, sB, tx);
      __syncthreads();
      tile(s0, p.go, p.gos, p.goh, h, nullptr);
      tile(s1, p.v, p.vs, p.vh, hk, p.mask);
      tile(s2, p.cc, p.ccs, p.cch, hk, p.mask);
      __syncthreads();
      tile_nt<T, C::RI, C::RJ, C::TX, C::DP, C::LD>(dp, s0, i0, s1, tx);
      tile_nt<T, C::RI, C::RJ, C::TX, C::DP, C::LD>(e, s0, i0, s2, tx);
      bool ok[C::RJ];
#pragma unroll
      for (int c = 0; c < C::RJ; ++c) ok[c] = allowed(part.row + tx + C::TX * c, part.hi, p.mask);
#pragma unroll
      for (int r = 0; r < C::RI; ++r) {
        T top = neg_inf<T>();
#pragma unroll
        for (int c = 0; c < C::RJ; ++c) {
          s[r][c] = ok[c] ? s[r][c] * c2 : neg_inf<T>();
          top = s[r][c] > top ? s[r][c] : top;
        }
        top = row_max<C::TX>(top);
        const T base = top == neg_inf<T>() ? T(0) : top;
        T sum = T(0);
#pragma unroll
        for (int c = 0; c < C::RJ; ++c) { s[r][c] = pow2(s[r][c] - base); sum += s[r][c]; }
        sum = row_sum<C::TX>(sum);
        const T inv = (top == neg_inf<T>() && sum == T(0)) || part.row + i0 + r >= part.hi ? T(0) : T(1) / sum;
        T D = T(0), R = T(0), U = T(0);
#pragma unroll
        for (int c = 0; c < C::RJ; ++c) {
          s[r][c] = ok[c] ? s[r][c] * inv : T(0);
          t[r][c] *= p.scale;
          D += ok[c] ? s[r][c] * dp[r][c] : T(0);
          R += ok[c] ? s[r][c] * t[r][c] : T(0);
          U += ok[c] ? s[r][c] * (t[r][c] * dp[r][c] + e[r][c]) : T(0);
        }
        D = row_sum<C::TX>(D);
        R = row_sum<C::TX>(R);
        U = row_sum<C::TX>(U) - D * R;
#pragma unroll
        for (int c = 0; c < C::RJ; ++c) {
          const int w = (i0 + r) * C::LDP + tx + C::TX * c;
          sP[w] = s[r][c];
          sT[w] = ok[c] ? s[r][c] * (t[r][c] - R) : T(0);
          sM[w] = ok[c] ? s[r][c] * ((t[r][c] - R) * (dp[r][c] - D) + e[r][c] - U) : T(0);
          sS[w] = ok[c] ? s[r][c] * (dp[r][c] - D) : T(0);
        }
      }
      __syncthreads();
      tile_nn<T, C::RI, C::BK, C::TX, C::DP, C::LDP, C::LD>(dout, sT, i0, s1, tx, used);
      tile_nn<T, C::RI, C::BK, C::TX, C::DP, C::LDP, C::LD>(dout, sP, i0, s2, tx, used);
      tile_tn<T, C::RI, C::BK, C::TX, C::DP, C::LDP, C::LD>(dv, sT, i0, s0, tx, used);
      __syncthreads();
      tile(s0, p.q, p.qs, p.qh, h, nullptr);
      tile(s1, p.k, p.ks, p.kh, hk, p.mask);
      tile(s2, p.ca, p.cas, p.cah, h, nullptr);
      __syncthreads();
      tile_nn<T, C::RI, C::BK, C::TX, C::DP, C::LDP, C::LD>(dq, sM, i0, s1, tx, used);
      tile_nn<T, C::RI, C::BK, C::TX, C::DP, C::LDP, C::LD>(dq, sS, i0, sB, tx, used);
      tile_tn<T, C::RI, C::BK, C::TX, C::DP, C::LDP, C::LD>(dk, sM, i0, s0, tx, used);
      tile_tn<T, C::RI, C::BK, C::TX, C::DP, C::LDP, C::LD>(dk, sS, i0, s2, tx, used);
      __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < C::RI; ++r) {
      const int row = part.row + i0 + r;
      if (row >= part.hi) continue;
      const int64_t at = ((int64_t)row * p.H + h) * p.D;
      store_row<T, C::DP, C::TX>(p.out0 + at, dq[r], p.scale * good, p.D, tx);
      store_row<T, C::DP, C::TX>(p.out3 + at, dout[r], good, p.D, tx);
    }
  }
#pragma unroll
  for (int r = 0; r < C::RI; ++r) {
    const int row = part.row + i0 + r;
    if (row >= part.hi) continue;
    hide(dk[r], dv[r], p.mask != nullptr && !p.mask[row]);
    const int64_t at = ((int64_t)row * p.HK + hk) * p.D;
    store_row<T, C::DP, C::TX>(p.out1 + at, dk[r], p.scale * good, p.D, tx);
    store_row<T, C::DP, C::TX>(p.out2 + at, dv[r], good, p.D, tx);
  }
}

// ------------------------------------------------------------------------------------------ launches
template <typename T, typename C, auto KERNEL>
cudaError_t launch(const Params<T>& p, int heads, int row_tiles, int key_tiles, int squares, cudaStream_t s) {
  const size_t bytes = sizeof(T) * ((size_t)row_tiles * C::BQ * C::LD + (size_t)key_tiles * C::BK * C::LD +
                                    (size_t)squares * C::BQ * C::LDP);
  const cudaError_t e = raise_smem_limit<KERNEL>(bytes);
  if (e != cudaSuccess) return e;
  const dim3 grid(part_blocks(p, C::BQ), heads);
  KERNEL<<<grid, C::NT, bytes, s>>>(p);
  return cudaGetLastError();
}

// The square tiles of 32 rows. float: a 2 x 4 corner of the scores a thread (one molecule of 21 atoms at 64 columns: 5 us with
// 128 threads, 9 with 64 and 4 x 4 corners; 4000 of 8-31 x 4 heads: 253 and 279 us, of 49 to move the data: reads of shared
// memory bound it). double: 2 x 2, since the accumulators of 4 x 4 alone would take 128 registers at 128 columns.
template <typename T, int DP> struct Small;
template <int DP> struct Small<float, DP> { using C = Cfg<float, 32, 32, DP, 2, 8>; };
template <int DP> struct Small<double, DP> { using C = Cfg<double, 32, 32, DP, 2, 16>; };
// the short backward pass at 128 float columns: 256 threads (2000 structures: 138 us against 186 with 128 threads). Corners of
// 4 x 4 read less of the tiles, but leave half the warps (64 columns, 4000 x 4 heads: 531 us against 505; 512 structures of one
// head: 27 and 23).
template <typename T, int DP> struct Short { using C = typename Small<T, DP>::C; };
template <> struct Short<float, 128> { using C = Cfg<float, 32, 32, 128, 2, 16>; };

#define XNN_ATTN_DIM(D_, ...)                            \
  if ((D_) <= 32) { constexpr int DP = 32; __VA_ARGS__; } \
  if ((D_) <= 64) { constexpr int DP = 64; __VA_ARGS__; } \
  { constexpr int DP = 128; __VA_ARGS__; }

}  // namespace

template <typename T>
cudaError_t forward(const Params<T>& p, cudaStream_t s) {
  XNN_ATTN_DIM(p.D, using C = typename Small<T, DP>::C; return (launch<T, C, fwd_kernel<T, C>>(p, p.H, 1, 2, 1, s)))
}
template <typename T>
cudaError_t forward_join(const Params<T>& p, cudaStream_t s) {
  const int64_t rows = (int64_t)p.H * p.N;
  join_kernel<T><<<(unsigned)((rows + 3) / 4), 128, 0, s>>>(p);
  return cudaGetLastError();
}
template <typename T>
cudaError_t sum_splits(int64_t n, int splits, const T* work, T* out0, T* out1, cudaStream_t s) {
  sum_kernel<T><<<dim3((unsigned)((n + 255) / 256), out1 ? 2 : 1), 256, 0, s>>>(n, splits, work, out0, out1);
  return cudaGetLastError();
}
template <typename T>
cudaError_t backward_short(const Params<T>& p, cudaStream_t s) {
  XNN_ATTN_DIM(p.D, using C = typename Short<T, DP>::C; return (launch<T, C, bwd_short_kernel<T, C>>(p, p.HK, 2, 2, 2, s)))
}
template <typename T>
cudaError_t second_short(const Params<T>& p, cudaStream_t s) {
  XNN_ATTN_DIM(p.D, using C = typename Small<T, DP>::C; return (launch<T, C, second_short_kernel<T, C>>(p, p.HK, 2, 2, 4, s)))
}

#define XNN_ATTN_INST(T)                                                                  \
  template cudaError_t forward<T>(const Params<T>&, cudaStream_t);                        \
  template cudaError_t forward_join<T>(const Params<T>&, cudaStream_t);                   \
  template cudaError_t sum_splits<T>(int64_t, int, const T*, T*, T*, cudaStream_t);       \
  template cudaError_t backward_short<T>(const Params<T>&, cudaStream_t);                 \
  template cudaError_t second_short<T>(const Params<T>&, cudaStream_t);
XNN_ATTN_INST(float)
XNN_ATTN_INST(double)

}  // namespace attn
