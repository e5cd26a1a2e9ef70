// Softmax attention over the atoms of each structure of a packed batch, its backward pass and the
// backward pass of that, on the FP32 / FP64 pipes; the matrix of probabilities never leaves the chip.
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
// D = do.o per row and head: a warp each
template <typename T>
__global__ void __launch_bounds__(128) delta_kernel(const Params<T> p) {
  const int64_t i = (int64_t)blockIdx.x * 4 + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  if (i >= (int64_t)p.H * p.N) return;
  const int h = (int)(i % p.H), row = (int)(i / p.H);
  const T *a = p.go + (int64_t)row * p.gos + h * p.goh, *b = p.o + (int64_t)row * p.os + h * p.oh;
  T s = T(0);
  for (int d = lane; d < p.D; d += 32) s += a[d] * b[d];
  s = row_sum<32>(s);
  if (lane == 0) p.delta[(int64_t)h * p.N + row] = s;
}

// structures of at most BQ atoms: one block holds the whole probability matrix of a head, so that the
// softmax is formed at once (neither the forward output nor its statistics are read) and dq, dk, dv
// come from one launch and one reading of the inputs
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
#pragma unroll
      for (int r = 0; r < C::RI; ++r) {
        T top = neg_inf<T>();
#pragma unroll
        for (int c = 0; c < C::RJ; ++c) {
          s[r][c] = allowed(part.row + tx + C::TX * c, part.hi, p.mask) ? s[r][c] * c2 : neg_inf<T>();
          top = s[r][c] > top ? s[r][c] : top;
        }
        top = row_max<C::TX>(top);
        const T base = top == neg_inf<T>() ? T(0) : top;
        T sum = T(0);
#pragma unroll
        for (int c = 0; c < C::RJ; ++c) { s[r][c] = pow2(s[r][c] - base); sum += s[r][c]; }
        sum = row_sum<C::TX>(sum);
        const T inv = top == neg_inf<T>() || part.row + i0 + r >= part.hi ? T(0) : T(1) / sum;
        T D = T(0);
#pragma unroll
        for (int c = 0; c < C::RJ; ++c) { s[r][c] *= inv; D += s[r][c] * dp[r][c]; }
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
    const int64_t at = ((int64_t)row * p.HK + hk) * p.D;
    store_row<T, C::DP, C::TX>(p.out1 + at, dk[r], p.scale * good, p.D, tx);
    store_row<T, C::DP, C::TX>(p.out2 + at, dv[r], good, p.D, tx);
  }
}

// ------------------------------------------------------------------------------------------ second derivative
// rows: q' and do'; the first walk over the keys gives r, c and do', the second q'
template <typename T, typename C>
__global__ void __launch_bounds__(C::NT) second_row_kernel(const Params<T> p) {
  extern __shared__ __align__(16) char smem_raw[];
  T* sQ = reinterpret_cast<T*>(smem_raw);
  T* sO = sQ + C::BQ * C::LD;
  T* sA = sO + C::BQ * C::LD;
  T* sK = sA + C::BQ * C::LD;
  T* sV = sK + C::BK * C::LD;
  T* sB = sV + C::BK * C::LD;
  T* sC = sB + C::BK * C::LD;
  T* sP = sC + C::BK * C::LD;
  T* sS = sP + C::BQ * C::LDP;
  Part part;
  if (!find_part<C::BQ>(p, blockIdx.x, part)) return;
  const int h = blockIdx.y, hk = h / (p.H / p.HK);
  const int tx = threadIdx.x % C::TX, i0 = threadIdx.x / C::TX * C::RI;
  const int k_lo = part.lo, k_hi = part.keys ? part.hi : part.lo;
  const T c2 = p.scale * log2e<T>();
  T L[C::RI], D[C::RI], R[C::RI], U[C::RI], acc[C::RI][C::DP / C::TX];
#pragma unroll
  for (int r = 0; r < C::RI; ++r) {
    const int row = part.row + i0 + r;
    L[r] = row < part.hi ? p.lse[(int64_t)h * p.N + row] : T(0);
    D[r] = row < part.hi ? p.delta[(int64_t)h * p.N + row] : T(0);
    R[r] = U[r] = T(0);
#pragma unroll
    for (int n = 0; n < C::DP / C::TX; ++n) acc[r][n] = T(0);
  }
  if (k_lo < k_hi) {
    load_tile<T, C::BQ, C::DP, C::LD, C::NT>(sQ, p.q + h * p.qh, p.qs, part.row, part.hi, p.D, vec_ok(p.q, p.qs, p.qh, p.D));
    load_tile<T, C::BQ, C::DP, C::LD, C::NT>(sO, p.go + h * p.goh, p.gos, part.row, part.hi, p.D, vec_ok(p.go, p.gos, p.goh, p.D));
    load_tile<T, C::BQ, C::DP, C::LD, C::NT>(sA, p.ca + h * p.cah, p.cas, part.row, part.hi, p.D, vec_ok(p.ca, p.cas, p.cah, p.D));
  }
  const bool one = k_hi - k_lo <= C::BK;                 // the second walk finds the keys still in place
  for (int walk = 0; walk < 2; ++walk) {
    for (int k0 = k_lo; k0 < k_hi; k0 += C::BK) {
      if (walk == 0 || !one) {
        load_tile<T, C::BK, C::DP, C::LD, C::NT>(sK, p.k + hk * p.kh, p.ks, k0, k_hi, p.D, vec_ok(p.k, p.ks, p.kh, p.D), p.mask);
        load_tile<T, C::BK, C::DP, C::LD, C::NT>(sV, p.v + hk * p.vh, p.vs, k0, k_hi, p.D, vec_ok(p.v, p.vs, p.vh, p.D), p.mask);
        load_tile<T, C::BK, C::DP, C::LD, C::NT>(sB, p.cb + hk * p.cbh, p.cbs, k0, k_hi, p.D, vec_ok(p.cb, p.cbs, p.cbh, p.D), p.mask);
        load_tile<T, C::BK, C::DP, C::LD, C::NT>(sC, p.cc + hk * p.cch, p.ccs, k0, k_hi, p.D, vec_ok(p.cc, p.ccs, p.cch, p.D), p.mask);
      }
      __syncthreads();
      T s[C::RI][C::RJ] = {}, t[C::RI][C::RJ] = {}, dp[C::RI][C::RJ] = {}, e[C::RI][C::RJ] = {};
      tile_nt<T, C::RI, C::RJ, C::TX, C::DP, C::LD>(s, sQ, i0, sK, tx);
      tile_nt<T, C::RI, C::RJ, C::TX, C::DP, C::LD>(t, sA, i0, sK, tx);
      tile_nt<T, C::RI, C::RJ, C::TX, C::DP, C::LD>(t, sQ, i0, sB, tx);
      tile_nt<T, C::RI, C::RJ, C::TX, C::DP, C::LD>(dp, sO, i0, sV, tx);
      tile_nt<T, C::RI, C::RJ, C::TX, C::DP, C::LD>(e, sO, i0, sC, tx);
#pragma unroll
      for (int c = 0; c < C::RJ; ++c) {
        const bool ok = allowed(k0 + tx + C::TX * c, k_hi, p.mask);
#pragma unroll
        for (int r = 0; r < C::RI; ++r) {
          const T pr = ok ? pow2(s[r][c] * c2 - L[r]) : T(0);
          const T tt = t[r][c] * p.scale;
          T a, b;
          if (walk == 0) {
            a = pr * tt;
            b = pr;
            R[r] += a;
            U[r] += pr * (tt * dp[r][c] + e[r][c]);
          } else {
            a = pr * ((tt - R[r]) * (dp[r][c] - D[r]) + e[r][c] - U[r]);
            b = pr * (dp[r][c] - D[r]);
          }
          sP[(i0 + r) * C::LDP + tx + C::TX * c] = ok ? a : T(0);
          sS[(i0 + r) * C::LDP + tx + C::TX * c] = ok ? b : T(0);
        }
      }
      __syncthreads();
      tile_nn<T, C::RI, C::BK, C::TX, C::DP, C::LDP, C::LD>(acc, sP, i0, walk == 0 ? sV : sK, tx);
      tile_nn<T, C::RI, C::BK, C::TX, C::DP, C::LDP, C::LD>(acc, sS, i0, walk == 0 ? sC : sB, tx);
      __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < C::RI; ++r) {
      const int row = part.row + i0 + r;
      const bool in = row < part.hi;
      T* out = (walk == 0 ? p.out3 : p.out0) + ((int64_t)row * p.H + h) * p.D;
      if (walk == 0) {
        R[r] = row_sum<C::TX>(R[r]);
        U[r] = row_sum<C::TX>(U[r]) - D[r] * R[r];
        if (in) {
          using K = Cols<T, C::DP, C::TX>;
          const T* o = p.o + (int64_t)row * p.os + h * p.oh;
#pragma unroll
          for (int n = 0; n < K::NC; ++n)
#pragma unroll
            for (int w = 0; w < K::VW; ++w) {
              const int d = n * C::TX * K::VW + tx * K::VW + w;
              if (d < p.D) acc[r][n * K::VW + w] -= R[r] * o[d];
            }
          if (tx == 0) {
            p.r[(int64_t)h * p.N + row] = R[r];
            p.c[(int64_t)h * p.N + row] = U[r];
          }
        }
      }
      if (in) store_row<T, C::DP, C::TX>(out, acc[r], walk == 0 ? T(1) : p.scale, p.D, tx);
#pragma unroll
      for (int n = 0; n < C::DP / C::TX; ++n) acc[r][n] = T(0);
    }
  }
}

// keys: k' and v' of BQ keys of one key head, over the queries of every head that shares it
template <typename T, typename C>
__global__ void __launch_bounds__(C::NT) second_key_kernel(const Params<T> p) {
  extern __shared__ __align__(16) char smem_raw[];
  T* sK = reinterpret_cast<T*>(smem_raw);
  T* sV = sK + C::BQ * C::LD;
  T* sB = sV + C::BQ * C::LD;
  T* sC = sB + C::BQ * C::LD;
  T* sQ = sC + C::BQ * C::LD;
  T* sO = sQ + C::BK * C::LD;
  T* sA = sO + C::BK * C::LD;
  T* sM = sA + C::BK * C::LD;
  T* sS = sM + C::BQ * C::LDP;
  T* sT = sS + C::BQ * C::LDP;
  Part part;
  if (!find_part<C::BQ>(p, blockIdx.x, part)) return;
  const int hk = blockIdx.y, group = p.H / p.HK;
  const int tx = threadIdx.x % C::TX, i0 = threadIdx.x / C::TX * C::RI;
  const int q_lo = part.lo, q_hi = part.keys ? part.hi : part.lo;
  const T c2 = p.scale * log2e<T>();
  T dk[C::RI][C::DP / C::TX] = {}, dv[C::RI][C::DP / C::TX] = {};
  bool ok[C::RI];
#pragma unroll
  for (int r = 0; r < C::RI; ++r) ok[r] = allowed(part.row + i0 + r, part.hi, p.mask);
  if (q_lo < q_hi) {
    load_tile<T, C::BQ, C::DP, C::LD, C::NT>(sK, p.k + hk * p.kh, p.ks, part.row, part.hi, p.D, vec_ok(p.k, p.ks, p.kh, p.D), p.mask);
    load_tile<T, C::BQ, C::DP, C::LD, C::NT>(sV, p.v + hk * p.vh, p.vs, part.row, part.hi, p.D, vec_ok(p.v, p.vs, p.vh, p.D), p.mask);
    load_tile<T, C::BQ, C::DP, C::LD, C::NT>(sB, p.cb + hk * p.cbh, p.cbs, part.row, part.hi, p.D, vec_ok(p.cb, p.cbs, p.cbh, p.D), p.mask);
    load_tile<T, C::BQ, C::DP, C::LD, C::NT>(sC, p.cc + hk * p.cch, p.ccs, part.row, part.hi, p.D, vec_ok(p.cc, p.ccs, p.cch, p.D), p.mask);
  }
  for (int g = 0; g < group; ++g) {
    const int h = hk * group + g;
    for (int q0 = q_lo; q0 < q_hi; q0 += C::BK) {
      load_tile<T, C::BK, C::DP, C::LD, C::NT>(sQ, p.q + h * p.qh, p.qs, q0, q_hi, p.D, vec_ok(p.q, p.qs, p.qh, p.D));
      load_tile<T, C::BK, C::DP, C::LD, C::NT>(sO, p.go + h * p.goh, p.gos, q0, q_hi, p.D, vec_ok(p.go, p.gos, p.goh, p.D));
      load_tile<T, C::BK, C::DP, C::LD, C::NT>(sA, p.ca + h * p.cah, p.cas, q0, q_hi, p.D, vec_ok(p.ca, p.cas, p.cah, p.D));
      __syncthreads();
      T s[C::RI][C::RJ] = {}, t[C::RI][C::RJ] = {}, dp[C::RI][C::RJ] = {}, e[C::RI][C::RJ] = {};
      tile_nt<T, C::RI, C::RJ, C::TX, C::DP, C::LD>(s, sK, i0, sQ, tx);
      tile_nt<T, C::RI, C::RJ, C::TX, C::DP, C::LD>(t, sK, i0, sA, tx);
      tile_nt<T, C::RI, C::RJ, C::TX, C::DP, C::LD>(t, sB, i0, sQ, tx);
      tile_nt<T, C::RI, C::RJ, C::TX, C::DP, C::LD>(dp, sV, i0, sO, tx);
      tile_nt<T, C::RI, C::RJ, C::TX, C::DP, C::LD>(e, sC, i0, sO, tx);
#pragma unroll
      for (int c = 0; c < C::RJ; ++c) {
        const int row = q0 + tx + C::TX * c;
        const bool in = row < q_hi;
        const int64_t at = (int64_t)h * p.N + (in ? row : q_lo);
        const T L = p.lse[at], D = p.delta[at], R = p.r[at], U = p.c[at];
#pragma unroll
        for (int r = 0; r < C::RI; ++r) {
          const bool on = in && ok[r];
          const T pr = on ? pow2(s[r][c] * c2 - L) : T(0);
          const T tt = t[r][c] * p.scale;
          const int w = (i0 + r) * C::LDP + tx + C::TX * c;
          sM[w] = on ? pr * ((tt - R) * (dp[r][c] - D) + e[r][c] - U) : T(0);
          sS[w] = on ? pr * (dp[r][c] - D) : T(0);
          sT[w] = on ? pr * (tt - R) : T(0);
        }
      }
      __syncthreads();
      tile_nn<T, C::RI, C::BK, C::TX, C::DP, C::LDP, C::LD>(dk, sM, i0, sQ, tx);
      tile_nn<T, C::RI, C::BK, C::TX, C::DP, C::LDP, C::LD>(dk, sS, i0, sA, tx);
      tile_nn<T, C::RI, C::BK, C::TX, C::DP, C::LDP, C::LD>(dv, sT, i0, sO, tx);
      __syncthreads();
    }
  }
#pragma unroll
  for (int r = 0; r < C::RI; ++r) {
    const int row = part.row + i0 + r;
    if (row >= part.hi) continue;
    const int64_t at = ((int64_t)row * p.HK + hk) * p.D;
    store_row<T, C::DP, C::TX>(p.out1 + at, dk[r], p.scale, p.D, tx);
    store_row<T, C::DP, C::TX>(p.out2 + at, dv[r], T(1), p.D, tx);
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

// The square tiles of 32 rows. float: a 2 x 4 corner of the scores a thread (one molecule of 21 atoms at 64 columns:
// 6.1 us with 128 threads, 9.1 with 64 and 4 x 4 corners; 4000 x 4 heads: 236 and 279 us). double: 2 x 2, since the
// accumulators of 4 x 4 alone would take 128 registers at 128 columns.
template <typename T, int DP> struct Small;
template <int DP> struct Small<float, DP> { using C = Cfg<float, 32, 32, DP, 2, 8>; };
template <int DP> struct Small<double, DP> { using C = Cfg<double, 32, 32, DP, 2, 16>; };
// The short backward pass has five products on a tile and reads less of it with 4 x 4 corners, up to 64 columns (64: 532
// and 565 us for 4000 x 4 heads; 128: 186 and, with 256 threads, 153 us for 2000).
template <typename T, int DP> struct Short { using C = typename Small<T, DP>::C; };
template <int DP> struct Short<float, DP> { using C = Cfg<float, 32, 32, DP, 4, 8>; };
template <> struct Short<float, 128> { using C = Cfg<float, 32, 32, 128, 2, 16>; };
// the second derivative holds seven tiles: 128 double columns leave room for 16 streamed rows
template <typename T, int DP> struct Second { using C = typename Small<T, DP>::C; };
template <int DP> struct Second<float, DP> { using C = Cfg<float, 32, 64, DP, 2, 16>; };
template <> struct Second<double, 128> { using C = Cfg<double, 32, 16, 128, 2, 16>; };

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
cudaError_t row_delta(const Params<T>& p, cudaStream_t s) {
  const int64_t rows = (int64_t)p.H * p.N;
  delta_kernel<T><<<(unsigned)((rows + 3) / 4), 128, 0, s>>>(p);
  return cudaGetLastError();
}
template <typename T>
cudaError_t backward_short(const Params<T>& p, cudaStream_t s) {
  XNN_ATTN_DIM(p.D, using C = typename Short<T, DP>::C; return (launch<T, C, bwd_short_kernel<T, C>>(p, p.HK, 2, 2, 2, s)))
}
template <typename T>
cudaError_t second_rows(const Params<T>& p, cudaStream_t s) {
  XNN_ATTN_DIM(p.D, using C = typename Second<T, DP>::C; return (launch<T, C, second_row_kernel<T, C>>(p, p.H, 3, 4, 2, s)))
}
template <typename T>
cudaError_t second_keys(const Params<T>& p, cudaStream_t s) {
  XNN_ATTN_DIM(p.D, using C = typename Second<T, DP>::C; return (launch<T, C, second_key_kernel<T, C>>(p, p.HK, 4, 3, 3, s)))
}

#define XNN_ATTN_INST(T)                                                                  \
  template cudaError_t forward<T>(const Params<T>&, cudaStream_t);                        \
  template cudaError_t forward_join<T>(const Params<T>&, cudaStream_t);                   \
  template cudaError_t sum_splits<T>(int64_t, int, const T*, T*, T*, cudaStream_t);       \
  template cudaError_t row_delta<T>(const Params<T>&, cudaStream_t);                      \
  template cudaError_t backward_short<T>(const Params<T>&, cudaStream_t);                 \
  template cudaError_t second_rows<T>(const Params<T>&, cudaStream_t);                    \
  template cudaError_t second_keys<T>(const Params<T>&, cudaStream_t);
XNN_ATTN_INST(float)
XNN_ATTN_INST(double)

}  // namespace attn
