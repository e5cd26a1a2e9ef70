// Shared pieces of the structure-attention kernels: which rows a block owns, tiles in shared memory
// and the register-tiled products over them.
//
// The rows of a packed batch belong to structures given by a CSR pointer (num + 1 entries). With the
// rows before the first and behind the last structure as two more parts that have no keys, the parts
// are p = 0 .. num + 1 with the bounds 0, ptr[0], .., ptr[num], N. A part of x rows needs ceil(x / Q)
// tiles of Q rows; numbering them from floor(start / Q) + p leaves room for all of them, since
// floor((s + x) / Q) - floor(s / Q) + 1 >= ceil(x / Q). So a block finds its part from the pointer alone
// (a warp-wide 32-ary search), the grid is floor(N / Q) + num + 2 whatever the lengths are, and no
// host copy of the lengths is needed. Bounds are clamped to [0, N]: no pointer value leaves the arrays.
#pragma once
#include <atomic>
#include <limits>

#include "attention_params.h"
#include "common.cuh"

namespace attn {

struct Part { int lo, hi, row, index; bool keys; };   // the part's rows, the block's first row, the part, whether it has keys

__device__ __forceinline__ int part_bound(const int64_t* ptr, int num, int N, int p) {
  if (p <= 0) return 0;
  if (p >= num + 2) return N;
  const int64_t v = ptr[p - 1];
  return (int)(v < 0 ? 0 : (v > N ? N : v));
}

// the last part p of 0 .. num + 1 for which ok(p) holds (it holds up to some part and from there on no more). All lanes of
// a warp call it together.
template <typename F>
__device__ __forceinline__ int last_part(int num, F ok) {
  const int lane = threadIdx.x & 31;
  int at = 0, n = num + 2;
  while (n > 1) {
    const int step = (n + 31) / 32, i = lane * step;
    const unsigned b = __ballot_sync(0xffffffffu, i < n && ok(at + i));
    const int c = max(__popc(b) - 1, 0);
    at += c * step;
    n = min(step, n - c * step);
  }
  return at;
}

// The part and first row of block `t` of Q rows; false where the number is one of the unused ones.
template <int Q, typename T>
__device__ __forceinline__ bool find_part(const Params<T>& p, int t, Part& out) {
  const int64_t* ptr = p.ptr;
  const int num = p.num, N = p.N;
  if (p.compact) {
    // Structures of more than 32 atoms alone, numbered from floor(start / 32): floor(x / 32) >= ceil(x / 64) numbers lie
    // before the next one, however many short structures there are. Row 32 t + 31 is in the structure that owns t.
    out.index = last_part(num, [&](int i) { return part_bound(ptr, num, N, i) <= min(32 * (int64_t)t + 31, (int64_t)N - 1); });
  } else {
    out.index = last_part(num, [&](int i) { return part_bound(ptr, num, N, i) / Q + i <= t; });
  }
  out.lo = part_bound(ptr, num, N, out.index);
  out.hi = max(part_bound(ptr, num, N, out.index + 1), out.lo);
  out.keys = out.index > 0 && out.index <= num;
  const int first = p.compact ? out.lo / 32 : out.lo / Q + out.index;
  const int64_t row = (int64_t)out.lo + (int64_t)(t - first) * Q;
  out.row = (int)row;
  const int len = out.hi - out.lo;
  if (p.compact && len <= 32) return false;
  return row >= out.lo && row < out.hi && (out.keys ? len >= p.min_len && len <= p.max_len : p.rest != 0);
}

// how many blocks of Q rows there may be
template <typename T>
__host__ __device__ __forceinline__ int part_blocks(const Params<T>& p, int Q) { return p.compact ? p.N / 32 + 1 : p.N / Q + p.num + 2; }

template <typename T> __device__ __forceinline__ T log2e() { return T(1.4426950408889634074); }

// the share of split z of the tiles of `B` rows in [lo, hi)
template <int B>
__device__ __forceinline__ void split_range(int& lo, int& hi, int z, int splits) {
  const int tiles = (hi - lo + B - 1) / B, per = (tiles + splits - 1) / splits;
  const int end = hi;
  hi = min(end, lo + min(tiles, (z + 1) * per) * B);
  lo = min(end, lo + min(tiles, z * per) * B);
}

template <typename T> struct Vec { static constexpr int W = 16 / sizeof(T); };
template <typename T> struct alignas(16) V16 { T x[16 / sizeof(T)]; };
template <typename T> struct alignas(2 * sizeof(T)) V2 { T x, y; };

__device__ __forceinline__ float pow2(float x) { return exp2f(x); }
__device__ __forceinline__ double pow2(double x) { return exp2(x); }
__device__ __forceinline__ float lg2(float x) { return log2f(x); }
__device__ __forceinline__ double lg2(double x) { return log2(x); }
template <typename T> __device__ __forceinline__ T neg_inf();
template <> __device__ __forceinline__ float neg_inf<float>() { return __int_as_float(0xff800000); }
template <> __device__ __forceinline__ double neg_inf<double>() { return __longlong_as_double(0xfff0000000000000LL); }

// whether 16-byte accesses are allowed for rows at p (+ any head) with these strides
template <typename T>
__host__ __device__ __forceinline__ bool vec_ok(const T* p, int64_t rs, int64_t hs, int D) {
  constexpr int W = Vec<T>::W;
  return (reinterpret_cast<uintptr_t>(p) % 16 == 0) && rs % W == 0 && hs % W == 0 && D % W == 0;
}

// Rows row0 (< end) .. row0 + ROWS of g into s (row stride LD), zero behind `end`, behind column D and where the mask is 0:
// what is masked or belongs to another structure never enters a product, NaN included. Eight loads are in flight a
// thread: they go to addresses that exist and what is not wanted is dropped afterwards, since a load under a condition
// waits for the one before.
template <typename T, int ROWS, int DP, int LD, int NT>
__device__ __forceinline__ void load_tile(T* s, const T* g, int64_t stride, int row0, int end, int D, bool vec,
                                          const uint8_t* mask = nullptr) {
  constexpr int W = Vec<T>::W, CH = DP / W, N = ROWS * CH, U = N / NT < 8 ? (N / NT < 1 ? 1 : N / NT) : 8;
#pragma unroll 1
  for (int i0 = threadIdx.x; i0 < N; i0 += U * NT) {
    V16<T> v[U];
    bool on[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(i0 + u * NT, N - 1), r = i / CH, c = (i % CH) * W, row = min(row0 + r, end - 1);
      on[u] = row0 + r < end && c < D;
      const T* p = g + (int64_t)row * stride + (c < D ? c : 0);
      if (vec) {
        v[u] = *reinterpret_cast<const V16<T>*>(p);
      } else {
#pragma unroll
        for (int e = 0; e < W; ++e) v[u].x[e] = p[c + e < D ? e : 0];
      }
      if (mask) on[u] = on[u] && mask[row];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * NT;
      if (i < N) {
        const int c = (i % CH) * W;
#pragma unroll
        for (int e = 0; e < W; ++e)
          if (!on[u] || c + e >= D) v[u].x[e] = T(0);
        *reinterpret_cast<V16<T>*>(s + i / CH * LD + c) = v[u];
      }
    }
  }
}

// acc[r][c] += sum_d A[i0 + r][d] B[j0 + TX c][d]: row-major tiles, rows of A contiguous per thread and
// columns strided by TX so that a warp's 16-byte reads of B fall into different banks (LD = DP + 16 bytes)
template <typename T, int RI, int RJ, int TX, int DP, int LD>
__device__ __forceinline__ void tile_nt(T (&acc)[RI][RJ], const T* A, int i0, const T* B, int j0) {
  constexpr int W = Vec<T>::W;
#pragma unroll 4
  for (int d = 0; d < DP; d += W) {
    V16<T> a[RI], b[RJ];
#pragma unroll
    for (int r = 0; r < RI; ++r) a[r] = *reinterpret_cast<const V16<T>*>(A + (i0 + r) * LD + d);
#pragma unroll
    for (int c = 0; c < RJ; ++c) b[c] = *reinterpret_cast<const V16<T>*>(B + (j0 + TX * c) * LD + d);
#pragma unroll
    for (int e = 0; e < W; ++e)
#pragma unroll
      for (int r = 0; r < RI; ++r)
#pragma unroll
        for (int c = 0; c < RJ; ++c) acc[r][c] += a[r].x[e] * b[c].x[e];
  }
}

// how a thread's DP / TX output columns are laid out: NC groups of VW neighbours, TX * VW apart
template <typename T, int DP, int TX>
struct Cols {
  static constexpr int PER = DP / TX;
  static constexpr int VW = PER < Vec<T>::W ? PER : Vec<T>::W;
  static constexpr int NC = PER / VW;
};

// acc[r][.] += sum_{j < J} P[i0 + r][j] V[j][columns of tx]; from the first `used` on, P is zero
template <typename T, int RI, int J, int TX, int DP, int LDP, int LD>
__device__ __forceinline__ void tile_nn(T (&acc)[RI][DP / TX], const T* P, int i0, const T* V, int tx, int used = J) {
  using C = Cols<T, DP, TX>;
  constexpr int W = Vec<T>::W;
  const int end = used < J ? used : J;
#pragma unroll 2
  for (int j = 0; j < end; j += W) {
    V16<T> p[RI];
#pragma unroll
    for (int r = 0; r < RI; ++r) p[r] = *reinterpret_cast<const V16<T>*>(P + (i0 + r) * LDP + j);
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const T* row = V + (j + e) * LD + tx * C::VW;
#pragma unroll
      for (int n = 0; n < C::NC; ++n) {
        T v[C::VW];
        if constexpr (C::VW == W) {
          *reinterpret_cast<V16<T>*>(v) = *reinterpret_cast<const V16<T>*>(row + n * TX * C::VW);
        } else {
#pragma unroll
          for (int w = 0; w < C::VW; ++w) v[w] = row[n * TX * C::VW + w];
        }
#pragma unroll
        for (int r = 0; r < RI; ++r)
#pragma unroll
          for (int w = 0; w < C::VW; ++w) acc[r][n * C::VW + w] += p[r].x[e] * v[w];
      }
    }
  }
}

// acc[r][.] += sum_{j < J} P[j][i0 + r] V[j][columns of tx] (P read transposed; RI neighbouring columns)
template <typename T, int RI, int J, int TX, int DP, int LDP, int LD>
__device__ __forceinline__ void tile_tn(T (&acc)[RI][DP / TX], const T* P, int i0, const T* V, int tx, int used = J) {
  using C = Cols<T, DP, TX>;
  constexpr int G = RI < Vec<T>::W ? RI : Vec<T>::W;       // columns a load takes
  struct alignas(G * sizeof(T)) Group { T x[G]; };
  const int end = used < J ? used : J;
#pragma unroll 4
  for (int j = 0; j < end; ++j) {
    T p[RI];
#pragma unroll
    for (int r = 0; r < RI; r += G) {
      const Group at = *reinterpret_cast<const Group*>(P + j * LDP + i0 + r);
#pragma unroll
      for (int x = 0; x < G; ++x) p[r + x] = at.x[x];
    }
    const T* row = V + j * LD + tx * C::VW;
#pragma unroll
    for (int n = 0; n < C::NC; ++n) {
      T v[C::VW];
#pragma unroll
      for (int w = 0; w < C::VW; ++w) v[w] = row[n * TX * C::VW + w];
#pragma unroll
      for (int r = 0; r < RI; ++r)
#pragma unroll
        for (int w = 0; w < C::VW; ++w) acc[r][n * C::VW + w] += p[r] * v[w];
    }
  }
}

// columns of tx of one row: out[column] = f * acc, guarded by D
template <typename T, int DP, int TX>
__device__ __forceinline__ void store_row(T* out, const T (&acc)[DP / TX], T f, int D, int tx) {
  using C = Cols<T, DP, TX>;
#pragma unroll
  for (int n = 0; n < C::NC; ++n)
#pragma unroll
    for (int w = 0; w < C::VW; ++w) {
      const int d = n * TX * C::VW + tx * C::VW + w;
      if (d < D) out[d] = f * acc[n * C::VW + w];
    }
}

// sum / maximum over the TX lanes that share a row
template <int TX, typename T>
__device__ __forceinline__ T row_sum(T v) {
#pragma unroll
  for (int o = TX / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int TX, typename T>
__device__ __forceinline__ T row_max(T v) {
#pragma unroll
  for (int o = TX / 2; o; o >>= 1) { const T u = __shfl_xor_sync(0xffffffffu, v, o); v = v > u ? v : u; }
  return v;
}

// Shared memory beyond the default 48 KB is asked for once a kernel and device, not at every launch.
template <auto KERNEL>
cudaError_t raise_smem_limit(size_t bytes) {
  static std::atomic<uint64_t> done{0};                  // a bit per device
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess || bytes <= 48 * 1024) return e;
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

}  // namespace attn
