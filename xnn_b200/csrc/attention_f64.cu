// Structure attention in 64 bits on the FP64 tensor instructions (formulas: attention.cu), for structures of more than a
// tile: forward, backward and second derivative of float64 operands, and the second derivative of float32 operands of
// more than 64 columns a head, whose parts the FP16-type tensor cores' memory does not hold (the operands are widened
// as they are read; 64-bit products run at half the FP32 pipes' rate but need a third of their shared-memory traffic).
//
// The streamed tiles come by asynchronous copies in two groups: those that a walk only takes for one kind of product are
// free while the others are at work, so the next tile's copies run under the products without a second set of buffers.
//
// A block owns 32 rows and streams tiles of the other side through shared memory. Its warps are RG groups of rows by KG
// groups of the streamed rows: a warp forms the weights of its 8 RB rows and its own slice of each tile, multiplies
// them on at once, and the KG partial results (with their own running maxima in the forward pass) are joined at the
// end. With m8n8k4 products a lane holds, of 8 x 8 scores, row lane / 4 and columns 2 (lane % 4) + {0, 1}; the next
// product takes a row's weights as they lie, four columns at a time: step s takes column 2 t + (s ^ t / 2) from lane t,
// so that the four matching rows of the other operand fall into different banks (rows are 4 mod 16 numbers long; float32
// rows, 4 mod 32 long, are conflict-free with column 2 t + s).
#include <type_traits>

#include "attention.h"
#include "attention_tile.cuh"

namespace attn {
namespace {

template <int DP_, int RB_, int RG_, int KG_, int NT_>
struct Shape {
  static constexpr int DP = DP_, RB = RB_, RG = RG_, KG = KG_, NT = NT_;
  static constexpr int ROWS = 8 * RB * RG, TILE = 8 * KG * NT, THREADS = 32 * RG * KG;
  static_assert(ROWS == 32, "a block owns 32 rows");
};

template <typename IN>
__host__ __device__ constexpr int row_length(int D) {
  return sizeof(IN) == 8 ? (D + 15) / 16 * 16 + 4 : (D + 31) / 32 * 32 + 4;
}

__device__ __forceinline__ void mma(double (&c)[2], double a, double b) {
  asm("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};" : "+d"(c[0]), "+d"(c[1]) : "d"(a), "d"(b));
}

// BYTES to shared memory, zero if not `on`
template <int BYTES>
__device__ __forceinline__ void copy_async(void* s, const void* g, bool on) {
  const uint32_t dst = (uint32_t)__cvta_generic_to_shared(s);
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(g), "n"(BYTES), "r"(on ? BYTES : 0) : "memory");
}
__device__ __forceinline__ void end_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// waits for the copies of all groups but the latest LEFT, the whole block's
template <int LEFT>
__device__ __forceinline__ void arrive() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
  __syncthreads();
}

// starts the copies of `rows` rows of g from row0 (< end) on; zero behind `end`, behind column D (up to the next multiple of
// 8) and where masked
template <int THREADS, typename IN>
__device__ __forceinline__ void copy_rows(IN* s, int ld, const IN* g, int64_t stride, int64_t head, int row0, int rows, int end, int D,
                                          const uint8_t* mask = nullptr) {
  const bool vec = reinterpret_cast<uintptr_t>(g) % (2 * sizeof(IN)) == 0 && stride % 2 == 0 && head % 2 == 0 && D % 2 == 0;
  const uint32_t pairs = (D + 7) / 8 * 4, by = ((1u << 20) + pairs - 1) / pairs;      // i / pairs = i by / 2^20 for i < 2^13
  const uint32_t n = rows * pairs;
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
    const int r = i * by >> 20, c = (i - r * pairs) * 2, row = min(row0 + r, end - 1);
    const bool on = row0 + r < end && c < D && (mask == nullptr || mask[row]);
    const IN* p = g + row * stride + (c < D ? c : 0);
    IN* to = s + r * ld + c;
    if (vec) {
      copy_async<2 * sizeof(IN)>(to, p, on);
    } else {
      copy_async<sizeof(IN)>(to, p, on);
      copy_async<sizeof(IN)>(to + 1, p + (c + 1 < D), on && c + 1 < D);
    }
  }
}

// where a lane's numbers lie
template <class S>
struct Lane {
  int g, t, rg, kg, ld;
  __device__ __forceinline__ explicit Lane(int ld_) : g(threadIdx.x % 32 / 4), t(threadIdx.x % 4), ld(ld_) {
    rg = threadIdx.x / 32 / S::KG;
    kg = threadIdx.x / 32 % S::KG;
  }
  __device__ __forceinline__ int own(int rb) const { return (rg * S::RB + rb) * 8 + g; }            // own row of block rb
  __device__ __forceinline__ int col(int nt) const { return (kg * S::NT + nt) * 8; }                 // first streamed row of block nt
};

template <class S> using Scores = double[S::RB][S::NT][2];
template <class S> using Sums = double[S::RB][S::DP / 8][2];

template <class S>
__device__ __forceinline__ void zero(Scores<S>& x) {
#pragma unroll
  for (int rb = 0; rb < S::RB; ++rb)
#pragma unroll
    for (int nt = 0; nt < S::NT; ++nt) x[rb][nt][0] = x[rb][nt][1] = 0.0;
}
template <class S>
__device__ __forceinline__ void clear(Sums<S>& x) {
#pragma unroll
  for (int rb = 0; rb < S::RB; ++rb)
#pragma unroll
    for (int n = 0; n < S::DP / 8; ++n) x[rb][n][0] = x[rb][n][1] = 0.0;
}

// a masked key's gradients are zero whatever its queries hold (0 NaN is NaN)
template <class S>
__device__ __forceinline__ void hide(Sums<S>& x, const bool (&ok)[S::RB]) {
#pragma unroll
  for (int rb = 0; rb < S::RB; ++rb)
#pragma unroll
    for (int n = 0; n < S::DP / 8; ++n) {
      x[rb][n][0] = ok[rb] ? x[rb][n][0] : 0.0;
      x[rb][n][1] = ok[rb] ? x[rb][n][1] : 0.0;
    }
}

// x += own rows of A times streamed rows of B
template <class S, typename IN>
__device__ __forceinline__ void scores(Scores<S>& x, const Lane<S>& l, const IN* A, const IN* B, int D) {
#pragma unroll 4
  for (int k = 0; k < D; k += 4) {
    double a[S::RB], b[S::NT];
#pragma unroll
    for (int rb = 0; rb < S::RB; ++rb) a[rb] = (double)A[l.own(rb) * l.ld + k + l.t];
#pragma unroll
    for (int nt = 0; nt < S::NT; ++nt) b[nt] = (double)B[(l.col(nt) + l.g) * l.ld + k + l.t];
#pragma unroll
    for (int rb = 0; rb < S::RB; ++rb)
#pragma unroll
      for (int nt = 0; nt < S::NT; ++nt) mma(x[rb][nt], a[rb], b[nt]);
  }
}

// acc += weights (own rows x streamed rows) times streamed rows of V
template <class S, typename IN>
__device__ __forceinline__ void sums(Sums<S>& acc, const Lane<S>& l, const Scores<S>& w, const IN* V, int D) {
#pragma unroll
  for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int e = sizeof(IN) == 8 ? s ^ (l.t >> 1) : s;
      const IN* row = V + (l.col(nt) + 2 * l.t + e) * l.ld + l.g;
      double a[S::RB];
#pragma unroll
      for (int rb = 0; rb < S::RB; ++rb) a[rb] = e ? w[rb][nt][1] : w[rb][nt][0];
#pragma unroll
      for (int n = 0; n < S::DP / 8; ++n) {
        if (n * 8 < D) {
          const double b = (double)row[n * 8];
#pragma unroll
          for (int rb = 0; rb < S::RB; ++rb) mma(acc[rb][n], a[rb], b);
        }
      }
    }
}

// The KG warps' partial results of the block's rows, each times f (one a row block), joined in their order into
// out[row] (rows `stride` apart), times `scale`. `red` holds KG x 32 rows.
template <class S, typename OUT>
__device__ __forceinline__ void join_rows(double* red, const Lane<S>& l, const Sums<S>& acc, const double (&f)[S::RB], OUT* out,
                                          int64_t stride, int rows, int D, double scale) {
  const int ld = row_length<double>(D);
  __syncthreads();
#pragma unroll
  for (int rb = 0; rb < S::RB; ++rb)
#pragma unroll
    for (int n = 0; n < S::DP / 8; ++n)
      if (n * 8 < D)
        *reinterpret_cast<double2*>(red + (l.kg * 32 + l.own(rb)) * ld + n * 8 + 2 * l.t) =
            make_double2(f[rb] * acc[rb][n][0], f[rb] * acc[rb][n][1]);
  __syncthreads();
  for (int i = threadIdx.x; i < rows * D; i += S::THREADS) {
    const int r = i / D, d = i - r * D;
    double x = 0.0;
#pragma unroll
    for (int kg = 0; kg < S::KG; ++kg) x += red[(kg * 32 + r) * ld + d];
    out[r * stride + d] = (OUT)(scale * x);
  }
}

__device__ __forceinline__ double quad_sum(double v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

__device__ __forceinline__ bool may(int j, int hi, const uint8_t* mask) { return j < hi && (mask == nullptr || mask[j]); }

// ------------------------------------------------------------------------------------------ forward
template <class S>
__global__ void __launch_bounds__(S::THREADS) fwd64_kernel(const Params<double> p) {
  extern __shared__ __align__(16) double smem64[];
  __shared__ double top[S::KG][32], total[S::KG][32];
  Part part;
  if (!find_part<32>(p, blockIdx.x, part)) return;
  const Lane<S> l(row_length<double>(p.D));
  const int h = blockIdx.y, hk = h / (p.H / p.HK);
  double *sQ = smem64, *sK = sQ + 32 * l.ld, *sV = sK + S::TILE * l.ld;
  int lo = part.lo, hi = part.keys ? part.hi : part.lo;
  split_range<S::TILE>(lo, hi, blockIdx.z, p.splits);
  const double c2 = p.scale * log2e<double>();
  double m[S::RB], sum[S::RB];
  Sums<S> acc;
  clear<S>(acc);
#pragma unroll
  for (int rb = 0; rb < S::RB; ++rb) {
    m[rb] = neg_inf<double>();
    sum[rb] = 0.0;
  }
  const auto next_k = [&](int k0) {
    if (k0 < hi) copy_rows<S::THREADS>(sK, l.ld, p.k + hk * p.kh, p.ks, p.kh, k0, S::TILE, hi, p.D, p.mask);
    end_group();
  };
  const auto next_v = [&](int k0) {
    if (k0 < hi) copy_rows<S::THREADS>(sV, l.ld, p.v + hk * p.vh, p.vs, p.vh, k0, S::TILE, hi, p.D, p.mask);
    end_group();
  };
  if (lo < hi) copy_rows<S::THREADS>(sQ, l.ld, p.q + h * p.qh, p.qs, p.qh, part.row, 32, part.hi, p.D);
  next_k(lo);
  next_v(lo);
  for (int k0 = lo; k0 < hi; k0 += S::TILE) {
    arrive<1>();
    Scores<S> s;
    zero<S>(s);
    scores<S>(s, l, sQ, sK, p.D);
#pragma unroll
    for (int rb = 0; rb < S::RB; ++rb) {
      double mx = neg_inf<double>();
#pragma unroll
      for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[rb][nt][e] = may(k0 + l.col(nt) + 2 * l.t + e, hi, p.mask) ? s[rb][nt][e] * c2 : neg_inf<double>();
          mx = s[rb][nt][e] > mx ? s[rb][nt][e] : mx;
        }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        const double u = __shfl_xor_sync(0xffffffffu, mx, o);
        mx = u > mx ? u : mx;
      }
      const double mn = mx > m[rb] ? mx : m[rb], base = mn == neg_inf<double>() ? 0.0 : mn, f = exp2(m[rb] - base);
      double u = 0.0;
#pragma unroll
      for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[rb][nt][e] = exp2(s[rb][nt][e] - base);
          u += s[rb][nt][e];
        }
      sum[rb] = sum[rb] * f + quad_sum(u);
      m[rb] = mn;
#pragma unroll
      for (int n = 0; n < S::DP / 8; ++n) {
        acc[rb][n][0] *= f;
        acc[rb][n][1] *= f;
      }
    }
    arrive<0>();
    next_k(k0 + S::TILE);
    sums<S>(acc, l, s, sV, p.D);
    __syncthreads();
    next_v(k0 + S::TILE);
  }
  if (l.t == 0) {
#pragma unroll
    for (int rb = 0; rb < S::RB; ++rb) {
      top[l.kg][l.own(rb)] = m[rb];
      total[l.kg][l.own(rb)] = sum[rb];
    }
  }
  __syncthreads();
  double f[S::RB];
  const int rows = min(32, part.hi - part.row);
  const int64_t all = (int64_t)p.H * p.N;
#pragma unroll
  for (int rb = 0; rb < S::RB; ++rb) {
    const int r = l.own(rb);
    double mx = neg_inf<double>(), tot = 0.0;
#pragma unroll
    for (int kg = 0; kg < S::KG; ++kg) mx = top[kg][r] > mx ? top[kg][r] : mx;
    const double base = mx == neg_inf<double>() ? 0.0 : mx;
#pragma unroll
    for (int kg = 0; kg < S::KG; ++kg) tot += exp2(top[kg][r] - base) * total[kg][r];
    const bool none = mx == neg_inf<double>() && tot == 0.0;               // NaN scores are not an empty row
    f[rb] = exp2(m[rb] - base) * (p.splits > 1 ? 1.0 : none ? 0.0 : 1.0 / tot);
    if (l.kg == 0 && l.t == 0 && r < rows) {
      const int64_t at = (int64_t)h * p.N + part.row + r;
      if (p.splits > 1) {
        double* stats = p.work + p.splits * all * p.D;
        stats[blockIdx.z * all + at] = mx;
        stats[(p.splits + blockIdx.z) * all + at] = tot;
      } else if (p.lse) {
        p.lse[at] = none ? -neg_inf<double>() : mx + log2(tot);
      }
    }
  }
  double* out = p.splits > 1 ? p.work + (blockIdx.z * all + (int64_t)h * p.N + part.row) * p.D : p.out0 + ((int64_t)part.row * p.H + h) * p.D;
  join_rows<S, double>(smem64, l, acc, f, out, p.splits > 1 ? p.D : (int64_t)p.H * p.D, rows, p.D, 1.0);
}

// ------------------------------------------------------------------------------------------ backward
template <class S>
__global__ void __launch_bounds__(S::THREADS) dq64_kernel(const Params<double> p) {
  extern __shared__ __align__(16) double smem64[];
  Part part;
  if (!find_part<32>(p, blockIdx.x, part)) return;
  const Lane<S> l(row_length<double>(p.D));
  const int h = blockIdx.y, hk = h / (p.H / p.HK);
  double *sQ = smem64, *sO = sQ + 32 * l.ld, *sK = sO + 32 * l.ld, *sV = sK + S::TILE * l.ld;
  int lo = part.lo, hi = part.keys ? part.hi : part.lo;
  split_range<S::TILE>(lo, hi, blockIdx.z, p.splits);
  const double c2 = p.scale * log2e<double>();
  double L[S::RB], D[S::RB], one[S::RB];
  Sums<S> acc;
  clear<S>(acc);
#pragma unroll
  for (int rb = 0; rb < S::RB; ++rb) {
    const int row = part.row + l.own(rb);
    L[rb] = row < part.hi ? p.lse[(int64_t)h * p.N + row] : 0.0;
    D[rb] = row < part.hi ? p.delta[(int64_t)h * p.N + row] : 0.0;
    one[rb] = 1.0;
  }
  const auto next_k = [&](int k0) {
    if (k0 < hi) copy_rows<S::THREADS>(sK, l.ld, p.k + hk * p.kh, p.ks, p.kh, k0, S::TILE, hi, p.D, p.mask);
    end_group();
  };
  const auto next_v = [&](int k0) {
    if (k0 < hi) copy_rows<S::THREADS>(sV, l.ld, p.v + hk * p.vh, p.vs, p.vh, k0, S::TILE, hi, p.D, p.mask);
    end_group();
  };
  if (lo < hi) {
    copy_rows<S::THREADS>(sQ, l.ld, p.q + h * p.qh, p.qs, p.qh, part.row, 32, part.hi, p.D);
    copy_rows<S::THREADS>(sO, l.ld, p.go + h * p.goh, p.gos, p.goh, part.row, 32, part.hi, p.D);
  }
  next_v(lo);
  next_k(lo);
  for (int k0 = lo; k0 < hi; k0 += S::TILE) {
    arrive<1>();
    Scores<S> s, dp;
    zero<S>(s);
    zero<S>(dp);
    scores<S>(dp, l, sO, sV, p.D);
    arrive<0>();
    next_v(k0 + S::TILE);
    scores<S>(s, l, sQ, sK, p.D);
#pragma unroll
    for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const bool ok = may(k0 + l.col(nt) + 2 * l.t + e, hi, p.mask);
#pragma unroll
        for (int rb = 0; rb < S::RB; ++rb) s[rb][nt][e] = ok ? exp2(s[rb][nt][e] * c2 - L[rb]) * (dp[rb][nt][e] - D[rb]) : 0.0;
      }
    sums<S>(acc, l, s, sK, p.D);
    __syncthreads();
    next_k(k0 + S::TILE);
  }
  double* out = p.splits > 1 ? p.work + (int64_t)blockIdx.z * p.N * p.H * p.D : p.out0;
  join_rows<S, double>(smem64, l, acc, one, out + ((int64_t)part.row * p.H + h) * p.D, (int64_t)p.H * p.D, min(32, part.hi - part.row),
                       p.D, p.scale);
}

template <class S>
__global__ void __launch_bounds__(S::THREADS) dkv64_kernel(const Params<double> p) {
  extern __shared__ __align__(16) double smem64[];
  Part part;
  if (!find_part<32>(p, blockIdx.x, part)) return;
  const Lane<S> l(row_length<double>(p.D));
  const int hk = blockIdx.y, group = p.H / p.HK;
  double *sK = smem64, *sV = sK + 32 * l.ld, *sQ = sV + 32 * l.ld, *sO = sQ + S::TILE * l.ld;
  int lo = part.lo, hi = part.keys ? part.hi : part.lo;
  split_range<S::TILE>(lo, hi, blockIdx.z, p.splits_k);
  const double c2 = p.scale * log2e<double>();
  bool ok[S::RB];
  double one[S::RB];
  Sums<S> dk, dv;
  clear<S>(dk);
  clear<S>(dv);
#pragma unroll
  for (int rb = 0; rb < S::RB; ++rb) {
    ok[rb] = may(part.row + l.own(rb), part.hi, p.mask);
    one[rb] = 1.0;
  }
  if (lo < hi) {
    copy_rows<S::THREADS>(sK, l.ld, p.k + hk * p.kh, p.ks, p.kh, part.row, 32, part.hi, p.D, p.mask);
    copy_rows<S::THREADS>(sV, l.ld, p.v + hk * p.vh, p.vs, p.vh, part.row, 32, part.hi, p.D, p.mask);
  }
  const auto next_q = [&](int h, int q0) {
    if (q0 < hi) copy_rows<S::THREADS>(sQ, l.ld, p.q + h * p.qh, p.qs, p.qh, q0, S::TILE, hi, p.D);
    end_group();
  };
  const auto next_o = [&](int h, int q0) {
    if (q0 < hi) copy_rows<S::THREADS>(sO, l.ld, p.go + h * p.goh, p.gos, p.goh, q0, S::TILE, hi, p.D);
    end_group();
  };
  next_o(hk * group, lo);
  next_q(hk * group, lo);
  for (int gh = 0; gh < group; ++gh) {
    const int h = hk * group + gh;
    for (int q0 = lo; q0 < hi; q0 += S::TILE) {
      const bool last = q0 + S::TILE >= hi;                                // the next tile is the next head's first, or none
      const int h1 = last ? h + 1 : h, q1 = !last ? q0 + S::TILE : gh + 1 < group ? lo : hi;
      arrive<1>();
      Scores<S> s, dp;
      zero<S>(s);
      zero<S>(dp);
      scores<S>(dp, l, sV, sO, p.D);
      arrive<0>();
      scores<S>(s, l, sK, sQ, p.D);
#pragma unroll
      for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = q0 + l.col(nt) + 2 * l.t + e;
          const bool in = row < hi;
          const int64_t at = (int64_t)h * p.N + (in ? row : q0);
          const double L = p.lse[at], D = p.delta[at];
#pragma unroll
          for (int rb = 0; rb < S::RB; ++rb) {
            const bool on = in && ok[rb];
            s[rb][nt][e] = on ? exp2(s[rb][nt][e] * c2 - L) : 0.0;
            dp[rb][nt][e] = on ? s[rb][nt][e] * (dp[rb][nt][e] - D) : 0.0;
          }
        }
      sums<S>(dv, l, s, sO, p.D);
      __syncthreads();
      next_o(h1, q1);
      sums<S>(dk, l, dp, sQ, p.D);
      __syncthreads();
      next_q(h1, q1);
    }
  }
  hide<S>(dk, ok);
  hide<S>(dv, ok);
  const int64_t all = (int64_t)p.N * p.HK * p.D, at = ((int64_t)part.row * p.HK + hk) * p.D;
  double *ok_ = p.out1, *ov_ = p.out2;
  if (p.splits_k > 1) {
    ok_ = p.work_k + blockIdx.z * all;
    ov_ = p.work_k + (p.splits_k + blockIdx.z) * all;
  }
  const int rows = min(32, part.hi - part.row);
  join_rows<S, double>(smem64, l, dk, one, ok_ + at, (int64_t)p.HK * p.D, rows, p.D, p.scale);
  join_rows<S, double>(smem64, l, dv, one, ov_ + at, (int64_t)p.HK * p.D, rows, p.D, 1.0);
}

// ------------------------------------------------------------------------------------------ second derivative
// rows: walk 0 gives r, sum P (T dP + E) and P T V + P C, walk 1 the products of q'; `wide` is where 64-bit partial results go
template <class S, typename IN, int WALK>
__global__ void __launch_bounds__(S::THREADS) rows64_kernel(const Params<IN> p, double* __restrict__ part_out, double* __restrict__ part_rc,
                                                            const double* __restrict__ stats) {
  extern __shared__ __align__(16) double smem64[];
  __shared__ double share[2][S::KG][32];
  Part part;
  if (!find_part<32>(p, blockIdx.x, part)) return;
  const Lane<S> l(row_length<IN>(p.D));
  const int h = blockIdx.y, hk = h / (p.H / p.HK);
  IN *sQ = reinterpret_cast<IN*>(smem64), *sO = sQ + 32 * l.ld, *sA = sO + 32 * l.ld, *sK = sA + 32 * l.ld, *sV = sK + S::TILE * l.ld,
     *sB = sV + S::TILE * l.ld, *sC = sB + S::TILE * l.ld;
  int lo = part.lo, hi = part.keys ? part.hi : part.lo;
  split_range<S::TILE>(lo, hi, blockIdx.z, p.splits);
  const double scale = (double)p.scale, c2 = scale * log2e<double>();
  const int64_t all = (int64_t)p.H * p.N;
  double L[S::RB], D[S::RB], r[S::RB], c[S::RB], R[S::RB], U[S::RB], one[S::RB];
  Sums<S> acc;
  clear<S>(acc);
#pragma unroll
  for (int rb = 0; rb < S::RB; ++rb) {
    const int row = part.row + l.own(rb);
    const bool in = row < part.hi;
    const int64_t at = (int64_t)h * p.N + (in ? row : part.row);
    L[rb] = (double)p.lse[at];
    D[rb] = stats[at];
    r[rb] = WALK == 1 ? stats[all + at] : 0.0;
    c[rb] = WALK == 1 ? stats[2 * all + at] : 0.0;
    R[rb] = U[rb] = 0.0;
    one[rb] = 1.0;
  }
  const auto next_kb = [&](int k0) {
    if (k0 < hi) {
      copy_rows<S::THREADS>(sK, l.ld, p.k + hk * p.kh, p.ks, p.kh, k0, S::TILE, hi, p.D, p.mask);
      copy_rows<S::THREADS>(sB, l.ld, p.cb + hk * p.cbh, p.cbs, p.cbh, k0, S::TILE, hi, p.D, p.mask);
    }
    end_group();
  };
  const auto next_vc = [&](int k0) {
    if (k0 < hi) {
      copy_rows<S::THREADS>(sV, l.ld, p.v + hk * p.vh, p.vs, p.vh, k0, S::TILE, hi, p.D, p.mask);
      copy_rows<S::THREADS>(sC, l.ld, p.cc + hk * p.cch, p.ccs, p.cch, k0, S::TILE, hi, p.D, p.mask);
    }
    end_group();
  };
  // the pair that the walk's last products do not take comes first
  const auto first = [&](int k0) {
    if (WALK == 0) next_kb(k0); else next_vc(k0);
  };
  const auto second = [&](int k0) {
    if (WALK == 0) next_vc(k0); else next_kb(k0);
  };
  if (lo < hi) {
    copy_rows<S::THREADS>(sQ, l.ld, p.q + h * p.qh, p.qs, p.qh, part.row, 32, part.hi, p.D);
    copy_rows<S::THREADS>(sO, l.ld, p.go + h * p.goh, p.gos, p.goh, part.row, 32, part.hi, p.D);
    copy_rows<S::THREADS>(sA, l.ld, p.ca + h * p.cah, p.cas, p.cah, part.row, 32, part.hi, p.D);
  }
  first(lo);
  second(lo);
  for (int k0 = lo; k0 < hi; k0 += S::TILE) {
    arrive<1>();
    Scores<S> s, t, dp, e;
    zero<S>(s);
    zero<S>(t);
    zero<S>(dp);
    zero<S>(e);
    const auto with_kb = [&] {
      scores<S>(s, l, sQ, sK, p.D);
      scores<S>(t, l, sA, sK, p.D);
      scores<S>(t, l, sQ, sB, p.D);
    };
    const auto with_vc = [&] {
      scores<S>(dp, l, sO, sV, p.D);
      scores<S>(e, l, sO, sC, p.D);
    };
    if (WALK == 0) with_kb(); else with_vc();
    arrive<0>();
    first(k0 + S::TILE);
    if (WALK == 0) with_vc(); else with_kb();
#pragma unroll
    for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const bool ok = may(k0 + l.col(nt) + 2 * l.t + x, hi, p.mask);
#pragma unroll
        for (int rb = 0; rb < S::RB; ++rb) {
          const double pr = ok ? exp2(s[rb][nt][x] * c2 - L[rb]) : 0.0, tt = t[rb][nt][x] * scale, d = dp[rb][nt][x] - D[rb];
          if (WALK == 0) {
            s[rb][nt][x] = ok ? pr * tt : 0.0;
            t[rb][nt][x] = pr;
            R[rb] += s[rb][nt][x];
            U[rb] += ok ? pr * (tt * dp[rb][nt][x] + e[rb][nt][x]) : 0.0;
          } else {
            s[rb][nt][x] = ok ? pr * ((tt - r[rb]) * d + e[rb][nt][x] - c[rb]) : 0.0;
            t[rb][nt][x] = ok ? pr * d : 0.0;
          }
        }
      }
    sums<S>(acc, l, s, WALK == 0 ? sV : sK, p.D);
    sums<S>(acc, l, t, WALK == 0 ? sC : sB, p.D);
    __syncthreads();
    second(k0 + S::TILE);
  }
  const int rows = min(32, part.hi - part.row);
  if (WALK == 0) {
#pragma unroll
    for (int rb = 0; rb < S::RB; ++rb) {
      R[rb] = quad_sum(R[rb]);
      U[rb] = quad_sum(U[rb]);
      if (l.t == 0) {
        share[0][l.kg][l.own(rb)] = R[rb];
        share[1][l.kg][l.own(rb)] = U[rb];
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * rows; i += S::THREADS) {
      const int w = i / rows, q = i - w * rows;
      double x = 0.0;
#pragma unroll
      for (int kg = 0; kg < S::KG; ++kg) x += share[w][kg][q];
      part_rc[(2 * (int64_t)blockIdx.z + w) * all + (int64_t)h * p.N + part.row + q] = x;
    }
  }
  const int64_t at = ((int64_t)part.row * p.H + h) * p.D;
  if (WALK == 1 && p.splits == 1)
    join_rows<S, IN>(smem64, l, acc, one, p.out0 + at, (int64_t)p.H * p.D, rows, p.D, scale);
  else
    join_rows<S, double>(smem64, l, acc, one, part_out + blockIdx.z * all * p.D + at, (int64_t)p.H * p.D, rows, p.D, WALK == 0 ? 1.0 : scale);
}

// D = do.o, a warp per (row, head)
template <typename IN>
__global__ void __launch_bounds__(128) delta64_kernel(const Params<IN> p, double* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * 4 + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  if (i >= (int64_t)p.H * p.N) return;
  const int h = (int)(i % p.H), row = (int)(i / p.H);
  const IN *a = p.go + (int64_t)row * p.gos + h * p.goh, *b = p.o + (int64_t)row * p.os + h * p.oh;
  double s = 0.0;
  for (int d = lane; d < p.D; d += 32) s += (double)a[d] * (double)b[d];
  s = row_sum<32>(s);
  if (lane == 0) out[(int64_t)h * p.N + row] = s;
}

// r, c and do' of a row from the splits (at most 32), a warp per (row, head)
template <typename IN>
__global__ void __launch_bounds__(128) join64_kernel(const Params<IN> p, const double* __restrict__ part_out,
                                                     const double* __restrict__ part_rc, double* __restrict__ stats) {
  const int64_t i = (int64_t)blockIdx.x * 4 + threadIdx.x / 32, all = (int64_t)p.H * p.N;
  const int lane = threadIdx.x % 32;
  if (i >= all) return;
  const int h = (int)(i % p.H), row = (int)(i / p.H);
  const int64_t at = (int64_t)h * p.N + row, out = ((int64_t)row * p.H + h) * p.D;
  const bool mine = lane < p.splits;
  const double r = row_sum<32>(mine ? part_rc[2 * (int64_t)lane * all + at] : 0.0);
  const double u = row_sum<32>(mine ? part_rc[(2 * (int64_t)lane + 1) * all + at] : 0.0);
  for (int d = lane; d < p.D; d += 32) {
    double v = 0.0;
#pragma unroll 4
    for (int z = 0; z < p.splits; ++z) v += part_out[z * all * p.D + out + d];
    p.out3[out + d] = (IN)(v - r * (double)p.o[(int64_t)row * p.os + h * p.oh + d]);
  }
  if (lane == 0) {
    stats[all + at] = r;
    stats[2 * all + at] = u - stats[at] * r;
  }
}

// out = the splits' 64-bit partial results added in their order; a second result's splits follow the first's
template <typename IN>
__global__ void __launch_bounds__(256) sum64_kernel(int64_t n, int splits, const double* __restrict__ work, IN* __restrict__ out0,
                                                    IN* __restrict__ out1) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  work += blockIdx.y * splits * n;
  double a = 0.0;
#pragma unroll 4
  for (int z = 0; z < splits; ++z) a += work[z * n + i];
  (blockIdx.y ? out1 : out0)[i] = (IN)a;
}

template <class S, typename IN>
__global__ void __launch_bounds__(S::THREADS) keys64_kernel(const Params<IN> p, double* __restrict__ part_out, const double* __restrict__ stats) {
  extern __shared__ __align__(16) double smem64[];
  Part part;
  if (!find_part<32>(p, blockIdx.x, part)) return;
  const Lane<S> l(row_length<IN>(p.D));
  const int hk = blockIdx.y, group = p.H / p.HK;
  IN *sK = reinterpret_cast<IN*>(smem64), *sV = sK + 32 * l.ld, *sB = sV + 32 * l.ld, *sC = sB + 32 * l.ld, *sQ = sC + 32 * l.ld,
     *sO = sQ + S::TILE * l.ld, *sA = sO + S::TILE * l.ld;
  int lo = part.lo, hi = part.keys ? part.hi : part.lo;
  split_range<S::TILE>(lo, hi, blockIdx.z, p.splits_k);
  const double scale = (double)p.scale, c2 = scale * log2e<double>();
  const int64_t all = (int64_t)p.H * p.N;
  bool ok[S::RB];
  double one[S::RB];
  Sums<S> dk, dv;
  clear<S>(dk);
  clear<S>(dv);
#pragma unroll
  for (int rb = 0; rb < S::RB; ++rb) {
    ok[rb] = may(part.row + l.own(rb), part.hi, p.mask);
    one[rb] = 1.0;
  }
  if (lo < hi) {
    copy_rows<S::THREADS>(sK, l.ld, p.k + hk * p.kh, p.ks, p.kh, part.row, 32, part.hi, p.D, p.mask);
    copy_rows<S::THREADS>(sV, l.ld, p.v + hk * p.vh, p.vs, p.vh, part.row, 32, part.hi, p.D, p.mask);
    copy_rows<S::THREADS>(sB, l.ld, p.cb + hk * p.cbh, p.cbs, p.cbh, part.row, 32, part.hi, p.D, p.mask);
    copy_rows<S::THREADS>(sC, l.ld, p.cc + hk * p.cch, p.ccs, p.cch, part.row, 32, part.hi, p.D, p.mask);
  }
  const auto next_qa = [&](int h, int q0) {
    if (q0 < hi) {
      copy_rows<S::THREADS>(sQ, l.ld, p.q + h * p.qh, p.qs, p.qh, q0, S::TILE, hi, p.D);
      copy_rows<S::THREADS>(sA, l.ld, p.ca + h * p.cah, p.cas, p.cah, q0, S::TILE, hi, p.D);
    }
    end_group();
  };
  const auto next_o = [&](int h, int q0) {
    if (q0 < hi) copy_rows<S::THREADS>(sO, l.ld, p.go + h * p.goh, p.gos, p.goh, q0, S::TILE, hi, p.D);
    end_group();
  };
  next_o(hk * group, lo);
  next_qa(hk * group, lo);
  for (int gh = 0; gh < group; ++gh) {
    const int h = hk * group + gh;
    for (int q0 = lo; q0 < hi; q0 += S::TILE) {
      const bool last = q0 + S::TILE >= hi;                                // the next tile is the next head's first, or none
      const int h1 = last ? h + 1 : h, q1 = !last ? q0 + S::TILE : gh + 1 < group ? lo : hi;
      arrive<1>();
      Scores<S> s, t, dp, e;
      zero<S>(s);
      zero<S>(t);
      zero<S>(dp);
      zero<S>(e);
      scores<S>(dp, l, sV, sO, p.D);
      scores<S>(e, l, sC, sO, p.D);
      arrive<0>();
      scores<S>(s, l, sK, sQ, p.D);
      scores<S>(t, l, sK, sA, p.D);
      scores<S>(t, l, sB, sQ, p.D);
#pragma unroll
      for (int nt = 0; nt < S::NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int row = q0 + l.col(nt) + 2 * l.t + x;
          const bool in = row < hi;
          const int64_t at = (int64_t)h * p.N + (in ? row : q0);
          const double L = (double)p.lse[at], D = stats[at], r = stats[all + at], c = stats[2 * all + at];
#pragma unroll
          for (int rb = 0; rb < S::RB; ++rb) {
            const bool on = in && ok[rb];
            const double pr = on ? exp2(s[rb][nt][x] * c2 - L) : 0.0, tt = t[rb][nt][x] * scale - r, d = dp[rb][nt][x] - D;
            s[rb][nt][x] = on ? pr * (tt * d + e[rb][nt][x] - c) : 0.0;
            t[rb][nt][x] = on ? pr * d : 0.0;
            dp[rb][nt][x] = on ? pr * tt : 0.0;
          }
        }
      sums<S>(dv, l, dp, sO, p.D);
      __syncthreads();
      next_o(h1, q1);
      sums<S>(dk, l, s, sQ, p.D);
      sums<S>(dk, l, t, sA, p.D);
      __syncthreads();
      next_qa(h1, q1);
    }
  }
  hide<S>(dk, ok);
  hide<S>(dv, ok);
  const int64_t n = (int64_t)p.N * p.HK * p.D, at = ((int64_t)part.row * p.HK + hk) * p.D;
  const int rows = min(32, part.hi - part.row);
  if (p.splits_k == 1) {
    join_rows<S, IN>(smem64, l, dk, one, p.out1 + at, (int64_t)p.HK * p.D, rows, p.D, scale);
    join_rows<S, IN>(smem64, l, dv, one, p.out2 + at, (int64_t)p.HK * p.D, rows, p.D, 1.0);
  } else {
    join_rows<S, double>(smem64, l, dk, one, part_out + blockIdx.z * n + at, (int64_t)p.HK * p.D, rows, p.D, scale);
    join_rows<S, double>(smem64, l, dv, one, part_out + (p.splits_k + blockIdx.z) * n + at, (int64_t)p.HK * p.D, rows, p.D, 1.0);
  }
}

// ------------------------------------------------------------------------------------------ launches
// shared memory: the tiles, or the KG partial results that replace them in the end
template <class S, typename IN>
size_t smem_bytes(int D, int own, int streamed) {
  const size_t tiles = sizeof(IN) * row_length<IN>(D) * (own * 32 + streamed * S::TILE), ends = sizeof(double) * row_length<double>(D) * S::KG * 32;
  return tiles > ends ? tiles : ends;
}

template <class S, auto KERNEL, typename T, typename... A>
cudaError_t launch64(const Params<T>& p, int heads, int splits, int own, int streamed, cudaStream_t s, A... more) {
  const size_t bytes = smem_bytes<S, T>(p.D, own, streamed);
  const cudaError_t e = raise_smem_limit<KERNEL>(232448 - 4096);       // the kernels' own static arrays stay below 4 KB
  if (e != cudaSuccess) return e;
  KERNEL<<<dim3(part_blocks(p, 32), heads, splits), S::THREADS, bytes, s>>>(p, more...);
  return cudaGetLastError();
}

#define XNN_F64_DIM(D_, ...)                              \
  if ((D_) <= 32) { constexpr int DP = 32; __VA_ARGS__; } \
  if ((D_) <= 64) { constexpr int DP = 64; __VA_ARGS__; } \
  { constexpr int DP = 128; __VA_ARGS__; }

}  // namespace

// Two blocks of rows a warp read less of the streamed tile, one leaves registers for twice the warps: 16 an SM instead of 8
// at 65-128 columns, where the forward pass takes 259 us instead of 391 (1500 atoms x 4 heads x 96). At 33-64 columns the
// forward pass (two blocks of eight warps fit) is 4% faster with two, the others up to a quarter slower.
template <int DP, int NT, int FROM>
using Rows64 = std::conditional_t<DP >= FROM, Shape<DP, 1, 4, 4, NT>, Shape<DP, 2, 2, 4, NT>>;

cudaError_t forward64(const Params<double>& p, cudaStream_t s) {
  XNN_F64_DIM(p.D, using S = Rows64<DP, 2, 128>; return (launch64<S, fwd64_kernel<S>>(p, p.H, p.splits, 1, 2, s)))
}

cudaError_t backward64(const Params<double>& p, cudaStream_t s) {
  delta64_kernel<double><<<(unsigned)(((int64_t)p.H * p.N + 3) / 4), 128, 0, s>>>(p, p.delta);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  // two sums of 128 columns leave no registers for more than eight warps
  XNN_F64_DIM(p.D, using S = Rows64<DP, 2, 64>; using K = std::conditional_t<DP == 64, Shape<DP, 1, 4, 4, 2>, Shape<DP, 1, 4, 2, 4>>;
              if ((e = launch64<S, dq64_kernel<S>>(p, p.H, p.splits, 2, 2, s)) != cudaSuccess) return e;
              return (launch64<K, dkv64_kernel<K>>(p, p.HK, p.splits_k, 2, 2, s)))
}

// 64-bit words: D, r, c; the splits' r and c; the splits' results over keys, and over queries
template <typename IN>
int64_t second64_words(const Params<IN>& p) {
  const int64_t rows = (int64_t)p.H * p.N;
  const int64_t over_k = (int64_t)p.splits * rows * p.D, over_q = p.splits_k > 1 ? 2 * (int64_t)p.splits_k * p.HK * p.N * p.D : 0;
  return 3 * rows + 2 * p.splits * rows + (over_k > over_q ? over_k : over_q);
}

template <typename IN, int DP, bool NARROW>
cudaError_t second64_dp(const Params<IN>& p, double* work, cudaStream_t s) {
  // float64 of 113 .. 128 columns: three slices of the keys and half the queries a tile, so that seven tiles fit
  using R = std::conditional_t<NARROW, Shape<DP, 1, 4, 3, 1>, Rows64<DP, 1, 64>>;
  using K = std::conditional_t<DP == 64, Shape<DP, 1, 4, 4, 1>, Shape<DP, 1, 4, 2, NARROW ? 1 : 2>>;
  const int64_t rows = (int64_t)p.H * p.N, nq = rows * p.D, nk = (int64_t)p.N * p.HK * p.D;
  double *stats = work, *rc = stats + 3 * rows, *out = rc + 2 * p.splits * rows;
  const unsigned row_warps = (unsigned)((rows + 3) / 4);
  delta64_kernel<IN><<<row_warps, 128, 0, s>>>(p, stats);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  if ((e = launch64<R, rows64_kernel<R, IN, 0>>(p, p.H, p.splits, 3, 4, s, out, rc, (const double*)stats)) != cudaSuccess) return e;
  join64_kernel<IN><<<row_warps, 128, 0, s>>>(p, out, rc, stats);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  if ((e = launch64<R, rows64_kernel<R, IN, 1>>(p, p.H, p.splits, 3, 4, s, out, rc, (const double*)stats)) != cudaSuccess) return e;
  if (p.splits > 1) {
    sum64_kernel<IN><<<dim3((unsigned)((nq + 255) / 256)), 256, 0, s>>>(nq, p.splits, out, p.out0, nullptr);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
  }
  if ((e = launch64<K, keys64_kernel<K, IN>>(p, p.HK, p.splits_k, 4, 3, s, out, (const double*)stats)) != cudaSuccess) return e;
  if (p.splits_k > 1)
    sum64_kernel<IN><<<dim3((unsigned)((nk + 255) / 256), 2), 256, 0, s>>>(nk, p.splits_k, out, p.out1, p.out2);
  return cudaGetLastError();
}

template <typename IN>
cudaError_t second64(const Params<IN>& p, double* work, cudaStream_t s) {
  if constexpr (sizeof(IN) == 4) {
    return second64_dp<IN, 128, false>(p, work, s);      // up to 64 columns are attention_tc_second.cu's
  } else {
    if (p.D > 112) return second64_dp<IN, 128, true>(p, work, s);
    XNN_F64_DIM(p.D, return (second64_dp<IN, DP, false>(p, work, s)))
  }
}

template int64_t second64_words<float>(const Params<float>&);
template int64_t second64_words<double>(const Params<double>&);
template cudaError_t second64<float>(const Params<float>&, double*, cudaStream_t);
template cudaError_t second64<double>(const Params<double>&, double*, cudaStream_t);

}  // namespace attn
