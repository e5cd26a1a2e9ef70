// Dropout from a counter-based generator: the keep mask of an element is a function of (seed, offset,
// element number), so the backward pass forms it again and no mask is stored.
//
// The generator is Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", SC 2011): key = the seed's two words, counter = (block, block >> 32, offset, offset >> 32) with
// block = element / 4; word element % 4 of the result is compared with floor(p 2^32).
//
// x is (outer, shared, inner); one mask entry serves all `shared` copies of (outer, inner). Per four
// entries the ten rounds are some 80 integer instructions; the passes stay bound by memory (one read and
// one write of x), so a thread forms four words once and walks its share of the copies with them.
#include "common.cuh"

namespace {

struct alignas(16) Words { uint32_t w[4]; };

__device__ __forceinline__ Words philox(uint64_t block, uint64_t offset, uint64_t seed) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Words{{c0, c1, c2, c3}};
}

template <typename T> struct alignas(16) Four { T x[4]; };

// y = keep ? factor x : 0 (a select: what is dropped is zero whatever it was). VEC: the four elements of
// a block are neighbours in memory on 16-byte boundaries (without sharing, all but a last incomplete block of any tensor).
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dropout_kernel(int64_t n, int64_t inner, int shared, int copies, uint64_t threshold,
                                                      T factor, const int64_t* __restrict__ rng,
                                                      const T* __restrict__ x, T* __restrict__ y) {
  const int64_t block = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t e0 = block * 4;
  if (VEC && e0 >= n) return;
  const Words bits = philox((uint64_t)block, (uint64_t)rng[1], (uint64_t)rng[0]);
  const int s0 = blockIdx.y * copies, s1 = min(shared, s0 + copies);
  if constexpr (VEC) {
    if (shared == 1 && e0 + 4 > n) {                     // the last block of a tensor whose size is no multiple of four
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (e0 + e < n) y[e0 + e] = bits.w[e] >= threshold ? x[e0 + e] * factor : T(0);
      return;
    }
    const int64_t o = shared == 1 ? 0 : e0 / inner, i = e0 - o * inner;
    const int64_t base = o * shared * inner + i;
#pragma unroll 4
    for (int s = s0; s < s1; ++s) {
      Four<T> v = *reinterpret_cast<const Four<T>*>(x + base + s * inner);
#pragma unroll
      for (int e = 0; e < 4; ++e) v.x[e] = bits.w[e] >= threshold ? v.x[e] * factor : T(0);
      *reinterpret_cast<Four<T>*>(y + base + s * inner) = v;
    }
  } else {
    // a warp's 128 entries go round, so that lane l has the entries l, l + 32, l + 64, l + 96 and whole lines are moved
    // (8000 x 49 x 127 floats: 117 us, 164 with a thread's four entries as neighbours)
    const int lane = threadIdx.x & 31;
    const int64_t first = e0 - 4 * lane;
    bool keep[4], in[4];
    int64_t at[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t w = 0;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint32_t u = __shfl_sync(0xffffffffu, bits.w[c], 8 * e + lane / 4);
        w = (lane & 3) == c ? u : w;
      }
      const int64_t entry = first + 32 * e + lane, k = entry < n ? entry : n - 1, o = shared == 1 ? 0 : k / inner;
      keep[e] = w >= threshold;
      in[e] = entry < n;
      at[e] = (o * shared + s0) * inner + (k - o * inner);
    }
#pragma unroll 4
    for (int s = s0; s < s1; ++s) {
      T v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = x[at[e]];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (in[e]) y[at[e]] = keep[e] ? v[e] * factor : T(0);
        at[e] += inner;
      }
    }
  }
}

}  // namespace

template <typename T>
cudaError_t counter_dropout(int64_t outer, int64_t shared, int64_t inner, double p, const int64_t* rng, const T* x, T* y,
                            cudaStream_t s) {
  const int64_t n = outer * inner, blocks = (n + 3) / 4, ctas = (blocks + 255) / 256;
  const bool vec = (shared == 1 || inner % 4 == 0) && reinterpret_cast<uintptr_t>(x) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(y) % 16 == 0;
  // enough blocks for eight a multiprocessor; beyond that a thread keeps its words for several copies
  const int64_t want = (148 * 8 + ctas - 1) / ctas;
  const int parts = (int)(want < shared ? want : shared);
  const int copies = (int)((shared + parts - 1) / parts);
  const dim3 grid((unsigned)ctas, (unsigned)((shared + copies - 1) / copies));
  const uint64_t threshold = (uint64_t)(p * 4294967296.0);          // 2^32 at p = 1: nothing is kept
  const T factor = p < 1.0 ? (T)(1.0 / (1.0 - p)) : T(0);
  if (vec)
    dropout_kernel<T, true><<<grid, 256, 0, s>>>(n, inner, (int)shared, copies, threshold, factor, rng, x, y);
  else
    dropout_kernel<T, false><<<grid, 256, 0, s>>>(n, inner, (int)shared, copies, threshold, factor, rng, x, y);
  return cudaGetLastError();
}
template cudaError_t counter_dropout<float>(int64_t, int64_t, int64_t, double, const int64_t*, const float*, float*, cudaStream_t);
template cudaError_t counter_dropout<double>(int64_t, int64_t, int64_t, double, const int64_t*, const double*, double*, cudaStream_t);
