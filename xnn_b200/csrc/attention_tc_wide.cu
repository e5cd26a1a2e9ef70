// The backward pass of structure attention on the tensor cores for 65 .. 128 columns a head.
//
// At that width tensor memory does not hold the parts of two operands and the results of both dk and dv. One kernel
// in three modes keeps the first operand's parts there and the second's in shared memory, and streams halves of images:
//   DQ  a block owns 128 queries:  dS = P (dP - D) over keys,     out = dS K     (first q, second do; K, V)
//   DK  a block owns 128 keys:     dS^T over queries,             out = dS^T Q   (first k, second v; Q, do)
//   DV  a block owns 128 keys:     P^T over queries,              out = P^T do   (first k; Q, do)
// S is formed three times instead of twice (8 products instead of 7), which costs less than a smaller tile would.
// Scores of the next tile run while the rows' threads form the weights of this one.
#include "attention.h"
#include "attention_tc.cuh"

namespace attn {
namespace {

enum Mode { DQ, DK, DV };

template <int DP, int MODE>
struct Wide {
  static constexpr int HB = half_bytes<DP>();
  // a ring of three for the images that the sums read too, of two for the others
  static constexpr int SECOND = MODE == DV ? 0 : PLANES * 128 * DP * 2, Y = SECOND, X = Y + 3 * HB, ST = X + 2 * HB,
                       BARS = ST + 3 * 2 * HALF * 4, SMEM = BARS + 128;
  static constexpr int S = 3 * DP / 2, T = S + HALF, W = T + HALF, OUT = W + 3 * HALF / 2;
  static_assert(OUT + DP <= 512 && SMEM <= 232448, "tensor and shared memory");
};

// first, second: images of the owned rows' operands, a, b: of the streamed ones
template <int DP, int MODE>
__device__ __forceinline__ void wide_block(const Params<float>& p, const Part& part, const Job& job, const Images& first,
                                           const Images& second, const Images& a, const Images& b, const float* __restrict__ stats,
                                           int* status) {
  using B = Wide<DP, MODE>;
  extern __shared__ __align__(128) char smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + B::BARS);
  uint64_t *full_x = bars, *full_y = bars + 2, *full_2 = bars + 5, *scored = bars + 6, *summed = bars + 7, *taken = bars + 8,
           *ready = bars + 9;
  uint32_t* slot = reinterpret_cast<uint32_t*>(bars + 10);
  volatile int* dead = reinterpret_cast<volatile int*>(bars + 11);
  const int warp = threadIdx.x / 32, group = p.H / p.HK, own = job.head;
  int lo = part.lo, hi = part.keys ? part.hi : part.lo;
  split_range<SLOT>(lo, hi, job.split, job.splits);
  const int tiles = (hi - lo + HALF - 1) / HALF, n = MODE == DQ ? tiles : tiles * group;
  const int slot0 = first_slot(p, part) + (lo - part.lo) / SLOT, own_slot = first_slot(p, part) + (part.row - part.lo) / SLOT;
  if (warp == 8) tmem_alloc(slot, 512);
  if (threadIdx.x == 0) {
    for (int i = 0; i < 8; ++i) tc::mbar_init(bars + i, 1);
    tc::mbar_init(taken, 8);
    tc::mbar_init(ready, 8);
    tc::mbar_init(bars + DRAINED, 1);
    *dead = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *slot;
  // the images of tile i: the sums read b (do) for dv, a otherwise
  const auto load = [&](int i, bool y) {
    if (elect()) {
      const int head = MODE == DQ ? own / group : own * group + i / tiles, t = MODE == DQ ? i : i % tiles;
      uint64_t* bar = y ? full_y + i % 3 : full_x + i % 2;
      char* to = smem + (y ? B::Y + i % 3 * B::HB : B::X + i % 2 * B::HB);
      const bool with_stats = y && MODE != DQ;
      tc::mbar_arrive_expect_tx(bar, B::HB + (with_stats ? 2 * HALF * 4 : 0));
      load_half<DP>(to, image<DP>(y == (MODE == DV) ? b : a, head, slot0 + t / 2), t % 2, bar);
      if (with_stats) {
        const float* st = stats + ((int64_t)head * a.slots + slot0 + t / 2) * 2 * SLOT + t % 2 * HALF;
        char* at = smem + B::ST + i % 3 * (2 * HALF * 4);
        tc::bulk_g2s(at, st, HALF * 4, bar);
        tc::bulk_g2s(at + HALF * 4, st + SLOT, HALF * 4, bar);
      }
    }
  };
  int loaded_x = min(n, 2), loaded_y = min(n, 3);
  if (warp == 8 && n > 0) {                             // the copies run while the other warps stage their rows
    if (MODE != DV && elect()) {
      tc::mbar_arrive_expect_tx(full_2, B::SECOND);
      load_block<DP>(smem, image<DP>(second, own, own_slot), full_2);
    }
    __syncwarp();
    for (int i = 0; i < loaded_x; ++i) load(i, false);
    for (int i = 0; i < loaded_y; ++i) load(i, true);
  } else if (n > 0) {
    stage_image<DP, DP / 2>(tmem + ((uint32_t)(warp & 3) << 21), image<DP>(first, own, own_slot), threadIdx.x & 127,
                            warp / 4 * (DP / 2));
    tmem_st_wait();
    tc::tc_fence_before();
  }
  __syncthreads();
  tc::tc_fence_after();

  if (warp == 8) {
    if (n > 0) {
      const uint32_t base = tc::smem_u32(smem);
      const auto scores = [&](int i) {
        if (elect()) {
          const uint32_t x = base + B::X + i % 2 * B::HB, y = base + B::Y + i % 3 * B::HB;
          mma_scores<DP, HALF>(tmem + B::S, tmem, MODE == DV ? x : y);
          if (MODE != DV) mma_scores_ss<DP, HALF>(tmem + B::T, base, x);
          tc::commit_to(scored);
        }
      };
      bool ok = (MODE == DV || wait_all(full_2, 0, dead, status)) && wait_all(full_x, 0, dead, status) &&
                (MODE == DV || wait_all(full_y, 0, dead, status));
      if (ok) scores(0);
      for (int i = 0; ok && i < n; ++i) {
        if (!(ok = wait_all(taken, i & 1, dead, status))) break;
        tc::tc_fence_after();
        if (i + 2 < n) { load(i + 2, false); loaded_x = i + 3; }
        if (i + 1 < n) {
          if (!(ok = wait_all(full_x + (i + 1) % 2, ((i + 1) / 2) & 1, dead, status))) break;
          if (MODE != DV && !(ok = wait_all(full_y + (i + 1) % 3, ((i + 1) / 3) & 1, dead, status))) break;
          scores(i + 1);
        }
        if (!(ok = wait_all(ready, i & 1, dead, status))) break;
        tc::tc_fence_after();
        if (i > 0 && i + 2 < n) { load(i + 2, true); loaded_y = i + 3; }      // the sums of tile i - 1 are done
        if (!(ok = wait_all(full_y + i % 3, (i / 3) & 1, dead, status))) break;
        if (elect()) {
          mma_sums<DP, HALF, Linear<HALF / 2>>(tmem + B::OUT, tmem + B::W, base + B::Y + i % 3 * B::HB);
          tc::commit_to(summed);
        }
      }
      if (!ok) {                                        // copies in flight must land before the block ends
        if (MODE != DV) tc::mbar_wait(full_2, 0, SPINS);
        for (int i = max(0, loaded_x - 2); i < loaded_x; ++i) tc::mbar_wait(full_x + i % 2, (i / 2) & 1, SPINS);
        for (int i = max(0, loaded_y - 3); i < loaded_y; ++i) tc::mbar_wait(full_y + i % 3, (i / 3) & 1, SPINS);
      }
    }
    drain(bars + DRAINED);
  } else {
    const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);
    const int half = warp / 4, row = part.row + (threadIdx.x & 127);
    const bool on = row < part.hi;
    const float c2 = p.scale * log2e<float>();
    float L = -neg_inf<float>(), D = 0.f, acc[DP / 2];
    if (MODE == DQ && on && n > 0) {
      const float* at = stats + ((int64_t)own * a.slots + first_slot(p, part) + (row - part.lo) / SLOT) * 2 * SLOT;
      L = at[(row - part.lo) % SLOT];
      D = at[SLOT + (row - part.lo) % SLOT];
    }
#pragma unroll
    for (int d = 0; d < DP / 2; ++d) acc[d] = 0.f;
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const uint32_t bits = MODE == DQ ? allowed_half(lo + i * HALF, hi, p.mask) >> (16 * half) : 0;
      if (!(ok = wait_all(scored, i & 1, dead, status))) break;
      if (MODE != DQ && !(ok = wait_all(full_y + i % 3, (i / 3) & 1, dead, status))) break;
      tc::tc_fence_after();
      float s[16], dp[16];
      tmem_ld16(lanes + B::S + 16 * half, s);
      if (MODE != DV) tmem_ld16(lanes + B::T + 16 * half, dp);
      tmem_ld_wait();
      tc::tc_fence_before();
      arrive(taken);
      if (MODE == DQ) {
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = (bits >> j) & 1 ? ex2(fmaf(s[j], c2, -L)) * (dp[j] - D) : 0.f;
      } else {
        const float* st = reinterpret_cast<const float*>(smem + B::ST + i % 3 * (2 * HALF * 4)) + 16 * half;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          s[j] = ex2(fmaf(s[j], c2, -st[j]));
          if (MODE == DK) s[j] *= dp[j] - st[HALF + j];
        }
      }
      if (i > 0) {
        if (!(ok = wait_all(summed, (i - 1) & 1, dead, status))) break;
        tc::tc_fence_after();
        add_columns<DP / 2>(lanes + B::OUT + half * (DP / 2), acc);
      }
      store_parts16<Linear<HALF / 2>>(lanes + B::W, half, s);
      tmem_st_wait();
      tc::tc_fence_before();
      arrive(ready);
    }
    if (ok && n > 0 && (ok = wait_all(summed, (n - 1) & 1, dead, status))) {
      tc::tc_fence_after();
      add_columns<DP / 2>(lanes + B::OUT + half * (DP / 2), acc);
    }
    const bool hidden = MODE != DQ && on && p.mask != nullptr && !p.mask[row];
#pragma unroll
    for (int d = 0; d < DP / 2; ++d) acc[d] = hidden ? 0.f : MODE == DV ? acc[d] : p.scale * acc[d];
    const int heads = MODE == DQ ? p.H : p.HK, row0 = part.row + 32 * (warp & 3);
    const int64_t all = (int64_t)p.N * heads * p.D;
    float* out = MODE == DQ ? p.out0 : MODE == DK ? p.out1 : p.out2;
    if (job.splits > 1) out = (MODE == DQ ? p.work : p.work_k) + ((MODE == DV ? job.splits : 0) + (int64_t)job.split) * all;
    store_rows<DP / 2>(scratch_of<DP / 2>(smem, warp), acc, out + ((int64_t)row0 * heads + own) * p.D, (int64_t)heads * p.D,
                       min(32, part.hi - row0), half * (DP / 2), p.D, ok);
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc::tc_fence_after();
    tmem_free(tmem, 512);
  }
}

// the three in one launch: the blocks of the keys first
template <int DP>
__global__ void __launch_bounds__(ROW_THREADS, 1) wide_kernel(const Params<float> p, const Images k, const Images v, const Images q,
                                                              const Images o, const float* __restrict__ stats, int* status) {
  const int tiles = part_blocks(p, 128), rest = blockIdx.x / tiles, keys = p.HK * p.splits_k;
  Part part;
  if (!find_part<128>(p, blockIdx.x % tiles, part)) return;
  const Job job{rest % keys % p.HK, rest % keys / p.HK, p.splits_k};
  if (rest < keys) wide_block<DP, DK>(p, part, job, k, v, q, o, stats, status);
  else if (rest < 2 * keys) wide_block<DP, DV>(p, part, job, k, v, q, o, stats, status);
  else wide_block<DP, DQ>(p, part, {(rest - 2 * keys) % p.H, (rest - 2 * keys) / p.H, p.splits}, q, o, k, v, stats, status);
}

}  // namespace

cudaError_t tc_wide_backward(const Params<float>& p, char* work, int* status, cudaStream_t s) {
  constexpr int DP = 128, SMEM = Wide<DP, DQ>::SMEM;     // of the three the first two need most
  const int slots = image_slots(p);
  char *ik = work, *iv = ik + image_bytes<DP>(p, p.HK), *iq = iv + image_bytes<DP>(p, p.HK), *io = iq + image_bytes<DP>(p, p.H);
  const float* stats = reinterpret_cast<const float*>(io + image_bytes<DP>(p, p.H));
  const cudaError_t e = raise_smem_limit<wide_kernel<DP>>(SMEM);
  if (e != cudaSuccess) return e;
  const int64_t blocks = (int64_t)(part_blocks(p, 128)) * (2 * p.HK * p.splits_k + p.H * p.splits);
  wide_kernel<DP><<<(unsigned)blocks, ROW_THREADS, SMEM, s>>>(p, Images{ik, slots}, Images{iv, slots}, Images{iq, slots},
                                                             Images{io, slots}, stats, status);
  return cudaGetLastError();
}

}  // namespace attn
