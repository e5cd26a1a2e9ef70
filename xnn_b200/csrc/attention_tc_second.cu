// The second derivative of structure attention on the tensor cores, up to 64 columns a head (formulas: attention.cu).
//
// rows   a block owns 128 queries with the parts of q, A and do in tensor memory and streams halves of the images of
//        k, v, B, C. Walk 0 forms r = sum P T, sum P (T dP + E) and sum_j (P T) V + P C; walk 1 the products of q'.
//        Between them a small kernel joins the splits: r, c and do' = sum - r O.
// keys   a block owns 128 keys with the parts of k and B in tensor memory, those of v and C in shared memory, and streams
//        q, do and A: k' and v'.
// The weights' parts take the scores' place in tensor memory. At 64 columns that memory is full: the score products of a
// tile follow the sums of the tile before in one stretch, and the threads' work is not hidden under them. Up to 32 columns
// it holds two sets of scores, and those of the next tile run while the threads form the weights of this one.
#include "attention.h"
#include "attention_tc.cuh"

namespace attn {
namespace {

constexpr int KINDS = 4;                                // L, D, r, c of a slot's rows

template <int DP> constexpr int SETS = DP <= 32 ? 2 : 1;  // sets of scores in tensor memory
template <int DP> constexpr int RING = SETS<DP> + 2;      // images: of the tiles with scores, of the sums before, on the way

struct Streams { Images a, b, c, d; };

// the end of the part's last slot
__device__ __forceinline__ int slots_end(const Part& part) { return part.lo + (part.hi - part.lo + SLOT - 1) / SLOT * SLOT; }

template <int DP>
struct Rows {
  static constexpr int HB = half_bytes<DP>(), STAGE = 4 * HB, BARS = RING<DP> * STAGE, SUMS = BARS + 128, SMEM = SUMS + 4 * 128 * 4;
  static constexpr int P = 3 * DP / 2, S = 3 * P, T = S + HALF, DPO = T + HALF, E = DPO + HALF, W0 = S, W1 = DPO, SET = 4 * HALF,
                       OUT = S + SETS<DP> * SET;
  using Weights = OverHalves<0, 8, HALF>;               // two planes over S or dP, one over T or E, each half over its own
  static_assert(OUT + DP <= 512 && SMEM <= 232448, "tensor and shared memory");
};

// copies in flight must land before the block ends
template <int DP>
__device__ __forceinline__ void give_up(int loaded, uint64_t* full, uint64_t* more = nullptr) {
  if (more) tc::mbar_wait(more, 0, SPINS);
  for (int i = max(0, loaded - RING<DP>); i < loaded; ++i) tc::mbar_wait(full + i % RING<DP>, i / RING<DP> & 1, SPINS);
}

// The ninth warp's turns. Products run in the order of their issue, so the scores of tile i + SETS may be issued behind the
// sums of tile i, whose weights they overwrite; the weights of tile i come after the threads have the sums of tile i - 1,
// whose images are then free.
template <int DP, class Load, class Score, class Sum>
__device__ __forceinline__ void issue(int n, int loaded, uint64_t* full, uint64_t* ready, volatile int* dead, int* status, const Load& load,
                                      const Score& score, const Sum& sum) {
  bool ok = true;
  for (int i = 0; ok && i < SETS<DP> && i < n; ++i)
    if ((ok = wait_all(full + i, 0, dead, status))) score(i);
  for (int i = 0; ok && i < n; ++i) {
    if (!(ok = wait_all(ready, i & 1, dead, status))) break;
    tc::tc_fence_after();
    sum(i);
    const int next = i + SETS<DP>;
    if (next < n) {
      if (!(ok = wait_all(full + next % RING<DP>, next / RING<DP> & 1, dead, status))) break;
      score(next);
    }
    if (i > 0 && i - 1 + RING<DP> < n) { load(i - 1 + RING<DP>); loaded = i + RING<DP>; }
  }
  if (!ok) give_up<DP>(loaded, full);
}

template <int DP, int WALK>
__device__ __forceinline__ void rows_block(const Params<float>& p, const Part& part, const Job& job, const Streams& im, const Streams& own,
                                           float* __restrict__ stats, float* __restrict__ parts, int* status) {
  using B = Rows<DP>;
  constexpr int HB = B::HB;
  extern __shared__ __align__(128) char smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + B::BARS);
  uint64_t *full = bars, *scored = bars + 4, *summed = bars + 6, *ready = bars + 7;
  uint32_t* slot = reinterpret_cast<uint32_t*>(bars + 9);
  volatile int* dead = reinterpret_cast<volatile int*>(bars + 10);
  float* sums = reinterpret_cast<float*>(smem + B::SUMS);
  const int warp = threadIdx.x / 32, h = job.head, hk = h / (p.H / p.HK);
  int lo = part.lo, hi = part.keys ? part.hi : part.lo;
  split_range<SLOT>(lo, hi, job.split, job.splits);
  const int n = (hi - lo + HALF - 1) / HALF, slot0 = first_slot(p, part) + (lo - part.lo) / SLOT;
  if (warp == 8) tmem_alloc(slot, 512);
  if (threadIdx.x == 0) {
    for (int i = 0; i < 7; ++i) tc::mbar_init(bars + i, 1);
    tc::mbar_init(ready, 8);
    tc::mbar_init(bars + DRAINED, 1);
    *dead = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *slot, lanes = tmem + ((uint32_t)(warp & 3) << 21);
  const int row = part.row + (threadIdx.x & 127), half = warp / 4;
  const bool on = warp < 8 && row < part.hi;
  const auto load = [&](int i) {
    if (elect()) {
      char* to = smem + i % RING<DP> * B::STAGE;
      uint64_t* bar = full + i % RING<DP>;
      tc::mbar_arrive_expect_tx(bar, B::STAGE);
      load_half<DP>(to, image<DP>(im.a, hk, slot0 + i / 2), i % 2, bar);
      load_half<DP>(to + HB, image<DP>(im.b, hk, slot0 + i / 2), i % 2, bar);
      load_half<DP>(to + 2 * HB, image<DP>(im.c, hk, slot0 + i / 2), i % 2, bar);
      load_half<DP>(to + 3 * HB, image<DP>(im.d, hk, slot0 + i / 2), i % 2, bar);
    }
  };
  int loaded = min(n, RING<DP>);
  if (warp == 8) {                                      // the copies run while the other warps stage their rows
    for (int i = 0; i < loaded; ++i) load(i);
  } else if (n > 0) {
    const int mine = first_slot(p, part) + (part.row - part.lo) / SLOT;   // own: q, A and do
    if (half == 0) {
      stage_image<DP>(lanes, image<DP>(own.a, h, mine), threadIdx.x & 127);
    } else {
      stage_image<DP>(lanes + B::P, image<DP>(own.b, h, mine), threadIdx.x & 127);
    }
    stage_image<DP, DP / 2>(lanes + 2 * B::P, image<DP>(own.c, h, mine), threadIdx.x & 127, half * (DP / 2));
    tmem_st_wait();
    tc::tc_fence_before();
  }
  __syncthreads();
  tc::tc_fence_after();
  bool ok = true;
  float acc[DP / 2], R = 0.f, U = 0.f;
#pragma unroll
  for (int d = 0; d < DP / 2; ++d) acc[d] = 0.f;

  if (warp == 8) {
    if (n > 0) {
      const uint32_t base = tc::smem_u32(smem);
      const auto score = [&](int i) {
        if (elect()) {
          const uint32_t at = base + i % RING<DP> * B::STAGE, set = tmem + i % SETS<DP> * B::SET;
          mma_scores<DP, HALF>(set + B::S, tmem, at);
          mma_scores<DP, HALF>(set + B::T, tmem + B::P, at, tmem, at + 2 * HB);
          mma_scores<DP, HALF>(set + B::DPO, tmem + 2 * B::P, at + HB);
          mma_scores<DP, HALF>(set + B::E, tmem + 2 * B::P, at + 3 * HB);
          tc::commit_to(scored + i % SETS<DP>);
        }
      };
      const auto sum = [&](int i) {
        if (elect()) {
          const uint32_t at = base + i % RING<DP> * B::STAGE, set = tmem + i % SETS<DP> * B::SET;
          mma_sums<DP, HALF, typename B::Weights, typename B::Weights>(tmem + B::OUT, set + B::W0, at + (WALK == 0 ? HB : 0),
                                                                       set + B::W1, at + (WALK == 0 ? 3 * HB : 2 * HB));
          tc::commit_to(summed);
        }
      };
      issue<DP>(n, loaded, full, ready, dead, status, load, score, sum);
    }
    drain(bars + DRAINED);
  } else {
    const float c2 = p.scale * log2e<float>();
    float L = -neg_inf<float>(), D = 0.f, r = 0.f, c = 0.f;
    if (on && n > 0) {
      const float* at = stats + ((int64_t)h * im.a.slots + first_slot(p, part) + (row - part.lo) / SLOT) * KINDS * SLOT + (row - part.lo) % SLOT;
      L = at[0];
      D = at[SLOT];
      if (WALK == 1) { r = at[2 * SLOT]; c = at[3 * SLOT]; }
    }
    for (int i = 0; i < n; ++i) {
      const uint32_t bits = allowed_half(lo + i * HALF, hi, p.mask) >> (16 * half);
      if (!(ok = wait_all(scored + i % SETS<DP>, i / SETS<DP> & 1, dead, status))) break;
      tc::tc_fence_after();
      const uint32_t set = lanes + i % SETS<DP> * B::SET;
      float s[16], t[16], dp[16], e[16];
      tmem_ld16(set + B::S + 16 * half, s);
      tmem_ld16(set + B::T + 16 * half, t);
      tmem_ld16(set + B::DPO + 16 * half, dp);
      tmem_ld16(set + B::E + 16 * half, e);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const bool in = (bits >> j) & 1;
        const float pr = in ? ex2(fmaf(s[j], c2, -L)) : 0.f, tt = t[j] * p.scale;
        if (WALK == 0) {
          s[j] = in ? pr * tt : 0.f;
          t[j] = pr;
          R += s[j];
          U += in ? pr * fmaf(tt, dp[j], e[j]) : 0.f;
        } else {
          s[j] = in ? pr * (fmaf(tt - r, dp[j] - D, e[j]) - c) : 0.f;
          t[j] = in ? pr * (dp[j] - D) : 0.f;
        }
      }
      if (i > 0) {
        if (!(ok = wait_all(summed, (i - 1) & 1, dead, status))) break;
        tc::tc_fence_after();
        add_columns<DP / 2>(lanes + B::OUT + half * (DP / 2), acc);
      }
      store_parts16<typename B::Weights>(set + B::W0, half, s);
      store_parts16<typename B::Weights>(set + B::W1, half, t);
      tmem_st_wait();
      tc::tc_fence_before();
      arrive(ready);
    }
    if (ok && n > 0 && (ok = wait_all(summed, (n - 1) & 1, dead, status))) {
      tc::tc_fence_after();
      add_columns<DP / 2>(lanes + B::OUT + half * (DP / 2), acc);
    }
    if (WALK == 0) {                                    // each half of a row's columns has its share of r and c
      sums[128 * half + (threadIdx.x & 127)] = ok ? R : __int_as_float(0x7fc00000);
      sums[256 + 128 * half + (threadIdx.x & 127)] = U;
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp < 8) {
    const int64_t rows = (int64_t)p.H * p.N, at = (int64_t)h * p.N + row;
    float* out = job.splits > 1 ? p.work + (int64_t)job.split * rows * p.D : WALK == 0 ? p.out3 : p.out0;
    if (WALK == 0) {
      R = sums[threadIdx.x & 127] + sums[128 + (threadIdx.x & 127)];
      U = sums[256 + (threadIdx.x & 127)] + sums[384 + (threadIdx.x & 127)];
      if (job.splits > 1) {
        if (on && half == 0) {
          parts[(2 * (int64_t)job.split) * rows + at] = R;
          parts[(2 * (int64_t)job.split + 1) * rows + at] = U;
        }
      } else if (part.keys && row < slots_end(part)) {  // nothing to join: r, c and do' at once, zeros behind the last row
        float* st = stats + ((int64_t)h * im.a.slots + first_slot(p, part) + (row - part.lo) / SLOT) * KINDS * SLOT + (row - part.lo) % SLOT;
        if (half == 0) {
          st[2 * SLOT] = on ? R : 0.f;
          st[3 * SLOT] = on ? U - st[SLOT] * R : 0.f;
        }
        if (on) {
          const float* o = p.o + row * p.os + h * p.oh + half * (DP / 2);
#pragma unroll
          for (int d = 0; d < DP / 2; ++d)
            if (half * (DP / 2) + d < p.D) acc[d] -= R * o[d];
        }
      }
    }
    if (WALK == 1) {
#pragma unroll
      for (int d = 0; d < DP / 2; ++d) acc[d] *= p.scale;
    }
    const int row0 = part.row + 32 * (warp & 3);
    store_rows<DP / 2>(scratch_of<DP / 2>(smem, warp), acc, out + ((int64_t)row0 * p.H + h) * p.D, (int64_t)p.H * p.D,
                       min(32, part.hi - row0), half * (DP / 2), p.D, ok);
  }
  if (warp == 8) {
    tc::tc_fence_after();
    tmem_free(tmem, 512);
  }
}

// Two rows a warp of a quarter of a (slot, head): r, c and do' from the splits; rows without keys give zero.
__global__ void __launch_bounds__(256) second_join_kernel(const Params<float> p, float* __restrict__ stats,
                                                          const float* __restrict__ parts, int slots) {
  Part part;
  if (!find_part<SLOT>(p, blockIdx.x, part)) return;
  const int h = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t rows = (int64_t)p.H * p.N;
  float* st = stats + ((int64_t)h * slots + first_slot(p, part) + (part.row - part.lo) / SLOT) * KINDS * SLOT;
#pragma unroll
  for (int i = blockIdx.z * 16 + warp; i < (int)blockIdx.z * 16 + 16; i += 8) {
    const int row = part.row + i;
    const bool in = row < part.hi, live = in && part.keys;
    const int64_t at = (int64_t)h * p.N + (live ? row : 0);
    const bool mine = live && lane < p.splits;           // a lane per split (at most 32)
    const float r = row_sum<32>(mine ? parts[(2 * (int64_t)lane) * rows + at] : 0.f);
    const float u = row_sum<32>(mine ? parts[(2 * (int64_t)lane + 1) * rows + at] : 0.f);
    for (int d = lane; d < p.D; d += 32) {
      float v = 0.f;
      if (live) {
#pragma unroll 4
        for (int z = 0; z < p.splits; ++z) v += p.work[(z * rows + (int64_t)row * p.H + h) * p.D + d];
        v -= r * p.o[row * p.os + h * p.oh + d];
      }
      if (in) p.out3[((int64_t)row * p.H + h) * p.D + d] = v;
    }
    if (lane == 0 && part.keys) {
      st[2 * SLOT + i] = r;
      st[3 * SLOT + i] = live ? u - st[SLOT + i] * r : 0.f;
    }
  }
}

template <int DP>
struct Keys {
  static constexpr int HB = half_bytes<DP>(), BLOCK = PLANES * 128 * DP * 2, ST = 2 * BLOCK, STAGE = 3 * HB + KINDS * HALF * 4,
                       BARS = ST + RING<DP> * STAGE, SMEM = BARS + 128;
  static constexpr int P = 3 * DP / 2, S = 2 * P, T = S + HALF, DPO = T + HALF, E = DPO + HALF, SET = 4 * HALF + 16,
                       K2 = S + SETS<DP> * SET, V2 = K2 + DP;
  // the parts of M, dS and P (T - r) over the four score regions and 16 columns more, each half over its own columns
  using M = OverHalves<0, 8, HALF>;
  using DS = OverHalves<HALF + 8, 2 * HALF, 2 * HALF + 8>;
  using PT = OverHalves<3 * HALF, 3 * HALF + 8, 4 * HALF, 16, 16, 8>;
  static_assert(V2 + DP <= 512 && SMEM <= 232448, "tensor and shared memory");
};

template <int DP>
__device__ __forceinline__ void keys_block(const Params<float>& p, const Part& part, const Job& job, const Streams& own, const Streams& im,
                                           const float* __restrict__ stats, int* status) {
  using B = Keys<DP>;
  constexpr int HB = B::HB;
  extern __shared__ __align__(128) char smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + B::BARS);
  uint64_t *full = bars, *full_2 = bars + 4, *scored = bars + 5, *summed = bars + 7, *ready = bars + 8;
  uint32_t* slot = reinterpret_cast<uint32_t*>(bars + 10);
  volatile int* dead = reinterpret_cast<volatile int*>(bars + 11);
  const int warp = threadIdx.x / 32, hk = job.head, group = p.H / p.HK;
  int lo = part.lo, hi = part.keys ? part.hi : part.lo;
  split_range<SLOT>(lo, hi, job.split, job.splits);
  const int mine = first_slot(p, part) + (part.row - part.lo) / SLOT;     // own: k, v, B, C
  const int tiles = (hi - lo + HALF - 1) / HALF, n = tiles * group, slot0 = first_slot(p, part) + (lo - part.lo) / SLOT;
  if (warp == 8) tmem_alloc(slot, 512);
  if (threadIdx.x == 0) {
    for (int i = 0; i < 8; ++i) tc::mbar_init(bars + i, 1);
    tc::mbar_init(ready, 8);
    tc::mbar_init(bars + DRAINED, 1);
    *dead = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *slot, lanes = tmem + ((uint32_t)(warp & 3) << 21);
  const int row = part.row + (threadIdx.x & 127), half = warp / 4;
  const auto load = [&](int i) {                    // q, do, A and the statistics of tile i
    if (elect()) {
      char* to = smem + B::ST + i % RING<DP> * B::STAGE;
      uint64_t* bar = full + i % RING<DP>;
      const int head = hk * group + i / tiles, t = i % tiles;
      tc::mbar_arrive_expect_tx(bar, B::STAGE);
      load_half<DP>(to, image<DP>(im.a, head, slot0 + t / 2), t % 2, bar);
      load_half<DP>(to + HB, image<DP>(im.b, head, slot0 + t / 2), t % 2, bar);
      load_half<DP>(to + 2 * HB, image<DP>(im.c, head, slot0 + t / 2), t % 2, bar);
      const float* st = stats + ((int64_t)head * im.a.slots + slot0 + t / 2) * KINDS * SLOT + t % 2 * HALF;
#pragma unroll
      for (int x = 0; x < KINDS; ++x) tc::bulk_g2s(to + 3 * HB + x * HALF * 4, st + x * SLOT, HALF * 4, bar);
    }
  };
  int loaded = min(n, RING<DP>);
  if (warp == 8 && n > 0) {
    if (elect()) {
      tc::mbar_arrive_expect_tx(full_2, 2 * B::BLOCK);
      load_block<DP>(smem, image<DP>(own.b, hk, mine), full_2);
      load_block<DP>(smem + B::BLOCK, image<DP>(own.d, hk, mine), full_2);
    }
    __syncwarp();
    for (int i = 0; i < loaded; ++i) load(i);
  } else if (n > 0) {
    stage_image<DP>(lanes + (half ? B::P : 0), image<DP>(half ? own.c : own.a, hk, mine), threadIdx.x & 127);
    tmem_st_wait();
    tc::tc_fence_before();
  }
  __syncthreads();
  tc::tc_fence_after();

  if (warp == 8) {
    if (n > 0) {
      const uint32_t base = tc::smem_u32(smem), ring = base + B::ST;
      const auto score = [&](int i) {
        if (elect()) {
          const uint32_t at = ring + i % RING<DP> * B::STAGE, set = tmem + i % SETS<DP> * B::SET;
          mma_scores<DP, HALF>(set + B::S, tmem, at);
          mma_scores<DP, HALF>(set + B::T, tmem, at + 2 * HB, tmem + B::P, at);
          mma_scores_ss<DP, HALF>(set + B::DPO, base, at + HB);
          mma_scores_ss<DP, HALF>(set + B::E, base + B::BLOCK, at + HB);
          tc::commit_to(scored + i % SETS<DP>);
        }
      };
      const auto sum = [&](int i) {
        if (elect()) {
          const uint32_t at = ring + i % RING<DP> * B::STAGE, set = tmem + i % SETS<DP> * B::SET;
          mma_sums<DP, HALF, typename B::M, typename B::DS>(tmem + B::K2, set + B::S, at, set + B::S, at + 2 * HB);
          mma_sums<DP, HALF, typename B::PT>(tmem + B::V2, set + B::S, at + HB);
          tc::commit_to(summed);
        }
      };
      if (wait_all(full_2, 0, dead, status)) issue<DP>(n, loaded, full, ready, dead, status, load, score, sum);
      else give_up<DP>(loaded, full, full_2);
    }
    drain(bars + DRAINED);
  } else {
    const float c2 = p.scale * log2e<float>();
    float acc[DP];                                      // the first half of the warps adds up k', the second v'
#pragma unroll
    for (int d = 0; d < DP; ++d) acc[d] = 0.f;
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      if (!(ok = wait_all(scored + i % SETS<DP>, i / SETS<DP> & 1, dead, status))) break;
      if (!(ok = wait_all(full + i % RING<DP>, i / RING<DP> & 1, dead, status))) break;
      tc::tc_fence_after();
      const float* st = reinterpret_cast<const float*>(smem + B::ST + i % RING<DP> * B::STAGE + 3 * HB) + 16 * half;
      const uint32_t set = lanes + i % SETS<DP> * B::SET;
      float s[16], t[16], dp[16], e[16];
      tmem_ld16(set + B::S + 16 * half, s);
      tmem_ld16(set + B::T + 16 * half, t);
      tmem_ld16(set + B::DPO + 16 * half, dp);
      tmem_ld16(set + B::E + 16 * half, e);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float pr = ex2(fmaf(s[j], c2, -st[j])), x = fmaf(t[j], p.scale, -st[2 * HALF + j]), y = dp[j] - st[HALF + j];
        s[j] = pr * (fmaf(x, y, e[j]) - st[3 * HALF + j]);
        t[j] = pr * y;
        dp[j] = pr * x;
      }
      if (i > 0) {
        if (!(ok = wait_all(summed, (i - 1) & 1, dead, status))) break;
        tc::tc_fence_after();
        add_columns<DP>(lanes + (half ? B::V2 : B::K2), acc);
      }
      store_parts16<typename B::M>(set + B::S, half, s);
      store_parts16<typename B::DS>(set + B::S, half, t);
      store_parts16<typename B::PT>(set + B::S, half, dp);
      tmem_st_wait();
      tc::tc_fence_before();
      arrive(ready);
    }
    if (ok && n > 0 && (ok = wait_all(summed, (n - 1) & 1, dead, status))) {
      tc::tc_fence_after();
      add_columns<DP>(lanes + (half ? B::V2 : B::K2), acc);
    }
    const bool hidden = row < part.hi && p.mask != nullptr && !p.mask[row];
#pragma unroll
    for (int d = 0; d < DP; ++d) acc[d] = hidden ? 0.f : half ? acc[d] : p.scale * acc[d];
    const int row0 = part.row + 32 * (warp & 3);
    const int64_t all = (int64_t)p.N * p.HK * p.D;
    float* out = job.splits > 1 ? p.work_k + ((half ? job.splits : 0) + (int64_t)job.split) * all : half ? p.out2 : p.out1;
    store_rows<DP>(scratch_of<DP>(smem, warp), acc, out + ((int64_t)row0 * p.HK + hk) * p.D, (int64_t)p.HK * p.D,
                   min(32, part.hi - row0), 0, p.D, ok);
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc::tc_fence_after();
    tmem_free(tmem, 512);
  }
}

template <int DP>
__global__ void __launch_bounds__(ROW_THREADS, 1) second_first_kernel(const Params<float> p, const Streams k, const Streams q,
                                                                      float* __restrict__ stats, float* __restrict__ parts, int* status) {
  Part part;
  if (!find_part<128>(p, blockIdx.x, part)) return;
  rows_block<DP, 0>(p, part, {(int)blockIdx.y, (int)blockIdx.z, p.splits}, k, q, stats, parts, status);
}

// what needs r and c, in one launch: the longer blocks of the keys first, then the second walk of the rows
template <int DP>
__global__ void __launch_bounds__(ROW_THREADS, 1) second_last_kernel(const Params<float> p, const Streams k, const Streams q,
                                                                     float* __restrict__ stats, float* __restrict__ parts, int* status) {
  const int tiles = part_blocks(p, 128), rest = blockIdx.x / tiles, keys = p.HK * p.splits_k;
  Part part;
  if (!find_part<128>(p, blockIdx.x % tiles, part)) return;
  if (rest < keys) keys_block<DP>(p, part, {rest % p.HK, rest / p.HK, p.splits_k}, k, {q.a, q.c, q.b, q.b}, stats, status);
  else rows_block<DP, 1>(p, part, {(rest - keys) % p.H, (rest - keys) / p.H, p.splits}, k, q, stats, parts, status);
}

// where things lie in the workspace: images of k, v, B, C, then q, A, do, the statistics, the splits' r and c
template <int DP>
struct Layout {
  char* at[7];
  float *stats, *parts;
  int slots;
  Layout(const Params<float>& p, char* work) : slots(image_slots(p)) {
    for (int i = 0; i < 7; ++i) {
      at[i] = work;
      work += image_bytes<DP>(p, i < 4 ? p.HK : p.H);
    }
    stats = reinterpret_cast<float*>(work);
    parts = stats + (int64_t)p.H * slots * KINDS * SLOT;
  }
  Images operator[](int i) const { return Images{at[i], slots}; }
};

template <int DP>
cudaError_t second(const Params<float>& p, char* work, int* status, cudaStream_t s) {
  const Layout<DP> w(p, work);
  Sources src{};
  src.s[0] = {p.k, p.ks, p.kh, p.HK, p.mask, w.at[0]};
  src.s[1] = {p.v, p.vs, p.vh, p.HK, p.mask, w.at[1]};
  src.s[2] = {p.cb, p.cbs, p.cbh, p.HK, p.mask, w.at[2]};
  src.s[3] = {p.cc, p.ccs, p.cch, p.HK, p.mask, w.at[3]};
  src.s[4] = {p.q, p.qs, p.qh, p.H, nullptr, w.at[4]};
  src.s[5] = {p.ca, p.cas, p.cah, p.H, nullptr, w.at[5]};
  src.s[6] = {p.go, p.gos, p.goh, p.H, nullptr, w.at[6]};
  cudaError_t e = write_images<DP>(p, src, 7, w.stats, KINDS, s);
  constexpr int SMEM = Rows<DP>::SMEM > Keys<DP>::SMEM ? Rows<DP>::SMEM : Keys<DP>::SMEM;
  if (e != cudaSuccess || (e = raise_smem_limit<second_first_kernel<DP>>(Rows<DP>::SMEM)) != cudaSuccess ||
      (e = raise_smem_limit<second_last_kernel<DP>>(SMEM)) != cudaSuccess)
    return e;
  const int tiles = part_blocks(p, 128);
  const Streams k{w[0], w[1], w[2], w[3]}, q{w[4], w[5], w[6], w[6]};
  second_first_kernel<DP><<<dim3(tiles, p.H, p.splits), ROW_THREADS, Rows<DP>::SMEM, s>>>(p, k, q, w.stats, w.parts, status);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  if (p.splits > 1) {
    second_join_kernel<<<dim3(part_blocks(p, SLOT), p.H, 4), 256, 0, s>>>(p, w.stats, w.parts, w.slots);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
  }
  const int64_t blocks = (int64_t)tiles * (p.HK * p.splits_k + p.H * p.splits);
  second_last_kernel<DP><<<(unsigned)blocks, ROW_THREADS, SMEM, s>>>(p, k, q, w.stats, w.parts, status);
  return cudaGetLastError();
}

template <int DP>
int64_t bytes(const Params<float>& p) {
  return image_bytes<DP>(p, 4 * p.HK + 3 * p.H) + (int64_t)p.H * (image_slots(p) * KINDS * SLOT + 2 * (int64_t)p.splits * p.N) * 4;
}

}  // namespace

int64_t tc_second_bytes(const Params<float>& p) { return p.D <= 32 ? bytes<32>(p) : bytes<64>(p); }
cudaError_t tc_second(const Params<float>& p, char* work, int* status, cudaStream_t s) {
  return p.D <= 32 ? second<32>(p, work, status, s) : second<64>(p, work, status, s);
}

}  // namespace attn
