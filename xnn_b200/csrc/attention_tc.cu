// Structure attention of float32 operands on the tensor cores (tcgen05), for structures of some hundred atoms on.
//
// The streamed operands are first written as images of bf16 parts (attention_tc.cuh), once per call: 10 bytes
// moved an element against the hundred times that every image is read again from L2. A block then owns 128
// rows (the lanes of tensor memory), keeps their parts in tensor memory and lets bulk copies bring the
// images through shared memory; products run with the left operand in tensor memory, since with both in
// shared memory a 128 x 64 x 16 step would read 6 KB in the 32 cycles that it takes.
#include <limits>

#include "attention.h"
#include "attention_tc.cuh"

namespace attn {
namespace {

// L and D of the rows of a slot, D = do.o: `kinds` x 64 numbers a (head, slot), L = +inf behind the last row, so that P is
// zero there. A warp takes eight rows at once, their loads overlap.
__device__ __forceinline__ void slot_stats(const Params<float>& p, const Part& part, int h, float* at) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const bool vec = vec_ok(p.go, p.gos, p.goh, p.D) && vec_ok(p.o, p.os, p.oh, p.D);
  float s[SLOT / 8], L[SLOT / 8];
#pragma unroll
  for (int i = 0; i < SLOT / 8; ++i) {
    const int row = part.row + warp + 8 * i;
    s[i] = 0.f;
    L[i] = row < part.hi ? p.lse[(int64_t)h * p.N + row] : -neg_inf<float>();
    if (row >= part.hi) continue;
    const float *a = p.go + row * p.gos + h * p.goh, *b = p.o + row * p.os + h * p.oh;
    if (vec) {
      if (4 * lane < p.D) {
        const float4 x = *reinterpret_cast<const float4*>(a + 4 * lane), y = *reinterpret_cast<const float4*>(b + 4 * lane);
        s[i] = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, x.w * y.w)));
      }
    } else {
      for (int d = lane; d < p.D; d += 32) s[i] = fmaf(a[d], b[d], s[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < SLOT / 8; ++i) {
    const float v = row_sum<32>(s[i]);
    if (lane == 0) {
      at[warp + 8 * i] = L[i];
      at[SLOT + warp + 8 * i] = v;
    }
  }
}

// The images of up to seven tensors, and the rows' statistics where they are asked for: a block per (slot, head, tensor).
// Zeros behind the structure's last row, behind column D and where the mask is 0.
template <int DP>
__global__ void __launch_bounds__(256) image_kernel(const Params<float> p, const Sources src, int count, int slots, float* stats,
                                                    int kinds) {
  const bool rows = (int)blockIdx.z == count;
  const Source s = src.s[rows ? 0 : blockIdx.z];
  if (!rows && (int)blockIdx.y >= s.heads) return;
  Part part;
  if (!find_part<SLOT>(p, blockIdx.x, part) || !part.keys) return;
  const int64_t slot = (int64_t)blockIdx.y * slots + first_slot(p, part) + (part.row - part.lo) / SLOT;
  if (rows) {
    slot_stats(p, part, blockIdx.y, stats + slot * kinds * SLOT);
    return;
  }
  const float* g = s.at + blockIdx.y * s.head;
  const bool vec = vec_ok(s.at, s.row, s.head, p.D);
  uint4* out = reinterpret_cast<uint4*>(s.out + slot * Image<DP>::BYTES);
#pragma unroll 2
  for (int i = threadIdx.x; i < SLOT * DP / 8; i += 256) {
    const int r = i / DP * 8 + i % 8, c = i / 8 % (DP / 8) * 8, row = part.row + r;
    alignas(16) float v[8] = {};
    if (row < part.hi && (s.mask == nullptr || s.mask[row])) {
      const float* x = g + row * s.row + c;
      if (vec && c + 8 <= p.D) {
        *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(x);
        *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(x + 4);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < p.D) v[e] = x[e];
      }
    }
    uint32_t w[3][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) split_pair(v[2 * e], v[2 * e + 1], w[0][e], w[1][e], w[2][e]);
#pragma unroll
    for (int x = 0; x < 3; ++x) out[x * (Image<DP>::PLANE / 16) + i] = make_uint4(w[x][0], w[x][1], w[x][2], w[x][3]);
  }
}

// ------------------------------------------------------------------------------------------ forward
// Eight warps of rows, two threads a row (half of a tile's keys and of the output's columns each), and a ninth that
// copies and issues. Tensor memory: the rows' parts, one region that holds S and then the parts of P in its place, and
// the product P V of one tile, which the rows' threads add to their accumulators in registers (rounded to nearest,
// which a sum over thousands of keys inside the tensor core is not). At 64 columns that is 256 of 512 columns and
// 97 KB, so two blocks share an SM and one's softmax runs under the other's products. One thread a row left the
// tensor cores idle a third of the time: its 800 instructions a tile took longer than the other block's products.
template <int DP>
struct Fwd {
  static constexpr int Q = 0, S = 3 * DP / 2, O = S + 96, COLUMNS = O + DP <= 256 ? 256 : 512;
  static constexpr int BARS = 4 * Image<DP>::BYTES, TOPS = BARS + 128, SMEM = TOPS + 2 * 128 * 4;
  static constexpr int BLOCKS = COLUMNS == 256 ? 2 : 1;
};

template <int DP>
__global__ void __launch_bounds__(ROW_THREADS, Fwd<DP>::BLOCKS) tc_fwd_kernel(const Params<float> p, const Images ik,
                                                                              const Images iv, int* status) {
  using F = Fwd<DP>;
  constexpr int BYTES = Image<DP>::BYTES;
  extern __shared__ __align__(128) char smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + F::BARS);
  uint64_t *full_k = bars, *full_v = bars + 2, *s_done = bars + 4, *o_done = bars + 5, *p_ready = bars + 6;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 7);
  volatile int* dead = reinterpret_cast<volatile int*>(bars + 8);
  float* tops = reinterpret_cast<float*>(smem + F::TOPS);
  Part part;
  if (!find_part<128>(p, blockIdx.x, part)) return;
  const int tid = threadIdx.x, warp = tid / 32;
  const int h = blockIdx.y, hk = h / (p.H / p.HK);
  int k_lo = part.lo, k_hi = part.keys ? part.hi : part.lo;
  split_range<SLOT>(k_lo, k_hi, blockIdx.z, p.splits);
  const int n = (k_hi - k_lo + SLOT - 1) / SLOT, slot0 = first_slot(p, part) + (k_lo - part.lo) / SLOT;
  if (warp == 8) tmem_alloc(tmem_slot, F::COLUMNS);
  if (tid == 0) {
    for (int i = 0; i < 6; ++i) tc::mbar_init(bars + i, 1);
    tc::mbar_init(p_ready, 8);
    tc::mbar_init(bars + DRAINED, 1);
    *dead = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot, lanes = tmem + ((uint32_t)(warp & 3) << 21);
  const int r = tid & 127, row = part.row + r, half = warp / 4;
  const bool on = warp < 8 && row < part.hi;
  const auto load = [&](uint64_t* bar, int at, const Images& im, int i) {
    if (elect()) {
      tc::mbar_arrive_expect_tx(bar, BYTES);
      tc::bulk_g2s(smem + at * BYTES, image<DP>(im, hk, slot0 + i), BYTES, bar);
    }
  };
  int loaded_k = min(n, 2), loaded_v = min(n, 2);
  if (warp == 8) {                                      // the copies run while the other warps stage their rows
    for (int i = 0; i < loaded_k; ++i) {
      load(full_k + i, i, ik, i);
      load(full_v + i, 2 + i, iv, i);
    }
  } else if (n > 0) {
    stage_row<DP, DP / 2>(lanes + F::Q, p.q + row * p.qs + h * p.qh, on, vec_ok(p.q, p.qs, p.qh, p.D), p.D,
                          p.scale * log2e<float>(), half * (DP / 2));
    tmem_st_wait();
    tc::tc_fence_before();
  }
  __syncthreads();
  tc::tc_fence_after();
  bool ok = true;
  float m = neg_inf<float>(), l = 0.f, acc[DP / 2];
#pragma unroll
  for (int d = 0; d < DP / 2; ++d) acc[d] = 0.f;

  if (warp == 8) {
    if (n > 0) {
      const uint32_t sk = tc::smem_u32(smem), sv = sk + 2 * BYTES;
      const auto scores = [&](int i) {
        if (elect()) {
          mma_scores<DP>(tmem + F::S, tmem + F::Q, sk + (i & 1) * BYTES);
          tc::commit_to(s_done);
        }
      };
      ok = wait_all(full_k, 0, dead, status);
      if (ok) scores(0);
      for (int i = 0; ok && i < n; ++i) {
        // the probabilities of tile i are there, so S(i) and P V(i - 1) are done and their images free
        if (!(ok = wait_all(p_ready, i & 1, dead, status))) break;
        tc::tc_fence_after();
        if (!(ok = wait_all(full_v + (i & 1), (i >> 1) & 1, dead, status))) break;
        if (elect()) {
          mma_sums<DP, SLOT, OverScores>(tmem + F::O, tmem + F::S, sv + (i & 1) * BYTES);
          tc::commit_to(o_done);
        }
        if (i + 1 < n) {
          if (!(ok = wait_all(full_k + ((i + 1) & 1), ((i + 1) >> 1) & 1, dead, status))) break;
          scores(i + 1);
        }
        if (i + 2 < n) { load(full_k + (i & 1), i & 1, ik, i + 2); loaded_k = i + 3; }
        if (i > 0 && i + 1 < n) { load(full_v + ((i + 1) & 1), 2 + ((i + 1) & 1), iv, i + 1); loaded_v = i + 2; }
      }
      if (!ok) {                                        // copies in flight must land before the block ends
        for (int i = max(0, loaded_k - 2); i < loaded_k; ++i) tc::mbar_wait(full_k + (i & 1), (i >> 1) & 1, SPINS);
        for (int i = max(0, loaded_v - 2); i < loaded_v; ++i) tc::mbar_wait(full_v + (i & 1), (i >> 1) & 1, SPINS);
      }
    }
    drain(bars + DRAINED);
  } else {
    float f = 1.f;
    const auto add = [&] {                              // P V of the tile before, relative to its maximum
      const Two ff = two(f, f);
#pragma unroll
      for (int c = 0; c < DP / 2; c += 16) {
        float o[16];
        tmem_ld16(lanes + F::O + half * (DP / 2) + c, o);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; j += 2)
          get(fma2(two(acc[c + j], acc[c + j + 1]), ff, two(o[j], o[j + 1])), acc[c + j], acc[c + j + 1]);
      }
    };
    for (int i = 0; i < n; ++i) {
      const uint32_t bits = (uint32_t)(allowed_bits(k_lo + i * SLOT, k_hi, p.mask) >> (32 * half));
      if (i > 0) {                                      // under the scores of this tile
        if (!(ok = wait_all(o_done, (i - 1) & 1, dead, status))) break;
        tc::tc_fence_after();
        add();
      }
      if (!(ok = wait_all(s_done, i & 1, dead, status))) break;
      tc::tc_fence_after();
      float s[32];
      tmem_ld32(lanes + F::S + 32 * half, s);
      tmem_ld_wait();
      if (bits != ~0u) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (!((bits >> j) & 1)) s[j] = neg_inf<float>();
      }
      float t0 = s[0], t1 = s[1], t2 = s[2], t3 = s[3];
#pragma unroll
      for (int j = 4; j < 32; j += 4) {
        t0 = fmaxf(t0, s[j]); t1 = fmaxf(t1, s[j + 1]); t2 = fmaxf(t2, s[j + 2]); t3 = fmaxf(t3, s[j + 3]);
      }
      const float mine = fmaxf(fmaxf(t0, t1), fmaxf(t2, t3));
      tops[half * 128 + r] = mine;
      pair_sync(warp & 3);                              // the maximum of the row's other half of the keys
      const float mn = fmaxf(m, fmaxf(mine, tops[(half ^ 1) * 128 + r]));
      const float base = mn == neg_inf<float>() ? 0.f : mn;
      f = ex2(m - base);
      m = mn;
      const Two down = two(-base, -base);
      Two u = two(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < 32; c += 16) {
#pragma unroll
        for (int j = c; j < c + 16; j += 2) {
          get(two(s[j], s[j + 1]) + down, s[j], s[j + 1]);
          s[j] = ex2(s[j]);
          s[j + 1] = ex2(s[j + 1]);
          u = u + two(s[j], s[j + 1]);
        }
        store_parts16<OverScores>(lanes + F::S, 2 * half + c / 16, s + c);
      }
      float u0, u1;
      get(u, u0, u1);
      l = fmaf(l, f, u0 + u1);
      tmem_st_wait();
      tc::tc_fence_before();
      arrive(p_ready);
    }
    if (!ok) pair_leave(warp & 3);
    if (ok && n > 0 && (ok = wait_all(o_done, (n - 1) & 1, dead, status))) {
      tc::tc_fence_after();
      add();
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp < 8) tops[half * 128 + r] = ok ? l : __int_as_float(0x7fc00000);
  __syncthreads();
  if (warp < 8) {
    l = tops[r] + tops[128 + r];
    const bool none = m == neg_inf<float>() && l == 0.f;
    const bool split = p.splits > 1;
    const int64_t rows = (int64_t)p.H * p.N, at = blockIdx.z * rows + (int64_t)h * p.N + row;
    const float g = split ? 1.f : none ? 0.f : 1.f / l;
    const int row0 = part.row + 32 * (warp & 3);         // the warp's first row
    float* out = split ? p.work + (blockIdx.z * rows + (int64_t)h * p.N + row0) * p.D : p.out0 + ((int64_t)row0 * p.H + h) * p.D;
#pragma unroll
    for (int d = 0; d < DP / 2; ++d) acc[d] *= g;
    store_rows<DP / 2>(scratch_of<DP / 2>(smem, warp), acc, out, split ? p.D : (int64_t)p.H * p.D, min(32, part.hi - row0),
                       half * (DP / 2), p.D, ok);
    if (half == 0 && on) {
      if (split) {
        float* stats = p.work + p.splits * rows * p.D;
        stats[at] = m;
        stats[p.splits * rows + at] = l;
      } else if (p.lse) {
        p.lse[(int64_t)h * p.N + row] = none ? -neg_inf<float>() : m + log2f(l);
      }
    }
  }
  if (warp == 8) {
    tc::tc_fence_after();
    tmem_free(tmem, F::COLUMNS);
  }
}

// ------------------------------------------------------------------------------------------ backward
// Eight warps of rows: warp w reaches the lanes 32 (w % 4) .. of tensor memory and takes half w / 4 of the columns;
// a ninth copies and issues. A ring of three stages holds the streamed images.
constexpr int STAGES = 3;

template <int DP>
struct Bwd {
  static constexpr int PARTS = 3 * DP / 2;
  static constexpr int STAGE = 2 * Image<DP>::BYTES + 2 * SLOT * 4;
  static constexpr int SMEM = STAGES * STAGE + 128;
  // dq: parts of q and do, S, dP, the parts of dS, the product of one tile
  static constexpr int Q_S = 2 * PARTS, Q_DP = Q_S + SLOT, Q_DS = Q_DP + SLOT, Q_OUT = Q_DS + 96;
  // dk, dv: parts of k and v, S^T then P^T, dP^T then dS^T, the products of one tile
  static constexpr int K_S = 2 * PARTS, K_DP = K_S + 96, K_DV = K_DP + 96, K_DK = K_DV + DP;
  static_assert(Q_OUT + DP <= 512 && K_DK + DP <= 512, "tensor memory");
};

struct Block {                                          // what the two kernels set up alike
  uint64_t *full, *bars;
  volatile int* dead;
  uint32_t tmem;
  int warp;
};

// barriers and tensor memory
template <int DP>
__device__ __forceinline__ Block set_up(char* smem) {
  Block k;
  k.full = reinterpret_cast<uint64_t*>(smem + STAGES * Bwd<DP>::STAGE);
  k.bars = k.full + STAGES;
  uint32_t* slot = reinterpret_cast<uint32_t*>(k.bars + 4);
  k.dead = reinterpret_cast<volatile int*>(k.bars + 5);
  k.warp = threadIdx.x / 32;
  if (k.warp == 8) tmem_alloc(slot, 512);
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) tc::mbar_init(k.full + i, 1);
    tc::mbar_init(k.bars, 1);
    tc::mbar_init(k.bars + 1, 1);
    tc::mbar_init(k.bars + 2, 8);
    tc::mbar_init(k.bars + 3, 8);
    tc::mbar_init(k.full + DRAINED, 1);
    *k.dead = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  k.tmem = *slot;
  return k;
}

// the parts of the two resident operands: a by the first four warps, b by the others
template <int DP>
__device__ __forceinline__ void stage_rows(const Block& k, const char* a, const char* b) {
  const uint32_t lanes = k.tmem + ((uint32_t)(k.warp & 3) << 21);
  stage_image<DP>(lanes + (k.warp < 4 ? 0 : Bwd<DP>::PARTS), k.warp < 4 ? a : b, threadIdx.x & 127);
  tmem_st_wait();
  tc::tc_fence_before();
}

__device__ __forceinline__ void tear_down(const Block& k) {
  tc::tc_fence_before();
  __syncthreads();
  if (k.warp == 8) {
    tc::tc_fence_after();
    tmem_free(k.tmem, 512);
  }
}

// dq of 128 queries. S and dP of the next tile run while the rows' threads form dS of this one.
template <int DP>
__device__ __forceinline__ void dq_block(const Params<float>& p, const Part& part, const Job& job, const Images& ik, const Images& iv,
                                         const Images& iq, const Images& io, const float* __restrict__ stats, int* status) {
  using B = Bwd<DP>;
  constexpr int BYTES = Image<DP>::BYTES;
  extern __shared__ __align__(128) char smem[];
  const int h = job.head, hk = h / (p.H / p.HK);
  int k_lo = part.lo, k_hi = part.keys ? part.hi : part.lo;
  split_range<SLOT>(k_lo, k_hi, job.split, job.splits);
  const int n = (k_hi - k_lo + SLOT - 1) / SLOT, slot0 = first_slot(p, part) + (k_lo - part.lo) / SLOT;
  const Block k = set_up<DP>(smem);
  const auto load = [&](int i) {
    if (elect()) {
      char* at = smem + (i % STAGES) * B::STAGE;
      tc::mbar_arrive_expect_tx(k.full + i % STAGES, 2 * BYTES);
      tc::bulk_g2s(at, image<DP>(ik, hk, slot0 + i), BYTES, k.full + i % STAGES);
      tc::bulk_g2s(at + BYTES, image<DP>(iv, hk, slot0 + i), BYTES, k.full + i % STAGES);
    }
  };
  int loaded = min(n, STAGES);
  if (k.warp == 8) {                                    // the copies run while the other warps stage their rows
    for (int i = 0; i < loaded; ++i) load(i);
  } else if (n > 0) {
    const int own = first_slot(p, part) + (part.row - part.lo) / SLOT;
    stage_rows<DP>(k, image<DP>(iq, h, own), image<DP>(io, h, own));
  }
  __syncthreads();
  tc::tc_fence_after();
  uint64_t *sd_done = k.bars, *dq_done = k.bars + 1, *taken = k.bars + 2, *ds_ready = k.bars + 3;
  if (k.warp == 8) {
    if (n > 0) {
      const uint32_t base = tc::smem_u32(smem);
      const auto scores = [&](int i) {
        if (elect()) {
          const uint32_t at = base + (i % STAGES) * B::STAGE;
          mma_scores<DP>(k.tmem + B::Q_S, k.tmem, at);
          mma_scores<DP>(k.tmem + B::Q_DP, k.tmem + B::PARTS, at + BYTES);
          tc::commit_to(sd_done);
        }
      };
      bool ok = wait_all(k.full, 0, k.dead, status);
      if (ok) scores(0);
      for (int i = 0; ok && i < n; ++i) {
        if (!(ok = wait_all(taken, i & 1, k.dead, status))) break;
        tc::tc_fence_after();
        if (i + 1 < n) {
          if (!(ok = wait_all(k.full + (i + 1) % STAGES, ((i + 1) / STAGES) & 1, k.dead, status))) break;
          scores(i + 1);
        }
        if (!(ok = wait_all(ds_ready, i & 1, k.dead, status))) break;
        tc::tc_fence_after();
        // dq of tile i - 1 is done: its stage is free
        if (i > 0 && i + 2 < n) { load(i + 2); loaded = i + 3; }
        if (elect()) {
          mma_sums<DP, SLOT, Linear<SLOT / 2>>(k.tmem + B::Q_OUT, k.tmem + B::Q_DS, base + (i % STAGES) * B::STAGE);
          tc::commit_to(dq_done);
        }
      }
      if (!ok)
        for (int i = max(0, loaded - STAGES); i < loaded; ++i) tc::mbar_wait(k.full + i % STAGES, (i / STAGES) & 1, SPINS);
    }
    drain(k.full + DRAINED);
  } else {
    const uint32_t lanes = k.tmem + ((uint32_t)(k.warp & 3) << 21);
    const int half = k.warp / 4, r = threadIdx.x & 127, row = part.row + r;
    const bool on = row < part.hi;
    const float c2 = p.scale * log2e<float>();
    float L = -neg_inf<float>(), D = 0.f, acc[DP / 2];
    if (on && n > 0) {
      const float* at = stats + ((int64_t)h * ik.slots + first_slot(p, part) + (row - part.lo) / SLOT) * 2 * SLOT;
      L = at[(row - part.lo) % SLOT];
      D = at[SLOT + (row - part.lo) % SLOT];
    }
#pragma unroll
    for (int d = 0; d < DP / 2; ++d) acc[d] = 0.f;
    bool ok = true;
    const auto add = [&] { add_columns<DP / 2>(lanes + B::Q_OUT + half * (DP / 2), acc); };
    for (int i = 0; i < n; ++i) {
      const uint32_t bits = (uint32_t)(allowed_bits(k_lo + i * SLOT, k_hi, p.mask) >> (32 * half));
      if (!(ok = wait_all(sd_done, i & 1, k.dead, status))) break;
      tc::tc_fence_after();
      float s[32], dp[32];
      tmem_ld32(lanes + B::Q_S + 32 * half, s);
      tmem_ld32(lanes + B::Q_DP + 32 * half, dp);
      tmem_ld_wait();
      tc::tc_fence_before();
      arrive(taken);
      const Two low = two(-L, -L), down = two(-D, -D), by = two(c2, c2);
#pragma unroll
      for (int j = 0; j < 32; j += 2) {
        get(fma2(two(s[j], s[j + 1]), by, low), s[j], s[j + 1]);
        get(two(ex2(s[j]), ex2(s[j + 1])) * (two(dp[j], dp[j + 1]) + down), s[j], s[j + 1]);
      }
      if (bits != ~0u) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (!((bits >> j) & 1)) s[j] = 0.f;
      }
      if (i > 0) {
        if (!(ok = wait_all(dq_done, (i - 1) & 1, k.dead, status))) break;
        tc::tc_fence_after();
        add();
      }
      store_parts16<Linear<SLOT / 2>>(lanes + B::Q_DS, 2 * half, s);
      store_parts16<Linear<SLOT / 2>>(lanes + B::Q_DS, 2 * half + 1, s + 16);
      tmem_st_wait();
      tc::tc_fence_before();
      arrive(ds_ready);
    }
    if (ok && n > 0 && (ok = wait_all(dq_done, (n - 1) & 1, k.dead, status))) {
      tc::tc_fence_after();
      add();
    }
#pragma unroll
    for (int d = 0; d < DP / 2; ++d) acc[d] *= p.scale;
    const int row0 = part.row + 32 * (k.warp & 3);
    float* out = job.splits > 1 ? p.work + (int64_t)job.split * p.N * p.H * p.D : p.out0;
    store_rows<DP / 2>(scratch_of<DP / 2>(smem, k.warp), acc, out + ((int64_t)row0 * p.H + h) * p.D, (int64_t)p.H * p.D,
                       min(32, part.hi - row0), half * (DP / 2), p.D, ok);
  }
  tear_down(k);
}

// dk and dv of 128 keys of one key head, over the queries of every head that shares it. Two chains share the
// tensor cores: while the threads form P^T of a tile, dK of the tile before and dP^T of this one run; while they form
// dS^T, dV of this tile and S^T of the next.
template <int DP>
__device__ __forceinline__ void dkv_block(const Params<float>& p, const Part& part, const Job& job, const Images& ik, const Images& iv,
                                          const Images& iq, const Images& io, const float* __restrict__ stats, int* status) {
  using B = Bwd<DP>;
  constexpr int BYTES = Image<DP>::BYTES;
  extern __shared__ __align__(128) char smem[];
  const int hk = job.head, group = p.H / p.HK;
  int q_lo = part.lo, q_hi = part.keys ? part.hi : part.lo;
  split_range<SLOT>(q_lo, q_hi, job.split, job.splits);
  const int tiles = (q_hi - q_lo + SLOT - 1) / SLOT, n = tiles * group, slot0 = first_slot(p, part) + (q_lo - part.lo) / SLOT;
  const Block k = set_up<DP>(smem);
  const auto load = [&](int i) {
    if (elect()) {
      char* at = smem + (i % STAGES) * B::STAGE;
      uint64_t* bar = k.full + i % STAGES;
      const int h = hk * group + i / tiles, slot = slot0 + i % tiles;
      tc::mbar_arrive_expect_tx(bar, B::STAGE);
      tc::bulk_g2s(at, image<DP>(iq, h, slot), BYTES, bar);
      tc::bulk_g2s(at + BYTES, image<DP>(io, h, slot), BYTES, bar);
      tc::bulk_g2s(at + 2 * BYTES, stats + ((int64_t)h * iq.slots + slot) * 2 * SLOT, 2 * SLOT * 4, bar);
    }
  };
  int loaded = min(n, STAGES);
  if (k.warp == 8) {                                    // the copies run while the other warps stage their rows
    for (int i = 0; i < loaded; ++i) load(i);
  } else if (n > 0) {
    const int own = first_slot(p, part) + (part.row - part.lo) / SLOT;
    stage_rows<DP>(k, image<DP>(ik, hk, own), image<DP>(iv, hk, own));
  }
  __syncthreads();
  tc::tc_fence_after();
  uint64_t *s_done = k.bars, *dp_done = k.bars + 1, *p_ready = k.bars + 2, *ds_ready = k.bars + 3;
  if (k.warp == 8) {
    if (n > 0) {
      const uint32_t base = tc::smem_u32(smem);
      const auto stage = [&](int i) { return base + (i % STAGES) * B::STAGE; };
      // a product of tile i and the score product of the next tile (or of none) behind it
      const auto step = [&](uint32_t sum, uint32_t a, uint32_t rows, uint32_t d, uint32_t parts, uint32_t image, bool next, uint64_t* bar) {
        if (elect()) {
          mma_sums<DP, SLOT, OverScores>(sum, a, rows);
          if (next) mma_scores<DP>(d, parts, image);
          tc::commit_to(bar);
        }
      };
      const uint32_t s = k.tmem + B::K_S, dp = k.tmem + B::K_DP, kp = k.tmem, vp = k.tmem + B::PARTS;
      bool ok = wait_all(k.full, 0, k.dead, status);
      if (ok && elect()) {
        mma_scores<DP>(s, kp, stage(0));
        tc::commit_to(s_done);
        mma_scores<DP>(dp, vp, stage(0) + BYTES);
        tc::commit_to(dp_done);
      }
      for (int i = 0; ok && i < n; ++i) {
        const bool next = i + 1 < n;
        if (!(ok = wait_all(p_ready, i & 1, k.dead, status))) break;
        tc::tc_fence_after();
        if (next && !(ok = wait_all(k.full + (i + 1) % STAGES, ((i + 1) / STAGES) & 1, k.dead, status))) break;
        step(k.tmem + B::K_DV, s, stage(i) + BYTES, s, kp, stage(i + 1), next, s_done);
        if (!(ok = wait_all(ds_ready, i & 1, k.dead, status))) break;
        tc::tc_fence_after();
        // dK of tile i - 1, the last to read its stage, is done
        if (i > 0 && i + 2 < n) { load(i + 2); loaded = i + 3; }
        step(k.tmem + B::K_DK, dp, stage(i), dp, vp, stage(i + 1) + BYTES, next, dp_done);
      }
      if (!ok)
        for (int i = max(0, loaded - STAGES); i < loaded; ++i) tc::mbar_wait(k.full + i % STAGES, (i / STAGES) & 1, SPINS);
    }
    drain(k.full + DRAINED);
  } else {
    const uint32_t lanes = k.tmem + ((uint32_t)(k.warp & 3) << 21);
    const int half = k.warp / 4, row = part.row + (threadIdx.x & 127);
    const float c2 = p.scale * log2e<float>();
    // the first half of the warps adds up dV, the second dK
    float acc[DP];
#pragma unroll
    for (int d = 0; d < DP; ++d) acc[d] = 0.f;
    const auto add = [&](int column) { add_columns<DP>(lanes + column, acc); };
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const float* st = reinterpret_cast<const float*>(smem + (i % STAGES) * B::STAGE + 2 * BYTES) + 32 * half;
      float s[32], dp[32];
      if (!(ok = wait_all(s_done, i & 1, k.dead, status))) break;
      // the statistics came with the tile's images: its barrier is passed (the issuing lane waited for it),
      // this thread's own wait makes them visible to it
      if (!(ok = wait_all(k.full + i % STAGES, (i / STAGES) & 1, k.dead, status))) break;
      tc::tc_fence_after();
      tmem_ld32(lanes + B::K_S + 32 * half, s);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 32; j += 4) {
        const float4 L = *reinterpret_cast<const float4*>(st + j);
        s[j] = ex2(fmaf(s[j], c2, -L.x));
        s[j + 1] = ex2(fmaf(s[j + 1], c2, -L.y));
        s[j + 2] = ex2(fmaf(s[j + 2], c2, -L.z));
        s[j + 3] = ex2(fmaf(s[j + 3], c2, -L.w));
      }
      if (half == 0 && i > 0) add(B::K_DV);
      store_parts16<OverScores>(lanes + B::K_S, 2 * half, s);
      store_parts16<OverScores>(lanes + B::K_S, 2 * half + 1, s + 16);
      tmem_st_wait();
      tc::tc_fence_before();
      arrive(p_ready);
      if (!(ok = wait_all(dp_done, i & 1, k.dead, status))) break;
      tc::tc_fence_after();
      tmem_ld32(lanes + B::K_DP + 32 * half, dp);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 32; j += 4) {
        const float4 D = *reinterpret_cast<const float4*>(st + SLOT + j);
        s[j] *= dp[j] - D.x; s[j + 1] *= dp[j + 1] - D.y; s[j + 2] *= dp[j + 2] - D.z; s[j + 3] *= dp[j + 3] - D.w;
      }
      if (half == 1 && i > 0) add(B::K_DK);
      store_parts16<OverScores>(lanes + B::K_DP, 2 * half, s);
      store_parts16<OverScores>(lanes + B::K_DP, 2 * half + 1, s + 16);
      tmem_st_wait();
      tc::tc_fence_before();
      arrive(ds_ready);
    }
    if (ok && n > 0 && (ok = wait_all(s_done, n & 1, k.dead, status)) && (ok = wait_all(dp_done, n & 1, k.dead, status))) {
      tc::tc_fence_after();
      add(half ? B::K_DK : B::K_DV);
    }
    const bool hidden = row < part.hi && p.mask != nullptr && !p.mask[row];
#pragma unroll
    for (int d = 0; d < DP; ++d) acc[d] = hidden ? 0.f : half ? p.scale * acc[d] : acc[d];
    const int row0 = part.row + 32 * (k.warp & 3);
    const int64_t all = (int64_t)p.N * p.HK * p.D;
    float* out = job.splits > 1 ? p.work_k + ((half ? 0 : job.splits) + (int64_t)job.split) * all : half ? p.out1 : p.out2;
    store_rows<DP>(scratch_of<DP>(smem, k.warp), acc, out + ((int64_t)row0 * p.HK + hk) * p.D, (int64_t)p.HK * p.D,
                   min(32, part.hi - row0), 0, p.D, ok);
  }
  tear_down(k);
}

// Both in one launch, the longer blocks of the keys first, so that neither waits for the other's last blocks.
template <int DP>
__global__ void __launch_bounds__(ROW_THREADS, 1) tc_bwd_kernel(const Params<float> p, const Images ik, const Images iv, const Images iq,
                                                                const Images io, const float* __restrict__ stats, int* status) {
  const int tiles = part_blocks(p, 128), rest = blockIdx.x / tiles, keys = p.HK * p.splits_k;
  Part part;
  if (!find_part<128>(p, blockIdx.x % tiles, part)) return;
  if (rest < keys) dkv_block<DP>(p, part, {rest % p.HK, rest / p.HK, p.splits_k}, ik, iv, iq, io, stats, status);
  else dq_block<DP>(p, part, {(rest - keys) % p.H, (rest - keys) / p.H, p.splits}, ik, iv, iq, io, stats, status);
}

template <int DP>
cudaError_t forward_dp(const Params<float>& p, char* work, int* status, cudaStream_t s) {
  const int slots = image_slots(p);
  char *ik = work, *iv = ik + image_bytes<DP>(p, p.HK);
  Sources src{};
  src.s[0] = {p.k, p.ks, p.kh, p.HK, p.mask, ik};
  src.s[1] = {p.v, p.vs, p.vh, p.HK, p.mask, iv};
  cudaError_t e = write_images<DP>(p, src, 2, nullptr, 0, s);
  if (e != cudaSuccess) return e;
  if ((e = raise_smem_limit<tc_fwd_kernel<DP>>(Fwd<DP>::SMEM)) != cudaSuccess) return e;
  tc_fwd_kernel<DP><<<dim3(part_blocks(p, 128), p.H, p.splits), ROW_THREADS, Fwd<DP>::SMEM, s>>>(p, Images{ik, slots}, Images{iv, slots}, status);
  return cudaGetLastError();
}

template <int DP>
cudaError_t prepare_dp(const Params<float>& p, char* work, cudaStream_t s) {
  char *ik = work, *iv = ik + image_bytes<DP>(p, p.HK), *iq = iv + image_bytes<DP>(p, p.HK), *io = iq + image_bytes<DP>(p, p.H);
  float* stats = reinterpret_cast<float*>(io + image_bytes<DP>(p, p.H));
  Sources src{};
  src.s[0] = {p.k, p.ks, p.kh, p.HK, p.mask, ik};
  src.s[1] = {p.v, p.vs, p.vh, p.HK, p.mask, iv};
  src.s[2] = {p.q, p.qs, p.qh, p.H, nullptr, iq};
  src.s[3] = {p.go, p.gos, p.goh, p.H, nullptr, io};
  return write_images<DP>(p, src, 4, stats, 2, s);
}

template <int DP>
cudaError_t backward_dp(const Params<float>& p, char* work, int* status, cudaStream_t s) {
  const int slots = image_slots(p);
  char *ik = work, *iv = ik + image_bytes<DP>(p, p.HK), *iq = iv + image_bytes<DP>(p, p.HK), *io = iq + image_bytes<DP>(p, p.H);
  const float* stats = reinterpret_cast<const float*>(io + image_bytes<DP>(p, p.H));
  const cudaError_t e = raise_smem_limit<tc_bwd_kernel<DP>>(Bwd<DP>::SMEM);
  if (e != cudaSuccess) return e;
  const int64_t blocks = (int64_t)(part_blocks(p, 128)) * (p.HK * p.splits_k + p.H * p.splits);
  tc_bwd_kernel<DP><<<(unsigned)blocks, ROW_THREADS, Bwd<DP>::SMEM, s>>>(p, Images{ik, slots}, Images{iv, slots}, Images{iq, slots},
                                                                        Images{io, slots}, stats, status);
  return cudaGetLastError();
}

}  // namespace

template <int DP>
cudaError_t write_images(const Params<float>& p, const Sources& src, int count, float* stats, int kinds, cudaStream_t s) {
  const dim3 grid(part_blocks(p, SLOT), p.H, count + (stats != nullptr));
  image_kernel<DP><<<grid, 256, 0, s>>>(p, src, count, image_slots(p), stats, kinds);
  return cudaGetLastError();
}
template cudaError_t write_images<32>(const Params<float>&, const Sources&, int, float*, int, cudaStream_t);
template cudaError_t write_images<64>(const Params<float>&, const Sources&, int, float*, int, cudaStream_t);
template cudaError_t write_images<128>(const Params<float>&, const Sources&, int, float*, int, cudaStream_t);

int64_t tc_forward_bytes(const Params<float>& p) {
  return 2 * (p.D <= 32 ? image_bytes<32>(p, p.HK) : p.D <= 64 ? image_bytes<64>(p, p.HK) : image_bytes<128>(p, p.HK));
}
int64_t tc_backward_bytes(const Params<float>& p) {
  return 2 * (p.D <= 32 ? image_bytes<32>(p, p.HK + p.H) : p.D <= 64 ? image_bytes<64>(p, p.HK + p.H) : image_bytes<128>(p, p.HK + p.H)) +
         (int64_t)p.H * image_slots(p) * 2 * SLOT * 4;
}
cudaError_t tc_forward(const Params<float>& p, char* work, int* status, cudaStream_t s) {
  return p.D <= 32 ? forward_dp<32>(p, work, status, s) : p.D <= 64 ? forward_dp<64>(p, work, status, s) : forward_dp<128>(p, work, status, s);
}
cudaError_t tc_backward(const Params<float>& p, char* work, int* status, cudaStream_t s) {
  cudaError_t e = p.D <= 32 ? prepare_dp<32>(p, work, s) : p.D <= 64 ? prepare_dp<64>(p, work, s) : prepare_dp<128>(p, work, s);
  if (e != cudaSuccess) return e;
  return p.D <= 32 ? backward_dp<32>(p, work, status, s) : p.D <= 64 ? backward_dp<64>(p, work, status, s) : tc_wide_backward(p, work, status, s);
}

}  // namespace attn
