// Pieces of the tensor-core attention kernels: float32 operands as three bf16 parts, their images in memory, tcgen05 issue
// with the left operand in tensor memory, and bounded waits.
//
// A float32 number is exactly x1 + x2 + x3 with bf16 parts (8 significant bits each, rounded to nearest, the
// remainders exact), so a product of two is six products of parts up to terms below 2^-24 of it:
//   x3 y1 + x1 y3 + x2 y2 + x2 y1 + x1 y2 + x1 y1,
// added by the tensor cores in 32 bits from the smallest to the largest. Six bf16 products cost what three
// TF32 products would and keep 24 bits instead of 22, in six bytes an element instead of eight.
#pragma once
#include "attention_tile.cuh"
#include "tc_common.cuh"

namespace attn {

constexpr int PLANES = 3, SLOT = 64;                   // bf16 parts of a number, rows of an image

// An image holds SLOT rows of one head as PLANES planes of bf16 core matrices (8 rows x 16 bytes, 128 bytes
// each): element (r, d) of a plane at (r / 8) DP 16 + (d / 8) 128 + (r % 8) 16 + (d % 8) 2 bytes. As a K-major operand
// (rows x d) its strides are 128 between columns of 16 bytes and DP 16 between groups of 8 rows; as an MN-major one
// (d x rows) the two change places. One bulk copy brings an image to shared memory.
template <int DP> struct Image {
  static constexpr int PLANE = SLOT * DP * 2, BYTES = PLANES * PLANE;
};

struct Images {                                        // of a tensor: head h, slot t at ((h slots) + t) BYTES
  const char* at;
  int slots;
};

template <int DP>
__device__ __forceinline__ const char* image(const Images& im, int head, int slot) {
  return im.at + ((int64_t)head * im.slots + slot) * Image<DP>::BYTES;
}

// the slot of a part's first rows (parts start at slots as they do at tiles of SLOT rows)
__device__ __forceinline__ int first_slot(const Params<float>& p, const Part& part) {
  return p.compact ? part.lo / 32 : part.lo / SLOT + part.index;
}

// two float32 in a register pair: one instruction adds, multiplies or fuses both
struct Two { uint64_t v; };
__device__ __forceinline__ Two two(float a, float b) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void get(Two x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
__device__ __forceinline__ Two operator+(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two operator*(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// two numbers as three packed pairs of bf16, the first number in the low half
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void split_pair(float a, float b, uint32_t& p0, uint32_t& p1, uint32_t& p2) {
  const Two minus = two(-1.f, -1.f);
  p0 = pack_bf16(a, b);
  Two x = fma2(two(__uint_as_float(p0 << 16), __uint_as_float(p0 & 0xffff0000u)), minus, two(a, b));
  get(x, a, b);
  p1 = pack_bf16(a, b);
  x = fma2(two(__uint_as_float(p1 << 16), __uint_as_float(p1 & 0xffff0000u)), minus, x);
  get(x, a, b);
  p2 = pack_bf16(a, b);
}

__device__ __forceinline__ uint32_t idesc_bf16(int n, int b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}

// One lane of a converged warp. Issued under this predicate a run of 128 x 64 x 16 products takes 34 cycles each, under
// `lane == 0` 48: the compiler then keeps the operands in uniform registers.
__device__ __forceinline__ bool elect() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(p));
  return p != 0;
}

// D (128 x N, tensor memory) (+)= A (tensor memory) B (shared memory, descriptor in two words)
template <int ACCUMULATE>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}\n"
      :: "r"(d), "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "n"(ACCUMULATE) : "memory");
}

// Where the parts of a left operand lie in tensor memory: the column of plane x, 16 K elements (8 columns) k.
template <int PLANE> struct Linear {
  static __host__ __device__ constexpr uint32_t col(int x, int k) { return x * PLANE + 8 * k; }
};
// Over 64 columns of scores and 32 more, each half of the keys (and of the threads of a row) in its own 32 columns and
// its own 16 of the rest: no thread writes where another one's scores may still be.
struct OverScores {
  static __host__ __device__ constexpr uint32_t col(int x, int k) { return (x < 2 ? k / 2 * 32 + x * 16 : 64 + k / 2 * 16) + k % 2 * 8; }
};
// the same over regions of 32 columns, a half of the keys a step: plane x at Cx + Sx k
template <int C0, int C1, int C2, int S0 = 16, int S1 = 16, int S2 = 16> struct OverHalves {
  static __host__ __device__ constexpr uint32_t col(int x, int k) { return x == 0 ? C0 + S0 * k : x == 1 ? C1 + S1 * k : C2 + S2 * k; }
};

// one of the six products of parts: A's plane x, B's plane at b + y B_PLANE bytes, B_STEP bytes of B a step
template <class A, int KSTEPS, int B_PLANE, int B_STEP, int LBO, int SBO>
__device__ __forceinline__ void mma_part(uint32_t d, uint32_t a, uint32_t b, int x, int y, uint32_t idesc, bool first) {
  constexpr uint32_t hi = (SBO >> 4) | (1u << 14);      // bit 46: descriptor version
  const uint32_t lo = (b >> 4) | ((LBO >> 4) << 16);
#pragma unroll
  for (int k = 0; k < KSTEPS; ++k) {
    const uint32_t at = lo + (y * B_PLANE + k * B_STEP) / 16;
    if (first && k == 0) mma_ts<0>(d, a + A::col(x, k), at, hi, idesc);
    else mma_ts<1>(d, a + A::col(x, k), at, hi, idesc);
  }
}
// the six (x, y), smallest product first: (2 0) (0 2) (1 1) (1 0) (0 1) (0 0)
__host__ __device__ constexpr int part_x(int i) { return i == 0 ? 2 : i == 2 || i == 3 ? 1 : 0; }
__host__ __device__ constexpr int part_y(int i) { return i == 1 ? 2 : i == 2 || i == 4 ? 1 : 0; }
// An operand image of ROWS rows as rows x d (scores) and as d x rows (sums over the rows); the forms with two operands
// give the sum of two products, part by part: the tensor cores cut what a sum does not hold, so nothing small should
// come after something large.
template <int DP, int ROWS = SLOT>
__device__ __forceinline__ void mma_scores(uint32_t d, uint32_t a, uint32_t b) {
#pragma unroll
  for (int i = 0; i < 6; ++i)
    mma_part<Linear<DP / 2>, DP / 16, ROWS * DP * 2, 256, 128, DP * 16>(d, a, b, part_x(i), part_y(i), idesc_bf16(ROWS, 0), i == 0);
}
template <int DP, int ROWS>
__device__ __forceinline__ void mma_scores(uint32_t d, uint32_t a0, uint32_t b0, uint32_t a1, uint32_t b1) {
#pragma unroll
  for (int i = 0; i < 6; ++i) {
    mma_part<Linear<DP / 2>, DP / 16, ROWS * DP * 2, 256, 128, DP * 16>(d, a0, b0, part_x(i), part_y(i), idesc_bf16(ROWS, 0), i == 0);
    mma_part<Linear<DP / 2>, DP / 16, ROWS * DP * 2, 256, 128, DP * 16>(d, a1, b1, part_x(i), part_y(i), idesc_bf16(ROWS, 0), false);
  }
}
template <int DP, int ROWS, class A>
__device__ __forceinline__ void mma_sums(uint32_t d, uint32_t a, uint32_t b) {
#pragma unroll
  for (int i = 0; i < 6; ++i)
    mma_part<A, ROWS / 16, ROWS * DP * 2, DP * 32, DP * 16, 128>(d, a, b, part_x(i), part_y(i), idesc_bf16(DP, 1), i == 0);
}
template <int DP, int ROWS, class A0, class A1>
__device__ __forceinline__ void mma_sums(uint32_t d, uint32_t a0, uint32_t b0, uint32_t a1, uint32_t b1) {
#pragma unroll
  for (int i = 0; i < 6; ++i) {
    mma_part<A0, ROWS / 16, ROWS * DP * 2, DP * 32, DP * 16, 128>(d, a0, b0, part_x(i), part_y(i), idesc_bf16(DP, 1), i == 0);
    mma_part<A1, ROWS / 16, ROWS * DP * 2, DP * 32, DP * 16, 128>(d, a1, b1, part_x(i), part_y(i), idesc_bf16(DP, 1), false);
  }
}

// the scores with the left operand's parts in shared memory too: 128 rows, planes of 128 DP 2 bytes
template <int ACCUMULATE>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %3};\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}\n"
      :: "r"(d), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "n"(ACCUMULATE) : "memory");
}
template <int DP, int ROWS>
__device__ __forceinline__ void mma_scores_ss(uint32_t d, uint32_t a, uint32_t b) {
  constexpr int X[6] = {2, 0, 1, 1, 0, 0}, Y[6] = {0, 2, 1, 0, 1, 0};
  const uint32_t lo_a = (a >> 4) | (8u << 16), lo_b = (b >> 4) | (8u << 16);
  constexpr uint32_t hi = (uint32_t)DP | (1u << 14);    // DP 16 bytes between groups of 8 rows
#pragma unroll
  for (int i = 0; i < 6; ++i)
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
      const uint32_t x = lo_a + X[i] * (DP * 16) + k * 16, y = lo_b + Y[i] * (ROWS * DP / 8) + k * 16;
      if (i + k) mma_ss<1>(d, x, y, hi, idesc_bf16(ROWS, 0));
      else mma_ss<0>(d, x, y, hi, idesc_bf16(ROWS, 0));
    }
}

__device__ __forceinline__ void tmem_ld32(uint32_t addr, float* v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float* v) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               :: "r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// sixteen neighbouring numbers of a row (K elements 16 k ..) as three planes of eight columns in layout A
template <class A>
__device__ __forceinline__ void store_parts16(uint32_t addr, int k, const float* v) {
  uint32_t a[8], b[8], c[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) split_pair(v[2 * j], v[2 * j + 1], a[j], b[j], c[j]);
  tmem_st8(addr + A::col(0, k), a);
  tmem_st8(addr + A::col(1, k), b);
  tmem_st8(addr + A::col(2, k), c);
}

// N columns from c0 on of a row of D numbers times f (zero where `on` is false) as three planes of DP / 2 columns. The
// loads come first, all of them in flight.
template <int DP, int N = DP>
__device__ __forceinline__ void stage_row(uint32_t addr, const float* row, bool on, bool vec, int D, float f, int c0 = 0) {
  constexpr int STEP = N < 64 ? N : 64;
#pragma unroll
  for (int b = 0; b < N; b += STEP) {
    float v[STEP];
#pragma unroll
    for (int e = 0; e < STEP; e += 4) {
      const int c = c0 + b + e;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (on && c < D) {
        if (vec) {
          x = *reinterpret_cast<const float4*>(row + c);
        } else {
          x.x = row[c];
          if (c + 1 < D) x.y = row[c + 1];
          if (c + 2 < D) x.z = row[c + 2];
          if (c + 3 < D) x.w = row[c + 3];
        }
      }
      v[e] = f * x.x; v[e + 1] = f * x.y; v[e + 2] = f * x.z; v[e + 3] = f * x.w;
    }
#pragma unroll
    for (int e = 0; e < STEP; e += 16) store_parts16<Linear<DP / 2>>(addr, (c0 + b + e) / 16, v + e);
  }
}

__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(tc::smem_u32(slot)), "r"(columns) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(addr), "r"(columns));
}
// one arrival a warp
__device__ __forceinline__ void arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(tc::smem_u32(bar)) : "memory");
}

// one phase of a barrier; false after SPINS polls or once another role of the block gave up. Whoever gives
// up first records it; the block then writes NaN instead of results.
constexpr int SPINS = 1 << 20;
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* dead, int* status) {
  for (int n = 0; n < SPINS; ++n) {
    if (tc::mbar_try_wait(bar, parity)) return true;
    if ((n & 63) == 63 && *dead) return false;
  }
  *dead = 1;
  atomicExch(status, 7);
  return false;
}

// the same for a whole warp, with one answer for its lanes: they leave a loop together or not at all
__device__ __forceinline__ bool wait_all(uint64_t* bar, uint32_t parity, volatile int* dead, int* status) {
  return __all_sync(0xffffffffu, wait(bar, parity, dead, status));
}

// The issuing warp's last step: all its products are complete (or a limit ran out), whoever gave up, so that tensor memory
// may be freed and the images overwritten. The barrier takes the last eight of the 128 bytes that each block has for them.
constexpr int DRAINED = 15;
__device__ __forceinline__ void drain(uint64_t* bar) {
  if (elect()) tc::commit_to(bar);
  __syncwarp();
  tc::mbar_wait(bar, 0, SPINS);
}

// The two warps that share a quarter of the lanes (one half of a row's columns each) meet. No wait of their loops lies
// between the meeting and the loop's next turn, so a warp that leaves its loop early owes its partner one arrival: the
// partner then finds the block given up at its next wait.
__device__ __forceinline__ void pair_sync(int quarter) { asm volatile("bar.sync %0, 64;" :: "r"(quarter + 1) : "memory"); }
__device__ __forceinline__ void pair_leave(int quarter) { asm volatile("bar.arrive %0, 64;" :: "r"(quarter + 1) : "memory"); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// which of the SLOT keys from k0 on may be attended to (all lanes of a warp together)
__device__ __forceinline__ uint64_t allowed_bits(int k0, int hi, const uint8_t* mask) {
  const int left = hi - k0;
  uint64_t bits = left >= SLOT ? ~0ull : (1ull << (left > 0 ? left : 0)) - 1;
  if (mask) {
    const int lane = threadIdx.x & 31;
    const uint64_t a = __ballot_sync(0xffffffffu, k0 + lane < hi && mask[k0 + lane]);
    const uint64_t b = __ballot_sync(0xffffffffu, k0 + 32 + lane < hi && mask[k0 + 32 + lane]);
    bits &= a | (b << 32);
  }
  return bits;
}

// ---- kernels that stream halves of images: eight warps of rows, a ninth that copies and issues ----
constexpr int HALF = SLOT / 2, ROW_THREADS = 288;
// which head and which share of the other axis a block takes
struct Job { int head, split, splits; };
template <int DP> constexpr int half_bytes() { return PLANES * HALF * DP * 2; }

// half `half` of an image: its planes one behind the other
template <int DP>
__device__ __forceinline__ void load_half(char* to, const char* im, int half, uint64_t* bar) {
  constexpr int PLANE = HALF * DP * 2;
#pragma unroll
  for (int x = 0; x < PLANES; ++x) tc::bulk_g2s(to + x * PLANE, im + x * Image<DP>::PLANE + half * PLANE, PLANE, bar);
}
// two neighbouring images as one operand of 128 rows (what the second holds of other structures ends in rows that are not stored)
template <int DP>
__device__ __forceinline__ void load_block(char* to, const char* im, uint64_t* bar) {
#pragma unroll
  for (int x = 0; x < PLANES; ++x)
#pragma unroll
    for (int s = 0; s < 2; ++s)
      tc::bulk_g2s(to + (2 * x + s) * Image<DP>::PLANE, im + s * Image<DP>::BYTES + x * Image<DP>::PLANE, Image<DP>::PLANE, bar);
}

// which of the HALF keys from k0 on may be attended to (all lanes of a warp together)
__device__ __forceinline__ uint32_t allowed_half(int k0, int hi, const uint8_t* mask) {
  const int k = k0 + (threadIdx.x & 31);
  return __ballot_sync(0xffffffffu, k < hi && (mask == nullptr || mask[k]));
}

// N columns from c0 on of row r of a block of 128 rows, from the images of its slots: neighbouring lanes read neighbouring
// 16 bytes, where rows of the tensor itself would be a line of memory apart
template <int DP, int N = DP>
__device__ __forceinline__ void stage_image(uint32_t addr, const char* im, int r, int c0 = 0) {
  const char* at = im + r / SLOT * Image<DP>::BYTES + r % SLOT / 8 * (DP * 16) + r % 8 * 16 + c0 * 16;
  uint4 v[PLANES][N / 8];
#pragma unroll
  for (int x = 0; x < PLANES; ++x)
#pragma unroll
    for (int c = 0; c < N / 8; ++c) v[x][c] = *reinterpret_cast<const uint4*>(at + x * Image<DP>::PLANE + c * 128);
#pragma unroll
  for (int x = 0; x < PLANES; ++x)
#pragma unroll
    for (int c = 0; c < N / 8; c += 2)
      tmem_st8(addr + x * (DP / 2) + c0 / 2 + c * 4, reinterpret_cast<const uint32_t*>(&v[x][c]));
}

// N columns from c0 on of a warp's 32 rows (a lane has a row), through shared memory so that whole lines are written;
// `rows` of them exist. NaN where the block gave up.
template <int N>
__device__ __forceinline__ void store_rows(float* scratch, const float* v, float* out, int64_t stride, int rows, int c0, int D, bool ok) {
  constexpr int LD = N + 4, PER = N / 4;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < N; j += 4) *reinterpret_cast<float4*>(scratch + lane * LD + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
  __syncwarp();
  const int c = lane % PER * 4;
  for (int r = lane / PER; r < rows; r += 32 / PER) {
    float4 x = *reinterpret_cast<const float4*>(scratch + r * LD + c);
    if (!ok) x.x = x.y = x.z = x.w = __int_as_float(0x7fc00000);
    float* to = out + r * stride + c0 + c;
    if (D % 4 == 0) {
      if (c0 + c < D) *reinterpret_cast<float4*>(to) = x;
    } else {
      if (c0 + c < D) to[0] = x.x;
      if (c0 + c + 1 < D) to[1] = x.y;
      if (c0 + c + 2 < D) to[2] = x.z;
      if (c0 + c + 3 < D) to[3] = x.w;
    }
  }
}
template <int N>
__device__ __forceinline__ float* scratch_of(char* smem, int warp) { return reinterpret_cast<float*>(smem) + warp * 32 * (N + 4); }

// acc += N columns of tensor memory
template <int N>
__device__ __forceinline__ void add_columns(uint32_t addr, float* acc) {
#pragma unroll
  for (int c = 0; c < N; c += 16) {
    float o[16];
    tmem_ld16(addr + c, o);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 16; j += 2) get(two(acc[c + j], acc[c + j + 1]) + two(o[j], o[j + 1]), acc[c + j], acc[c + j + 1]);
  }
}

// ---- images on the host side ----
struct Source { const float* at; int64_t row, head; int heads; const uint8_t* mask; char* out; };
constexpr int MAX_SOURCES = 7;
struct Sources { Source s[MAX_SOURCES]; };

inline int image_slots(const Params<float>& p) { return part_blocks(p, SLOT) + 1; }   // the last: read behind the end by load_block
template <int DP> int64_t image_bytes(const Params<float>& p, int heads) { return (int64_t)heads * image_slots(p) * Image<DP>::BYTES; }
// the images of `count` tensors and, with `stats`, L and D (and room for more) of the rows of each slot: `kinds` x SLOT
// numbers a (head, slot)
template <int DP>
cudaError_t write_images(const Params<float>& p, const Sources& src, int count, float* stats, int kinds, cudaStream_t s);

}  // namespace attn
