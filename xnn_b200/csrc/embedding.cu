// Lookup of table rows by id with a scale, and its gradient by sorted ids.
//
//   out[n] = scale table[id_n]        (zero where id_n is outside the table: a padded entry)
//   gtable[v] = scale sum_{n: id_n = v} g[n]
//
// The gradient sorts the ids (stable radix sort, eight bits a pass, (key, row) pairs), then walks the sorted
// order in chunks: a warp sums the rows of each run of equal ids inside its chunk. A run inside one chunk
// goes to the table; the part of a run that began before the chunk, and the one that goes on behind it, are
// written to one of the chunk's two partial rows. A warp (or, for long runs, a block) per table row then adds the partials of its run in their order
// and writes zeros where no id came. Every sum has a fixed order; there are no atomics on values.
// Small inputs (rule at `collects`) skip the sort: a block per table row collects its ids itself.
#include "common.cuh"
#include "embedding_impl.h"

namespace {

template <typename T> struct alignas(16) Pack { T x[16 / sizeof(T)]; };

// Sums of eight terms as a tree, so that a sum is a chain of an eighth of its terms; where that may still be long, the running
// correction of compensated summation (Kahan, CACM 8, 1965) keeps the error at two roundings of the terms' magnitudes. An
// infinite or NaN sum stays what it is. Together a table row is off by fewer than 100 roundings (half a step each) of its terms'
// magnitudes, however many there are: in a chunk 3 + MOST / 8 and up to 14 for what is not eight of one id, of its partials
// 3 + 2, of a block's warps 3 + 4, the scale 1. (Sums in 64 bits: 400000 ids of 7569 rows x 128 111 us, this way 83.)
constexpr int TREE = 8, MOST = 512;

template <typename T>
__device__ __forceinline__ T tree(const T (&x)[TREE]) {
  return ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
}

template <typename T>
__device__ __forceinline__ void add(T& s, T& low, T x) {
  const T y = x - low, t = s + y, d = (t - s) - y;
  low = isfinite(d) ? d : T(0);
  s = t;
}

// A thread takes LOOKUPS pieces of 16 bytes, a block apart, so that its id and row loads overlap; what is
// written is not read again here, so it goes past the caches. 400000 rows of 128 floats: 34 us, 6.1 TB/s written.
constexpr int LOOKUPS = 4;

template <typename T, typename I>
__global__ void __launch_bounds__(256) lookup_kernel(uint32_t items, uint32_t per, int64_t V, int C, const T* __restrict__ table,
                                                     const I* __restrict__ ids, T scale, T* __restrict__ out) {
  constexpr int W = 16 / sizeof(T);
  const uint32_t first = blockIdx.x * (256u * LOOKUPS) + threadIdx.x;
  int64_t v[LOOKUPS];
  uint32_t n[LOOKUPS], c[LOOKUPS];
#pragma unroll
  for (int u = 0; u < LOOKUPS; ++u) {
    const uint32_t i = first + u * 256u;
    n[u] = i / per;
    c[u] = (i - n[u] * per) * W;
    v[u] = i < items ? row_of(ids, n[u], V) : -1;
  }
  Pack<T> a[LOOKUPS];
#pragma unroll
  for (int u = 0; u < LOOKUPS; ++u) {
#pragma unroll
    for (int e = 0; e < W; ++e) a[u].x[e] = T(0);
    if (v[u] >= 0) a[u] = *reinterpret_cast<const Pack<T>*>(table + v[u] * C + c[u]);
  }
#pragma unroll
  for (int u = 0; u < LOOKUPS; ++u) {
#pragma unroll
    for (int e = 0; e < W; ++e) a[u].x[e] *= scale;
    if (first + u * 256u < items) __stcs(reinterpret_cast<float4*>(out + (int64_t)n[u] * C + c[u]), *reinterpret_cast<float4*>(&a[u]));
  }
}

// Rows that are no whole number of 16 bytes (or not on such boundaries): a thread writes 16 bytes of the output, whatever rows
// they are of. 400000 rows of 127 floats: 58 us (97 with single
// elements, each with its own division).
template <typename T, typename I>
__global__ void __launch_bounds__(256) lookup_odd_kernel(uint32_t items, uint32_t C, int64_t V, const T* __restrict__ table,
                                                         const I* __restrict__ ids, T scale, T* __restrict__ out) {
  constexpr int W = 16 / sizeof(T);
  const uint32_t e0 = (blockIdx.x * 256u + threadIdx.x) * W;
  if (e0 >= items) return;
  if (e0 + W <= items) {
    Pack<T> a;
    walk_elements<W, true>(e0, items, C, V, ids, [&](int e, int64_t v, uint32_t c) { a.x[e] = v < 0 ? T(0) : table[v * C + c]; });
#pragma unroll
    for (int e = 0; e < W; ++e) a.x[e] *= scale;
    __stcs(reinterpret_cast<float4*>(out + e0), *reinterpret_cast<float4*>(&a));
  } else {
    walk_elements<W, false>(e0, items, C, V, ids,
                            [&](int e, int64_t v, uint32_t c) { out[e0 + e] = v < 0 ? T(0) : scale * table[v * C + c]; });
  }
}

// ---- sort: each block takes `tile` pairs, each of its 32 warps a contiguous share, in strips of 32 ----
constexpr int SORT_WARPS = 32;

template <typename I>
__device__ __forceinline__ int key_at(const I* ids, const int* keys, int64_t i, int64_t V) {
  if (keys) return keys[i];
  const int64_t v = row_of(ids, i, V);
  return v < 0 ? (int)V : (int)v;                       // padded entries sort behind the table
}

template <typename I>
__global__ void __launch_bounds__(256) count_kernel(int N, int64_t V, int tile, int shift, const I* __restrict__ ids,
                                                    const int* __restrict__ keys, int* __restrict__ counts) {
  __shared__ int c[256];
  c[threadIdx.x] = 0;
  __syncthreads();
  const int end = min(N, (int)(blockIdx.x + 1) * tile);
  for (int i = blockIdx.x * tile + threadIdx.x; i < end; i += 256) atomicAdd(&c[(key_at(ids, keys, i, V) >> shift) & 255], 1);
  __syncthreads();
  counts[blockIdx.x * 256 + threadIdx.x] = c[threadIdx.x];
}

template <typename I>
__global__ void __launch_bounds__(1024) place_kernel(int N, int64_t V, int tile, int shift, const I* __restrict__ ids,
                                                     const int* __restrict__ keys, const int* __restrict__ rows,
                                                     const int* __restrict__ counts, int* __restrict__ keys_out,
                                                     int* __restrict__ rows_out) {
  __shared__ int base[SORT_WARPS][256];
  __shared__ int scan[8];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, digit = t & 255, quarter = t >> 8;
  // where this block's entries of a digit start: entries of smaller digits, then those of earlier blocks; each
  // quarter of the block adds up a quarter of the blocks' counts
  int before = 0, total = 0;
  const int share = ((int)gridDim.x + 3) / 4, b1 = min((int)gridDim.x, (quarter + 1) * share);
#pragma unroll 16
  for (int b = quarter * share; b < b1; ++b) {
    const int v = counts[b * 256 + digit];
    before += b < (int)blockIdx.x ? v : 0;
    total += v;
  }
  base[quarter][digit] = before;
  base[4 + quarter][digit] = total;
  __syncthreads();
  int start = 0, incl = 0;
  if (t < 256) {
#pragma unroll
    for (int x = 0; x < 4; ++x) { start += base[x][t]; incl += base[4 + x][t]; }
    start -= incl;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int u = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += u; }
    start += incl;
    if (lane == 31) scan[warp] = incl;
  }
  __syncthreads();
#pragma unroll
  for (int x = 0; x < SORT_WARPS / 4; ++x) base[quarter + 4 * x][digit] = 0;
  if (t < 256)
    for (int w = 0; w < warp; ++w) start += scan[w];
  __syncthreads();
  const int per = tile / SORT_WARPS;
  const int end = min(N, (int)(blockIdx.x + 1) * tile);
  const int first = blockIdx.x * tile + warp * per, last = min(end, first + per);
  for (int i = first + lane; i < last; i += 32) atomicAdd(&base[warp][(key_at(ids, keys, i, V) >> shift) & 255], 1);
  __syncthreads();
  if (t < 256) {
#pragma unroll 8
    for (int w = 0; w < SORT_WARPS; ++w) { const int c = base[w][t]; base[w][t] = start; start += c; }
  }
  __syncthreads();
  for (int i0 = first; i0 < last; i0 += 32) {
    const int i = i0 + lane;
    const bool in = i < last;
    const int key = in ? key_at(ids, keys, i, V) : 0, d = in ? (key >> shift) & 255 : 256;
    const unsigned same = __match_any_sync(0xffffffffu, d);
    const int rank = __popc(same & ((1u << lane) - 1));
    int at = 0;
    if (in) at = base[warp][d] + rank;
    __syncwarp();
    if (in && rank == 0) base[warp][d] += __popc(same);
    __syncwarp();
    if (in) {
      keys_out[at] = key;
      rows_out[at] = rows ? rows[i] : i;
    }
  }
}

// ---- sums over the sorted order: a warp per (chunk of R entries, 32 W columns) ----
template <typename T, int W>
__device__ __forceinline__ void put(T* row, const T (&a)[W], T f, int c, int C) {
#pragma unroll
  for (int e = 0; e < W; ++e)
    if (c + e < C) row[c + e] = f * a[e];
}

template <typename T, int W>
__device__ __forceinline__ void get(const T* row, T (&a)[W], int c, int C) {
  if constexpr (W == 1) {
    a[0] = c < C ? row[c] : T(0);
  } else {
    Pack<T> v;
    if (c < C) v = *reinterpret_cast<const Pack<T>*>(row + c);
#pragma unroll
    for (int e = 0; e < W; ++e) a[e] = c < C ? v.x[e] : T(0);
  }
}

// The lanes fetch the keys and rows of 32 entries at once (one dependent load for 32 entries) and pass them round;
// eight gradient rows are then in flight a warp, and eight of one id are added as a tree.
template <typename T, int W>
__global__ void __launch_bounds__(128, 6) runs_kernel(int N, int V, int C, int R, const int* __restrict__ keys,
                                                   const int* __restrict__ rows, const T* __restrict__ g, T scale,
                                                   T* __restrict__ table, T* __restrict__ part) {
  const int chunk = blockIdx.x * 4 + threadIdx.x / 32, lane = threadIdx.x & 31;
  const int64_t first = (int64_t)chunk * R;
  if (first >= N) return;
  const int last = (int)(first + R < N ? first + R : N), i0 = (int)first;
  const int c = (blockIdx.y * 32 + lane) * W;
  T acc[W] = {};
  int key = keys[i0];
  bool open = i0 > 0 && keys[i0 - 1] == key;            // the run began in an earlier chunk
  const auto leave = [&](int next) {                    // the run ends within the chunk
    if (key < V) {
      if (open) put<T, W>(part + (int64_t)(2 * chunk) * C, acc, T(1), c, C);
      else put<T, W>(table + (int64_t)key * C, acc, scale, c, C);
    }
    open = false;
    key = next;
#pragma unroll
    for (int e = 0; e < W; ++e) acc[e] = T(0);
  };
  constexpr int U = TREE;
  int next_key = i0 + lane < last ? keys[i0 + lane] : V, next_row = i0 + lane < last ? rows[i0 + lane] : 0;
  for (int i = i0; i < last; i += 32) {
    const int my_key = next_key, my_row = next_row;
    const int j = i + 32 + lane;
    next_key = j < last ? keys[j] : V;
    next_row = j < last ? rows[j] : 0;
    const int count = min(32, last - i);
    for (int s = 0; s < count; s += U) {
      int k[U];
      T v[U][W];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        k[u] = __shfl_sync(0xffffffffu, my_key, s + u);
        const int row = __shfl_sync(0xffffffffu, my_row, s + u);
        if (k[u] < V) get<T, W>(g + (int64_t)row * C, v[u], c, C);
      }
      if (k[0] == k[U - 1] && s + U <= count) {         // eight of one id
        if (k[0] != key) leave(k[0]);
        if (key < V) {
#pragma unroll
          for (int e = 0; e < W; ++e) acc[e] += tree<T>({v[0][e], v[1][e], v[2][e], v[3][e], v[4][e], v[5][e], v[6][e], v[7][e]});
        }
        continue;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (s + u >= count) break;
        if (k[u] != key) leave(k[u]);
        if (key < V) {
#pragma unroll
          for (int e = 0; e < W; ++e) acc[e] += v[u][e];
        }
      }
    }
  }
  if (key < V) {
    const bool goes_on = last < N && keys[last] == key;
    if (open) put<T, W>(part + (int64_t)(2 * chunk) * C, acc, T(1), c, C);
    else if (goes_on) put<T, W>(part + (int64_t)(2 * chunk + 1) * C, acc, T(1), c, C);
    else put<T, W>(table + (int64_t)key * C, acc, scale, c, C);
  }
}

// first sorted position with a key >= v (all lanes of a warp together)
__device__ __forceinline__ int lower_bound(const int* keys, int N, int v) {
  const int lane = threadIdx.x & 31;
  int at = 0, n = N;                                    // the answer is in [at, at + n]
  while (n > 0) {
    const int step = (n + 31) / 32;
    const int i = lane * step + step - 1;
    const bool less = i < n && keys[at + i] < v;
    const int c = __popc(__ballot_sync(0xffffffffu, less));
    at += c * step;
    n = min(step - 1, n - c * step);
    if (n < 0) n = 0;
  }
  return at;
}

// sum of the partials j0 .. j1 - 1 of a run that begins in chunk c0; the first chunk's share is in its second partial row
template <typename T, int W>
__device__ __forceinline__ void run_part(const T* part, int c0, int j0, int j1, int C, int c, T (&s)[W]) {
#pragma unroll
  for (int e = 0; e < W; ++e) s[e] = T(0);
  T low[W] = {};
  for (int j = j0; j < j1; j += TREE) {
    T v[TREE][W];
#pragma unroll
    for (int u = 0; u < TREE; ++u) get<T, W>(part + (int64_t)(2 * (c0 + j + u) + (j + u == 0 ? 1 : 0)) * C, v[u], j + u < j1 ? c : C, C);
#pragma unroll
    for (int e = 0; e < W; ++e) add(s[e], low[e], tree<T>({v[0][e], v[1][e], v[2][e], v[3][e], v[4][e], v[5][e], v[6][e], v[7][e]}));
  }
}

// A warp per table row and 32 W columns: zeros where no id came, the partials of a run over several chunks added up. Rows of
// more than MANY partials (the few elements that most atoms are) are left to the whole block. A block's rows lie gridDim.x
// apart, so that the popular ids, which are neighbours, meet in different blocks; a table of at most a row an SM has a block
// of 32 warps a row (gradient of 400000 ids of 5 elements, 512 columns: 171 us, 747 with eight rows in one block).
constexpr int MANY = 32;

template <typename T, int W, int WARPS, int ROWS>
__global__ void __launch_bounds__(32 * WARPS) rows_kernel(int N, int V, int C, int R, const int* __restrict__ keys,
                                                          const T* __restrict__ part, T scale, T* __restrict__ table) {
  __shared__ T sums[WARPS][32 * W];
  __shared__ int heavy_first[ROWS], heavy_count[ROWS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = (blockIdx.y * 32 + lane) * W;
  T s[W];
  if (warp < ROWS) {
    const int v = blockIdx.x + warp * gridDim.x;
    int n = 0, c0 = 0;
    if (v < V) {
      const int a = lower_bound(keys, N, v), b = lower_bound(keys, N, v + 1);
      T* out = table + (int64_t)v * C;
      if (a == b) {
#pragma unroll
        for (int e = 0; e < W; ++e) s[e] = T(0);
        put<T, W>(out, s, scale, c, C);
      } else {
        c0 = a / R;
        n = (b - 1) / R - c0 + 1;                       // 1: one chunk had the whole run and has written it
        if (n > 1 && n <= MANY) {
          run_part<T, W>(part, c0, 0, n, C, c, s);
          put<T, W>(out, s, scale, c, C);
        }
      }
    }
    if (lane == 0) {
      heavy_first[warp] = c0;
      heavy_count[warp] = n > MANY ? n : 0;
    }
  }
  __syncthreads();
  for (int w = 0; w < ROWS; ++w) {
    const int m = heavy_count[w];
    if (m == 0) continue;
    const int per = (m + WARPS - 1) / WARPS;
    run_part<T, W>(part, heavy_first[w], min(m, warp * per), min(m, (warp + 1) * per), C, c, s);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < W; ++e) sums[warp][lane * W + e] = s[e];
    __syncthreads();
    if (warp == 0) {
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const int at = lane * W + e;
        s[e] = T(0);
        for (int k = 0; k < WARPS; k += TREE)
          s[e] += tree<T>({sums[k][at], sums[k + 1][at], sums[k + 2][at], sums[k + 3][at], sums[k + 4][at], sums[k + 5][at], sums[k + 6][at], sums[k + 7][at]});
      }
      put<T, W>(table + (int64_t)(blockIdx.x + w * gridDim.x) * C, s, scale, c, C);
    }
  }
}

// ---- small inputs: a block per table row lists its entries in order, then sums them ----
template <typename T, typename I>
__global__ void __launch_bounds__(256) collect_kernel(int N, int64_t V, int C, const I* __restrict__ ids,
                                                      const T* __restrict__ g, T scale, T* __restrict__ table) {
  extern __shared__ __align__(16) char raw[];
  T* sums = reinterpret_cast<T*>(raw);
  int* list = reinterpret_cast<int*>(sums + 256);
  __shared__ int warp_n[8];
  const int v = blockIdx.x, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  int n = 0;
  // four neighbouring ids a thread, so that a turn with its two meetings covers 1024
  const unsigned before = (1u << lane) - 1;
  for (int i0 = 0; i0 < N; i0 += 1024) {
    const int i = i0 + 4 * t;
    bool hit[4];
    int mine = 0, all = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) hit[j] = i + j < N && (int64_t)ids[min(i + j, N - 1)] == v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned b = __ballot_sync(0xffffffffu, hit[j]);
      mine += __popc(b & before);
      all += __popc(b);
    }
    if (lane == 0) warp_n[warp] = all;
    __syncthreads();
    int at = n + mine;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      at += w < warp ? warp_n[w] : 0;
      n += warp_n[w];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (hit[j]) list[at++] = i + j;
    __syncthreads();
  }
  T* out = table + (int64_t)v * C;
  const int lanes = C <= 32 ? 32 : (C <= 64 ? 64 : (C <= 128 ? 128 : 256)), groups = 256 / lanes, group = t / lanes;
  const int per = (n + groups - 1) / groups;
  for (int cb = 0; cb < C; cb += lanes) {
    const int c = cb + t % lanes;
    T s = T(0), low = T(0);
    if (c < C) {
      const int j1 = min(n, (group + 1) * per);
      for (int j = group * per; j < j1; j += TREE) {
        T v[TREE];
#pragma unroll
        for (int u = 0; u < TREE; ++u) v[u] = j + u < j1 ? g[(int64_t)list[j + u] * C + c] : T(0);
        add(s, low, tree(v));
      }
    }
    __syncthreads();
    sums[t] = s;
    __syncthreads();
    if (group == 0 && c < C) {
      for (int k = 1; k < groups; ++k) s += sums[k * lanes + t];
      out[c] = scale * s;
    }
  }
}

constexpr int SMALL_ROWS = 8192;                        // the list of a row's entries is in shared memory

// pairs a sort block takes: at most 148 blocks (each reads every block's counts), 1024 pairs at least
int sort_tile(int64_t N) {
  const int64_t t = (N + 147) / 148;
  return (int)((t + 1023) / 1024 * 1024);
}
// entries a summing warp takes: 32, more when that would pass WARPS_AT_ONCE (eight rows in flight in each of them are enough
// for the memory's latency, and longer chunks leave fewer partial rows), MOST at most, in whole rounds of the warps
constexpr int64_t WARPS_AT_ONCE = 148 * 24;
int run_chunk(int64_t N) {
  const int64_t rounds = (N + WARPS_AT_ONCE * MOST - 1) / (WARPS_AT_ONCE * MOST);
  const int64_t r = (N + rounds * WARPS_AT_ONCE - 1) / (rounds * WARPS_AT_ONCE);
  return (int)(r < 32 ? 32 : (r + 7) / 8 * 8);
}
// Collecting costs N V id reads in all, a block a table row, and sums a row's entries, in the worst case all of them, in one
// block; the sort costs four to ten launches, 15-25 us on the device and as much of the host. Device, collected and sorted, in us:
// 4868 ids of 1777 rows x 11 columns 16 and 22, 8192 of 2000 x 16 27 and 23, of 4000 x 16 49 and 25, of 4 x 16 18 and 15, of
// 4 x 128 53 and 15, of 4 x 512 202 and 15, 611 of 87 x 64 3 and 14; the blocks alone, 16 ids x 64 columns: of 8192 rows 18 and
// 18 (the call 53 and 71), of 16384 35 and 20 (53 and 71), of 32768 68 and 25 (72 and 72), of 2^20 2058 and 223.
constexpr int64_t COLLECTED_ROWS = 16384;
bool collects(int64_t N, int64_t V, int64_t C) {
  return N <= SMALL_ROWS && V <= COLLECTED_ROWS && N * V <= (int64_t)1 << 24 && N * C <= (int64_t)1 << 17;
}

template <typename T, int W>
void add_partials(int N, int V, int C, int R, const int* keys, const T* part, T scale, T* table, cudaStream_t s) {
  const unsigned columns = (unsigned)((C + 32 * W - 1) / (32 * W));
  if (V <= 148) rows_kernel<T, W, 32, 1><<<dim3(V, columns), 1024, 0, s>>>(N, V, C, R, keys, part, scale, table);
  else rows_kernel<T, W, 8, 8><<<dim3((V + 7) / 8, columns), 256, 0, s>>>(N, V, C, R, keys, part, scale, table);
}

}  // namespace

template <typename T, typename I>
cudaError_t embedding_lookup(int64_t N, int64_t V, int C, const T* table, const I* ids, double scale, T* out, cudaStream_t s) {
  constexpr int W = 16 / sizeof(T);
  const bool vec = C % W == 0 && reinterpret_cast<uintptr_t>(table) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  const int64_t per = vec ? C / W : C;
  // pieces are counted in 32 bits: rows in groups that fit, each on a 16-byte boundary of the output
  const int64_t group = ((int64_t)1 << 31) / per / W * W;
  for (int64_t n0 = 0; n0 < N; n0 += group) {
    const int64_t n = N - n0 < group ? N - n0 : group;
    const uint32_t items = (uint32_t)(n * per);
    const unsigned each = vec ? 256 * LOOKUPS : 256 * W, grid = (unsigned)(((int64_t)items + each - 1) / each);
    if (vec) lookup_kernel<T, I><<<grid, 256, 0, s>>>(items, (uint32_t)per, V, C, table, ids + n0, (T)scale, out + n0 * C);
    else lookup_odd_kernel<T, I><<<grid, 256, 0, s>>>(items, (uint32_t)C, V, table, ids + n0, (T)scale, out + n0 * C);
  }
  return cudaGetLastError();
}

// int32 words of workspace for the sort, and elements of T for the partial rows
int64_t embedding_grad_ints(int64_t N, int64_t V, int64_t C) {
  if (collects(N, V, C)) return 0;
  const int64_t tile = sort_tile(N);
  return 4 * N + (N + tile - 1) / tile * 256;
}
int64_t embedding_grad_partials(int64_t N, int64_t V, int64_t C) {
  if (collects(N, V, C)) return 0;
  const int64_t R = run_chunk(N);
  return (N + R - 1) / R * 2 * C;
}

template <typename T, typename I>
cudaError_t embedding_grad(int64_t N, int64_t V, int C, const I* ids, const T* g, double scale, int* ints, T* partials,
                           T* table, cudaStream_t s) {
  if (collects(N, V, C)) {
    collect_kernel<T, I><<<(unsigned)V, 256, 256 * sizeof(T) + sizeof(int) * (size_t)N, s>>>((int)N, V, C, ids, g, (T)scale, table);
    return cudaGetLastError();
  }
  const int tile = sort_tile(N), blocks = (int)((N + tile - 1) / tile);
  int *keys[2] = {ints, ints + N}, *rows[2] = {ints + 2 * N, ints + 3 * N}, *counts = ints + 4 * N;
  int bits = 1;
  while (((int64_t)1 << bits) <= V) ++bits;             // keys 0 .. V
  int at = 0;
  for (int shift = 0; shift < bits; shift += 8) {
    const int* kin = shift ? keys[at ^ 1] : nullptr;
    const int* rin = shift ? rows[at ^ 1] : nullptr;
    count_kernel<I><<<blocks, 256, 0, s>>>((int)N, V, tile, shift, ids, kin, counts);
    place_kernel<I><<<blocks, 1024, 0, s>>>((int)N, V, tile, shift, ids, kin, rin, counts, keys[at], rows[at]);
    at ^= 1;
  }
  const int *k = keys[at ^ 1], *r = rows[at ^ 1];
  const int R = run_chunk(N), chunks = (int)((N + R - 1) / R);
  constexpr int W = 16 / sizeof(T);
  const bool vec = C % W == 0 && reinterpret_cast<uintptr_t>(g) % 16 == 0;
  const int cols = 32 * (vec ? W : 1);
  const dim3 grid((chunks + 3) / 4, (C + cols - 1) / cols);
  if (vec) runs_kernel<T, W><<<grid, 128, 0, s>>>((int)N, (int)V, C, R, k, r, g, (T)scale, table, partials);
  else runs_kernel<T, 1><<<grid, 128, 0, s>>>((int)N, (int)V, C, R, k, r, g, (T)scale, table, partials);
  // partial rows start on 16-byte boundaries where a whole number of vectors makes a row
  if (C % W == 0) add_partials<T, W>((int)N, (int)V, C, R, k, partials, (T)scale, table, s);
  else add_partials<T, 1>((int)N, (int)V, C, R, k, partials, (T)scale, table, s);
  return cudaGetLastError();
}

#define XNN_EMB_INST(T, I)                                                                                          \
  template cudaError_t embedding_lookup<T, I>(int64_t, int64_t, int, const T*, const I*, double, T*, cudaStream_t); \
  template cudaError_t embedding_grad<T, I>(int64_t, int64_t, int, const I*, const T*, double, int*, T*, T*, cudaStream_t);
XNN_EMB_INST(float, int64_t)
XNN_EMB_INST(float, int)
XNN_EMB_INST(double, int64_t)
XNN_EMB_INST(double, int)
