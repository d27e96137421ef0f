// Token embedding: rows of a table by id, and the gradient of the table (include/pmg_lm.h).
//
//   y_n = scale W[id_n]            dW_v = scale sum_{n : id_n = v, v != padding} dy_n
//
// Both are bound by memory.  The gradient has no atomics: the positions are sorted by id (stable, so that
// the sum over a token's positions has one order), cut into chunks of equal length whatever the ids are, and
// each chunk sums runs of equal ids; a run that crosses chunks leaves partial rows that are joined
// afterwards in a fixed order.  A frequent token (padding apart, which is dropped) therefore spreads over
// the chip like any other rows, and equal inputs give equal bits.
//   1. sort    N <= 2048: one workgroup, bitonic in LDS;  else LSD radix, up to 9 bits a pass, three launches
//              a pass (digit counts per tile, their scan per digit, stable scatter)
//   2. reduce  runs -> rows of dW or partial rows; other workgroups of the same launch write the zero rows
//              of tokens that do not occur, so every row of dW is written once
//   3. join    partial rows of runs that cross chunks
#include "pmg_types.h"

namespace {

constexpr int THREADS = 256;
constexpr int SMALL_N = 2048;   // one-workgroup sort: 66 steps in LDS, less than the radix passes' launches
constexpr int ROUND = 256;      // keys a workgroup of the radix sort takes at a time: 4 waves x 64
constexpr int MAX_BITS = 9;     // digit bits a pass: 17 bits of ids (128 k tokens) in two passes
constexpr int MAX_BINS = 1 << MAX_BITS;
constexpr int FILL_ROWS = 64;   // table rows a workgroup checks and zeroes
constexpr int JOIN_THREADS = 256;
constexpr int HELD = 2048;      // sorted keys and positions that a workgroup of the reduction holds in LDS
// Workgroups a launch: of 2^32 threads or more in a dimension only some run, without an error.
constexpr int64_t MOST_GROUPS = 1 << 23;

// ids outside [0, V) and the padding id sort behind all tokens and take no part
template <typename I> __device__ __forceinline__ uint32_t key_of(I id, int64_t V, int64_t pad) {
  const int64_t v = (int64_t)id;
  return (v < 0 || v >= V || v == pad) ? (uint32_t)V : (uint32_t)v;
}

// ------------------------------------------------------------------------------------------ forward
// tpr threads (a power of two) share a row, 16 bytes each; ROWS rows a thread keep several loads in flight.
template <typename T, typename I, int ROWS>
__global__ __launch_bounds__(THREADS) void embed_fwd_kernel(const T* __restrict__ W, int64_t ldw,
                                                            const I* __restrict__ ids, int64_t N, int64_t V, int64_t E,
                                                            float scale, int tpr, T* __restrict__ out) {
  constexpr int VEC = pmg_vec16<T>::N;
  const int rpw = THREADS / tpr;
  const int64_t c = ((int64_t)blockIdx.y * tpr + (threadIdx.x & (tpr - 1))) * VEC;
  if (c >= E) return;
  const int64_t row0 = (int64_t)blockIdx.x * rpw * ROWS + threadIdx.x / tpr;
  typename pmg_vec16<T>::vec x[ROWS];
  bool ok[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int64_t n = row0 + (int64_t)r * rpw;
    const int64_t id = n < N ? (int64_t)ids[n] : 0;
    ok[r] = id >= 0 && id < V;
    if (n < N) x[r] = pmg_vec16<T>::load(W + (ok[r] ? id : 0) * ldw + c, E - c);
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int64_t n = row0 + (int64_t)r * rpw;
    if (n >= N) break;
    float y[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) y[j] = ok[r] ? (float)x[r][j] * scale : __builtin_nanf("");
    pmg_vec16<T>::store(out + n * E + c, y, E - c);
  }
}

// ------------------------------------------------------------------------------------------ sort
template <typename I>
__global__ __launch_bounds__(1024) void embed_sort_small_kernel(const I* __restrict__ ids, int N, int64_t V, int64_t pad,
                                                                uint32_t* __restrict__ keys, uint32_t* __restrict__ pos) {
  __shared__ uint64_t s[SMALL_N];
  int size = 64;
  while (size < N) size <<= 1;
  for (int i = threadIdx.x; i < size; i += 1024)
    s[i] = i < N ? ((uint64_t)key_of(ids[i], V, pad) << 32) | (uint32_t)i : ~(uint64_t)0;
  __syncthreads();
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      const int t = threadIdx.x;
      if (t < size / 2) {
        const int a = ((t & ~(j - 1)) << 1) | (t & (j - 1)), b = a | j;
        const uint64_t x = s[a], y = s[b];
        if ((x > y) == ((a & k) == 0)) {
          s[a] = y;
          s[b] = x;
        }
      }
      __syncthreads();
    }
  for (int i = threadIdx.x; i < N; i += 1024) {
    keys[i] = (uint32_t)(s[i] >> 32);
    pos[i] = (uint32_t)s[i];
  }
}

// Where a radix pass takes its keys from: the ids themselves (first pass) or the pass before.
template <typename I> struct FromIds {
  const I* ids;
  int64_t V, pad;
  __device__ __forceinline__ uint32_t key(int64_t i) const { return key_of(ids[i], V, pad); }
  __device__ __forceinline__ uint32_t pos(int64_t i) const { return (uint32_t)i; }
};
struct FromKeys {
  const uint32_t *keys, *at;
  __device__ __forceinline__ uint32_t key(int64_t i) const { return keys[i]; }
  __device__ __forceinline__ uint32_t pos(int64_t i) const { return at[i]; }
};

// count[digit * tiles + tile]
template <typename Src, int ROUNDS>
__global__ __launch_bounds__(THREADS) void embed_count_kernel(const Src src, int64_t N, int shift, int bits, int tiles,
                                                              int* __restrict__ count) {
  __shared__ int bin[MAX_BINS];
  const int bins = 1 << bits;
  for (int b = threadIdx.x; b < bins; b += THREADS) bin[b] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * (ROUNDS * ROUND);
  uint32_t key[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int64_t i = base + r * THREADS + threadIdx.x;
    key[r] = src.key(i < N ? i : N - 1);
  }
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r)
    if (base + r * THREADS + threadIdx.x < N) atomicAdd(&bin[(key[r] >> shift) & (bins - 1)], 1);  // integers: any order, one result
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += THREADS) count[(int64_t)b * tiles + blockIdx.x] = bin[b];
}

__device__ __forceinline__ int wave_scan(int v) {  // inclusive
  const int lane = threadIdx.x & 63;
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}

// One workgroup a digit: exclusive scan of its counts over the tiles, in place; total[digit].
__global__ __launch_bounds__(THREADS) void embed_scan_kernel(int* __restrict__ count, int tiles, int* __restrict__ total) {
  __shared__ int wsum[THREADS / 64];
  int* row = count + (int64_t)blockIdx.x * tiles;
  int carry = 0;
  for (int base = 0; base < tiles; base += THREADS) {
    const int i = base + threadIdx.x;
    const int v = i < tiles ? row[i] : 0;
    const int inc = wave_scan(v);
    if ((threadIdx.x & 63) == 63) wsum[threadIdx.x >> 6] = inc;
    __syncthreads();
    int pre = carry;
    for (int w = 0; w < (int)(threadIdx.x >> 6); ++w) pre += wsum[w];
    if (i < tiles) row[i] = pre + inc - v;
    carry += (wsum[0] + wsum[1]) + (wsum[2] + wsum[3]);
    __syncthreads();
  }
  if (threadIdx.x == 0) total[blockIdx.x] = carry;
}

// LDS written by other lanes of the wave is read behind this: a wave runs in step, the compiler has to be told.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Stable: a wave takes ROUNDS x 64 consecutive keys in rounds of 64; keys of one digit in a round are ranked by
// lane, rounds and waves by running counts.
template <typename Src, int ROUNDS>
__global__ __launch_bounds__(THREADS) void embed_scatter_kernel(const Src src, int64_t N, int shift, int bits, int tiles,
                                                                const int* __restrict__ count,
                                                                const int* __restrict__ total,
                                                                uint32_t* __restrict__ keys, uint32_t* __restrict__ pos) {
  __shared__ int place[THREADS / 64][MAX_BINS];  // counts of a wave's keys, then where its next key of a digit goes
  __shared__ int start[MAX_BINS];
  __shared__ int wsum[THREADS / 64];
  const int bins = 1 << bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int b = lane; b < bins; b += 64) place[wave][b] = 0;
  // first position of every digit: exclusive scan of the totals
  int carry = 0;
  for (int base = 0; base < bins; base += THREADS) {
    const int b = base + threadIdx.x;
    const int v = b < bins ? total[b] : 0;
    const int inc = wave_scan(v);
    if (lane == 63) wsum[wave] = inc;
    __syncthreads();
    int pre = carry;
    for (int w = 0; w < wave; ++w) pre += wsum[w];
    if (b < bins) start[b] = pre + inc - v;
    carry += (wsum[0] + wsum[1]) + (wsum[2] + wsum[3]);
    __syncthreads();
  }
  const int64_t base = (int64_t)blockIdx.x * (ROUNDS * ROUND) + wave * (ROUNDS * 64) + lane;
  uint32_t key[ROUNDS], from[ROUNDS];
  uint64_t same[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int64_t i = base + r * 64 < N ? base + r * 64 : N - 1;
    key[r] = src.key(i);
    from[r] = src.pos(i);
  }
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const bool in = base + r * 64 < N;
    const int d = (key[r] >> shift) & (bins - 1);
    uint64_t m = __ballot(in);
    for (int b = 0; b < bits; ++b) {
      const uint64_t v = __ballot((d >> b) & 1);
      m &= ((d >> b) & 1) ? v : ~v;
    }
    same[r] = in ? m : 0;
    if (in && (m & ((1ull << lane) - 1)) == 0) place[wave][d] += __popcll(m);  // first lane of the digit
    wave_sync();
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += THREADS) {
    int at = start[b] + count[(int64_t)b * tiles + blockIdx.x];
    for (int w = 0; w < THREADS / 64; ++w) {
      const int n = place[w][b];
      place[w][b] = at;
      at += n;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    if (same[r]) {
      const int d = (key[r] >> shift) & (bins - 1);
      const int rank = __popcll(same[r] & ((1ull << lane) - 1));
      const int at = place[wave][d];
      wave_sync();
      keys[at + rank] = key[r];
      pos[at + rank] = from[r];
      if (rank == 0) place[wave][d] = at + __popcll(same[r]);
    }
    wave_sync();
  }
}

// ------------------------------------------------------------------------------------------ reduce
struct ReduceArgs {
  int64_t N, V, E, ldg;
  float scale;
  int tpr, chunk;            // threads a row piece, sorted positions a chunk
  int64_t chunks, reduce_blocks;
  const uint32_t *keys, *pos;
  float* part;               // [chunks][2][E]: [0] of the run that began earlier, [1] of the run that goes on
  int64_t join_from;         // the first chunk of a launch that joins
};

// WHOLE: rows of 16 bytes or more; the last 16 bytes of a row that is no multiple of them overlap those before (both
// threads form and write the same values), so that no load needs a branch: loads with branches between them wait for each
// other (32767 x 2048 bf16: 74 us, 79 with branches; 417792 x 128 fp32: 52 and 61; 524288 x 512 bf16: 160 and 173, joining
// 34 and 48).
template <typename T, bool WHOLE>
__global__ __launch_bounds__(THREADS) void embed_reduce_kernel(const ReduceArgs a, const T* __restrict__ g,
                                                               T* __restrict__ dW) {
  constexpr int VEC = pmg_vec16<T>::N;
  constexpr int U = 8;  // rows loaded ahead of their sum
  if ((int64_t)blockIdx.x >= a.reduce_blocks) {
    // rows of tokens that do not occur
    __shared__ int absent[FILL_ROWS];
    if (blockIdx.y > 0) return;
    const int64_t v0 = ((int64_t)blockIdx.x - a.reduce_blocks) * FILL_ROWS;
    if (threadIdx.x < FILL_ROWS) {
      const int64_t v = v0 + threadIdx.x;
      int64_t lo = 0, hi = a.N;
      while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if ((int64_t)a.keys[mid] < v) lo = mid + 1;
        else hi = mid;
      }
      absent[threadIdx.x] = v < a.V && !(lo < a.N && (int64_t)a.keys[lo] == v);
    }
    __syncthreads();
    const float zero[VEC] = {};
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int r = wave; r < FILL_ROWS; r += THREADS / 64)
      if (absent[r])
        for (int64_t c = lane * VEC; c < a.E; c += 64 * VEC) pmg_vec16<T>::store(dW + (v0 + r) * a.E + c, zero, a.E - c);
    return;
  }
  // the workgroup's keys and positions, and the keys next to them
  __shared__ uint32_t key[HELD + 2], pos[HELD];
  const int per = THREADS / a.tpr * a.chunk;
  const int64_t first = (int64_t)blockIdx.x * per;
  for (int i = threadIdx.x; i < per + 2; i += THREADS) {
    const int64_t p = first + i - 1;
    key[i] = p >= 0 && p < a.N ? a.keys[p] : ~0u;
    if (i >= 1 && i <= per && p < a.N) pos[i - 1] = a.pos[p];
  }
  __syncthreads();
  int64_t c = ((int64_t)blockIdx.y * a.tpr + (threadIdx.x & (a.tpr - 1))) * VEC;
  const int grp = threadIdx.x / a.tpr;
  const int64_t ch = (int64_t)blockIdx.x * (THREADS / a.tpr) + grp;
  if (c >= a.E || ch >= a.chunks) return;
  if (WHOLE && c > a.E - VEC) c = a.E - VEC;
  const int lo = grp * a.chunk, n = (int)(a.N - ch * a.chunk < a.chunk ? a.N - ch * a.chunk : a.chunk);
  const uint32_t* k = key + 1 + lo;  // k[-1] and k[n]: the neighbours
  const uint32_t* at = pos + lo;
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
  uint32_t cur = k[0];
  if (cur >= (uint32_t)a.V) return;  // dropped positions sort last
  bool before = k[-1] == cur;
  auto put_part = [&](int slot) __attribute__((always_inline)) {
    float* p = a.part + (ch * 2 + slot) * a.E + c;
#pragma unroll
    for (int j = 0; j < VEC; j += 4) {
      if (WHOLE || c + j < a.E) pmg_store4(p + j, f32x4{acc[j], acc[j + 1], acc[j + 2], acc[j + 3]}, WHOLE ? 4 : a.E - c - j);
    }
  };
  auto put_row = [&]() __attribute__((always_inline)) {
    float y[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) y[j] = acc[j] * a.scale;
    pmg_vec16<T>::store(dW + (int64_t)cur * a.E + c, y, WHOLE ? VEC : a.E - c);
  };
  typedef typename pmg_vec16<T>::vec vec;
  vec x[2][U];
  // no branches between the loads (behind the end the last row again; dropped positions have a row too)
  auto load = [&](vec(&v)[U], int i) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      v[u] = pmg_vec16<T>::load(g + (int64_t)at[i + u < n ? i + u : n - 1] * a.ldg + c, WHOLE ? VEC : a.E - c);
  };
  // false: what follows takes no part (dropped positions sort last)
  auto add = [&](const vec(&v)[U], int i) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u < n) {
        const uint32_t q = k[i + u];
        if (q != cur) {
          if (before) put_part(0);
          else put_row();
          before = false;
          cur = q;
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
        }
        if (cur >= (uint32_t)a.V) return false;
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += (float)v[u][j];
      }
    }
    return true;
  };
  load(x[0], 0);
  for (int i = 0; i < n; i += 2 * U) {  // the rows of one set are under way while the other is added up
    load(x[1], i + U);
    if (!add(x[0], i)) return;
    load(x[0], i + 2 * U);
    if (!add(x[1], i + U)) return;
  }
  if (before) put_part(0);
  else if (k[n] == cur) put_part(1);
  else put_row();
}

// One workgroup a chunk and column block; only a chunk whose last run begins in it and goes on has work (most do where
// tokens are frequent, with two or three parts each: small workgroups, 43 us with 1024 threads at 32767 x 2048): the
// parts of the run are dealt to the workgroup's groups of tpr threads in turn, and the groups' sums are
// added in order.
template <typename T, bool WHOLE>
__global__ __launch_bounds__(JOIN_THREADS) void embed_join_kernel(const ReduceArgs a, T* __restrict__ dW) {
  constexpr int VEC = pmg_vec16<T>::N;
  __shared__ float sum[JOIN_THREADS * VEC];
  const int64_t ch = a.join_from + blockIdx.x, lo = ch * a.chunk, hi = lo + a.chunk;
  if (hi >= a.N) return;
  const uint32_t cur = a.keys[hi];
  if (cur >= (uint32_t)a.V || a.keys[hi - 1] != cur) return;
  if (a.keys[lo] == cur && lo > 0 && a.keys[lo - 1] == cur) return;  // began earlier: another chunk's run
  // the last chunk that begins inside the run: all threads look at the chunks behind this one
  __shared__ int ends;
  int64_t last = ch + 1;
  for (int64_t base = ch + 1;; base += JOIN_THREADS) {
    if (threadIdx.x == 0) ends = JOIN_THREADS;
    __syncthreads();
    const int64_t k = base + threadIdx.x;
    if (k >= a.chunks || a.keys[k * a.chunk] != cur) atomicMin(&ends, (int)threadIdx.x);
    __syncthreads();
    const int e = ends;
    last = base + e - 1;
    if (e < JOIN_THREADS) break;
    __syncthreads();
  }
  const int groups = JOIN_THREADS / a.tpr, grp = threadIdx.x / a.tpr, t = threadIdx.x & (a.tpr - 1);
  int64_t c = ((int64_t)blockIdx.y * a.tpr + t) * VEC;
  const bool in = c < a.E;
  if (WHOLE && c > a.E - VEC) c = a.E - VEC;
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
  if (in) {
#pragma unroll 16
    for (int64_t k = ch + grp; k <= last; k += groups) {  // long runs: many loads under way
      const float* p = a.part + (k * 2 + (k == ch ? 1 : 0)) * a.E + c;
#pragma unroll
      for (int j = 0; j < VEC; j += 4) {
        if (WHOLE || c + j < a.E) {
          const f32x4 x = pmg_load4(p + j, WHOLE ? 4 : a.E - c - j);
          acc[j] += x.x; acc[j + 1] += x.y; acc[j + 2] += x.z; acc[j + 3] += x.w;
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) sum[j * JOIN_THREADS + threadIdx.x] = acc[j];
  __syncthreads();
  if (grp == 0 && in) {
    float y[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      float s = 0.0f;
      for (int q = 0; q < groups; ++q) s += sum[j * JOIN_THREADS + q * a.tpr + t];
      y[j] = s * a.scale;
    }
    pmg_vec16<T>::store(dW + (int64_t)cur * a.E + c, y, WHOLE ? VEC : a.E - c);
  }
}

// ------------------------------------------------------------------------------------------ host
int threads_per_row(int64_t E, int vec) {  // a power of two up to a wave
  const int64_t v = (E + vec - 1) / vec;
  int t = 1;
  while (t < v && t < 64) t <<= 1;
  return t;
}

// Sorted positions a chunk: 8, so that few positions spread over the chip; doubled up to 64, so that the partial rows stay
// a small part of what is read, while that leaves a workgroup for every CU (32258 x 20 over 7914: 32 us with 8, 47 with
// 32) and a thousand chunks.
int chunk_of(int64_t N, int64_t E, int vec, int tpr) {
  const int64_t cols = (E + (int64_t)tpr * vec - 1) / ((int64_t)tpr * vec), rpw = THREADS / tpr;
  int c = 8;
  while (c < 64 && N / c > 1024 && N / c / rpw * cols > 256 && c * 2 * rpw <= HELD) c <<= 1;
  return c;
}

int key_bits(int64_t V) {  // keys 0 .. V
  int b = 1;
  while (((int64_t)1 << b) <= V) ++b;
  return b;
}

struct BwdLayout {
  size_t keys[2], pos[2], count, total, part, bytes;
  int64_t tiles, chunks;
  int chunk, tpr, rounds;
};

BwdLayout bwd_layout(int64_t N, int64_t E, int dtype) {
  BwdLayout L;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t p = at;
    at += (bytes + 255) & ~(size_t)255;
    return p;
  };
  // rounds of 256 keys a workgroup of the sort: fewer where there would be few workgroups
  L.rounds = N >= 256 * 2048 ? 8 : 2;
  L.tiles = (N + L.rounds * ROUND - 1) / (L.rounds * ROUND);
  L.tpr = threads_per_row(E, 16 / (int)pmg_elem_bytes(dtype));
  L.chunk = chunk_of(N, E, 16 / (int)pmg_elem_bytes(dtype), L.tpr);
  L.chunks = (N + L.chunk - 1) / L.chunk;
  const bool small = N <= SMALL_N;
  for (int i = 0; i < 2; ++i) {
    L.keys[i] = i == 1 && small ? L.keys[0] : take((size_t)N * 4);
    L.pos[i] = i == 1 && small ? L.pos[0] : take((size_t)N * 4);
  }
  L.count = take(small ? 0 : (size_t)L.tiles * MAX_BINS * 4);
  L.total = take(small ? 0 : MAX_BINS * 4);
  L.part = take((size_t)L.chunks * 2 * (size_t)E * 4);
  L.bytes = at ? at : 256;
  return L;
}

int embed_args_ok(int64_t N, int64_t V, int64_t E, int dtype, int id_bits) {
  if (N < 0 || V < 1 || E < 1 || N > 0x7fffffff - 8 * ROUND || V > 0x7ffffffe || E > ((int64_t)1 << 22)) return PMG_E_ARG;
  if (!pmg_dtype_ok(dtype)) return PMG_E_DTYPE;
  if (id_bits != 32 && id_bits != 64) return PMG_E_DTYPE;
  return PMG_OK;
}

template <typename T, typename I>
int fwd(const void* W, int64_t ldw, const void* ids, int64_t N, int64_t V, int64_t E, float scale, void* out, hipStream_t st) {
  const int tpr = threads_per_row(E, pmg_vec16<T>::N), rpw = THREADS / tpr;
  const int64_t cols = (E + (int64_t)tpr * pmg_vec16<T>::N - 1) / ((int64_t)tpr * pmg_vec16<T>::N);
  if (cols > 65535) return PMG_E_ARG;
  // four rows a thread once that leaves enough workgroups for the chip
  const int rows = (N / rpw) * cols >= 4 * 1024 ? 4 : 1;
  const int64_t most = MOST_GROUPS * rpw * rows;
  for (int64_t n0 = 0; n0 < N; n0 += most) {
    const int64_t n = N - n0 < most ? N - n0 : most;
    const dim3 grid((unsigned)((n + (int64_t)rpw * rows - 1) / ((int64_t)rpw * rows)), (unsigned)cols);
    const I* id = (const I*)ids + n0;
    T* to = (T*)out + n0 * E;
    if (rows == 4) hipLaunchKernelGGL((embed_fwd_kernel<T, I, 4>), grid, dim3(THREADS), 0, st, (const T*)W, ldw, id, n, V, E, scale, tpr, to);
    else hipLaunchKernelGGL((embed_fwd_kernel<T, I, 1>), grid, dim3(THREADS), 0, st, (const T*)W, ldw, id, n, V, E, scale, tpr, to);
  }
  return (int)hipGetLastError();
}

template <typename Src, int ROUNDS>
void radix_pass_of(const Src& src, int64_t N, int shift, int bits, const BwdLayout& L, char* ws, int to, hipStream_t st) {
  int *count = (int*)(ws + L.count), *total = (int*)(ws + L.total);
  const dim3 grid((unsigned)L.tiles), block(THREADS);
  hipLaunchKernelGGL((embed_count_kernel<Src, ROUNDS>), grid, block, 0, st, src, N, shift, bits, (int)L.tiles, count);
  hipLaunchKernelGGL(embed_scan_kernel, dim3(1u << bits), block, 0, st, count, (int)L.tiles, total);
  hipLaunchKernelGGL((embed_scatter_kernel<Src, ROUNDS>), grid, block, 0, st, src, N, shift, bits, (int)L.tiles, count, total,
                     (uint32_t*)(ws + L.keys[to]), (uint32_t*)(ws + L.pos[to]));
}
template <typename Src>
void radix_pass(const Src& src, int64_t N, int shift, int bits, const BwdLayout& L, char* ws, int to, hipStream_t st) {
  if (L.rounds == 8) radix_pass_of<Src, 8>(src, N, shift, bits, L, ws, to, st);
  else radix_pass_of<Src, 2>(src, N, shift, bits, L, ws, to, st);
}

// Returns which of the two key buffers holds the sorted keys.
template <typename I>
int sort_ids(const I* ids, int64_t N, int64_t V, int64_t pad, const BwdLayout& L, char* ws, hipStream_t st) {
  if (N <= SMALL_N) {
    hipLaunchKernelGGL(embed_sort_small_kernel<I>, dim3(1), dim3(1024), 0, st, ids, (int)N, V, pad,
                       (uint32_t*)(ws + L.keys[0]), (uint32_t*)(ws + L.pos[0]));
    return 0;
  }
  const int all = key_bits(V), passes = (all + MAX_BITS - 1) / MAX_BITS, bits = (all + passes - 1) / passes;
  int to = 0;
  for (int p = 0; p < passes; ++p) {
    to = p & 1;
    if (p == 0) radix_pass(FromIds<I>{ids, V, pad}, N, 0, bits, L, ws, to, st);
    else
      radix_pass(FromKeys{(const uint32_t*)(ws + L.keys[1 - to]), (const uint32_t*)(ws + L.pos[1 - to])}, N, p * bits, bits, L,
                 ws, to, st);
  }
  return to;
}

template <typename T>
int bwd(const void* g, int64_t ldg, const void* ids, int id_bits, int64_t N, int64_t V, int64_t E, float scale, int64_t pad,
        void* dW, char* ws, hipStream_t st) {
  const int dtype = sizeof(T) == 4 ? PMG_F32 : PMG_BF16;
  const BwdLayout L = bwd_layout(N, E, dtype);
  const int tpr = L.tpr;
  const int64_t cols = (E + (int64_t)tpr * pmg_vec16<T>::N - 1) / ((int64_t)tpr * pmg_vec16<T>::N);
  const int rpw = THREADS / tpr;
  const int64_t reduce_blocks = (L.chunks + rpw - 1) / rpw, blocks = reduce_blocks + (V + FILL_ROWS - 1) / FILL_ROWS;
  if (cols > 65535 || blocks >= ((int64_t)1 << 32) / THREADS) return PMG_E_ARG;
  int at = 0;
  if (N > 0) at = id_bits == 64 ? sort_ids((const int64_t*)ids, N, V, pad, L, ws, st) : sort_ids((const int32_t*)ids, N, V, pad, L, ws, st);
  ReduceArgs a;
  a.N = N; a.V = V; a.E = E; a.ldg = ldg; a.scale = scale; a.tpr = tpr; a.chunk = L.chunk; a.chunks = L.chunks;
  a.reduce_blocks = reduce_blocks;
  a.keys = (const uint32_t*)(ws + L.keys[at]);
  a.pos = (const uint32_t*)(ws + L.pos[at]);
  a.part = (float*)(ws + L.part);
  a.join_from = 0;
  const dim3 grid((unsigned)blocks, (unsigned)cols);
  const bool whole = E >= pmg_vec16<T>::N;
  if (whole) hipLaunchKernelGGL((embed_reduce_kernel<T, true>), grid, dim3(THREADS), 0, st, a, (const T*)g, (T*)dW);
  else hipLaunchKernelGGL((embed_reduce_kernel<T, false>), grid, dim3(THREADS), 0, st, a, (const T*)g, (T*)dW);
  for (a.join_from = 0; L.chunks > 1 && a.join_from < L.chunks; a.join_from += MOST_GROUPS) {
    const dim3 joins((unsigned)(L.chunks - a.join_from < MOST_GROUPS ? L.chunks - a.join_from : MOST_GROUPS), (unsigned)cols);
    if (whole) hipLaunchKernelGGL((embed_join_kernel<T, true>), joins, dim3(JOIN_THREADS), 0, st, a, (T*)dW);
    else hipLaunchKernelGGL((embed_join_kernel<T, false>), joins, dim3(JOIN_THREADS), 0, st, a, (T*)dW);
  }
  return (int)hipGetLastError();
}

}  // namespace

extern "C" int pmg_embedding_fwd(const void* weight, int64_t ld_weight, const void* ids, int id_bits, int64_t N, int64_t V,
                                 int64_t E, int dtype, float scale, void* out, pmg_stream stream) {
  const int rc = embed_args_ok(N, V, E, dtype, id_bits);
  if (rc) return rc;
  if (N == 0) return PMG_OK;
  if (!weight || !ids || !out) return PMG_E_NULL;
  if (ld_weight < E) return PMG_E_ARG;
  if ((((uintptr_t)weight | (uintptr_t)out) & (pmg_elem_bytes(dtype) - 1)) || ((uintptr_t)ids & (id_bits / 8 - 1)))
    return PMG_E_ALIGN;
  hipStream_t st = (hipStream_t)stream;
  const bool w = id_bits == 64;
  if (dtype == PMG_F32) return w ? fwd<float, int64_t>(weight, ld_weight, ids, N, V, E, scale, out, st) : fwd<float, int32_t>(weight, ld_weight, ids, N, V, E, scale, out, st);
  if (dtype == PMG_BF16) return w ? fwd<bf16_t, int64_t>(weight, ld_weight, ids, N, V, E, scale, out, st) : fwd<bf16_t, int32_t>(weight, ld_weight, ids, N, V, E, scale, out, st);
  return w ? fwd<f16_t, int64_t>(weight, ld_weight, ids, N, V, E, scale, out, st) : fwd<f16_t, int32_t>(weight, ld_weight, ids, N, V, E, scale, out, st);
}

extern "C" int pmg_embedding_bwd_workspace(int64_t N, int64_t V, int64_t E, int dtype, size_t* out) {
  if (!out) return PMG_E_NULL;
  const int rc = embed_args_ok(N, V, E, dtype, 64);
  if (rc) return rc;
  *out = bwd_layout(N, E, dtype).bytes;
  return PMG_OK;
}

extern "C" int pmg_embedding_bwd(const void* grad, int64_t ld_grad, const void* ids, int id_bits, int64_t N, int64_t V,
                                 int64_t E, int dtype, float scale, int64_t padding_idx, void* grad_weight, void* ws,
                                 pmg_stream stream) {
  const int rc = embed_args_ok(N, V, E, dtype, id_bits);
  if (rc) return rc;
  if (!grad_weight || !ws || (N > 0 && (!grad || !ids))) return PMG_E_NULL;
  if (N > 0 && ld_grad < E) return PMG_E_ARG;
  if (((uintptr_t)ws & 15) || (((uintptr_t)grad | (uintptr_t)grad_weight) & (pmg_elem_bytes(dtype) - 1)) ||
      ((uintptr_t)ids & (id_bits / 8 - 1)))
    return PMG_E_ALIGN;
  hipStream_t st = (hipStream_t)stream;
  char* w = (char*)ws;
  if (dtype == PMG_F32) return bwd<float>(grad, ld_grad, ids, id_bits, N, V, E, scale, padding_idx, grad_weight, w, st);
  if (dtype == PMG_BF16) return bwd<bf16_t>(grad, ld_grad, ids, id_bits, N, V, E, scale, padding_idx, grad_weight, w, st);
  return bwd<f16_t>(grad, ld_grad, ids, id_bits, N, V, E, scale, padding_idx, grad_weight, w, st);
}
