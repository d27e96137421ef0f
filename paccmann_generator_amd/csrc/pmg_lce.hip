// Cross entropy of a linear vocabulary projection, with its gradients (include/pmg_lm.h); the logits are
// not kept, unless the caller gives a place for them.
//
//   l = s (x W^T + b)     lse_n = log sum_v exp l_nv     nll_n = lse_n - l_{n,t_n}
//   dl_nv = a_n exp(l_nv - lse_n) - c_n [v = t_n]    dx = f dl W    dW = f dl^T x    db = f sum_n dl_n
// where f c_n / s is the slope of the loss in nll_n, f a_n / s that plus the slope in lse_n, and f what all rows have
// in common (the logits' scale, and of a reduced loss its slope and the mean's 1 / count).
//
// Forward: the tile product of pmg_gemm.h (m = vocabulary, n = tokens) whose epilogue leaves per token and
// vocabulary tile the largest logit and the sum of exponentials below it, and the target's logit: 8 bytes
// for 256 logits.  A second kernel joins them.  Few tokens (serving) take narrow tiles: W is streamed once.
// Backward: the vocabulary goes in pieces; of each piece the logits are formed again, dl is written in the
// operands' type (bf16: one rounding, relative 2^-8 at most, like the operands themselves; without f, so
// that the targets' -1 and the zeros stay exact and the roundings of the rows are not all the same; weights and slopes
// of single rows stay in, because dx and dW read the same dl, and a target's -c_n is then rounded too; the products sum
// in fp32) and read by the two products for dx and dW.  dx is summed over the pieces in fp32.  Long sums with
// few result tiles are split and joined in a fixed order.  No atomics: equal inputs give equal bits.
// Rows without a slope (ignored targets, zero weights) take no part in the backward: the others are listed, the
// products run over the list, and the rows left out get a zero gradient whatever they hold.
// Bound by the matrix units for many tokens (8 N V H operations, two of them for the second forming of the
// logits), by reading W for few.  With few vocabulary entries kept logits are much shorter than the hidden rows they are
// made of: the backward reads them and forms nothing again (524288 rows of 512 fp32 over 60: 126 MB in place of 1 GB and a
// quarter of the operations).
#include "pmg_gemm.h"

#include <type_traits>

namespace {

constexpr float LOG2E = 1.4426950408889634f;

template <typename T> __device__ __forceinline__ float exp_of(float x);
template <> __device__ __forceinline__ float exp_of<float>(float x) { return expf(x); }
// behind bf16 operands the hardware's 2^x of a rounded product is exact enough: relative 2^-24 |x| log2(e)
template <> __device__ __forceinline__ float exp_of<bf16_t>(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }

// ------------------------------------------------------------------------------------------ tile shapes
// Rows of m and n, waves along m and n, bytes of k a stage, stages, and workgroups that fit a CU.  Measured as plain
// products with fp32 result, bf16 (operands with k / m and k / m contiguous), TFLOP/s: the large square 1152 / 1281 /
// 1303 at 8192 x 8192 x 4096 (4096 x 8192 x 8192), the middle one 1067 / 1029 / 968; with two stages of 128 bytes the
// large one gets 950 / 1007 / 1216, with four waves the middle one 906 / 989 / 929.  fp32: 142, of 157 the units give.
// 64 words by 128 tokens, 524288 x 512 fp32 over 60: 321 us with the waves along the tokens, 340 in a square, 328 with 256
// tokens; weights' gradient there 336 in a square, 318 with 256 of m, which costs bf16 2 %, 408 with two waves.
struct Shape {
  int BM, BN, WM, WN, KB, stages, per_cu;
};
enum { S256, S128, S64, SN64, SM64, SK16W, SK16, SK32, SK64, SD64 };  // S: square, SN / SM / SD: 64 of n or m, SK: few tokens
constexpr Shape SHAPES[] = {{256, 256, 2, 4, 64, 3, 1}, {128, 128, 2, 4, 128, 2, 2}, {64, 64, 2, 2, 128, 2, 5},
                            {128, 64, 2, 2, 128, 2, 3}, {64, 128, 1, 4, 128, 2, 3},  {128, 16, 2, 1, 128, 2, 4},
                            {64, 16, 2, 1, 128, 2, 8},  {128, 32, 2, 1, 128, 2, 4},  {128, 64, 2, 1, 128, 2, 3},
                            {128, 64, 2, 2, 64, 2, 6}};
template <typename T, int S, bool AKC, bool BKC, bool ALIST, bool BLIST>
using TileOf = pmg_tile<T, SHAPES[S].BM, SHAPES[S].BN, SHAPES[S].WM, SHAPES[S].WN, AKC, BKC, ALIST, BLIST, SHAPES[S].KB,
                        SHAPES[S].stages>;
template <int S> constexpr int THREADS_OF = SHAPES[S].WM * SHAPES[S].WN * 64;
constexpr int LIST_SLACK = 256;  // entries behind the list of rows that a tile may read (and not use)

// a value in memory that is the same for the whole launch, into a scalar register
__device__ __forceinline__ int uniform_of(const int* p) { return *(const __attribute__((address_space(4))) int*)p; }

// Sums of exponentials are held below a maximum, (top, sum).  A top of -inf (nothing, or NaN) or +inf has no difference to
// itself: such a sum is held below 0, and one whose maximum stays is not rescaled.  A NaN logit is in no maximum and stays
// in the sum; below -inf the sum is 0 or NaN.
__device__ __forceinline__ float below(float top) { return fabsf(top) == __builtin_inff() ? 0.0f : top; }
template <typename T> __device__ __forceinline__ float rescaled(float2 p, float top) {
  return p.x == top ? p.y : p.y * exp_of<T>(p.x - top);
}

// ------------------------------------------------------------------------------------------ arguments
struct LogitArgs {
  const void *W, *X, *bias;
  int64_t ldw, ldx;
  int64_t V, N, K;       // vocabulary rows of this piece, tokens, hidden size
  int64_t v0;            // first vocabulary entry of the piece
  int tiles_m, tiles_n;
  float scale;
  const void* targets;
  int id_bits;
  float* kept;           // logits of all tokens, rows of ldk (a multiple of 4); forward: written, backward: read; or null
  int64_t ldk;
  // forward
  float2* part;          // [tiles_m][N]; or, where the hidden size is split,
  int splits;
  float* sums;           // [splits][N][ldk] products, and nothing else
  float* at_target;      // [N]
  // backward: over the listed rows
  const struct Row* row; // [count]
  const int* list;       // [count] their places in X
  const int* count;
  const float* factor;   // f
  void* dl;              // [count][ldl], columns V .. ldl zero
  int64_t ldl;
  float* dbias;          // [tiles_n][ldl] or null
};

__device__ __forceinline__ int64_t target_of(const void* t, int bits, int64_t n) {
  return bits == 64 ? ((const int64_t*)t)[n] : (int64_t)((const int32_t*)t)[n];
}

// A row that takes part in the backward
struct Row {
  float lse, a, c;       // a_n, c_n
  int target;            // -1: outside the vocabulary
};

// ------------------------------------------------------------------------------------------ logits
// Forward: whole, or a part of the hidden size; backward: forms the logits again, or reads those that were kept
enum { FORWARD, SPLIT, REFORM, KEPT };

template <typename T, int S, int WAY>
__global__ __launch_bounds__(THREADS_OF<S>) void lce_logits_kernel(const LogitArgs a) {
  constexpr bool BACKWARD = WAY == REFORM || WAY == KEPT;
  typedef TileOf<T, S, true, true, false, BACKWARD> Tile;
  constexpr int BM = SHAPES[S].BM, BN = SHAPES[S].BN, WM = SHAPES[S].WM, WN = SHAPES[S].WN;
  constexpr int MI = Tile::MI, NI = Tile::NI;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  int tm, tn;
  pmg_tile_of(blockIdx.x, a.tiles_m, a.tiles_n, &tm, &tn);
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
  const int64_t N = BACKWARD ? uniform_of(a.count) : a.N;
  if (BACKWARD && n0 >= N) return;
  int64_t k0 = 0, k1 = a.K;
  if constexpr (WAY == SPLIT) {
    const int64_t per = ((a.K + Tile::KSTEP - 1) / Tile::KSTEP + a.splits - 1) / a.splits * Tile::KSTEP;
    k0 = per * blockIdx.y;
    k1 = k0 + per < a.K ? k0 + per : a.K;
  }
  f32x4 acc[MI][NI];
  if constexpr (WAY != KEPT)
    Tile::run(acc, (lds_char*)smem, a.W, a.ldw, nullptr, m0, a.V, a.X, a.ldx, a.list, n0, N, k0, k1);

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;
  const int g = lane >> 4, col = lane & 15;
  const int64_t mw = m0 + wm * (BM / WM);               // this lane's rows: mw + row_of(i) + e
  const int rows = a.V - mw < BM ? (int)(a.V - mw) : BM;  // of them in the vocabulary (may be none)
  const T* bias = (const T*)a.bias;
  if constexpr (WAY == SPLIT) {
    float* sums = a.sums + (int64_t)blockIdx.y * a.N * a.ldk + mw;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int64_t n = n0 + wn * (BN / WN) + j * 16 + col;
#pragma unroll
      for (int i = 0; i < MI; ++i)
        if (n < N && Tile::row_of(i) < rows) *(f32x4*)(sums + n * a.ldk + Tile::row_of(i)) = acc[i][j];
    }
  } else if constexpr (WAY == KEPT) {
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int64_t n = n0 + wn * (BN / WN) + j * 16 + col;
      const float* from = a.kept + (n < N ? (int64_t)a.list[n] : 0) * a.ldk + a.v0 + mw;
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (n < N && Tile::row_of(i) < rows) acc[i][j] = *(const f32x4*)(from + Tile::row_of(i));
      }
    }
  } else {
    // logits; entries behind the vocabulary's end do not take part
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      f32x4 b = {0.f, 0.f, 0.f, 0.f};
      if (bias) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (Tile::row_of(i) + e < rows) b[e] = (float)bias[mw + Tile::row_of(i) + e];
      }
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc[i][j][e] = Tile::row_of(i) + e < rows ? (acc[i][j][e] + b[e]) * a.scale : -__builtin_inff();
    }
  }

  if constexpr (WAY == FORWARD) {
    if (a.kept) {
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const int64_t n = n0 + wn * (BN / WN) + j * 16 + col;
        float* to = a.kept + n * a.ldk + mw;
#pragma unroll
        for (int i = 0; i < MI; ++i)
          if (n < a.N && Tile::row_of(i) < rows) *(f32x4*)(to + Tile::row_of(i)) = acc[i][j];
      }
    }
    float2* red = (float2*)smem;  // [WM][BN]
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int64_t n = n0 + wn * (BN / WN) + j * 16 + col;
      float top = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, acc[i][j][e]);
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float base = below(top);
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += exp_of<T>(acc[i][j][e] - base);
      sum += __shfl_xor(sum, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
      if (g == 0) red[wm * BN + wn * (BN / WN) + j * 16 + col] = make_float2(top, sum);
      if (n < a.N) {
        const int64_t t = target_of(a.targets, a.id_bits, n) - a.v0 - mw;
        if (t >= 0 && t < rows) {
#pragma unroll
          for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (Tile::row_of(i) + e == (int)t) a.at_target[n] = acc[i][j][e];
        }
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < BN; c += Tile::THREADS) {
      float top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
      for (int w = 0; w < WM; ++w) top = fmaxf(top, red[w * BN + c].x);
#pragma unroll
      for (int w = 0; w < WM; ++w) sum += rescaled<T>(red[w * BN + c], top);
      if (n0 + c < a.N) a.part[(int64_t)tm * a.N + n0 + c] = make_float2(top, sum);
    }
  } else if constexpr (BACKWARD) {
    T* dl = (T*)a.dl;
    const int wide = a.ldl - mw < BM ? (int)(a.ldl - mw) : BM;  // ldl is a multiple of 64
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int64_t n = n0 + wn * (BN / WN) + j * 16 + col;
      Row r = {0.0f, 0.0f, 0.0f, -1};
      if (n < N) r = a.row[n];
      const int64_t behind = (int64_t)r.target - a.v0 - mw;
      const int t = behind >= 0 && behind < rows ? (int)behind : -1;
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // entries behind the vocabulary's end and rows behind the last are zero
          float x = n < N && Tile::row_of(i) + e < rows ? r.a * exp_of<T>(acc[i][j][e] - r.lse) : 0.0f;
          if (Tile::row_of(i) + e == t) x -= r.c;
          acc[i][j][e] = x;
        }
      if (n < N) {
        T* to = dl + n * a.ldl + mw;
#pragma unroll
        for (int i = 0; i < MI; i += 2) {
          if constexpr (Tile::PAIR) {
            const bool up = Tile::swapped();
            if (Tile::pair_of(i) < wide) pmg_store8(to + Tile::pair_of(i), up ? acc[i + 1][j] : acc[i][j], up ? acc[i][j] : acc[i + 1][j], 8);
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (Tile::row_of(i + h) < wide) pmg_store4(to + Tile::row_of(i + h), acc[i + h][j]);
          }
        }
      }
    }
    if (a.dbias) {
      float* red = (float*)smem;  // [WN][BM]
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float s = 0.0f;
#pragma unroll
          for (int j = 0; j < NI; ++j) s += acc[i][j][e];
          s += __shfl_xor(s, 1, 64);
          s += __shfl_xor(s, 2, 64);
          s += __shfl_xor(s, 4, 64);
          s += __shfl_xor(s, 8, 64);
          if (col == 0) red[wn * BM + wm * (BM / WM) + Tile::row_of(i) + e] = s;
        }
      __syncthreads();
      for (int r = threadIdx.x; r < BM; r += Tile::THREADS) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < WN; ++w) s += red[w * BM + r];
        if (m0 + r < a.ldl) a.dbias[(int64_t)tn * a.ldl + m0 + r] = s * a.factor[0];
      }
    }
  }
}

// ------------------------------------------------------------------------------------------ gradients
// out[n][m] (m contiguous) = sum_k A(m,k) B(n,k), A with m contiguous: dx (A = W, B = dl) and dW (A = x, B = dl).
struct GradArgs {
  const void *A, *B;
  int64_t lda, ldb;
  int64_t M, N, K;
  const int* list;       // of the rows that the backward takes, and their number:
  const int* count;      // dx: row n of the result is row list[n] of out, N = count; dW: rows k of A, K = count
  const float* factor;   // f
  int tiles_m, tiles_n, splits;
  void* out;             // of T, row stride ldo; or null: the fp32 sums go to acc
  int64_t ldo;
  float* acc;            // fp32 [splits][N][M], where the sums go (splits > 1) or are added up over pieces
  int add;               // add what acc holds
  const uint8_t* used;   // dx: which rows of the batch have a slope;
  void* zeroed;          // the others become zero here (null: not in this launch)
};

// Zero columns c0 .. H of rows of dx for 64 rows of the batch that have no slope; a wave takes one row after the other in turn.
template <typename T>
__device__ __forceinline__ void zero_rows(const uint8_t* __restrict__ used, int64_t n0, int64_t N, int64_t c0, int64_t H,
                                          int64_t ldo, T* __restrict__ dx) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  uint64_t left = __ballot(n0 + lane < N && !used[n0 + lane]);
  for (int k = 0; left; ++k, left &= left - 1) {
    if (k % waves != wave) continue;
    T* row = dx + (n0 + __ffsll((unsigned long long)left) - 1) * ldo;
    for (int64_t c = c0 + lane * 4; c < H; c += 256) pmg_store4(row + c, f32x4{0.f, 0.f, 0.f, 0.f}, H - c);
  }
}

template <typename T, int S, bool BKC>
__global__ __launch_bounds__(THREADS_OF<S>) void lce_grad_kernel(const GradArgs a) {
  typedef TileOf<T, S, false, BKC, !BKC, false> Tile;
  constexpr int BM = SHAPES[S].BM, BN = SHAPES[S].BN, WM = SHAPES[S].WM, WN = SHAPES[S].WN;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  if (BKC && (int64_t)blockIdx.x >= (int64_t)a.tiles_m * a.tiles_n) {  // behind the tiles
    if (blockIdx.y == 0) zero_rows(a.used, ((int64_t)blockIdx.x - (int64_t)a.tiles_m * a.tiles_n) * 64, a.N, 0, a.M, a.ldo, (T*)a.zeroed);
    return;
  }
  int tm, tn;
  pmg_tile_of(blockIdx.x, a.tiles_m, a.tiles_n, &tm, &tn);
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
  const int64_t rows = uniform_of(a.count), N = BKC ? rows : a.N, K = BKC ? a.K : rows;
  if (n0 >= N) return;
  const int64_t steps = (K + Tile::KSTEP - 1) / Tile::KSTEP, per = (steps + a.splits - 1) / a.splits * Tile::KSTEP;
  const int64_t k0 = per * blockIdx.y, k1 = k0 + per < K ? k0 + per : K;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t mw = m0 + (wave / WN) * (BM / WM), nw = n0 + (wave % WN) * (BN / WN) + (lane & 15);
  int place[Tile::NI];  // of this lane's rows of the result
  if (BKC) {
#pragma unroll
    for (int j = 0; j < Tile::NI; ++j) place[j] = nw + j * 16 < N ? a.list[nw + j * 16] : 0;
  }
  f32x4 acc[Tile::MI][Tile::NI];
  Tile::run(acc, (lds_char*)smem, a.A, a.lda, a.list, m0, a.M, a.B, a.ldb, nullptr, n0, N, k0, k1);
  const float f = a.factor[0];
  float* sums = a.acc ? a.acc + (int64_t)blockIdx.y * a.N * a.M : nullptr;
#pragma unroll
  for (int j = 0; j < Tile::NI; ++j) {
    const int64_t n = nw + j * 16;
    if (n >= N) continue;
    const int64_t o = BKC ? place[j] : n;
#pragma unroll
    for (int i = 0; i < Tile::MI; i += 2) {
      f32x4 x[2] = {acc[i][j] * f, acc[i + 1][j] * f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t m = mw + Tile::row_of(i + h), left = a.M - m;
        if (left <= 0) continue;
        float* s = sums + n * a.M + m;
        if (a.add) x[h] += pmg_load4(s, left);
        if (!a.out) pmg_store4(s, x[h], left);
        else if (!Tile::PAIR && S == SD64) pmg_store4_nt((T*)a.out + o * a.ldo + m, x[h], left);
        else if (!Tile::PAIR) pmg_store4((T*)a.out + o * a.ldo + m, x[h], left);
      }
      const int64_t m = mw + Tile::pair_of(i);
      const bool up = Tile::swapped();
      if (Tile::PAIR && a.out && m < a.M) pmg_store8((T*)a.out + o * a.ldo + m, up ? x[1] : x[0], up ? x[0] : x[1], a.M - m);
    }
  }
}

// dx over at most 64 vocabulary entries, bound by writing dx (fp32: and by the matrix units, 64 columns of k a token).  A
// wave keeps its 256 bytes of columns of W in registers, in the fragments' layout, and streams over tokens: the workgroup
// fetches the slopes of 64 tokens ahead, in whole rows, and passes them through LDS (16-byte pieces of a row permuted, so
// that the rows of a fragment lie in different banks).  Tokens are the products' m and columns their n, lane l & 15 of
// fragment i has column MI (l & 15) + i: a lane's results of a token are neighbours, and those of 16 lanes are 256 bytes in
// a row.  524288 x 512 fp32 over 60: 316 us (3.4 TB/s written, 109 Tflop/s); 185763 x 2944 bf16 over 17, half of the rows
// zero: 208 us (5.3 TB/s).  With the short sums' tiles 370 us and 370 us; with fragments read straight from memory, where
// neighbouring lanes read different rows, 452 and 234, and with products whose lanes are tokens, so that neighbouring lanes
// write different rows, 536 and 295.
constexpr int NARROW = 64, NARROW_TOKENS = 64, NARROW_PER_CU = 3;  // vocabulary entries, tokens at a time, workgroups a CU
template <typename T>
__global__ __launch_bounds__(256, NARROW_PER_CU) void lce_dx_narrow_kernel(const GradArgs a) {
  constexpr int E = 16 / sizeof(T), KK = NARROW / (4 * E), MI = E, COLS = MI * 16;
  constexpr int PIECES = NARROW / E, FETCH = NARROW_TOKENS * PIECES / 256;
  typedef typename pmg_frag<T>::type frag;
  __shared__ __attribute__((aligned(16))) frag slopes[2][NARROW_TOKENS * PIECES];
  __shared__ __attribute__((aligned(16))) unsigned places[2][NARROW_TOKENS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, i16 = lane & 15;
  const int64_t m0 = ((int64_t)blockIdx.y * 4 + wave) * COLS;
  const int N = uniform_of(a.count), step = gridDim.x * NARROW_TOKENS;
  if (N < a.N) {
    const int64_t c0 = (int64_t)blockIdx.y * 4 * COLS, c1 = c0 + 4 * COLS < a.M ? c0 + 4 * COLS : a.M;
    for (int64_t n0 = (int64_t)blockIdx.x * 64; n0 < a.N; n0 += (int64_t)gridDim.x * 64)
      zero_rows(a.used, n0, a.N, c0, c1, a.ldo, (T*)a.zeroed);
  }
  int t = blockIdx.x * NARROW_TOKENS;
  if (t >= N) return;
  const int64_t m = m0 + MI * i16, left = a.M - m;  // this lane's columns (may be none)
  frag w[MI][KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk)
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int k = kk * 4 * E + g * E + j;
      typename pmg_vec16<T>::vec x = {};
      if (k < a.K && left > 0) x = pmg_vec16<T>::load((const T*)a.A + k * a.lda + m, left);
#pragma unroll
      for (int i = 0; i < MI; ++i) w[i][kk][j] = x[i];
    }
  const float f = a.factor[0];
  frag next[FETCH];
  unsigned next_place;
  const auto fetch = [&](int at) {  // rows behind the last: the last one
    next_place = a.list[at + (threadIdx.x & 63)];
#pragma unroll
    for (int q = 0; q < FETCH; ++q) {
      const int piece = q * 256 + threadIdx.x, r = piece / PIECES, n = at + r < N ? at + r : N - 1;
      next[q] = *(const frag*)((const T*)a.B + (int64_t)n * a.ldb + piece % PIECES * E);
    }
  };
  const auto put = [&](int buf) {
    if (threadIdx.x < NARROW_TOKENS) places[buf][threadIdx.x] = next_place;
#pragma unroll
    for (int q = 0; q < FETCH; ++q) {
      const int piece = q * 256 + threadIdx.x, r = piece / PIECES;
      slopes[buf][r * PIECES + ((piece ^ r) & (PIECES - 1))] = next[q];
    }
  };
  // `whole`: all tokens and columns; without branches around the stores the compiler waits for the fetch alone, not for them
  const auto multiply = [&](int at, int buf, auto whole) {
#pragma unroll 1  // (more turns at a time take more registers than three workgroups a CU have)
    for (int q = 0; q < NARROW_TOKENS / 16; ++q) {
      const int r = q * 16 + i16;
      frag b[KK];
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) b[kk] = slopes[buf][r * PIECES + (((kk * 4 + g) ^ r) & (PIECES - 1))];
      f32x4 acc[MI];
#pragma unroll
      for (int i = 0; i < MI; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int i = 0; i < MI; ++i) acc[i] = pmg_frag<T>::mma(b[kk], w[i][kk], acc[i]);
        } else {
#pragma unroll
          for (int j = 0; j < E; ++j)
#pragma unroll
            for (int i = 0; i < MI; ++i) acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(b[kk][j], w[i][kk][j], acc[i], 0, 0, 0);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = q * 16 + 4 * g + e;
        T* out = (T*)a.out + (uint64_t)places[buf][row] * (uint64_t)a.ldo + m;
        f32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = acc[i][e] * f;
        if (!whole && (at + row >= N || left <= 0)) continue;
        if constexpr (MI == 8) {
          f32x4 y;
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = acc[4 + i][e] * f;
          pmg_store8(out, x, y, whole ? 8 : left);
        } else {
          pmg_store4(out, x, whole ? 4 : left);
        }
      }
    }
  };
  fetch(t);
  put(0);
  __syncthreads();
  for (int buf = 0;; buf ^= 1) {
    const bool last = t >= N - step;
    fetch(last ? t : t + step);
    __builtin_amdgcn_sched_barrier(0);  // ahead of the products, not behind
    if (m0 + COLS <= a.M && t + NARROW_TOKENS <= N) multiply(t, buf, std::true_type());
    else multiply(t, buf, std::false_type());
    if (last) break;
    put(buf ^ 1);
    __syncthreads();
    t += step;
  }
}

// out row r (list[r] with a list) = sum over the splits of acc[split][r], in order
template <typename T>
__global__ __launch_bounds__(256) void lce_join_kernel(const float* __restrict__ acc, int splits, int64_t rows, int64_t M,
                                                       const int* list, const int* count, T* __restrict__ out, int64_t ldo) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, total = rows * M;
  const int64_t r = i / M;
  if (i >= total || (list && r >= count[0])) return;
  float s = 0.0f;
#pragma unroll 8
  for (int k = 0; k < splits; ++k) s += acc[(int64_t)k * total + i];
  out[(list ? list[r] : r) * ldo + (i - r * M)] = (T)s;
}

// db[v] = sum over the tiles of BN tokens; 64 entries by 16 groups that take the tiles in turn, joined in order
template <typename T>
__global__ __launch_bounds__(1024) void lce_dbias_kernel(const float* __restrict__ part, int BN, const int* count, int64_t ldl,
                                                         int64_t V, T* __restrict__ db) {
  __shared__ float red[16][64];
  const int c = threadIdx.x & 63, grp = threadIdx.x >> 6, tiles = (uniform_of(count) + BN - 1) / BN;
  const int64_t v = (int64_t)blockIdx.x * 64 + c;
  float s = 0.0f;
  if (v < V) {
#pragma unroll 8
    for (int k = grp; k < tiles; k += 16) s += part[(int64_t)k * ldl + v];
  }
  red[grp][c] = s;
  __syncthreads();
  if (grp == 0 && v < V) {
    s = 0.0f;
#pragma unroll
    for (int g = 0; g < 16; ++g) s += red[g][c];
    db[v] = (T)s;
  }
}

// ------------------------------------------------------------------------------------------ rows
// A workgroup's 1024 threads are `r` rows by 1024 / r groups; a group joins every (1024 / r)-th part of its row.
struct RowArgs {
  const float2* part;
  const float* at_target;
  int tiles;
  int64_t N, V;
  const void* targets;
  int id_bits;
  int64_t ignore;
  const float* weight;   // [N] or null
  float* lse;
  float* nll;            // [N], weighted; null: not wanted
  struct LossPart* sums; // [workgroups] or null
  int rows;
  int mean;
  float *loss, *count;   // one workgroup: the reduced loss at once
};

struct LossPart {
  double sum;
  int64_t count;
};

// Sum over a workgroup of 1024; valid in thread 0.
__device__ __forceinline__ LossPart block_sum(double s, int64_t c) {
  __shared__ double ws[16];
  __shared__ long long wc[16];
  long long k = c;
  for (int o = 32; o > 0; o >>= 1) {
    s += __shfl_xor(s, o, 64);
    k += __shfl_xor(k, o, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    ws[threadIdx.x >> 6] = s;
    wc[threadIdx.x >> 6] = k;
  }
  __syncthreads();
  LossPart p = {0.0, 0};
  if (threadIdx.x == 0)
    for (int w = 0; w < 16; ++w) {
      p.sum += ws[w];
      p.count += wc[w];
    }
  return p;
}

__device__ __forceinline__ void reduced_loss(const LossPart& p, int mean, float* loss, float* count) {
  loss[0] = (float)(mean ? (p.count > 0 ? p.sum / (double)p.count : 0.0) : p.sum);
  count[0] = (float)p.count;
}

__global__ __launch_bounds__(1024) void lce_rows_kernel(const RowArgs a) {
  __shared__ float2 red[1024];
  const int r = threadIdx.x % a.rows, grp = threadIdx.x / a.rows, groups = 1024 / a.rows;
  const int64_t n = (int64_t)blockIdx.x * a.rows + r;
  float top = -__builtin_inff(), sum = 0.0f;
  if (n < a.N) {
#pragma unroll 4
    for (int t = grp; t < a.tiles; t += groups) {
      const float2 p = a.part[(int64_t)t * a.N + n];
      const float m = fmaxf(top, p.x);
      sum = rescaled<float>(make_float2(top, sum), m) + rescaled<float>(p, m);
      top = m;
    }
  }
  red[threadIdx.x] = make_float2(top, sum);
  for (int half = groups >> 1; half > 0; half >>= 1) {
    __syncthreads();
    if (grp < half) {
      const float2 p = red[threadIdx.x], q = red[threadIdx.x + half * a.rows];
      const float m = fmaxf(p.x, q.x);
      red[threadIdx.x] = make_float2(m, rescaled<float>(p, m) + rescaled<float>(q, m));
    }
  }
  float nll = 0.0f;
  bool in = false;
  if (grp == 0 && n < a.N) {
    const float2 p = red[threadIdx.x];
    const float lse = p.x + logf(p.y);
    a.lse[n] = lse;
    const int64_t t = target_of(a.targets, a.id_bits, n);
    in = t != a.ignore;
    if (in) nll = t >= 0 && t < a.V ? (lse - a.at_target[n]) * (a.weight ? a.weight[n] : 1.0f) : __builtin_nanf("");
    if (a.nll) a.nll[n] = nll;
  }
  if (a.sums) {
    const LossPart p = block_sum((double)nll, in);
    if (threadIdx.x == 0) {
      if (a.loss) reduced_loss(p, a.mean, a.loss, a.count);
      else a.sums[blockIdx.x] = p;
    }
  }
}

// The same from products split over the hidden size: a row's 1024 / rows threads (whole waves) add up the parts in order,
// four entries a thread, with the running maximum and sum of the exponentials.
struct SplitArgs {
  const float* sums;     // [splits][N][ldk]
  int splits;
  int64_t ldk;
  const void* bias;
  float scale;
  float* kept;           // [N][ldk] or null
};

template <typename T> __global__ __launch_bounds__(1024) void lce_split_rows_kernel(const SplitArgs b, const RowArgs a) {
  __shared__ float2 red[16];
  __shared__ float hit[16];
  const int per = 1024 / a.rows, i = threadIdx.x % per, row = threadIdx.x / per, wave = threadIdx.x >> 6;
  const int64_t n = (int64_t)blockIdx.x * a.rows + row;
  const bool here = n < a.N;
  const int64_t t = here ? target_of(a.targets, a.id_bits, n) : -1;
  if (i == 0) hit[row] = 0.0f;
  __syncthreads();
  float top = -__builtin_inff(), sum = 0.0f;
  for (int64_t v = i * 4; here && v < a.V; v += per * 4) {
    f32x4 x = {0.f, 0.f, 0.f, 0.f}, bias = x;
    if (b.bias) bias = pmg_load4((const T*)b.bias + v, a.V - v);
    const float* from = b.sums + n * b.ldk + v;
    for (int k = 0; k < b.splits; k += 8) {  // eight loads under way, added in order
      f32x4 y[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) y[u] = *(const f32x4*)(from + (int64_t)(k + u < b.splits ? k + u : 0) * a.N * b.ldk);
#pragma unroll
      for (int u = 0; u < 8; ++u) x += k + u < b.splits ? y[u] : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    float most = -__builtin_inff();
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = v + e < a.V ? (x[e] + bias[e]) * b.scale : -__builtin_inff();
      most = fmaxf(most, x[e]);
      if (v + e == t) hit[row] = x[e];
    }
    if (b.kept) *(f32x4*)(b.kept + n * b.ldk + v) = x;
    const float m = fmaxf(top, most), base = below(m);
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) s += expf(x[e] - base);
    sum = rescaled<float>(make_float2(top, sum), m) + s;
    top = m;
  }
  const auto join = [](float2 p, float2 q) {
    const float m = fmaxf(p.x, q.x);
    return make_float2(m, rescaled<float>(p, m) + rescaled<float>(q, m));
  };
  float2 p = make_float2(top, sum);
  for (int o = 32; o > 0; o >>= 1) p = join(p, make_float2(__shfl_xor(p.x, o, 64), __shfl_xor(p.y, o, 64)));
  if ((threadIdx.x & 63) == 0) red[wave] = p;
  __syncthreads();
  float nll = 0.0f;
  bool in = false;
  if (i == 0 && here) {
    for (int w = 1; w < per / 64; ++w) p = join(p, red[wave + w]);
    const float lse = p.x + logf(p.y);
    a.lse[n] = lse;
    in = t != a.ignore;
    if (in) nll = t >= 0 && t < a.V ? (lse - hit[row]) * (a.weight ? a.weight[n] : 1.0f) : __builtin_nanf("");
    if (a.nll) a.nll[n] = nll;
  }
  if (a.sums) {
    const LossPart q = block_sum((double)nll, in);
    if (threadIdx.x == 0) {
      if (a.loss) reduced_loss(q, a.mean, a.loss, a.count);
      else a.sums[blockIdx.x] = q;
    }
  }
}

// count[0] = rows with a target; loss[0] = sum of nll (mean: over those rows; 0 without any).  One workgroup
// over the workgroups of the rows, sums in fp64, in one order.
__global__ __launch_bounds__(1024) void lce_loss_kernel(const LossPart* __restrict__ sums, int n, int mean,
                                                        float* __restrict__ loss, float* __restrict__ count) {
  double s = 0.0;
  int64_t c = 0;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += 1024) {
    s += sums[i].sum;
    c += sums[i].count;
  }
  const LossPart p = block_sum(s, c);
  if (threadIdx.x == 0) reduced_loss(p, mean, loss, count);
}

// The rows with a slope, in their order.  Up to 16 groups of 1024 rows count the rows before theirs by themselves; of
// more groups the counts (WRITE false) are scanned between two launches.
constexpr int OWN_GROUPS = 16;
struct SlopeArgs {
  const float *g_loss, *g_lse, *lse, *count, *weight;
  int per_row, mean;
  const void* targets;
  int id_bits;
  int64_t ignore, N, V;
  int* first;            // [groups]: rows with a slope in a group, then before it
  int groups;
  Row* row;
  int* list;
  int* total;
  float scale;           // of the logits
  float* factor;         // f
  uint8_t* used;         // [N]
};

// What all rows have in common, without the logits' scale; 1 where that is 0 or not finite, and where it is so far from 1 that
// slopes of the log-sum-exps, which are divided by it, could leave fp32 (a loss of weight 1e-38 beside them, say).
__device__ __forceinline__ float common_of(const SlopeArgs& a) {
  if (a.per_row || !a.g_loss) return 1.0f;
  const float g = a.mean ? a.g_loss[0] / a.count[0] : a.g_loss[0];
  if (a.g_lse && !(fabsf(g) >= 0x1p-60f && fabsf(g) <= 0x1p60f)) return 1.0f;
  return g != 0.0f && fabsf(g) < __builtin_inff() ? g : 1.0f;
}

__device__ __forceinline__ Row slope_of(const SlopeArgs& a, int64_t n, float common) {
  Row r = {0.0f, 0.0f, 0.0f, -1};
  const int64_t t = target_of(a.targets, a.id_bits, n);
  if (t != a.ignore && a.g_loss) {
    r.c = a.weight ? a.weight[n] : 1.0f;
    if (a.per_row) r.c *= a.g_loss[n];
    else if (common == 1.0f) r.c *= a.mean ? a.g_loss[0] / a.count[0] : a.g_loss[0];
    if (t >= 0 && t < a.V) r.target = (int)t;
    else r.c = __builtin_nanf("");
  }
  r.a = r.c + (a.g_lse ? a.g_lse[n] / common : 0.0f);
  return r;
}

template <bool WRITE> __global__ __launch_bounds__(1024) void lce_slopes_kernel(const SlopeArgs a) {
  __shared__ int wsum[16];
  const int64_t n = (int64_t)blockIdx.x * 1024 + threadIdx.x;
  Row r = {0.0f, 0.0f, 0.0f, -1};
  const float common = common_of(a);
  if (n < a.N) r = slope_of(a, n, common);
  const bool used = r.a != 0.0f || r.c != 0.0f;
  const uint64_t mask = __ballot(used);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (lane == 0) wsum[wave] = __popcll(mask);
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < 16; ++w) {
    if (w < wave) before += wsum[w];
    all += wsum[w];
  }
  if (!WRITE) {
    if (threadIdx.x == 0) a.first[blockIdx.x] = all;
    return;
  }
  int base = a.groups > OWN_GROUPS ? a.first[blockIdx.x] : 0;
  if (a.groups <= OWN_GROUPS && blockIdx.x > 0) {
    int mine = 0;
#pragma unroll 4
    for (int g = 0; g < (int)blockIdx.x; ++g) {
      const Row q = slope_of(a, (int64_t)g * 1024 + threadIdx.x, common);
      mine += q.a != 0.0f || q.c != 0.0f;
    }
    for (int o = 32; o > 0; o >>= 1) mine += __shfl_xor(mine, o, 64);
    __shared__ int earlier[16];
    if (lane == 0) earlier[wave] = mine;
    __syncthreads();
    for (int w = 0; w < 16; ++w) base += earlier[w];
  }
  if (n < a.N) a.used[n] = used;
  if (used) {
    const int at = base + before + __popcll(mask & ((1ull << lane) - 1));
    r.lse = a.lse[n];
    a.row[at] = r;
    a.list[at] = (int)n;
  }
  if (threadIdx.x == 0 && blockIdx.x == (unsigned)a.groups - 1) {
    a.total[0] = base + all;
    a.factor[0] = common * a.scale;
  }
}

__global__ __launch_bounds__(1024) void lce_scan_kernel(int* __restrict__ first, int n) {
  __shared__ int wsum[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int carry = 0;
  for (int base = 0; base < n; base += 1024) {
    const int i = base + threadIdx.x, v = i < n ? first[i] : 0;
    int inc = v;
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(inc, o, 64);
      if (lane >= o) inc += u;
    }
    if (lane == 63) wsum[wave] = inc;
    __syncthreads();
    int before = carry;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) before += wsum[w];
      carry += wsum[w];
    }
    if (i < n) first[i] = before + inc - v;
    __syncthreads();
  }
}

// rows of `width` elements, `ld` apart, into rows of `wide` (a multiple of 16 bytes), zero behind the end; tpr threads (a
// power of two) a row, 16 bytes each at a time.  Bound by memory: 78869 x 1930 bf16, 610 MB, 107 us.
template <typename T>
__global__ __launch_bounds__(256) void lce_pack_kernel(const T* __restrict__ src, int64_t ld, int64_t rows, int64_t width,
                                                       T* __restrict__ dst, int64_t wide, int tpr) {
  typedef pmg_vec16<T> V;
  const int per = 256 / tpr;
  for (int64_t r = (int64_t)blockIdx.x * per + threadIdx.x / tpr; r < rows; r += (int64_t)gridDim.x * per)
#pragma unroll 4
    for (int64_t c = (threadIdx.x & (tpr - 1)) * V::N; c < wide; c += tpr * V::N)
      *(typename V::vec*)(dst + r * wide + c) = V::load(src + r * ld + c, width - c);
}

// ------------------------------------------------------------------------------------------ host
int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
int64_t div_up(int64_t x, int64_t by) { return (x + by - 1) / by; }

constexpr int CUS = 256;

int64_t tiles_of(int s, int64_t M, int64_t N) { return div_up(M, SHAPES[s].BM) * div_up(N, SHAPES[s].BN); }

// Whether one launch covers the tiles and `more` workgroups: of 2^32 threads or more only some run, without an error.
bool covers(int s, int64_t M, int64_t N, int64_t more = 0) {
  return (tiles_of(s, M, N) + more) * SHAPES[s].WM * SHAPES[s].WN * 64 < (int64_t)1 << 32;
}

// Parts of a long sum where there are too few tiles for the chip; at least eight stages a part.
int splits_of(int s, int64_t M, int64_t N, int64_t K, int64_t eb) {
  const int64_t tiles = tiles_of(s, M, N), slots = (int64_t)CUS * SHAPES[s].per_cu;
  if (tiles * 2 > slots) return 1;
  const int64_t want = slots / tiles, most = div_up(K * eb, (int64_t)SHAPES[s].KB * 8);
  return (int)(want < 1 || most < 1 ? 1 : want < most ? (want < 1024 ? want : 1024) : (most < 1024 ? most : 1024));
}

// Microseconds that a product of this shape takes, roughly: rounds of per_cu tiles on every CU, each as long as its
// products at the rate the shape reaches on a full chip (a CU: 4.6 Tflop/s in bf16, 0.55 in fp32; the middle square 0.85
// of it, the small one 0.6) and a start of 3 us; one tile a CU does not write its result under another's products;
// split sums are written and read once more.
double cost_of(int s, int64_t M, int64_t N, int64_t K, int64_t eb, bool split) {
  const Shape& h = SHAPES[s];
  const int splits = split ? splits_of(s, M, N, K, eb) : 1;
  const double rate = (eb == 2 ? 4.6e6 : 0.55e6) * (s == S256 ? 1.0 : s == S64 ? 0.6 : 0.85);
  const double rounds = (double)div_up(tiles_of(s, M, N) * splits, (int64_t)CUS * h.per_cu);
  const double area = (double)h.BM * h.BN, k = (double)div_up(K, splits);
  double us = rounds * (h.per_cu * area * k * 2 / rate + 3 + (h.per_cu == 1 ? area * (splits > 1 ? 4 : eb) * CUS / 4e6 : 0));
  if (splits > 1) us += 4 + (double)M * N * (8 * splits + eb) / 4e6;
  return us;
}

int best_square(int64_t M, int64_t N, int64_t K, int64_t eb, bool split) {
  int best = S256;
  for (int s = S128; s <= S64; ++s)
    if (cost_of(s, M, N, K, eb, split) < cost_of(best, M, N, K, eb, split)) best = s;
  return best;
}

int logits_shape(int64_t V, int64_t N, int64_t H, int64_t eb, bool backward) {
  if (!backward && N <= 64) {
    if (N <= 16) return div_up(V, 128) >= 3 * CUS ? SK16W : SK16;
    return N <= 32 ? SK32 : SK64;
  }
  if (V <= 64) return div_up(N, 128) >= CUS ? SM64 : S64;
  return best_square(V, N, H, eb, false);
}

// A short sum (65 to 256 vocabulary entries) is bound by writing dx: small tiles, six a CU, so that some write while
// others multiply (fp32 262144 x 512 over 65: 204 us, 305 with the best square; 131072 x 1024 over 250: 554 and 593; bf16
// 262144 x 1024 over 100: 222 and 239; 131072 x 2048 over 250: 284 and 304).
int dx_shape(int64_t H, int64_t N, int64_t K, int64_t eb, bool split) {
  return K <= 256 && H > 64 ? SD64 : best_square(H, N, K, eb, split);
}

int dw_shape(int64_t H, int64_t V, int64_t N, int64_t eb) {
  if (V <= 64 && H > 64) return SN64;
  return best_square(H, V, N, eb, true);
}

struct Problem {
  int64_t N, V, H;
  int dtype;
  bool pack_x, pack_w;
  int64_t Hp;       // hidden size of packed rows
  bool kept;        // logits
  size_t eb;
};

// Vocabulary entries of a backward piece: dl of a piece takes about 256 MB, or 256 entries where those are more (from 524288
// tokens in bf16).  8192 tokens over 128000 (2 GB in one piece):
// 27.4 ms a step with 256 MB, 27.2 with 128, 27.7 with 1024; 4095 over 32001 (250 MB): 1.80 ms, 1.90 in pieces of 128 MB.
constexpr int64_t PIECE_BYTES = 256 << 20;
int64_t piece_of(const Problem& p) {
  if (p.V <= 256) return p.V;
  int64_t v = PIECE_BYTES / (p.N * (int64_t)p.eb) / 256 * 256;
  // at least a chip's worth of tiles of the logits' product
  const int64_t fill = up(div_up((int64_t)CUS * 256, div_up(p.N, 256)), 256);
  if (v < fill) v = fill;
  if (v >= p.V) return p.V;
  return up(div_up(p.V, div_up(p.V, v)), 256);
}

struct Layout {
  size_t xp, wp, part, at, sums;                    // forward
  size_t row, list, total, factor, first, used, dl, dxacc, dwacc, dbias;  // backward
  size_t bytes;
};

struct Taker {
  size_t at = 0;
  size_t operator()(size_t bytes) {
    const size_t p = at;
    at += (bytes + 255) & ~(size_t)255;
    return p;
  }
};

// Rows a workgroup of the joining kernel takes.  Few parts: rows side by side; few rows: threads side by side on the
// parts of a row; 64 rows where there are as many, so that a wave reads neighbouring parts.
int rows_of(int64_t N, int64_t tiles) {
  int rows = 1;
  while (rows < 1024 && rows < N && 1024 / rows > tiles) rows <<= 1;
  while (rows < 64 && rows < N) rows <<= 1;
  return rows;
}

// Few tiles (a small batch over a small vocabulary) are bound by the latency of their stages, one after the other: the
// hidden size is split over the chip, into 16 parts at most of four stages at least (logits and rows; fp32 20 tokens of
// 4096 over 100: 148 us whole, 18 in 16 parts; 20 of 512 over 60: 27 whole, 13 in four parts).
// The statistics of the tiles (8 bytes for a token and a tile's words) are held for a block of tokens at a time, 256 MB of
// them: 524288 tokens over 128000 would leave 2.1 GB.  A block has 1024 tokens at least (rows a workgroup joins, and some
// tiles of tokens; then it is V that is long, and the statistics take 128 bytes a word at most).
constexpr int64_t PART_BYTES = 256 << 20;
struct FwdPlan {
  int s, splits, rows;   // tile shape; rows a workgroup joins
  int64_t groups, block; // of rows; tokens at a time
};

FwdPlan fwd_plan(const Problem& p) {
  FwdPlan f;
  f.s = logits_shape(p.V, p.N, p.Hp, (int64_t)p.eb, false);
  const int64_t tiles = tiles_of(f.s, p.V, p.N), want = 2 * CUS / tiles;
  const int64_t stages = p.Hp * (int64_t)p.eb / SHAPES[f.s].KB, most = stages / 4 < 16 ? stages / 4 : 16;
  f.splits = (int)(want < most ? want : most);
  if (f.splits < 2 || f.s == S256 || f.s == SM64) f.splits = 1;
  f.rows = f.splits > 1 ? (p.V <= 256 ? 16 : p.V <= 1024 ? 4 : 1) : rows_of(p.N, div_up(p.V, SHAPES[f.s].BM));
  f.groups = div_up(p.N, f.rows);
  f.block = p.N;
  const int64_t fit = PART_BYTES / ((int64_t)sizeof(float2) * div_up(p.V, SHAPES[f.s].BM));
  const int64_t most_tokens = fit < 1024 ? 1024 : fit / 1024 * 1024;
  if (f.splits == 1 && p.N > most_tokens) f.block = up(div_up(p.N, div_up(p.N, most_tokens)), 1024);
  return f;
}

Layout fwd_layout(const Problem& p) {
  Layout L = {};
  Taker take;
  L.xp = take(p.pack_x ? (size_t)p.N * p.Hp * p.eb : 0);
  L.wp = take(p.pack_w ? (size_t)p.V * p.Hp * p.eb : 0);
  const FwdPlan f = fwd_plan(p);
  L.part = take(f.splits > 1 ? (size_t)f.splits * p.N * up(p.V, 4) * 4 : (size_t)div_up(p.V, SHAPES[f.s].BM) * f.block * sizeof(float2));
  L.at = take((size_t)f.block * 4);
  L.sums = take((size_t)f.groups * sizeof(LossPart));
  L.bytes = take.at + 256;
  return L;
}

struct BwdPlan {
  int64_t piece, ldl;
  int s_dl, s_dx, s_dw, split_dx, split_dw;
  int64_t pieces;
};

BwdPlan bwd_plan(const Problem& p) {
  BwdPlan b;
  b.piece = piece_of(p);
  b.pieces = div_up(p.V, b.piece);
  b.ldl = up(b.piece, 64);
  const int64_t eb = (int64_t)p.eb;
  b.s_dl = p.kept ? SM64 : logits_shape(b.piece, p.N, p.Hp, eb, true);  // (kept: no product, any shape)
  b.s_dx = dx_shape(p.H, p.N, b.piece, eb, b.pieces == 1);
  b.s_dw = dw_shape(p.H, b.piece, p.N, eb);
  b.split_dx = b.pieces == 1 ? splits_of(b.s_dx, p.H, p.N, b.piece, eb) : 1;
  b.split_dw = splits_of(b.s_dw, p.H, b.piece, p.N, eb);
  return b;
}

Layout bwd_layout(const Problem& p, const BwdPlan& b) {
  Layout L = {};
  Taker take;
  L.xp = take(p.pack_x ? (size_t)p.N * p.Hp * p.eb : 0);
  L.wp = take(p.pack_w ? (size_t)p.V * p.Hp * p.eb : 0);
  L.row = take((size_t)p.N * sizeof(Row));
  L.list = take(((size_t)p.N + LIST_SLACK) * 4);
  L.total = take(4);
  L.factor = take(4);
  L.first = take((size_t)div_up(p.N, 1024) * 4);
  L.used = take((size_t)p.N);
  L.dl = take((size_t)p.N * b.ldl * p.eb);
  L.dxacc = take(b.pieces > 1 || b.split_dx > 1 ? (size_t)b.split_dx * p.N * p.H * 4 : 0);
  L.dwacc = take(b.split_dw > 1 ? (size_t)b.split_dw * b.piece * p.H * 4 : 0);
  L.dbias = take((size_t)div_up(p.N, 64) * b.ldl * 4);  // tiles of 64 tokens or more, with kept logits or without
  L.bytes = take.at + 256;
  return L;
}

int problem_of(const pmg_linear_ce* a, Problem* p) {
  if (a->N < 1 || a->V < 1 || a->H < 1 || a->N > 0x7fffff00 || a->V > 0x7fffff00 || a->H > 65536) return PMG_E_ARG;
  if (a->dtype != PMG_F32 && a->dtype != PMG_BF16) return PMG_E_DTYPE;
  if (a->id_bits != 32 && a->id_bits != 64) return PMG_E_DTYPE;
  if (a->ld_hidden < a->H || a->ld_weight < a->H) return PMG_E_ARG;
  if (a->reduction != PMG_REDUCE_NONE && a->reduction != PMG_REDUCE_SUM && a->reduction != PMG_REDUCE_MEAN) return PMG_E_ARG;
  p->N = a->N; p->V = a->V; p->H = a->H; p->dtype = a->dtype;
  p->eb = pmg_elem_bytes(a->dtype);
  const int64_t e16 = 16 / (int64_t)p->eb;
  p->Hp = up(a->H, e16);
  p->kept = a->logits != nullptr;
  // 16-byte loads: rows that do not begin at multiples of 16 bytes, or whose end does not, are copied to rows that do
  const bool tail = a->H % e16 != 0;
  p->pack_x = tail || a->ld_hidden % e16 != 0 || ((uintptr_t)a->hidden & 15) != 0;
  p->pack_w = tail || a->ld_weight % e16 != 0 || ((uintptr_t)a->weight & 15) != 0;
  const size_t eb = p->eb;
  if (((uintptr_t)a->hidden | (uintptr_t)a->weight | (uintptr_t)a->bias) & (eb - 1)) return PMG_E_ALIGN;
  if ((uintptr_t)a->logits & 15) return PMG_E_ALIGN;
  if (((uintptr_t)a->targets & (a->id_bits / 8 - 1)) || ((uintptr_t)a->row_weight & 3)) return PMG_E_ALIGN;
  return PMG_OK;
}

template <typename T, int S, int WAY> int launch_logits(const LogitArgs& a, hipStream_t st) {
  static std::atomic<unsigned long long> done{0};
  if (const hipError_t e = pmg_full_lds_once((const void*)&lce_logits_kernel<T, S, WAY>, &done)) return (int)e;
  // without the product only the sums over the tokens are in LDS
  constexpr int LDS = WAY == KEPT ? SHAPES[S].WN * SHAPES[S].BM * (int)sizeof(float) : TileOf<T, S, true, true, false, WAY == REFORM>::LDS;
  hipLaunchKernelGGL((lce_logits_kernel<T, S, WAY>), dim3((unsigned)((int64_t)a.tiles_m * a.tiles_n), WAY == SPLIT ? a.splits : 1),
                     dim3(THREADS_OF<S>), LDS, st, a);
  return (int)hipGetLastError();
}

template <typename T, int WAY> int logits(int s, LogitArgs a, hipStream_t st) {
  a.tiles_m = (int)div_up(a.V, SHAPES[s].BM);
  a.tiles_n = (int)div_up(a.N, SHAPES[s].BN);
  if constexpr (WAY != SPLIT) {
    if (s == SM64) return launch_logits<T, SM64, WAY>(a, st);
    if constexpr (WAY != KEPT)
      if (s == S256) return launch_logits<T, S256, WAY>(a, st);
    if constexpr (WAY == FORWARD)
      if (s == SK16W) return launch_logits<T, SK16W, WAY>(a, st);
  }
  if constexpr (WAY != KEPT) switch (s) {
      case S128: return launch_logits<T, S128, WAY>(a, st);
      case S64: return launch_logits<T, S64, WAY>(a, st);
    }
  if constexpr (WAY == FORWARD || WAY == SPLIT) switch (s) {
      case SK16: return launch_logits<T, SK16, WAY>(a, st);
      case SK32: return launch_logits<T, SK32, WAY>(a, st);
      case SK64: return launch_logits<T, SK64, WAY>(a, st);
    }
  return PMG_E_ARG;
}

template <typename T, int S, bool BKC> int launch_grad(const GradArgs& a, hipStream_t st) {
  static std::atomic<unsigned long long> done{0};
  if (const hipError_t e = pmg_full_lds_once((const void*)&lce_grad_kernel<T, S, BKC>, &done)) return (int)e;
  const int64_t blocks = (int64_t)a.tiles_m * a.tiles_n + (BKC && a.zeroed ? div_up(a.N, 64) : 0);
  hipLaunchKernelGGL((lce_grad_kernel<T, S, BKC>), dim3((unsigned)blocks, a.splits), dim3(THREADS_OF<S>),
                     (TileOf<T, S, false, BKC, !BKC, false>::LDS), st, a);
  return (int)hipGetLastError();
}

// The sums of a split go to acc and are joined into `out`.
template <typename T, bool BKC> int grad(int s, GradArgs a, hipStream_t st) {
  a.tiles_m = (int)div_up(a.M, SHAPES[s].BM);
  a.tiles_n = (int)div_up(a.N, SHAPES[s].BN);
  void* out = a.out;
  if (a.splits > 1) a.out = nullptr;
  int rc = PMG_E_ARG;
  switch (s) {
    case S256: rc = launch_grad<T, S256, BKC>(a, st); break;
    case S128: rc = launch_grad<T, S128, BKC>(a, st); break;
    case S64: rc = launch_grad<T, S64, BKC>(a, st); break;
    case SN64:
      if constexpr (!BKC) rc = launch_grad<T, SN64, BKC>(a, st);
      break;
    case SD64:
      if constexpr (BKC) rc = launch_grad<T, SD64, BKC>(a, st);
      break;
  }
  if (rc || a.splits == 1) return rc;
  const int64_t total = a.N * a.M;
  hipLaunchKernelGGL(lce_join_kernel<T>, dim3((unsigned)div_up(total, 256)), dim3(256), 0, st, a.acc, a.splits, a.N, a.M,
                     BKC ? a.list : nullptr, a.count, (T*)out, a.ldo);
  return (int)hipGetLastError();
}

template <typename T> int dx_narrow(GradArgs a, hipStream_t st) {
  const int64_t blocks_m = div_up(a.M, 1024 / (int64_t)sizeof(T)), chunks = div_up(a.N, NARROW_TOKENS);
  const int64_t most = up(div_up((int64_t)CUS * NARROW_PER_CU, blocks_m), 8);  // (8: the columns of a token on one XCD)
  const int64_t blocks = div_up(chunks, div_up(chunks, most));                 // as many turns for all
  hipLaunchKernelGGL(lce_dx_narrow_kernel<T>, dim3((unsigned)blocks, (unsigned)blocks_m), dim3(256), 0, st, a);
  return (int)hipGetLastError();
}

template <typename T> int pack(const void* src, int64_t ld, int64_t rows, const Problem& p, void* dst, hipStream_t st) {
  int tpr = 1;
  while (tpr < 256 && tpr * (16 / (int)sizeof(T)) < p.Hp) tpr <<= 1;
  const int64_t blocks = div_up(rows, 256 / tpr), most = 1 << 20;  // (a launch has fewer than 2^32 threads)
  hipLaunchKernelGGL(lce_pack_kernel<T>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, st, (const T*)src, ld, rows,
                     p.H, (T*)dst, p.Hp, tpr);
  return (int)hipGetLastError();
}

// Operands as the tile product reads them
template <typename T>
int operands(const pmg_linear_ce* a, const Problem& p, const Layout& L, char* ws, LogitArgs* l, hipStream_t st) {
  l->X = a->hidden; l->ldx = a->ld_hidden;
  l->W = a->weight; l->ldw = a->ld_weight;
  if (p.pack_x) {
    if (const int rc = pack<T>(a->hidden, a->ld_hidden, p.N, p, ws + L.xp, st)) return rc;
    l->X = ws + L.xp; l->ldx = p.Hp;
  }
  if (p.pack_w) {
    if (const int rc = pack<T>(a->weight, a->ld_weight, p.V, p, ws + L.wp, st)) return rc;
    l->W = ws + L.wp; l->ldw = p.Hp;
  }
  l->bias = a->bias;
  l->N = p.N;
  l->K = p.Hp;
  l->scale = a->logit_scale;
  l->targets = a->targets; l->id_bits = a->id_bits;
  l->kept = a->logits; l->ldk = up(p.V, 4);
  return PMG_OK;
}

template <typename T> int forward(const pmg_linear_ce* a, const Problem& p, char* ws, hipStream_t st) {
  const Layout L = fwd_layout(p);
  LogitArgs l = {};
  if (const int rc = operands<T>(a, p, L, ws, &l, st)) return rc;
  l.V = p.V;
  l.v0 = 0;
  l.part = (float2*)(ws + L.part);
  l.at_target = (float*)(ws + L.at);
  const FwdPlan f = fwd_plan(p);
  l.splits = f.splits;
  l.sums = (float*)(ws + L.part);
  RowArgs r = {};
  r.part = l.part;
  r.at_target = l.at_target;
  r.tiles = (int)div_up(p.V, SHAPES[f.s].BM);
  r.V = p.V;
  r.id_bits = a->id_bits; r.ignore = a->ignore_index;
  const bool none = a->reduction == PMG_REDUCE_NONE;
  LossPart* sums = (LossPart*)(ws + L.sums);
  r.rows = f.rows;
  r.mean = a->reduction == PMG_REDUCE_MEAN;
  if (f.groups == 1 && !none) {
    r.loss = a->loss;
    r.count = a->count;
  }
  const char *X = (const char*)l.X, *targets = (const char*)a->targets;
  for (int64_t n0 = 0; n0 < p.N; n0 += f.block) {
    const int64_t n = n0 + f.block < p.N ? f.block : p.N - n0;
    l.N = r.N = n;
    l.X = X + n0 * l.ldx * (int64_t)p.eb;
    l.targets = r.targets = targets + n0 * (a->id_bits / 8);
    l.kept = a->logits ? a->logits + n0 * l.ldk : nullptr;
    if (const int rc = f.splits > 1 ? logits<T, SPLIT>(f.s, l, st) : logits<T, FORWARD>(f.s, l, st)) return rc;
    r.weight = a->row_weight ? a->row_weight + n0 : nullptr;
    r.lse = a->lse + n0;
    r.nll = none ? a->loss + n0 : nullptr;
    r.sums = none ? nullptr : sums + n0 / f.rows;
    const dim3 groups((unsigned)div_up(n, f.rows));
    if (f.splits > 1) {
      const SplitArgs b = {l.sums, f.splits, l.ldk, a->bias, a->logit_scale, l.kept};
      hipLaunchKernelGGL(lce_split_rows_kernel<T>, groups, dim3(1024), 0, st, b, r);
    } else {
      hipLaunchKernelGGL(lce_rows_kernel, groups, dim3(1024), 0, st, r);
    }
  }
  if (!none && f.groups > 1)
    hipLaunchKernelGGL(lce_loss_kernel, dim3(1), dim3(1024), 0, st, sums, (int)f.groups, r.mean, a->loss, a->count);
  return (int)hipGetLastError();
}

template <typename T> int backward(const pmg_linear_ce* a, const Problem& p, char* ws, hipStream_t st) {
  const BwdPlan b = bwd_plan(p);
  const Layout L = bwd_layout(p, b);
  LogitArgs l = {};
  if (const int rc = operands<T>(a, p, L, ws, &l, st)) return rc;
  SlopeArgs sl = {};
  sl.g_loss = a->grad_loss; sl.g_lse = a->grad_lse; sl.lse = a->lse; sl.count = a->count; sl.weight = a->row_weight;
  sl.per_row = a->reduction == PMG_REDUCE_NONE;
  sl.mean = a->reduction == PMG_REDUCE_MEAN;
  sl.targets = a->targets; sl.id_bits = a->id_bits; sl.ignore = a->ignore_index;
  sl.N = p.N; sl.V = p.V;
  sl.first = (int*)(ws + L.first);
  sl.groups = (int)div_up(p.N, 1024);
  sl.row = (Row*)(ws + L.row);
  sl.list = (int*)(ws + L.list);
  sl.total = (int*)(ws + L.total);
  sl.scale = a->logit_scale;
  sl.factor = (float*)(ws + L.factor);
  sl.used = (uint8_t*)(ws + L.used);
  if (sl.groups > OWN_GROUPS) {
    hipLaunchKernelGGL(lce_slopes_kernel<false>, dim3(sl.groups), dim3(1024), 0, st, sl);
    hipLaunchKernelGGL(lce_scan_kernel, dim3(1), dim3(1024), 0, st, sl.first, sl.groups);
  }
  hipLaunchKernelGGL(lce_slopes_kernel<true>, dim3(sl.groups), dim3(1024), 0, st, sl);
  l.row = sl.row;
  l.list = sl.list;
  l.count = sl.total;
  l.factor = sl.factor;
  l.dl = ws + L.dl;
  l.ldl = b.ldl;
  l.dbias = a->grad_bias ? (float*)(ws + L.dbias) : nullptr;
  const char* W = (const char*)l.W;
  const char* bias = (const char*)a->bias;
  for (int64_t i = 0; i < b.pieces; ++i) {
    const int64_t v0 = i * b.piece, v = v0 + b.piece < p.V ? b.piece : p.V - v0;
    l.v0 = v0;
    l.V = v;
    l.W = W + v0 * l.ldw * (int64_t)p.eb;
    l.bias = bias ? bias + v0 * (int64_t)p.eb : nullptr;
    if (const int rc = l.kept ? logits<T, KEPT>(b.s_dl, l, st) : logits<T, REFORM>(b.s_dl, l, st)) return rc;
    if (a->grad_bias)
      hipLaunchKernelGGL(lce_dbias_kernel<T>, dim3((unsigned)div_up(v, 64)), dim3(1024), 0, st, l.dbias,
                         SHAPES[b.s_dl].BN, sl.total, b.ldl, v, (T*)a->grad_bias + v0);
    if (a->grad_hidden) {
      GradArgs g = {};
      g.A = l.W; g.lda = l.ldw; g.M = p.H;
      g.B = l.dl; g.ldb = b.ldl; g.N = p.N;
      g.K = v;
      g.list = sl.list;
      g.count = sl.total;
      g.factor = sl.factor;
      g.splits = b.split_dx;
      g.out = i == b.pieces - 1 ? a->grad_hidden : nullptr;
      g.ldo = p.H;
      g.acc = b.pieces > 1 || b.split_dx > 1 ? (float*)(ws + L.dxacc) : nullptr;
      g.add = i > 0;
      g.used = sl.used;
      g.zeroed = i == 0 ? a->grad_hidden : nullptr;
      if (const int rc = p.V <= NARROW ? dx_narrow<T>(g, st) : grad<T, true>(b.s_dx, g, st)) return rc;
    }
    if (a->grad_weight) {
      GradArgs g = {};
      g.A = l.X; g.lda = l.ldx; g.M = p.H;
      g.B = l.dl; g.ldb = b.ldl; g.N = v;
      g.K = p.N;
      g.list = sl.list;
      g.count = sl.total;
      g.factor = sl.factor;
      g.splits = b.split_dw;
      g.out = (T*)a->grad_weight + v0 * p.H;
      g.ldo = p.H;
      g.acc = b.split_dw > 1 ? (float*)(ws + L.dwacc) : nullptr;
      if (const int rc = grad<T, false>(b.s_dw, g, st)) return rc;
    }
  }
  return (int)hipGetLastError();
}

// What no launch covers (half a billion words or tokens) is refused before the first one.
int forward_fits(const Problem& p) {
  const FwdPlan f = fwd_plan(p);
  return covers(f.s, p.V, f.block) ? PMG_OK : PMG_E_ARG;
}
int backward_fits(const Problem& p) {
  const BwdPlan b = bwd_plan(p);
  const bool dx = p.V <= NARROW || covers(b.s_dx, p.H, p.N, div_up(p.N, 64));
  return covers(b.s_dl, b.piece, p.N) && dx && covers(b.s_dw, p.H, b.piece) ? PMG_OK : PMG_E_ARG;
}

}  // namespace

extern "C" int pmg_linear_ce_workspace(const pmg_linear_ce* a, int backward, size_t* out) {
  if (!a || !out) return PMG_E_NULL;
  Problem p;
  if (const int rc = problem_of(a, &p)) return rc;
  if (const int rc = backward ? backward_fits(p) : forward_fits(p)) return rc;
  *out = backward ? bwd_layout(p, bwd_plan(p)).bytes : fwd_layout(p).bytes;
  return PMG_OK;
}

extern "C" int pmg_linear_ce_fwd(const pmg_linear_ce* a, void* ws, pmg_stream stream) {
  if (!a || !ws || !a->hidden || !a->weight || !a->targets || !a->loss || !a->lse) return PMG_E_NULL;
  if (a->reduction != PMG_REDUCE_NONE && !a->count) return PMG_E_NULL;
  Problem p;
  if (const int rc = problem_of(a, &p)) return rc;
  if (const int rc = forward_fits(p)) return rc;
  if (((uintptr_t)ws & 15) || (((uintptr_t)a->loss | (uintptr_t)a->lse | (uintptr_t)a->count) & 3)) return PMG_E_ALIGN;
  hipStream_t st = (hipStream_t)stream;
  return a->dtype == PMG_F32 ? forward<float>(a, p, (char*)ws, st) : forward<bf16_t>(a, p, (char*)ws, st);
}

extern "C" int pmg_linear_ce_bwd(const pmg_linear_ce* a, void* ws, pmg_stream stream) {
  if (!a || !ws || !a->hidden || !a->weight || !a->targets || !a->lse) return PMG_E_NULL;
  if (a->reduction == PMG_REDUCE_MEAN && !a->count) return PMG_E_NULL;
  if (a->grad_bias && !a->bias) return PMG_E_NULL;
  Problem p;
  if (const int rc = problem_of(a, &p)) return rc;
  if (const int rc = backward_fits(p)) return rc;
  if (((uintptr_t)ws & 15) || (((uintptr_t)a->grad_loss | (uintptr_t)a->grad_lse | (uintptr_t)a->lse | (uintptr_t)a->count) & 3))
    return PMG_E_ALIGN;
  if (((uintptr_t)a->grad_hidden | (uintptr_t)a->grad_weight | (uintptr_t)a->grad_bias) & (p.eb - 1)) return PMG_E_ALIGN;
  if (!a->grad_hidden && !a->grad_weight && !a->grad_bias) return PMG_OK;
  hipStream_t st = (hipStream_t)stream;
  return a->dtype == PMG_F32 ? backward<float>(a, p, (char*)ws, st) : backward<bf16_t>(a, p, (char*)ws, st);
}
