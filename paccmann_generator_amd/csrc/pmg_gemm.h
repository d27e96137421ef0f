// The tile product behind the linear cross entropy (pmg_lce.hip):  D[m][n] = sum_k A(m,k) B(n,k)  for one
// BM x BN tile, on MFMA, operands in bf16 or fp32, sums in fp32.
//
// An operand lies in memory with k contiguous (rows of m or n) or with m / n contiguous (rows of k): the
// vocabulary projection and the hidden states enter the logits the first way and their own gradients the
// second way, so no transposed copy of either is made.
//
// LDS holds two stages of 128 bytes of k per row (64 bf16 or 32 fp32), filled by 16-byte loads that go
// straight to LDS; while a stage is multiplied the next one is in flight.  The loads write LDS linearly, so
// what keeps the reads free of bank conflicts is which global 16 bytes a lane fetches:
//   k contiguous: 16-byte piece c of row r lies at piece c ^ (r & 7); a fragment is one ds_read_b128
//   m contiguous: 32-byte (bf16) or 64-byte (fp32) pieces of row k lie at piece ^ f(k), f chosen so that the
//                 rows one read touches fall into different banks; a bf16 fragment is two transposing
//                 reads (ds_read_b64_tr_b16), an fp32 fragment four single ones
// An operand may be read through a list of its rows (of m or n where k is contiguous, of k otherwise): the
// training rows of a batch stay where they are.
// Lane l of a wave holds of a 16x16 tile of D column n = l & 15 and four rows m.  Which rows of m a fragment of A has is
// free: in bf16 two fragments share 32 rows so that a lane's eight are neighbours (8 (l >> 4) .. + 7, the first four in
// fragment i for even l >> 4 and in i + 1 for odd: half of the lanes read the other half of 16 bytes, which keeps all
// banks busy) and are stored as 16 bytes, 64 in a row with the lanes beside it; in fp32 four are 16 bytes already (m =
// 4 (l >> 4) .. + 3).
#pragma once
#include "pmg_kernels.h"
#include "pmg_types.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

typedef __attribute__((address_space(3))) char lds_char;

template <typename T> struct pmg_frag;  // 16 bytes of k of one row
template <> struct pmg_frag<bf16_t> {
  typedef bf16x8 type;
  static __device__ __forceinline__ f32x4 mma(type a, type b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct pmg_frag<float> {
  typedef f32x4 type;
  static __device__ __forceinline__ f32x4 mma(type a, type b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};

// 16 bytes that stand for operand elements behind the end of k
static __device__ const float4 pmg_zero16 = {0.f, 0.f, 0.f, 0.f};

__device__ __forceinline__ void pmg_load_lds16(const char* src, lds_char* dst) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                   (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}

// One operand's share of a stage: R rows of m (or n), 128 bytes of k.
//   KC: k contiguous.  WAVES waves fill it, 1 KB an instruction.  LIST: rows by a list.  PAIR: fragments share 32 rows.
template <typename T, int R, bool KC, int WAVES, bool LIST, int KB, bool PAIR> struct pmg_operand {
  static constexpr int E16 = 16 / sizeof(T);
  static constexpr int KSTEP = KB / sizeof(T);
  static constexpr int BYTES = R * KB;
  static constexpr int PER_ROW = KB / 16;         // 16-byte pieces of a row's k (k contiguous)
  static constexpr int CNT = BYTES / 1024 / WAVES;
  static constexpr int ROWB = R * sizeof(T);      // bytes of a row of k (m contiguous)
  static constexpr int PIECES = ROWB / 16;
  static_assert(BYTES % (1024 * WAVES) == 0, "whole instructions");
  static_assert(KC || PIECES >= 8, "the permutation stays inside a row");

  static __device__ __forceinline__ int perm(int k) {  // of the 16-byte pieces of row k (m contiguous)
    if (PAIR) return ((k & 1) | (((k >> 1) & 1) << 2) | (((k >> 3) & 1) << 3)) & (PIECES - 1);
    if (sizeof(T) == 2) return (((k & 3) | (((k >> 3) & 3) << 2)) & (PIECES / 2 - 1)) << 1;
    return (((k >> 2) & 3) << 2) & (PIECES - 1);
  }

  static __device__ __forceinline__ int perm_k(int row) {  // of the pieces of a row (k contiguous)
    if (PAIR) return KB == 128 ? ((row >> 1) & 1) | (((row >> 3) & 3) << 1) : (row >> 3) & 3;
    return KB == 128 ? row & 7 : (row >> 2) & 3;
  }

  const char* src[CNT];
  int64_t step;   // bytes from stage to stage
  int kofs[CNT];  // k of this lane's 16 bytes within a stage
  // m contiguous with a list: the entries of the rows that this wave fetches in the next stage.  An instruction that
  // covers one or two rows takes them through scalar loads, which do not count among the stages' vector loads; one that
  // covers more (narrow tiles, of two stages, which wait for all loads anyway) by a load per lane.
  typedef const __attribute__((address_space(4))) int* scalar_list;
  static constexpr int ROWS = KC ? 1 : CNT * 1024 / ROWB;  // of a wave
  static constexpr int RPI = ROWS / CNT > 0 ? ROWS / CNT : 1;
  static constexpr bool SCALAR = RPI <= 2;
  static constexpr bool BY_LIST = LIST && !KC;
  scalar_list list;
  const int* lane_list;
  int64_t row_bytes;
  int next[!BY_LIST ? 1 : SCALAR ? ROWS : CNT];

  __device__ __forceinline__ void look_up() {
    if constexpr (BY_LIST && SCALAR) {
#pragma unroll
      for (int j = 0; j < ROWS; ++j) next[j] = list[j];
      list += KSTEP;
    } else if constexpr (BY_LIST) {
#pragma unroll
      for (int j = 0; j < CNT; ++j) next[j] = lane_list[kofs[j]];
      lane_list += KSTEP;
    }
  }

  // rows row0 .. of R_all (clamped: rows behind the end repeat the last one and are not stored), k from k0
  __device__ __forceinline__ void init(const void* base, int64_t ld, const int* rows, int64_t row0, int64_t R_all,
                                       int64_t k0) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    step = KC ? KB : (int64_t)KSTEP * ld * (int64_t)sizeof(T);
#pragma unroll
    for (int j = 0; j < CNT; ++j) {
      const int byte = (wave * CNT + j) * 1024 + lane * 16;
      if (KC) {
        const int row = byte / KB, c = ((byte >> 4) & (PER_ROW - 1)) ^ perm_k(row);
        int64_t r = row0 + row < R_all ? row0 + row : R_all - 1;
        if (LIST) r = rows[r];
        kofs[j] = c * E16;
        src[j] = (const char*)base + (r * ld + k0 + kofs[j]) * (int64_t)sizeof(T);
      } else {
        const int k = byte / ROWB, c = ((byte % ROWB) >> 4) ^ perm(k);
        const int64_t last = ((R_all + E16 - 1) / E16 - 1) * E16;
        const int64_t m = row0 + c * E16 < last ? row0 + c * E16 : last;
        kofs[j] = k;
        src[j] = (const char*)base + ((LIST ? 0 : (k0 + k) * ld) + m) * (int64_t)sizeof(T);
      }
    }
    if (BY_LIST) {
      row_bytes = ld * (int64_t)sizeof(T);
      list = (scalar_list)(rows + k0) + __builtin_amdgcn_readfirstlane(wave) * ROWS;
      lane_list = rows + k0;
      look_up();
    }
  }

  // one stage into LDS at `dst`.  PART: only `left` of its k exist (the others read as zeros), and the operand stays
  // where it is; else it moves on by a stage.
  template <bool PART> __device__ __forceinline__ void fetch(lds_char* dst, int left) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    lds_char* d = dst + wave * (CNT * 1024);
#pragma unroll
    for (int j = 0; j < CNT; ++j) {
      const char* from = src[j];
      if constexpr (BY_LIST && SCALAR) {
        // (named scalar values: a choice between two elements would make the array's index depend on the lane)
        const int64_t at = __builtin_amdgcn_readfirstlane(next[j * RPI]) * row_bytes;
        const int64_t behind = __builtin_amdgcn_readfirstlane(next[j * RPI + RPI - 1]) * row_bytes;
        from += RPI == 2 && lane >= 32 ? behind : at;
      } else if constexpr (BY_LIST) {
        from += next[j] * row_bytes;
      } else if (!PART) {
        src[j] += step;
      }
      if (PART) from = kofs[j] < left ? from : (const char*)&pmg_zero16;
      pmg_load_lds16(from, d + j * 1024);
    }
    if (BY_LIST && !PART) look_up();
  }

  // behind a PART stage at the end of k: back by n stages
  __device__ __forceinline__ void back(int64_t n) {
    if constexpr (BY_LIST) {
      list -= (n + 1) * KSTEP;
      lane_list -= (n + 1) * KSTEP;
      look_up();
    } else {
#pragma unroll
      for (int j = 0; j < CNT; ++j) src[j] -= n * step;
    }
  }

  typedef typename pmg_frag<T>::type frag;
  // fragment f of the rows from `row` (of this operand's R) for half kk of the stage
  static __device__ __forceinline__ frag read(const lds_char* s, int row, int f, int kk) {
    const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
    // where the q-th four of its rows begins
    const auto quad = [&](int q) { return row + (PAIR ? (f >> 1) * 32 + 8 * q + 4 * ((f ^ q) & 1) : f * 16 + 4 * q); };
    if (KC) {
      const int r = quad(i >> 2) + (i & 3);
      return *(const __attribute__((address_space(3))) frag*)(s + r * KB + (((kk * 4 + g) ^ perm_k(r)) << 4));
    } else if constexpr (sizeof(T) == 2) {
      frag out;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = kk * 32 + 8 * g + 4 * h + (i >> 2);
        const int m = quad(i & 3), c = m >> 3;
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        const s16x4 t = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)(s + k * ROWB + ((c ^ perm(k)) << 4) + ((m & 4) << 1)));
        const bf16x4 v = __builtin_bit_cast(bf16x4, t);
#pragma unroll
        for (int j = 0; j < 4; ++j) out[4 * h + j] = v[j];
      }
      return out;
    } else {
      static_assert(!PAIR, "fp32");
      frag out;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = kk * 16 + 4 * g + j, m = quad(0) + i;
        out[j] = *(const __attribute__((address_space(3))) float*)(s + k * ROWB + (((m >> 2) ^ perm(k)) << 4) + ((m & 3) << 2));
      }
      return out;
    }
  }
};

// The tile of workgroup `id`: workgroups go round the 8 XCDs, so every XCD gets a run of neighbouring tiles
// (its L2 then serves the operands' rows that they share), in blocks of 8 tiles of m by all of n.
__device__ __forceinline__ void pmg_tile_of(int id, int tiles_m, int tiles_n, int* tm, int* tn) {
  const int total = tiles_m * tiles_n, q = total >> 3, r = total & 7, x = id & 7;
  const int t = x * q + (x < r ? x : r) + (id >> 3);
  const int width = 8 * tiles_n, g = t / width, first = g * 8;
  const int gm = tiles_m - first < 8 ? tiles_m - first : 8, in = t - g * width;
  *tm = first + in % gm;
  *tn = in / gm;
}

// acc[i][j]: the 16x16 tiles of wave (wm, wn)'s (BM / WM) x (BN / WN) part; k from k0 to k1 (k0 a multiple of the
// stage).  Ends behind a barrier: LDS is free.  A list of rows of k may be read up to two stages beyond k1.
template <typename T, int BM, int BN, int WM, int WN, bool AKC, bool BKC, bool ALIST, bool BLIST, int KB, int STAGES>
struct pmg_tile {
  static constexpr int WAVES = WM * WN, THREADS = WAVES * 64;
  static constexpr int MI = BM / WM / 16, NI = BN / WN / 16;
  static constexpr bool PAIR = sizeof(T) == 2;
  typedef pmg_operand<T, BM, AKC, WAVES, ALIST, KB, PAIR> OpA;
  typedef pmg_operand<T, BN, BKC, WAVES, BLIST, KB, false> OpB;
  static constexpr int STAGE = OpA::BYTES + OpB::BYTES;
  static constexpr int LDS = STAGES * STAGE;
  static constexpr int KSTEP = OpA::KSTEP;
  static constexpr int LOADS = OpA::CNT + OpB::CNT;  // of a wave and stage
  static constexpr int KK = KB / 64, HI = MI / 2;
  static_assert(MI % 2 == 0, "two halves");
  static_assert((!OpA::BY_LIST || OpA::SCALAR || STAGES == 2) && !OpB::BY_LIST, "loads that stage() does not count");

  // row of acc[i][.][0] of lane 0 .. 63 in the wave's part of m
  static __device__ __forceinline__ int row_of(int i) {
    const int g = (threadIdx.x & 63) >> 4;
    return PAIR ? (i >> 1) * 32 + 8 * g + 4 * ((i ^ g) & 1) : i * 16 + 4 * g;
  }

  // PAIR: the first row of a lane's eight in fragments i and i + 1 (i even), and whether fragment i has the upper four
  static __device__ __forceinline__ int pair_of(int i) { return (i >> 1) * 32 + 8 * ((threadIdx.x & 63) >> 4); }
  static __device__ __forceinline__ bool swapped() { return (threadIdx.x >> 4) & 1; }

  OpA a;
  OpB b;
  typename OpA::frag fa[2][HI];
  typename OpB::frag fb[2][NI];
  int rowA, rowB;

  __device__ __forceinline__ void read_a(const lds_char* s, int half, int kk) {
#pragma unroll
    for (int i = 0; i < HI; ++i) fa[half][i] = OpA::read(s, rowA, half * HI + i, kk);
  }
  __device__ __forceinline__ void read_b(const lds_char* s, int set, int kk) {
#pragma unroll
    for (int j = 0; j < NI; ++j) fb[set][j] = OpB::read(s + OpA::BYTES, rowB, j, kk);
  }
  __device__ __forceinline__ void multiply(f32x4 (&acc)[MI][NI], int half, int set) {
#pragma unroll
    for (int i = 0; i < HI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[half * HI + i][j] = pmg_frag<T>::mma(fa[half][i], fb[set][j], acc[half * HI + i][j]);
  }

  // One stage: it has landed (loads complete in order: those of the stages behind it may be under way), and every wave
  // has read what it needs of the stage before, whose place (`put`) the next fetch takes.  The two places never are the
  // same, which __restrict__ tells the compiler: else it would wait for the fetch before it reads.
  // The fragments of a half are read while the half before them is multiplied: the first products here are those of the
  // second half of the stage before (none in the FIRST one).
  template <bool FETCH, bool FIRST>
  __device__ __forceinline__ void stage(f32x4 (&acc)[MI][NI], lds_char* __restrict__ put, const lds_char* __restrict__ get) {
    if (FETCH) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((STAGES - 2) * LOADS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (FETCH) {
      a.template fetch<false>(put, 0);
      b.template fetch<false>(put + OpA::BYTES, 0);
    }
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      read_b(get, 1, kk);
      read_a(get, 0, kk);
      if (!FIRST || kk > 0) multiply(acc, 1, 0);
      read_a(get, 1, kk);
      multiply(acc, 0, 1);
#pragma unroll
      for (int j = 0; j < NI; ++j) fb[0][j] = fb[1][j];
    }
  }

  static __device__ __forceinline__ void run(f32x4 (&acc)[MI][NI], lds_char* lds, const void* A, int64_t lda, const int* rows_a,
                                             int64_t m0, int64_t M, const void* B, int64_t ldb, const int* rows_b, int64_t n0,
                                             int64_t N, int64_t k0, int64_t k1) {
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (k1 <= k0) return;
    pmg_tile t;
    t.rowA = (wave / WN) * (BM / WM);
    t.rowB = (wave % WN) * (BN / WN);
    const int full = (int)((k1 - k0) / KSTEP), part = (int)((k1 - k0) - (int64_t)full * KSTEP);
    const int steps = full + (part > 0);
    // the stage that is not whole comes first: the loop below has whole ones only
    t.a.init(A, lda, rows_a, m0, M, part ? k0 + (int64_t)full * KSTEP : k0);
    t.b.init(B, ldb, rows_b, n0, N, part ? k0 + (int64_t)full * KSTEP : k0);
    if (part) {
      t.a.template fetch<true>(lds, part);
      t.b.template fetch<true>(lds + OpA::BYTES, part);
      t.a.back(full);
      t.b.back(full);
    }
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s)
      if (s < steps && (s > 0 || !part)) {
        t.a.template fetch<false>(lds + s * STAGE, 0);
        t.b.template fetch<false>(lds + s * STAGE + OpA::BYTES, 0);
      }
    __builtin_amdgcn_s_waitcnt(0);
    int put = STAGES - 1, get = 1 % STAGES, s = 1;
    if (steps > STAGES - 1) {
      t.template stage<true, true>(acc, lds + put * STAGE, lds);
      put = 0;
    } else {
      t.template stage<false, true>(acc, lds, lds);
    }
    for (; s < steps - (STAGES - 1); ++s) {
      t.template stage<true, false>(acc, lds + put * STAGE, lds + get * STAGE);
      put = put + 1 == STAGES ? 0 : put + 1;
      get = get + 1 == STAGES ? 0 : get + 1;
    }
    for (; s < steps; ++s) {
      t.template stage<false, false>(acc, lds, lds + get * STAGE);
      get = get + 1 == STAGES ? 0 : get + 1;
    }
    t.multiply(acc, 1, 0);
    __syncthreads();
  }
};
