// Norm and clipping of many gradients, and the Adam / AdamW update of many parameters (include/pmg_lm.h).
//
// All of it is bound by memory: every element is read and written once and takes a handful of fp32
// operations.  Tensors are cut into chunks and a workgroup takes one chunk, so a launch covers many tensors
// of any size; the table of tensors travels in the kernel's arguments (up to 4 KB), so nothing has to be
// copied to the device first, nothing is kept between calls, and a captured graph holds what it needs.
#include "pmg_types.h"
#include <algorithm>
#include <new>
#include <cstdlib>

namespace {

constexpr int THREADS = 256;
// Workgroups a launch: of 2^32 threads or more only some run, without an error.
constexpr int64_t MOST_GROUPS = (((int64_t)1 << 32) - 1) / THREADS;

// The tensor that owns chunk `c`: first[0] = 0, first[k] <= c < first[k+1].  Uniform: scalar loads.
template <typename Table> __device__ __forceinline__ int owner(const Table& t, int c) {
  int lo = 0, hi = t.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= c) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ float clip_factor(const float* norm, double max_norm) {
  const double c = max_norm / ((double)norm[0] + 1e-6);
  return (float)(c > 1.0 ? 1.0 : c);  // a NaN norm stays NaN
}

// ------------------------------------------------------------------------------------------ norm, clip
constexpr int GT_MAX = 160;
struct GradTable {
  void* g[GT_MAX];
  int64_t n_el[GT_MAX];
  int first[GT_MAX];
  uint8_t dtype[GT_MAX];
  int n;
};
static_assert(sizeof(GradTable) <= 3800, "kernel arguments");

template <typename T>
__device__ __forceinline__ double square_sum(const T* __restrict__ g, int64_t n, int64_t lo, int chunk) {
  double s = 0.0;
  // whole: loads of 16 bytes without a branch between them, eight under way (468 M bf16: 208 us, 229 with the loop below)
  if (n - lo >= chunk) {
    constexpr int VEC = pmg_vec16<T>::N;
    for (int i = threadIdx.x * VEC; i < chunk; i += THREADS * VEC * 8) {
      typename pmg_vec16<T>::vec x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (i + u * THREADS * VEC < chunk) x[u] = pmg_vec16<T>::load(g + lo + i + u * THREADS * VEC, VEC);
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (i + u * THREADS * VEC < chunk) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) s = fma((double)(float)x[u][j], (double)(float)x[u][j], s);
        }
    }
    return s;
  }
#pragma unroll 4
  for (int i = threadIdx.x * 4; i < chunk; i += THREADS * 4) {
    const int64_t left = n - lo - i;
    if (left <= 0) break;
    const f32x4 x = pmg_load4(g + lo + i, left);
#pragma unroll
    for (int j = 0; j < 4; ++j) s = fma((double)x[j], (double)x[j], s);
  }
  return s;
}

__device__ __forceinline__ double wave_sum(double s) {
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  return s;
}

// part[base + chunk] = sum of the chunk's squares, in fp64: squares of fp32 gradients overflow and
// underflow fp32, and the fp64 rate is far above what four bytes an element from memory ask for.
__global__ __launch_bounds__(THREADS) void norm_part_kernel(const GradTable t, int chunk, int base,
                                                            double* __restrict__ part) {
  __shared__ double wsum[THREADS / 64];
  const int k = owner(t, blockIdx.x);
  const int64_t lo = (int64_t)(blockIdx.x - t.first[k]) * chunk;
  double s;
  if (t.dtype[k] == PMG_F32) s = square_sum((const float*)t.g[k], t.n_el[k], lo, chunk);
  else if (t.dtype[k] == PMG_BF16) s = square_sum((const bf16_t*)t.g[k], t.n_el[k], lo, chunk);
  else s = square_sum((const f16_t*)t.g[k], t.n_el[k], lo, chunk);
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) wsum[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[base + blockIdx.x] = (wsum[0] + wsum[1]) + (wsum[2] + wsum[3]);
}

__global__ __launch_bounds__(1024) void norm_join_kernel(const double* __restrict__ part, int n,
                                                         float* __restrict__ norm) {
  __shared__ double wsum[16];
  double s = 0.0;
#pragma unroll 8
  for (int i = threadIdx.x; i < n; i += 1024) s += part[i];
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) wsum[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double a = 0.0;
    for (int w = 0; w < 16; ++w) a += wsum[w];
    norm[0] = (float)sqrt(a);
  }
}

template <typename T>
__device__ __forceinline__ void scale_chunk(T* __restrict__ g, int64_t n, int64_t lo, int chunk, float c) {
#pragma unroll 4
  for (int i = threadIdx.x * 4; i < chunk; i += THREADS * 4) {
    const int64_t left = n - lo - i;
    if (left <= 0) break;
    f32x4 x = pmg_load4(g + lo + i, left);
    x *= c;
    pmg_store4(g + lo + i, x, left);
  }
}

__global__ __launch_bounds__(THREADS) void clip_kernel(const GradTable t, int chunk, const float* __restrict__ norm,
                                                       double max_norm) {
  const float c = clip_factor(norm, max_norm);
  if (c == 1.0f) return;  // times one: nothing changes
  const int k = owner(t, blockIdx.x);
  const int64_t lo = (int64_t)(blockIdx.x - t.first[k]) * chunk;
  if (t.dtype[k] == PMG_F32) scale_chunk((float*)t.g[k], t.n_el[k], lo, chunk, c);
  else if (t.dtype[k] == PMG_BF16) scale_chunk((bf16_t*)t.g[k], t.n_el[k], lo, chunk, c);
  else scale_chunk((f16_t*)t.g[k], t.n_el[k], lo, chunk, c);
}

// Elements a workgroup takes: 16384 (64 a thread: enough loads in flight, few partial sums); a quarter of
// the chip's worth of chunks or less, 2048, so that a small model's gradients spread over more CUs.
int norm_chunk(const int64_t* numel, int n) {
  int64_t total = 0;
  for (int i = 0; i < n; ++i) total += numel[i];
  return total >= (int64_t)16384 * 256 ? 16384 : 2048;
}

int grad_args_ok(const void* const* g, const int64_t* numel, const int* dtype, int n) {
  if (n < 0) return PMG_E_ARG;
  if (n > 0 && (!g || !numel || !dtype)) return PMG_E_NULL;
  for (int i = 0; i < n; ++i) {
    if (numel[i] < 0 || numel[i] > ((int64_t)1 << 40)) return PMG_E_ARG;
    if (!pmg_dtype_ok(dtype[i])) return PMG_E_DTYPE;
    if (numel[i] > 0 && !g[i]) return PMG_E_NULL;
    if ((uintptr_t)g[i] & (pmg_elem_bytes(dtype[i]) - 1)) return PMG_E_ALIGN;
  }
  return PMG_OK;
}

struct Range {
  uintptr_t lo, hi;
  int written;
};

// PMG_OK if no written range meets another one (read-only ranges may overlap each other).
int check_disjoint(Range* r, int n) {
  std::sort(r, r + n, [](const Range& a, const Range& b) { return a.lo < b.lo; });
  uintptr_t end = 0, wend = 0;  // furthest end so far: of any range, of a written one
  for (int i = 0; i < n; ++i) {
    if (r[i].lo < (r[i].written ? end : wend)) return PMG_E_OVERLAP;
    end = std::max(end, r[i].hi);
    if (r[i].written) wend = std::max(wend, r[i].hi);
  }
  return PMG_OK;
}

// Calls launch(table, chunks, base) for runs of at most MAX tensors; empty tensors take no place.
template <typename Table, int MAX, typename Fill, typename Launch>
void batches(const int64_t* numel, int n, int chunk, Fill fill, Launch launch) {
  Table t;
  t.n = 0;
  int chunks = 0, base = 0;
  for (int i = 0; i < n; ++i) {
    if (numel[i] > 0) {
      const int64_t c = (numel[i] + chunk - 1) / chunk;
      fill(t, t.n, i);
      t.n_el[t.n] = numel[i];
      t.first[t.n] = chunks;
      ++t.n;
      chunks += (int)c;
    }
    if (t.n == MAX || (i == n - 1 && t.n > 0)) {
      launch(t, chunks, base);
      base += chunks;
      t.n = 0;
      chunks = 0;
    }
  }
}

// ------------------------------------------------------------------------------------------------ AdamW
constexpr int AW_MAX = 56;
struct AdamwTable {
  void* p[AW_MAX];
  const void* g[AW_MAX];
  void* m[AW_MAX];
  void* v[AW_MAX];
  float* mt[AW_MAX];
  float* vt[AW_MAX];
  float* w[AW_MAX];
  int64_t n_el[AW_MAX];
  int first[AW_MAX];
  int n;
};
struct AdamwConst {
  float b1, c1, b2, c2, eps, wd;  // c = 1 - b, rounded from fp64
  int decoupled;
};
static_assert(sizeof(AdamwTable) + sizeof(AdamwConst) + 16 <= 4096, "kernel arguments");

// What depends on the step, the learning rate and the norm, once for the whole update.
struct AdamwScalars {
  float rate, root, factor, keep;
};

__global__ void adamw_prep_kernel(int64_t* step, const float* lr_dev, const float* norm, double lr, double b1, double b2,
                                  double wd, double max_norm, int decoupled, AdamwScalars* out) {
  if (threadIdx.x != 0) return;
  const int64_t t = step[0] + 1;
  step[0] = t;
  const double rate = lr_dev ? (double)lr_dev[0] : lr;
  out->rate = (float)(rate / (1.0 - pow(b1, (double)t)));
  out->root = (float)(1.0 / sqrt(1.0 - pow(b2, (double)t)));
  out->factor = norm ? clip_factor(norm, max_norm) : 1.0f;
  out->keep = decoupled ? (float)(1.0 - rate * wd) : 1.0f;
}

// The largest magnitude over the wave's 256 values; as unsigned integers, so that a NaN wins.
__device__ __forceinline__ float wave_top(f32x4 x) {
  unsigned a = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) a = max(a, __float_as_uint(x[j]) & 0x7fffffffu);
  for (int o = 32; o > 0; o >>= 1) a = max(a, (unsigned)__shfl_xor((int)a, o, 64));
  return __uint_as_float(a);
}

__device__ __forceinline__ float share_of(float top) {
  return top >= 1.17549435e-38f ? 1.0f / top : 0.0f;  // a NaN fails the comparison
}

constexpr int AW_ITER = 4;
constexpr int AW_CHUNK = THREADS * 4 * AW_ITER;  // 4096 elements a workgroup: 16 a thread, all loads in flight at once

__device__ __forceinline__ f32x4 decode_m(int c4, float top) {
#pragma clang fp contract(off)
  f32x4 x;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float c = (float)(int8_t)(c4 >> (8 * j)) * (1.0f / 127.0f);
    x[j] = (c * fabsf(c)) * top;
  }
  return x;
}
__device__ __forceinline__ f32x4 decode_v(int c4, float top) {
#pragma clang fp contract(off)
  f32x4 x;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float c = (float)(uint8_t)(c4 >> (8 * j)) * (1.0f / 255.0f);
    c = c * c;
    x[j] = (c * c) * top;
  }
  return x;
}
__device__ __forceinline__ int encode_m(f32x4 x, float share) {
#pragma clang fp contract(off)
  int c4 = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float q = rintf(sqrtf(fabsf(x[j]) * share) * 127.0f);
    q = q == q ? q : 0.0f;
    c4 |= ((int)copysignf(q, x[j]) & 0xff) << (8 * j);
  }
  return c4;
}
__device__ __forceinline__ int encode_v(f32x4 x, float share) {
#pragma clang fp contract(off)
  int c4 = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float q = rintf(sqrtf(sqrtf(x[j] * share)) * 255.0f);
    q = q == q ? q : 0.0f;
    if (x[j] > 0.0f) q = fmaxf(q, 1.0f);
    c4 |= (int)q << (8 * j);
  }
  return c4;
}

typedef int __attribute__((aligned(1))) codes4;
__device__ __forceinline__ int load_codes(const uint8_t* p, int64_t left) {
  if (left >= 4) return *reinterpret_cast<const codes4*>(p);
  int c = 0;
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (j < left) c |= (int)p[j] << (8 * j);
  return c;
}
__device__ __forceinline__ void store_codes(uint8_t* p, int c, int64_t left) {
  if (left >= 4) {
    *reinterpret_cast<codes4*>(p) = c;
    return;
  }
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (j < left) p[j] = (uint8_t)(c >> (8 * j));
}

// One chunk of one tensor.  A wave's 64 x 4 consecutive elements are one block of an 8-bit state, so its
// scale is a reduction within the wave.  Products, sums, quotients and roots are rounded one by one (no
// contraction), as the formulas of pmg_lm.h are written: an 8-bit code near the border of two is then the
// same wherever these formulas are evaluated in fp32.
template <typename P, typename G, int BITS>
__global__ __launch_bounds__(THREADS) void adamw_kernel(const AdamwTable t, const AdamwConst k,
                                                        const AdamwScalars* __restrict__ sc) {
#pragma clang fp contract(off)
  const int i = owner(t, blockIdx.x);
  const int64_t n = t.n_el[i];
  const int64_t lo = (int64_t)(blockIdx.x - t.first[i]) * AW_CHUNK + threadIdx.x * 4;
  P* __restrict__ p = (P*)t.p[i];
  const G* __restrict__ g = (const G*)t.g[i];
  float* __restrict__ w = t.w[i];
  const float rate = sc->rate, root = sc->root, factor = sc->factor, keep = sc->keep;

  f32x4 gx[AW_ITER], px[AW_ITER], mx[AW_ITER], vx[AW_ITER];
  int mc[AW_ITER], vc[AW_ITER];
  float mt[AW_ITER], vt[AW_ITER];
#pragma unroll
  for (int u = 0; u < AW_ITER; ++u) {
    const int64_t e = lo + u * (THREADS * 4), left = n - e;
    gx[u] = px[u] = mx[u] = vx[u] = f32x4{0.f, 0.f, 0.f, 0.f};
    mc[u] = vc[u] = 0;
    mt[u] = vt[u] = 0.0f;
    if (left > 0) {
      gx[u] = pmg_load4(g + e, left);
      px[u] = w ? pmg_load4(w + e, left) : pmg_load4(p + e, left);
      if (BITS == 32) {
        mx[u] = pmg_load4((const float*)t.m[i] + e, left);
        vx[u] = pmg_load4((const float*)t.v[i] + e, left);
      } else {
        mc[u] = load_codes((const uint8_t*)t.m[i] + e, left);
        vc[u] = load_codes((const uint8_t*)t.v[i] + e, left);
        mt[u] = t.mt[i][e / PMG_STATE_BLOCK];
        vt[u] = t.vt[i][e / PMG_STATE_BLOCK];
      }
    }
  }
#pragma unroll
  for (int u = 0; u < AW_ITER; ++u) {
    const int64_t e = lo + u * (THREADS * 4), left = n - e;
    f32x4 m, v, x;
    if (BITS == 8) {
      mx[u] = decode_m(mc[u], mt[u]);
      vx[u] = decode_v(vc[u], vt[u]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float gj = gx[u][j] * factor;
      if (!k.decoupled) gj = gj + k.wd * px[u][j];
      m[j] = mx[u][j] * k.b1 + gj * k.c1;
      v[j] = vx[u][j] * k.b2 + (gj * gj) * k.c2;
      const float move = (m[j] * rate) / (sqrtf(v[j]) * root + k.eps);
      x[j] = px[u][j] * keep - move;
    }
    if (BITS == 8) {
      // elements behind the tensor's end take no part in the scale
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j >= left) m[j] = v[j] = 0.0f;
      const float top_m = wave_top(m), top_v = wave_top(v);
      if (left > 0) {
        store_codes((uint8_t*)t.m[i] + e, encode_m(m, share_of(top_m)), left);
        store_codes((uint8_t*)t.v[i] + e, encode_v(v, share_of(top_v)), left);
        if ((threadIdx.x & 63) == 0) {
          t.mt[i][e / PMG_STATE_BLOCK] = top_m;
          t.vt[i][e / PMG_STATE_BLOCK] = top_v;
        }
      }
    }
    if (left > 0) {
      if (BITS == 32) {
        pmg_store4((float*)t.m[i] + e, m, left);
        pmg_store4((float*)t.v[i] + e, v, left);
      }
      if (w) pmg_store4(w + e, x, left);
      pmg_store4(p + e, x, left);
    }
  }
}

template <bool SIGNED>
__global__ __launch_bounds__(THREADS) void values_kernel(const uint8_t* __restrict__ code, const float* __restrict__ top,
                                                         int64_t n, float* __restrict__ out) {
  const int64_t lo = (int64_t)blockIdx.x * AW_CHUNK + threadIdx.x * 4;
#pragma unroll
  for (int u = 0; u < AW_ITER; ++u) {
    const int64_t e = lo + u * (THREADS * 4), left = n - e;
    if (left <= 0) break;
    const int c = load_codes(code + e, left);
    const float s = top[e / PMG_STATE_BLOCK];
    pmg_store4(out + e, SIGNED ? decode_m(c, s) : decode_v(c, s), left);
  }
}

template <typename P, typename G>
void launch_adamw(const AdamwTable& t, const AdamwConst& k, const AdamwScalars* sc, int bits, int chunks, hipStream_t st) {
  if (bits == 32) hipLaunchKernelGGL((adamw_kernel<P, G, 32>), dim3(chunks), dim3(THREADS), 0, st, t, k, sc);
  else hipLaunchKernelGGL((adamw_kernel<P, G, 8>), dim3(chunks), dim3(THREADS), 0, st, t, k, sc);
}

}  // namespace

extern "C" int pmg_grad_norm_workspace(const int64_t* numel, int n, size_t* out) {
  if (!out || (n > 0 && !numel)) return PMG_E_NULL;
  if (n < 0) return PMG_E_ARG;
  const int chunk = norm_chunk(numel, n);
  size_t chunks = 1;
  for (int i = 0; i < n; ++i) {
    if (numel[i] < 0 || numel[i] > ((int64_t)1 << 40)) return PMG_E_ARG;
    chunks += (size_t)((numel[i] + chunk - 1) / chunk);
  }
  if (chunks > (size_t)MOST_GROUPS) return PMG_E_ARG;
  *out = chunks * sizeof(double);
  return PMG_OK;
}

extern "C" int pmg_grad_norm(const void* const* grads, const int64_t* numel, const int* dtype, int n, float* norm,
                             void* ws, pmg_stream stream) {
  if (!norm || !ws) return PMG_E_NULL;
  const int rc = grad_args_ok(grads, numel, dtype, n);
  if (rc) return rc;
  size_t need;
  if (const int e = pmg_grad_norm_workspace(numel, n, &need)) return e;
  if ((uintptr_t)ws & 15) return PMG_E_ALIGN;
  hipStream_t st = (hipStream_t)stream;
  const int chunk = norm_chunk(numel, n);
  double* part = (double*)ws;
  int total = 0;
  batches<GradTable, GT_MAX>(
      numel, n, chunk,
      [&](GradTable& t, int k, int i) {
        t.g[k] = const_cast<void*>(grads[i]);
        t.dtype[k] = (uint8_t)dtype[i];
      },
      [&](const GradTable& t, int chunks, int base) {
        hipLaunchKernelGGL(norm_part_kernel, dim3(chunks), dim3(THREADS), 0, st, t, chunk, base, part);
        total = base + chunks;
      });
  hipLaunchKernelGGL(norm_join_kernel, dim3(1), dim3(1024), 0, st, part, total, norm);
  return (int)hipGetLastError();
}

extern "C" int pmg_grad_clip_check(void* const* grads, const int64_t* numel, const int* dtype, int n, float max_norm) {
  if (!(max_norm > 0.0f)) return PMG_E_ARG;
  const int rc = grad_args_ok((const void* const*)grads, numel, dtype, n);
  if (rc) return rc;
  size_t need;
  if (const int e = pmg_grad_norm_workspace(numel, n, &need)) return e;  // chunks within a launch's reach
  if (n == 0) return PMG_OK;
  Range* r = new (std::nothrow) Range[n];
  if (!r) return PMG_E_ARG;
  int nr = 0;
  for (int i = 0; i < n; ++i)  // an empty tensor has no elements to share, wherever it points
    if (numel[i] > 0) r[nr++] = Range{(uintptr_t)grads[i], (uintptr_t)grads[i] + (size_t)numel[i] * pmg_elem_bytes(dtype[i]), 1};
  const int ov = check_disjoint(r, nr);
  delete[] r;
  return ov;
}

extern "C" int pmg_grad_clip(void* const* grads, const int64_t* numel, const int* dtype, int n, const float* norm,
                             float max_norm, pmg_stream stream) {
  if (!norm) return PMG_E_NULL;
  if (const int rc = pmg_grad_clip_check(grads, numel, dtype, n, max_norm)) return rc;
  hipStream_t st = (hipStream_t)stream;
  const int chunk = norm_chunk(numel, n);
  batches<GradTable, GT_MAX>(
      numel, n, chunk,
      [&](GradTable& t, int k, int i) {
        t.g[k] = grads[i];
        t.dtype[k] = (uint8_t)dtype[i];
      },
      [&](const GradTable& t, int chunks, int) {
        hipLaunchKernelGGL(clip_kernel, dim3(chunks), dim3(THREADS), 0, st, t, chunk, norm, (double)max_norm);
      });
  return (int)hipGetLastError();
}

extern "C" int pmg_adamw_step(const pmg_adamw* a, void* ws, pmg_stream stream) {
  if (!a || !ws || !a->step) return PMG_E_NULL;
  if (a->n < 0) return PMG_E_ARG;
  if (a->n > 0 && (!a->numel || !a->param || !a->grad || !a->m || !a->v)) return PMG_E_NULL;
  if (a->state_bits != 32 && a->state_bits != 8) return PMG_E_ARG;
  if (a->state_bits == 8 && a->n > 0 && (!a->m_top || !a->v_top)) return PMG_E_NULL;
  if (!pmg_dtype_ok(a->dtype)) return PMG_E_DTYPE;
  if (a->grad_dtype != a->dtype && a->grad_dtype != PMG_F32) return PMG_E_DTYPE;
  if (a->master && a->dtype == PMG_F32) return PMG_E_DTYPE;
  if (!(a->beta1 >= 0 && a->beta1 < 1 && a->beta2 >= 0 && a->beta2 < 1 && a->eps >= 0 && a->lr >= 0 && a->weight_decay >= 0))
    return PMG_E_ARG;
  if (a->norm && !(a->max_norm > 0)) return PMG_E_ARG;
  if (((uintptr_t)ws & 15) || ((uintptr_t)a->step & 7)) return PMG_E_ALIGN;
  const bool q = a->state_bits == 8;
  const size_t pb = pmg_elem_bytes(a->dtype), gb = pmg_elem_bytes(a->grad_dtype), sb = q ? 1 : 4;
  int64_t chunks_all = 0;
  for (int i = 0; i < a->n; ++i) {
    if (a->numel[i] < 0 || a->numel[i] > ((int64_t)1 << 40)) return PMG_E_ARG;
    if (a->numel[i] == 0) continue;
    chunks_all += (a->numel[i] + AW_CHUNK - 1) / AW_CHUNK;
    if (!a->param[i] || !a->grad[i] || !a->m[i] || !a->v[i] || (q && (!a->m_top[i] || !a->v_top[i])) ||
        (a->master && !a->master[i]))
      return PMG_E_NULL;
    uintptr_t bad = ((uintptr_t)a->param[i] & (pb - 1)) | ((uintptr_t)a->grad[i] & (gb - 1));
    bad |= ((uintptr_t)a->m[i] | (uintptr_t)a->v[i]) & (sb - 1);
    if (q) bad |= ((uintptr_t)a->m_top[i] | (uintptr_t)a->v_top[i]) & 3;
    if (a->master) bad |= (uintptr_t)a->master[i] & 3;
    if (bad) return PMG_E_ALIGN;
  }
  if (chunks_all > MOST_GROUPS) return PMG_E_ARG;
  Range* r = new (std::nothrow) Range[(size_t)a->n * 7 + 4];
  if (!r) return PMG_E_ARG;
  int nr = 0;
  auto add = [&](const void* p, size_t bytes, int written) {
    r[nr++] = Range{(uintptr_t)p, (uintptr_t)p + bytes, written};
  };
  add(a->step, 8, 1);
  add(ws, PMG_ADAMW_WS, 1);
  if (a->lr_dev) add(a->lr_dev, 4, 0);
  if (a->norm) add(a->norm, 4, 0);
  for (int i = 0; i < a->n; ++i) {
    const size_t n = (size_t)a->numel[i], nb = (n + PMG_STATE_BLOCK - 1) / PMG_STATE_BLOCK;
    if (n == 0) continue;
    add(a->param[i], n * pb, 1);
    add(a->grad[i], n * gb, 0);
    add(a->m[i], n * sb, 1);
    add(a->v[i], n * sb, 1);
    if (q) {
      add(a->m_top[i], nb * 4, 1);
      add(a->v_top[i], nb * 4, 1);
    }
    if (a->master) add(a->master[i], n * 4, 1);
  }
  const int ov = check_disjoint(r, nr);
  delete[] r;
  if (ov) return ov;

  hipStream_t st = (hipStream_t)stream;
  AdamwScalars* sc = (AdamwScalars*)ws;
  hipLaunchKernelGGL(adamw_prep_kernel, dim3(1), dim3(64), 0, st, a->step, a->lr_dev, a->norm, a->lr, a->beta1, a->beta2,
                     a->weight_decay, a->max_norm, a->decoupled, sc);
  const AdamwConst k = {(float)a->beta1, (float)(1.0 - a->beta1), (float)a->beta2, (float)(1.0 - a->beta2),
                        (float)a->eps, (float)a->weight_decay, a->decoupled};
  batches<AdamwTable, AW_MAX>(
      a->numel, a->n, AW_CHUNK,
      [&](AdamwTable& t, int j, int i) {
        t.p[j] = a->param[i];
        t.g[j] = a->grad[i];
        t.m[j] = a->m[i];
        t.v[j] = a->v[i];
        t.mt[j] = q ? a->m_top[i] : nullptr;
        t.vt[j] = q ? a->v_top[i] : nullptr;
        t.w[j] = a->master ? a->master[i] : nullptr;
      },
      [&](const AdamwTable& t, int chunks, int) {
        if (a->dtype == PMG_F32) launch_adamw<float, float>(t, k, sc, a->state_bits, chunks, st);
        else if (a->dtype == PMG_BF16 && a->grad_dtype == PMG_BF16) launch_adamw<bf16_t, bf16_t>(t, k, sc, a->state_bits, chunks, st);
        else if (a->dtype == PMG_BF16) launch_adamw<bf16_t, float>(t, k, sc, a->state_bits, chunks, st);
        else if (a->grad_dtype == PMG_F16) launch_adamw<f16_t, f16_t>(t, k, sc, a->state_bits, chunks, st);
        else launch_adamw<f16_t, float>(t, k, sc, a->state_bits, chunks, st);
      });
  return (int)hipGetLastError();
}

extern "C" int pmg_adamw_values(const void* code, const float* top, int64_t numel, int is_signed, float* out,
                                pmg_stream stream) {
  if (numel < 0 || numel > MOST_GROUPS * AW_CHUNK) return PMG_E_ARG;
  if (numel == 0) return PMG_OK;
  if (!code || !top || !out) return PMG_E_NULL;
  if (((uintptr_t)top | (uintptr_t)out) & 3) return PMG_E_ALIGN;
  const dim3 grid((unsigned)((numel + AW_CHUNK - 1) / AW_CHUNK));
  hipStream_t st = (hipStream_t)stream;
  if (is_signed) hipLaunchKernelGGL(values_kernel<true>, grid, dim3(THREADS), 0, st, (const uint8_t*)code, top, numel, out);
  else hipLaunchKernelGGL(values_kernel<false>, grid, dim3(THREADS), 0, st, (const uint8_t*)code, top, numel, out);
  return (int)hipGetLastError();
}
