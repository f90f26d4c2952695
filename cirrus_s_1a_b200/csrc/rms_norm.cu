// RMSNorm of rows, and its gradient.
//
//   y = x r w, r = (mean x^2 + eps)^-1/2
//   dx = r (g w - x r mean(g w x r))          dw = sum over rows of g x r
//
// Bound by memory: a row is read once and held in the registers of a warp, or where rows are
// few or long of a CTA, while its sums are taken.  The gradient's warps or CTAs go through
// rows in turn and add their part of dw up as they do; the parts of a CTA's warps, then of the
// CTAs, are added in order, so that the sum does not depend on timing.  Rows that are not
// 16-byte aligned are taken by single elements.  Rows too long to be held (more than 8192
// columns, 4096 of single elements) are read twice, with dw over fixed groups of rows.
// Measured, 65537 x 1024 in float32: 78 us (6.9 TB/s) and, the gradient, 125 us (6.4 TB/s);
// 16384 x 768 in bf16, both, 33 us; 16384 x 4096 in bf16, both, 139 us (4.8 TB/s), x 769 63 us.
#include <algorithm>
#include <type_traits>

#include "ends.cuh"

namespace cb {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kGroup = 64;  // rows whose part of dw one CTA sums (rows taken by CTAs)

// A thread's elements of w beside VEC of x.
template <typename W, int VEC>
__device__ __forceinline__ void load_w(const W* w, float (&o)[VEC]) {
  constexpr int kN = std::min(VEC, 16 / (int)sizeof(W));
#pragma unroll
  for (int i = 0; i < VEC; i += kN) {
    const Vec<W, kN> v = *reinterpret_cast<const Vec<W, kN>*>(w + i);
#pragma unroll
    for (int k = 0; k < kN; ++k) o[i + k] = Elem<W>::get(v.v[k]);
  }
}

// A warp to a row: NV pieces of VEC elements a lane, 16 bytes or one element.
template <typename T, typename W, int VEC, int NV>
__global__ void __launch_bounds__(kThreads) rms_norm_warp_kernel(const T* x, int64_t ld, const W* w, int rows, int d,
                                                                 float eps, T* y) {
  const int lane = threadIdx.x & 31, n = blockIdx.x * kWarps + (threadIdx.x >> 5);
  await_before();
  start_next();
  if (n >= rows) return;
  Vec<T, VEC> v[NV];
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = (i * 32 + lane) * VEC;
    if (j < d) v[i] = *reinterpret_cast<const Vec<T, VEC>*>(x + n * ld + j);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if ((i * 32 + lane) * VEC < d)
#pragma unroll
      for (int k = 0; k < VEC; ++k) s += Elem<T>::get(v[i].v[k]) * Elem<T>::get(v[i].v[k]);
  const float r = rsqrtf(warp_sum(s) / d + eps);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = (i * 32 + lane) * VEC;
    if (j >= d) continue;
    float u[VEC];
    load_w<W, VEC>(w + j, u);
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[i].v[k] = Elem<T>::put(Elem<T>::get(v[i].v[k]) * r * u[k]);
    *reinterpret_cast<Vec<T, VEC>*>(y + (int64_t)n * d + j) = v[i];
  }
}

// part[cta][d]
template <typename T, typename W, int VEC, int NV>
__global__ void __launch_bounds__(kThreads) rms_norm_grad_warp_kernel(const T* x, int64_t ld, const T* g, int64_t ldg,
                                                                      const W* w, int rows, int d, float eps, T* dx,
                                                                      float* part) {
  constexpr int kWide = NV * VEC * 32;   // columns of NV pieces a lane, d of them or more
  __shared__ float s_part[kWarps / 2][kWide];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float acc[NV][VEC] = {};
  await_before();
  start_next();
  for (int n = blockIdx.x * kWarps + warp; n < rows; n += gridDim.x * kWarps) {
    Vec<T, VEC> v[NV], up[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * 32 + lane) * VEC;
      if (j < d) {
        v[i] = *reinterpret_cast<const Vec<T, VEC>*>(x + n * ld + j);
        up[i] = *reinterpret_cast<const Vec<T, VEC>*>(g + n * ldg + j);
      }
    }
    float s = 0.0f, c = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * 32 + lane) * VEC;
      if (j >= d) continue;
      float u[VEC];
      load_w<W, VEC>(w + j, u);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float a = Elem<T>::get(v[i].v[k]);
        s += a * a;
        c += Elem<T>::get(up[i].v[k]) * u[k] * a;
      }
    }
    const float r = rsqrtf(warp_sum(s) / d + eps);
    const float m = warp_sum(c) * r / d * r;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * 32 + lane) * VEC;
      if (j >= d) continue;
      float u[VEC];
      load_w<W, VEC>(w + j, u);
      Vec<T, VEC> o;
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float a = Elem<T>::get(v[i].v[k]), b = Elem<T>::get(up[i].v[k]);
        o.v[k] = Elem<T>::put(r * (b * u[k] - a * m));
        acc[i][k] += b * (a * r);
      }
      *reinterpret_cast<Vec<T, VEC>*>(dx + (int64_t)n * d + j) = o;
    }
  }
  // the warps' parts, halved until one is left
  for (int half = kWarps / 2; half > 0; half /= 2) {
    __syncthreads();
    if (warp >= half && warp < 2 * half)
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k)
          s_part[warp - half][(i * VEC + k) * 32 + lane] = acc[i][k];
    __syncthreads();
    if (warp < half)
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k)
          acc[i][k] += s_part[warp][(i * VEC + k) * 32 + lane];
  }
  if (warp > 0) return;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const int j = (i * 32 + lane) * VEC + k;
      if (j < d) part[(int64_t)blockIdx.x * d + j] = acc[i][k];
    }
}

// dw = the sum of `parts` rows: 32 columns a CTA, its warps' sums added in order.
template <typename W>
__global__ void __launch_bounds__(1024) rms_norm_dw_kernel(const float* part, int parts, int d, W* dw) {
  __shared__ float s_sum[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = blockIdx.x * 32 + lane;
  float s[4] = {};
  await_before();
  start_next();
  if (j < d) {
    int i = warp;
    for (; i + 96 < parts; i += 128)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k] += part[(int64_t)(i + 32 * k) * d + j];
    for (; i < parts; i += 32) s[0] += part[(int64_t)i * d + j];
  }
  s_sum[warp][lane] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (warp == 0 && j < d) {
    float t = 0.0f;
    for (int k = 0; k < 32; ++k) t += s_sum[k][lane];
    dw[j] = Elem<W>::put(t);
  }
}

// A CTA to a row that it holds: NV pieces of VEC elements a thread.
template <typename T, typename W, int VEC, int NV>
__global__ void __launch_bounds__(kThreads) rms_norm_cta_kernel(const T* x, int64_t ld, const W* w, int d, float eps,
                                                                T* y) {
  __shared__ float red[33];
  await_before();
  start_next();
  Vec<T, VEC> v[NV];
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = (i * kThreads + threadIdx.x) * VEC;
    if (j < d) v[i] = *reinterpret_cast<const Vec<T, VEC>*>(x + blockIdx.x * ld + j);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if ((i * kThreads + threadIdx.x) * VEC < d)
#pragma unroll
      for (int k = 0; k < VEC; ++k) s += Elem<T>::get(v[i].v[k]) * Elem<T>::get(v[i].v[k]);
  const float r = rsqrtf(block_sum(s, red) / d + eps);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = (i * kThreads + threadIdx.x) * VEC;
    if (j >= d) continue;
    float u[VEC];
    load_w<W, VEC>(w + j, u);
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[i].v[k] = Elem<T>::put(Elem<T>::get(v[i].v[k]) * r * u[k]);
    *reinterpret_cast<Vec<T, VEC>*>(y + (int64_t)blockIdx.x * d + j) = v[i];
  }
}

// CTAs take rows in turn, row_ctas (for so many columns a thread) to an SM: 16384 x 4096 in bf16
// 139 us, 160 with registers for three.  (Four leave 64 registers a thread, of which 16 columns
// spill 16 to 48 bytes: seven forms.)  part[cta][d]
constexpr int row_ctas(int columns) { return columns <= 16 ? 4 : 2; }
template <typename T, typename W, int VEC, int NV>
__global__ void __launch_bounds__(kThreads, row_ctas(NV * VEC))
    rms_norm_grad_cta_kernel(const T* x, int64_t ld, const T* g, int64_t ldg, const W* w, int rows, int d, float eps, T* dx,
                             float* part) {
  __shared__ float2 s_sum[2][kWarps];  // one is read while the next row's is written
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float acc[NV][VEC] = {};
  int which = 0;
  await_before();
  start_next();
  // The next row is on its way meanwhile where registers allow (16384 x 2047 in float32 131 us,
  // with it 114; 16 columns a thread: x 4096 213 and 284).
  constexpr bool kNext = NV * VEC <= 8;
  Vec<T, VEC> v[NV], up[NV], next_v[kNext ? NV : 1], next_up[kNext ? NV : 1];
  auto load = [&](int n, auto& to_v, auto& to_up) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * kThreads + threadIdx.x) * VEC;
      if (n < rows && j < d) {
        to_v[i] = *reinterpret_cast<const Vec<T, VEC>*>(x + n * ld + j);
        to_up[i] = *reinterpret_cast<const Vec<T, VEC>*>(g + n * ldg + j);
      }
    }
  };
  if constexpr (kNext) load(blockIdx.x, next_v, next_up);
  for (int n = blockIdx.x; n < rows; n += gridDim.x, which ^= 1) {
    if constexpr (kNext) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        v[i] = next_v[i];
        up[i] = next_up[i];
      }
      load(n + gridDim.x, next_v, next_up);
    } else {
      load(n, v, up);
    }
    float s = 0.0f, c = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * kThreads + threadIdx.x) * VEC;
      if (j >= d) continue;
      float u[VEC];
      load_w<W, VEC>(w + j, u);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float a = Elem<T>::get(v[i].v[k]);
        s += a * a;
        c += Elem<T>::get(up[i].v[k]) * u[k] * a;
      }
    }
    s = warp_sum(s);
    c = warp_sum(c);
    if (lane == 0) s_sum[which][warp] = make_float2(s, c);
    __syncthreads();
    s = c = 0.0f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) {
      s += s_sum[which][k].x;
      c += s_sum[which][k].y;
    }
    const float r = rsqrtf(s / d + eps), m = c * r / d * r;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * kThreads + threadIdx.x) * VEC;
      if (j >= d) continue;
      float u[VEC];
      load_w<W, VEC>(w + j, u);
      Vec<T, VEC> o;
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float a = Elem<T>::get(v[i].v[k]), b = Elem<T>::get(up[i].v[k]);
        o.v[k] = Elem<T>::put(r * (b * u[k] - a * m));
        acc[i][k] += b * (a * r);
      }
      *reinterpret_cast<Vec<T, VEC>*>(dx + (int64_t)n * d + j) = o;
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const int j = (i * kThreads + threadIdx.x) * VEC + k;
      if (j < d) part[(int64_t)blockIdx.x * d + j] = acc[i][k];
    }
}

// Rows of any length, read twice.
template <typename T, typename W>
__global__ void __launch_bounds__(kThreads) rms_norm_kernel(const T* x, int64_t ld, const W* w, int d, float eps, T* y) {
  __shared__ float red[33];
  await_before();
  start_next();
  const T* row = x + blockIdx.x * ld;
  float s = 0.0f;
  for (int j = threadIdx.x; j < d; j += kThreads) {
    const float v = Elem<T>::get(row[j]);
    s += v * v;
  }
  const float r = rsqrtf(block_sum(s, red) / d + eps);
  for (int j = threadIdx.x; j < d; j += kThreads)
    y[(int64_t)blockIdx.x * d + j] = Elem<T>::put(Elem<T>::get(row[j]) * r * Elem<W>::get(w[j]));
}

template <typename T, typename W>
__global__ void __launch_bounds__(kThreads) rms_norm_dx_kernel(const T* x, int64_t ld, const T* g, int64_t ldg,
                                                               const W* w, int d, float eps, T* dx, float* rstd) {
  __shared__ float red[33];
  await_before();
  start_next();
  const T* row = x + blockIdx.x * ld;
  const T* up = g + blockIdx.x * ldg;
  float s = 0.0f, c = 0.0f;
  for (int j = threadIdx.x; j < d; j += kThreads) {
    const float v = Elem<T>::get(row[j]);
    s += v * v;
    c += Elem<T>::get(up[j]) * Elem<W>::get(w[j]) * v;
  }
  const float r = rsqrtf(block_sum(s, red) / d + eps);
  const float m = block_sum(c, red) * r / d * r;
  if (threadIdx.x == 0) rstd[blockIdx.x] = r;
  for (int j = threadIdx.x; j < d; j += kThreads)
    dx[(int64_t)blockIdx.x * d + j] =
        Elem<T>::put(r * (Elem<T>::get(up[j]) * Elem<W>::get(w[j]) - Elem<T>::get(row[j]) * m));
}

template <typename T>
__global__ void __launch_bounds__(kThreads) rms_norm_dw_part_kernel(const T* x, int64_t ld, const T* g, int64_t ldg,
                                                                    const float* rstd, int rows, int d, float* part) {
  const int j = blockIdx.y * kThreads + threadIdx.x;
  await_before();
  start_next();
  if (j >= d) return;
  const int64_t from = (int64_t)blockIdx.x * kGroup;
  const int64_t to = min(from + kGroup, (int64_t)rows);
  float s = 0.0f;
  for (int64_t n = from; n < to; ++n) s += Elem<T>::get(g[n * ldg + j]) * (Elem<T>::get(x[n * ld + j]) * rstd[n]);
  part[(int64_t)blockIdx.x * d + j] = s;
}

// Whether a row's pieces can be 16 bytes.
bool in_pieces(const void* x, int64_t ld, int rows, int d, int size) {
  return d * size % 16 == 0 && aligned_to(x, 16) && (rows == 1 || ld * size % 16 == 0);
}

// Whether warps take a row each: enough rows (768 columns of float32: 300 rows 2.5 us, by CTAs
// 1.8, 2400 rows 2.9 and 3.9; both directions 300 rows 7.7 and 6.5, 600 rows 8.2 and 9.9) of up
// to 4096 bytes, in the gradient 1024 columns, whose sums fill the registers (16384 x 1536 in
// bf16 87 us, by CTAs 74, in float32 140 and 93; x 1024 39 and 62, 61 and 76), and 512 of
// single elements (16384 x 255 24 us, by CTAs 61; x 769 122 and 64).
bool in_a_warp(int rows, int d, int size, bool pieces, bool grad) {
  return rows > (grad ? 3 : 6) * num_sms() && (!pieces ? d <= 512 : grad ? d <= 1024 : d * size <= 4096);
}
// Whether CTAs hold a row each.
bool in_a_cta(int d, bool pieces) { return d <= (pieces ? 8192 : 4096); }

// f(elements of a piece, pieces a thread): the first of NV that holds n pieces.
template <int VEC, int NV, int... MORE, typename F>
int first_of(int n, F&& f) {
  if constexpr (sizeof...(MORE) > 0)
    if (n > NV) return first_of<VEC, MORE...>(n, f);
  return f(std::integral_constant<int, VEC>{}, std::integral_constant<int, NV>{});
}
template <typename T, typename F>
int warp_pieces(int d, bool pieces, F&& f) {
  constexpr int VEC = 16 / sizeof(T);
  const int n = ceil_div(d, 32 * (pieces ? VEC : 1));
  if (!pieces) return first_of<1, 4, 8, 16>(n, f);
  return first_of<VEC, 1, 2, 3, 4, 6, 8>(n, f);
}
template <typename T, typename F>
int cta_pieces(int d, bool pieces, F&& f) {
  constexpr int VEC = 16 / sizeof(T);
  const int n = ceil_div(d, kThreads * (pieces ? VEC : 1));
  if (!pieces) return first_of<1, 3, 4, 6, 8, 16>(n, f);
  if constexpr (sizeof(T) == 4) return first_of<VEC, 2, 4, 8>(n, f);
  else return first_of<VEC, 1, 2, 4>(n, f);
}

// CTAs of the gradient: of warps at most two to an SM (bf16, 65537 x 768 with the forward: 103
// us, 121 with three), of those that hold a row two or four.
int warp_ctas(int rows) { return std::min(ceil_div(rows, kWarps), 2 * num_sms()); }
int row_ctas(int rows, int columns) { return std::min(rows, row_ctas(columns) * num_sms()); }

template <typename F>
int with_types(int32_t dtype, int32_t w_dtype, F&& f) {
  return with_type(dtype, [&](auto t) { return w_dtype == CB_F32 ? f(t, float{}) : f(t, t); });
}

bool bad(const void* x, int32_t dtype, int64_t ld, const void* w, int32_t w_dtype, int32_t rows, int32_t d) {
  return !x || !w || rows <= 0 || d <= 0 || ld < 0 || !is_dtype(dtype) || (w_dtype != CB_F32 && w_dtype != dtype) ||
         !aligned_to(x, dtype_size(dtype)) || !aligned_to(w, dtype_size(w_dtype));
}

}  // namespace
}  // namespace cb

using namespace cb;

extern "C" int cb_rms_norm(const void* x, int32_t dtype, int64_t ld, const void* w, int32_t w_dtype, int32_t rows,
                           int32_t d, float eps, void* y, void* stream) {
  if (bad(x, dtype, ld, w, w_dtype, rows, d) || !y || !aligned_to(y, dtype_size(dtype))) return CB_ERR_ARG;
  if (rows > CB_ENDS_MAX_ROWS || d > CB_ENDS_MAX_DIM) return CB_ERR_SHAPE;
  cudaStream_t st = (cudaStream_t)stream;
  const bool pieces = in_pieces(x, ld, rows, d, dtype_size(dtype)) && aligned_to(y, 16) && aligned_to(w, 16);
  return with_types(dtype, w_dtype, [&](auto t, auto u) {
    using T = decltype(t);
    using W = decltype(u);
    const T* in = static_cast<const T*>(x);
    const W* weight = static_cast<const W*>(w);
    if (!in_a_cta(d, pieces)) {
      return launch_after(rms_norm_kernel<T, W>, dim3(rows), kThreads, 0, st, in, ld, weight, d, eps, static_cast<T*>(y));
    }
    if (!in_a_warp(rows, d, dtype_size(dtype), pieces, false))
      return cta_pieces<T>(d, pieces, [&](auto vec, auto nv) {
        return launch_after(rms_norm_cta_kernel<T, W, decltype(vec)::value, decltype(nv)::value>, dim3(rows), kThreads, 0,
                            st, in, ld, weight, d, eps, static_cast<T*>(y));
      });
    return warp_pieces<T>(d, pieces, [&](auto vec, auto nv) {
      return launch_after(rms_norm_warp_kernel<T, W, decltype(vec)::value, decltype(nv)::value>,
                          dim3(ceil_div(rows, kWarps)), kThreads, 0, st, in, ld, weight, rows, d, eps, static_cast<T*>(y));
    });
  });
}

extern "C" size_t cb_rms_norm_grad_scratch_bytes(int32_t rows, int32_t d) {
  if (rows <= 0 || d <= 0 || rows > CB_ENDS_MAX_ROWS || d > CB_ENDS_MAX_DIM) return 0;
  return ((size_t)rows + (size_t)std::max(ceil_div(rows, kGroup), row_ctas(rows, 1)) * d) * sizeof(float);
}

extern "C" int cb_rms_norm_grad(const void* x, int32_t dtype, int64_t ld, const void* g, int64_t ldg, const void* w,
                                int32_t w_dtype, int32_t rows, int32_t d, float eps, void* dx, void* dw, void* scratch,
                                size_t scratch_bytes, void* stream) {
  if (bad(x, dtype, ld, w, w_dtype, rows, d) || !g || !dx || !dw || !scratch || ldg < 0) return CB_ERR_ARG;
  if (!aligned_to(g, dtype_size(dtype)) || !aligned_to(dx, dtype_size(dtype)) || !aligned_to(dw, dtype_size(w_dtype)) ||
      !aligned_to(scratch, 16))
    return CB_ERR_ARG;
  const size_t need = cb_rms_norm_grad_scratch_bytes(rows, d);
  if (!need) return CB_ERR_SHAPE;
  if (scratch_bytes < need) return CB_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t)stream;
  const int size = dtype_size(dtype);
  const bool pieces = in_pieces(x, ld, rows, d, size) && in_pieces(g, ldg, rows, d, size) && aligned_to(dx, 16) &&
                      aligned_to(w, 16);
  return with_types(dtype, w_dtype, [&](auto t, auto u) {
    using T = decltype(t);
    using W = decltype(u);
    const T *in = static_cast<const T*>(x), *up = static_cast<const T*>(g);
    const W* weight = static_cast<const W*>(w);
    float* rstd = static_cast<float*>(scratch);
    float* part = rstd + rows;
    int parts;
    if (in_a_warp(rows, d, size, pieces, true)) {
      part = rstd;
      parts = warp_ctas(rows);
      const int rc = warp_pieces<T>(d, pieces, [&](auto vec, auto nv) {
        return launch_after(rms_norm_grad_warp_kernel<T, W, decltype(vec)::value, decltype(nv)::value>, dim3(parts),
                            kThreads, 0, st, in, ld, up, ldg, weight, rows, d, eps, static_cast<T*>(dx), part);
      });
      if (rc) return rc;
    } else if (in_a_cta(d, pieces)) {
      part = rstd;
      const int rc = cta_pieces<T>(d, pieces, [&](auto vec, auto nv) {
        parts = row_ctas(rows, vec * nv);
        return launch_after(rms_norm_grad_cta_kernel<T, W, decltype(vec)::value, decltype(nv)::value>, dim3(parts),
                            kThreads, 0, st, in, ld, up, ldg, weight, rows, d, eps, static_cast<T*>(dx), part);
      });
      if (rc) return rc;
    } else {
      parts = ceil_div(rows, kGroup);
      if (int rc = launch_after(rms_norm_dx_kernel<T, W>, dim3(rows), kThreads, 0, st, in, ld, up, ldg, weight, d, eps,
                                static_cast<T*>(dx), rstd))
        return rc;
      if (int rc = launch_after(rms_norm_dw_part_kernel<T>, dim3(parts, ceil_div(d, kThreads)), kThreads, 0, st, in, ld,
                                up, ldg, rstd, rows, d, part))
        return rc;
    }
    return launch_after(rms_norm_dw_kernel<W>, dim3(ceil_div(d, 32)), 1024, 0, st, part, parts, d, static_cast<W*>(dw));
  });
}
