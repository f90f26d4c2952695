// RMSNorm of rows, and its gradient.
//
//   y = x r w, r = (mean x^2 + eps)^-1/2
//   dx = r (g w - x r mean(g w x r))          dw = sum over rows of g x r
//
// Bound by memory.  Sums are float32; dw is summed over fixed groups of rows, then over
// the groups, so that its order does not depend on timing.
#include "ends.cuh"

namespace cb {
namespace {

constexpr int kThreads = 256;
constexpr int kGroup = 64;  // rows whose part of dw one CTA sums

template <typename T, typename W>
__global__ void __launch_bounds__(kThreads) rms_norm_kernel(const T* x, int64_t ld, const W* w, int d, float eps, T* y) {
  __shared__ float red[33];
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
  if (j >= d) return;
  const int64_t from = (int64_t)blockIdx.x * kGroup;
  const int64_t to = min(from + kGroup, (int64_t)rows);
  float s = 0.0f;
  for (int64_t n = from; n < to; ++n) s += Elem<T>::get(g[n * ldg + j]) * (Elem<T>::get(x[n * ld + j]) * rstd[n]);
  part[(int64_t)blockIdx.x * d + j] = s;
}

template <typename W>
__global__ void __launch_bounds__(kThreads) rms_norm_dw_kernel(const float* part, int parts, int d, W* dw) {
  const int j = blockIdx.x * kThreads + threadIdx.x;
  if (j >= d) return;
  float s = 0.0f;
  for (int64_t i = 0; i < parts; ++i) s += part[i * d + j];
  dw[j] = Elem<W>::put(s);
}

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
  return with_types(dtype, w_dtype, [&](auto t, auto u) {
    using T = decltype(t);
    using W = decltype(u);
    rms_norm_kernel<T, W><<<rows, kThreads, 0, (cudaStream_t)stream>>>(static_cast<const T*>(x), ld,
                                                                       static_cast<const W*>(w), d, eps,
                                                                       static_cast<T*>(y));
    return launched();
  });
}

extern "C" size_t cb_rms_norm_grad_scratch_bytes(int32_t rows, int32_t d) {
  if (rows <= 0 || d <= 0 || rows > CB_ENDS_MAX_ROWS || d > CB_ENDS_MAX_DIM) return 0;
  return ((size_t)rows + (size_t)ceil_div(rows, kGroup) * d) * sizeof(float);
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
  return with_types(dtype, w_dtype, [&](auto t, auto u) {
    using T = decltype(t);
    using W = decltype(u);
    float* rstd = static_cast<float*>(scratch);
    float* part = rstd + rows;
    const int parts = ceil_div(rows, kGroup);
    rms_norm_dx_kernel<T, W><<<rows, kThreads, 0, st>>>(static_cast<const T*>(x), ld, static_cast<const T*>(g), ldg,
                                                        static_cast<const W*>(w), d, eps, static_cast<T*>(dx), rstd);
    if (int rc = launched()) return rc;
    rms_norm_dw_part_kernel<T><<<dim3(parts, ceil_div(d, kThreads)), kThreads, 0, st>>>(
        static_cast<const T*>(x), ld, static_cast<const T*>(g), ldg, rstd, rows, d, part);
    if (int rc = launched()) return rc;
    rms_norm_dw_kernel<W><<<ceil_div(d, kThreads), kThreads, 0, st>>>(part, parts, d, static_cast<W*>(dw));
    return launched();
  });
}
