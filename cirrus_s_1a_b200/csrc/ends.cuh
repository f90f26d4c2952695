// What the operators at the ends of a model share (embedding.cu, rms_norm.cu,
// linear_ce.cu): element types, rows of a matrix, token ids.
#pragma once

#include "common.cuh"

namespace cb {

template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int code = CB_F32;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int code = CB_BF16;
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem<__half> {
  static constexpr int code = CB_F16;
  static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};

inline bool is_dtype(int32_t t) { return t == CB_F32 || t == CB_BF16 || t == CB_F16; }
inline int dtype_size(int32_t t) { return t == CB_F32 ? 4 : 2; }
inline bool aligned_to(const void* p, int64_t bytes) { return (uintptr_t)p % (uintptr_t)bytes == 0; }

// Token ids in 32 or 64 bits.
struct Ids {
  const void* p;
  int wide;
  __device__ __forceinline__ int64_t operator[](int64_t i) const {
    return wide ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
  }
};

// f(T{}) for the C type of a dtype code.
template <typename F>
int with_type(int32_t dtype, F&& f) {
  if (dtype == CB_F32) return f(float{});
  if (dtype == CB_BF16) return f(__nv_bfloat16{});
  return f(__half{});
}

inline int launched() {
  count_launch();
  return cudaGetLastError() == cudaSuccess ? CB_OK : CB_ERR_CUDA;
}

}  // namespace cb
