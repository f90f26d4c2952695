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

// Launches a kernel as the programmatic dependent of the one before it: its blocks may
// start while that one ends, and touch memory only after await_before() (2 to 4 us less
// between two short kernels).  Every kernel of these files waits, so that a kernel's end
// implies the end of all before it.
template <typename... P, typename... A>
int launch_after(void (*fn)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, A&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, fn, static_cast<P>(args)...) != cudaSuccess) {
    (void)cudaGetLastError();
    return CB_ERR_CUDA;
  }
  count_launch();
  return CB_OK;
}
__device__ __forceinline__ void await_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Lets the next kernel's blocks start.
__device__ __forceinline__ void start_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// 16 bytes of a row, or one element where rows are not 16-byte aligned.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
  T v[VEC];
};

}  // namespace cb
