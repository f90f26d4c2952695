// Device helpers of the 8-bit K/V cache (kv8_*.cu) and of the log probabilities.
//
// The cache holds codes in 8 bits, [batch][kv head][slot][dim], and one scale
// for each block of kKv8Block slots and head.  A scale is a power of two, the
// smallest 2^e with absmax <= qmax * 2^e, so multiplying and dividing by it is
// exact in float32 and a code moved onto a larger scale is rounded once on a
// grid that contains the new one.  Every code (|int8| <= 127, every finite
// E4M3 value) is exact in f16, so a product with an f16 operand is exact too.
#pragma once

#include "common.cuh"

namespace cb {

constexpr int kKv8Block = CB_KV8_BLOCK;
constexpr int kKv8EMin = -100, kKv8EMax = 120;

// 2^e for -126 <= e <= 127.
__host__ __device__ __forceinline__ float kv8_pow2(int e) {
#ifdef __CUDA_ARCH__
  return __int_as_float((e + 127) << 23);
#else
  union { int i; float f; } u;
  u.i = (e + 127) << 23;
  return u.f;
#endif
}

// Exponent of a power of two in the normal range.
__device__ __forceinline__ int kv8_exponent(float s) { return (__float_as_int(s) >> 23) - 127; }

// The smallest e with absmax <= qmax * 2^e (qmax 448 = 1.75 * 2^8 for E4M3,
// 127 = 1.984375 * 2^6 for int8), within [kKv8EMin, kKv8EMax]; absmax finite, >= 0.
template <int FMT>
__device__ __forceinline__ int kv8_need(float absmax) {
  const int bits = __float_as_int(absmax);
  const int ex = (bits >> 23) - 127, mant = bits & 0x7fffff;
  const int e = FMT == CB_KV8_E4M3 ? ex - 8 + (mant > 0x600000) : ex - 6 + (mant > 0x7e0000);
  return min(max(e, kKv8EMin), kKv8EMax);
}

// y = x / scale -> code: nearest, ties to even.  Infinities saturate; a NaN is
// kept by E4M3 and becomes 0 in int8, which has none.
template <int FMT>
__device__ __forceinline__ uint32_t kv8_encode(float y) {
  if (FMT == CB_KV8_E4M3) return f32_to_e4m3(y);
  return (uint32_t)(min(max(__float2int_rn(y), -127), 127) & 0xFF);
}

template <int FMT>
__device__ __forceinline__ float kv8_decode(uint32_t b) {
  if (FMT == CB_KV8_E4M3) return e4m3_to_f32(b & 0xFF);
  return (float)(int8_t)(b & 0xFF);
}

// Waits on an mbarrier phase, at most kTimeoutNs.
constexpr unsigned long long kTimeoutNs = 200ull * 1000 * 1000;
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ unsigned long long timer_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) {
  if (mbar_try(bar, parity)) return true;
  const unsigned long long t0 = timer_ns();
  while (!mbar_try(bar, parity))
    if (timer_ns() - t0 > kTimeoutNs) return false;
  return true;
}

// 2^x to about 2^-22; 0 below 2^-126.
__device__ __forceinline__ float exp2a(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 1 / l for sums of 2^-135 to 2^115, in two factors.
struct Inverse {
  float f, inv;
  __device__ __forceinline__ explicit Inverse(float l) : f(l < 1.0f ? 4294967296.0f : 2.3283064e-10f), inv(1.0f / (l * f)) {}
  __device__ __forceinline__ float of(float o) const { return o * f * inv; }
};

// A softmax's sum l * 2^m, m = -infinity: nothing yet.  l may be 2^100 and its share of the
// whole 1, so it is scaled in two steps of half the exponent.
struct Sum {
  float m, l;
  __device__ __forceinline__ void clear() { m = -INFINITY, l = 0.0f; }
  // The root of the factor that takes what is against m to `to`.
  static __device__ __forceinline__ float half(float m, float to) { return m == -INFINITY ? 0.0f : exp2a(0.5f * (m - to)); }
  // Adds l2 * 2^m2; returns the factors that take what is against m and m2 to the new m.
  __device__ __forceinline__ float2 add(float m2, float l2) {
    const float to = fmaxf(m, m2), g = half(m, to), g2 = half(m2, to);
    l = l * g * g + l2 * g2 * g2;
    m = to;
    return make_float2(g * g, g2 * g2);
  }
};

// The larger of two; NaN if either is one.
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// The smaller of two; NaN if either is one.
__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// An attention weight, 2^x: at most 1, also where scores are too coarse to say so.
__device__ __forceinline__ float weight(float x) { return exp2a(min_nan(x, 0.0f)); }

// Pairs of floats on the packed float32 units.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pack2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// Four codes of one word -> exact f16x2 of bytes (0, 1) and (2, 3).
template <int FMT>
__device__ __forceinline__ void codes_to_h2(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (FMT == CB_KV8_E4M3) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {
    // byte u = code + 128 under the exponent of 1024: the half 1024 + u, less 1152
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __floats2half2_rn(1152.0f, 1152.0f);
    lo = h2_bits(__hsub2(bits_h2(__byte_perm(u, 0x64646464u, 0x4140)), off));
    hi = h2_bits(__hsub2(bits_h2(__byte_perm(u, 0x64646464u, 0x4342)), off));
  }
}

// Two pairs of exact code values times a power of two f <= 2^15, rounded to four
// codes.  E4M3: the f16 product is exact down to 2^-24, far below half the
// smallest code.  int8: v * f + 1536 rounds to an integer (ties to even), whose
// low byte is the code.
template <int FMT>
__device__ __forceinline__ uint32_t h2_to_codes(uint32_t lo, uint32_t hi, __half2 f) {
  if (FMT == CB_KV8_E4M3) {
    const __half2 a = __hmul2(bits_h2(lo), f), b = __hmul2(bits_h2(hi), f);
    const uint32_t x = __nv_cvt_halfraw2_to_fp8x2(__half2_raw(a), __NV_SATFINITE, __NV_E4M3);
    const uint32_t y = __nv_cvt_halfraw2_to_fp8x2(__half2_raw(b), __NV_SATFINITE, __NV_E4M3);
    return x | (y << 16);
  }
  const __half2 magic = __floats2half2_rn(1536.0f, 1536.0f);
  return __byte_perm(h2_bits(__hfma2(bits_h2(lo), f, magic)), h2_bits(__hfma2(bits_h2(hi), f, magic)), 0x6420);
}

// Element i of an array of one of the three input types.
__device__ __forceinline__ float kv8_load(const void* p, int64_t i, int dtype) {
  if (dtype == CB_F32) return static_cast<const float*>(p)[i];
  const uint32_t u = static_cast<const uint16_t*>(p)[i];
  return dtype == CB_BF16 ? bf16_to_f32(u) : __half2float(__ushort_as_half((unsigned short)u));
}

}  // namespace cb
