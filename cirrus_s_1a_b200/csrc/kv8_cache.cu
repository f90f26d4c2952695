// cb_kv8_append: T new tokens per sequence into the 8-bit cache.
//
// One CTA owns one (sequence, KV head, block of 64 slots) of K or of V.  It
// reads the block's new values once, keeps them in registers, reduces their
// absmax, and writes codes and the scale.  A block that already holds tokens
// keeps the larger of its scale and the one the new tokens need; its old codes
// are rewritten only when the scale grows (each is then rounded once more, onto
// a grid 2^d times as coarse).  The result does not depend on the order of
// anything: absmax is order-free and every division by a scale is exact.
// Bound by memory in principle (input once, codes once); issue slots are 73 % busy
// with widening, comparing and rounding.  Measured: 16 sequences' prompts of up to
// 8192 tokens, 2 heads of 128 dims, bf16 -> int8: 27 us = 3.7 TB/s; one token: the
// launch.  256 threads: 128 and 512 took 43 and 41 us where they took 37.
#include <type_traits>

#include "kv8.cuh"
#include "kv8_attend.cuh"

namespace cb {
namespace {

constexpr int kAT = 256;

struct AppendParams {
  CbKv8 c;
  const void* k;
  const void* v;
  int dtype, T;
  int64_t ks[3], vs[3];  // element strides between sequences, tokens, heads
  const int32_t* pos;
  const int32_t* counts;
  int32_t* status;
};

// Eight values of one token as they come, widened where they are used (16-bit types
// hold a third fewer registers that way, and more CTAs an SM).
template <typename T>
struct Eight {
  uint4 v;
  static __device__ __forceinline__ float2 widen(uint32_t w) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
      return make_float2(bf16_to_f32(w), __uint_as_float(w & 0xFFFF0000u));
    else
      return __half22float2(bits_h2(w));
  }
  template <bool VEC>
  __device__ __forceinline__ void load(const T* p) {
    if (VEC) {
      v = __ldcs(reinterpret_cast<const uint4*>(p));
    } else {
      const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
      uint32_t* w = &v.x;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = (uint32_t)u[2 * j] | (uint32_t)u[2 * j + 1] << 16;
    }
  }
  __device__ __forceinline__ float2 pair(int j) const { return widen((&v.x)[j]); }
};
template <>
struct Eight<float> {
  float4 a, b;
  template <bool VEC>
  __device__ __forceinline__ void load(const float* p) {
    if (VEC) {
      a = __ldcs(reinterpret_cast<const float4*>(p));
      b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
    } else {
      a = make_float4(p[0], p[1], p[2], p[3]);
      b = make_float4(p[4], p[5], p[6], p[7]);
    }
  }
  __device__ __forceinline__ float2 pair(int j) const {
    return j == 0 ? make_float2(a.x, a.y) : j == 1 ? make_float2(a.z, a.w) : j == 2 ? make_float2(b.x, b.y) : make_float2(b.z, b.w);
  }
};

// Eight values times 1 / s as codes.  fast (int8): every |x / s| <= 127, and x / s +
// 1.5 * 2^23 rounds to an integer (ties to even) whose low byte is the code.
template <int FMT, typename T>
__device__ __forceinline__ uint2 encode8(const Eight<T>& x, float inv, bool fast) {
  uint32_t w[2] = {0u, 0u};
  if (FMT == CB_KV8_INT8 && fast) {
    uint32_t u[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = x.pair(j);
      u[2 * j] = __float_as_uint(fmaf(f.x, inv, 12582912.0f));
      u[2 * j + 1] = __float_as_uint(fmaf(f.y, inv, 12582912.0f));
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
      w[j] = __byte_perm(__byte_perm(u[4 * j], u[4 * j + 1], 0x0040), __byte_perm(u[4 * j + 2], u[4 * j + 3], 0x0040), 0x5410);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = x.pair(j);
      if (FMT == CB_KV8_E4M3)
        w[j / 2] |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(f.x * inv, f.y * inv), __NV_SATFINITE, __NV_E4M3) << (16 * (j & 1));
      else
        w[j / 2] |= (kv8_encode<FMT>(f.x * inv) | kv8_encode<FMT>(f.y * inv) << 8) << (16 * (j & 1));
    }
  }
  return make_uint2(w[0], w[1]);
}

template <int D, int FMT, typename T, bool VEC>
__global__ void __launch_bounds__(kAT) kv8_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int kPer = D / 8;                                     // 8-value pieces of one token
  constexpr int kPieces = kKv8Block * kPer;                       // of one block
  constexpr int kMine = (kPieces + kAT - 1) / kAT;                // of one thread
  __shared__ float red[33];
  const int h = blockIdx.y % p.c.n_kv_heads, b = blockIdx.y / p.c.n_kv_heads;
  const bool is_v = blockIdx.z != 0;
  const int pos = p.pos[b];
  const int cnt = p.counts ? min(max(p.counts[b], 0), p.T) : p.T;
  if (pos < 0 || cnt == 0) return;
  const int blk = pos / kKv8Block + (int)blockIdx.x, first = blk * kKv8Block;
  // the block's slots [lo, hi) get new tokens, [first, lo) hold old ones
  const int64_t end = (int64_t)pos + cnt;
  if (end > p.c.max_len && blockIdx.x == 0 && threadIdx.x == 0) set_status(p.status, CB_ERR_CTX_FULL);
  const int lo = max(pos, first), hi = (int)min(end, (int64_t)min(first + kKv8Block, p.c.max_len));
  if (lo >= hi) return;
  const int64_t row = (int64_t)b * p.c.n_kv_heads + h;
  const T* src = static_cast<const T*>(is_v ? p.v : p.k);
  const int64_t* st = is_v ? p.vs : p.ks;
  uint8_t* codes = (is_v ? p.c.v : p.c.k) + (row * p.c.max_len + first) * D;
  float* scale = (is_v ? p.c.v_scale : p.c.k_scale) + row * (p.c.max_len / kKv8Block) + blk;

  Eight<T> x[kMine];
  float top = 0.0f, odd = 0.0f;  // odd: NaN where an infinity or a NaN passed
  const T* from = src + (int64_t)b * st[0] + (int64_t)(first - pos) * st[1] + h * st[2];
#pragma unroll
  for (int m = 0; m < kMine; ++m) {
    const int piece = threadIdx.x + m * kAT, slot = first + piece / kPer;
    if (slot >= lo && slot < hi && piece < kPieces)
      x[m].template load<VEC>(from + (int64_t)(piece / kPer) * st[1] + (piece % kPer) * 8);
  }
#pragma unroll
  for (int m = 0; m < kMine; ++m) {
    const int piece = threadIdx.x + m * kAT, slot = first + piece / kPer;
    if (slot < lo || slot >= hi || piece >= kPieces) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = x[m].pair(j);
      top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
      odd = fmaf(f.x, 0.0f, fmaf(f.y, 0.0f, odd));
    }
  }
  const bool plain = odd == 0.0f;
  if (!plain) {  // infinities and NaN leave the scale alone
    top = 0.0f;
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      const int piece = threadIdx.x + m * kAT, slot = first + piece / kPer;
      if (slot < lo || slot >= hi || piece >= kPieces) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = x[m].pair(j);
        if (fabsf(f.x) < INFINITY) top = fmaxf(top, fabsf(f.x));
        if (fabsf(f.y) < INFINITY) top = fmaxf(top, fabsf(f.y));
      }
    }
  }
  top = block_max(top, red);
  const float old = lo > first ? *scale : 0.0f;
  __syncthreads();  // every thread has read the old scale
  int e = kv8_need<FMT>(top);
  if (lo > first) e = max(e, kv8_exponent(old));
  const float s = kv8_pow2(e), inv = kv8_pow2(-e);
  if (threadIdx.x == 0) *scale = s;
  if (!is_v && p.c.mass && threadIdx.x < hi - lo) p.c.mass[row * p.c.max_len + lo + threadIdx.x] = 0.0f;
  const bool grow = lo > first && s > old;
#pragma unroll
  for (int m = 0; m < kMine; ++m) {
    const int piece = threadIdx.x + m * kAT, slot = first + piece / kPer;
    if (slot >= hi || piece >= kPieces || (slot < lo && !grow)) continue;
    uint2* dst = reinterpret_cast<uint2*>(codes + piece * 8);
    if (slot < lo) {
      const uint2 c = *dst;
      const uint32_t was[2] = {c.x, c.y};
      uint32_t w[2] = {0u, 0u};
      const float f = old * inv;  // 2^-d
#pragma unroll
      for (int j = 0; j < 8; ++j)
        w[j / 4] |= kv8_encode<FMT>(kv8_decode<FMT>(was[j / 4] >> (8 * (j & 3))) * f) << (8 * (j & 3));
      *dst = make_uint2(w[0], w[1]);
    } else {
      *dst = encode8<FMT, T>(x[m], inv, plain && e < kKv8EMax);
    }
  }
}

template <int D, int FMT, typename T>
void launch(const AppendParams& p, dim3 grid, bool vec, cudaStream_t st) {
  if (vec) kv8_append_kernel<D, FMT, T, true><<<grid, kAT, 0, st>>>(p);
  else kv8_append_kernel<D, FMT, T, false><<<grid, kAT, 0, st>>>(p);
}

template <int D, int FMT>
void launch(const AppendParams& p, dim3 grid, bool vec, cudaStream_t st) {
  if (p.dtype == CB_F32) launch<D, FMT, float>(p, grid, vec, st);
  else if (p.dtype == CB_BF16) launch<D, FMT, __nv_bfloat16>(p, grid, vec, st);
  else launch<D, FMT, __half>(p, grid, vec, st);
}

template <int D>
void launch(const AppendParams& p, dim3 grid, bool vec, cudaStream_t st) {
  if (p.c.format == CB_KV8_E4M3) launch<D, CB_KV8_E4M3>(p, grid, vec, st);
  else launch<D, CB_KV8_INT8>(p, grid, vec, st);
}

}  // namespace

int kv8_check(const CbKv8* c) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return CB_ERR_ARG;
  if (c->batch <= 0 || c->n_kv_heads <= 0 || c->max_len <= 0) return CB_ERR_ARG;
  if (c->format != CB_KV8_E4M3 && c->format != CB_KV8_INT8) return CB_ERR_ARG;
  if (c->max_len % kKv8Block) return CB_ERR_SHAPE;
  if (c->head_dim != 16 && c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128) return CB_ERR_SHAPE;
  if ((int64_t)c->batch * c->n_kv_heads > 65535) return CB_ERR_SHAPE;
  // codes are copied 16 bytes at a time
  if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) return CB_ERR_ARG;
  return CB_OK;
}

bool kv8_dtype_ok(int dtype) { return dtype == CB_F32 || dtype == CB_BF16 || dtype == CB_F16; }

}  // namespace cb

using namespace cb;

extern "C" int cb_kv8_append(const CbKv8* c, const void* k, const void* v, int32_t dtype, const int64_t* k_strides,
                             const int64_t* v_strides, int32_t T, const int32_t* pos, const int32_t* counts,
                             int32_t* status, void* stream) {
  const int rc = kv8_check(c);
  if (rc != CB_OK) return rc;
  if (!k || !v || !k_strides || !v_strides || !pos || T <= 0 || T > c->max_len || !kv8_dtype_ok(dtype))
    return CB_ERR_ARG;
  AppendParams p{};
  p.c = *c;
  p.k = k;
  p.v = v;
  p.dtype = dtype;
  p.T = T;
  const int size = dtype == CB_F32 ? 4 : 2, lane = 16 / size;
  bool vec = (((uintptr_t)k | (uintptr_t)v) & 15) == 0;
  for (int i = 0; i < 3; ++i) {
    p.ks[i] = k_strides[i];
    p.vs[i] = v_strides[i];
    vec = vec && k_strides[i] % lane == 0 && v_strides[i] % lane == 0;
  }
  p.pos = pos;
  p.counts = counts;
  p.status = status;
  // T tokens from any slot of a block on touch at most this many blocks
  const dim3 grid((unsigned)((T + 2 * kKv8Block - 2) / kKv8Block), (unsigned)(c->batch * c->n_kv_heads), 2);
  cudaStream_t st = (cudaStream_t)stream;
  switch (c->head_dim) {
    case 16: launch<16>(p, grid, vec, st); break;
    case 32: launch<32>(p, grid, vec, st); break;
    case 64: launch<64>(p, grid, vec, st); break;
    default: launch<128>(p, grid, vec, st); break;
  }
  count_launch();
  return cudaGetLastError() == cudaSuccess ? CB_OK : CB_ERR_CUDA;
}
