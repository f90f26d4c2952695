// cb_kv8_append: T new tokens per sequence into the 8-bit cache.
//
// One CTA owns one (sequence, KV head, block of 64 slots) of K or of V.  It
// reads the block's new values once, keeps them in registers, reduces their
// absmax, and writes codes and the scale.  A block that already holds tokens
// keeps the larger of its scale and the one the new tokens need; its old codes
// are rewritten only when the scale grows (each is then rounded once more, onto
// a grid 2^d times as coarse).  The result does not depend on the order of
// anything: absmax is order-free and every division by a scale is exact.
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

// Eight values of one token, from 16-byte vectors (VEC) or one by one.
template <bool VEC>
__device__ __forceinline__ void load8(const void* base, int64_t i, int dtype, float (&x)[8]) {
  if (VEC && dtype == CB_F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + i);
    const float4 a = __ldcs(p), b = __ldcs(p + 1);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else if (VEC) {
    const uint4 a = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + i));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (dtype == CB_BF16) {
        x[2 * j] = bf16_to_f32(w[j]);
        x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        x[2 * j] = f.x;
        x[2 * j + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = kv8_load(base, i + j, dtype);
  }
}

template <int D, int FMT, bool VEC>
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
  const void* src = is_v ? p.v : p.k;
  const int64_t* st = is_v ? p.vs : p.ks;
  uint8_t* codes = (is_v ? p.c.v : p.c.k) + (row * p.c.max_len + first) * D;
  float* scale = (is_v ? p.c.v_scale : p.c.k_scale) + row * (p.c.max_len / kKv8Block) + blk;

  float x[kMine][8];
  float top = 0.0f;
#pragma unroll
  for (int m = 0; m < kMine; ++m) {
    const int piece = threadIdx.x + m * kAT, slot = first + piece / kPer;
    if (slot < lo || slot >= hi || piece >= kPieces) continue;
    load8<VEC>(src, (int64_t)b * st[0] + (int64_t)(slot - pos) * st[1] + h * st[2] + (piece % kPer) * 8, p.dtype, x[m]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float a = fabsf(x[m][j]);
      if (a < INFINITY) top = fmaxf(top, a);  // infinities and NaN leave the scale alone
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
    uint32_t w[2] = {0u, 0u};
    if (slot < lo) {
      const uint2 c = *dst;
      const uint32_t was[2] = {c.x, c.y};
      const float f = old * inv;  // 2^-d
#pragma unroll
      for (int j = 0; j < 8; ++j)
        w[j / 4] |= kv8_encode<FMT>(kv8_decode<FMT>(was[j / 4] >> (8 * (j & 3))) * f) << (8 * (j & 3));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j / 4] |= kv8_encode<FMT>(x[m][j] * inv) << (8 * (j & 3));
    }
    *dst = make_uint2(w[0], w[1]);
  }
}

template <int D>
void launch(const AppendParams& p, dim3 grid, bool vec, cudaStream_t st) {
  const bool e4m3 = p.c.format == CB_KV8_E4M3;
  if (e4m3 && vec) kv8_append_kernel<D, CB_KV8_E4M3, true><<<grid, kAT, 0, st>>>(p);
  else if (e4m3) kv8_append_kernel<D, CB_KV8_E4M3, false><<<grid, kAT, 0, st>>>(p);
  else if (vec) kv8_append_kernel<D, CB_KV8_INT8, true><<<grid, kAT, 0, st>>>(p);
  else kv8_append_kernel<D, CB_KV8_INT8, false><<<grid, kAT, 0, st>>>(p);
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
