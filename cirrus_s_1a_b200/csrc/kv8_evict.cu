// cb_kv8_evict: brings every sequence that holds more than `keep` tokens down to
// `keep`, per KV head: the `recent` last slots stay, and of the older ones the
// keep - recent with the largest accumulated attention weight (ties to the
// lowest slot).  The kept tokens move to slots 0 .. keep - 1 in order, in place.
//
// One CTA per (sequence, KV head): a radix select over the weights' order keys
// (8 bits a pass), an ordered scan that writes the kept slots, then the blocks
// of 64 kept tokens one after another.  In place is safe in that order: the
// token for slot j comes from a slot >= j, so what block i overwrites (slots
// below 64 (i + 1)) is read by no later block.  A new block's scale is the one
// its values need; a code is rounded again only where its scale grows.
#include "kv8.cuh"
#include "kv8_attend.cuh"

namespace cb {
namespace {

constexpr int kET = 1024;

struct EvictParams {
  CbKv8 c;
  const int32_t* pos;
  int keep, recent;
  int32_t* kept;
  int32_t* new_pos;
};

// Order key of a weight: larger weight, larger key; NaN below everything.
__device__ __forceinline__ uint32_t weight_key(float w) { return w != w ? 0u : score_key(w); }

// Exclusive prefix sum over the CTA of one int per thread; total to *all.
__device__ __forceinline__ int block_scan(int v, int* red, int* all) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) red[w] = x;
  __syncthreads();
  if (w == 0) {
    int y = red[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int z = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) y += z;
    }
    red[lane] = y;
  }
  __syncthreads();
  *all = red[31];
  return x - v + (w ? red[w - 1] : 0);
}

template <int D, int FMT>
__global__ void __launch_bounds__(kET) kv8_evict_kernel(const __grid_constant__ EvictParams p) {
  __shared__ int hist[256];
  __shared__ int red[32];
  __shared__ float fred[33];
  __shared__ uint32_t s_prefix;
  __shared__ int s_rest;
  const int h = blockIdx.x % p.c.n_kv_heads, b = blockIdx.x / p.c.n_kv_heads, tid = threadIdx.x;
  const int n = min(max(p.pos[b], 0), p.c.max_len), keep = p.keep;
  const int64_t head = blockIdx.x;
  int32_t* kept = p.kept + head * keep;
  if (h == 0 && tid == 0) p.new_pos[b] = min(n, keep);
  if (n <= keep) {
    for (int j = tid; j < keep; j += kET) kept[j] = j < n ? j : -1;
    return;
  }
  float* mass = p.c.mass + head * p.c.max_len;
  const int old = n - p.recent;       // candidates: slots below this
  const int want = keep - p.recent;   // how many of them stay, < old

  // the want-th largest key: `prefix`, and how many of its ties stay
  uint32_t prefix = 0, mask = 0;
  int rest = want;
  if (want > 0)
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kET) hist[i] = 0;
      __syncthreads();
      for (int j = tid; j < old; j += kET) {
        const uint32_t u = weight_key(mass[j]);
        if ((u & mask) == prefix) atomicAdd(&hist[(u >> shift) & 255], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int d = 255, left = rest;
        while (hist[d] < left) left -= hist[d--];
        s_prefix = prefix | ((uint32_t)d << shift);
        s_rest = left;
      }
      __syncthreads();
      prefix = s_prefix;
      rest = s_rest;
      mask |= 255u << shift;
      __syncthreads();
    }

  // kept slots in order
  int base = 0, ties = 0;
  for (int j0 = 0; j0 < n; j0 += kET) {
    const int j = j0 + tid;
    bool above = false, tie = false;
    if (j < old && want > 0) {
      const uint32_t u = weight_key(mass[j]);
      above = u > prefix;
      tie = u == prefix;
    }
    int nt;
    const int tb = ties + block_scan(tie, red, &nt);
    const bool stay = j < n && (j >= old || above || (tie && tb < rest));
    ties += nt;
    int ns;
    const int at = base + block_scan(stay, red, &ns);
    if (stay) kept[at] = j;
    base += ns;
  }
  __syncthreads();

  // blocks of 64 kept tokens
  constexpr int kPer = D / 8, kPieces = kKv8Block * kPer;
  constexpr int kMine = (kPieces + kET - 1) / kET;
  const int64_t nb = p.c.max_len / kKv8Block;
  for (int first = 0; first < keep; first += kKv8Block) {
    const int cnt = min(kKv8Block, keep - first);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      uint8_t* codes = (kv ? p.c.v : p.c.k) + head * p.c.max_len * D;
      float* scale = (kv ? p.c.v_scale : p.c.k_scale) + head * nb;
      float x[kMine][8];
      float top = 0.0f;
#pragma unroll
      for (int m = 0; m < kMine; ++m) {
        const int piece = tid + m * kET, tok = piece / kPer;
        if (tok >= cnt) continue;
        const int src = kept[first + tok];
        const uint2 c = *reinterpret_cast<const uint2*>(codes + (int64_t)src * D + (piece % kPer) * 8);
        const float s = scale[src / kKv8Block];
        const uint32_t w[2] = {c.x, c.y};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[m][i] = kv8_decode<FMT>(w[i / 4] >> (8 * (i & 3))) * s;
          if (fabsf(x[m][i]) < INFINITY) top = fmaxf(top, fabsf(x[m][i]));
        }
      }
      top = block_max(top, fred);  // its barriers end the reads of this block
      const int e = kv8_need<FMT>(top);
      const float inv = kv8_pow2(-e);
#pragma unroll
      for (int m = 0; m < kMine; ++m) {
        const int piece = tid + m * kET, tok = piece / kPer;
        if (tok >= cnt) continue;
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i / 4] |= kv8_encode<FMT>(x[m][i] * inv) << (8 * (i & 3));
        *reinterpret_cast<uint2*>(codes + (int64_t)first * D + piece * 8) = make_uint2(w[0], w[1]);
      }
      if (tid == 0) scale[first / kKv8Block] = kv8_pow2(e);
    }
    float w = 0.0f;
    if (tid < cnt) w = mass[kept[first + tid]];
    __syncthreads();
    if (tid < cnt) mass[first + tid] = w;
    __syncthreads();
  }
}

template <int D>
void launch(const EvictParams& p, cudaStream_t st) {
  const int grid = p.c.batch * p.c.n_kv_heads;
  if (p.c.format == CB_KV8_E4M3) kv8_evict_kernel<D, CB_KV8_E4M3><<<grid, kET, 0, st>>>(p);
  else kv8_evict_kernel<D, CB_KV8_INT8><<<grid, kET, 0, st>>>(p);
}

}  // namespace
}  // namespace cb

using namespace cb;

extern "C" int cb_kv8_evict(const CbKv8* c, const int32_t* pos, int32_t keep, int32_t recent, int32_t* kept,
                            int32_t* new_pos, void* stream) {
  const int rc = kv8_check(c);
  if (rc != CB_OK) return rc;
  if (!c->mass || !pos || !kept || !new_pos || new_pos == pos) return CB_ERR_ARG;
  if (keep <= 0 || recent < 0 || recent > keep || keep > c->max_len) return CB_ERR_ARG;
  const EvictParams p{*c, pos, keep, recent, kept, new_pos};
  cudaStream_t st = (cudaStream_t)stream;
  switch (c->head_dim) {
    case 16: launch<16>(p, st); break;
    case 32: launch<32>(p, st); break;
    case 64: launch<64>(p, st); break;
    default: launch<128>(p, st); break;
  }
  count_launch();
  return cudaGetLastError() == cudaSuccess ? CB_OK : CB_ERR_CUDA;
}
