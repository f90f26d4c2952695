// Attention over the 8-bit K/V cache: cb_kv8_attend.
//
//   x[r][j] = q_r . k_j * scale      j <= pos[b] + t   (k_j = code * block scale)
//   lse_r   = log sum_j exp(x[r][j])
//   out_r   = sum_j exp(x[r][j] - lse_r) v_j
//   mass_j += sum over the KV head's rows r of exp(x[r][j] - lse_r)     (add_mass)
//
// The rows of a KV head are its G query heads of the T tokens, r = t * G + g, so
// the codes are read once for all of them.  kv8_attend_kernel runs on warp-level
// matrix products (m16n8k16, f16 operands, f32 sums).  Codes are exact in f16;
// the products' free index order is used so that no operand needs a transpose
// through shared memory:
//   * S = Q K^T: lane (g, t) = (lane / 4, lane % 4) reads D/4 contiguous bytes of
//     one key row, so a warp's load covers whole rows; the four k positions a
//     lane feeds in step s are the dims t * D/4 + 4 s .. + 3, and the query
//     fragments are loaded in that order.
//   * O = P V: the softmax of S leaves P in the layout of an A operand.  The key
//     behind column c of key tile j is 8 j + 4 (c & 1) + c / 2, so the four keys
//     a lane feeds in a step are 16 s + t + {0, 4, 8, 12}: four rows in a row
//     across t.  The lane reads D/8 contiguous bytes of each (dims g * D/8 ..)
//     and pairs the keys' bytes with byte permutes.
// Queries: a row is scaled by a power of two that brings its largest element to
// [256, 512) and rounded to f16.  bf16 and f16 queries are exact in that (up to
// 2^-33 of the row's largest element); float32 queries and their P are carried
// as a head and a tail (about 22 bits), two products each.  f16 P (11 bits) for
// 16-bit outputs adds less than the output's own rounding.
// Softmax statistics, the sums over V and the joins of parts are float32.
#include <algorithm>

#include "kv8.cuh"
#include "kv8_attend.cuh"

namespace cb {
namespace {

constexpr int kWarps = 4;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// N bytes (2, 4, 8, 16 or 32, aligned to min(N, 16)) as words.
template <int N>
__device__ __forceinline__ void load_bytes(const uint8_t* p, uint32_t (&w)[(N + 3) / 4]) {
  if constexpr (N == 2) {
    w[0] = *reinterpret_cast<const uint16_t*>(p);
  } else if constexpr (N == 4) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 8) {
    const uint2 a = *reinterpret_cast<const uint2*>(p);
    w[0] = a.x, w[1] = a.y;
  } else {
#pragma unroll
    for (int i = 0; i < N / 16; ++i) {
      const uint4 a = reinterpret_cast<const uint4*>(p)[i];
      w[4 * i] = a.x, w[4 * i + 1] = a.y, w[4 * i + 2] = a.z, w[4 * i + 3] = a.w;
    }
  }
}

// Query rows row0 .. row0 + 15 of a KV head as A fragments: lane (g, t) holds
// rows g and g + 8.  `back` gets the factor that undoes each row's power of two,
// times scale * log2(e).  HL: the tails too.
template <int D, bool HL>
__device__ __forceinline__ void load_q(const AttendParams& p, int b, int hk, int row0, uint32_t (&qh)[D / 16][4],
                                       uint32_t (&ql)[HL ? D / 16 : 1][4], float (&back)[2]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = row0 + g + 8 * half;
    float x[D / 4];
    float top = 0.0f;
    const bool live = r < p.rows;
    const int t = r / p.G, hq = hk * p.G + r % p.G;
    const int64_t base = (int64_t)b * p.qs[0] + (int64_t)t * p.qs[1] + hq * p.qs[2] + t4 * (D / 4);
#pragma unroll
    for (int i = 0; i < D / 4; ++i) {
      x[i] = live ? kv8_load(p.q, base + i, p.dtype) : 0.0f;
      top = fmaxf(top, fabsf(x[i]));
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    int e = 0;  // top in [2^e, 2^(e+1)); rows of zeros, infinities and the ends of the range keep e = 0
    if (top > 0.0f && top < INFINITY) e = min(max((__float_as_int(top) >> 23) - 127, -100), 100);
    const float f = kv8_pow2(8 - e);
    back[half] = kv8_pow2(e - 8) * p.scale * kLog2e;
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float u = x[4 * s + 2 * i] * f, v = x[4 * s + 2 * i + 1] * f;
        const __half2 h = __floats2half2_rn(u, v);
        qh[s][half + 2 * i] = h2_bits(h);
        if (HL) {
          const float2 back2 = __half22float2(h);
          ql[HL ? s : 0][half + 2 * i] = h2_bits(__floats2half2_rn(u - back2.x, v - back2.y));
        }
      }
  }
}

// The last slot query row r sees; -1: none.
__device__ __forceinline__ int row_limit(const AttendParams& p, int r, int pos, int cnt) {
  const int t = r / p.G;
  if (r >= p.rows || t >= cnt) return -1;
  return min(pos + t, p.c.max_len - 1);
}

// S of 16 query rows against the 64 keys of a block (codes only): c[j] is key tile j.
template <int D, int FMT, bool HL>
__device__ __forceinline__ void scores(const uint8_t* kb, const uint32_t (&qh)[D / 16][4],
                                       const uint32_t (&ql)[HL ? D / 16 : 1][4], float (&c)[8][4]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    uint32_t w[D / 16];
    load_bytes<D / 4>(kb + (8 * j + (g & 1) * 4 + (g >> 1)) * D + t4 * (D / 4), w);
    c[j][0] = c[j][1] = c[j][2] = c[j][3] = 0.0f;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      uint32_t b0, b1;
      codes_to_h2<FMT>(w[s], b0, b1);
      mma16816(c[j], qh[s], b0, b1);
      if (HL) mma16816(c[j], ql[HL ? s : 0], b0, b1);
    }
  }
}

// Key (within its block) behind element i of key tile j of this lane's S.
__device__ __forceinline__ int key_of(int j, int i) { return 8 * j + 4 * (i & 1) + (threadIdx.x & 3); }

template <int D, int FMT, bool HL>
__global__ void __launch_bounds__(kWarps * 32) kv8_attend_kernel(const __grid_constant__ AttendParams p) {
  __shared__ float s_m[kWarps][16], s_l[kWarps][16];
  extern __shared__ float s_o[];  // [kWarps][16][D]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
  const int hk = blockIdx.z % p.c.n_kv_heads, b = blockIdx.z / p.c.n_kv_heads;
  const int split = blockIdx.x, row0 = blockIdx.y * 16;
  const int pos = p.pos[b], cnt = p.counts ? min(max(p.counts[b], 0), p.T) : p.T;
  const int lim[2] = {row_limit(p, row0 + g, pos, cnt), row_limit(p, row0 + g + 8, pos, cnt)};
  // blocks of 64 keys the rows of this CTA see, dealt out to the splits in runs
  int last = -1;
  for (int r = row0; r < min(row0 + 16, p.rows); ++r) last = max(last, row_limit(p, r, pos, cnt));
  const int blocks = (last + kKv8Block) / kKv8Block;
  const int per = (blocks + p.splits - 1) / p.splits;
  const int beg = min(blocks, split * per), end = min(blocks, beg + per);
  const int64_t head = (int64_t)b * p.c.n_kv_heads + hk;
  const uint8_t* kbase = p.c.k + head * p.c.max_len * D;
  const uint8_t* vbase = p.c.v + head * p.c.max_len * D;
  const float* ksc = p.c.k_scale + head * (p.c.max_len / kKv8Block);
  const float* vsc = p.c.v_scale + head * (p.c.max_len / kKv8Block);

  uint32_t qh[D / 16][4], ql[HL ? D / 16 : 1][4];
  float back[2];
  load_q<D, HL>(p, b, hk, row0, qh, ql, back);
  float o[D / 8][4] = {};
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

  for (int blk = beg + warp; blk < end; blk += kWarps) {
    float c[8][4];
    scores<D, FMT, HL>(kbase + (int64_t)blk * kKv8Block * D, qh, ql, c);
    const float f0 = back[0] * ksc[blk], f1 = back[1] * ksc[blk];
    const int key0 = blk * kKv8Block;
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int half = i >> 1;
        c[j][i] = key0 + key_of(j, i) <= lim[half] ? c[j][i] * (half ? f1 : f0) : -INFINITY;
        top[half] = fmaxf(top[half], c[j][i]);
      }
    float alpha[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      top[half] = fmaxf(top[half], __shfl_xor_sync(0xffffffffu, top[half], 1));
      top[half] = fmaxf(top[half], __shfl_xor_sync(0xffffffffu, top[half], 2));
      const float now = fmaxf(m[half], top[half]);
      alpha[half] = m[half] == -INFINITY ? 0.0f : exp2a(m[half] - now);
      m[half] = now;
      l[half] *= alpha[half];
    }
    const float sub[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
    float pv[D / 8][4] = {};
    const uint8_t* vb = vbase + (int64_t)blk * kKv8Block * D;
    const bool tail = key0 + kKv8Block > last + 1;  // the block ends past the last visible slot
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      uint32_t ph[4], pl[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {  // A registers: (tile 2s, rows g / g+8), (tile 2s+1, rows g / g+8)
        const int j = 2 * s + (q >> 1), half = q & 1;
        const float e0 = exp2a(c[j][2 * half] - sub[half]), e1 = exp2a(c[j][2 * half + 1] - sub[half]);
        l[half] += e0 + e1;
        const __half2 h = __floats2half2_rn(e0, e1);
        ph[q] = h2_bits(h);
        if (HL) {
          const float2 hb = __half22float2(h);
          pl[q] = h2_bits(__floats2half2_rn(e0 - hb.x, e1 - hb.y));
        }
      }
      constexpr int NB = D / 8;  // bytes of a row this lane feeds
      uint32_t w[4][(NB + 3) / 4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int key = 16 * s + 4 * u + t4;
        load_bytes<NB>(vb + key * D + g * NB, w[u]);
        // slots no row sees may hold anything, an E4M3 NaN too: 0 * NaN is not 0
        if (tail && key0 + key > last)
#pragma unroll
          for (int z = 0; z < (NB + 3) / 4; ++z) w[u][z] = 0u;
      }
#pragma unroll
      for (int z = 0; z < (NB + 3) / 4; ++z)
#pragma unroll
        for (int y = 0; y < (NB < 4 ? 1 : 2); ++y) {
          // keys' bytes side by side: dims 4z + 2y and 4z + 2y + 1
          const uint32_t sel = y ? 0x7362u : 0x5140u;
          const uint32_t a = __byte_perm(w[0][z], w[1][z], sel), d = __byte_perm(w[2][z], w[3][z], sel);
          uint32_t a0, a1, d0, d1;
          codes_to_h2<FMT>(a, a0, a1);
          codes_to_h2<FMT>(d, d0, d1);
          const int n = 4 * z + 2 * y;
          mma16816(pv[n], ph, a0, d0);
          mma16816(pv[n + 1], ph, a1, d1);
          if (HL) {
            mma16816(pv[n], pl, a0, d0);
            mma16816(pv[n + 1], pl, a1, d1);
          }
        }
    }
    const float vs = vsc[blk];
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][i] = fmaf(pv[n][i], vs, o[n][i] * alpha[i >> 1]);
  }

  // join the warps, in warp order
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
    l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
    if (t4 == 0) {
      s_m[warp][g + 8 * half] = m[half];
      s_l[warp][g + 8 * half] = l[half];
    }
  }
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      s_o[(warp * 16 + g + 8 * (i >> 1)) * D + (2 * t4 + (i & 1)) * (D / 8) + n] = o[n][i];
  __syncthreads();
  for (int e = threadIdx.x; e < 16 * D; e += kWarps * 32) {
    const int rr = e / D, d = e % D, r = row0 + rr;
    if (r >= p.rows) break;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_m[w][rr]);
    float ll = 0.0f, oo = 0.0f;
    if (mm > -INFINITY) {
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = exp2a(s_m[w][rr] - mm);
        ll = fmaf(s_l[w][rr], f, ll);
        oo = fmaf(s_o[(w * 16 + rr) * D + d], f, oo);
      }
    }
    const int64_t at = (head * p.rows + r) * p.splits + split;
    p.part_o[at * D + d] = oo;
    if (d == 0) {
      p.part_ml[2 * at] = mm;
      p.part_ml[2 * at + 1] = ll;
    }
  }
}

// Joins the splits' parts of one row, in split order: one CTA of D threads per
// row (all its splits' maxima and sums are a few KB, read from L2).
__global__ void kv8_join_kernel(const __grid_constant__ AttendParams p) {
  const int D = p.c.head_dim, d = threadIdx.x;
  const int r = blockIdx.x;
  const int64_t head = blockIdx.y;
  const int hk = (int)(head % p.c.n_kv_heads), b = (int)(head / p.c.n_kv_heads);
  const int t = r / p.G, hq = hk * p.G + r % p.G;
  const int64_t at = (head * p.rows + r) * p.splits;
  float mm = -INFINITY;
  for (int s = 0; s < p.splits; ++s) mm = fmaxf(mm, p.part_ml[2 * (at + s)]);
  float ll = 0.0f, oo = 0.0f;
  if (mm > -INFINITY)
    for (int s = 0; s < p.splits; ++s) {
      const float f = exp2a(p.part_ml[2 * (at + s)] - mm);
      ll = fmaf(p.part_ml[2 * (at + s) + 1], f, ll);
      oo = fmaf(p.part_o[(at + s) * D + d], f, oo);
    }
  const int64_t orow = ((int64_t)b * p.T + t) * (p.G * p.c.n_kv_heads) + hq;
  const float y = ll > 0.0f ? oo / ll : (mm > -INFINITY ? oo / ll : 0.0f);
  if (p.dtype == CB_F32) static_cast<float*>(p.out)[orow * D + d] = y;
  else if (p.dtype == CB_BF16) static_cast<uint16_t*>(p.out)[orow * D + d] = f32_to_bf16(y);
  else static_cast<__half*>(p.out)[orow * D + d] = __float2half_rn(y);
  if (d == 0) p.lse[orow] = mm > -INFINITY ? (mm + log2f(ll)) * kLn2 : -INFINITY;
}

// mass_j += sum_r exp(x[r][j] - lse_r): a warp owns a block of 64 keys and walks
// the head's query rows 16 at a time, so every slot has one writer and one order.
template <int D, int FMT, bool HL>
__global__ void __launch_bounds__(kWarps * 32) kv8_mass_kernel(const __grid_constant__ AttendParams p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2;
  const int hk = blockIdx.y % p.c.n_kv_heads, b = blockIdx.y / p.c.n_kv_heads;
  const int pos = p.pos[b], cnt = p.counts ? min(max(p.counts[b], 0), p.T) : p.T;
  const int last = cnt > 0 ? min(pos + cnt, p.c.max_len) - 1 : -1;
  const int64_t head = (int64_t)b * p.c.n_kv_heads + hk;
  for (int blk = blockIdx.x * kWarps + warp; blk * kKv8Block <= last; blk += gridDim.x * kWarps) {
    const int key0 = blk * kKv8Block;
    const uint8_t* kb = p.c.k + (head * p.c.max_len + key0) * D;
    const float ks = p.c.k_scale[head * (p.c.max_len / kKv8Block) + blk];
    float sum[8][2] = {};
    const int first_t = max(0, key0 - pos);  // rows of earlier tokens do not see this block
    for (int row0 = first_t * p.G / 16 * 16; row0 < cnt * p.G; row0 += 16) {
      uint32_t qh[D / 16][4], ql[HL ? D / 16 : 1][4];
      float back[2], lse[2];
      load_q<D, HL>(p, b, hk, row0, qh, ql, back);
      int lim[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = row0 + g + 8 * half;
        lim[half] = row_limit(p, r, pos, cnt);
        lse[half] = 0.0f;
        if (lim[half] >= 0)
          lse[half] = p.lse[((int64_t)b * p.T + r / p.G) * (p.G * p.c.n_kv_heads) + hk * p.G + r % p.G] * kLog2e;
      }
      float c[8][4];
      scores<D, FMT, HL>(kb, qh, ql, c);
      const float f[2] = {back[0] * ks, back[1] * ks};
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int half = i >> 1;
          if (key0 + key_of(j, i) <= lim[half]) sum[j][i & 1] += exp2a(fmaf(c[j][i], f[half], -lse[half]));
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float v = sum[j][i];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        const int key = key0 + key_of(j, i);
        if (g == 0 && key <= last) p.c.mass[head * p.c.max_len + key] += v;
      }
  }
}

template <int D, int FMT, bool HL>
int launch_dfh(const AttendParams& p, int bh, int longest, cudaStream_t st) {
  if (p.row_tiles > 0) {
    if (const int rc = kv8_prompt_launch(p, bh, st)) return rc;
  } else {
    const int smem = kWarps * 16 * D * (int)sizeof(float);
    auto fn = kv8_attend_kernel<D, FMT, HL>;
    if (const int rc = ensure_smem_attr((const void*)fn, smem)) return rc;
    fn<<<dim3(p.splits, ceil_div(p.rows, 16), bh), kWarps * 32, smem, st>>>(p);
    count_launch();
  }
  if (p.row_tiles == 0 || p.splits > 1) {
    kv8_join_kernel<<<dim3(p.rows, bh), D, 0, st>>>(p);
    count_launch();
  }
  if (p.add_mass && p.row_tiles > 0) {
    if (const int rc = kv8_prompt_mass_launch(p, bh, longest, st)) return rc;
  } else if (p.add_mass) {
    kv8_mass_kernel<D, FMT, HL><<<dim3(ceil_div(longest, kWarps * kKv8Block), bh), kWarps * 32, 0, st>>>(p);
    count_launch();
  }
  return cudaGetLastError() == cudaSuccess ? CB_OK : CB_ERR_CUDA;
}

template <int D>
int launch_d(const AttendParams& p, int bh, int longest, cudaStream_t st) {
  const bool e = p.c.format == CB_KV8_E4M3, hl = p.dtype == CB_F32;
  if (e && hl) return launch_dfh<D, CB_KV8_E4M3, true>(p, bh, longest, st);
  if (e) return launch_dfh<D, CB_KV8_E4M3, false>(p, bh, longest, st);
  if (hl) return launch_dfh<D, CB_KV8_INT8, true>(p, bh, longest, st);
  return launch_dfh<D, CB_KV8_INT8, false>(p, bh, longest, st);
}

// How a call is cut up, and where its parts lie in the scratch.
struct Plan {
  int rows = 0, row_tiles = 0, splits = 0;
  size_t o = 0, q16 = 0, back = 0, bytes = 0;  // part_ml at 0
};

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

Plan plan_of(const CbKv8& c, int dtype, int n_q_heads, int T, int longest) {
  Plan pl;
  const int bh = c.batch * c.n_kv_heads;
  pl.rows = T * (n_q_heads / c.n_kv_heads);
  // From 33 rows on the tensor cores' 128-row tiles pay for the rows they leave empty.
  if (pl.rows > 32 && c.head_dim >= 64 && dtype != CB_F32) {
    pl.row_tiles = ceil_div(pl.rows, 128);
    // runs of key tiles that leave the fewest tile times (and three more a CTA to
    // start and end) on the busiest SM
    const int items = bh * ceil_div(pl.row_tiles, 2), tiles = ceil_div(longest, 8192 / c.head_dim);
    long best = 0;
    for (int s = 1; s <= 32 && s <= ceil_div(tiles, 2); ++s) {
      const long cost = (long)ceil_div(items * s, 148) * (ceil_div(tiles, s) + 3);
      if (pl.splits == 0 || cost < best) {
        pl.splits = s;
        best = cost;
      }
    }
  } else {
    // enough CTAs for about four on every SM, each with at least one block of 64
    // keys for each of its warps
    const int items = bh * ceil_div(pl.rows, 16);
    pl.splits = std::max(1, std::min(ceil_div(148 * 4, items), ceil_div(longest, kWarps * kKv8Block)));
  }
  const int64_t parts = (int64_t)bh * pl.rows * pl.splits;
  pl.o = align256((size_t)parts * 2 * sizeof(float));
  pl.q16 = pl.o + align256((size_t)parts * c.head_dim * sizeof(float));
  pl.back = pl.q16 + (size_t)bh * pl.row_tiles * 128 * c.head_dim * 2;
  pl.bytes = pl.back + (size_t)bh * pl.row_tiles * 128 * sizeof(float);
  return pl;
}

int check_call(const CbKv8* c, int dtype, int n_q_heads, int T, int longest) {
  if (const int rc = kv8_check(c)) return rc;
  if (T <= 0 || longest <= 0 || !kv8_dtype_ok(dtype)) return CB_ERR_ARG;
  if (n_q_heads <= 0 || n_q_heads % c->n_kv_heads) return CB_ERR_SHAPE;
  if ((int64_t)T * (n_q_heads / c->n_kv_heads) > 65535 * 16) return CB_ERR_SHAPE;
  return CB_OK;
}

}  // namespace
}  // namespace cb

using namespace cb;

extern "C" size_t cb_kv8_attend_scratch_bytes(const CbKv8* c, int32_t dtype, int32_t n_q_heads, int32_t T,
                                              int32_t longest) {
  if (check_call(c, dtype, n_q_heads, T, longest) != CB_OK) return 0;
  return plan_of(*c, dtype, n_q_heads, T, std::min(longest, c->max_len)).bytes;
}

extern "C" int cb_kv8_attend(const CbKv8* c, const void* q, int32_t dtype, const int64_t* q_strides, int32_t n_q_heads,
                             int32_t T, const int32_t* pos, const int32_t* counts, int32_t longest, float scale,
                             int32_t add_mass, void* out, float* lse, void* scratch, size_t scratch_bytes,
                             int32_t* status, void* stream) {
  if (const int rc = check_call(c, dtype, n_q_heads, T, longest)) return rc;
  if (!q || !q_strides || !pos || !out || !lse || !scratch || ((uintptr_t)scratch & 15) || ((uintptr_t)out & 15))
    return CB_ERR_ARG;
  if (add_mass && !c->mass) return CB_ERR_ARG;
  longest = std::min(longest, c->max_len);
  const Plan pl = plan_of(*c, dtype, n_q_heads, T, longest);
  if (scratch_bytes < pl.bytes) return CB_ERR_WORKSPACE;
  AttendParams p{};
  p.c = *c;
  p.q = q;
  p.dtype = dtype;
  for (int i = 0; i < 3; ++i) p.qs[i] = q_strides[i];
  p.G = n_q_heads / c->n_kv_heads;
  p.T = T;
  p.rows = pl.rows;
  p.pos = pos;
  p.counts = counts;
  p.scale = scale;
  p.add_mass = add_mass != 0;
  p.out = out;
  p.lse = lse;
  p.splits = pl.splits;
  uint8_t* base = static_cast<uint8_t*>(scratch);
  p.part_ml = reinterpret_cast<float*>(base);
  p.part_o = reinterpret_cast<float*>(base + pl.o);
  p.row_tiles = pl.row_tiles;
  p.q16 = base + pl.q16;
  p.q_back = reinterpret_cast<float*>(base + pl.back);
  p.status = status;
  const int bh = c->batch * c->n_kv_heads;
  cudaStream_t st = (cudaStream_t)stream;
  switch (c->head_dim) {
    case 16: return launch_d<16>(p, bh, longest, st);
    case 32: return launch_d<32>(p, bh, longest, st);
    case 64: return launch_d<64>(p, bh, longest, st);
    default: return launch_d<128>(p, bh, longest, st);
  }
}
