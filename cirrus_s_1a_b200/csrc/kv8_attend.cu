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
//
// Work is dealt out by blocks of 64 keys: the visible blocks of all KV heads, one
// after another, are cut into equal runs, one per CTA (with sequences of different
// lengths, equal runs of each head left half of the SMs idle).  A run that crosses
// heads leaves a part for each; (CTA + head) numbers the parts without a table.
// Each warp takes every fourth block of a run; K and V blocks arrive by bulk copies
// in a ring of slots of its own, two or three ahead, across the ends of heads.  The
// CTA that finishes a head last joins its parts in their order and writes the
// output, so a call is one launch (two with attention weights).
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
  return min(pos + t, p.limit - 1);
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

// Writes the output and lse of one row's four dims: `o` is the sum against the
// maximum mm, ll its weights' sum.
__device__ __forceinline__ void write_row(const AttendParams& p, int b, int hk, int r, int d, float4 o, float mm, float ll) {
  const int64_t at = ((int64_t)b * p.T + r / p.G) * (p.G * p.c.n_kv_heads) + hk * p.G + r % p.G;
  const float inv = mm > -INFINITY || mm != mm ? 1.0f / ll : 0.0f;
  if (mm == -INFINITY) o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  const float y[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
  if (p.dtype == CB_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at * p.c.head_dim + d) = make_float4(y[0], y[1], y[2], y[3]);
  } else {
    uint2 u;
    if (p.dtype == CB_BF16)
      u = make_uint2((uint32_t)f32_to_bf16(y[0]) | (uint32_t)f32_to_bf16(y[1]) << 16,
                     (uint32_t)f32_to_bf16(y[2]) | (uint32_t)f32_to_bf16(y[3]) << 16);
    else
      u = make_uint2(h2_bits(__floats2half2_rn(y[0], y[1])), h2_bits(__floats2half2_rn(y[2], y[3])));
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at * p.c.head_dim + d) = u;
  }
  if (d == 0) p.lse[at] = mm == -INFINITY ? -INFINITY : (mm + log2f(ll)) * kLn2;
}

// Visible blocks of sequence b for the query rows up to last_row (exclusive).
__device__ __forceinline__ int visible_blocks(const AttendParams& p, int b, int row0, int rows_end, int& last) {
  const int cnt = p.counts ? min(max(p.counts[b], 0), p.T) : p.T;
  const int end = min(rows_end, cnt * p.G);  // rows of real tokens
  last = end > row0 ? max(-1, min(p.pos[b] + (end - 1) / p.G, p.limit - 1)) : -1;
  return (last + kKv8Block) / kKv8Block;
}

// This warp's way through the blocks of its CTA's run.
struct Cursor {
  int b, h;        // sequence, KV head
  int blocks, last;  // the sequence's visible blocks, and its last visible slot
  int blk, end;    // next block of this warp in the head, and the run's end in it
  int64_t left;    // blocks of the run in the heads after this one
};

template <int D, int FMT, bool HL>
__global__ void __launch_bounds__(kWarps * 32) kv8_attend_kernel(const __grid_constant__ AttendParams p) {
  constexpr int kSlot = kKv8Block * D, kSlots = D == 128 ? 3 : 4;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) unsigned long long bars[kWarps][kSlots];
  __shared__ float s_m[kWarps][16], s_l[kWarps][16];
  __shared__ long long s_total;
  __shared__ int s_b, s_last;
  __shared__ long long s_before;
  float* s_join = reinterpret_cast<float*>(smem + kWarps * kSlots * kSlot);  // [2][16 * D]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const int H = p.c.n_kv_heads, B = p.c.batch;
  const int row0 = blockIdx.y * 16, rows_end = min(row0 + 16, p.rows);
  const int64_t cta = blockIdx.x;

  // ------------------------------------------- this CTA's run of blocks
  if (tid == 0) s_total = 0;
  __syncthreads();
  {
    long long mine = 0;
    int last;
    for (int b = tid; b < B; b += kWarps * 32) mine += visible_blocks(p, b, row0, rows_end, last);
    if (mine) atomicAdd(reinterpret_cast<unsigned long long*>(&s_total), (unsigned long long)mine);
  }
  __syncthreads();
  const int64_t all = s_total * H;  // every run holds a block: fewer CTAs work where there are fewer
  const int64_t ctas = min((long long)gridDim.x, (long long)all);
  // heads without a visible slot belong to no run
  for (int b = (int)cta; b < B; b += (int)gridDim.x) {
    int last;
    if (visible_blocks(p, b, row0, rows_end, last) == 0)
      for (int e = tid; e < H * (rows_end - row0) * (D / 4); e += kWarps * 32) {
        const int h = e / ((rows_end - row0) * (D / 4)), r = row0 + e / (D / 4) % (rows_end - row0);
        write_row(p, b, h, r, e % (D / 4) * 4, make_float4(0, 0, 0, 0), -INFINITY, 0.0f);
      }
  }
  if (cta >= ctas) return;
  const int64_t u0 = cta * all / ctas, u1 = (cta + 1) * all / ctas;
  // the sequence that holds block u0
  long long base = 0;  // blocks (of one head) of the sequences before this tile of them
  for (int b0 = 0; b0 < B; b0 += kWarps * 32) {
    const int b = b0 + tid;
    int last;
    const int mine = b < B ? visible_blocks(p, b, row0, rows_end, last) : 0;
    int x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) s_m[warp][0] = __int_as_float(x);
    __syncthreads();
    long long before = base + x - mine, tile = 0;
    for (int w = 0; w < kWarps; ++w) {
      const int n = __float_as_int(s_m[w][0]);
      before += w < warp ? n : 0;
      tile += n;
    }
    if (mine && before * H <= u0 && u0 < (before + mine) * H) {
      s_b = b;
      s_before = before;
    }
    base += tile;
    if (base * H > u0) break;
  }
  __syncthreads();

  Cursor at;
  at.b = s_b;
  at.blocks = visible_blocks(p, at.b, row0, rows_end, at.last);
  {
    const int64_t in = u0 - s_before * H;  // blocks of this sequence's heads before the run
    at.h = (int)(in / at.blocks);
    const int off = (int)(in % at.blocks);
    at.end = (int)min((int64_t)at.blocks, off + (u1 - u0));
    at.blk = off + warp;
    at.left = u1 - u0 - (at.end - off);
  }
  auto next_head = [&](Cursor& c) {
    if (++c.h == H) {
      c.h = 0;
      do ++c.b;
      while ((c.blocks = visible_blocks(p, c.b, row0, rows_end, c.last)) == 0);
    }
    c.end = (int)min((int64_t)c.blocks, c.left);
    c.left -= c.end;
    c.blk = warp;
  };

  // ----------------------------------------------------- the warp's ring
  const uint32_t bar0 = smem_u32(&bars[warp][0]);
  uint8_t* ring = smem + warp * kSlots * kSlot;
  if (lane == 0) {
    for (int i = 0; i < kSlots; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar0 + 8 * i));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  Cursor ahead = at;   // what is copied next: K of its block, then V
  bool more = true, ahead_v = false;
  int put = 0;         // copies issued
  bool ok = true;
  auto find = [&] {    // to the warp's next block, if it has one left
    while (more && ahead.blk >= ahead.end) {
      if (ahead.left > 0) next_head(ahead);
      else more = false;
    }
  };
  auto copy = [&] {
    find();
    if (!more || !ok) return;
    if (lane == 0) {
      const uint32_t bar = bar0 + 8 * (put % kSlots);
      const uint8_t* src = (ahead_v ? p.c.v : p.c.k) +
                           (((int64_t)ahead.b * H + ahead.h) * p.c.max_len + (int64_t)ahead.blk * kKv8Block) * D;
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "n"(kSlot) : "memory");
      asm volatile(
          "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
              smem_u32(ring + put % kSlots * kSlot)),
          "l"(src), "n"(kSlot), "r"(bar)
          : "memory");
    }
    ++put;
    if (ahead_v) ahead.blk += kWarps;
    ahead_v = !ahead_v;
  };
  for (int i = 0; i < kSlots; ++i) copy();
  int got = 0;  // copies waited for; after a wait that gave up, only those in flight
  auto arrive = [&]() -> const uint8_t* {
    if (got < put && !mbar_wait(bar0 + 8 * (got % kSlots), (got / kSlots) & 1)) ok = false;
    return ring + got++ % kSlots * kSlot;
  };

  while (true) {
    const int64_t head = (int64_t)at.b * H + at.h;
    const int first = at.blk - warp, seg_end = at.end;  // the run's blocks in this head
    const int pos = p.pos[at.b], cnt = p.counts ? min(max(p.counts[at.b], 0), p.T) : p.T;
    const int lim[2] = {row_limit(p, row0 + g, pos, cnt), row_limit(p, row0 + g + 8, pos, cnt)};
    const float* ksc = p.c.k_scale + head * (p.c.max_len / kKv8Block);
    const float* vsc = p.c.v_scale + head * (p.c.max_len / kKv8Block);
    uint32_t qh[D / 16][4], ql[HL ? D / 16 : 1][4];
    float back[2];
    float ks = 0.0f, vs = 0.0f;
    if (at.blk < seg_end) {
      ks = __ldg(ksc + at.blk);
      vs = __ldg(vsc + at.blk);
    }
    load_q<D, HL>(p, at.b, at.h, row0, qh, ql, back);
    float o[D / 8][4] = {};
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

    for (; at.blk < seg_end; at.blk += kWarps) {
      const float f0 = back[0] * ks, f1 = back[1] * ks, vsn = vs;
      if (at.blk + kWarps < seg_end) {
        ks = __ldg(ksc + at.blk + kWarps);
        vs = __ldg(vsc + at.blk + kWarps);
      }
      float c[8][4];
      const uint8_t* kb = arrive();
      scores<D, FMT, HL>(kb, qh, ql, c);
      __syncwarp();
      copy();  // into the slot of these keys
      const int key0 = at.blk * kKv8Block;
      float top[2] = {-INFINITY, -INFINITY};
      const bool whole = key0 + kKv8Block - 1 <= lim[0] && key0 + kKv8Block - 1 <= lim[1];
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int half = i >> 1;
          c[j][i] *= half ? f1 : f0;
          if (!whole && key0 + key_of(j, i) > lim[half]) c[j][i] = -INFINITY;
          top[half] = fmaxf(top[half], c[j][i]);
        }
      if (p.scores) {
        // log2 units, for the rows' attention weights
#pragma unroll
        for (int half = 0; half < 2; ++half)
          if (row0 + g + 8 * half < p.rows) {
            float* x = p.scores + (head * p.rows + row0 + g + 8 * half) * p.ld_scores + key0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              x[key_of(j, 0)] = c[j][2 * half];
              x[key_of(j, 1)] = c[j][2 * half + 1];
            }
          }
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
      const uint8_t* vb = arrive();
      const bool tail = key0 + kKv8Block > at.last + 1;  // the block ends past the last visible slot
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
          if (tail && key0 + key > at.last)
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
      __syncwarp();
      copy();  // into the slot of these values
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][i] = fmaf(pv[n][i], vsn, o[n][i] * alpha[i >> 1]);
    }

    // join the warps: 2 and 3 into 0 and 1, then 1 into 0
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
      l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
    }
#pragma unroll
    for (int step = kWarps / 2; step > 0; step >>= 1) {
      if (warp >= step && warp < 2 * step) {
        float* to = s_join + (warp - step) * 16 * D;
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) to[(n * 4 + i) * 32 + lane] = o[n][i];
        if (t4 == 0) {
          s_m[warp][g] = m[0], s_m[warp][g + 8] = m[1];
          s_l[warp][g] = l[0], s_l[warp][g + 8] = l[1];
        }
      }
      __syncthreads();
      if (warp < step) {
        const float* from = s_join + warp * 16 * D;
        float a[2], c[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float om = s_m[warp + step][g + 8 * half], now = fmaxf(m[half], om);
          a[half] = m[half] == -INFINITY ? 0.0f : exp2a(m[half] - now);
          c[half] = om == -INFINITY ? 0.0f : exp2a(om - now);
          l[half] = l[half] * a[half] + s_l[warp + step][g + 8 * half] * c[half];
          m[half] = now;
        }
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            o[n][i] = o[n][i] * a[i >> 1] + from[(n * 4 + i) * 32 + lane] * c[i >> 1];
      }
      __syncthreads();
    }
    // parts of this head: from the CTA with its first block to the one with its last
    const int64_t head_u = u0 + (u1 - u0) - at.left - (seg_end - first) - first;  // its first block's number
    const int64_t c0 = ((head_u + 1) * ctas - 1) / all, c1 = ((head_u + at.blocks) * ctas - 1) / all;
    const int64_t slot = (cta + head) * 16;
    if (warp == 0) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int rr = g + 8 * half, r = row0 + rr;
        if (r >= p.rows) continue;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int n = 0; n < D / 8; n += (D / 8 < 4 ? 2 : 4)) {
            const int d = (2 * t4 + i) * (D / 8) + n;
            if constexpr (D / 8 >= 4) {
              const float4 v = make_float4(o[n][2 * half + i], o[n + 1][2 * half + i], o[n + 2][2 * half + i], o[n + 3][2 * half + i]);
              *reinterpret_cast<float4*>(p.part_o + ((int64_t)blockIdx.y * p.part_rows + slot + rr) * D + d) = v;
            } else {
              *reinterpret_cast<float2*>(p.part_o + ((int64_t)blockIdx.y * p.part_rows + slot + rr) * D + d) =
                  make_float2(o[n][2 * half + i], o[n + 1][2 * half + i]);
            }
          }
        if (t4 == 0)
          *reinterpret_cast<float2*>(p.part_ml + ((int64_t)blockIdx.y * p.part_rows + slot + rr) * 2) =
              make_float2(m[half], l[half]);
      }
      __threadfence();
    }
    __syncthreads();
    if (tid == 0) {
      int* count = p.arrived + (int64_t)blockIdx.y * (int64_t)B * H + head;
      const int last = atomicAdd(count, 1) == (int)(c1 - c0);
      if (last) *count = 0;  // as the next call finds it
      s_last = last;
    }
    __syncthreads();
    if (s_last) {
      __threadfence();
      const int64_t part0 = (int64_t)blockIdx.y * p.part_rows + (c0 + head) * 16;
      const int parts = (int)(c1 - c0) + 1, rows = rows_end - row0;
      for (int e = tid; e < rows * (D / 4); e += kWarps * 32) {
        const int rr = e / (D / 4), d = e % (D / 4) * 4;
        float mm = -INFINITY;
        for (int q = 0; q < parts; ++q) mm = fmaxf(mm, __ldcg(p.part_ml + 2 * (part0 + 16 * q + rr)));
        float ll = 0.0f;
        float4 oo = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (mm > -INFINITY) {
#pragma unroll 4
          for (int q = 0; q < parts; ++q) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.part_ml) + part0 + 16 * q + rr);
            const float4 v = __ldcg(reinterpret_cast<const float4*>(p.part_o + (part0 + 16 * q + rr) * D + d));
            const float f = exp2a(ml.x - mm);
            ll = fmaf(ml.y, f, ll);
            oo.x = fmaf(v.x, f, oo.x), oo.y = fmaf(v.y, f, oo.y);
            oo.z = fmaf(v.z, f, oo.z), oo.w = fmaf(v.w, f, oo.w);
          }
        }
        write_row(p, at.b, at.h, row0 + rr, d, oo, mm, ll);
      }
    }
    if (at.left == 0) break;
    next_head(at);
  }
  if (!ok) set_status(p.status, CB_ERR_TIMEOUT);
}

// Joins the runs' parts of one row of the prompt form, in order: one CTA of D threads per row.
__global__ void kv8_join_kernel(const __grid_constant__ AttendParams p) {
  const int D = p.c.head_dim, d = threadIdx.x;
  const int r = blockIdx.x;
  const int64_t head = blockIdx.y;
  const int hk = (int)(head % p.c.n_kv_heads), b = (int)(head / p.c.n_kv_heads);
  const int64_t at = (head * p.rows + r) * p.splits;
  float mm = -INFINITY;
  for (int s = 0; s < p.splits; ++s) mm = fmaxf(mm, p.part_ml[2 * (at + s)]);
  float ll = 0.0f;
  float4 oo = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (mm > -INFINITY)
    for (int s = 0; s < p.splits; ++s) {
      const float f = exp2a(p.part_ml[2 * (at + s)] - mm);
      const float4 v = *reinterpret_cast<const float4*>(p.part_o + (at + s) * D + 4 * d);
      ll = fmaf(p.part_ml[2 * (at + s) + 1], f, ll);
      oo.x = fmaf(v.x, f, oo.x), oo.y = fmaf(v.y, f, oo.y);
      oo.z = fmaf(v.z, f, oo.z), oo.w = fmaf(v.w, f, oo.w);
    }
  write_row(p, b, hk, r, 4 * d, oo, mm, ll);
}

// mass_j += sum_r exp(x[r][j] - lse_r) from the scores that the attention left: four
// keys a thread.
__global__ void __launch_bounds__(256) kv8_scores_mass_kernel(const __grid_constant__ AttendParams p) {
  const int64_t head = blockIdx.y;
  const int b = (int)(head / p.c.n_kv_heads), hk = (int)(head % p.c.n_kv_heads);
  const int key = (blockIdx.x * 256 + threadIdx.x) * 4;
  int last;
  visible_blocks(p, b, 0, p.rows, last);
  if (key > last) return;
  float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int r = 0; r < p.rows; ++r) {
    const float lse = p.lse[((int64_t)b * p.T + r / p.G) * (p.G * p.c.n_kv_heads) + hk * p.G + r % p.G] * kLog2e;
    if (lse == -INFINITY) continue;  // its scores were not all written
    const float4 x = *reinterpret_cast<const float4*>(p.scores + (head * p.rows + r) * p.ld_scores + key);
    sum.x += exp2a(x.x - lse), sum.y += exp2a(x.y - lse);
    sum.z += exp2a(x.z - lse), sum.w += exp2a(x.w - lse);
  }
  float* to = p.c.mass + head * p.c.max_len + key;
  const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (key + i <= last) to[i] += v[i];
}

// mass_j += sum_r exp(x[r][j] - lse_r): a warp owns a block of 64 keys and walks
// the head's query rows 16 at a time, so every slot has one writer and one order.
template <int D, int FMT, bool HL>
__global__ void __launch_bounds__(kWarps * 32) kv8_mass_kernel(const __grid_constant__ AttendParams p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2;
  const int hk = blockIdx.y % p.c.n_kv_heads, b = blockIdx.y / p.c.n_kv_heads;
  const int pos = p.pos[b], cnt = p.counts ? min(max(p.counts[b], 0), p.T) : p.T;
  const int last = cnt > 0 ? min(pos + cnt, p.limit) - 1 : -1;
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
    if (p.splits > 1) {
      kv8_join_kernel<<<dim3(p.rows, bh), D / 4, 0, st>>>(p);
      count_launch();
    }
    if (p.add_mass) return kv8_prompt_mass_launch(p, bh, longest, st);
  } else {
    const int smem = kWarps * (D == 128 ? 3 : 4) * kKv8Block * D + 2 * 16 * D * (int)sizeof(float);
    auto fn = kv8_attend_kernel<D, FMT, HL>;
    if (const int rc = ensure_smem_attr((const void*)fn, smem)) return rc;
    fn<<<dim3(p.splits, ceil_div(p.rows, 16)), kWarps * 32, smem, st>>>(p);
    count_launch();
    if (p.scores) {
      kv8_scores_mass_kernel<<<dim3(ceil_div(longest, 1024), bh), 256, 0, st>>>(p);
      count_launch();
    } else if (p.add_mass) {
      kv8_mass_kernel<D, FMT, HL><<<dim3(ceil_div(longest, kWarps * kKv8Block), bh), kWarps * 32, 0, st>>>(p);
      count_launch();
    }
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

// How a call is cut up, and where its parts lie in the scratch.  The counters come
// first, in every call's layout: they are zero between calls.
constexpr size_t kCounters = 65536;
struct Plan {
  int rows = 0, row_tiles = 0, splits = 0;
  int64_t part_rows = 0, ld_scores = 0;
  size_t ml = 0, o = 0, q16 = 0, back = 0, scores = 0, bytes = 0;
};

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

Plan plan_of(const CbKv8& c, int dtype, int n_q_heads, int T, int longest, bool add_mass) {
  Plan pl;
  const int bh = c.batch * c.n_kv_heads;
  pl.rows = T * (n_q_heads / c.n_kv_heads);
  pl.ml = kCounters * sizeof(int);
  int64_t parts;
  // From 33 rows on the tensor cores' 128-row tiles pay for the rows they leave empty.
  if (pl.rows > 32 && c.head_dim >= 64 && dtype != CB_F32) {
    pl.row_tiles = ceil_div(pl.rows, 128);
    // runs of key tiles that leave the fewest tile times (and three more a CTA to
    // start and end) on the busiest SM
    const int items = bh * ceil_div(pl.row_tiles, 2), tiles = ceil_div(longest, 8192 / c.head_dim);
    long best = 0;
    for (int s = 1; s <= 32 && s <= ceil_div(tiles, 2); ++s) {
      const long cost = (long)ceil_div(items * s, num_sms()) * (ceil_div(tiles, s) + 3);
      if (pl.splits == 0 || cost < best) {
        pl.splits = s;
        best = cost;
      }
    }
    parts = (int64_t)bh * pl.rows * pl.splits;
  } else {
    // CTAs that are resident at once (three to an SM of 48 KB rings, two of 96), at
    // least one block of 64 keys for each warp, and no more than 48 parts a head
    const int blocks = ceil_div(pl.rows, 16);
    const int64_t fit = std::max(1, num_sms() * (c.head_dim == 128 ? 2 : 3) / blocks);
    const int64_t work = std::max<int64_t>(1, (int64_t)bh * ceil_div(longest, kKv8Block) / kWarps);
    pl.splits = (int)std::min(std::min(fit, work), (int64_t)bh * 48);
    pl.part_rows = ((int64_t)bh + pl.splits) * 16;
    parts = pl.part_rows * blocks;
    // rows' scores cost 8 bytes a key to write and read, taking them again head_dim
    if (add_mass && pl.rows * 8 <= c.head_dim) pl.ld_scores = ceil_div(longest, kKv8Block) * kKv8Block;
  }
  pl.o = pl.ml + align256((size_t)parts * 2 * sizeof(float));
  pl.q16 = pl.o + align256((size_t)parts * c.head_dim * sizeof(float));
  pl.back = pl.q16 + (size_t)bh * pl.row_tiles * 128 * c.head_dim * 2;
  pl.scores = pl.back + (size_t)bh * pl.row_tiles * 128 * sizeof(float);
  pl.bytes = pl.scores + (size_t)bh * pl.rows * pl.ld_scores * sizeof(float);
  return pl;
}

int check_call(const CbKv8* c, int dtype, int n_q_heads, int T, int longest) {
  if (const int rc = kv8_check(c)) return rc;
  if (T <= 0 || longest <= 0 || !kv8_dtype_ok(dtype)) return CB_ERR_ARG;
  if (n_q_heads <= 0 || n_q_heads % c->n_kv_heads) return CB_ERR_SHAPE;
  const int64_t rows = (int64_t)T * (n_q_heads / c->n_kv_heads);
  if (rows > 65535 * 16) return CB_ERR_SHAPE;
  // a counter for each head and 16 rows
  if ((rows <= 32 || dtype == CB_F32 || c->head_dim < 64) &&
      (rows + 15) / 16 * c->batch * c->n_kv_heads > (int64_t)kCounters)
    return CB_ERR_SHAPE;
  return CB_OK;
}

}  // namespace
}  // namespace cb

using namespace cb;

extern "C" size_t cb_kv8_attend_scratch_bytes(const CbKv8* c, int32_t dtype, int32_t n_q_heads, int32_t T,
                                              int32_t longest, int32_t add_mass) {
  if (check_call(c, dtype, n_q_heads, T, longest) != CB_OK) return 0;
  return plan_of(*c, dtype, n_q_heads, T, std::min(longest, c->max_len), add_mass != 0).bytes;
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
  const Plan pl = plan_of(*c, dtype, n_q_heads, T, longest, add_mass != 0);
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
  p.limit = longest;
  p.scale = scale;
  p.add_mass = add_mass != 0;
  p.out = out;
  p.lse = lse;
  p.splits = pl.splits;
  uint8_t* base = static_cast<uint8_t*>(scratch);
  p.arrived = reinterpret_cast<int*>(base);
  p.part_ml = reinterpret_cast<float*>(base + pl.ml);
  p.part_rows = pl.part_rows;
  p.ld_scores = pl.ld_scores;
  p.scores = pl.ld_scores ? reinterpret_cast<float*>(base + pl.scores) : nullptr;
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
