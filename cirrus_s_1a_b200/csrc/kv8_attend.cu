// Attention over the 8-bit K/V cache: cb_kv8_attend.
//
//   x[r][j] = q_r . k_j * scale      j <= pos[b] + t   (k_j = code * block scale)
//   lse_r   = log sum_j exp(x[r][j])
//   out_r   = sum_j exp(x[r][j] - lse_r) v_j
//   mass_j += sum over the KV head's rows r of exp(x[r][j] - lse_r)     (add_mass)
//
// The rows of a KV head are its G query heads of the T tokens, r = t * G + g, so
// the codes are read once for all of them.  kv8_attend_kernel runs on warp-level
// matrix products (m16n8k16, f16 operands, f32 sums) with the codes as their left
// operand: 16 keys, or 16 dims, by 8 NT query rows, so that a decode step's few rows
// leave half of an 8-row operand empty, not of a 16-row one.  Codes are exact in
// f16; the products' free index order is used so that no operand needs a transpose
// through shared memory:
//   * S^T = K Q^T: lane (g, t) = (lane / 4, lane % 4) reads D/4 contiguous bytes of
//     a key row, so a warp's load covers whole rows; the four k positions a lane
//     feeds in step s are the dims t * D/4 + 4 s .. + 3, and the query fragments are
//     loaded in that order.
//   * O^T = V^T P^T: P leaves the softmax with keys along lanes and is turned by
//     movmatrix, 8 x 8 at a time.  Row i of an 8-key group is its key
//     4 (i & 1) + i / 2, so the four keys a lane feeds in a step are t + {0, 4, 8,
//     12}: four rows in a row across t.  The lane reads D/8 contiguous bytes of each
//     (dims g * D/8 ..) and pairs the keys' bytes with byte permutes.
// Queries: a row is scaled by a power of two that brings its largest element to
// [256, 512) and rounded to f16.  bf16 and f16 queries are exact in that (up to
// 2^-33 of the row's largest element); float32 queries and their P are carried
// as a head and a tail (about 22 bits), two products each, and each block's product
// is added up in float32 registers.  f16 P (11 bits) for 16-bit outputs adds less
// than the output's own rounding.
// With x = S * a_b (a_b = row factor * block b's key scale, log2 units) and e_b the
// exponent of its value scale, P = exp2(x + e_b - m') against m' = max (x + e_b):
// P times the bare codes is the sum over values, its f16 rounding relative to what
// the row adds up, whatever the blocks' scales.  The row's sum is
// l 2^m', l = sum_b 2^-e_b sum P, added up against an exponent e_ref near the blocks' own;
// blocks far below it (zeros) are summed for themselves (kNear).
// out = O / l.  O is rescaled only when m' has grown by more than 2^12
// (float32: 2^15, and m' is 11 powers below the maximum, for the tails).
// Softmax statistics and the joins of parts are float32.
//
// Work is dealt out by blocks of 64 keys: the visible blocks of all KV heads, one
// after another, are cut into equal runs, one per CTA (with sequences of different
// lengths, equal runs of each head left half of the SMs idle).  A run that crosses
// heads leaves a part for each; (CTA + head) numbers the parts without a table.
// Each warp takes every fourth block of a run; K and V blocks arrive by bulk copies
// in a ring of slots of its own, two or three ahead, across the ends of heads.  The
// CTA that finishes a head last joins its parts in their order and writes the
// output, so a call is one launch (two with attention weights).
//
// Bound by memory in principle (2 D bytes a key for all rows of its head), by issue
// and the latency of its chains in fact.  Measured: 64 sequences x 1 token at 32K,
// 128 dims, E4M3, with weights 221 us, 5 TB/s in the attention itself (30 % of
// issue slots); 16 x 5 tokens at up to 128K, 64 dims, int8 155 to 172 us, 4 TB/s (53 % of
// issue slots, 49 % of the integer pipe: int8 codes take 5 instructions for four,
// E4M3 two); one token at 32K 18 us, of which the blocks take 4, placing the CTA and
// the query 4, and joining 48 parts the rest.  Prompts of 16 and 32 dims: 1000 tokens at 8K,
// 16 dims (2 heads, bf16) 38 us, with weights 218; 32 dims (4 heads, float32) 66 and 152.
#include <algorithm>
#include <climits>

#include "kv8.cuh"
#include "kv8_attend.cuh"

namespace cb {
namespace {

constexpr int kWarps = 4;
// Growth of the maximum, in powers of two, that O follows (f16 P ends at 2^16), and what a
// row's largest P lies above 1 when it does: a tail of P then ends at 2^-35 of the largest.
template <bool HL>
constexpr float kLazy = HL ? 15.0f : 12.0f;
template <bool HL>
constexpr float kLift = HL ? 11.0f : 0.0f;
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

// Query rows row0 .. row0 + 8 NT - 1 of a KV head as right operands: lane (g, t)
// feeds row g of each eight.  `back`: the factors that undo the powers of two, times
// scale * log2(e), of the rows 2 t and 2 t + 1 that the lane's scores belong to.  A row with
// a NaN or an infinity is taken as zeros with a NaN for its factor, which makes NaN of its
// results.  HL: the tails too.
template <int D, bool HL, int NT>
struct Query {
  uint32_t h[NT][D / 16][2], l[HL ? NT : 1][HL ? D / 16 : 1][2];
  float back[NT][2];
  __device__ __forceinline__ void load(const AttendParams& p, int b, int hk, int row0) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = row0 + 8 * nt + g;
      float x[D / 4];
      float top = 0.0f;
      const bool live = r < p.rows;
      const int t = r / p.G, hq = hk * p.G + r % p.G;
      const int64_t base = (int64_t)b * p.qs[0] + (int64_t)t * p.qs[1] + hq * p.qs[2] + t4 * (D / 4);
      if (D >= 32 && p.q_wide) {  // rows of 16-byte pieces
        if (HL) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (live) v = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + base) + i);
            x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
          }
        } else {
          uint32_t w[D / 8];
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (live) v = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + base) + i);
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
          }
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            const float2 f = p.dtype == CB_BF16 ? make_float2(bf16_to_f32(w[i]), __uint_as_float(w[i] & 0xFFFF0000u))
                                                : __half22float2(bits_h2(w[i]));
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < D / 4; ++i) x[i] = live ? kv8_load(p.q, base + i, p.dtype) : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < D / 4; ++i) top = max_nan(top, fabsf(x[i]));
      top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const bool bad = !(top < INFINITY);
      int e = 0;  // top in [2^e, 2^(e+1)); rows of zeros keep e = 0
      if (top > 0.0f && !bad) e = max((__float_as_int(top) >> 23) - 127, -100);
      const float f = copysignf(kv8_pow2(8 - e), p.scale), undo = bad ? NAN : kv8_pow2(e - 8) * fabsf(p.scale) * kLog2e;
      back[nt][0] = __shfl_sync(0xffffffffu, undo, 8 * t4);
      back[nt][1] = __shfl_sync(0xffffffffu, undo, 8 * t4 + 4);
#pragma unroll
      for (int s = 0; s < D / 16; ++s)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float u = bad ? 0.0f : x[4 * s + 2 * i] * f, v = bad ? 0.0f : x[4 * s + 2 * i + 1] * f;
          const __half2 hd = __floats2half2_rn(u, v);
          h[nt][s][i] = h2_bits(hd);
          if (HL) {
            const float2 hb = __half22float2(hd);
            l[HL ? nt : 0][HL ? s : 0][i] = h2_bits(__floats2half2_rn(u - hb.x, v - hb.y));
          }
        }
    }
  }
};

// Key (within 16) behind row g (+ 8) of a left operand of keys.
__device__ __forceinline__ int key_row(int g) { return 4 * (g & 1) + (g >> 1); }

// S^T of 16 keys (codes) against the query rows: c[nt] is (key g, rows 2t, 2t + 1),
// (key g + 8, the same rows).
template <int D, int FMT, bool HL, int NT>
__device__ __forceinline__ void scores(const uint8_t* kb, const Query<D, HL, NT>& q, float (&c)[NT][4]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  uint32_t w0[D / 16], w1[D / 16];
  load_bytes<D / 4>(kb + key_row(g) * D + t4 * (D / 4), w0);
  load_bytes<D / 4>(kb + (8 + key_row(g)) * D + t4 * (D / 4), w1);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) c[nt][0] = c[nt][1] = c[nt][2] = c[nt][3] = 0.0f;
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    uint32_t a[4];
    codes_to_h2<FMT>(w0[s], a[0], a[2]);
    codes_to_h2<FMT>(w1[s], a[1], a[3]);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      mma16816(c[nt], a, q.h[nt][s][0], q.h[nt][s][1]);
      if (HL) mma16816(c[nt], a, q.l[HL ? nt : 0][HL ? s : 0][0], q.l[HL ? nt : 0][HL ? s : 0][1]);
    }
  }
}

__device__ __forceinline__ uint32_t turn(uint32_t m) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(m));
  return r;
}

// The last slot query row r sees; -1: none.
__device__ __forceinline__ int row_limit(const AttendParams& p, int r, int pos, int cnt) {
  const int t = r / p.G;
  if (r >= p.rows || t >= cnt) return -1;
  return min(pos + t, p.limit - 1);
}

// Writes the output and lse of one row's four dims: `o` against the sum's m.
__device__ __forceinline__ void write_row(const AttendParams& p, int b, int hk, int r, int d, float4 o, Sum s) {
  const int64_t at = ((int64_t)b * p.T + r / p.G) * (p.G * p.c.n_kv_heads) + hk * p.G + r % p.G;
  const bool none = s.m == -INFINITY;
  const Inverse by(none ? 1.0f : s.l);
  if (none) o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  const float y[4] = {by.of(o.x), by.of(o.y), by.of(o.z), by.of(o.w)};
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
  if (d == 0) {
    const float lse2 = none ? -INFINITY : s.m + log2f(s.l);
    p.lse[at] = lse2 * kLn2;
    if (p.add_mass) p.lse2[((int64_t)b * p.c.n_kv_heads + hk) * p.rows + r] = lse2;
  }
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

template <int D>
constexpr int kRing = D == 128 ? 2 : 3;
// CTAs of an SM to aim at
template <int D, bool HL, int NT>
constexpr int kResident = HL || NT == 4 ? 1 : D == 128 ? (NT == 1 ? 3 : 2) : (NT == 1 ? 4 : 3);

template <int D, int FMT, bool HL, int NT>
__global__ void __launch_bounds__(kWarps * 32, kResident<D, HL, NT>) kv8_attend_kernel(const __grid_constant__ AttendParams p) {
  constexpr int kSlot = kKv8Block * D, kSlots = kRing<D>, kRows = 8 * NT;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) unsigned long long bars[kWarps][kSlots];
  __shared__ Sum s_sum[kWarps][kRows], s_aside[2 * NT][kWarps * 32];
  __shared__ int s_scan[kWarps];
  __shared__ long long s_before;
  __shared__ int s_b, s_blocks, s_slot, s_last;
  float* s_join = reinterpret_cast<float*>(smem + kWarps * kSlots * kSlot);  // [2][kRows * D]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const int H = p.c.n_kv_heads, B = p.c.batch;
  const int row0 = (p.block0 + blockIdx.y) * kRows, rows_end = min(row0 + kRows, p.rows);
  const int64_t cta = blockIdx.x;

  // ------------------------------------------- this CTA's run of blocks
  // blocks (of one head) of the sequences before a thread's one in a tile of them
  auto scan = [&](int mine, long long& tile) {
    int x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) s_scan[warp] = x;
    __syncthreads();
    long long before = x - mine;
    tile = 0;
    for (int w = 0; w < kWarps; ++w) {
      const int n = s_scan[w];
      before += w < warp ? n : 0;
      tile += n;
    }
    return before;
  };
  long long total = 0, before = 0;
  int mine = 0, mine_last = -1;
  for (int b0 = 0; b0 < B; b0 += kWarps * 32) {
    const int b = b0 + tid;
    mine = b < B ? visible_blocks(p, b, row0, rows_end, mine_last) : 0;
    long long tile;
    before = total + scan(mine, tile);
    total += tile;
  }
  const int64_t all = total * H;  // every run holds a block: fewer CTAs work where there are fewer
  const int64_t ctas = min((long long)gridDim.x, (long long)all);
  // heads without a visible slot belong to no run
  for (int b = (int)cta; b < B; b += (int)gridDim.x) {
    int last;
    if (visible_blocks(p, b, row0, rows_end, last) == 0)
      for (int e = tid; e < H * (rows_end - row0) * (D / 4); e += kWarps * 32) {
        const int h = e / ((rows_end - row0) * (D / 4)), r = row0 + e / (D / 4) % (rows_end - row0);
        write_row(p, b, h, r, e % (D / 4) * 4, make_float4(0, 0, 0, 0), Sum{-INFINITY, 0.0f});
      }
  }
  if (cta >= ctas) return;
  const int64_t u0 = cta * all / ctas, u1 = (cta + 1) * all / ctas;
  // the sequence that holds block u0
  auto found = [&](int b) {
    if (mine && before * H <= u0 && u0 < (before + mine) * H) {
      s_b = b;
      s_blocks = mine;
      s_slot = mine_last;
      s_before = before;
    }
  };
  if (B <= kWarps * 32) {
    found(tid);
  } else {
    long long base = 0;
    for (int b0 = 0; base * H <= u0; b0 += kWarps * 32) {
      mine = b0 + tid < B ? visible_blocks(p, b0 + tid, row0, rows_end, mine_last) : 0;
      long long tile;
      before = base + scan(mine, tile);
      base += tile;
      found(b0 + tid);
    }
  }
  __syncthreads();

  Cursor at;
  at.b = s_b;
  at.blocks = s_blocks;
  at.last = s_slot;
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
  int put = 0, put_at = 0;  // copies issued, and the next one's slot
  bool ok = true;
  int64_t ahead_at = 0;  // its block in k and v
  auto locate = [&] { ahead_at = (((int64_t)ahead.b * H + ahead.h) * p.c.max_len + (int64_t)ahead.blk * kKv8Block) * D; };
  locate();
  auto copy = [&] {
    if (ahead.blk >= ahead.end) {  // to the warp's next block, if it has one left
      while (more && ahead.blk >= ahead.end) {
        if (ahead.left > 0) next_head(ahead);
        else more = false;
      }
      locate();
    }
    if (!more || !ok) return;
    if (lane == 0) {
      const uint32_t bar = bar0 + 8 * put_at;
      const uint8_t* src = (ahead_v ? p.c.v : p.c.k) + ahead_at;
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "n"(kSlot) : "memory");
      asm volatile(
          "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
              smem_u32(ring) + put_at * kSlot),
          "l"(src), "n"(kSlot), "r"(bar)
          : "memory");
    }
    ++put;
    if (++put_at == kSlots) put_at = 0;
    if (ahead_v) {
      ahead.blk += kWarps;
      ahead_at += kWarps * kSlot;
    }
    ahead_v = !ahead_v;
  };
  for (int i = 0; i < kSlots; ++i) copy();
  // copies waited for, the next one's slot and its phase; after a wait that gave up,
  // only those in flight
  int got = 0, got_at = 0, phase = 0;
  auto arrive = [&]() -> const uint8_t* {
    if (got < put && !mbar_wait(bar0 + 8 * got_at, phase)) ok = false;
    const uint8_t* slot = ring + got_at * kSlot;
    ++got;
    if (++got_at == kSlots) got_at = 0, phase ^= 1;
    return slot;
  };

  while (true) {
    const int64_t head = (int64_t)at.b * H + at.h;
    const int first = at.blk - warp, seg_end = at.end;  // the run's blocks in this head
    const int pos = p.pos[at.b], cnt = p.counts ? min(max(p.counts[at.b], 0), p.T) : p.T;
    const float* ksc = p.c.k_scale + head * (p.c.max_len / kKv8Block);
    const float* vsc = p.c.v_scale + head * (p.c.max_len / kKv8Block);
    float ks = 0.0f, vs = 1.0f;
    if (at.blk < seg_end) {
      ks = __ldg(ksc + at.blk);
      vs = __ldg(vsc + at.blk);
    }
    Query<D, HL, NT> q;
    q.load(p, at.b, at.h, row0);
    float o[D / 16][NT][4] = {};
    float m[NT][2], l[NT][2];  // of rows 2 t4, 2 t4 + 1; l: this lane's keys
    bool has_aside = false, far = false;
    int e_ref = kv8_exponent(vs);
    int lim[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        m[nt][i] = -INFINITY;
        l[nt][i] = 0.0f;
        lim[nt][i] = row_limit(p, row0 + 8 * nt + 2 * t4 + i, pos, cnt);
      }

    // blocks that end by here are seen whole by every row
    const int seen = cnt < p.T ? -1 : min(pos + row0 / p.G, p.limit - 1);
    for (; at.blk < seg_end; at.blk += kWarps) {
      const float kf = ks;
      const int ev = kv8_exponent(vs);
      if (abs(ev - e_ref) > kNear) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            Sum& s = s_aside[2 * nt + i][tid];
            if (!has_aside) s.clear();
            if (ev > e_ref) {
              s.add(m[nt][i], l[nt][i] * kv8_pow2(-e_ref));
              l[nt][i] = 0.0f;
            }
          }
        has_aside = true;
        e_ref = max(ev, e_ref);
      }
      if (at.blk + kWarps < seg_end) {
        ks = __ldg(ksc + at.blk + kWarps);
        vs = __ldg(vsc + at.blk + kWarps);
      }
      const int key0 = at.blk * kKv8Block;
      float c[4][NT][4];
      const uint8_t* kb = arrive();
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) scores<D, FMT, HL, NT>(kb + 16 * mt * D, q, c[mt]);
      __syncwarp();
      copy();  // into the slot of these keys
      const bool partly = key0 + kKv8Block - 1 > seen;  // the first row (or a row without a token) does not see all of it
      if (partly) {
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (key0 + 16 * mt + 8 * (i >> 1) + key_row(g) > lim[nt][i & 1]) c[mt][nt][i] = -INFINITY;
      }
      // the largest x + e of this lane's keys: only where one passes m' by kLazy do
      // the lanes of a row compare
      float a[NT][2], now[NT][2];
      bool any = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          a[nt][i] = max_nan(q.back[nt][i] * kf, 1.2e-38f);  // above 0: a masked score times it stays -infinity
          float t = fmaxf(c[0][nt][i], c[0][nt][i + 2]);
#pragma unroll
          for (int mt = 1; mt < 4; ++mt) t = fmaxf(fmaxf(t, c[mt][nt][i]), c[mt][nt][i + 2]);
          now[nt][i] = fmaf(t, a[nt][i], (float)ev);
          any = any || now[nt][i] > m[nt][i] + kLazy<HL>;  // -infinity passes nothing, anything passes -infinity
        }
      if (p.scores) {
        // log2 units, for the rows' attention weights
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (row0 + 8 * nt + 2 * t4 + i < p.rows) {
              float* x = p.scores + (head * p.rows + row0 + 8 * nt + 2 * t4 + i) * p.ld_scores + key0 + key_row(g);
#pragma unroll
              for (int mt = 0; mt < 4; ++mt) {
                x[16 * mt] = c[mt][nt][i] * a[nt][i];
                x[16 * mt + 8] = c[mt][nt][i + 2] * a[nt][i];
              }
            }
      }
      if (__any_sync(0xffffffffu, any)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float alpha[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float to = now[nt][i];
            to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, 4));
            to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, 8));
            to = fmaxf(m[nt][i], fmaxf(to, __shfl_xor_sync(0xffffffffu, to, 16)) - kLift<HL>);
            alpha[i] = m[nt][i] == -INFINITY ? 0.0f : exp2a(m[nt][i] - to);
            m[nt][i] = to;
            l[nt][i] *= alpha[i];
          }
#pragma unroll
          for (int j = 0; j < D / 16; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[j][nt][i] *= alpha[i & 1];
        }
        bool any_far = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) any_far = any_far || fabsf(m[nt][0]) > kFarScore || fabsf(m[nt][1]) > kFarScore;
        far = __any_sync(0xffffffffu, any_far);
      }
      const bool low = ev < e_ref - kNear;
      if (low) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (now[nt][i] > -INFINITY) {
              float sum = 0.0f;
#pragma unroll
              for (int mt = 0; mt < 4; ++mt)
                sum += exp2a(fmaf(c[mt][nt][i], a[nt][i], (float)ev) - now[nt][i]) +
                       exp2a(fmaf(c[mt][nt][i + 2], a[nt][i], (float)ev) - now[nt][i]);
              s_aside[2 * nt + i][tid].add(now[nt][i], sum * kv8_pow2(-ev));
            }
      }
      const float back_l = low ? 0.0f : kv8_pow2(e_ref - ev);
      float add[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) add[nt][i] = (float)ev - (m[nt][i] == -INFINITY ? 0.0f : m[nt][i]);
      if (far) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (m[nt][i] > -INFINITY) {
#pragma unroll
              for (int mt = 0; mt < 4; ++mt)
#pragma unroll
                for (int half = 0; half < 4; half += 2)
                  c[mt][nt][i + half] = min_nan(fmaf(c[mt][nt][i + half], a[nt][i], (float)ev) - m[nt][i], kFarMost);
              a[nt][i] = 1.0f;
              add[nt][i] = 0.0f;
            }
      }
      const uint8_t* vb = arrive();
      bool any_nan = false;
      float pv[HL ? D / 16 : 1][HL ? NT : 1][4] = {};
      float sum[NT][2] = {};
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        uint32_t ph[NT][2], pl[HL ? NT : 1][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float e[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              e[i] = exp2a(fmaf(c[s][nt][2 * half + i], a[nt][i], add[nt][i]));
              sum[nt][i] += e[i];
            }
            const __half2 h = __floats2half2_rn(e[0], e[1]);
            ph[nt][half] = turn(h2_bits(h));
            if (HL) {
              const float2 hb = __half22float2(h);
              pl[HL ? nt : 0][half] = turn(h2_bits(__floats2half2_rn(e[0] - hb.x, e[1] - hb.y)));
            }
          }
        constexpr int NB = D / 8;  // bytes of a key row this lane feeds
        uint32_t w[4][(NB + 3) / 4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int key = 16 * s + 4 * u + t4;
          load_bytes<NB>(vb + key * D + g * NB, w[u]);
          if (partly) {
            // 0 * NaN is not 0: slots no row sees may hold anything and read as 0, and so do
            // E4M3 NaNs, which then reach the rows that see them below
#pragma unroll
            for (int z = 0; z < (NB + 3) / 4; ++z) {
              if (key0 + key > at.last) w[u][z] = 0u;
              if (FMT == CB_KV8_E4M3) {
                const uint32_t nan = __vcmpeq4(w[u][z] & 0x7F7F7F7Fu, 0x7F7F7F7Fu);
                w[u][z] &= ~nan;
                any_nan = any_nan || nan;
              }
            }
          }
        }
#pragma unroll
        for (int z = 0; z < (NB + 3) / 4; ++z)
#pragma unroll
          for (int y = 0; y < (NB < 4 ? 1 : 2); ++y) {
            // keys' bytes side by side: dims 4z + 2y and 4z + 2y + 1, rows g and g + 8 of the operand
            const uint32_t sel = y ? 0x7362u : 0x5140u;
            uint32_t va[4];
            codes_to_h2<FMT>(__byte_perm(w[0][z], w[1][z], sel), va[0], va[1]);
            codes_to_h2<FMT>(__byte_perm(w[2][z], w[3][z], sel), va[2], va[3]);
            const int j = 2 * z + y;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (HL) {
                mma16816(pv[HL ? j : 0][HL ? nt : 0], va, ph[nt][0], ph[nt][1]);
                mma16816(pv[HL ? j : 0][HL ? nt : 0], va, pl[HL ? nt : 0][0], pl[HL ? nt : 0][1]);
              } else {
                mma16816(o[j][nt], va, ph[nt][0], ph[nt][1]);
              }
            }
          }
      }
      if (FMT == CB_KV8_E4M3 && partly && __any_sync(0xffffffffu, any_nan)) {
        // the first NaN of each of this lane's dims, for the rows that see it
#pragma unroll
        for (int y = 0; y < D / 8; ++y) {
          int first = INT_MAX;
#pragma unroll 1
          for (int key = 63; key >= 0; --key)
            if (key0 + key <= at.last && (vb[key * D + g * (D / 8) + y] & 0x7F) == 0x7F) first = key0 + key;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (first <= lim[nt][i]) o[y / 2][nt][2 * (y & 1) + i] = NAN;
        }
      }
      __syncwarp();
      copy();  // into the slot of these values
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 2; ++i) l[nt][i] = fmaf(sum[nt][i], back_l, l[nt][i]);
        if (HL)
#pragma unroll
          for (int j = 0; j < D / 16; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[j][nt][i] += pv[HL ? j : 0][HL ? nt : 0][i];
      }
    }

    // join the warps: 2 and 3 into 0 and 1, then 1 into 0
    const float undo = kv8_pow2(-e_ref);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[nt][i] *= undo;
        if (has_aside) {  // (its m passes the row's by no more than a maximum lags)
          const Sum s = s_aside[2 * nt + i][tid];
          const float g = Sum::half(s.m, m[nt][i]);
          l[nt][i] += s.l * g * g;
        }
        float v = l[nt][i];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        l[nt][i] = v + __shfl_xor_sync(0xffffffffu, v, 16);
        // NaN scores raise no maximum, but the row has seen something all the same
        if (l[nt][i] != l[nt][i] && lim[nt][i] >= 0 && m[nt][i] == -INFINITY) m[nt][i] = 0.0f;
      }
#pragma unroll
    for (int step = kWarps / 2; step > 0; step >>= 1) {
      if (warp >= step && warp < 2 * step) {
        float* to = s_join + (warp - step) * kRows * D;
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) to[((j * NT + nt) * 4 + i) * 32 + lane] = o[j][nt][i];
        if (g == 0)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              s_sum[warp][8 * nt + 2 * t4 + i] = Sum{m[nt][i], l[nt][i]};
            }
      }
      __syncthreads();
      if (warp < step) {
        const float* from = s_join + warp * kRows * D;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float mine[2], theirs[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            Sum s{m[nt][i], l[nt][i]};
            const Sum other = s_sum[warp + step][8 * nt + 2 * t4 + i];
            const float2 f = s.add(other.m, other.l);
            mine[i] = f.x;
            theirs[i] = f.y;
            m[nt][i] = s.m;
            l[nt][i] = s.l;
          }
#pragma unroll
          for (int j = 0; j < D / 16; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              o[j][nt][i] = o[j][nt][i] * mine[i & 1] + from[((j * NT + nt) * 4 + i) * 32 + lane] * theirs[i & 1];
        }
      }
      __syncthreads();
    }
    // parts of this head: from the CTA with its first block to the one with its last
    const int64_t head_u = u0 + (u1 - u0) - at.left - (seg_end - first) - first;  // its first block's number
    const int64_t c0 = ((head_u + 1) * ctas - 1) / all, c1 = ((head_u + at.blocks) * ctas - 1) / all;
    const int64_t slot = (int64_t)blockIdx.y * p.part_rows + (cta + head) * kRows;
    if (warp == 0) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int rr = 8 * nt + 2 * t4 + i;
          if (row0 + rr >= p.rows) continue;
          float* to = p.part_o + (slot + rr) * D + g * (D / 8);
          if constexpr (D >= 32) {
#pragma unroll
            for (int j = 0; j < D / 16; j += 2)
              *reinterpret_cast<float4*>(to + 2 * j) =
                  make_float4(o[j][nt][i], o[j][nt][i + 2], o[j + 1][nt][i], o[j + 1][nt][i + 2]);
          } else {
            *reinterpret_cast<float2*>(to) = make_float2(o[0][nt][i], o[0][nt][i + 2]);
          }
          if (g == 0) p.part_ml[slot + rr] = Sum{m[nt][i], l[nt][i]};
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
      const int64_t part0 = (int64_t)blockIdx.y * p.part_rows + (c0 + head) * kRows;
      const int parts = (int)(c1 - c0) + 1, rows = rows_end - row0;
      for (int e = tid; e < rows * (D / 4); e += kWarps * 32) {
        const int rr = e / (D / 4), d = e % (D / 4) * 4;
        Sum sum{-INFINITY, 0.0f};
#pragma unroll 8
        for (int k = 0; k < parts; ++k) sum.m = fmaxf(sum.m, __ldcg(&p.part_ml[part0 + kRows * k + rr].m));
        float4 oo = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (sum.m > -INFINITY) {
#pragma unroll 8
          for (int k = 0; k < parts; ++k) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.part_ml) + part0 + kRows * k + rr);
            const float4 v = __ldcg(reinterpret_cast<const float4*>(p.part_o + (part0 + kRows * k + rr) * D + d));
            const float g = exp2a(0.5f * (ml.x - sum.m)), f = g * g;
            sum.l = fmaf(ml.y * g, g, sum.l);
            oo.x = fmaf(v.x, f, oo.x), oo.y = fmaf(v.y, f, oo.y);
            oo.z = fmaf(v.z, f, oo.z), oo.w = fmaf(v.w, f, oo.w);
          }
        }
        write_row(p, at.b, at.h, row0 + rr, d, oo, sum);
      }
    }
    if (at.left == 0) break;
    next_head(at);
  }
  if (!ok) set_status(p.status, CB_ERR_TIMEOUT);
}

// Joins the runs' parts of the prompt form's rows, in order: four dims a thread, 256
// threads to a CTA (16000 rows of 128 dims in two parts: 9.7 us; a CTA for each row took 20, most of it launching).
__global__ void __launch_bounds__(256) kv8_join_kernel(const __grid_constant__ AttendParams p) {
  const int lanes = p.c.head_dim / 4, d = threadIdx.x % lanes * 4;
  const int r = blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
  if (r >= p.rows) return;
  const int64_t head = blockIdx.y;
  const int hk = (int)(head % p.c.n_kv_heads), b = (int)(head / p.c.n_kv_heads);
  const int64_t at = (head * p.rows + r) * p.splits;
  Sum sum{-INFINITY, 0.0f};
  for (int s = 0; s < p.splits; ++s) sum.m = fmaxf(sum.m, p.part_ml[at + s].m);
  float4 oo = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (sum.m > -INFINITY)
    for (int s = 0; s < p.splits; ++s) {
      const Sum part = p.part_ml[at + s];
      const float g = exp2a(0.5f * (part.m - sum.m)), f = g * g;
      const float4 v = *reinterpret_cast<const float4*>(p.part_o + (at + s) * p.c.head_dim + d);
      sum.l = fmaf(part.l * g, g, sum.l);
      oo.x = fmaf(v.x, f, oo.x), oo.y = fmaf(v.y, f, oo.y);
      oo.z = fmaf(v.z, f, oo.z), oo.w = fmaf(v.w, f, oo.w);
    }
  write_row(p, b, hk, r, d, oo, sum);
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
    const float lse = p.lse2[head * p.rows + r];
    const int t = r / p.G;
    // past a row's last slot its scores were not all written
    if (key > p.pos[b] + t || t >= (p.counts ? min(p.counts[b], p.T) : p.T)) continue;
    if (lse != lse) {  // every slot that the row sees
      const int n = p.pos[b] + t - key;
      sum.x = NAN;
      if (n >= 1) sum.y = NAN;
      if (n >= 2) sum.z = NAN;
      if (n >= 3) sum.w = NAN;
      continue;
    }
    const float4 x = *reinterpret_cast<const float4*>(p.scores + (head * p.rows + r) * p.ld_scores + key);
    sum.x += weight(x.x - lse), sum.y += weight(x.y - lse);
    sum.z += weight(x.z - lse), sum.w += weight(x.w - lse);
  }
  float* to = p.c.mass + head * p.c.max_len + key;
  const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (key + i <= last) to[i] += v[i];
}

// mass_j += sum_r exp(x[r][j] - lse_r): a warp owns a block of 64 keys and walks
// the head's query rows 8 NT at a time, so every slot has one writer and one order.
template <int D, int FMT, bool HL, int NT>
__global__ void __launch_bounds__(kWarps * 32) kv8_mass_kernel(const __grid_constant__ AttendParams p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
  const int hk = blockIdx.y % p.c.n_kv_heads, b = blockIdx.y / p.c.n_kv_heads;
  const int pos = p.pos[b], cnt = p.counts ? min(max(p.counts[b], 0), p.T) : p.T;
  const int last = cnt > 0 ? min(pos + cnt, p.limit) - 1 : -1;
  const int64_t head = (int64_t)b * p.c.n_kv_heads + hk;
  const int blk = blockIdx.x * kWarps + warp, key0 = blk * kKv8Block;
  if (key0 > last) return;
  const uint8_t* kb = p.c.k + (head * p.c.max_len + key0) * D;
  const float ks = p.c.k_scale[head * (p.c.max_len / kKv8Block) + blk];
  float sum[4][2] = {};                    // keys g and g + 8 of each 16
  const int first_t = max(0, key0 - pos);  // rows of earlier tokens do not see this block
  for (int row0 = first_t * p.G / (8 * NT) * (8 * NT); row0 < cnt * p.G; row0 += 8 * NT) {
    Query<D, HL, NT> q;
    q.load(p, b, hk, row0);
    float lse[NT][2];
    int lim[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = row0 + 8 * nt + 2 * t4 + i;
        lim[nt][i] = row_limit(p, r, pos, cnt);
        lse[nt][i] = 0.0f;
        if (lim[nt][i] >= 0)
          lse[nt][i] = p.lse2[head * p.rows + r];
      }
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
      float c[NT][4];
      scores<D, FMT, HL, NT>(kb + 16 * mt * D, q, c);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (key0 + 16 * mt + 8 * (i >> 1) + key_row(g) <= lim[nt][i & 1])
            sum[mt][i >> 1] += weight(__fmul_rn(c[nt][i], q.back[nt][i & 1] * ks) - lse[nt][i & 1]);
    }
  }
#pragma unroll
  for (int mt = 0; mt < 4; ++mt)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float v = sum[mt][half];
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      v += __shfl_xor_sync(0xffffffffu, v, 2);
      const int key = key0 + 16 * mt + 8 * half + key_row(g);
      if (t4 == 0 && key <= last) p.c.mass[head * p.c.max_len + key] += v;
    }
}

// The decode form's kernels of a call, and their shared memory.
struct Form {
  void (*attend)(AttendParams);
  void (*mass)(AttendParams);
  int rows, smem;  // query rows of a CTA
};

template <int D, int FMT, bool HL, int NT>
Form form_of() {
  return {kv8_attend_kernel<D, FMT, HL, NT>, kv8_mass_kernel<D, FMT, HL, NT>, 8 * NT,
          kWarps * kRing<D> * kKv8Block * D + 2 * 8 * NT * D * (int)sizeof(float)};
}

// As many query rows to a CTA as there are, up to what its registers hold: 32 rows
// of 64 dims, 16 of 128 (half with heads and tails).
template <int D, int FMT, bool HL>
Form form_of(int rows) {
  constexpr int kMost = (D == 128 ? 2 : 4) / (HL && D >= 64 ? 2 : 1);
  if constexpr (kMost >= 4)
    if (rows > 16) return form_of<D, FMT, HL, 4>();
  if constexpr (kMost >= 2)
    if (rows > 8) return form_of<D, FMT, HL, 2>();
  return form_of<D, FMT, HL, 1>();
}

template <int D>
Form form_of(int format, bool hl, int rows) {
  if (format == CB_KV8_E4M3) return hl ? form_of<D, CB_KV8_E4M3, true>(rows) : form_of<D, CB_KV8_E4M3, false>(rows);
  return hl ? form_of<D, CB_KV8_INT8, true>(rows) : form_of<D, CB_KV8_INT8, false>(rows);
}

Form form_of(const CbKv8& c, int dtype, int rows) {
  const bool hl = dtype == CB_F32;
  switch (c.head_dim) {
    case 16: return form_of<16>(c.format, hl, rows);
    case 32: return form_of<32>(c.format, hl, rows);
    case 64: return form_of<64>(c.format, hl, rows);
    default: return form_of<128>(c.format, hl, rows);
  }
}

// How a call is cut up, and where its parts lie in the scratch.  The counters come
// first, in every call's layout: they are zero between calls.  A call with more 8-row
// blocks over all heads than there are counters takes its rows in several launches.
constexpr size_t kCounters = CB_KV8_ZEROED / sizeof(int);
struct Plan {
  int rows = 0, row_tiles = 0, splits = 0;
  int blocks = 0;  // of query rows, in a launch of the decode form
  int64_t part_rows = 0, ld_scores = 0;
  size_t ml = 0, o = 0, q16 = 0, back = 0, lse2 = 0, scores = 0, bytes = 0;
};

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

Plan plan_of(const CbKv8& c, int dtype, int n_q_heads, int T, int longest, bool add_mass) {
  Plan pl;
  const int bh = c.batch * c.n_kv_heads;
  pl.rows = T * (n_q_heads / c.n_kv_heads);
  pl.ml = kCounters * sizeof(int);
  int64_t parts;
  // From 33 rows on the tensor cores' 128-row tiles pay for the rows they leave empty
  // (float32, 128 dims: 16 sequences x 36 rows at 2K 29 us, 40 on the warp-level form; one
  // of 80 rows at 32K 45 and 49, but of 36 rows 47 and 38).
  if (pl.rows > 32 && c.head_dim >= 64) {
    pl.row_tiles = ceil_div(pl.rows, 128);
    // runs of key tiles that leave the fewest tile times (and three more a CTA to
    // start and end) on the busiest SM
    const int items = bh * ceil_div(pl.row_tiles, 2), tiles = ceil_div(longest, dtype == CB_F32 ? 64 : 8192 / c.head_dim);
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
    // CTAs that are resident at once, at least one block of 64 keys for each warp,
    // and no more than 48 parts a head
    const Form f = form_of(c, dtype, pl.rows);
    int resident = 1;  // without a device: only the layout is asked for
    if (ensure_smem_attr((const void*)f.attend, f.smem) == CB_OK)
      resident = std::max(1, resident_ctas((const void*)f.attend, kWarps * 32, f.smem));
    pl.blocks = std::min({ceil_div(pl.rows, f.rows), (int)kCounters / bh, 65535});
    const int64_t fit = std::max(1, num_sms() * resident / pl.blocks);
    const int64_t work = std::max<int64_t>(1, (int64_t)bh * ceil_div(longest, kKv8Block) / kWarps);
    pl.splits = (int)std::min(std::min(fit, work), (int64_t)bh * 48);
    pl.part_rows = ((int64_t)bh + pl.splits) * f.rows;
    parts = pl.part_rows * pl.blocks;
    // rows' scores cost 8 bytes a key to write and read, taking them again head_dim
    if (add_mass && pl.rows * 8 <= c.head_dim) pl.ld_scores = ceil_div(longest, kKv8Block) * kKv8Block;
  }
  pl.o = pl.ml + align256((size_t)parts * sizeof(Sum));
  pl.q16 = pl.o + align256((size_t)parts * c.head_dim * sizeof(float));
  pl.back = pl.q16 + (size_t)bh * pl.row_tiles * 128 * c.head_dim * (dtype == CB_F32 ? 4 : 2);
  pl.lse2 = pl.back + (size_t)bh * pl.row_tiles * 128 * sizeof(float);
  pl.scores = pl.lse2 + (add_mass ? align256((size_t)bh * pl.rows * sizeof(float)) : 0);
  pl.bytes = pl.scores + (size_t)bh * pl.rows * pl.ld_scores * sizeof(float);
  return pl;
}

int check_call(const CbKv8* c, int dtype, int n_q_heads, int T, int longest) {
  if (const int rc = kv8_check(c)) return rc;
  if (T <= 0 || longest <= 0 || !kv8_dtype_ok(dtype)) return CB_ERR_ARG;
  if (n_q_heads <= 0 || n_q_heads % c->n_kv_heads) return CB_ERR_SHAPE;
  const int64_t rows = (int64_t)T * (n_q_heads / c->n_kv_heads);
  if (rows > 65535 * 16) return CB_ERR_SHAPE;
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
  const int wide = dtype == CB_F32 ? 4 : 8;
  p.q_wide = ((uintptr_t)q & 15) == 0;
  for (int i = 0; i < 3; ++i) {
    p.qs[i] = q_strides[i];
    p.q_wide = p.q_wide && q_strides[i] % wide == 0;
  }
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
  p.part_ml = reinterpret_cast<Sum*>(base + pl.ml);
  p.part_rows = pl.part_rows;
  p.ld_scores = pl.ld_scores;
  p.scores = pl.ld_scores ? reinterpret_cast<float*>(base + pl.scores) : nullptr;
  p.part_o = reinterpret_cast<float*>(base + pl.o);
  p.row_tiles = pl.row_tiles;
  p.q16 = base + pl.q16;
  p.q_back = reinterpret_cast<float*>(base + pl.back);
  p.lse2 = reinterpret_cast<float*>(base + pl.lse2);
  p.status = status;
  const int bh = c->batch * c->n_kv_heads;
  cudaStream_t st = (cudaStream_t)stream;
  if (p.row_tiles > 0) {
    if (const int rc = kv8_prompt_launch(p, bh, st)) return rc;
    if (p.splits > 1) {
      kv8_join_kernel<<<dim3(ceil_div(p.rows, 1024 / c->head_dim), bh), 256, 0, st>>>(p);
      count_launch();
    }
    if (p.add_mass) return kv8_prompt_mass_launch(p, bh, longest, st);
  } else {
    const Form f = form_of(*c, dtype, p.rows);
    if (const int rc = ensure_smem_attr((const void*)f.attend, f.smem)) return rc;
    for (const int all = ceil_div(p.rows, f.rows); p.block0 < all; p.block0 += pl.blocks) {
      f.attend<<<dim3(p.splits, std::min(pl.blocks, all - p.block0)), kWarps * 32, f.smem, st>>>(p);
      count_launch();
    }
    if (p.scores) {
      kv8_scores_mass_kernel<<<dim3(ceil_div(longest, 1024), bh), 256, 0, st>>>(p);
      count_launch();
    } else if (p.add_mass) {
      f.mass<<<dim3(ceil_div(longest, kWarps * kKv8Block), bh), kWarps * 32, 0, st>>>(p);
      count_launch();
    }
  }
  return cudaGetLastError() == cudaSuccess ? CB_OK : CB_ERR_CUDA;
}
