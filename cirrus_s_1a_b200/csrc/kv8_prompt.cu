// Attention of many query rows over the 8-bit K/V cache on the 5th-generation
// tensor cores: the prompt form of cb_kv8_attend for head_dim 64 and 128.
//
// kv8_query_kernel prepares the query rows once: each scaled by a power of two
// (largest element in [256, 512)), rounded to f16 and written as swizzled 128-row
// operand tiles, with the factor that undoes the scaling; float32 rows as two such
// tiles, the f16 head and what it leaves.
//
// kv8_prompt_kernel: a CTA owns 256 query rows of one KV head (two tiles of 128)
// and a run of key tiles (128 keys for 64 dims, 64 for 128 and for float32).
//   * 4 warps turn codes into f16 operands in shared memory (two stages each of K
//     and V), exact; no scale is applied there.
//   * one thread (two for 128 dims) issues tcgen05.mma kind::f16: S = Q K^T into tensor memory, and
//     O += P V with P read from tensor memory (V's dims are its contiguous
//     direction, an MN-major operand).
//   * two warpgroups, a thread per row, do the softmax.  With x = S * a_b
//     (a_b = row factor * block b's key scale, in log2 units) and e_b the exponent
//     of its value scale, a thread keeps m' = max (x + e_b) and writes
//       P = exp2(x + e_b - m')
//     so that P times the bare codes is the sum over values, and neither a block
//     of tiny values nor one of huge ones costs the others precision: P's f16
//     rounding is relative to what the row adds up.  The row's sum (before P is rounded)
//     is l 2^m', l = sum_b 2^-e_b sum P, added up against an exponent e_ref near the blocks'
//     own; blocks far below it (zeros) are summed for themselves (kNear).  out = O / l.
//   * a thread reads its row of S into registers at once, so that the next tile's
//     scores can follow, and takes P against the maximum so far.  Only where the
//     tile's passes it by more than 2^15 (f16 P ends at 2^16) is it raised, and O
//     rescaled in tensor memory.
// The next tile's scores are taken while the exponentials of this one run, and its
// product with V while the next ones do; the two warpgroups take turns at the
// exponentials and at what lies between them.  The exponentials bound it for head_dim 64: 128 x 128 per tile at 16 a
// clock take 1024 clocks, its products 512.
// With several runs per row tile, kv8_join_kernel joins them (kv8_attend.cu).
// Measured: 4096 tokens behind 28600, 12 query heads on 4 KV heads of 64 dims, E4M3:
// 593 us = 650 TFLOP/s, the exponential unit 66 % busy, the tensor pipe 33 %.  Tried
// and slower: a share of the exponentials as a polynomial on the FMA units (636 to
// 757 us, at 639 then), three row tiles of 64 keys (703; with strict turns at the
// exponentials 696, turns passed on at half 624), Q K^T and P V issued by two warps (641).
// For 128 dims, 2 x 1000 tokens at up to 8K (171 us then): tiles of 128 keys with P in
// the columns of its scores (180), a second P a tile (171).
// float32, heads and tails of Q and of P as products of their own: 5 x 191 tokens at up
// to 15.5K, 8 query heads of 128 dims 134 us, 4096 tokens behind 28600 as above 865 us
// (twice the products; the warp-level form took 383 and 3287 us).
// Every wait is bounded (%globaltimer); one that gives up sets CB_ERR_TIMEOUT in the
// status word, and the rows that waited are not written.
#include <climits>

#include "kv8.cuh"
#include "kv8_attend.cuh"

namespace cb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kRows = 128;                 // of a tile (MMA M)
constexpr int kTiles = 2;                  // row tiles of a CTA
constexpr int kStages = 2;
constexpr int kSoftWarps = 4 * kTiles;
constexpr int kConvThreads = 128;
constexpr int kThreads = kSoftWarps * 32 + kConvThreads + 128;
// Registers a thread of the four warpgroups, out of the 128 at launch, where a thread
// holds 128 scores: two warpgroups of softmax, one that converts, one that issues the products.
constexpr int kSoftRegs = 192, kConvRegs = 88, kMmaRegs = 40;
static_assert(2 * kSoftRegs + kConvRegs + kMmaRegs <= 4 * 128, "the shares fit what the block was launched with");
constexpr float kLazy = 15.0f;             // growth of the maximum, in powers of two, that O follows: f16 P ends at 2^16

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Operand tiles lie in rows of 128 bytes (64 elements), 16-byte piece c of row r at
// piece c ^ (r % 8), the 128-byte swizzle; elements 64 on start a second block of rows.
// Offset of 8-element piece kb of a row, in a tile of ROWS rows.
template <int ROWS>
__device__ __forceinline__ uint32_t swizzled(int row, int kb) {
  return (uint32_t)((kb >> 3) * ROWS * 128 + row * 128 + (((kb & 7) ^ (row & 7)) << 4));
}

// One thread of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(is));
  return is != 0;
}

// Shared-memory matrix descriptor, 128-byte swizzle (2 at bits 61-63), version 1
// (bits 46-47), 8-row groups 1024 bytes apart.  lbo, for an operand whose rows run
// along K (MN-major): between its blocks of 64 elements.
__device__ __forceinline__ uint64_t mat_desc(uint32_t saddr, uint32_t lbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)((lbo >> 4) & 0x3FFF) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// Instruction descriptor, kind::f16: D f32, A and B f16; bit 16: B is MN-major.
__host__ __device__ constexpr uint32_t idesc(int m, int n, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"((uint32_t)add)
      : "memory");
}

__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"((uint32_t)add)
      : "memory");
}

// 32 columns of the warp's 32 lanes of tensor memory, and back.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float* v) {
  uint32_t* u = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
      "%30,%31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
        "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
        "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&u)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&u)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
      "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 16 codes as f16 operand values.
template <int FMT>
__device__ __forceinline__ void to_operand(uint4 c, uint4& lo, uint4& hi) {
  codes_to_h2<FMT>(c.x, lo.x, lo.y);
  codes_to_h2<FMT>(c.y, lo.z, lo.w);
  codes_to_h2<FMT>(c.z, hi.x, hi.y);
  codes_to_h2<FMT>(c.w, hi.z, hi.w);
}

// The last slot row r of a KV head sees (rows of padding tokens: -1).
__device__ __forceinline__ int row_limit(const AttendParams& p, int r, int pos, int cnt) {
  const int t = r / p.G;
  if (r >= p.rows || t >= cnt) return -1;
  return min(pos + t, p.limit - 1);
}

// ------------------------------------------------------------------ queries
// D/8 lanes per row, 8 elements each.
template <int D, int HL>
__global__ void __launch_bounds__(256) kv8_query_kernel(const __grid_constant__ AttendParams p) {
  constexpr int kLanes = D / 8;
  const int64_t head = blockIdx.y;
  const int hk = (int)(head % p.c.n_kv_heads), b = (int)(head / p.c.n_kv_heads);
  const int r = (int)(blockIdx.x * 256 + threadIdx.x) / kLanes, kb = threadIdx.x % kLanes;
  if (r >= p.row_tiles * kRows) return;  // whole rows leave together
  float x[8];
  float top = 0.0f;
  const bool live = r < p.rows;
  const int64_t base =
      (int64_t)b * p.qs[0] + (int64_t)(r / p.G) * p.qs[1] + (hk * p.G + r % p.G) * p.qs[2] + kb * 8;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = live ? kv8_load(p.q, base + i, p.dtype) : 0.0f;
    top = max_nan(top, fabsf(x[i]));
  }
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  // a row with a NaN or an infinity: zeros, and a NaN for its factor
  const bool bad = !(top < INFINITY);
  if (bad)
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.0f;
  int e = 0;
  if (top > 0.0f && !bad) e = max((__float_as_int(top) >> 23) - 127, -100);
  const float f = copysignf(kv8_pow2(8 - e), p.scale);
  uint8_t* tile = p.q16 + (head * p.row_tiles + r / kRows) * (int64_t)((1 + HL) * kRows * D * 2);
#pragma unroll
  for (int part = 0; part <= HL; ++part) {  // head, and what it leaves
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float y0 = part ? x[2 * i] : x[2 * i] * f, y1 = part ? x[2 * i + 1] : x[2 * i + 1] * f;
      const __half2 y = __floats2half2_rn(y0, y1);
      h[i] = h2_bits(y);
      x[2 * i] = y0 - __low2float(y);
      x[2 * i + 1] = y1 - __high2float(y);
    }
    *reinterpret_cast<uint4*>(tile + part * kRows * D * 2 + swizzled<kRows>(r % kRows, kb)) =
        make_uint4(h[0], h[1], h[2], h[3]);
  }
  if (kb == 0) p.q_back[head * p.row_tiles * kRows + r] = bad ? NAN : live ? kv8_pow2(e - 8) * fabsf(p.scale) * kLog2e : 0.0f;
}

// --------------------------------------------------------------- attention
// HL: float32 queries, carried as f16 head and tail, and so is P (22 bits).
template <int D, int HL>
struct Prompt {
  static constexpr int kKeys = HL ? 64 : 8192 / D;  // of a key tile: S, P and O of two tiles fit tensor memory
  static constexpr int kHalves = kKeys / kKv8Block;
  static constexpr int kHead = kRows * D * 2;
  static constexpr int kQ = (1 + HL) * kHead;   // bytes of a query tile
  static constexpr int kKV = kKeys * D * 2;     // of a K or V tile
  static constexpr int kSmem = kTiles * kQ + 2 * kStages * kKV + 1024;
  // tensor memory: S, P (f16, half as many columns) and O of both tiles
  static constexpr int kPCols = (1 + HL) * kKeys / 2;
  static constexpr int kP = kTiles * kKeys, kO = 512 - kTiles * D;
  static_assert(kP + kTiles * kPCols <= kO, "S, P and O fit 512 columns");
  // What the row's largest P lies above 1, in powers of two: with a tail of P, its last
  // bit (2^-24, the smallest f16) then is 2^-35 of the largest, and O follows growth by 2^4.
  static constexpr float kLift = HL ? 11.0f : 0.0f;
  // Warps that issue the products.  One keeps two tiles of 128 keys busy, in a fixed
  // order that keeps the softmax warpgroups out of step (64 dims, 4096 tokens at 32K:
  // 584 us, a warp to each tile 637).  With 64 keys its own waits and issue bounded a
  // tile (128 dims, 2 x 1000 tokens at 8K with weights: 171 us
  // with one warp, 161 with two; 2048 tokens at 32K: 341, 327).
  static constexpr int kIssuers = kKeys == 64 ? 2 : 1;
  // With 64 scores a thread, the softmax leaves registers to the others.
  static constexpr int kSoftRegs = kKeys == 64 ? 160 : cb::kSoftRegs, kConvRegs = kKeys == 64 ? 104 : cb::kConvRegs,
                       kMmaRegs = kKeys == 64 ? 88 : cb::kMmaRegs;
  static_assert(2 * kSoftRegs + kConvRegs + kMmaRegs <= 4 * 128, "the shares fit what the block was launched with");
  static constexpr int kPieces = kKeys * D / 16 / kConvThreads;  // 16-byte pieces of a tile per converting thread
  static constexpr int kRow = D / 16;                            // of a key
};

// NaN over a row's results in the dims where a slot that it sees, from `first` on, holds a
// NaN (thread for row, after the CTA's results).  Rarely called: it finds its place anew, so
// that nothing is kept for it through the loops.
template <int D, int HL>
__device__ void nan_values(const AttendParams& p, int first, int end) {
  uint32_t bx, by, tid;
  asm volatile("mov.u32 %0, %%ctaid.x;\n\tmov.u32 %1, %%ctaid.y;\n\tmov.u32 %2, %%tid.x;" : "=r"(bx), "=r"(by), "=r"(tid));
  const int64_t head = by;
  const int hk = (int)(by % p.c.n_kv_heads), b = (int)(by / p.c.n_kv_heads);
  const int split = bx % p.splits, r = bx / p.splits * kTiles * kRows + tid;
  if (tid >= kTiles * kRows || r >= p.rows) return;
  const int cnt = p.counts ? min(max(p.counts[b], 0), p.T) : p.T;
  const int lim = min(row_limit(p, r, p.pos[b], cnt), end - 1);
  const int64_t at = p.splits > 1 ? (head * p.rows + r) * p.splits + split
                                  : ((int64_t)b * p.T + r / p.G) * (p.G * p.c.n_kv_heads) + hk * p.G + r % p.G;
#pragma unroll 1
  for (int slot = first; slot <= lim; ++slot)
#pragma unroll 1
    for (int d = 0; d < D; ++d) {
      if ((p.c.v[(head * p.c.max_len + slot) * D + d] & 0x7F) != 0x7F) continue;
      if (p.splits > 1) p.part_o[at * D + d] = NAN;
      else if (HL > 0) static_cast<float*>(p.out)[at * D + d] = NAN;
      else static_cast<uint16_t*>(p.out)[at * D + d] = 0x7FFF;  // a NaN of either type
    }
}

template <int D, int FMT, int HL>
__global__ void __launch_bounds__(kThreads, 1) kv8_prompt_kernel(const __grid_constant__ AttendParams p) {
  using C = Prompt<D, HL>;
  constexpr int kKeys = C::kKeys, kHalves = C::kHalves;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023);  // the swizzle counts from 1024-byte boundaries
  __shared__ __align__(8) unsigned long long bars[20];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ Sum s_aside[kTiles * kRows];
  __shared__ int s_nan;  // the first slot with an E4M3 NaN among values that not all rows see
  __shared__ int s_end;  // the end of the run's slots
  uint8_t* sq = smem;
  uint8_t* sk = smem + kTiles * C::kQ;
  uint8_t* sv = sk + kStages * C::kKV;
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t q_full = bar0, k_full = bar0 + 8, k_free = bar0 + 24, v_full = bar0 + 40, v_free = bar0 + 56,
                 s_full = bar0 + 72, s_free = bar0 + 88, p_full = bar0 + 104, o_full = bar0 + 120, end = bar0 + 136;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t head = blockIdx.y;
  const int b = (int)(head / p.c.n_kv_heads);
  const int pair = blockIdx.x / p.splits, split = blockIdx.x % p.splits;
  const int row0 = pair * kTiles * kRows;
  const int tiles = min(kTiles, p.row_tiles - pair * kTiles);
  const int pos = p.pos[b], cnt = p.counts ? min(max(p.counts[b], 0), p.T) : p.T;
  // the last slot any of the CTA's rows sees, and this run of key tiles
  int last = -1;
  {
    const int rl = min(min(row0 + tiles * kRows, p.rows), cnt * p.G) - 1;
    if (rl >= row0) last = max(last, row_limit(p, rl, pos, cnt));
  }
  const int all = (last + kKeys) / kKeys, per = (all + p.splits - 1) / p.splits;
  const int beg = min(all, split * per), n = min(all, beg + per) - beg;

  if (tid == 0) {
    const uint32_t one[] = {q_full, s_full, s_full + 8, o_full, o_full + 8, end, end + 8};
    for (uint32_t bar : one) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar));
    for (int i = 0; i < 2; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(k_full + 8 * i), "n"(kConvThreads));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(v_full + 8 * i), "n"(kConvThreads));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(k_free + 8 * i), "r"(min(tiles, C::kIssuers)));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(v_free + 8 * i), "r"(min(tiles, C::kIssuers)));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(s_free + 8 * i), "n"(kRows));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(p_full + 8 * i), "n"(kRows));
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_abort = 0;
    s_nan = INT_MAX;
    s_end = (beg + n) * kKeys;
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s_tmem)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = 0;  // all 512 columns are this CTA's: they start at 0
  bool ok = true;
  auto wait = [&](uint32_t bar, int phase) {
    if (ok && !mbar_wait(bar, phase & 1)) {
      ok = false;
      s_abort = 1;
    }
    return ok;
  };

  if (warp < kSoftWarps) {
    // ---------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kSoftRegs));
    const int tile = warp / 4, r = row0 + tile * kRows + (warp % 4) * 32 + lane;
    if (tile < tiles) {
      const uint32_t lanes = (uint32_t)(warp % 4) << 21;  // this warp's lanes of tensor memory (bits 16-31)
      const uint32_t ts = tmem + lanes + tile * kKeys, tp = tmem + lanes + C::kP + tile * C::kPCols,
                     to = tmem + lanes + C::kO + tile * D;
      const int lim = row_limit(p, r, pos, cnt);
      const float back = p.q_back[head * p.row_tiles * kRows + r];
      const float* ksc = p.c.k_scale + head * (p.c.max_len / kKv8Block);
      const float* vsc = p.c.v_scale + head * (p.c.max_len / kKv8Block);
      const int vis = last / kKv8Block;  // the last block any row sees
      float m = -INFINITY, l = 0.0f;
      Sum& aside = s_aside[tid];
      aside.clear();
      // the run's largest value exponent, and whether any lies far below it
      int e_ref = 0;
      bool wide = false;
      {
        uint32_t most = 0u, least = ~0u;  // bits of positive floats
        for (int blk = kHalves * beg + lane; blk <= min(vis, kHalves * (beg + n) - 1); blk += 32) {
          const uint32_t u = __float_as_uint(__ldg(vsc + blk));
          most = max(most, u), least = min(least, u);
        }
        most = __reduce_max_sync(0xffffffffu, most);
        least = __reduce_min_sync(0xffffffffu, least);
        if (n > 0) {
          e_ref = kv8_exponent(__uint_as_float(most));
          wide = kv8_exponent(__uint_as_float(least)) < e_ref - kNear;
        }
      }
      float ks[kHalves], vs[kHalves];
      auto scales = [&](int j) {
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          const int blk = min(kHalves * (beg + j) + h, vis);
          ks[h] = __ldg(ksc + blk);
          vs[h] = __ldg(vsc + blk);
        }
      };
      if (n > 0) scales(0);
      for (int j = 0; j < n; ++j) {
        const int key0 = (beg + j) * kKeys;
        float a[kHalves];
        int ev[kHalves];
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          a[h] = max_nan(back * ks[h], 1.2e-38f);  // above 0: a masked score times it stays -infinity
          ev[h] = kv8_exponent(vs[h]);
        }
        if (j + 1 < n) scales(j + 1);
        wait(s_full + 8 * tile, j);  // (where it gives up no lane leaves the loop: what follows takes whole warps)
        fence_after();
        if (wide && min(ev[0], ev[kHalves - 1]) < e_ref - kNear) {
#pragma unroll 1
          for (int q = 0; q < kKeys / 16; ++q) {
            const bool first = q < kKv8Block / 16;
            if ((first ? ev[0] : ev[kHalves - 1]) >= e_ref - kNear) continue;
            const float by = first ? a[0] : a[kHalves - 1];
            uint32_t u[16];
            tmem_ld16(ts + q * 16, u);
            tmem_ld_wait();
            float x = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if (key0 + q * 16 + i > lim) u[i] = __float_as_uint(-INFINITY);
              x = fmaxf(x, __uint_as_float(u[i]));
            }
            if (x > -INFINITY) {
              const int e = first ? ev[0] : ev[kHalves - 1];
              x = fmaf(x, by, (float)e);
              float sum = 0.0f;
#pragma unroll
              for (int i = 0; i < 16; ++i) sum += exp2a(fmaf(__uint_as_float(u[i]), by, (float)e) - x);
              aside.add(x, sum * kv8_pow2(-e));
            }
            __syncwarp();
          }
        }
        const bool whole = __all_sync(0xffffffffu, lim >= key0 + kKeys - 1);
        float s[kKeys];
#pragma unroll
        for (int q = 0; q < kKeys / 32; ++q) tmem_ld32(ts + q * 32, s + q * 32);
        tmem_ld_wait();
        fence_before();
        mbar_arrive(s_free + 8 * tile);  // the next tile's scores may replace them
        if (!whole) {
#pragma unroll
          for (int i = 0; i < kKeys; ++i)
            if (key0 + i > lim) s[i] = -INFINITY;
        }
        float now = -INFINITY;
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          const float* v = s + h * 64;
          float t[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) t[k] = v[k];
#pragma unroll
          for (int i = 4; i < 60; i += 8)
#pragma unroll
            for (int k = 0; k < 4; ++k) t[k] = fmaxf(fmaxf(t[k], v[i + k]), v[i + 4 + k]);
#pragma unroll
          for (int k = 0; k < 4; ++k) t[k] = fmaxf(t[k], v[60 + k]);
          const float top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
          if (top > -INFINITY) now = fmaxf(now, fmaf(top, a[h], (float)ev[h]));
        }
        const bool grow = now > m + kLazy || (m == -INFINITY && now > m);
        if (j > 0) {  // the product with the last tile's P has read it, and O is at rest
          wait(o_full + 8 * tile, j - 1);
          fence_after();
        }
        float at_m = m == -INFINITY ? 0.0f : m;
        if (__any_sync(0xffffffffu, grow || fabsf(at_m) > kFarScore)) {
          const float ref = now - C::kLift, alpha = !grow ? 1.0f : m > -INFINITY ? exp2a(m - ref) : 0.0f;
          if (grow) m = ref;
          l *= alpha;
          if (j > 0) {
#pragma unroll
            for (int c = 0; c < D; c += 16) {
              uint32_t u[16];
              tmem_ld16(to + c, u);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) u[i] = __float_as_uint(__uint_as_float(u[i]) * alpha);
              tmem_st16(to + c, u);
            }
          }
          at_m = m == -INFINITY ? 0.0f : m;
          if (fabsf(at_m) > kFarScore) {
#pragma unroll
            for (int i = 0; i < kKeys; ++i)
              s[i] = min_nan(fmaf(s[i], a[i / 64], (float)ev[i / 64]) - at_m, kFarMost) - (float)ev[i / 64];
#pragma unroll
            for (int h = 0; h < kHalves; ++h) a[h] = 1.0f;
            at_m = 0.0f;
          }
        }
        float sum_l = 0.0f;
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          const float add = (float)ev[h] - at_m;
          const f32x2 a2 = pack2(a[h], a[h]), c2 = pack2(add, add);
          f32x2 sum[2] = {0, 0};  // pairs of zeros
#pragma unroll
          for (int q = 2 * h; q < 2 * h + 2; ++q) {
            uint32_t ph[16], pt[HL ? 16 : 1];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 d = unpack2(fma2(pack2(s[q * 32 + 2 * i], s[q * 32 + 2 * i + 1]), a2, c2));
              const float y0 = exp2a(d.x), y1 = exp2a(d.y);
              sum[i & 1] = add2(sum[i & 1], pack2(y0, y1));
              const __half2 y = __floats2half2_rn(y0, y1);
              ph[i] = h2_bits(y);
              if constexpr (HL > 0) pt[i] = h2_bits(__floats2half2_rn(y0 - __low2float(y), y1 - __high2float(y)));
            }
            tmem_st16(tp + q * 16, ph);
            if constexpr (HL > 0) tmem_st16(tp + kKeys / 2 + q * 16, pt);
          }
          const float2 both = unpack2(add2(sum[0], sum[1]));
          const int d = e_ref - ev[h];  // 2^-127 is written as 0
          sum_l = fmaf(both.x + both.y, kv8_pow2(d > kNear ? -127 : d), sum_l);
        }
        l += sum_l;
        tmem_st_wait();
        fence_before();
        mbar_arrive(p_full + 8 * tile);
      }
      // results: O, and the sum.  (Products n - 2 and before are known done.)
      if (n > 0) wait(o_full + 8 * tile, n - 1);
      fence_after();
      l *= kv8_pow2(-e_ref);
      if (wide) {  // (its m passes the row's by no more than a maximum lags)
        const float g = Sum::half(aside.m, m);
        l += aside.l * g * g;
      }
      const int t = r / p.G, hq = (int)(head % p.c.n_kv_heads) * p.G + r % p.G;
      const int64_t orow = ((int64_t)b * p.T + t) * (p.G * p.c.n_kv_heads) + hq;
      const int64_t at = (head * p.rows + r) * p.splits + split;
      // NaN scores raise no maximum, but the row has seen something all the same
      const bool none = lim < 0 || l == 0.0f;
      const Inverse inv(none ? 1.0f : l);
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        float o[32];
        if (n > 0) {
          tmem_ld32(to + c, o);
          tmem_ld_wait();
        }
        if (r >= p.rows || !ok) continue;
        if (none)
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0.0f;
        if (p.splits > 1) {
          float4* dst = reinterpret_cast<float4*>(p.part_o + at * D + c);
#pragma unroll
          for (int i = 0; i < 8; ++i) dst[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        } else if constexpr (HL > 0) {
          float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.out) + orow * D + c);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            dst[i] = make_float4(inv.of(o[4 * i]), inv.of(o[4 * i + 1]), inv.of(o[4 * i + 2]), inv.of(o[4 * i + 3]));
        } else {
          uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + orow * D + c);
          uint32_t u[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float y0 = inv.of(o[2 * i]), y1 = inv.of(o[2 * i + 1]);
            u[i] = p.dtype == CB_BF16 ? (uint32_t)f32_to_bf16(y0) | (uint32_t)f32_to_bf16(y1) << 16
                                      : h2_bits(__floats2half2_rn(y0, y1));
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) dst[i] = make_uint4(u[4 * i], u[4 * i + 1], u[4 * i + 2], u[4 * i + 3]);
        }
      }
      if (r < p.rows && ok) {
        if (p.splits > 1) {
          p.part_ml[at] = none ? Sum{-INFINITY, 0.0f} : Sum{fmaxf(m, -3e38f), l};
        } else {
          const float lse2 = none ? -INFINITY : m + log2f(l);
          p.lse[orow] = lse2 * kLn2;
          if (p.add_mass) p.lse2[head * p.rows + r] = lse2;
        }
      }
    }
  } else if (warp < kSoftWarps + kConvThreads / 32) {
    // ------------------------------------------------- codes to operands
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kConvRegs));
    const int d = tid - kSoftWarps * 32;
    const uint8_t* src[2] = {p.c.k + head * p.c.max_len * D, p.c.v + head * p.c.max_len * D};
    uint4 raw[2][C::kPieces];
    // piece i: 16 bytes of one key, 8 consecutive keys to 8 consecutive threads
    auto key_of = [&](int i) { return (d & 7) + 8 * ((i * kConvThreads + d) / (8 * C::kRow)); };
    auto chunk_of = [&](int i) { return (i * kConvThreads + d) / 8 % C::kRow; };
    auto load = [&](int kv, int j) {
#pragma unroll
      for (int i = 0; i < C::kPieces; ++i) {
        const int key = (beg + j) * kKeys + key_of(i);
        // slots no row sees may hold anything, an E4M3 NaN too: they read as 0
        raw[kv][i] = j < n && key <= last
                         ? __ldg(reinterpret_cast<const uint4*>(src[kv] + (int64_t)key * D) + chunk_of(i))
                         : make_uint4(0u, 0u, 0u, 0u);
      }
    };
    load(0, 0);
    load(1, 0);
    // tiles that end by here are seen whole by every row
    const int seen = row0 + tiles * kRows > cnt * p.G ? -1 : min(pos + row0 / p.G, p.limit - 1);
    for (int j = 0; j < n; ++j) {
      const int st = j & 1;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        if (j >= kStages && !wait((kv ? v_free : k_free) + 8 * st, (j - kStages) / kStages)) break;
        uint8_t* dst = (kv ? sv : sk) + st * C::kKV;
#pragma unroll
        for (int i = 0; i < C::kPieces; ++i) {
          const int key = key_of(i), c = chunk_of(i);
          uint4 lo, hi;
          if (FMT == CB_KV8_E4M3 && kv == 1 && (beg + j + 1) * kKeys - 1 > seen) {
            // 0 * NaN is not 0: a NaN reads as 0 here, and reaches the rows that see it at the end
            uint32_t* w = &raw[kv][i].x;
            uint32_t any = 0;
#pragma unroll
            for (int z = 0; z < 4; ++z) {
              const uint32_t nan = __vcmpeq4(w[z] & 0x7F7F7F7Fu, 0x7F7F7F7Fu);
              w[z] &= ~nan;
              any |= nan;
            }
            if (any) atomicMin(&s_nan, (beg + j) * kKeys + key);
          }
          to_operand<FMT>(raw[kv][i], lo, hi);
          *reinterpret_cast<uint4*>(dst + swizzled<kKeys>(key, 2 * c)) = lo;
          *reinterpret_cast<uint4*>(dst + swizzled<kKeys>(key, 2 * c + 1)) = hi;
        }
        load(kv, j + 1);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive((kv ? v_full : k_full) + 8 * st);
      }
      if (!ok) break;
    }
  } else {
    // ---------------------------------------------------------- products
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kMmaRegs));
    const int issuer = warp - kSoftWarps - kConvThreads / 32;
    if (issuer < C::kIssuers && issuer < tiles && n > 0) {
      const int first = C::kIssuers > 1 ? issuer : 0;  // its row tiles: first, first + kIssuers ...
      // The whole warp walks the loop, so that addresses and descriptors stay in
      // uniform registers; one elected thread issues.  (A branch of one thread moved
      // them there for every instruction: 90 to 140 clocks each instead of 32 or 64.)
      const bool lead = elect_one();
      const uint32_t q_at = smem_u32(sq), k_at = smem_u32(sk), v_at = smem_u32(sv);
      if (lead && first == 0) {
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(q_full), "r"(tiles * C::kQ) : "memory");
        asm volatile(
            "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(q_at),
            "l"(p.q16 + (head * p.row_tiles + pair * kTiles) * (int64_t)C::kQ), "r"(tiles * C::kQ), "r"(q_full)
            : "memory");
      }
      constexpr uint32_t kIdS = idesc(kRows, kKeys, false), kIdO = idesc(kRows, D, true);
      auto qk = [&](int t, int st) {
        const uint64_t qd = mat_desc(q_at + t * C::kQ, 16), kd = mat_desc(k_at + st * C::kKV, 16);
        if (lead) {
#pragma unroll
          for (int s = 0; s < (1 + HL) * (D / 16); ++s) {
            const int k = s % (D / 16);
            mma_ss(t * kKeys, qd + (s / (D / 16) * C::kHead + k / 4 * (kRows * 128) + k % 4 * 32) / 16,
                   kd + (k / 4 * (kKeys * 128) + k % 4 * 32) / 16, kIdS, s > 0);
          }
          commit(s_full + 8 * t);
          if (t + C::kIssuers >= tiles) commit(k_free + 8 * st);
        }
      };
      auto all_wait = [&](uint32_t bar, int phase) { return __all_sync(0xffffffffu, wait(bar, phase)); };
      bool go = all_wait(q_full, 0) && all_wait(k_full, 0);
      if (go)
        for (int t = first; t < tiles; t += C::kIssuers) qk(t, 0);
      for (int j = 0; j < n && go; ++j) {
        const int st = j & 1, next = (j + 1) & 1;
        for (int t = first; t < tiles && go; t += C::kIssuers) {
          if (j + 1 < n) {
            go = (t > first || all_wait(k_full + 8 * next, (j + 1) / 2)) && all_wait(s_free + 8 * t, j);
            if (!go) break;
            fence_after();
            qk(t, next);
          }
          go = all_wait(p_full + 8 * t, j) && (t > first || all_wait(v_full + 8 * st, j / 2));
          if (!go) break;
          fence_after();
          const uint64_t vd = mat_desc(v_at + st * C::kKV, kKeys * 128);
          if (lead) {
#pragma unroll
            for (int s = 0; s < C::kPCols / 8; ++s)
              mma_ts(C::kO + t * D, C::kP + t * C::kPCols + s * 8, vd + s % (kKeys / 16) * 2048 / 16, kIdO, j > 0 || s > 0);
            commit(o_full + 8 * t);
            if (t + C::kIssuers >= tiles) commit(v_free + 8 * st);
          }
        }
      }
      // the copy and the products in flight end before their memory goes
      if (!go) mbar_wait(q_full, 0);
      if (lead) commit(end + 8 * first);
      mbar_wait(end + 8 * first, 0);
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (FMT == CB_KV8_E4M3 && s_nan != INT_MAX && !s_abort) nan_values<D, HL>(p, s_nan, s_end);
  if (tid == 0 && s_abort) set_status(p.status, CB_ERR_TIMEOUT);
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(s_tmem));
}

// ----------------------------------------------------------------- weights
// mass_j += sum_r exp(x[r][j] - lse_r) for the query rows of a KV head: the scores
// are taken again, transposed (keys in the 128 lanes, 128 query rows in the
// columns), so that a thread owns a key and adds its probabilities up in one fixed
// order, without atomics.  A CTA owns 128 keys, turned into an operand once; query
// tiles and their rows' factors stream through four stages, the scores through four
// buffers of tensor memory, two warpgroups take them in turn.  Bound by the
// exponentials and by whole CTAs to an SM: 2 x 1000 tokens at up to 8K, 8 query heads
// of 128 dims: 70 us (206 key tiles on 148 SMs), the exponential unit 59 % busy.
// (float32 queries of 128 dims, with their tails: two stages and two buffers.)
template <int D, int HL>
struct Mass {
  static constexpr int kStages = HL && D == 128 ? 2 : 4;
  static constexpr int kHead = kRows * D * 2;
  static constexpr int kQ = (1 + HL) * kHead;
  static constexpr int kInfo = kRows * 8;  // of each row: the factor of its scores, and -lse (log2 units)
  static constexpr int kSmem = kHead + kStages * (kQ + kInfo) + 1024;
};

template <int D, int FMT, int HL>
__global__ void __launch_bounds__(kThreads, 1) kv8_prompt_mass_kernel(const __grid_constant__ AttendParams p) {
  using C = Mass<D, HL>;
  constexpr int kMassStages = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sk = smem_raw + (-smem_u32(smem_raw) & 1023);
  uint8_t* sq = sk + C::kHead;
  float* s_info = reinterpret_cast<float*>(sq + kMassStages * C::kQ);  // [stage][2][128]
  __shared__ __align__(8) unsigned long long bars[3 * kMassStages + 1];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ float s_sum[kRows];
  __shared__ int s_nan_t;  // the last token with a row whose lse is NaN: every slot it sees is one too
  const uint32_t q_full = smem_u32(bars), q_free = q_full + 8 * kMassStages, s_full = q_free + 8 * kMassStages,
                 end = s_full + 8 * kMassStages;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t head = blockIdx.y;
  const int b = (int)(head / p.c.n_kv_heads);
  const int key0 = blockIdx.x * kRows;
  const int pos = p.pos[b], cnt = p.counts ? min(max(p.counts[b], 0), p.T) : p.T;
  const int last = cnt > 0 ? min(pos + cnt, p.limit) - 1 : -1;
  if (key0 > last) return;
  // row tiles from the first row that sees key0
  const int first = max(0, key0 - pos) * p.G / kRows, n = ceil_div(cnt * p.G, kRows) - first;

  if (tid == 0) {
    for (int i = 0; i < kMassStages; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(q_full + 8 * i), "n"(kConvThreads + 1));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(q_free + 8 * i), "n"(kRows + 1));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(s_full + 8 * i));
    }
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(end));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_abort = 0;
    s_nan_t = INT_MIN / 2;
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s_tmem)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  // the keys, slots no row sees as 0
  const uint8_t* src = p.c.k + head * p.c.max_len * D;
  for (int i = tid; i < kRows * (D / 16); i += kThreads) {
    const int key = (i & 7) + 8 * (i / (8 * (D / 16))), c = i / 8 % (D / 16);
    uint4 raw = make_uint4(0u, 0u, 0u, 0u), lo, hi;
    if (key0 + key <= last) raw = __ldg(reinterpret_cast<const uint4*>(src + (int64_t)(key0 + key) * D) + c);
    to_operand<FMT>(raw, lo, hi);
    *reinterpret_cast<uint4*>(sk + swizzled<kRows>(key, 2 * c)) = lo;
    *reinterpret_cast<uint4*>(sk + swizzled<kRows>(key, 2 * c + 1)) = hi;
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  fence_before();
  __syncthreads();
  fence_after();
  bool ok = true;
  auto wait = [&](uint32_t bar, int phase) {
    if (ok && !mbar_wait(bar, phase & 1)) {
      ok = false;
      s_abort = 1;
    }
    return ok;
  };
  float mine = 0.0f;
  if (warp < kSoftWarps) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
    const int group = warp / 4, key = key0 + (warp % 4) * 32 + lane;
    const float ks = p.c.k_scale[head * (p.c.max_len / kKv8Block) + min(key, last) / kKv8Block];
    const f32x2 ks2 = pack2(ks, ks);
    f32x2 sum[2] = {0, 0};
    for (int k = group; k < n; k += 2) {
      const int st = k % kMassStages;
      wait(s_full + 8 * st, k / kMassStages);  // (no lane leaves the loop alone)
      fence_after();
      float s[kRows];
#pragma unroll
      for (int q = 0; q < 4; ++q) tmem_ld32(((uint32_t)(warp % 4) << 21) + st * kRows + q * 32, s + q * 32);
      tmem_ld_wait();
      fence_before();
      const int row0 = (first + k) * kRows;
      // the tile's first row sees the least: a key past it is not seen by all of them
      if (!__all_sync(0xffffffffu, key <= pos + row0 / p.G)) {
#pragma unroll
        for (int i = 0; i < kRows; ++i)
          if (key > pos + (row0 + i) / p.G) s[i] = -INFINITY;
      }
      const float* f = s_info + st * 2 * kRows;
#pragma unroll
      for (int i = 0; i < kRows; i += 4) {
        const float4 by = *reinterpret_cast<const float4*>(f + i), sub = *reinterpret_cast<const float4*>(f + kRows + i);
        const float2 x = unpack2(add2(mul2(mul2(pack2(s[i], s[i + 1]), ks2), pack2(by.x, by.y)), pack2(sub.x, sub.y)));
        const float2 y = unpack2(add2(mul2(mul2(pack2(s[i + 2], s[i + 3]), ks2), pack2(by.z, by.w)), pack2(sub.z, sub.w)));
        sum[0] = add2(sum[0], pack2(weight(x.x), weight(x.y)));
        sum[1] = add2(sum[1], pack2(weight(y.x), weight(y.y)));
      }
      mbar_arrive(q_free + 8 * st);
    }
    const float2 both = unpack2(add2(sum[0], sum[1]));
    mine = both.x + both.y;
    if (group == 1) s_sum[(warp % 4) * 32 + lane] = mine;
  } else if (warp < kSoftWarps + kConvThreads / 32) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kConvRegs));
    const int d = tid - kSoftWarps * 32;
    for (int k = 0; k < n; ++k) {
      const int st = k % kMassStages, tile = first + k, r = tile * kRows + d, t = r / p.G;
      if (k >= kMassStages && !wait(q_free + 8 * st, k / kMassStages - 1)) break;
      if (d == 0) {
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(q_full + 8 * st), "r"(C::kQ) : "memory");
        asm volatile(
            "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                smem_u32(sq) + st * C::kQ),
            "l"(p.q16 + (head * p.row_tiles + tile) * (int64_t)C::kQ), "r"(C::kQ), "r"(q_full + 8 * st)
            : "memory");
      }
      // rows that see nothing (or NaN): a factor that leaves any score finite, and -infinity
      float by = 1.2e-38f, sub = -INFINITY;
      if (t < cnt && pos + t >= 0) {
        const float lse = p.lse2[head * p.rows + r];
        by = fmaxf(p.q_back[head * p.row_tiles * kRows + r], 1.2e-38f);
        sub = lse == lse ? -lse : -INFINITY;
        if (lse != lse) atomicMax(&s_nan_t, t);
      }
      s_info[st * 2 * kRows + d] = by;
      s_info[st * 2 * kRows + kRows + d] = sub;
      mbar_arrive(q_full + 8 * st);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMmaRegs));
    if (warp == kSoftWarps + kConvThreads / 32) {
      const bool lead = elect_one();
      const uint32_t k_at = smem_u32(sk), q_at = smem_u32(sq);
      bool go = true;
      for (int k = 0; k < n && go; ++k) {
        const int st = k % kMassStages;
        // the stage's query tile is new, so its scores' buffer has been read
        go = __all_sync(0xffffffffu, wait(q_full + 8 * st, k / kMassStages));
        if (!go) break;
        fence_after();
        const uint64_t kd = mat_desc(k_at, 16), qd = mat_desc(q_at + st * C::kQ, 16);
        if (lead) {
#pragma unroll
          for (int s = 0; s < (1 + HL) * (D / 16); ++s) {
            const int k16 = s % (D / 16), at = k16 / 4 * (kRows * 128) + k16 % 4 * 32;
            mma_ss(st * kRows, kd + at / 16, qd + (s / (D / 16) * C::kHead + at) / 16, idesc(kRows, kRows, false), s > 0);
          }
          commit(s_full + 8 * st);
          commit(q_free + 8 * st);
        }
      }
      // the products and copies in flight end before their memory goes
      if (lead) commit(end);
      mbar_wait(end, 0);
      for (int k = max(0, n - kMassStages); k < n && !go; ++k) mbar_wait(q_full + 8 * (k % kMassStages), k / kMassStages & 1);
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (tid < kRows && key0 + tid <= last && !s_abort)
    p.c.mass[head * p.c.max_len + key0 + tid] += key0 + tid <= pos + s_nan_t ? NAN : mine + s_sum[tid];
  if (tid == 0 && s_abort) set_status(p.status, CB_ERR_TIMEOUT);
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(s_tmem));
}

template <int D, int HL>
int launch_prompt(const AttendParams& p, int bh, cudaStream_t st) {
  kv8_query_kernel<D, HL><<<dim3(ceil_div(p.row_tiles * kRows * (D / 8), 256), bh), 256, 0, st>>>(p);
  count_launch();
  const dim3 grid(ceil_div(p.row_tiles, kTiles) * p.splits, bh);
  constexpr int kSmem = Prompt<D, HL>::kSmem;
  auto fn = p.c.format == CB_KV8_E4M3 ? kv8_prompt_kernel<D, CB_KV8_E4M3, HL> : kv8_prompt_kernel<D, CB_KV8_INT8, HL>;
  if (const int rc = ensure_smem_attr((const void*)fn, kSmem)) return rc;
  fn<<<grid, kThreads, kSmem, st>>>(p);
  count_launch();
  return cudaGetLastError() == cudaSuccess ? CB_OK : CB_ERR_CUDA;
}

template <int D, int HL>
int launch_mass(const AttendParams& p, int bh, int longest, cudaStream_t st) {
  constexpr int kSmem = Mass<D, HL>::kSmem;
  auto fn = p.c.format == CB_KV8_E4M3 ? kv8_prompt_mass_kernel<D, CB_KV8_E4M3, HL>
                                      : kv8_prompt_mass_kernel<D, CB_KV8_INT8, HL>;
  if (const int rc = ensure_smem_attr((const void*)fn, kSmem)) return rc;
  fn<<<dim3(ceil_div(longest, kRows), bh), kThreads, kSmem, st>>>(p);
  count_launch();
  return cudaGetLastError() == cudaSuccess ? CB_OK : CB_ERR_CUDA;
}

}  // namespace

int kv8_prompt_mass_launch(const AttendParams& p, int bh, int longest, cudaStream_t st) {
  if (p.dtype == CB_F32)
    return p.c.head_dim == 64 ? launch_mass<64, 1>(p, bh, longest, st) : launch_mass<128, 1>(p, bh, longest, st);
  return p.c.head_dim == 64 ? launch_mass<64, 0>(p, bh, longest, st) : launch_mass<128, 0>(p, bh, longest, st);
}

int kv8_prompt_launch(const AttendParams& p, int bh, cudaStream_t st) {
  if (p.dtype == CB_F32) return p.c.head_dim == 64 ? launch_prompt<64, 1>(p, bh, st) : launch_prompt<128, 1>(p, bh, st);
  return p.c.head_dim == 64 ? launch_prompt<64, 0>(p, bh, st) : launch_prompt<128, 0>(p, bh, st);
}

}  // namespace cb
