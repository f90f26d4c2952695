// Softmax cross entropy over a vocabulary from hidden rows, without keeping the logits.
//
//   x = h W^T       lse_n = log sum_v exp x_nv       loss_n = lse_n - x_n,t(n)
//   G_nv = a_n p_nv - b_n [v = t(n)],  p = exp(x - lse),  a = dL/dloss + dL/dlse,  b = dL/dloss
//   dh = G W        dW = G^T h
//
// Bound by the matrix products: 2 N V d operations forward, 6 N V d backward (the logits
// again, and two products), against N d + V d elements read.  All of them run in one
// kernel on the 5th-generation tensor cores:
//   * a pair of CTAs (cta_group::2) owns a 256 x 256 tile: each holds 128 of its rows, the
//     accumulator in tensor memory (two of them, so that a tile's products run under the
//     last tile's epilogue), and brings half of the columns' operand;
//   * a thread of each CTA copies 64-wide steps of K by TMA into six or seven stages, one of
//     the pair issues tcgen05.mma, eight warps a CTA take the accumulators out of tensor
//     memory;
//   * operands lie as the caller has them: logits read h and W along K; dh reads W, and dW
//     reads G and h, across it (MN-major operands), so that nothing is transposed.
// Forward: a pair takes a run of tiles along the vocabulary and keeps its rows' maximum and
// sum over them; a second kernel joins the runs in order.  Backward: G of a piece of the
// vocabulary goes to memory in the operands' type, both products of the piece follow in one
// launch; dh adds the pieces up in float32.
// float32 operands are two f16 parts each (11 + 11 bits, of the value times a power of two),
// three products of parts (what is left out is up to 2^-22 of a product), where the values
// lie in the range that this is right for, which the kernel that makes the parts finds out;
// else three bf16 parts (8 + 8 + 8 bits, and float32's range), six products.  Against bf16,
// which is one part: two products and three.
// Measured, 16384 x 32000 x 768 in bf16, back to back, which the power limit holds down: loss
// 590 us = 1.36 PFLOP/s (530 to 640 as it sets in), with the gradient 2780 us = 1.16 PFLOP/s.
// Single launches under ncu, tensor pipe: the logits 87 %, G's pass 74 % (its epilogue; it holds
// 128 logits a thread and spills 48 bytes of 168 registers), the products 90 %.  5 rows 15.5 us,
// 128 rows of float32 against bf16 23 us, of which one read of W is 7.5.
// Every wait is bounded (%globaltimer).  One that gives up sets CB_ERR_TIMEOUT, and what its
// CTA had still to give is NaN, so that a caller without a status word sees it too.
#include <cuda.h>

#include <algorithm>
#include <atomic>

#include "ends.cuh"

namespace cb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTileM = 256, kTileN = 256;  // of a pair
constexpr int kStep = 64;                  // of K: 128 bytes, a swizzled row
constexpr int kMaxStages = 12;
constexpr int kHalfBytes = 128 * kStep * 2;  // one CTA's rows of one operand's step
constexpr int kStageBytes = 2 * kHalfBytes;
constexpr int kEpiWarps = 8;
constexpr int kBoxBytes = 32 * 128;  // a box on its way out: a warp's 32 rows, 128 bytes of each
constexpr int kSmem = 7 * kStageBytes + 1024;
constexpr int kThreads = kEpiWarps * 32 + 64;
constexpr int kMaxPasses = 6, kMaxPairs = 128;
// Sums in tensor memory are cut off, not rounded, after every 16 products, and each product two
// bits further down: over 1500 additions of float32 parts the gradients were 4e-5 off.  So a
// span of K is added up there, and the spans in registers, rounded: 1024 of K, or 256 where float32
// parts are multiplied.
// Logits, whose errors nothing averages: 768 of K, of float16, whose products have more bits to
// be cut, 512.  lse of rows of 1024 is then 5.4e-7 (bf16) and 5.7e-7 (f16) off, in spans of 1024
// 8.6e-7 and 1.2e-6, the plain float32 form 2.5e-7 and 3.8e-7; 16384 x 32000 x 768 takes 615 us in
// bf16 (640 in spans of 512) and 661 in f16 (647 in spans of 1024, 715 of 256).  256 for up to 64
// rows, which wait for W (5 rows of 768 columns in bf16 8e-8 off, 17.5 us; one span 2.4e-7, 16.5).
constexpr int kSpan16 = 16, kSpan32 = 4, kSpanBf16Logits = 12, kSpanF16Logits = 8, kSpan32Rows = 64;
constexpr uint64_t kWaitNs = 2000000000ull, kDrainNs = 10000000ull;
// cb_linear_ce_set_wait_limit's
std::atomic<uint64_t> wait_limit{kWaitNs};
std::atomic<int32_t> stalled_pair{-1};

// 16-bit rows up to which the backward pass holds G in two parts.  One part is off by half a
// step, as the results' own rounding is: over many rows their errors come to 1.2 to 1.4 of what
// rounding the results alone gives, but of few rows single roundings show (3 rows of f16, dW 1.7
// times).  The second part takes 8 to 14 % of the loss with its gradient up to 128 rows (32000 x
// 768 in bf16: 3 rows 80 us and 89, 128 rows 86 and 97), 18 to 45 % of 256 to 1001 rows (256 rows
// 92 and 108, over 200000 x 1024 461 and 664; 1001 rows 184 and 269).
constexpr int kTwoRows = 128;

// Rows up to which the forward has them as columns and the vocabulary as rows of its tiles.
constexpr int kFew = 128;

enum { STATS = 0, FEW = 1, GRAD = 2, PRODUCTS = 3 };
enum { OUT_STORE = 0, OUT_ADD = 1 };
// Stages of 32 KiB out of seven; the last is for what goes out.  (Two boxes a warp and five
// stages: 159 us instead of 152 for G of 16384 x 8192 x 768, the copies in are what waits.)
constexpr int stages_of(int mode) { return mode == STATS ? 7 : 6; }
static_assert(kEpiWarps * kBoxBytes == kStageBytes, "a box for each warp takes a stage");

// One matrix product D[m][n] = sum over passes and k of A[m][k] B[n][k].  An operand is a
// 16-bit matrix read along K (its rows are m or n) or across it (its rows are k); pass i
// adds a_part[i] / b_part[i] to the column it is read at, the place of a part of its values.
struct alignas(64) Gemm {
  CUtensorMap a, b, out;
  int a_mn;                        // PRODUCTS: A is read across K, as B always is there
  int a_base, b_base;              // added to the row it is read at
  // for operands in bf16 (or 16 bits as they came), and for float32 ones in f16
  int passes[2], a_part[2][kMaxPasses], b_part[2][kMaxPasses];
  int span[2];                     // steps of K that are added up in tensor memory
  int apart;                       // bf16 parts: the passes before the last, step by step, are a sum of their own
  int m_tiles, n_tiles, k_steps;   // k_steps of a pass
  int splits;                      // of K, each with an output of its own
  int out_f32, out_mode, split_mode;  // of the first split and of the others
  int out_rows;                    // between the splits' outputs
  const float* top;                // PRODUCTS: the output is final, G's units to be multiplied in (null: not yet)
};

constexpr uint32_t kKindF16 = 1u << 4, kKindBf16 = 1u << 4 | 1u << 7 | 1u << 10;  // D float32; A and B

struct alignas(64) Args {
  Gemm g[2];                       // STATS, GRAD: one; PRODUCTS: dW, dh
  int pairs;
  int whole;                       // PRODUCTS: items of dW, dealt in turn
  int from[kMaxPairs + 1];         // and where each pair's steps of dh begin
  const uint32_t* wide;            // 0 where the parts are f16 (null: not tried)
  uint32_t kind;                   // instruction descriptor without sizes and directions
  int tile_m, tile_n;              // rows and columns of a tile (PRODUCTS: kTileM, kTileN)
  int share;                       // FEW: parts of the rows' operand that a step of the vocabulary's meets, 1 or 3
  int part_cols;                   // and the columns between them
  int stages, stage_bytes;         // FEW
  // STATS, FEW and GRAD: rows, vocabulary rows, the vocabulary row that the tiles start at, and how many
  int N, V, v0, vp;
  Ids targets;
  float2* part;                    // of a row's sum.  STATS: [run][2][N]; FEW: [tile][2][N]
  float* xt;                       // [N]
  uint32_t* counter;               // set to 0
  const float* row_scale;          // STATS, FEW, f16 parts: what a row's logits are multiplied by
  const float4* rows;              // GRAD: (a, b, lse, that) of each row
  const float* top;                // and their largest factor
  const float* common;             // PRODUCTS, f16 parts: the largest value of h as dW's operand
  int g_parts, g_cols;             // of G: columns of one part
  int is_f16;                      // 16-bit operands are f16
  int32_t* status;
  uint64_t wait_ns;                // limit of a wait
  int stalled;                     // the pair that copies nothing (tests; none: -1)
};

// ------------------------------------------------------------- primitives
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint64_t now_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ bool try_wait(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, "
      "p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
__device__ __noinline__ bool slow_wait(uint32_t bar, uint32_t parity, uint64_t limit) {
  const uint64_t end = now_ns() + limit;
  while (!try_wait(bar, parity))
    if (now_ns() > end) return false;
  return true;
}
__device__ __forceinline__ bool bounded_wait(uint32_t bar, uint32_t parity, uint64_t limit) {
  for (int i = 0; i < 64; ++i)
    if (try_wait(bar, parity)) return true;
  return slow_wait(bar, parity, limit);
}
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(is));
  return is != 0;
}
// Whether any of the 128 threads of a half of the epilogue says so; a barrier of theirs.
__device__ __forceinline__ bool any_of_half(int half, bool is) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"((uint32_t)is), "r"(half + 1)
      : "memory");
  return any != 0;
}
__device__ __forceinline__ uint32_t in_leader(uint32_t addr) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ void copy_in(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
      "[%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void copy_out(const CUtensorMap* map, int x, int y, uint32_t src, int mode) {
  if (mode == OUT_ADD)
    asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map),
                 "r"(src), "r"(x), "r"(y)
                 : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(src),
                 "r"(x), "r"(y)
                 : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// The pair's products issued so far arrive at this barrier of both CTAs.
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"((uint32_t)add)
      : "memory");
}
// Operand of 128-byte swizzled rows (2 at bits 61-63, version 1 at bits 46-47), 8-row groups
// 1024 bytes apart; read across K, its 64-element column blocks lie a step's rows apart.
__device__ __forceinline__ uint64_t operand(uint32_t saddr) {
  constexpr uint32_t kBlock = kStep * 128;
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)(kBlock >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ void load32(uint32_t addr, float* v) {
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
__device__ __forceinline__ void load16(uint32_t addr, float* v) {
  uint32_t* u = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
      : "r"(addr));
}
__device__ __forceinline__ void loads_done() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two float32 operations in one instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Two values in 16 bits, the first in the low half.
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ float2 unpack_bf16(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
}
__device__ __forceinline__ float2 unpack_f16(uint32_t u) { return __half22float2(reinterpret_cast<const __half2&>(u)); }

// float32 as two f16 parts.  W: of the value times 2^8, right for values below 255 in rows
// whose largest is 2^-10 or more, against which what lies below f16's range, 2^-33, is 2^-23;
// W alone decides, so that both directions take the logits alike (a logit of thousands that
// came out another way would not be the one its lse is of).  h in front of the logits: of the
// row times the power of two that brings its largest value to [2^14, 2^15), so that no row
// depends on another.  h as dW's operand: of the rows times one power of two, that of their
// largest value (rows more than 2^17 below it lose bits of their part of dW).
constexpr int kNarrowShift = 8;
constexpr float kNarrowMost = 255.0f, kNarrowLeast = 1.0f / 1024;
// The exponent that brings `top` to [2^14, 2^15).
__device__ __forceinline__ int exponent_to_15(float top) {
  int e = 0;
  if (top > 0.0f && top < INFINITY) frexpf(top, &e);
  return 15 - min(max(e, -100), 128);
}

// G is held in units of the largest |a| or |b| of the call, `top`: a mean's G is p - [v = t]
// itself, whose largest entries lie below 1, where their rounding is smallest against them.
// float16, whose range ends soon: G of row n is held times 2^(13 + e), e >= 0 the exponent
// by which the row's |a| + |b| falls behind the largest it can be, so that it stays below
// 2^15 and a probability of 2^-26 is a normal number; dh is scaled back by rows, for dW the
// row of h is multiplied by 2^-e.
constexpr int kF16Shift = 13;
__device__ __forceinline__ bool has_gradient(float4 row) { return row.x != 0.0f || row.y != 0.0f; }
__device__ __forceinline__ float scale_of(float top) { return top > 0.0f ? top : 1.0f; }
// -e; 0 for rows whose factors are not finite.
__device__ __forceinline__ int row_exponent(float4 row, float top) {
  const float size = (fabsf(row.x) + fabsf(row.y)) / scale_of(top);
  int e = 0;
  if (size > 0.0f && size < INFINITY) frexpf(size, &e);
  return min(max(e - 2, -100), 0);
}
// What a product of G (16 bits or parts of float32) is multiplied by, beside top and rows'
// exponents; common: of h as dW's operand (null: of W).
__device__ __forceinline__ float product_scale(bool f16, bool narrow, const float* common) {
  if (!f16) return 1.0f;
  return ldexpf(1.0f, -kF16Shift - (!narrow ? 0 : common ? exponent_to_15(*common) : kNarrowShift));
}

// ------------------------------------------------------------------- work
struct Item {
  int gemm, m0, n0, first, steps, split;  // steps `first` .. of K; times the passes
  int tile;                               // along n
};

// The i-th item of a pair.  STATS and GRAD: a run of equal length of all tiles, rows after
// rows of tiles.  PRODUCTS: tiles of dW (or splits of them), dealt in turn, and then a run of
// all steps of all tiles of dh, as long as what it takes for all pairs to end together; a
// tile that lies in several runs has its sum in parts, in slots of their own.
template <int MODE>
__device__ __forceinline__ bool item_of(const Args& p, int pair, int i, Item& it) {
  if (MODE != PRODUCTS) {
    const Gemm& g = p.g[0];
    const int64_t all = (int64_t)g.m_tiles * g.n_tiles;
    const int64_t u = all * pair / p.pairs + i;
    if (u >= all * (pair + 1) / p.pairs) return false;
    it.gemm = 0;
    it.m0 = (int)(u / g.n_tiles) * p.tile_m;
    it.tile = (int)(u % g.n_tiles);
    it.n0 = it.tile * p.tile_n;
    it.first = 0;
    it.steps = g.k_steps;
    it.split = 0;
    return true;
  }
  const int mine = (p.whole - pair + p.pairs - 1) / p.pairs;
  it.gemm = i >= mine;
  const Gemm& g = p.g[it.gemm];
  int tile;
  if (!it.gemm) {
    const int idx = pair + i * p.pairs;
    it.split = idx % g.splits;
    tile = idx / g.splits;
    it.first = (int)((int64_t)g.k_steps * it.split / g.splits);
    it.steps = (int)((int64_t)g.k_steps * (it.split + 1) / g.splits) - it.first;
  } else {
    const int begin = p.from[pair], end = p.from[pair + 1];
    tile = begin / max(g.k_steps, 1) + i - mine;
    const int tile_at = tile * g.k_steps, at = max(begin, tile_at);
    if (at >= end) return false;
    it.first = at - tile_at;
    it.steps = min(end, tile_at + g.k_steps) - at;
    it.split = 0;
    for (int c = pair; p.from[c] > tile_at && at == begin; --c) it.split += p.from[c] > p.from[c - 1];
  }
  // dW's tiles go by rows of tiles, in turn: pairs that work at one time share their rows of
  // G^T.  dh's go by columns: the pairs a column of tiles apart share their rows of G.
  it.tile = it.gemm ? tile / g.m_tiles : tile % g.n_tiles;
  it.n0 = it.tile * kTileN;
  it.m0 = (it.gemm ? tile % g.m_tiles : tile / g.n_tiles) * kTileM;
  return true;
}

// One 128-byte row of a box, word j of which is f(j): eight 16-byte pieces, piece c at c ^ (row % 8).
template <typename F>
__device__ __forceinline__ void put_row(uint32_t box, int row, F&& f) {
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const uint32_t u0 = f(4 * c), u1 = f(4 * c + 1), u2 = f(4 * c + 2), u3 = f(4 * c + 3);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(box + row * 128 + ((c ^ (row & 7)) << 4)), "r"(u0),
                 "r"(u1), "r"(u2), "r"(u3)
                 : "memory");
  }
}

template <int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) gemm_kernel(const __grid_constant__ Args p) {
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t bars[2 * kMaxStages + 4];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x & 1, pair = blockIdx.x >> 1;
  const uint32_t base = (smem_u32(raw) + 1023) & ~1023u;
  const uint32_t out_at = base + stages_of(MODE) * kStageBytes;
  const int stages = MODE == FEW ? p.stages : stages_of(MODE), stage_bytes = MODE == FEW ? p.stage_bytes : kStageBytes;
  const int a_bytes = MODE == FEW ? p.tile_m * 64 : kHalfBytes;  // of a stage
  const uint32_t full = smem_u32(bars), empty = full + 8 * kMaxStages, done = empty + 8 * kMaxStages, freed = done + 16;

  if (tid == 0) {
    for (int i = 0; i < kMaxStages; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(full + 8 * i));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(empty + 8 * i));
    }
    for (int i = 0; i < 2; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(done + 8 * i));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(freed + 8 * i), "n"(2 * kEpiWarps));
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_abort = 0;
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s_tmem)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  cluster_sync();
  fence_after();
  await_before();
  if (MODE <= FEW && blockIdx.x == 0 && tid == 0) *p.counter = 0;
  const uint32_t tmem = s_tmem;
  const bool narrow = p.wide && *p.wide == 0;  // float32 in f16 parts
  volatile int* abort_flag = &s_abort;
  auto wait = [&](uint32_t bar, uint32_t parity) {
    if (*abort_flag) return false;
    if (bounded_wait(bar, parity, p.wait_ns)) return true;
    *abort_flag = 1;
    return false;
  };

  if (warp == kEpiWarps) {
    // ---------------------------------------------------------- copies in
    if (elect_one()) {
      int n = 0;  // steps so far
      Item it;
      bool go = pair != p.stalled;
      for (int i = 0; go && item_of<MODE>(p, pair, i, it); ++i) {
        const Gemm& g = p.g[MODE == PRODUCTS ? it.gemm : 0];
        const int n_rows = MODE == PRODUCTS ? kTileN / 2 : p.tile_n / 2, m_rows = MODE == FEW ? p.tile_m / 2 : 128;
        const int m = it.m0 + rank * m_rows, c = it.n0 + rank * n_rows;
        const uint32_t bytes = 2 * (m_rows + (MODE == FEW ? p.share : 1) * n_rows) * 128;
        // a span of K at a time, all passes over it, or those apart and then the last
        const int span = g.span[narrow], passes = g.passes[narrow];
        const bool apart = (MODE == STATS || MODE == GRAD) && g.apart && !narrow;
        for (int from = 0; go && from < it.steps; from += span)
          for (int k = 0, pass = 0, end = min(span, it.steps - from); pass < passes; ++n) {
            const int ap = g.a_part[narrow][pass], bp = g.b_part[narrow][pass];
            const int st = n % stages, k0 = (it.first + from + k) * kStep;
            if (n >= stages && !wait(empty + 8 * st, (n / stages - 1) & 1)) {
              go = false;
              break;
            }
            const uint32_t bar = in_leader(full + 8 * st), at = base + st * stage_bytes, bt = at + a_bytes;
            if (rank == 0)
              asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full + 8 * st), "r"(bytes)
                           : "memory");
            if (MODE == PRODUCTS && g.a_mn) {
              copy_in(at, &g.a, m + ap, g.a_base + k0, bar);
              copy_in(at + kHalfBytes / 2, &g.a, m + 64 + ap, g.a_base + k0, bar);
            } else {
              copy_in(at, &g.a, k0 + ap, g.a_base + m, bar);
            }
            if (MODE == PRODUCTS) {  // both products read their second operand across K
              copy_in(bt, &g.b, c + bp, g.b_base + k0, bar);
              copy_in(bt + kHalfBytes / 2, &g.b, c + 64 + bp, g.b_base + k0, bar);
            } else {
              const bool shared = MODE == FEW && p.share > 1;
              copy_in(shared ? bt + rank * n_rows * 128 : bt, &g.b, k0 + bp, g.b_base + c, bar);
              if (shared) {
                copy_in(bt + (rank ^ 1) * n_rows * 128, &g.b, k0 + p.part_cols, c, bar);
                copy_in(bt + 2 * n_rows * 128, &g.b, k0 + 2 * p.part_cols, c, bar);
              }
            }
            if (apart && pass < passes - 1) {
              if (++pass < passes - 1) continue;
              pass = ++k < end ? 0 : passes - 1;
              if (k == end) k = 0;
            } else if (++k == end) {
              k = 0;
              ++pass;
            }
          }
      }
    }
    __syncwarp();
  } else if (warp == kEpiWarps + 1) {
    // ----------------------------------------------------------- products
    if (rank == 0) {
      const bool lead = elect_one();
      int n = 0, sums = 0;
      Item it;
      bool go = true;
      for (int i = 0; go && item_of<MODE>(p, pair, i, it); ++i) {
        const Gemm& g = p.g[MODE == PRODUCTS ? it.gemm : 0];
        const bool a_mn = MODE == PRODUCTS && g.a_mn;
        const uint32_t id = (narrow ? kKindF16 : p.kind) | (a_mn ? 1u << 15 : 0u) | (MODE == PRODUCTS ? 1u << 16 : 0u) |
                            (uint32_t)((MODE == PRODUCTS ? kTileN : p.tile_n) >> 3) << 17 | (uint32_t)(kTileM >> 4) << 24;
        // 16 of K: 32 bytes of a row, or 16 rows
        const uint32_t a_step = a_mn ? 2048 / 16 : 2, b_step = MODE == PRODUCTS ? 2048 / 16 : 2;
        const int span = g.span[narrow], passes = g.passes[narrow];
        const int apart = (MODE == STATS || MODE == GRAD) && g.apart && !narrow;
        for (int from = 0, last = !apart; go && from < it.steps;
             from += last ? span : 0, last = !apart || !last, ++sums) {
          const int acc = sums & 1, steps = min(span, it.steps - from) * (!apart ? passes : last ? 1 : passes - 1);
          if (sums >= 2) go = __all_sync(0xffffffffu, wait(freed + 8 * acc, (sums / 2 - 1) & 1));
          fence_after();
          const uint32_t d = tmem + acc * kTileN;
          for (int k = 0; k < steps && go; ++k, ++n) {
            const int st = n % stages;
            go = __all_sync(0xffffffffu, wait(full + 8 * st, (n / stages) & 1));
            if (!go) break;
            fence_after();
            if (lead) {
              const uint64_t a = operand(base + st * stage_bytes), b = operand(base + st * stage_bytes + a_bytes);
              // Parts that share a step: the first two in one product of twice the columns, the
              // third on to the second's, which lie side by side: half a product's columns come
              // from either CTA, and the right one holds the two parts the other way round.
              const bool shared = MODE == FEW && p.share > 1;
              const uint32_t id0 = shared ? id + ((uint32_t)(p.tile_n >> 3) << 17) : id;
#pragma unroll
              for (int s = 0; s < kStep / 16; ++s) mma(d, a + s * a_step, b + s * b_step, id0, k > 0 || s > 0);
              if (shared)
#pragma unroll
                for (int s = 0; s < kStep / 16; ++s)
                  mma(d + p.tile_n / 2, a + s * a_step, b + 2 * p.tile_n * 4 + s * b_step, id, true);
              commit(empty + 8 * st);
            }
            __syncwarp();
          }
          if (go && lead) commit(done + 8 * acc);
          __syncwarp();
        }
      }
      if (!go) {  // what is in flight ends before the memory goes
        for (int k = 0; k < stages; ++k) {
          const int last = n - 1 - k;
          if (last >= 0) bounded_wait(empty + 8 * (last % stages), (last / stages) & 1, kDrainNs);
        }
        for (int k = 0; k < stages; ++k) bounded_wait(full + 8 * ((n + k) % stages), ((n + k) / stages) & 1, kDrainNs);
      }
    }
  } else {
    // ----------------------------------------------------------- epilogue
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const bool f16 = p.is_f16 || narrow;
    const uint32_t lane_at = (uint32_t)((warp & 3) * 32) << 16;
    auto half_sync = [&] { asm volatile("bar.sync %0, 128;" ::"r"(half + 1) : "memory"); };
    auto warp_bar = [&] { asm volatile("bar.sync %0, 32;" ::"r"(warp + 3) : "memory"); };
    // the warp's rows, 128 bytes of each, go out as a box
    auto send = [&](const CUtensorMap* map, int x, int y, int mode, auto&& word) {
      const uint32_t box = out_at + warp * kBoxBytes;
      if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      warp_bar();
      put_row(box, lane, word);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      warp_bar();
      if (lane == 0) copy_out(map, x, y + (warp & 3) * 32, box, mode);
    };
    float m = -INFINITY, l = 0.0f;  // STATS: of the row over the run
    int run = -1, slot = 0;
    int64_t target = -1;
    float4 f = make_float4(0, 0, 0, 0);
    auto leave = [&] {  // STATS: the run's part of the row's sum
      if (run >= 0 && run + rank * 128 + row < p.N)
        p.part[((int64_t)slot * 2 + half) * p.N + run + rank * 128 + row] = make_float2(m, l);
    };
    // FEW: the thread's one or two rows, over a quarter of each tile
    const int quarter = warp & 3;
    const uint32_t few_box = out_at + half * 4 * kBoxBytes;  // [32][128] logits
    int few_row[2], few_target[2];
    float few_unit[2], few_m[2] = {-INFINITY, -INFINITY}, few_l[2] = {};
    if constexpr (MODE == FEW)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int c = b * 32 + lane, r = half * (p.tile_n / 2) + c;
        few_row[b] = c < p.tile_n / 2 && r < p.N ? r : -1;
        const int64_t t = few_row[b] >= 0 ? p.targets[r] : -1;
        few_target[b] = t < p.V ? (int)t : -1;
        few_unit[b] = few_row[b] >= 0 && narrow ? p.row_scale[r] : 1.0f;
      }
    Item it;
    int sums = 0;
    for (int i = 0; item_of<MODE>(p, pair, i, it); ++i) {
      const int n = it.m0 + rank * 128 + row;
      const bool live = MODE != PRODUCTS && n < p.N;
      if ((MODE == STATS || MODE == GRAD) && it.m0 != run) {
        if (MODE == STATS) leave();
        run = it.m0;
        m = -INFINITY;
        l = 0.0f;
        target = live ? p.targets[n] : -1;
        if (target >= p.V) target = -1;
        if (MODE == GRAD) {
          f = live ? p.rows[n] : make_float4(0, 0, 0, 0);
          const float by = f16 ? ldexpf(1.0f, kF16Shift - row_exponent(f, *p.top)) : 1.0f;
          f.x = f.x / scale_of(*p.top) * by;
          f.y = f.y / scale_of(*p.top) * by;
        }
        if (MODE == STATS) {
          f.w = live && narrow ? p.row_scale[n] : 1.0f;
          // which of the runs over these rows this one is
          const int64_t all = (int64_t)p.g[0].m_tiles * p.g[0].n_tiles, from = (int64_t)(it.m0 / kTileM) * p.g[0].n_tiles;
          slot = pair - (int)(((from + 1) * p.pairs - 1) / all);
        }
      }
      constexpr int kCols = MODE == FEW ? kFew / 2 : 128;  // a thread's
      float x[kCols];
      // this half's columns
      const int cols = MODE == PRODUCTS ? 128 : MODE == FEW ? p.tile_n / 2 : min(128, p.tile_n - half * 128);
      const Gemm& mine = p.g[MODE == PRODUCTS ? it.gemm : 0];
      const int spans = (it.steps + mine.span[narrow] - 1) / mine.span[narrow];
      bool go = true;
      for (int q = (MODE == STATS || MODE == GRAD) && mine.apart && !narrow ? 2 * spans : spans, first = 1; q > 0;
           --q, first = 0, ++sums) {
        const int acc = sums & 1;
        go = __all_sync(0xffffffffu, wait(done + 8 * acc, (sums / 2) & 1));
        if (!go) break;
        fence_after();
        // the half's columns; of parts that share a step the small ones' first, then the large one's
        const bool shared = MODE == FEW && p.share > 1;
        const uint32_t acc_at = tmem + lane_at + acc * kTileN;
        const uint32_t at = acc_at + (shared ? (1 + half) * cols : half * (MODE == FEW ? cols : 128));
        if (first) {
#pragma unroll
          for (int c = 0; c < kCols / 32; ++c)
            if (c * 32 < cols) load32(at + c * 32, x + c * 32);
          loads_done();
        }
        constexpr int kAtOnce = MODE == FEW ? 32 : 16;
        for (int more = first; more < (shared ? 2 : 1); ++more)
#pragma unroll
          for (int c = 0; c < kCols / kAtOnce; ++c)
            if (c * kAtOnce < cols) {
              float y[kAtOnce];
              if constexpr (MODE == FEW)
                load32((more ? acc_at + half * 3 * cols : at) + c * 32, y);
              else
                load16(at + c * 16, y);
              loads_done();
#pragma unroll
              for (int j = 0; j < kAtOnce; ++j) x[c * kAtOnce + j] += y[j];
            }
        fence_before();
        __syncwarp();
        if (lane == 0)
          asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(in_leader(freed + 8 * acc))
                       : "memory");
      }
      // The half's four warps agree.  After a wait that gave up all that follow do at once, and
      // what the CTA has still to give is NaN.
      if (any_of_half(half, !go))
#pragma unroll
        for (int c = 0; c < kCols; ++c) x[c] = NAN;
      if ((MODE == STATS || MODE == GRAD) && narrow)
#pragma unroll
        for (int c = 0; c < kCols; ++c) x[c] *= f.w;
      const int v = it.n0 + half * 128;  // of the piece, or of d
      const int at = (int)(target - p.v0 - v);  // the target's column
      const bool hit = (MODE == STATS || MODE == GRAD) && target >= 0 && at >= 0 && at < cols;
      if constexpr (MODE == PRODUCTS) {
        const Gemm& g = p.g[it.gemm];
        const int y = it.m0 + rank * 128 + it.split * g.out_rows;
        if (g.top) {
          const float s = scale_of(*g.top) * product_scale(f16, narrow, p.common);
#pragma unroll
          for (int c = 0; c < 128; ++c) x[c] *= s;
        }
        if (g.out_f32) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            send(&g.out, v + c * 32, y, it.split ? g.split_mode : g.out_mode,
                 [&](int j) { return __float_as_uint(x[c * 32 + j]); });
        } else {
#pragma unroll
          for (int c = 0; c < 2; ++c)
            send(&g.out, v + c * 64, y, OUT_STORE, [&](int j) {
              const float lo = x[c * 64 + 2 * j], hi = x[c * 64 + 2 * j + 1];
              return p.is_f16 ? pack_f16(lo, hi) : pack_bf16(lo, hi);
            });
        }
      }
      if constexpr (MODE == FEW) {
        // Lanes hold vocabulary rows, columns the few rows.  Turned over in shared memory, 32
        // columns at a time (word j * 128 + (row ^ j), free of bank conflicts both ways), a
        // thread takes a quarter of the tile's logits of one row.
        const int v0 = it.m0 + rank * (p.tile_m / 2), valid = min(p.tile_m / 2, p.V - v0);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          if (b * 32 >= cols) break;
          if (b) half_sync();
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (b * 32 + (j & 16) < cols)
              asm volatile("st.shared.f32 [%0], %1;" ::"r"(few_box + (j * 128 + (row ^ j)) * 4), "f"(x[b * 32 + j])
                           : "memory");
          half_sync();
          if (few_row[b] < 0) continue;
          float y[32], t = few_m[b];
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            asm volatile("ld.shared.f32 %0, [%1];"
                         : "=f"(y[k])
                         : "r"(few_box + (lane * 128 + ((quarter * 32 + k) ^ lane)) * 4));
            y[k] = quarter * 32 + k < valid ? y[k] * few_unit[b] : -INFINITY;
          }
#pragma unroll
          for (int k = 0; k < 32; k += 2) t = max3(t, y[k], y[k + 1]);
          const float ref = t == -INFINITY ? 0.0f : t;
          float e[4] = {};
#pragma unroll
          for (int k = 0; k < 32; ++k) e[k & 3] += exp2_of((y[k] - ref) * kLog2e);
          few_l[b] = fmaf(few_l[b], exp2_of((few_m[b] - ref) * kLog2e), (e[0] + e[1]) + (e[2] + e[3]));
          few_m[b] = t;
          const int own = few_target[b] - v0;
          if (few_target[b] >= 0 && own >= quarter * 32 && own < min(valid, quarter * 32 + 32)) {
            float at_target;
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(at_target) : "r"(few_box + (lane * 128 + (own ^ lane)) * 4));
            p.xt[few_row[b]] = at_target * few_unit[b];
          }
        }
      }
      if constexpr (MODE == STATS) {
        if (v + cols > p.vp)  // the last tile
#pragma unroll
          for (int c = 0; c < 128; ++c)
            if (v + c >= p.vp) x[c] = -INFINITY;
        if (__any_sync(0xffffffffu, hit)) {
          float t = 0.0f;
#pragma unroll
          for (int c = 0; c < 128; ++c) t = c == at ? x[c] : t;
          if (hit) p.xt[n] = t;
        }
        float top[4] = {m, m, m, m};
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (g * 32 < cols)
#pragma unroll
            for (int c = g * 32; c < g * 32 + 32; c += 2) top[c / 2 & 3] = max3(top[c / 2 & 3], x[c], x[c + 1]);
        const float t = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        const float ref = t == -INFINITY ? 0.0f : t;
        const float2 off = make_float2(-ref, -ref), scale = make_float2(kLog2e, kLog2e);
        // The tile's own sum first: against the run's, which grows long, each of its terms would be
        // rounded (a run of 2^20 vocabulary rows: lse 4e-5 off in the mean square, so below 2.4e-6).
        float2 s[4] = {};
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (g * 32 < cols)
#pragma unroll
            for (int c = g * 32; c < g * 32 + 32; c += 2) {
              const float2 e = mul2(add2(make_float2(x[c], x[c + 1]), off), scale);
              s[c / 2 & 3] = add2(s[c / 2 & 3], make_float2(exp2_of(e.x), exp2_of(e.y)));
            }
        const float2 both = add2(add2(s[0], s[1]), add2(s[2], s[3]));
        l = fmaf(l, exp2_of((m - ref) * kLog2e), both.x + both.y);
        m = t;
      }
      if constexpr (MODE == GRAD) {
        const float2 off = make_float2(-f.z, -f.z), scale = make_float2(kLog2e, kLog2e), by = make_float2(f.x, f.x);
#pragma unroll
        for (int c = 0; c < 128; c += 2) {
          const float2 e = mul2(add2(make_float2(x[c], x[c + 1]), off), scale);
          const float2 g = mul2(make_float2(exp2_of(e.x), exp2_of(e.y)), by);
          x[c] = g.x;
          x[c + 1] = g.y;
        }
        if (__any_sync(0xffffffffu, hit)) {
#pragma unroll
          for (int c = 0; c < 128; ++c) x[c] = hit && c == at ? x[c] - f.y : x[c];
        }
        if (v + cols > p.vp)
#pragma unroll
          for (int c = 0; c < 128; ++c)
            if (v + c >= p.vp) x[c] = 0.0f;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (v + c * 64 >= p.g_cols) continue;
          const int parts = narrow ? 2 : p.g_parts, y = it.m0 + rank * 128;
          int at_part = v + c * 64;
          for (int part = 1; part < parts; ++part, at_part += p.g_cols)
            send(&p.g[0].out, at_part, y, OUT_STORE, [&](int j) {
              float &lo = x[c * 64 + 2 * j], &hi = x[c * 64 + 2 * j + 1];
              const uint32_t u = f16 ? pack_f16(lo, hi) : pack_bf16(lo, hi);
              const float2 is = f16 ? unpack_f16(u) : unpack_bf16(u);
              lo -= is.x;  // what is left for the next part
              hi -= is.y;
              return u;
            });
          if (f16)
            send(&p.g[0].out, at_part, y, OUT_STORE,
                 [&](int j) { return pack_f16(x[c * 64 + 2 * j], x[c * 64 + 2 * j + 1]); });
          else
            send(&p.g[0].out, at_part, y, OUT_STORE,
                 [&](int j) { return pack_bf16(x[c * 64 + 2 * j], x[c * 64 + 2 * j + 1]); });
        }
      }
    }
    if (MODE == STATS) leave();
    if constexpr (MODE == FEW) {  // a warp joins the quarters
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        half_sync();
        asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(few_box + (quarter * 32 + lane) * 8), "f"(few_m[b]),
                     "f"(few_l[b])
                     : "memory");
        half_sync();
        if (quarter == 0 && few_row[b] >= 0) {
          float2 q[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];"
                         : "=f"(q[k].x), "=f"(q[k].y)
                         : "r"(few_box + (k * 32 + lane) * 8));
          const float t = fmaxf(fmaxf(q[0].x, q[1].x), fmaxf(q[2].x, q[3].x)), ref = t == -INFINITY ? 0.0f : t;
          float sum = 0.0f;
#pragma unroll
          for (int k = 0; k < 4; ++k) sum += q[k].y * exp2_of((q[k].x - ref) * kLog2e);
          p.part[((int64_t)pair * 2 + rank) * p.N + few_row[b]] = make_float2(t, sum);
        }
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  // (at the start it would have small kernels wait beside these CTAs: 33 us instead of 27 for 128 rows of float32)
  start_next();
  fence_before();
  __syncthreads();
  cluster_sync();  // no CTA leaves while the pair's products or arrivals may reach it
  fence_after();
  if (tid == 0 && s_abort) set_status(p.status, CB_ERR_TIMEOUT);
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

// --------------------------------------------------------- before and after
struct Problem {
  int N, V, d;
  Ids targets;
};

__device__ __forceinline__ int64_t target_of(const Problem& p, int n) {
  const int64_t t = p.targets[n];
  return t >= 0 && t < p.V ? t : -1;
}

constexpr int kRowThreads = 256;

// Joins the runs' parts of a row's sum, LANES threads to a row (32 where few rows are in many
// parts).  A reduced loss: the CTAs' sums, which the last CTA adds up in order.
template <int LANES>
__global__ void __launch_bounds__(kRowThreads) join_kernel(Problem p, int few, int n_tiles, int m_tiles, int pairs,
                                                           const float2* part, const float* xt, float* rows, float* lse,
                                                           int reduction, float* loss, int32_t* count, float* rest,
                                                           double2* sums, uint32_t* counter,
                                                           int32_t* status) {
  __shared__ double s_sum[kRowThreads / 32], s_count[kRowThreads / 32];
  __shared__ int s_last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = (blockIdx.x * kRowThreads + threadIdx.x) / LANES;
  await_before();
  start_next();
  double sum = 0.0, has = 0.0;
  const int64_t all = (int64_t)m_tiles * n_tiles, from = (int64_t)(n / kTileM) * n_tiles;
  const int parts =
      n >= p.N ? 0
      : few    ? 2 * pairs
               : 2 * ((int)(((from + n_tiles) * pairs - 1) / all) - (int)(((from + 1) * pairs - 1) / all) + 1);
  float m = -INFINITY, l = 0.0f;
  for (int i = threadIdx.x % LANES; i < parts; i += 4 * LANES) {
    float2 q[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      q[k] = i + k * LANES < parts ? part[(int64_t)(i + k * LANES) * p.N + n] : make_float2(-INFINITY, 0.0f);
    const float t = fmaxf(m, fmaxf(fmaxf(q[0].x, q[1].x), fmaxf(q[2].x, q[3].x))), ref = t == -INFINITY ? 0.0f : t;
    l *= expf(m - ref);
#pragma unroll
    for (int k = 0; k < 4; ++k) l += q[k].y * expf(q[k].x - ref);
    m = t;
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    const float qm = __shfl_xor_sync(0xffffffffu, m, o), ql = __shfl_xor_sync(0xffffffffu, l, o);
    const float t = fmaxf(m, qm), ref = t == -INFINITY ? 0.0f : t;
    l = l * expf(m - ref) + ql * expf(qm - ref);
    m = t;
  }
  if (n < p.N && threadIdx.x % LANES == 0) {
    // (in 64 bits: log l is off by as much as the sum is rounded, and a loss near 0 is a difference)
    const double log_l = log((double)l), whole = (double)m + log_l;
    const float rounded = (float)whole;
    lse[n] = rounded;
    if (rest) rest[n] = fabsf(rounded) < INFINITY ? (float)(whole - (double)rounded) : 0.0f;
    const int64_t t = p.targets[n];
    float row = 0.0f;
    if (t >= p.V) set_status(status, CB_ERR_TOKEN);
    if (t >= 0 && t < p.V) {
      row = (float)(((double)m - (double)xt[n]) + log_l);
      sum = row;
      has = 1.0;
    }
    if (reduction == CB_REDUCE_NONE) rows[n] = row;
  }
  if (reduction == CB_REDUCE_NONE) return;
  auto block_add = [&] {  // to thread 0
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      has += __shfl_xor_sync(0xffffffffu, has, o);
    }
    if (lane == 0) {
      s_sum[warp] = sum;
      s_count[warp] = has;
    }
    __syncthreads();
    sum = has = 0.0;
    if (threadIdx.x == 0)
      for (int w = 0; w < kRowThreads / 32; ++w) {
        sum += s_sum[w];
        has += s_count[w];
      }
  };
  block_add();
  if (threadIdx.x == 0) {
    if (gridDim.x > 1) {
      sums[blockIdx.x] = make_double2(sum, has);
      __threadfence();
      s_last = atomicAdd(counter, 1u) == gridDim.x - 1;
      __threadfence();
    } else {
      s_last = 1;
    }
  }
  __syncthreads();
  if (!s_last) return;
  if (gridDim.x > 1) {
    sum = has = 0.0;
    for (int i = threadIdx.x; i < gridDim.x; i += kRowThreads) {
      const double2 q = __ldcg(sums + i);
      sum += q.x;
      has += q.y;
    }
    block_add();
  }
  if (threadIdx.x == 0) {
    *loss = (float)(reduction == CB_REDUCE_MEAN ? sum / fmax(has, 1.0) : sum);
    *count = (int)has;
  }
}

struct Upstream {
  const float *loss, *lse;  // either may be null
  int64_t loss_step, lse_step;
  const int32_t* count;  // mean: rows with a target
  int reduction;
  const float* rest;     // what rounding took off lse (may be null)
};

// rows[n] = (a, b, lse, -) as they come from above, and *top = the largest |a| or |b|: one
// for all rows of a reduced loss; else a maximum (which does not depend on the order it is
// taken in), *top starting at 0.
__global__ void __launch_bounds__(kRowThreads) factors_kernel(Problem p, Upstream u, const float* lse, float4* rows,
                                                              float* top, float* common, uint32_t* wide) {
  const int n = blockIdx.x * kRowThreads + threadIdx.x;
  const bool one_top = u.reduction != CB_REDUCE_NONE && !u.lse;
  await_before();
  start_next();
  if (wide && n == 0) *wide = 0;
  if (common && n == 0) *common = 0.0f;
  float one = u.loss && u.reduction != CB_REDUCE_NONE ? *u.loss : 0.0f;
  if (u.reduction == CB_REDUCE_MEAN) one /= (float)max(*u.count, 1);
  if (one_top && n == 0) *top = fabsf(one) < INFINITY ? fabsf(one) : 0.0f;
  float size = 0.0f;
  if (n < p.N) {
    float b = 0.0f;
    if (u.loss && target_of(p, n) >= 0) b = u.reduction == CB_REDUCE_NONE ? u.loss[n * u.loss_step] : one;
    const float a = b + (u.lse ? u.lse[n * u.lse_step] : 0.0f);
    // (a row without a gradient is read as zeros, and its G is 0 whatever its own lse is)
    // p = exp(x - lse - rest)
    const float of_p = u.rest && a != 0.0f ? a * expf(-u.rest[n]) : a;
    rows[n] = make_float4(of_p, b, a == 0.0f && b == 0.0f ? 0.0f : lse[n], 0.0f);
    size = fmaxf(fabsf(a), fabsf(b));
    if (!(size < INFINITY)) size = 0.0f;
  }
  if (one_top) return;
  size = warp_max(size);
  if ((threadIdx.x & 31) == 0 && size > 0.0f) atomicMax(reinterpret_cast<int*>(top), __float_as_int(size));
}

// A matrix to be made an operand: rows of dp columns a part.  rows given: rows without a
// gradient become zeros.  scaled given: a second copy for dW, f16 rows multiplied by
// 2^row_exponent.
enum { SCALE_FIXED = 0, SCALE_ROW = 1, SCALE_COMMON = 2 };  // of f16 parts of float32, see kNarrowShift
struct Source {
  const void* x;
  int64_t ld, n;
  float4* rows;
  uint16_t *out, *scaled;
  int scale;
  float* unit;  // SCALE_ROW: what the row's logits are to be multiplied by
  int64_t unit_step;
};
struct Sources {
  Source s[2];
  int d, dp;
  const float* top;
  float* common;   // SCALE_ROW: raised to the rows' largest value; SCALE_COMMON: that (null: not wanted)
  uint32_t* wide;  // set where f16 parts do not fit (null: not tried)
};

// Eight columns of a row.  WIDE: rows are 16-byte aligned and d a multiple of 8.
template <typename T, bool WIDE>
__device__ __forceinline__ Vec<T, 8> load8(const T* row, int j0, int d) {
  Vec<T, 8> v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v.v[j] = Elem<T>::put(0.0f);
  if (WIDE) {
    if (j0 < d)
#pragma unroll
      for (int k = 0; k < 8; k += 16 / sizeof(T))
        *reinterpret_cast<uint4*>(&v.v[k]) = *reinterpret_cast<const uint4*>(row + j0 + k);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j0 + j < d) v.v[j] = row[j0 + j];
  }
  return v;
}

// 16-bit rows as they are, float32 ones as three bf16 parts; after a try in f16 parts only
// where *wide is set.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kRowThreads) operand_kernel(Sources p, int64_t first, int64_t blocks) {
  constexpr int kParts = sizeof(T) == 4 ? 3 : 1;
  await_before();
  start_next();
  if (p.wide && *p.wide == 0) return;
  for (int64_t block = blockIdx.x; block < blocks; block += gridDim.x) {
    const bool second = block >= first;
    const Source& s = p.s[second];
    const int64_t i = (block - (second ? first : 0)) * kRowThreads + threadIdx.x;
    const uint32_t pieces = p.dp / 8;
    const int64_t n = i < (1ll << 32) ? (int64_t)((uint32_t)i / pieces) : i / pieces;
    if (n >= s.n) continue;
    const int j0 = (int)(i - n * pieces) * 8;
    const float4 row = s.rows ? s.rows[n] : make_float4(1.0f, 0.0f, 0.0f, 0.0f);
    Vec<T, 8> v = load8<T, WIDE>(static_cast<const T*>(s.x) + n * s.ld, j0, has_gradient(row) ? p.d : 0);
    if constexpr (kParts == 1) {
      *reinterpret_cast<uint4*>(s.out + n * p.dp + j0) = *reinterpret_cast<const uint4*>(&v);
      if (!s.scaled) continue;
      const float by = ldexpf(1.0f, row_exponent(row, *p.top));
#pragma unroll
      for (int j = 0; j < 8; ++j) v.v[j] = Elem<T>::put(Elem<T>::get(v.v[j]) * by);
      *reinterpret_cast<uint4*>(s.scaled + n * p.dp + j0) = *reinterpret_cast<const uint4*>(&v);
    } else {
#pragma unroll
      for (int k = 0; k < kParts; ++k) {
        uint32_t u[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          u[j] = pack_bf16(v.v[2 * j], v.v[2 * j + 1]);
          const float2 is = unpack_bf16(u[j]);
          v.v[2 * j] -= is.x;
          v.v[2 * j + 1] -= is.y;
        }
        const int64_t at = (n * kParts + k) * p.dp + j0;
        *reinterpret_cast<uint4*>(s.out + at) = make_uint4(u[0], u[1], u[2], u[3]);
        if (s.scaled) *reinterpret_cast<uint4*>(s.scaled + at) = make_uint4(u[0], u[1], u[2], u[3]);
      }
    }
  }
}

// Eight values, times `by`, as f16 parts dp columns apart: two of float32, one of bf16, which
// f16 holds whole.
template <typename T>
__device__ __forceinline__ void put_parts(uint16_t* out, int dp, const Vec<T, 8>& v, float by) {
  float r[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = Elem<T>::get(v.v[j]) * by;
#pragma unroll
  for (int k = 0; k < (int)sizeof(T) / 2; ++k) {
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      u[j] = pack_f16(r[2 * j], r[2 * j + 1]);
      const float2 part = unpack_f16(u[j]);
      r[2 * j] -= part.x;
      r[2 * j + 1] -= part.y;
    }
    *reinterpret_cast<uint4*>(out + k * dp) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}

// float32 rows as two f16 parts (in rows laid out for three), bf16 rows as one, LANES threads
// to a row; sets *wide where values of W do not fit.  (A value that is not finite makes its
// sums NaN in any form, and is left to.)
template <typename T, bool WIDE, int LANES>
__global__ void __launch_bounds__(kRowThreads) narrow_kernel(Sources p, int64_t first) {
  constexpr int kLaid = sizeof(T) == 4 ? 3 : 1;
  const bool second = blockIdx.x >= first;
  const Source& s = p.s[second];
  const int lane = threadIdx.x % LANES;
  const int64_t n = ((blockIdx.x - (second ? first : 0)) * kRowThreads + threadIdx.x) / LANES;
  await_before();
  start_next();
  const bool is = n < s.n;
  if (s.scale == SCALE_COMMON && *p.wide) return;  // dW takes the bf16 parts
  const float4 row = is && s.rows ? s.rows[n] : make_float4(1.0f, 0.0f, 0.0f, 0.0f);
  const int d = is && has_gradient(row) ? p.d : 0, dp = is ? p.dp : 0;
  const T* x = static_cast<const T*>(s.x) + n * s.ld;
  uint16_t* out = s.out + n * kLaid * p.dp;
  constexpr int kAhead = 3;  // pieces in flight: a row of 768
  float top = 0.0f;
  auto reduce_top = [&] {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  };
  int e = kNarrowShift;
  if (s.scale == SCALE_ROW) {
    for (int j0 = lane * 8; j0 < dp; j0 += LANES * 8) {
      const Vec<T, 8> v = load8<T, WIDE>(x, j0, d);
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(Elem<T>::get(v.v[j])));
    }
    reduce_top();
    e = exponent_to_15(top);
    if (is && lane == 0) {
      s.unit[n * s.unit_step] = ldexpf(1.0f, -e - kNarrowShift);
      const float mine = p.common && top < INFINITY ? ldexpf(top, row_exponent(row, *p.top)) : 0.0f;
      if (mine > 0.0f) atomicMax(reinterpret_cast<int*>(p.common), __float_as_int(mine));
    }
  }
  if (s.scale == SCALE_COMMON) e = exponent_to_15(*p.common) + row_exponent(row, *p.top);
  const float by = ldexpf(1.0f, e);
  for (int j0 = lane * 8; j0 < dp; j0 += kAhead * LANES * 8) {
    Vec<T, 8> v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) v[i] = load8<T, WIDE>(x, j0 + i * LANES * 8, d);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int j = j0 + i * LANES * 8;
      if (j >= dp) break;
      if (s.scale == SCALE_FIXED)
#pragma unroll
        for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(Elem<T>::get(v[i].v[k])));
      put_parts(out + j, p.dp, v[i], by);
    }
  }
  if (s.scale != SCALE_FIXED) return;
  reduce_top();
  if (lane == 0 && top < INFINITY && (top >= kNarrowMost || (top > 0.0f && top < kNarrowLeast))) *p.wide = 1;
}

// out[r][j] = the sum of the splits' results, scaled back; 0 in a row without a gradient.
// VEC columns a thread: 4 where d is a multiple of it.
template <typename T, int VEC>
__global__ void __launch_bounds__(kRowThreads) finish_kernel(const float* acc, int splits, int64_t split_rows, int da,
                                                             int64_t n_rows, int d, const float4* rows, const float* top,
                                                             const float* common, int f16, const uint32_t* wide, T* out) {
  const int64_t i = (int64_t)blockIdx.x * kRowThreads + threadIdx.x;
  const uint32_t pieces = d / VEC;
  const int64_t n = i < (1ll << 32) ? (int64_t)((uint32_t)i / pieces) : i / pieces;
  await_before();
  start_next();
  if (n >= n_rows) return;
  const int j = (int)(i - n * pieces) * VEC;
  float s[VEC] = {};
  for (int k = 0; k < splits; ++k) {
    const Vec<float, VEC> q = *reinterpret_cast<const Vec<float, VEC>*>(acc + (k * split_rows + n) * da + j);
#pragma unroll
    for (int c = 0; c < VEC; ++c) s[c] += q.v[c];
  }
  const bool live = !rows || has_gradient(rows[n]);
  const bool narrow = wide && *wide == 0;
  float by = scale_of(*top) * product_scale(f16 || narrow, narrow, common);
  if (rows && (f16 || narrow)) by = ldexpf(by, row_exponent(rows[n], *top));
  Vec<T, VEC> o;
#pragma unroll
  for (int c = 0; c < VEC; ++c) o.v[c] = Elem<T>::put(live ? s[c] * by : 0.0f);
  *reinterpret_cast<Vec<T, VEC>*>(out + n * d + j) = o;
}

// ------------------------------------------------------------------- host
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encoder() {
  static const EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult how;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &how) != cudaSuccess ||
        how != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeFn>(f);
  }();
  return fn;
}

// A matrix of rows `ld` elements apart, in boxes of 128 bytes x box_rows.
bool map_of(CUtensorMap* map, const void* at, CUtensorMapDataType type, int64_t rows, int64_t cols, int64_t ld,
            int box_rows) {
  const int size = type == CU_TENSOR_MAP_DATA_TYPE_FLOAT32 ? 4 : 2;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)(ld * size)};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / size), (cuuint32_t)box_rows}, steps[2] = {1, 1};
  return encoder() && encoder()(map, type, 2, const_cast<void*>(at), dims, strides, box, steps,
                                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool bad(const void* h, int32_t h_dtype, int64_t ldh, const void* w, int32_t w_dtype, int64_t ldw, int32_t N, int32_t V,
         int32_t d, const void* targets, int32_t targets_64, int32_t reduction) {
  if (!h || !w || !targets || N <= 0 || V <= 0 || d <= 0 || !is_dtype(h_dtype) || !is_dtype(w_dtype)) return true;
  if (h_dtype != w_dtype && !(h_dtype == CB_F32 && w_dtype == CB_BF16)) return true;
  if (ldh < 0 || (V > 1 && ldw < d)) return true;
  const int32_t by = reduction & ~CB_REDUCE_REST;
  if (by != CB_REDUCE_NONE && by != CB_REDUCE_MEAN && by != CB_REDUCE_SUM) return true;
  return !aligned_to(h, dtype_size(h_dtype)) || !aligned_to(w, dtype_size(w_dtype)) ||
         !aligned_to(targets, targets_64 ? 8 : 4);
}

bool too_large(int32_t N, int32_t V, int32_t d) {
  return N > CB_ENDS_MAX_ROWS || V > CB_ENDS_MAX_VOCAB || d > CB_ENDS_MAX_DIM;
}

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// Whether a 16-bit matrix can be copied by TMA where it lies: a tensor map's rows are aligned
// and do not overlap.
bool direct(const void* x, int32_t dtype, int64_t ld, int64_t rows, int d) {
  return dtype != CB_F32 && aligned_to(x, 16) && (rows == 1 || (ld % 8 == 0 && ld >= d));
}

// Whether TMA can write contiguous rows of d columns there.
bool tma_rows(const void* x, int32_t dtype, int d) { return aligned_to(x, 16) && d * dtype_size(dtype) % 16 == 0; }

// Vocabulary rows whose G is held at a time: whole tiles, 256 MiB of G at most.
int piece_of(int32_t N, int32_t V, int parts) {
  const int64_t most = std::max<int64_t>(kTileM, (int64_t)(256 << 20) / ((int64_t)N * parts * 2) / kTileM * kTileM);
  const int pieces = (int)((V + most - 1) / most);
  return (int)up((V + pieces - 1) / pieces, kTileM);
}

// The products of parts that matter, those of a smaller part first: what tensor memory cuts
// off a sum is in proportion to the sum so far.  `least`: the orders of parts, the two added,
// that are left in.
int passes_of(Gemm& g, int narrow, int a_parts, int b_parts, int a_cols, int b_cols, int least = 2) {
  int n = 0;
  for (int both = least; both >= 0; --both)
    for (int i = std::min(both, a_parts - 1); i >= 0 && both - i < b_parts; --i) {
      g.a_part[narrow][n] = i * a_cols;
      g.b_part[narrow][n++] = (both - i) * b_cols;
    }
  g.passes[narrow] = n;
  g.span[narrow] = n == 1 ? kSpan16 : kSpan32;
  return n;
}

// How the two products are dealt: dW's tiles split `w` times along K, and the steps of dh
// that go to each pair.
struct Deal {
  int w, h_slots;
  int from[kMaxPairs + 1];
};

// When the last pair ends, if dh's steps fill what dW's items, dealt in turn, leave of a
// common end, and that end.
struct End {
  double last, common;
};
End end_of(int pairs, int items, double cost, double work) {
  const int odd = items % pairs, low = items / pairs;  // `odd` pairs have one item more
  double common = low * cost + work / (pairs - odd);   // if only the others get steps
  if (common > (low + 1) * cost || odd == 0) common = (items * cost + work) / pairs;
  return {std::max(common, items ? (low + (odd > 0)) * cost : 0.0), common};
}

// dW's split is the one whose pairs end first, counted in steps of K, with what a tile costs
// beside them and what the splits' float32 results cost in memory.
Deal deal(int pairs, int h_tiles, int h_steps, int h_passes, int w_tiles, int w_steps, int w_passes, double w_bytes,
          int w_most) {
  constexpr int kTileCost = 2;             // of filling and emptying, in steps
  constexpr double kBytesPerStep = 900e3;  // written and read back in a step's time by the whole device
  const double steps = (double)h_tiles * h_steps, work = steps * h_passes;
  Deal o;
  o.w = 1;
  double least = 1e30;
  auto cost = [&](int w) { return (double)w_steps * w_passes / w + kTileCost; };
  for (int w = 1; w_tiles && w <= 64 && w <= w_steps && w <= w_most; w *= 2) {
    const double t = end_of(pairs, w_tiles * w, cost(w), work).last + (w > 1 ? w * w_bytes / kBytesPerStep : 0.0);
    if (t < least * 0.99) {
      least = t;
      o.w = w;
    }
  }
  const int items = w_tiles * o.w, odd = items % pairs, low = items / pairs;
  const double end = end_of(pairs, items, cost(o.w), work).common;
  const double most = std::max(0.0, end - low * cost(o.w)) / h_passes;
  const double less = std::max(0.0, end - (low + 1) * cost(o.w)) / h_passes;
  for (int c = 0; c < pairs; ++c) o.from[c] = (int)std::min(steps, c < odd ? c * less : odd * less + (c - odd) * most);
  o.from[pairs] = (int)steps;
  // the most parts that a tile of dh lies in
  o.h_slots = 1;
  for (int c = 0, parts = 1; c < pairs && h_tiles; ++c) {
    if (o.from[c] == o.from[c + 1]) continue;
    parts = o.from[c] % h_steps == 0 ? 1 : parts + 1;
    o.h_slots = std::max(o.h_slots, parts);
    if (o.from[c + 1] / h_steps > o.from[c] / h_steps) parts = 1;
  }
  return o;
}

struct Shape {
  int N, V, d, dp;          // dp: columns of a part
  int h_parts, w_parts, g_parts;
  bool tried;               // float32 rows, in f16 parts if they fit
  CUtensorMapDataType type;  // of operands
  int f16;
  int pairs;                // on this device
  int piece;                // backward
  Shape(int32_t h_dtype, int32_t w_dtype, int N_, int V_, int d_) : N(N_), V(V_), d(d_), dp((int)up(d_, kStep)) {
    h_parts = h_dtype == CB_F32 ? 3 : 1;
    w_parts = w_dtype == CB_F32 ? 3 : 1;
    g_parts = h_parts == 1 && N <= kTwoRows ? 2 : h_parts;
    // bf16 W would be read where it lies for bf16 parts: worth a copy in f16 for many rows (the loss of 1100 rows, 32000
    // x 768: 110 us, 121 in bf16 parts; of 16384 1310 and 2050)
    tried = w_parts == 3 || (h_parts == 3 && N > 1024);
    f16 = h_dtype == CB_F16;
    type = f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    pairs = std::min(std::max(1, num_sms() / 2), kMaxPairs);
    piece = piece_of(N, V, g_parts);
  }
  uint32_t kind() const { return f16 ? kKindF16 : kKindBf16; }
  // The logits' passes.  Of float32 against bf16 the smaller parts of a step follow each other,
  // as they do where few rows share it: every form of the forward and the backward pass adds
  // alike.
  void logit_passes(Gemm& g, bool swapped) const {
    passes(g, h_parts, w_parts, dp, dp);
    if (h_parts == 1) g.span[0] = N <= kSpan32Rows ? kSpan32 : f16 ? kSpanF16Logits : kSpanBf16Logits;
    g.apart = h_parts > w_parts;
    if (g.apart) std::swap(g.a_part[0][0], g.a_part[0][1]);
    if (swapped) std::swap(g.a_part, g.b_part);
  }
  // The passes of a product of these parts, and of the f16 parts that take their place (two of
  // float32, one of bf16).  Returns how many there will be, as a rule.
  int passes(Gemm& g, int a_parts, int b_parts, int a_cols, int b_cols) const {
    const int n = passes_of(g, 0, a_parts, b_parts, a_cols, b_cols);
    return tried ? passes_of(g, 1, std::min(a_parts, 2), std::min(b_parts, 2), a_cols, b_cols, 1) : n;
  }
  // dW = G^T h; where dW is bf16, two of three bf16 parts will do
  int dw_passes(Gemm& g, int g_cols) const {
    const int n = passes(g, g_parts, h_parts, g_cols, dp);
    if (w_parts == h_parts) return n;
    passes_of(g, 0, g_parts, h_parts, g_cols, dp, 1);
    return g.passes[tried];
  }
  // whether W is read where it lies
  bool reads_w(const void* w, int32_t w_dtype, int64_t ldw) const { return !tried && direct(w, w_dtype, ldw, V, d); }
  int da() const { return (int)up(d, 4); }  // columns of a float32 result
};

// How a piece is dealt; scratch is laid out for the first, the largest.
Deal deal_of(const Shape& s, bool dh, bool dw, int vp, int w_most) {
  Gemm t;
  const int nt = ceil_div(s.d, kTileN);
  return deal(s.pairs, dh ? ceil_div(s.N, kTileM) * nt : 0, ceil_div(vp, kStep), s.passes(t, s.g_parts, s.w_parts, 0, 0),
              dw ? ceil_div(vp, kTileM) * nt : 0, ceil_div(s.N, kStep), s.dw_passes(t, 0),
              2.0 * vp * s.d * 4, w_most);
}

// Scratch, part by part; `at` null only counts.
struct Layout {
  char* at;
  size_t used = 0;
  template <typename T>
  T* take(int64_t n) {
    T* p = reinterpret_cast<T*>(at + used);
    used += (size_t)up(n * (int64_t)sizeof(T), 256);
    return p;
  }
};

struct Forward {
  uint16_t *h, *w;
  float2* part;
  float* xt;
  double2* sums;
  uint32_t *counter, *wide;
  float* unit;
  int few, tile_m, tile_n, m_tiles, n_tiles, pairs, slots;
  Forward(Layout& a, const Shape& s, bool h_direct, bool w_direct) {
    // Float32 rows against bf16 meet each step of the vocabulary once (128 rows, 32000 x 768: 27 us, 36 as rows of a
    // tile, three passes).  Otherwise it is read at memory's speed by tiles enough, with a quarter of the columns or
    // less (64 rows of bf16: 24000 x 768 16 us, as rows of a tile 18, 152000 x 1024 60 and 63; but 8192 x 1024 16 and
    // 13; 128 rows, 32000 x 768: 19 and 18.5).
    few = s.N <= (s.h_parts > s.w_parts ? kFew : s.V > 192 * s.pairs ? 64 : 16);
    if (few) {
      // the vocabulary in as many tiles as there are CTAs, or twice, .. as many, of equal height
      const int rounds = ceil_div(s.V, 256 * s.pairs);
      tile_m = 2 * std::min(128, (int)up(ceil_div(s.V, 2 * s.pairs * rounds), 8));
      tile_n = (int)up(s.N, 32);
      m_tiles = ceil_div(s.V, tile_m);
      n_tiles = 1;
    } else {
      tile_m = kTileM;
      tile_n = kTileN;
      m_tiles = ceil_div(s.N, kTileM);
      n_tiles = ceil_div(s.V, tile_n);
    }
    pairs = (int)std::min<int64_t>(s.pairs, (int64_t)m_tiles * n_tiles);
    slots = few ? pairs : ceil_div(pairs, m_tiles) + 1;
    h = h_direct ? nullptr : a.take<uint16_t>((int64_t)s.N * s.h_parts * s.dp);
    w = w_direct ? nullptr : a.take<uint16_t>((int64_t)s.V * s.w_parts * s.dp);
    part = a.take<float2>((int64_t)slots * 2 * s.N);
    xt = a.take<float>(s.N);
    sums = a.take<double2>(join_ctas(s.N));
    counter = a.take<uint32_t>(1);
    wide = s.tried ? a.take<uint32_t>(1) : nullptr;
    unit = s.tried ? a.take<float>(s.N) : nullptr;
  }
  int lanes() const { return 2 * slots > 16 ? 32 : 4; }  // of a row's parts
  int join_ctas(int N) const { return ceil_div(N, kRowThreads / lanes()); }
};

struct Backward {
  float4* rows;
  float *top, *common;
  uint32_t* wide;
  uint16_t *h, *hs, *w, *G;
  float *acc, *dw;
  Deal first;
  int h_slots, dw_direct;
  Backward(Layout& a, const Shape& s, bool w_direct, bool want_h, bool want_w, bool dw_aligned) {
    const int vp = std::min(s.piece, s.V);
    first = deal_of(s, want_h, want_w, vp, 64);
    dw_direct = dw_aligned && first.w == 1;
    h_slots = first.h_slots;
    if (s.V % s.piece) h_slots = std::max(h_slots, deal_of(s, want_h, want_w, s.V % s.piece, first.w).h_slots);
    rows = a.take<float4>(s.N);
    top = a.take<float>(1);
    common = s.tried && want_w ? a.take<float>(1) : nullptr;
    h = a.take<uint16_t>((int64_t)s.N * s.h_parts * s.dp);
    wide = s.tried ? a.take<uint32_t>(1) : nullptr;
    hs = (s.f16 || s.tried) && want_w ? a.take<uint16_t>((int64_t)s.N * s.h_parts * s.dp) : h;
    w = w_direct ? nullptr : a.take<uint16_t>((int64_t)s.V * s.w_parts * s.dp);
    G = a.take<uint16_t>((int64_t)s.N * s.g_parts * up(vp, kStep));
    acc = want_h ? a.take<float>((int64_t)h_slots * up(s.N, kTileM) * s.da()) : nullptr;
    dw = want_w && !dw_direct ? a.take<float>((int64_t)first.w * up(vp, kTileM) * s.da()) : nullptr;
  }
};

template <int MODE>
int launch(Args& p, cudaStream_t st) {
  p.wait_ns = wait_limit;
  p.stalled = stalled_pair;
  if (int rc = ensure_smem_attr((const void*)gemm_kernel<MODE>, kSmem)) return rc;
  return launch_after(gemm_kernel<MODE>, dim3(2 * p.pairs), kThreads, kSmem, st, p);
}

template <typename F>
int with_f32_or_bf16(int32_t dtype, F&& f) {
  return dtype == CB_F32 ? f(float{}) : f(__nv_bfloat16{});
}

// Up to two matrices of a type, and whether their rows can be read 16 bytes at a time.
struct Made {
  Sources p;
  int32_t dtype;
  bool aligned;
  Made(int32_t dtype_, const Shape& s, const Source& one, const Source& two, const float* top, float* common,
       uint32_t* wide)
      : p{{one, two}, s.d, s.dp, top, common, wide}, dtype(dtype_) {
    auto pieces = [&](const Source& x) { return !x.n || (aligned_to(x.x, 16) && x.ld * dtype_size(dtype) % 16 == 0); };
    aligned = s.d % 8 == 0 && pieces(one) && pieces(two);
  }
  // in f16 parts
  int narrow(cudaStream_t st) const {
    const int lanes = p.dp <= 64 ? 8 : 32;
    auto ctas = [&](const Source& x) { return (x.n * lanes + kRowThreads - 1) / kRowThreads; };
    return with_f32_or_bf16(dtype, [&](auto t) {
      using T = decltype(t);
      auto* fn = lanes == 8 ? (aligned ? narrow_kernel<T, true, 8> : narrow_kernel<T, false, 8>)
                            : (aligned ? narrow_kernel<T, true, 32> : narrow_kernel<T, false, 32>);
      return launch_after(fn, dim3((unsigned)(ctas(p.s[0]) + ctas(p.s[1]))), kRowThreads, 0, st, p, ctas(p.s[0]));
    });
  }
  // as they are, or in bf16 parts; after a try in f16 parts there is rarely anything to do
  int whole(cudaStream_t st) const {
    auto ctas = [&](const Source& x) { return (x.n * (p.dp / 8) + kRowThreads - 1) / kRowThreads; };
    const int64_t blocks = ctas(p.s[0]) + ctas(p.s[1]);
    const unsigned grid = (unsigned)(p.wide ? std::min<int64_t>(blocks, 8 * num_sms()) : blocks);
    return with_type(dtype, [&](auto t) {
      using T = decltype(t);
      return launch_after(aligned ? operand_kernel<T, true> : operand_kernel<T, false>, dim3(grid), kRowThreads, 0, st, p,
                          ctas(p.s[0]), blocks);
    });
  }
};

// h's and W's operands, as far as they have to be made.  f16 parts are tried for both before
// either is made in another form: one matrix that does not fit decides for both.
int make_operands(int32_t h_dtype, int32_t w_dtype, const Shape& s, const Source& h, const Source& w, const float* top,
                  float* common, uint32_t* wide, cudaStream_t st) {
  const bool together = h_dtype == w_dtype && h.out && w.out;
  const Made first(w_dtype, s, w, together ? h : Source{}, top, common, wide);
  const Made second(h_dtype, s, h, Source{}, top, common, wide);
  const bool has_first = w.out, has_second = h.out && !together;
  if (wide) {
    if (has_first)
      if (int rc = first.narrow(st)) return rc;
    if (has_second)
      if (int rc = second.narrow(st)) return rc;
    if (h.scaled) {
      Source dw = h;
      dw.out = h.scaled;
      dw.scale = SCALE_COMMON;
      if (int rc = Made(h_dtype, s, dw, Source{}, top, common, wide).narrow(st)) return rc;
    }
  }
  if (has_first)
    if (int rc = first.whole(st)) return rc;
  return has_second ? second.whole(st) : (int)CB_OK;
}

int finish(int32_t dtype, const float* acc, int splits, int64_t split_rows, const Shape& s, int64_t n_rows,
           const float4* rows, const float* top, const float* common, const uint32_t* wide, void* out, cudaStream_t st) {
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    const bool vecs = s.d % 4 == 0 && aligned_to(out, 4 * sizeof(T));
    const int64_t n = n_rows * (vecs ? s.d / 4 : s.d);
    return launch_after(vecs ? finish_kernel<T, 4> : finish_kernel<T, 1>,
                        dim3((unsigned)((n + kRowThreads - 1) / kRowThreads)), kRowThreads, 0, st, acc, splits, split_rows,
                        s.da(), n_rows, s.d, rows, top, common, s.f16, wide, static_cast<T*>(out));
  });
}

// An operand in memory: the caller's matrix, or one made from it.
struct Operand {
  const void* at;
  int64_t cols, ld;
  Operand(const void* x, int64_t ld_, int64_t rows, const uint16_t* made, int parts, const Shape& s) {
    at = made ? made : x;
    cols = made ? (int64_t)parts * s.dp : s.d;
    ld = made ? cols : rows == 1 ? up(s.d, 8) : ld_;
  }
};

}  // namespace
}  // namespace cb

using namespace cb;

extern "C" size_t cb_linear_ce_scratch_bytes(const void* h, int32_t h_dtype, int64_t ldh, const void* w, int32_t w_dtype,
                                             int64_t ldw, int32_t N, int32_t V, int32_t d, const void* dw,
                                             int32_t gradients) {
  if (N <= 0 || V <= 0 || d <= 0 || too_large(N, V, d) || !is_dtype(h_dtype) || !is_dtype(w_dtype) || gradients < 0 ||
      gradients > 3)
    return 0;
  const Shape s(h_dtype, w_dtype, N, V, d);
  Layout a{nullptr};
  const bool w_direct = s.reads_w(w, w_dtype, ldw);
  if (!gradients) {
    Forward f(a, s, direct(h, h_dtype, ldh, N, d), w_direct);
  } else {
    Backward f(a, s, w_direct, gradients & 1, gradients & 2, tma_rows(dw, w_dtype, d));
  }
  return a.used;
}

extern "C" int cb_linear_ce(const void* h, int32_t h_dtype, int64_t ldh, const void* w, int32_t w_dtype, int64_t ldw,
                            int32_t N, int32_t V, int32_t d, const void* targets, int32_t targets_64, int32_t reduction,
                            float* loss, float* lse, int32_t* count, void* scratch, size_t scratch_bytes,
                            int32_t* status, void* stream) {
  if (bad(h, h_dtype, ldh, w, w_dtype, ldw, N, V, d, targets, targets_64, reduction) || !loss || !lse || !scratch ||
      !aligned_to(scratch, 256) || (reduction != CB_REDUCE_NONE && !count))
    return CB_ERR_ARG;
  float* rest = reduction & CB_REDUCE_REST ? reinterpret_cast<float*>(count + 1) : nullptr;
  reduction &= ~CB_REDUCE_REST;
  if (too_large(N, V, d)) return CB_ERR_SHAPE;
  cudaStream_t st = (cudaStream_t)stream;
  const Shape s(h_dtype, w_dtype, N, V, d);
  Layout a{static_cast<char*>(scratch)};
  const Forward f(a, s, direct(h, h_dtype, ldh, N, d), s.reads_w(w, w_dtype, ldw));
  if (scratch_bytes < a.used) return CB_ERR_WORKSPACE;
  const Source hs{h, ldh, N, nullptr, f.h, nullptr, SCALE_ROW, f.unit, 1}, ws{w, ldw, V, nullptr, f.w};
  if (s.tried && cudaMemsetAsync(f.wide, 0, sizeof(uint32_t), st) != cudaSuccess) return CB_ERR_CUDA;
  if (int rc = make_operands(h_dtype, w_dtype, s, hs, ws, nullptr, nullptr, f.wide, st)) return rc;
  const Operand ho(h, ldh, N, f.h, s.h_parts, s), wo(w, ldw, V, f.w, s.w_parts, s);
  Args p{};
  Gemm& g = p.g[0];
  const Operand &ao = f.few ? wo : ho, &bo = f.few ? ho : wo;
  if (!map_of(&g.a, ao.at, s.type, f.few ? V : N, ao.cols, ao.ld, f.tile_m / 2) ||
      !map_of(&g.b, bo.at, s.type, f.few ? N : V, bo.cols, bo.ld, f.tile_n / 2))
    return CB_ERR_CUDA;
  p.share = 1;
  s.logit_passes(g, f.few);
  if (f.few && s.h_parts > s.w_parts) {
    // the rows' parts meet a step of the vocabulary together, which is then read once
    g.passes[0] = 1;
    g.b_part[0][0] = g.apart = 0;
    p.share = s.h_parts;
  }
  p.part_cols = s.dp;
  p.stage_bytes = f.tile_m * 64 + p.share * f.tile_n * 64;
  p.stages = std::min(kMaxStages, stages_of(FEW) * kStageBytes / p.stage_bytes);
  g.m_tiles = f.m_tiles;
  g.n_tiles = f.n_tiles;
  g.k_steps = s.dp / kStep;
  p.pairs = f.pairs;
  p.kind = s.kind();
  p.tile_m = f.tile_m;
  p.tile_n = f.tile_n;
  p.N = N;
  p.V = p.vp = V;
  p.targets = Ids{targets, targets_64};
  p.part = f.part;
  p.xt = f.xt;
  p.counter = f.counter;
  p.wide = f.wide;
  p.row_scale = f.unit;
  p.status = status;
  if (int rc = f.few ? launch<FEW>(p, st) : launch<STATS>(p, st)) return rc;
  const int lanes = f.lanes();
  return launch_after(lanes == 32 ? join_kernel<32> : join_kernel<4>, dim3(f.join_ctas(N)), kRowThreads, 0, st,
                      Problem{N, V, d, p.targets}, f.few, f.n_tiles, f.m_tiles, f.pairs, f.part, f.xt, loss, lse, reduction,
                      loss, count, rest, f.sums, f.counter, status);
}

extern "C" int cb_linear_ce_grad(const void* h, int32_t h_dtype, int64_t ldh, const void* w, int32_t w_dtype,
                                 int64_t ldw, int32_t N, int32_t V, int32_t d, const void* targets, int32_t targets_64,
                                 int32_t reduction, const float* lse, const int32_t* count, const float* g_loss,
                                 int64_t g_loss_step, const float* g_lse, int64_t g_lse_step, void* dh, void* dw,
                                 void* scratch, size_t scratch_bytes, int32_t* status, void* stream) {
  if (bad(h, h_dtype, ldh, w, w_dtype, ldw, N, V, d, targets, targets_64, reduction) || !lse || !scratch ||
      !aligned_to(scratch, 256) || (reduction != CB_REDUCE_NONE && reduction != CB_REDUCE_SUM && !count) || g_loss_step < 0 || g_lse_step < 0 ||
      (!dh && !dw) || !aligned_to(dh, dtype_size(h_dtype)) || !aligned_to(dw, dtype_size(w_dtype)))
    return CB_ERR_ARG;
  const float* rest = reduction & CB_REDUCE_REST ? reinterpret_cast<const float*>(count + 1) : nullptr;
  reduction &= ~CB_REDUCE_REST;
  if (too_large(N, V, d)) return CB_ERR_SHAPE;
  cudaStream_t st = (cudaStream_t)stream;
  const Shape s(h_dtype, w_dtype, N, V, d);
  Layout a{static_cast<char*>(scratch)};
  const Backward f(a, s, s.reads_w(w, w_dtype, ldw), dh != nullptr, dw != nullptr, tma_rows(dw, w_dtype, d));
  if (scratch_bytes < a.used) return CB_ERR_WORKSPACE;
  const Problem pb{N, V, d, Ids{targets, targets_64}};
  const Upstream u{g_loss, g_lse, g_loss_step, g_lse_step, count, reduction, rest};
  if ((reduction == CB_REDUCE_NONE || g_lse) && cudaMemsetAsync(f.top, 0, sizeof(float), st) != cudaSuccess)
    return CB_ERR_CUDA;
  if (int rc = launch_after(factors_kernel, dim3(ceil_div(N, kRowThreads)), kRowThreads, 0, st, pb, u, lse, f.rows, f.top,
                            f.common, f.wide))
    return rc;
  const Source ws{w, ldw, V, nullptr, f.w};
  const Source hs{h, ldh, N, f.rows, f.h, f.hs != f.h ? f.hs : nullptr, SCALE_ROW, s.tried ? &f.rows->w : nullptr, 4};
  if (int rc = make_operands(h_dtype, w_dtype, s, hs, ws, f.top, f.common, f.wide, st)) return rc;
  const Operand wo(w, ldw, V, f.w, s.w_parts, s);
  const int64_t h_cols = (int64_t)s.h_parts * s.dp;
  const int nt = ceil_div(d, kTileN), m_tiles = ceil_div(N, kTileM);

  Args q{};  // G of a piece
  Gemm& g = q.g[0];
  if (!map_of(&g.a, f.h, s.type, N, h_cols, h_cols, 128) || !map_of(&g.b, wo.at, s.type, V, wo.cols, wo.ld, kTileN / 2))
    return CB_ERR_CUDA;
  s.logit_passes(g, false);
  g.m_tiles = m_tiles;
  g.k_steps = s.dp / kStep;
  q.kind = s.kind();
  q.tile_m = kTileM;
  q.tile_n = kTileN;
  q.N = N;
  q.V = V;
  q.targets = pb.targets;
  q.rows = f.rows;
  q.top = f.top;
  q.g_parts = s.g_parts;
  q.is_f16 = s.f16;
  q.wide = f.wide;
  q.status = status;
  Args r{};  // both products of a piece
  r.kind = q.kind;
  r.is_f16 = s.f16;
  r.wide = f.wide;
  r.common = f.common;
  r.status = status;
  const int64_t slot = up(N, kTileM) * s.da();  // floats of one of dh's
  if (dh && f.h_slots > 1 && cudaMemsetAsync(f.acc + slot, 0, (f.h_slots - 1) * slot * sizeof(float), st) != cudaSuccess)
    return CB_ERR_CUDA;
  for (int v0 = 0; v0 < V; v0 += s.piece) {
    const int vp = std::min(s.piece, V - v0), cols = (int)up(vp, kStep);
    const int64_t g_ld = (int64_t)s.g_parts * cols;
    if (!map_of(&g.out, f.G, s.type, N, g_ld, g_ld, 32)) return CB_ERR_CUDA;
    g.b_base = q.v0 = v0;
    g.n_tiles = ceil_div(vp, kTileN);
    q.vp = vp;
    q.g_cols = cols;
    q.pairs = (int)std::min<int64_t>(s.pairs, (int64_t)m_tiles * g.n_tiles);
    if (int rc = launch<GRAD>(q, st)) return rc;

    const Deal sp = vp == std::min(s.piece, V) ? f.first : deal_of(s, dh != nullptr, dw != nullptr, vp, f.first.w);
    Gemm &gw = r.g[0], &gh = r.g[1];
    gh = gw = Gemm{};
    r.whole = 0;
    std::copy(sp.from, sp.from + s.pairs + 1, r.from);
    if (dh) {
      if (!map_of(&gh.a, f.G, s.type, N, g_ld, g_ld, 128) || !map_of(&gh.b, wo.at, s.type, V, wo.cols, wo.ld, 64) ||
          !map_of(&gh.out, f.acc, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, f.h_slots * up(N, kTileM), s.da(), s.da(), 32))
        return CB_ERR_CUDA;
      s.passes(gh, s.g_parts, s.w_parts, cols, s.dp);
      gh.b_base = v0;
      gh.m_tiles = m_tiles;
      gh.n_tiles = nt;
      gh.k_steps = cols / kStep;
      gh.out_f32 = 1;
      gh.out_mode = v0 ? OUT_ADD : OUT_STORE;
      gh.split_mode = OUT_ADD;
      gh.out_rows = (int)up(N, kTileM);
    }
    if (dw) {
      if (!map_of(&gw.a, f.G, s.type, N, g_ld, g_ld, 64) ||
          !map_of(&gw.b, f.hs, s.type, N, h_cols, h_cols, 64))
        return CB_ERR_CUDA;
      const bool ok =
          f.dw_direct
              ? map_of(&gw.out, static_cast<char*>(dw) + (int64_t)v0 * d * dtype_size(w_dtype),
                       w_dtype == CB_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : s.type, vp, d, d, 32)
              : map_of(&gw.out, f.dw, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, f.first.w * up(std::min(s.piece, V), kTileM), s.da(),
                       s.da(), 32);
      if (!ok) return CB_ERR_CUDA;
      s.dw_passes(gw, cols);
      gw.a_mn = 1;
      gw.m_tiles = ceil_div(vp, kTileM);
      gw.n_tiles = nt;
      gw.k_steps = ceil_div(N, kStep);
      gw.splits = sp.w;
      gw.out_f32 = !f.dw_direct || w_dtype == CB_F32;
      gw.out_rows = (int)up(std::min(s.piece, V), kTileM);
      if (f.dw_direct) gw.top = f.top;
      r.whole = gw.m_tiles * nt * sp.w;
    }
    r.pairs = s.pairs;
    if (int rc = launch<PRODUCTS>(r, st)) return rc;
    if (dw && !f.dw_direct)
      if (int rc = finish(w_dtype, f.dw, sp.w, up(std::min(s.piece, V), kTileM), s, vp, nullptr, f.top, f.common, f.wide,
                          static_cast<char*>(dw) + (int64_t)v0 * d * dtype_size(w_dtype), st))
        return rc;
  }
  if (!dh) return CB_OK;
  return finish(h_dtype, f.acc, f.h_slots, up(N, kTileM), s, N, f.rows, f.top, nullptr, f.wide, dh, st);
}

extern "C" int cb_linear_ce_set_wait_limit(uint64_t limit_ns, int32_t stall_pair) {
  if (stall_pair < 0) return CB_ERR_ARG;
  wait_limit = limit_ns ? limit_ns : kWaitNs;
  stalled_pair = stall_pair - 1;
  return CB_OK;
}
