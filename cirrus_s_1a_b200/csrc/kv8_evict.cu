// cb_kv8_evict: brings every sequence that holds more than `keep` tokens down to
// `keep`, per KV head: the `recent` last slots stay, and of the older ones the
// keep - recent with the largest accumulated attention weight (ties to the
// lowest slot).  The kept tokens move to slots 0 .. keep - 1 in order, in place.
//
// One cluster of CTAs per (sequence, KV head).
//   1. The smallest weight that stays: a radix select over the weights' order
//      keys in three passes of 11, 11 and 10 bits.  Each CTA counts a stretch of
//      the slots; each adds up its share of the bins over all histograms through
//      distributed shared memory, and all read the sums and find the same digit.
//      (Every CTA reading all histograms took 24 us a pass in a cluster of 16.)
//   2. The kept slots in order: each warp counts its stretch, the counts are
//      shared, and a second walk writes the slot numbers.
//   3. The move, in rounds of 32 KB of codes per CTA.  The token for slot j comes
//      from a slot >= j, so what a round writes is read by no later round, and
//      copies run two rounds ahead (cp.async into a ring of three stages); within
//      a round every CTA has read before any writes, which takes one cluster
//      barrier, arrived at when the round's copies have landed.
// A new block takes the scale its values need; a code is rounded again only
// where its scale grows, and copied as it is where the scale stays.
// Bound by memory in principle (the weights once, each kept token read and written),
// in fact by issue (52 % of the slots, 50 % of the integer pipe) and the rounds'
// barriers.  Measured: 32 sequences of up to 64K down to 32K, 2 heads of 128 dims,
// E4M3: 292 us = 2.5 TB/s (uniform lengths: 314 us = 3.6 TB/s); one sequence of 16.5K
// down to 16K, 4 heads of 64: 33 us, the selection's dependent passes and the rounds' latency.
#include <cooperative_groups.h>

#include "kv8.cuh"
#include "kv8_attend.cuh"

namespace cb {
namespace {

namespace cg = cooperative_groups;

constexpr int kET = 512;
constexpr int kEWarps = kET / 32;
constexpr int kBins = 2048;
constexpr int kPieces = 4;  // 16-byte pieces of one thread in a round
constexpr int kMaxCluster = 16;
constexpr int kStages = 3;
constexpr int kSrcRing = 4;

struct EvictParams {
  CbKv8 c;
  const int32_t* pos;
  int keep, recent;
  int32_t* kept;
  int32_t* new_pos;
};

// Order key of a weight: larger weight, larger key; NaN below everything.
__device__ __forceinline__ uint32_t weight_key(float w) { return w != w ? 0u : score_key(w); }

// Sum over the threads after this one (higher tid) of v; needs 32 ints of scratch.
__device__ __forceinline__ int sum_after(int v, int* red) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_down_sync(0xffffffffu, x, o);
    if (lane + o < 32) x += y;
  }
  __syncthreads();
  if (lane == 0) red[w] = x;
  __syncthreads();
  int after = x - v;
  for (int i = w + 1; i < kEWarps; ++i) after += red[i];
  return after;
}

// Largest magnitude of 16 codes (as f16 pairs); a NaN does not count.
__device__ __forceinline__ float piece_max(const uint32_t (&h)[8]) {
  __half2 a = __habs2(bits_h2(h[0]));
#pragma unroll
  for (int i = 1; i < 8; ++i) a = __hmax2(a, __habs2(bits_h2(h[i])));
  const float m = __half2float(__hmax(__low2half(a), __high2half(a)));
  return m == m ? m : 0.0f;
}

// Shared memory of the move: the ring of codes, then of each token's two scales
// and mass, then of source slots.  The selection's histograms lie under it.
template <int D>
struct Move {
  static constexpr int kRow = D / 16;                        // 16-byte pieces of a token
  static constexpr int kUnit = kKv8Block * kRow;             // of a block of K or V
  static constexpr int kUnits = kPieces * kET / kUnit;       // per round, K and V of a block in turn
  static constexpr int kBlocks = kUnits / 2;
  static constexpr int kTokens = kBlocks * kKv8Block;
  static constexpr int kCodes = kPieces * kET * 16;          // bytes of a stage
  static constexpr int kBytes = kStages * (kCodes + 3 * kTokens * 4) + kSrcRing * kTokens * 4;
  static_assert(kBytes >= 4 * kBins * 4, "the histograms lie under the ring");
};

__device__ __forceinline__ void cp16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
               : "memory");
}
__device__ __forceinline__ void cp4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
               : "memory");
}

template <int D, int FMT>
__global__ void __launch_bounds__(kET, 2) kv8_evict_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  int(*hist)[kBins] = reinterpret_cast<int(*)[kBins]>(smem);  // [3]
  int* total = reinterpret_cast<int*>(smem) + 3 * kBins;      // this CTA's share of the bins, all CTAs
  __shared__ int red[kEWarps];
  __shared__ uint32_t s_digit;
  __shared__ int s_rest;
  __shared__ int s_stay[kEWarps], s_tie[kEWarps];
  __shared__ int s_count[2];
  cg::cluster_group cl = cg::this_cluster();
  const int nc = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t head = blockIdx.x / nc;
  const int b = (int)(head / p.c.n_kv_heads);
  const int n = min(max(p.pos[b], 0), p.c.max_len), keep = p.keep;
  int32_t* kept = p.kept + head * keep;
  if (head % p.c.n_kv_heads == 0 && rank == 0 && tid == 0) p.new_pos[b] = min(n, keep);
  if (n <= keep) {  // the whole cluster takes this way
    for (int j = rank * kET + tid; j < keep; j += nc * kET) kept[j] = j < n ? j : -1;
    return;
  }
  float* mass = p.c.mass + head * p.c.max_len;
  const int old = n - p.recent;      // candidates: slots below this
  const int want = keep - p.recent;  // how many of them stay, < old
  // this CTA's stretch of the slots, whole warps' worth of 32 each
  const int seg = ceil_div(ceil_div(n, nc), kET) * 32, chunk = seg * kEWarps;
  const int beg = min(n, rank * chunk), end = min(n, beg + chunk);

  // 1. the want-th largest key, and how many of its equals stay
  for (int i = tid; i < 3 * kBins; i += kET) (&hist[0][0])[i] = 0;
  uint32_t key = 0, mask = 0;
  int rest = want;
  __syncthreads();
  if (want > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      int* h = hist[pass];
      for (int j = beg + tid; j < min(end, old); j += kET) {
        const uint32_t u = weight_key(mass[j]);
        if ((u & mask) == key) atomicAdd(&h[(u >> shift) & ((1 << bits) - 1)], 1);
      }
      cl.sync();  // the histograms are complete, and the last pass's totals read
      const int share = kBins / nc;
      for (int i = tid; i < share; i += kET) total[i] = 0;
      __syncthreads();
#pragma unroll
      for (int i = tid; i < kBins; i += kET)
        atomicAdd(&total[i % share], cl.map_shared_rank(h, i / share)[rank * share + i % share]);
      cl.sync();
      // bins 4 tid .. + 3
      const int4 c4 = *reinterpret_cast<const int4*>(cl.map_shared_rank(total, 4 * tid / share) + 4 * tid % share);
      const int c[kBins / kET] = {c4.x, c4.y, c4.z, c4.w};
      int mine = 0;
#pragma unroll
      for (int i = 0; i < kBins / kET; ++i) mine += c[i];
      int after = sum_after(mine, red);
      if (after < rest && after + mine >= rest) {
        int i = kBins / kET - 1;
        while (after + c[i] < rest) after += c[i--];
        s_digit = (uint32_t)(tid * (kBins / kET) + i);
        s_rest = rest - after;
      }
      __syncthreads();
      key |= s_digit << shift;
      mask |= ((1u << bits) - 1u) << shift;
      rest = s_rest;
      __syncthreads();
    }
  }

  // 2. the kept slots in order
  const int w0 = beg + warp * seg, w1 = min(end, w0 + seg);
  constexpr int kAhead = 8;  // loads of a warp in flight
  auto weights = [&](int j0, uint32_t (&u)[kAhead]) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int j = j0 + 32 * i + lane;
      u[i] = j < min(w1, old) ? weight_key(mass[j]) : 0u;
    }
  };
  auto stays = [&](int j, uint32_t u) { return j < w1 && (j >= old || (want > 0 && u > key)); };
  auto ties_in = [&](int j, uint32_t u) { return j < min(w1, old) && want > 0 && u == key; };
  int stay = 0, tie = 0;
  for (int j0 = w0; j0 < w1; j0 += 32 * kAhead) {
    uint32_t u[kAhead];
    weights(j0, u);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int j = j0 + 32 * i + lane;
      stay += __popc(__ballot_sync(0xffffffffu, stays(j, u[i])));
      tie += __popc(__ballot_sync(0xffffffffu, ties_in(j, u[i])));
    }
  }
  if (lane == 0) {
    s_stay[warp] = stay;
    s_tie[warp] = tie;
  }
  __syncthreads();
  int base = 0, ties = 0;  // of the warps before this one
  for (int w = 0; w < kEWarps; ++w) {
    if (tid == 0) {
      if (w == 0) s_count[0] = s_count[1] = 0;
      s_count[0] += s_stay[w];
      s_count[1] += s_tie[w];
    }
    base += w < warp ? s_stay[w] : 0;
    ties += w < warp ? s_tie[w] : 0;
  }
  cl.sync();
  for (int r = 0; r < rank; ++r) {
    const int* o = cl.map_shared_rank(s_count, r);
    base += o[0];
    ties += o[1];
  }
  for (int j0 = w0; j0 < w1; j0 += 32 * kAhead) {
    uint32_t u[kAhead];
    weights(j0, u);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int j = j0 + 32 * i + lane;
      const bool st = stays(j, u[i]), ti = ties_in(j, u[i]);
      const unsigned sb = __ballot_sync(0xffffffffu, st), tb = __ballot_sync(0xffffffffu, ti);
      const unsigned before = (1u << lane) - 1u;
      const int t = ties + __popc(tb & before);
      if (st || (ti && t < rest)) kept[base + __popc(sb & before) + min(rest, t)] = j;
      base += __popc(sb);
      ties += __popc(tb);
    }
  }
  cl.sync();  // every CTA's slot numbers are visible to the cluster

  // 3. the move.  Piece i of a round: 16 bytes of one token, in unit i / kUnit.
  using M = Move<D>;
  __shared__ unsigned s_max[2][M::kUnits];
  float* s_float = reinterpret_cast<float*>(smem + kStages * M::kCodes);                  // [stage][3][tokens]
  int* s_src = reinterpret_cast<int*>(s_float + kStages * 3 * M::kTokens);                // [ring][tokens]
  const int64_t nb = p.c.max_len / kKv8Block;
  auto codes = [&](int kv) { return (kv ? p.c.v : p.c.k) + head * p.c.max_len * D; };
  auto scales = [&](int kv) { return (kv ? p.c.v_scale : p.c.k_scale) + head * nb; };
  const int rounds = ceil_div(ceil_div(keep, kKv8Block), M::kBlocks * nc);
  if (tid < 2 * M::kUnits) (&s_max[0][0])[tid] = 0u;
  // destination slot of token t of this CTA in a round, -1: none
  auto dest = [&](int round, int t) {
    const int j = (round * nc + rank) * M::kTokens + t;
    return round < rounds && j < keep ? j : -1;
  };
  auto copy_src = [&](int round) {
    for (int t = tid; t < M::kTokens; t += kET)
      if (const int j = dest(round, t); j >= 0) cp4(s_src + round % kSrcRing * M::kTokens + t, kept + j);
  };
  auto copy_codes = [&](int round) {
    const int* src = s_src + round % kSrcRing * M::kTokens;
    float* f = s_float + round % kStages * 3 * M::kTokens;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int piece = tid + i * kET, unit = piece / M::kUnit, in = piece % M::kUnit;
      const int t = unit / 2 * kKv8Block + in / M::kRow;
      if (dest(round, t) >= 0)
        cp16(smem + round % kStages * M::kCodes + piece * 16,
             codes(unit & 1) + (int64_t)src[t] * D + in % M::kRow * 16);
    }
    for (int t = tid; t < M::kTokens; t += kET)
      if (dest(round, t) >= 0) {
        cp4(f + t, scales(0) + src[t] / kKv8Block);
        cp4(f + M::kTokens + t, scales(1) + src[t] / kKv8Block);
        cp4(f + 2 * M::kTokens + t, mass + src[t]);
      }
  };
  auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
  for (int r = 0; r < kSrcRing; ++r) copy_src(r);
  commit();
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  copy_codes(0);
  commit();
  copy_codes(1);
  commit();
  for (int round = 0; round < rounds; ++round) {
    // all but the newest group: this round's codes, and the sources of round + 2
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncthreads();
    cl.barrier_arrive();  // this CTA has read what this round's writes may lie over
    copy_codes(round + 2);
    copy_src(round + kSrcRing);
    commit();
    unsigned* top = s_max[round & 1];
    const uint8_t* stage = smem + round % kStages * M::kCodes;
    const float* f = s_float + round % kStages * 3 * M::kTokens;
    uint32_t h[kPieces][8];  // the codes' values, exact in f16
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int piece = tid + i * kET, unit = piece / M::kUnit, t = unit / 2 * kKv8Block + piece % M::kUnit / M::kRow;
      const uint4 c = *reinterpret_cast<const uint4*>(stage + piece * 16);
      codes_to_h2<FMT>(c.x, h[i][0], h[i][1]);
      codes_to_h2<FMT>(c.y, h[i][2], h[i][3]);
      codes_to_h2<FMT>(c.z, h[i][4], h[i][5]);
      codes_to_h2<FMT>(c.w, h[i][6], h[i][7]);
      const float a = dest(round, t) >= 0 ? piece_max(h[i]) * f[(unit & 1) * M::kTokens + t] : 0.0f;
      const unsigned m = __reduce_max_sync(0xffffffffu, __float_as_uint(a));
      if (lane == 0) atomicMax(&top[unit], m);
    }
    __syncthreads();
    if (tid < M::kUnits) s_max[(round + 1) & 1][tid] = 0u;  // read last before this round's first barrier
    cl.barrier_wait();
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int piece = tid + i * kET, unit = piece / M::kUnit, in = piece % M::kUnit;
      const int t = unit / 2 * kKv8Block + in / M::kRow, j = dest(round, t);
      if (j < 0) continue;
      const float was = f[(unit & 1) * M::kTokens + t];
      const int e = kv8_need<FMT>(__uint_as_float(top[unit]));
      const float now = kv8_pow2(e);
      uint4 o;
      if (was == now) {
        o = *reinterpret_cast<const uint4*>(stage + piece * 16);
      } else {
        // E4M3 codes may grow by up to 2^17: two factors of at most 2^15.  Only
        // codes of 0 see a larger one cut off.
        const float by = was * kv8_pow2(-e), by1 = fminf(by, 32768.0f);
        const __half2 f1 = __float2half2_rn(by1);
        if (FMT == CB_KV8_E4M3 && by > by1) {
          const __half2 f2 = __float2half2_rn(fminf(by * (1.0f / 32768.0f), 32768.0f));
#pragma unroll
          for (int k = 0; k < 8; ++k) h[i][k] = h2_bits(__hmul2(bits_h2(h[i][k]), f2));
        }
        o = make_uint4(h2_to_codes<FMT>(h[i][0], h[i][1], f1), h2_to_codes<FMT>(h[i][2], h[i][3], f1),
                       h2_to_codes<FMT>(h[i][4], h[i][5], f1), h2_to_codes<FMT>(h[i][6], h[i][7], f1));
      }
      *reinterpret_cast<uint4*>(codes(unit & 1) + (int64_t)j * D + in % M::kRow * 16) = o;
      if (in == 0) scales(unit & 1)[j / kKv8Block] = now;
    }
    for (int t = tid; t < M::kTokens; t += kET)
      if (const int j = dest(round, t); j >= 0) mass[j] = f[2 * M::kTokens + t];
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <int D, int FMT>
int launch_df(const EvictParams& p, cudaStream_t st) {
  // the largest cluster that leaves all of them resident at two CTAs per SM:
  // few heads get many CTAs each, many heads get few
  const int heads = p.c.batch * p.c.n_kv_heads;
  auto fn = kv8_evict_kernel<D, FMT>;
  if (const int rc = ensure_smem_attr((const void*)fn, Move<D>::kBytes)) return rc;
  int nc = kMaxCluster;
  while (nc > 1 && heads * nc > 2 * num_sms()) nc >>= 1;
  if (nc == kMaxCluster &&
      cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
    (void)cudaGetLastError();
    nc = 8;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(heads * nc);
  cfg.blockDim = dim3(kET);
  cfg.dynamicSmemBytes = Move<D>::kBytes;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = nc;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, fn, p);
  count_launch();
  return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? CB_OK : CB_ERR_CUDA;
}

template <int D>
int launch(const EvictParams& p, cudaStream_t st) {
  return p.c.format == CB_KV8_E4M3 ? launch_df<D, CB_KV8_E4M3>(p, st) : launch_df<D, CB_KV8_INT8>(p, st);
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
    case 16: return launch<16>(p, st);
    case 32: return launch<32>(p, st);
    case 64: return launch<64>(p, st);
    default: return launch<128>(p, st);
  }
}
