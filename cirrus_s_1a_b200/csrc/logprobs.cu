// cb_token_logprobs: for each row x of logits, with m = max x, l = sum exp(x - m):
//   logprob = x[token] - m - log l
//   entropy = log l - (1/l) sum (x - m) exp(x - m)
//   rank    = how many logits are larger than x[token]
//   the `top` largest logits in order (ties to the lowest token), as log probabilities
//
// One CTA per row, one pass over it.  Each thread keeps its own running maximum
// m, l and t = sum (x - m) exp(x - m); a larger maximum m' rescales them,
//   d = m - m':  t <- (t + d l) e^d,  l <- l e^d,
// so a batch of loaded values costs a branch, not a rescale per value.  The
// exponentials are in powers of two; -infinity is kept out of 0 * infinity by a
// floor of -200 under the exponent, where exp2 is 0 in float32 already.
//
// Alternatives need no second pass: the threads' maxima are folded to 64 groups,
// and the top-th largest of the 64 is a threshold with at least `top` values at
// or above it.  Only threads whose maximum passes it (about as many as there are
// alternatives) have their values read again, from L2; the values that pass
// (about 24 for top = 20) are ranked by counting.  Where more than kCand pass
// (ties, rows where a mask leaves less than `top` tokens), the ones above the
// threshold are ranked and equal ones follow in token order; where more than
// kCand are above it (values packed into few threads), it is one search per
// alternative.
//
// Bound by memory in principle (the row once), by issue in fact (77 % of the slots;
// the pass widens, compares, scales, exponentiates and adds each value).  Measured: 16384 rows of 32000 in bf16,
// 20 alternatives: 250 to 273 us = 4 TB/s (nine tenths masked by -1e9: 312); without
// alternatives 200 us = 5.2 TB/s; five rows in float32: 17 us, the host's part of the call.
// Rows with more than kCand equal negative values at the threshold (a finite mask that
// leaves less than `top` tokens) take the one search per alternative, 0.5 us a row.
#include "common.cuh"
#include "kv8.cuh"

namespace cb {
namespace {

constexpr int kGroups = 64;
constexpr int kCand = 512;
constexpr int kBatch = 4;  // 16-byte vectors in flight per thread
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
static_assert(CB_LOGPROB_MAX_TOP <= kGroups, "the threshold needs a group per alternative");
static_assert(8 * kBatch + 8 * kBatch <= 256, "counts between two takes are exact in bf16");

struct LogprobParams {
  const void* x;
  int64_t ld;
  int V, top;
  const int32_t* tokens;
  float* logprob;
  float* entropy;
  int32_t* rank;
  float* top_logprob;
  int32_t* top_token;
  int32_t* status;
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

// (value, token) as one key: larger value first, then the lower token.
__device__ __forceinline__ unsigned long long top_key(float v, int i) {
  return ((unsigned long long)score_key(v) << 32) | (uint32_t)~i;
}

// Running maximum m of one thread, and relative to a reference c near m * log2(e) the
// sums l = sum 2^(x log2(e) - c) and t = sum of exponent * 2^exponent, each in two
// halves.  Up to kFar, c is m * log2(e) rounded and every term is taken against the
// rounded value by one fused operation, so what the rounding leaves (up to half an ulp of
// c, 2^-4 there) is a factor common to all of them and cancels.  Beyond, that factor would
// leave the range of float32, and values 150 below m are no longer told from m: c is
// m * log2(e) itself and the exponents are (x - m) log2(e).
constexpr float kFar = 1048576.0f, kFloor = -200.0f;
constexpr float kHuge = 2e38f;  // from here on x * log2(e) overflows
__device__ __forceinline__ bool is_far(float m) { return fabsf(m) > kFar; }
struct Stat {
  float m = -INFINITY;
  f32x2 l = 0, t = 0;  // two zeros each
  __device__ __forceinline__ bool far() const { return is_far(m); }
  __device__ __forceinline__ float c() const { return __fmul_rn(m, kLog2e); }
  __device__ __forceinline__ void raise(float top) {
    if (top > m) {
      if (m > -INFINITY) {
        // from one reference to the other, whichever kind each is
        const float to = __fmul_rn(top, kLog2e);
        const float by = is_far(top) ? (far() ? (m - top) * kLog2e : -fmaf(top, kLog2e, -c()))
                                     : (far() ? fmaf(m, kLog2e, -to) : c() - to);
        const float d = fmaxf(by, kFloor), f = exp2a(d);
        t = mul2(fma2(pack2(d, d), l, t), pack2(f, f));
        l = mul2(l, pack2(f, f));
      }
      m = top;
    }
  }
  // any value, m already at least as large
  __device__ __forceinline__ void add(float x) {
    if (m > -INFINITY) {
      const float d = max_nan(far() ? (x - m) * kLog2e : fmaf(x, kLog2e, -c()), kFloor), e = exp2a(d);
      l = add2(l, pack2(e, 0.0f));
      t = add2(t, pack2(d * e, 0.0f));
    } else if (x != x) {  // nothing finite yet: only a NaN counts
      l = pack2(NAN, 0.0f);
    }
  }
};

template <typename T>
struct Vec;  // 16 bytes of a row
template <>
struct Vec<float> {
  static constexpr int N = 4;
  float4 v;
  struct Count {
    int n = 0;
    __device__ __forceinline__ int take() {
      const int r = n;
      n = 0;
      return r;
    }
  };
  __device__ __forceinline__ float get(int i) const { return (&v.x)[i]; }
  __device__ __forceinline__ float max() const { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); }
  // values below the floor, whose exponentials are 0, are raised to it
  using Floor = float;
  static __device__ __forceinline__ Floor floor_of(float m) { return m - 150.0f; }
  static __device__ __forceinline__ bool usable(Floor f) { return f > -INFINITY; }
  __device__ __forceinline__ void lift(Floor f) {
#pragma unroll
    for (int i = 0; i < N; ++i) (&v.x)[i] = max_nan((&v.x)[i], f);
  }
  __device__ __forceinline__ void above(float xt, Count& c) const {
    c.n += (v.x > xt) + (v.y > xt) + (v.z > xt) + (v.w > xt);
  }
};
// Two 16-bit types: pairs are compared and raised to a floor before they are widened.
template <typename T2>
struct Vec16 {
  static constexpr int N = 8;
  uint4 v;
  struct Count {  // a batch of kBatch vectors counts to 4 kBatch per half: exact in either type
    T2 n;
    __device__ __forceinline__ Count() { *reinterpret_cast<uint32_t*>(&n) = 0u; }
    __device__ __forceinline__ int take() {
      const int r = (int)(__low2float(n) + __high2float(n));
      *reinterpret_cast<uint32_t*>(&n) = 0u;
      return r;
    }
  };
  __device__ __forceinline__ T2 pair(int i) const { return reinterpret_cast<const T2*>(&v)[i]; }
  __device__ __forceinline__ float get(int i) const { return i & 1 ? __high2float(pair(i >> 1)) : __low2float(pair(i >> 1)); }
  __device__ __forceinline__ float max() const {
    const T2 a = __hmax2(__hmax2(pair(0), pair(1)), __hmax2(pair(2), pair(3)));
    return fmaxf(__low2float(a), __high2float(a));
  }
  using Floor = T2;
  static __device__ __forceinline__ bool usable(Floor f) { return __low2float(f) > -INFINITY; }
  __device__ __forceinline__ void lift(Floor f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<T2*>(&v)[i] = __hmax2_nan(pair(i), f);
  }
  __device__ __forceinline__ void above2(T2 xt, Count& c) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) c.n = __hadd2(c.n, __hgt2(pair(i), xt));
  }
};
template <>
struct Vec<__nv_bfloat16> : Vec16<__nv_bfloat162> {
  // rounded down: at most m - 150
  static __device__ __forceinline__ Floor floor_of(float m) { return __bfloat162bfloat162(__float2bfloat16_rd(m - 150.0f)); }
  __device__ __forceinline__ void above(float xt, Count& c) const { above2(__float2bfloat162_rn(xt), c); }
};
template <>
struct Vec<__half> : Vec16<__half2> {
  static __device__ __forceinline__ Floor floor_of(float m) { return __half2half2(__float2half_rd(m - 150.0f)); }
  __device__ __forceinline__ void above(float xt, Count& c) const { above2(__float2half2_rn(xt), c); }
};

// COUNT vectors into a thread's sums.
template <typename T, int COUNT>
__device__ __forceinline__ void add_vecs(Vec<T> (&v)[COUNT], Stat& s, typename Vec<T>::Floor& floor) {
  constexpr int N = Vec<T>::N;
  float top = v[0].max();
#pragma unroll
  for (int u = 1; u < COUNT; ++u) top = fmaxf(top, v[u].max());
  if (top > s.m) {
    s.raise(top);
    floor = Vec<T>::floor_of(s.m);
  }
  if (!s.far() && Vec<T>::usable(floor)) {
    const f32x2 L = pack2(kLog2e, kLog2e), c = pack2(-s.c(), -s.c());
#pragma unroll
    for (int u = 0; u < COUNT; ++u) {
      v[u].lift(floor);
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const f32x2 d = fma2(pack2(v[u].get(i), v[u].get(i + 1)), L, c);
        const float2 dd = unpack2(d);
        const f32x2 e = pack2(exp2a(dd.x), exp2a(dd.y));
        s.l = add2(s.l, e);
        s.t = fma2(d, e, s.t);
      }
    }
  } else {  // nothing finite yet, far from zero, or a floor past the type's range
#pragma unroll
    for (int u = 0; u < COUNT; ++u)
#pragma unroll
      for (int i = 0; i < N; ++i) s.add(v[u].get(i));
  }
}

template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* p) {
  Vec<T> r;
  r.v = __ldg(reinterpret_cast<const decltype(r.v)*>(p));
  return r;
}

__device__ __forceinline__ float warp_max_f32(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT) token_logprobs_kernel(const __grid_constant__ LogprobParams p) {
  constexpr int N = Vec<T>::N, kWarps = NT / 32;
  __shared__ float s_m[kWarps], s_l[kWarps], s_t[kWarps];
  __shared__ int s_above[kWarps];
  __shared__ __align__(16) uint32_t s_group[kGroups];
  __shared__ float s_tau;
  __shared__ int s_threads, s_cands;
  __shared__ int s_thread[NT];
  __shared__ unsigned long long s_cand[kCand];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r = blockIdx.x;
  const T* row = static_cast<const T*>(p.x) + r * p.ld;
  int tok = p.tokens[r];
  if (tok >= p.V) {
    if (tid == 0) set_status(p.status, CB_ERR_TOKEN);
    tok = -1;
  }
  const float xt = tok >= 0 ? to_f(row[tok]) : INFINITY;

  // the row: `head` values up to the first 16-byte boundary, vectors, a tail
  const int head = min(p.V, (int)(((16 - ((uintptr_t)row & 15)) & 15) / sizeof(T)));
  const int vecs = (p.V - head) / N, edge = p.V - vecs * N;  // edge: head and tail together, < 2 N
  const T* body = row + head;
  Stat s;
  int above = 0;
  typename Vec<T>::Count count;
  typename Vec<T>::Floor floor = Vec<T>::floor_of(-INFINITY);
  int j = tid;
  const T* at = body + (int64_t)tid * N;
  for (; j + (kBatch - 1) * NT < vecs; j += kBatch * NT, at += kBatch * NT * N) {
    Vec<T> v[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) v[u] = load_vec(at + u * NT * N);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) v[u].above(xt, count);
    above += count.take();
    add_vecs<T, kBatch>(v, s, floor);
  }
  for (; j < vecs; j += NT, at += NT * N) {
    Vec<T> v[1] = {load_vec(at)};
    v[0].above(xt, count);
    add_vecs<T, 1>(v, s, floor);
  }
  above += count.take();
  // the edge goes to the last threads
  const int mine = NT - 1 - tid;
  const int edge_at = mine < edge ? (mine < head ? mine : p.V - edge + mine) : -1;
  float edge_x = -INFINITY;
  if (edge_at >= 0) {
    edge_x = to_f(row[edge_at]);
    s.raise(edge_x);
    above += edge_x > xt;
    s.add(edge_x);
  }

  // join the threads
  const float mine_max = s.m;
  const float wm = warp_max_f32(s.m);
  if (lane == 0) s_m[warp] = wm;
  if (tid == 0) s_threads = s_cands = 0;
  if (p.top) {
    float gm = s.m;
#pragma unroll
    for (int o = 1; o < NT / kGroups; o <<= 1) gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, o));
    const int g = tid / (NT / kGroups);
    if (tid % (NT / kGroups) == 0) s_group[g] = (score_key(gm) & ~(kGroups - 1)) | (kGroups - 1 - g);
  }
  __syncthreads();
  float m = s_m[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) m = fmaxf(m, s_m[w]);
  s.raise(m);
  const float2 l2 = unpack2(s.l), t2 = unpack2(s.t);
  const float wl = warp_sum(l2.x + l2.y), wt = warp_sum(t2.x + t2.y);
  const int wa = __reduce_add_sync(0xffffffffu, above);
  if (lane == 0) {
    s_l[warp] = wl;
    s_t[warp] = wt;
    s_above[warp] = wa;
  }
  if (p.top && tid < kGroups) {
    // the top-th largest group maximum, rounded down where the group number tells equal ones apart
    const uint32_t me = s_group[tid];
    int ahead = 0;
#pragma unroll
    for (int g = 0; g < kGroups; g += 4) {
      const uint4 o = *reinterpret_cast<const uint4*>(s_group + g);
      ahead += (o.x > me) + (o.y > me) + (o.z > me) + (o.w > me);
    }
    if (ahead == p.top - 1) {
      const uint32_t u = me & ~(kGroups - 1);
      const float v = __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
      s_tau = v == v ? v : -INFINITY;
    }
  }
  __syncthreads();
  float l = 0.0f, t = 0.0f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    l += s_l[w];
    t += s_t[w];
  }
  const float log2l = log2f(l);
  s.m = m;
  const float c0 = s.c();
  const bool far = s.far();
  auto logp = [&](float x) {
    return far || fabsf(x) > kHuge ? (x - m) - log2l * kLn2 : (fmaf(x, kLog2e, -c0) - log2l) * kLn2;
  };
  if (tid == 0) {
    int n = 0;
    for (int w = 0; w < kWarps; ++w) n += s_above[w];
    p.logprob[r] = tok >= 0 ? logp(xt) : 0.0f;
    p.entropy[r] = (log2l - t / l) * kLn2;
    p.rank[r] = tok >= 0 ? n : -1;
  }
  if (!p.top) return;

  // Values at or above the threshold, from the threads that hold any.  Where too
  // many are equal to it, the ones above it alone, and equal ones in token order
  // afterwards.
  const float tau = s_tau;
  float* out_lp = p.top_logprob + r * p.top;
  int32_t* out_tok = p.top_token + r * p.top;
  const int per = (vecs + NT - 1) / NT, per_log2 = per > 1 ? 32 - __clz(per - 1) : 0;
  bool strict = tau == -INFINITY;
  int cands;
  while (true) {
    // v >= tau as v > the float below it: one comparison either way
    const float under = strict ? tau : nextafterf(tau, -INFINITY);
    auto passes = [&](float v) { return v > under; };
    auto take = [&](float v, int i) {
      const int at = atomicAdd(&s_cands, 1);
      if (at < kCand) s_cand[at] = top_key(v, i);
    };
    if (passes(mine_max)) s_thread[atomicAdd(&s_threads, 1)] = tid;
    if (edge_at >= 0 && passes(edge_x)) take(edge_x, edge_at);
    __syncthreads();
    // (thread, vector) pairs over all threads, two reads ahead
    const int jobs = s_threads << per_log2;
    for (int job = tid; job < jobs; job += 2 * NT) {
      int at[2];
      Vec<T> v[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int jb = job + u * NT;
        at[u] = jb < jobs ? s_thread[jb >> per_log2] + (jb & ((1 << per_log2) - 1)) * NT : vecs;
        if (at[u] < vecs) v[u] = load_vec(body + (int64_t)at[u] * N);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (at[u] >= vecs) continue;
        unsigned which = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) which |= passes(v[u].get(i)) ? 1u << i : 0u;
        for (; which && s_cands <= kCand; which &= which - 1) {
          const int i = head + at[u] * N + __ffs(which) - 1;
          take(to_f(row[i]), i);
        }
      }
    }
    __syncthreads();
    cands = s_cands;
    if (cands <= kCand || strict) break;
    strict = true;
    __syncthreads();
    if (tid == 0) s_threads = s_cands = 0;
    __syncthreads();
  }
  int filled = min(cands, p.top);
  if (cands <= kCand) {
    for (int c = tid; c < cands; c += NT) {
      const unsigned long long me = s_cand[c];
      int ahead = 0;
      for (int o = 0; o < cands; ++o) ahead += s_cand[o] > me;
      if (ahead < p.top) {
        const int i = (int)~(uint32_t)me;
        out_tok[ahead] = i;
        out_lp[ahead] = logp(to_f(row[i]));
      }
    }
  } else {
    unsigned long long below = ~0ull;
    for (int k = 0; k < p.top; ++k) {
      unsigned long long best = 0;
      for (int i = tid; i < p.V; i += NT) {
        const float v = to_f(row[i]);
        const unsigned long long u = v == v ? top_key(v, i) : 0;
        if (u < below && u > best) best = u;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long u = __shfl_xor_sync(0xffffffffu, best, o);
        best = u > best ? u : best;
      }
      __syncthreads();
      if (lane == 0) s_cand[warp] = best;
      __syncthreads();
      for (int w = 0; w < kWarps; ++w) best = s_cand[w] > best ? s_cand[w] : best;
      below = best;
      if (tid == 0) {
        const int i = (int)~(uint32_t)best;
        out_tok[k] = i;
        out_lp[k] = logp(to_f(row[i]));
      }
    }
  }
  for (int i0 = 0; strict && filled < p.top && i0 < p.V; i0 += NT) {
    const int i = i0 + tid;
    const bool is = i < p.V && to_f(row[i]) == tau;
    const unsigned ballot = __ballot_sync(0xffffffffu, is);
    __syncthreads();
    if (lane == 0) s_above[warp] = __popc(ballot);
    __syncthreads();
    int at = filled + __popc(ballot & ((1u << lane) - 1u));
    int n = 0;
    for (int w = 0; w < kWarps; ++w) {
      at += w < warp ? s_above[w] : 0;
      n += s_above[w];
    }
    if (is && at < p.top) {
      out_tok[at] = i;
      out_lp[at] = logp(tau);
    }
    filled = min(p.top, filled + n);
  }
  // a row of NaN may have less than `top` values that can be ranked
  for (int k = filled + tid; k < p.top; k += NT) {
    out_tok[k] = -1;
    out_lp[k] = NAN;
  }
}

template <typename T>
void launch(const LogprobParams& p, int rows, cudaStream_t st) {
  // 256 threads a row leave six rows to an SM, whose reads and reductions
  // overlap, and the rows in flight to L2 for the second look (with 128 threads
  // they passed it: 1.41 instead of 1.05 GB read); with at most a row per SM,
  // 1024 threads hold a row's reads in flight
  if (rows > num_sms()) token_logprobs_kernel<T, 256><<<rows, 256, 0, st>>>(p);
  else token_logprobs_kernel<T, 1024><<<rows, 1024, 0, st>>>(p);
}

}  // namespace
}  // namespace cb

using namespace cb;

extern "C" int cb_token_logprobs(const void* logits, int32_t dtype, int64_t ld, int32_t rows, int32_t V,
                                 const int32_t* tokens, int32_t top, float* logprob, float* entropy, int32_t* rank,
                                 float* top_logprob, int32_t* top_token, int32_t* status, void* stream) {
  if (!logits || !tokens || !logprob || !entropy || !rank || rows <= 0 || V <= 0 || (ld < V && ld != 0)) return CB_ERR_ARG;
  if (dtype != CB_F32 && dtype != CB_BF16 && dtype != CB_F16) return CB_ERR_ARG;
  if (top < 0 || top > V || (top > 0 && (!top_logprob || !top_token))) return CB_ERR_ARG;
  if (top > CB_LOGPROB_MAX_TOP || V > CB_LOGPROB_MAX_VOCAB) return CB_ERR_SHAPE;
  if ((uintptr_t)logits % (dtype == CB_F32 ? 4 : 2)) return CB_ERR_ARG;
  const LogprobParams p{logits, ld, V, top, tokens, logprob, entropy, rank, top_logprob, top_token, status};
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == CB_F32) launch<float>(p, rows, st);
  else if (dtype == CB_BF16) launch<__nv_bfloat16>(p, rows, st);
  else launch<__half>(p, rows, st);
  count_launch();
  return cudaGetLastError() == cudaSuccess ? CB_OK : CB_ERR_CUDA;
}
