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

__device__ __forceinline__ float exp2a(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The larger of two; NaN if either is one.
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// Running maximum, sum and entropy sum of one thread (t and the exponents in powers of two).
struct Stat {
  float m = -INFINITY, l = 0.0f, t = 0.0f;
  __device__ __forceinline__ void raise(float top) {
    if (top > m) {
      if (m > -INFINITY) {
        const float d = fmaxf((m - top) * kLog2e, -200.0f), f = exp2a(d);
        t = fmaf(d, l, t) * f;
        l *= f;
      }
      m = top;
    }
  }
  __device__ __forceinline__ void add(float x) {
    const float d = max_nan((x - m) * kLog2e, -200.0f), e = exp2a(d);
    l += e;
    t = fmaf(d, e, t);
  }
};

template <typename T>
struct Vec;  // 16 bytes of a row
template <>
struct Vec<float> {
  static constexpr int N = 4;
  float4 v;
  __device__ __forceinline__ float get(int i) const { return (&v.x)[i]; }
  __device__ __forceinline__ float max() const { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); }
  __device__ __forceinline__ int above(float xt) const { return (v.x > xt) + (v.y > xt) + (v.z > xt) + (v.w > xt); }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  uint4 v;
  __device__ __forceinline__ __nv_bfloat162 pair(int i) const { return reinterpret_cast<const __nv_bfloat162*>(&v)[i]; }
  __device__ __forceinline__ float get(int i) const {
    const uint32_t w = (&v.x)[i >> 1];
    return __uint_as_float(i & 1 ? w & 0xFFFF0000u : w << 16);
  }
  __device__ __forceinline__ float max() const {
    const __nv_bfloat162 a = __hmax2(__hmax2(pair(0), pair(1)), __hmax2(pair(2), pair(3)));
    return fmaxf(__low2float(a), __high2float(a));
  }
  __device__ __forceinline__ int above(float xt) const {  // counts to 8: exact in bf16
    const __nv_bfloat162 c = __float2bfloat162_rn(xt);
    const __nv_bfloat162 a =
        __hadd2(__hadd2(__hgt2(pair(0), c), __hgt2(pair(1), c)), __hadd2(__hgt2(pair(2), c), __hgt2(pair(3), c)));
    return (int)(__low2float(a) + __high2float(a));
  }
};
template <>
struct Vec<__half> {
  static constexpr int N = 8;
  uint4 v;
  __device__ __forceinline__ __half2 pair(int i) const { return reinterpret_cast<const __half2*>(&v)[i]; }
  __device__ __forceinline__ float get(int i) const {
    const __half2 h = pair(i >> 1);
    return i & 1 ? __high2float(h) : __low2float(h);
  }
  __device__ __forceinline__ float max() const {
    const __half2 a = __hmax2(__hmax2(pair(0), pair(1)), __hmax2(pair(2), pair(3)));
    return fmaxf(__low2float(a), __high2float(a));
  }
  __device__ __forceinline__ int above(float xt) const {
    const __half2 c = __float2half2_rn(xt);
    const __half2 a =
        __hadd2(__hadd2(__hgt2(pair(0), c), __hgt2(pair(1), c)), __hadd2(__hgt2(pair(2), c), __hgt2(pair(3), c)));
    return (int)(__low2float(a) + __high2float(a));
  }
};

template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* p) {
  Vec<T> r;
  r.v = __ldg(reinterpret_cast<const decltype(r.v)*>(p));
  return r;
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT) token_logprobs_kernel(const __grid_constant__ LogprobParams p) {
  constexpr int N = Vec<T>::N, kWarps = NT / 32;
  __shared__ float s_m[kWarps], s_l[kWarps], s_t[kWarps];
  __shared__ int s_above[kWarps];
  __shared__ float s_group[kGroups];
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
  for (int j = tid; j < vecs; j += kBatch * NT) {
    Vec<T> v[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (j + u * NT < vecs) v[u] = load_vec(body + (int64_t)(j + u * NT) * N);
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (j + u * NT < vecs) {
        s.raise(v[u].max());
        above += v[u].above(xt);
        if (s.m > -INFINITY) {
#pragma unroll
          for (int i = 0; i < N; ++i) s.add(v[u].get(i));
        } else {  // nothing finite yet: only a NaN counts
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (v[u].get(i) != v[u].get(i)) s.l = NAN;
        }
      }
  }
  // the edge goes to the last threads
  const int mine = NT - 1 - tid;
  const int edge_at = mine < edge ? (mine < head ? mine : p.V - edge + mine) : -1;
  float edge_x = -INFINITY;
  if (edge_at >= 0) {
    edge_x = to_f(row[edge_at]);
    s.raise(edge_x);
    above += edge_x > xt;
    if (s.m > -INFINITY || edge_x != edge_x) s.add(edge_x);
  }

  // join the threads
  const float mine_max = s.m;
  const float wm = warp_max(s.m);
  if (lane == 0) s_m[warp] = wm;
  if (tid == 0) s_threads = s_cands = 0;
  if (p.top) {
    float gm = s.m;
#pragma unroll
    for (int o = 1; o < NT / kGroups; o <<= 1) gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, o));
    if (tid % (NT / kGroups) == 0) s_group[tid / (NT / kGroups)] = gm;
  }
  __syncthreads();
  float m = s_m[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) m = fmaxf(m, s_m[w]);
  s.raise(m);
  const float wl = warp_sum(s.l), wt = warp_sum(s.t);
  const int wa = __reduce_add_sync(0xffffffffu, above);
  if (lane == 0) {
    s_l[warp] = wl;
    s_t[warp] = wt;
    s_above[warp] = wa;
  }
  if (p.top && tid < kGroups) {
    // the top-th largest group maximum (equal ones in group order)
    const float me = s_group[tid];
    int ahead = 0;
#pragma unroll 16
    for (int g = 0; g < kGroups; ++g) ahead += s_group[g] > me || (s_group[g] == me && g < tid);
    if (ahead == p.top - 1) s_tau = me;
  }
  __syncthreads();
  float l = 0.0f, t = 0.0f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    l += s_l[w];
    t += s_t[w];
  }
  const float log2l = log2f(l);
  if (tid == 0) {
    int n = 0;
    for (int w = 0; w < kWarps; ++w) n += s_above[w];
    p.logprob[r] = tok >= 0 ? (xt - m) - log2l * kLn2 : 0.0f;
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
  const int per = (vecs + NT - 1) / NT;
  bool strict = false;
  int cands;
  while (true) {
    auto passes = [&](float v) { return strict ? v > tau : v >= tau; };
    auto take = [&](float v, int i) {
      const int at = atomicAdd(&s_cands, 1);
      if (at < kCand) s_cand[at] = top_key(v, i);
    };
    if (passes(mine_max)) s_thread[atomicAdd(&s_threads, 1)] = tid;
    if (edge_at >= 0 && passes(edge_x)) take(edge_x, edge_at);
    __syncthreads();
    const int jobs = s_threads * per;
    for (int job = tid; job < jobs; job += NT) {
      const int j = s_thread[job / per] + (job % per) * NT;
      if (j >= vecs || s_cands > kCand) continue;
      const Vec<T> v = load_vec(body + (int64_t)j * N);
      if (!passes(v.max())) continue;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (passes(v.get(i))) take(v.get(i), head + j * N + i);
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
        out_lp[ahead] = (to_f(row[i]) - m) - log2l * kLn2;
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
        out_lp[k] = (to_f(row[i]) - m) - log2l * kLn2;
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
      out_lp[at] = (tau - m) - log2l * kLn2;
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
  // 256 threads a row leave eight rows to an SM, whose reductions and reads
  // overlap; with at most a row per SM, 1024 threads hold a row's reads in flight
  if (rows > num_sms()) token_logprobs_kernel<T, 256><<<rows, 256, 0, st>>>(p);
  else token_logprobs_kernel<T, 1024><<<rows, 1024, 0, st>>>(p);
}

}  // namespace
}  // namespace cb

using namespace cb;

extern "C" int cb_token_logprobs(const void* logits, int32_t dtype, int64_t ld, int32_t rows, int32_t V,
                                 const int32_t* tokens, int32_t top, float* logprob, float* entropy, int32_t* rank,
                                 float* top_logprob, int32_t* top_token, int32_t* status, void* stream) {
  if (!logits || !tokens || !logprob || !entropy || !rank || rows <= 0 || V <= 0 || ld < V) return CB_ERR_ARG;
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
