// cb_token_logprobs: for each row x of logits, with m = max x, l = sum exp(x - m):
//   logprob = x[token] - m - log l
//   entropy = log l - (1/l) sum (x - m) exp(x - m)
//   rank    = how many logits are larger than x[token]
//   the `top` largest logits in order (ties to the lowest token), as log probabilities
//
// One CTA per row: one pass for m, l, the entropy sum and the rank, then one
// pass over the row for each alternative.
#include "common.cuh"
#include "kv8.cuh"

namespace cb {
namespace {

constexpr int kLT = 256;

struct LogprobParams {
  const void* x;
  int dtype;
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

// (value, token) as one key: larger value first, then the lower token.
__device__ __forceinline__ unsigned long long top_key(float v, int i) {
  return ((unsigned long long)(v != v ? 0xFFFFFFFFu : score_key(v)) << 32) | (uint32_t)~i;
}

__global__ void __launch_bounds__(kLT) token_logprobs_kernel(const __grid_constant__ LogprobParams p) {
  __shared__ float red[33];
  __shared__ unsigned long long kred[kLT / 32];
  const int64_t r = blockIdx.x, base = r * p.ld;
  const int tid = threadIdx.x;
  int tok = p.tokens[r];
  if (tok >= p.V) {
    if (tid == 0) set_status(p.status, CB_ERR_TOKEN);
    tok = -1;
  }
  const float xt = tok >= 0 ? kv8_load(p.x, base + tok, p.dtype) : INFINITY;
  float m = -INFINITY;
  int above = 0;
  for (int i = tid; i < p.V; i += kLT) {
    const float v = kv8_load(p.x, base + i, p.dtype);
    m = fmaxf(m, v);
    above += v > xt;
  }
  m = block_max(m, red);
  float l = 0.0f, t = 0.0f;
  for (int i = tid; i < p.V; i += kLT) {
    const float d = kv8_load(p.x, base + i, p.dtype) - m, e = expf(d);
    l += e;
    if (e > 0.0f) t += d * e;
  }
  l = block_sum(l, red);
  t = block_sum(t, red);
  const float rank = block_sum((float)above, red);  // V < 2^24: exact
  const float logl = logf(l);
  if (tid == 0) {
    p.logprob[r] = tok >= 0 ? (xt - m) - logl : 0.0f;
    p.entropy[r] = logl - t / l;
    p.rank[r] = tok >= 0 ? (int)rank : -1;
  }
  unsigned long long below = ~0ull;
  for (int k = 0; k < p.top; ++k) {
    unsigned long long best = 0;
    for (int i = tid; i < p.V; i += kLT) {
      const unsigned long long u = top_key(kv8_load(p.x, base + i, p.dtype), i);
      if (u < below && u > best) best = u;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long u = __shfl_xor_sync(0xffffffffu, best, o);
      best = u > best ? u : best;
    }
    __syncthreads();
    if ((tid & 31) == 0) kred[tid >> 5] = best;
    __syncthreads();
    for (int w = 0; w < kLT / 32; ++w) best = kred[w] > best ? kred[w] : best;
    below = best;
    if (tid == 0) {
      const int i = (int)~(uint32_t)best;
      p.top_token[r * p.top + k] = i;
      p.top_logprob[r * p.top + k] = (kv8_load(p.x, base + i, p.dtype) - m) - logl;
    }
  }
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
  const LogprobParams p{logits, dtype, ld, V, top, tokens, logprob, entropy, rank, top_logprob, top_token, status};
  token_logprobs_kernel<<<rows, kLT, 0, (cudaStream_t)stream>>>(p);
  count_launch();
  return cudaGetLastError() == cudaSuccess ? CB_OK : CB_ERR_CUDA;
}
