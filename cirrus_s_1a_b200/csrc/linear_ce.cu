// Softmax cross entropy over a vocabulary from hidden rows, without keeping the logits.
//
//   x = h W^T       lse_n = log sum_v exp x_nv       loss_n = lse_n - x_n,t(n)
//   G_nv = a_n p_nv - b_n [v = t(n)],  p = exp(x - lse),  a = dL/dloss + dL/dlse,  b = dL/dloss
//   dh = G W        dW = G^T h
//
// Forward: each tile of logits leaves its rows' maximum and sum, which a second kernel
// joins in the order of the vocabulary.  Backward: the logits are taken again for a piece
// of the vocabulary at a time, and G of that piece goes into both products.
#include "ends.cuh"

namespace cb {
namespace {

constexpr int kTile = 64, kStep = 16, kThreads = 256;
constexpr int kPiece = 2048;  // vocabulary rows whose G is held at a time

struct Problem {
  const void *h, *w;
  int64_t ldh, ldw;
  int N, V, d;
  Ids targets;
};

__device__ __forceinline__ int64_t target_of(const Problem& p, int n) {
  const int64_t t = p.targets[n];
  return t >= 0 && t < p.V ? t : -1;
}

// acc[i][j] = sum_k A[r0 + ty * 4 + i][k] * B[c0 + tx * 4 + j][k], with A and B given as functions of (row, k).
template <typename FA, typename FB>
__device__ __forceinline__ void tile_product(float (&acc)[4][4], int K, FA&& a, FB&& b) {
  __shared__ float As[kStep][kTile + 1], Bs[kStep][kTile + 1];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  for (int k0 = 0; k0 < K; k0 += kStep) {
    __syncthreads();
    for (int e = tid; e < kTile * kStep; e += kThreads) {
      const int k = e % kStep, r = e / kStep;
      As[k][r] = k0 + k < K ? a(r, k0 + k) : 0.0f;
      Bs[k][r] = k0 + k < K ? b(r, k0 + k) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kStep; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(As[k][ty * 4 + i], Bs[k][tx * 4 + j], acc[i][j]);
  }
}

// part[tile][n] = (maximum, sum of exponentials against it) of the row's logits in the tile; xt[n] the target's logit.
template <typename TH, typename TW>
__global__ void __launch_bounds__(kThreads) stats_kernel(Problem p, float2* part, float* xt) {
  const int n0 = blockIdx.x * kTile, v0 = blockIdx.y * kTile;
  float x[4][4] = {};
  tile_product(
      x, p.d,
      [&](int r, int k) { return n0 + r < p.N ? Elem<TH>::get(static_cast<const TH*>(p.h)[(n0 + r) * p.ldh + k]) : 0.0f; },
      [&](int r, int k) { return v0 + r < p.V ? Elem<TW>::get(static_cast<const TW*>(p.w)[(v0 + r) * p.ldw + k]) : 0.0f; });
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = n0 + ty * 4 + i;
    const int64_t t = n < p.N ? target_of(p, n) : -1;
    float m = -INFINITY, l = 0.0f;
    bool nan = false;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (v0 + tx * 4 + j < p.V) {
        m = fmaxf(m, x[i][j]);
        nan |= x[i][j] != x[i][j];
        if (v0 + tx * 4 + j == t) xt[n] = x[i][j];
      }
    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (v0 + tx * 4 + j < p.V && m > -INFINITY) l += expf(x[i][j] - m);
    if (nan) l = NAN;
    for (int o = 8; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (tx == 0 && n < p.N) part[(int64_t)blockIdx.y * p.N + n] = make_float2(m, l);
  }
}

__global__ void __launch_bounds__(kThreads) join_kernel(Problem p, const float2* part, int tiles, const float* xt,
                                                        float* loss, float* lse, int32_t* status) {
  const int n = blockIdx.x * kThreads + threadIdx.x;
  if (n >= p.N) return;
  float m = -INFINITY, l = 0.0f;
  for (int i = 0; i < tiles; ++i) m = fmaxf(m, part[(int64_t)i * p.N + n].x);
  for (int i = 0; i < tiles; ++i) {
    const float2 q = part[(int64_t)i * p.N + n];
    l += q.y == 0.0f ? 0.0f : q.y * expf(q.x - m);
  }
  lse[n] = m + logf(l);
  const int64_t t = target_of(p, n);
  loss[n] = t >= 0 ? (m - xt[n]) + logf(l) : 0.0f;
  if (p.targets[n] >= p.V) set_status(status, CB_ERR_TOKEN);
}

__global__ void __launch_bounds__(1024) reduce_kernel(Problem p, const float* loss, int mean, float* out, int32_t* count) {
  __shared__ double sums[1024];
  __shared__ int counts[1024];
  double s = 0.0;
  int c = 0;
  for (int n = threadIdx.x; n < p.N; n += 1024) {
    c += target_of(p, n) >= 0;
    s += loss[n];
  }
  sums[threadIdx.x] = s;
  counts[threadIdx.x] = c;
  for (int o = 512; o > 0; o >>= 1) {
    __syncthreads();
    if (threadIdx.x < o) {
      sums[threadIdx.x] += sums[threadIdx.x + o];
      counts[threadIdx.x] += counts[threadIdx.x + o];
    }
  }
  if (threadIdx.x == 0) {
    *out = (float)(mean ? sums[0] / max(counts[0], 1) : sums[0]);
    *count = counts[0];
  }
}

struct Upstream {
  const float *loss, *lse;  // either may be null
  int64_t loss_step, lse_step;
  const int32_t* count;  // mean: rows with a target
  int reduction;
};

__global__ void __launch_bounds__(kThreads) factors_kernel(Problem p, Upstream u, float2* ab) {
  const int n = blockIdx.x * kThreads + threadIdx.x;
  if (n >= p.N) return;
  float b = 0.0f;
  if (u.loss && target_of(p, n) >= 0) {
    b = u.loss[u.reduction == CB_REDUCE_NONE ? n * u.loss_step : 0];
    if (u.reduction == CB_REDUCE_MEAN) b /= (float)max(*u.count, 1);
  }
  ab[n] = make_float2(b + (u.lse ? u.lse[n * u.lse_step] : 0.0f), b);
}

__device__ __forceinline__ bool dead(float2 ab) { return ab.x == 0.0f && ab.y == 0.0f; }

// G[n][v - v0] of the vocabulary rows v0 .. v0 + vp; a row without a gradient is 0 whatever it holds.
template <typename TH, typename TW>
__global__ void __launch_bounds__(kThreads) grad_kernel(Problem p, const float2* ab, const float* lse, int v0, int vp,
                                                        float* G) {
  const int n0 = blockIdx.x * kTile, c0 = blockIdx.y * kTile;
  float x[4][4] = {};
  tile_product(
      x, p.d,
      [&](int r, int k) { return n0 + r < p.N ? Elem<TH>::get(static_cast<const TH*>(p.h)[(n0 + r) * p.ldh + k]) : 0.0f; },
      [&](int r, int k) {
        return c0 + r < vp ? Elem<TW>::get(static_cast<const TW*>(p.w)[(v0 + c0 + r) * p.ldw + k]) : 0.0f;
      });
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = n0 + ty * 4 + i;
    if (n >= p.N) continue;
    const int64_t t = target_of(p, n);
    const float2 f = ab[n];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = c0 + tx * 4 + j;
      if (c >= vp) continue;
      G[(int64_t)n * vp + c] = dead(f) ? 0.0f : f.x * expf(x[i][j] - lse[n]) - (v0 + c == t ? f.y : 0.0f);
    }
  }
}

// acc (+)= G W of a piece.
template <typename TW>
__global__ void __launch_bounds__(kThreads) dh_kernel(Problem p, const float* G, int v0, int vp, float* acc) {
  const int n0 = blockIdx.x * kTile, c0 = blockIdx.y * kTile;
  float x[4][4] = {};
  tile_product(
      x, vp, [&](int r, int k) { return n0 + r < p.N ? G[(int64_t)(n0 + r) * vp + k] : 0.0f; },
      [&](int r, int k) {
        return c0 + r < p.d ? Elem<TW>::get(static_cast<const TW*>(p.w)[(v0 + k) * p.ldw + c0 + r]) : 0.0f;
      });
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + ty * 4 + i, c = c0 + tx * 4 + j;
      if (n < p.N && c < p.d) acc[(int64_t)n * p.d + c] = (v0 ? acc[(int64_t)n * p.d + c] : 0.0f) + x[i][j];
    }
}

template <typename TH>
__global__ void __launch_bounds__(kThreads) dh_out_kernel(Problem p, const float2* ab, const float* acc, TH* dh) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= (int64_t)p.N * p.d) return;
  dh[i] = Elem<TH>::put(dead(ab[i / p.d]) ? 0.0f : acc[i]);
}

// dW = G^T h of a piece; rows without a gradient are left out, whatever they hold.
template <typename TH, typename TW>
__global__ void __launch_bounds__(kThreads) dw_kernel(Problem p, const float2* ab, const float* G, int v0, int vp, TW* dw) {
  const int r0 = blockIdx.x * kTile, c0 = blockIdx.y * kTile;
  float x[4][4] = {};
  tile_product(
      x, p.N, [&](int r, int k) { return r0 + r < vp ? G[(int64_t)k * vp + r0 + r] : 0.0f; },
      [&](int r, int k) {
        return c0 + r < p.d && !dead(ab[k]) ? Elem<TH>::get(static_cast<const TH*>(p.h)[k * p.ldh + c0 + r]) : 0.0f;
      });
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = r0 + ty * 4 + i, c = c0 + tx * 4 + j;
      if (r < vp && c < p.d) dw[(int64_t)(v0 + r) * p.d + c] = Elem<TW>::put(x[i][j]);
    }
}

bool bad(const void* h, int32_t h_dtype, int64_t ldh, const void* w, int32_t w_dtype, int64_t ldw, int32_t N, int32_t V,
         int32_t d, const void* targets, int32_t targets_64, int32_t reduction) {
  if (!h || !w || !targets || N <= 0 || V <= 0 || d <= 0 || !is_dtype(h_dtype) || !is_dtype(w_dtype)) return true;
  if (h_dtype != w_dtype && !(h_dtype == CB_F32 && w_dtype == CB_BF16)) return true;
  if (ldh < 0 || (V > 1 && ldw < d)) return true;
  if (reduction != CB_REDUCE_NONE && reduction != CB_REDUCE_MEAN && reduction != CB_REDUCE_SUM) return true;
  return !aligned_to(h, dtype_size(h_dtype)) || !aligned_to(w, dtype_size(w_dtype)) || !aligned_to(targets, targets_64 ? 8 : 4);
}

bool too_large(int32_t N, int32_t V, int32_t d) {
  return N > CB_ENDS_MAX_ROWS || V > CB_ENDS_MAX_VOCAB || d > CB_ENDS_MAX_DIM;
}

size_t up16(size_t n) { return (n + 15) / 16 * 16; }

template <typename F>
int with_types(int32_t h_dtype, int32_t w_dtype, F&& f) {
  if (h_dtype == CB_F32) return w_dtype == CB_F32 ? f(float{}, float{}) : f(float{}, __nv_bfloat16{});
  return with_type(h_dtype, [&](auto t) { return f(t, t); });
}

}  // namespace
}  // namespace cb

using namespace cb;

extern "C" size_t cb_linear_ce_scratch_bytes(int32_t h_dtype, int32_t w_dtype, int32_t N, int32_t V, int32_t d,
                                             int32_t backward) {
  if (N <= 0 || V <= 0 || d <= 0 || too_large(N, V, d) || !is_dtype(h_dtype) || !is_dtype(w_dtype)) return 0;
  if (!backward) return up16((size_t)N * ceil_div(V, kTile) * sizeof(float2)) + up16((size_t)N * 4) * 2;
  return up16((size_t)N * sizeof(float2)) + up16((size_t)N * min(V, kPiece) * 4) + up16((size_t)N * d * 4);
}

extern "C" int cb_linear_ce(const void* h, int32_t h_dtype, int64_t ldh, const void* w, int32_t w_dtype, int64_t ldw,
                            int32_t N, int32_t V, int32_t d, const void* targets, int32_t targets_64, int32_t reduction,
                            float* loss, float* lse, int32_t* count, void* scratch, size_t scratch_bytes,
                            int32_t* status, void* stream) {
  if (bad(h, h_dtype, ldh, w, w_dtype, ldw, N, V, d, targets, targets_64, reduction) || !loss || !lse || !scratch ||
      !aligned_to(scratch, 16) || (reduction != CB_REDUCE_NONE && !count))
    return CB_ERR_ARG;
  if (too_large(N, V, d)) return CB_ERR_SHAPE;
  if (scratch_bytes < cb_linear_ce_scratch_bytes(h_dtype, w_dtype, N, V, d, 0)) return CB_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t)stream;
  const Problem p{h, w, ldh, ldw, N, V, d, Ids{targets, targets_64}};
  const int tiles = ceil_div(V, kTile);
  float2* part = static_cast<float2*>(scratch);
  float* xt = reinterpret_cast<float*>(static_cast<char*>(scratch) + up16((size_t)N * tiles * sizeof(float2)));
  float* rows = reduction == CB_REDUCE_NONE ? loss : xt + up16((size_t)N * 4) / 4;
  return with_types(h_dtype, w_dtype, [&](auto t, auto u) {
    using TH = decltype(t);
    using TW = decltype(u);
    stats_kernel<TH, TW><<<dim3(ceil_div(N, kTile), tiles), kThreads, 0, st>>>(p, part, xt);
    if (int rc = launched()) return rc;
    join_kernel<<<ceil_div(N, kThreads), kThreads, 0, st>>>(p, part, tiles, xt, rows, lse, status);
    if (int rc = launched()) return rc;
    if (reduction == CB_REDUCE_NONE) return (int)CB_OK;
    reduce_kernel<<<1, 1024, 0, st>>>(p, rows, reduction == CB_REDUCE_MEAN, loss, count);
    return launched();
  });
}

extern "C" int cb_linear_ce_grad(const void* h, int32_t h_dtype, int64_t ldh, const void* w, int32_t w_dtype,
                                 int64_t ldw, int32_t N, int32_t V, int32_t d, const void* targets, int32_t targets_64,
                                 int32_t reduction, const float* lse, const int32_t* count, const float* g_loss,
                                 int64_t g_loss_step, const float* g_lse, int64_t g_lse_step, void* dh, void* dw,
                                 void* scratch, size_t scratch_bytes, int32_t* status, void* stream) {
  (void)status;
  if (bad(h, h_dtype, ldh, w, w_dtype, ldw, N, V, d, targets, targets_64, reduction) || !lse || !scratch ||
      !aligned_to(scratch, 16) || (reduction == CB_REDUCE_MEAN && !count) || g_loss_step < 0 || g_lse_step < 0 ||
      (!dh && !dw) || (dh && !aligned_to(dh, dtype_size(h_dtype))) || (dw && !aligned_to(dw, dtype_size(w_dtype))))
    return CB_ERR_ARG;
  if (too_large(N, V, d)) return CB_ERR_SHAPE;
  if (scratch_bytes < cb_linear_ce_scratch_bytes(h_dtype, w_dtype, N, V, d, 1)) return CB_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t)stream;
  const Problem p{h, w, ldh, ldw, N, V, d, Ids{targets, targets_64}};
  char* at = static_cast<char*>(scratch);
  float2* ab = reinterpret_cast<float2*>(at);
  float* G = reinterpret_cast<float*>(at += up16((size_t)N * sizeof(float2)));
  float* acc = reinterpret_cast<float*>(at + up16((size_t)N * min(V, kPiece) * 4));
  factors_kernel<<<ceil_div(N, kThreads), kThreads, 0, st>>>(
      p, Upstream{g_loss, g_lse, g_loss_step, g_lse_step, count, reduction}, ab);
  if (int rc = launched()) return rc;
  return with_types(h_dtype, w_dtype, [&](auto t, auto u) {
    using TH = decltype(t);
    using TW = decltype(u);
    for (int v0 = 0; v0 < V; v0 += kPiece) {
      const int vp = min(kPiece, V - v0);
      grad_kernel<TH, TW><<<dim3(ceil_div(N, kTile), ceil_div(vp, kTile)), kThreads, 0, st>>>(p, ab, lse, v0, vp, G);
      if (int rc = launched()) return rc;
      if (dh) {
        dh_kernel<TW><<<dim3(ceil_div(N, kTile), ceil_div(d, kTile)), kThreads, 0, st>>>(p, G, v0, vp, acc);
        if (int rc = launched()) return rc;
      }
      if (dw) {
        dw_kernel<TH, TW><<<dim3(ceil_div(vp, kTile), ceil_div(d, kTile)), kThreads, 0, st>>>(p, ab, G, v0, vp,
                                                                                            static_cast<TW*>(dw));
        if (int rc = launched()) return rc;
      }
    }
    if (!dh) return (int)CB_OK;
    dh_out_kernel<TH><<<(unsigned)(((int64_t)N * d + kThreads - 1) / kThreads), kThreads, 0, st>>>(p, ab, acc,
                                                                                                  static_cast<TH*>(dh));
    return launched();
  });
}
