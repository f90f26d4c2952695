// Embedding lookup with scaling, and its gradient.
//
//   y[n] = scale * table[id_n]                dtable[v] = scale * sum of g[n] over the n with id_n = v
//
// Both are bound by memory.  The gradient is written by vocabulary rows, so that every
// row has one owner and its sum one order, that of the tokens, whatever their number.
#include "ends.cuh"

namespace cb {
namespace {

constexpr int kThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kThreads) embedding_kernel(const T* table, int64_t ld, int V, int d, Ids ids,
                                                             float scale, T* out, int32_t* status) {
  const int64_t n = blockIdx.x;
  const int64_t id = ids[n];
  const bool has = id >= 0 && id < V;
  if (id >= V && threadIdx.x == 0) set_status(status, CB_ERR_TOKEN);
  for (int j = threadIdx.x; j < d; j += kThreads)
    out[n * d + j] = has ? Elem<T>::put(Elem<T>::get(table[id * ld + j]) * scale) : Elem<T>::put(0.0f);
}

// A warp to 32 columns of a vocabulary row: it reads all ids in order.
template <typename T>
__global__ void __launch_bounds__(kThreads) embedding_grad_kernel(const T* g, int64_t ldg, Ids ids, int64_t n, int V,
                                                                  int d, float scale, T* dtable) {
  const int lane = threadIdx.x & 31;
  const int64_t v = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (v >= V) return;
  const int j = blockIdx.y * 32 + lane;
  float sum = 0.0f;
  for (int64_t i = 0; i < n; i += 32) {
    uint32_t hits = __ballot_sync(0xffffffffu, i + lane < n && ids[i + lane] == v);
    while (hits) {
      const int at = __ffs(hits) - 1;
      hits &= hits - 1;
      if (j < d) sum += Elem<T>::get(g[(i + at) * ldg + j]);
    }
  }
  if (j < d) dtable[v * d + j] = Elem<T>::put(sum * scale);
}

}  // namespace
}  // namespace cb

using namespace cb;

extern "C" int cb_embedding(const void* table, int32_t dtype, int64_t ld, int32_t V, int32_t d, const void* ids,
                            int32_t ids_64, int64_t n, float scale, void* out, int32_t* status, void* stream) {
  if (!table || !ids || !out || V <= 0 || d <= 0 || n <= 0 || (V > 1 && ld < d) || !is_dtype(dtype)) return CB_ERR_ARG;
  if (!aligned_to(table, dtype_size(dtype)) || !aligned_to(out, dtype_size(dtype)) || !aligned_to(ids, ids_64 ? 8 : 4))
    return CB_ERR_ARG;
  if (n > CB_ENDS_MAX_ROWS || V > CB_ENDS_MAX_VOCAB || d > CB_ENDS_MAX_DIM) return CB_ERR_SHAPE;
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    embedding_kernel<T><<<(unsigned)n, kThreads, 0, (cudaStream_t)stream>>>(
        static_cast<const T*>(table), ld, V, d, Ids{ids, ids_64}, scale, static_cast<T*>(out), status);
    return launched();
  });
}

extern "C" size_t cb_embedding_grad_scratch_bytes(int64_t n, int32_t V, int32_t d) {
  if (n <= 0 || V <= 0 || d <= 0 || n > CB_ENDS_MAX_ROWS || V > CB_ENDS_MAX_VOCAB || d > CB_ENDS_MAX_DIM) return 0;
  return 16;
}

extern "C" int cb_embedding_grad(const void* g, int32_t dtype, int64_t ldg, const void* ids, int32_t ids_64, int64_t n,
                                 int32_t V, int32_t d, float scale, void* dtable, void* scratch, size_t scratch_bytes,
                                 void* stream) {
  if (!g || !ids || !dtable || !scratch || V <= 0 || d <= 0 || n <= 0 || ldg < 0 || !is_dtype(dtype)) return CB_ERR_ARG;
  if (!aligned_to(g, dtype_size(dtype)) || !aligned_to(dtable, dtype_size(dtype)) || !aligned_to(ids, ids_64 ? 8 : 4) ||
      !aligned_to(scratch, 16))
    return CB_ERR_ARG;
  const size_t need = cb_embedding_grad_scratch_bytes(n, V, d);
  if (!need) return CB_ERR_SHAPE;
  if (scratch_bytes < need) return CB_ERR_WORKSPACE;
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    const dim3 grid((unsigned)ceil_div(V, kThreads / 32), (unsigned)ceil_div(d, 32));
    embedding_grad_kernel<T><<<grid, kThreads, 0, (cudaStream_t)stream>>>(static_cast<const T*>(g), ldg, Ids{ids, ids_64},
                                                                          n, V, d, scale, static_cast<T*>(dtable));
    return launched();
  });
}
