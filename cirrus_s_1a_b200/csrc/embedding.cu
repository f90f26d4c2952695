// Embedding lookup with scaling, and its gradient.
//
//   y[n] = scale * table[id_n]                dtable[v] = scale * sum of g[n] over the n with id_n = v
//
// Both are bound by memory: a row read and a row written for each token, and every row of
// dtable.  The gradient sorts the tokens by id, so that every row has one owner and its sum
// one order, that of the tokens:
//   * sort_kernel: a cluster of up to 16 CTAs sorts up to 131072 (id, token) pairs by 8-bit
//     digits, stable, exchanging counts and pairs through distributed shared memory; a CTA
//     orders its own pairs first, so that what it sends goes in runs (131072 pairs: 29 us,
//     35 with each pair sent from where it was);
//   * sum_kernel: a warp sums 32 sorted tokens over 512 bytes of columns, however the tokens
//     fall to rows, so that a frequent token is spread over many warps; a row whose tokens
//     end within them is written, one that goes on leaves its part (float32) in scratch;
//     other warps write the rows without a token;
//   * join_kernel: adds the parts of such rows in order.
// More tokens are taken in batches, added up in float32.
// Measured, 131072 tokens, 32768 x 1024 in float32: lookup 104 us (5.9 TB/s), sort 30, sums
// 110 (5.3 TB/s), join 26; 16384 tokens, 32000 x 768 in bf16: 11, 14, 20 and 7.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "ends.cuh"

namespace cb {
namespace {

constexpr int kThreads = 256;
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kPerCta = 8192, kMaxCluster = 16;
constexpr int64_t kBatch = (int64_t)kPerCta * kMaxCluster;
constexpr int kChunk = 32;  // sorted tokens of a warp

// ----------------------------------------------------------------- lookup
constexpr int kPieces = 4;  // of a thread, in flight together

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) embedding_kernel(const T* table, int64_t ld, int V, int vecs, Ids ids,
                                                             int64_t all, float scale, T* out, int32_t* status) {
  await_before();
  start_next();
  const int64_t first = (int64_t)blockIdx.x * (kPieces * kThreads) + threadIdx.x;
  Vec<T, VEC> x[kPieces];
#pragma unroll
  for (int p = 0; p < kPieces; ++p) {
    const int64_t i = first + p * kThreads;
    if (i >= all) break;
    const int64_t n = all < (1ll << 31) ? (int64_t)((uint32_t)i / (uint32_t)vecs) : i / vecs;
    const int j = (int)(i - n * vecs);
    const int64_t id = ids[n];
    if (id >= 0 && id < V) {
      x[p] = *reinterpret_cast<const Vec<T, VEC>*>(table + id * ld + j * VEC);
    } else {
      if (id >= V && j == 0) set_status(status, CB_ERR_TOKEN);
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[p].v[k] = Elem<T>::put(0.0f);
    }
  }
#pragma unroll
  for (int p = 0; p < kPieces; ++p) {
    const int64_t i = first + p * kThreads;
    if (i >= all) break;
    if (scale != 1.0f)
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[p].v[k] = Elem<T>::put(Elem<T>::get(x[p].v[k]) * scale);
    *reinterpret_cast<Vec<T, VEC>*>(out + i * VEC) = x[p];
  }
}

// ------------------------------------------------------------------- sort
struct SortShared {
  uint2 pairs[2][kPerCta];  // (key, token)
  uint16_t rank[kPerCta];   // of a pair among its digit's in its warp's segment
  uint16_t count[kSortWarps][256];
  uint32_t total[256], local[256], base[256], warp_sum[8];
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t at_rank(const void* p, int rank) {
  uint32_t a = (uint32_t)__cvta_generic_to_shared(p), r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}

// Tokens [0, n) of the batch by id, those without one (as id V) last: keys and order.
__global__ void __launch_bounds__(kSortThreads) sort_kernel(Ids ids, int64_t first, int n, int V, int passes,
                                                            uint32_t* keys, uint32_t* order) {
  extern __shared__ SortShared sort_shared[];
  SortShared& s = *sort_shared;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x, ctas = gridDim.x;  // one cluster
  await_before();
  start_next();
  const int per = (n + ctas - 1) / ctas, mine = max(0, min(per, n - rank * per));
  // a warp's segment
  const int seg = ((per + kSortWarps - 1) / kSortWarps + 31) / 32 * 32;
  const int from = min(mine, warp * seg), to = min(mine, from + seg);
#pragma unroll
  for (int k = 0; k < kPerCta / kSortThreads; ++k) {
    const int i = k * kSortThreads + tid;
    if (i < mine) {
      const int64_t id = ids[first + rank * per + i];
      s.pairs[0][i] = make_uint2(id >= 0 && id < V ? (uint32_t)id : (uint32_t)V, (uint32_t)(rank * per + i));
    }
  }
  uint2 *in = s.pairs[0], *ordered = s.pairs[1];
  // the sum of a value over threads 0 .. tid - 1 of the first 256
  auto scan256 = [&](uint32_t v) {
    uint32_t sum = v;
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += u;
    }
    if (tid < 256 && lane == 31) s.warp_sum[warp] = sum;
    __syncthreads();
    if (tid < 256)
      for (int w = 0; w < warp; ++w) sum += s.warp_sum[w];
    __syncthreads();
    return sum - v;
  };
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * 8;
    for (int i = lane; i < 256; i += 32) s.count[warp][i] = 0;
    __syncthreads();
    for (int i = from + lane; i - lane < to; i += 32) {
      const bool is = i < to;
      const uint32_t digit = is ? in[i].x >> shift & 255 : 0;
      // the lanes of the same digit: eight votes (a match instruction takes longer)
      uint32_t same = __ballot_sync(0xffffffffu, is);
#pragma unroll
      for (int bit = 0; bit < 8; ++bit) {
        const bool one = digit >> bit & 1;
        const uint32_t ones = __ballot_sync(0xffffffffu, one);
        same &= one ? ones : ~ones;
      }
      const int before = __popc(same & ((1u << lane) - 1));
      const int at = is ? s.count[warp][digit] : 0;
      __syncwarp();
      if (is) {
        s.rank[i] = (uint16_t)(at + before);
        if (before == 0) s.count[warp][digit] = (uint16_t)(at + __popc(same));
      }
      __syncwarp();
    }
    __syncthreads();
    uint32_t mine_of = 0;  // of digit tid
    if (tid < 256) {  // counts of the warps before, for each digit
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = s.count[w][tid];
        s.count[w][tid] = (uint16_t)mine_of;
        mine_of += c;
      }
      s.total[tid] = mine_of;
    }
    const uint32_t at_local = scan256(mine_of);
    if (tid < 256) s.local[tid] = at_local;
    __syncthreads();
    for (int i = from + lane; i < to; i += 32) {
      const uint2 p = in[i];
      const uint32_t digit = p.x >> shift & 255;
      ordered[s.local[digit] + s.count[warp][digit] + s.rank[i]] = p;
    }
    cluster_sync();  // totals are there, and every CTA has taken its pairs out of `in`
    uint32_t before = 0, all = 0;
    if (tid < 256) {
      uint32_t c[kMaxCluster];
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) {
        c[r] = 0;
        if (r < ctas) asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(c[r]) : "r"(at_rank(&s.total[tid], r)));
      }
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) {
        before += r < rank ? c[r] : 0;
        all += c[r];
      }
    }
    const uint32_t at_all = scan256(all);
    if (tid < 256) s.base[tid] = at_all + before - at_local;  // what a pair moves by
    __syncthreads();
    const bool last = pass == passes - 1;
    for (int i = tid; i < mine; i += kSortThreads) {
      const uint2 p = ordered[i];
      const uint32_t at = i + s.base[p.x >> shift & 255];
      if (last) {
        keys[at] = p.x;
        order[at] = p.y;
      } else {
        const uint32_t cta = at / per;
        asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(at_rank(in + (at - cta * per), cta)), "r"(p.x),
                     "r"(p.y)
                     : "memory");
      }
    }
    cluster_sync();  // pairs have arrived, and totals may be replaced
  }
}

// ------------------------------------------------------------------- sums
// What a row's sum goes to: the table itself, or the batches' float32 sums.
template <typename T, int VEC>
__device__ __forceinline__ void write_row(T* dtable, float* total, int64_t at, const float* sum, float scale) {
  if (total) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) total[at + k] += sum[k];
  } else {
    Vec<T, VEC> x;
#pragma unroll
    for (int k = 0; k < VEC; ++k) x.v[k] = Elem<T>::put(sum[k] * scale);
    *reinterpret_cast<Vec<T, VEC>*>(dtable + at) = x;
  }
}

// part[chunk][which][d]: 0 the sum of the tokens of the row that began before the chunk, 1 of
// one that begins in it and goes on.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, VEC > 4 ? 2 : 4)
    sum_kernel(const T* g, int64_t ldg, const uint32_t* keys, const uint32_t* order, int n, int V, int d, int slabs,
               float scale, T* dtable, float* total, float* part) {
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  await_before();
  start_next();
  const int chunks = (n + kChunk - 1) / kChunk;
  const int64_t sums = (int64_t)chunks * slabs;
  if (w >= sums) {
    // rows without a token, 32 at a time
    const int64_t v0 = (w - sums) * 32;
    if (total || v0 >= V) return;
    const uint32_t v = (uint32_t)v0 + lane;
    int lo = 0, hi = n;  // the first key of v or more
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (keys[mid] < v) lo = mid + 1;
      else hi = mid;
    }
    uint32_t empty = __ballot_sync(0xffffffffu, v < (uint32_t)V && (lo >= n || keys[lo] != v));
    Vec<T, VEC> zero;
#pragma unroll
    for (int k = 0; k < VEC; ++k) zero.v[k] = Elem<T>::put(0.0f);
    while (empty) {
      const int64_t row = v0 + __ffs(empty) - 1;
      empty &= empty - 1;
      for (int j = lane * VEC; j < d; j += 32 * VEC) *reinterpret_cast<Vec<T, VEC>*>(dtable + row * d + j) = zero;
    }
    return;
  }
  const int chunk = (int)(w / slabs), j = ((int)(w % slabs) * 32 + lane) * VEC;
  const int first = chunk * kChunk, count = min(kChunk, n - first);
  const uint32_t none = (uint32_t)V;
  const uint32_t key = lane < count ? keys[first + lane] : none, prev = first > 0 ? keys[first - 1] : none;
  const uint32_t next = first + count < n ? keys[first + count] : none;
  const T* at = g + (lane < count ? order[first + lane] * ldg : 0);
  const int valid = __popc(__ballot_sync(0xffffffffu, key < none));  // the tokens without an id are the last
  const uint32_t after = __shfl_down_sync(0xffffffffu, key, 1);
  // where a row's tokens in the chunk end; its first row may have begun before, its last go on
  const uint32_t ends = __ballot_sync(0xffffffffu, lane < valid && (lane == valid - 1 || after != key));
  const uint32_t key0 = __shfl_sync(0xffffffffu, key, 0), key_last = __shfl_sync(0xffffffffu, key, max(valid - 1, 0));
  bool began = valid > 0 && key0 == prev;
  const bool goes_on = valid == count && key_last == next;
  const bool live = j < d;
  float sum[VEC] = {};
  constexpr int kAhead = 8;  // rows in flight
  for (int i0 = 0; i0 < valid; i0 += kAhead) {
    Vec<T, VEC> x[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const T* row = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(at), i0 + i));
      if (live && i0 + i < valid) x[i] = *reinterpret_cast<const Vec<T, VEC>*>(row + j);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (i0 + i >= valid) break;
#pragma unroll
      for (int k = 0; k < VEC; ++k) sum[k] += Elem<T>::get(x[i].v[k]);
      if (!(ends >> (i0 + i) & 1)) continue;
      const uint32_t row_key = __shfl_sync(0xffffffffu, key, i0 + i);
      if (live) {
        if (began || (goes_on && i0 + i == valid - 1)) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) part[((int64_t)chunk * 2 + (began ? 0 : 1)) * d + j + k] = sum[k];
        } else {
          write_row<T, VEC>(dtable, total, (int64_t)row_key * d + j, sum, scale);
        }
      }
      began = false;
#pragma unroll
      for (int k = 0; k < VEC; ++k) sum[k] = 0.0f;
    }
  }
}

template <int VEC>
__device__ __forceinline__ void load_sum(const float* at, float (&x)[VEC]) {
  constexpr int kN = VEC < 4 ? VEC : 4;
#pragma unroll
  for (int i = 0; i < VEC; i += kN) {
    const Vec<float, kN> v = *reinterpret_cast<const Vec<float, kN>*>(at + i);
#pragma unroll
    for (int k = 0; k < kN; ++k) x[i + k] = v.v[k];
  }
}

// A warp to 512 bytes of columns of a chunk whose last row goes on: the row's parts in order.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) join_kernel(const uint32_t* keys, int n, int V, int d, int slabs, float scale,
                                                        T* dtable, float* total, const float* part) {
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const int chunk = (int)(w / slabs), j = ((int)(w % slabs) * 32 + lane) * VEC;
  const int end = (chunk + 1) * kChunk;
  await_before();
  start_next();
  if (end >= n) return;
  const uint32_t key = keys[end - 1];
  if (key >= (uint32_t)V || keys[end] != key) return;
  const int first = chunk * kChunk;
  if (keys[first] == key && first > 0 && keys[first - 1] == key) return;  // it began before
  float sum[VEC];
  if (j < d) load_sum<VEC>(part + ((int64_t)chunk * 2 + 1) * d + j, sum);
  constexpr int kAhead = 8;
  for (int c = chunk + 1, more = 32; more == 32; c += 32) {
    // how many of the next 32 chunks begin with the row
    const int at = c + lane;
    more = __popc(__ballot_sync(0xffffffffu, (int64_t)at * kChunk < n && keys[at * kChunk] == key));
    for (int i0 = 0; i0 < more; i0 += kAhead) {
      float x[kAhead][VEC];
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (i0 + i < more && j < d) load_sum<VEC>(part + (int64_t)(c + i0 + i) * 2 * d + j, x[i]);
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (i0 + i < more)
#pragma unroll
          for (int k = 0; k < VEC; ++k) sum[k] += x[i][k];
    }
  }
  if (j < d) write_row<T, VEC>(dtable, total, (int64_t)key * d + j, sum, scale);
}

// The batches' sums in the table's type.
template <typename T>
__global__ void __launch_bounds__(kThreads) scale_kernel(const float* total, int64_t all, float scale, T* dtable) {
  await_before();
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < all; i += (int64_t)gridDim.x * kThreads)
    dtable[i] = Elem<T>::put(total[i] * scale);
}

// ------------------------------------------------------------------- host
struct Scratch {
  uint32_t *keys, *order;
  float *part, *total;
  size_t used = 0;
  Scratch(void* at, int64_t n, int32_t V, int32_t d) {
    const int64_t batch = std::min(n, kBatch);
    auto take = [&](int64_t bytes) {
      char* p = static_cast<char*>(at) + used;
      used += (size_t)((bytes + 15) / 16 * 16);
      return p;
    };
    keys = reinterpret_cast<uint32_t*>(take(batch * 4));
    order = reinterpret_cast<uint32_t*>(take(batch * 4));
    part = reinterpret_cast<float*>(take((batch + kChunk - 1) / kChunk * 2 * d * 4));
    total = n > kBatch ? reinterpret_cast<float*>(take((int64_t)V * d * 4)) : nullptr;
  }
};

// f(elements of a piece): the most, up to 16 bytes, that divide a row, where the rows of both
// matrices begin at such pieces (16384 x 770 in bf16, lookup and gradient: 66 us, by single
// elements 82; x 772 54 and 81).
template <typename T, typename F>
int with_piece(const void* a, int64_t lda, const void* b, int d, F&& f) {
  auto fits = [&](int n) {
    return d % n == 0 && lda % n == 0 && aligned_to(a, n * sizeof(T)) && aligned_to(b, n * sizeof(T));
  };
  if constexpr (sizeof(T) == 2)
    if (fits(8)) return f(std::integral_constant<int, 8>{});
  if (fits(4)) return f(std::integral_constant<int, 4>{});
  return fits(2) ? f(std::integral_constant<int, 2>{}) : f(std::integral_constant<int, 1>{});
}

int launch_sort(Ids ids, int64_t first, int n, int V, const Scratch& s, cudaStream_t st) {
  int bits = 1;
  while (V >> bits) ++bits;  // keys go up to V
  // 2048 tokens a CTA where there are few (lookup and gradient of 5000 tokens: 34 us, 40 with
  // 8192 a CTA)
  int ctas = 1;
  while (ctas < kMaxCluster && ctas * 2048 < n) ctas *= 2;
  const void* fn = (const void*)sort_kernel;
  if (int rc = ensure_smem_attr(fn, sizeof(SortShared))) return rc;
  if (ctas > 8 && cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
    return CB_ERR_CUDA;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = sizeof(SortShared);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, sort_kernel, ids, first, n, V, (bits + 7) / 8, s.keys, s.order) != cudaSuccess) {
    (void)cudaGetLastError();
    return CB_ERR_CUDA;
  }
  count_launch();
  return CB_OK;
}

template <typename T, int VEC>
int grad(const T* g, int64_t ldg, Ids ids, int64_t n, int V, int d, float scale, T* dtable, const Scratch& s,
         cudaStream_t st) {
  if (s.total && cudaMemsetAsync(s.total, 0, (size_t)V * d * 4, st) != cudaSuccess) return CB_ERR_CUDA;
  const int slabs = ceil_div(d, 32 * VEC);
  for (int64_t first = 0; first < n; first += kBatch) {
    const int m = (int)std::min(kBatch, n - first);
    if (int rc = launch_sort(ids, first, m, V, s, st)) return rc;
    const int64_t sums = (int64_t)ceil_div(m, kChunk) * slabs, warps = sums + (s.total ? 0 : ceil_div(V, 32));
    constexpr int kWarps = kThreads / 32;
    if (int rc = launch_after(sum_kernel<T, VEC>, dim3((unsigned)((warps + kWarps - 1) / kWarps)), kThreads, 0, st,
                              g + first * ldg, ldg, s.keys, s.order, m, V, d, slabs, scale, dtable, s.total, s.part))
      return rc;
    if (m <= kChunk) continue;
    if (int rc = launch_after(join_kernel<T, VEC>, dim3((unsigned)((sums + kWarps - 1) / kWarps)), kThreads, 0, st, s.keys,
                              m, V, d, slabs, scale, dtable, s.total, s.part))
      return rc;
  }
  if (!s.total) return CB_OK;
  return launch_after(scale_kernel<T>, dim3(8 * num_sms()), kThreads, 0, st, s.total, (int64_t)V * d, scale, dtable);
}

}  // namespace
}  // namespace cb

using namespace cb;

extern "C" int cb_embedding(const void* table, int32_t dtype, int64_t ld, int32_t V, int32_t d, const void* ids,
                            int32_t ids_64, int64_t n, float scale, void* out, int32_t* status, void* stream) {
  if (!table || !ids || !out || V <= 0 || d <= 0 || n <= 0 || (V > 1 && ld < d) || !is_dtype(dtype) ||
      !std::isfinite(scale))
    return CB_ERR_ARG;
  const int size = dtype_size(dtype);
  if (!aligned_to(table, size) || !aligned_to(out, size) || !aligned_to(ids, ids_64 ? 8 : 4)) return CB_ERR_ARG;
  if (n > CB_ENDS_MAX_ROWS || V > CB_ENDS_MAX_VOCAB || d > CB_ENDS_MAX_DIM) return CB_ERR_SHAPE;
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto vec) {
      constexpr int VEC = decltype(vec)::value;
      const int64_t all = n * (d / VEC);
      const int64_t ctas = (all + kPieces * kThreads - 1) / (kPieces * kThreads);
      return launch_after(embedding_kernel<T, VEC>, dim3((unsigned)ctas), kThreads, 0, (cudaStream_t)stream,
                          static_cast<const T*>(table), ld, V, d / VEC, Ids{ids, ids_64},
                          all, scale, static_cast<T*>(out), status);
    };
    return with_piece<T>(table, V == 1 ? 0 : ld, out, d, go);
  });
}

extern "C" size_t cb_embedding_grad_scratch_bytes(int64_t n, int32_t V, int32_t d) {
  if (n <= 0 || V <= 0 || d <= 0 || n > CB_ENDS_MAX_ROWS || V > CB_ENDS_MAX_VOCAB || d > CB_ENDS_MAX_DIM) return 0;
  return Scratch(nullptr, n, V, d).used;
}

extern "C" int cb_embedding_grad(const void* g, int32_t dtype, int64_t ldg, const void* ids, int32_t ids_64, int64_t n,
                                 int32_t V, int32_t d, float scale, void* dtable, void* scratch, size_t scratch_bytes,
                                 void* stream) {
  if (!g || !ids || !dtable || !scratch || V <= 0 || d <= 0 || n <= 0 || ldg < 0 || !is_dtype(dtype) ||
      !std::isfinite(scale))
    return CB_ERR_ARG;
  const int size = dtype_size(dtype);
  if (!aligned_to(g, size) || !aligned_to(dtable, size) || !aligned_to(ids, ids_64 ? 8 : 4) || !aligned_to(scratch, 16))
    return CB_ERR_ARG;
  if (!cb_embedding_grad_scratch_bytes(n, V, d)) return CB_ERR_SHAPE;
  const Scratch s(scratch, n, V, d);
  if (scratch_bytes < s.used) return CB_ERR_WORKSPACE;
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto vec) {
      return grad<T, decltype(vec)::value>(static_cast<const T*>(g), ldg, Ids{ids, ids_64}, n, V, d, scale,
                                           static_cast<T*>(dtable), s, (cudaStream_t)stream);
    };
    return with_piece<T>(g, ldg, dtable, d, go);
  });
}
