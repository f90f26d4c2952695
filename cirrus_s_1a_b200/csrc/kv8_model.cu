// The 8-bit cache inside the forward (cb_forward_kv8): heads prepared for it, and
// the gate behind its attention.
#include "kv8.cuh"
#include "kv8_model.cuh"

namespace cb {
namespace {

// RMSNorm and RoPE of one head per warp (layers.py:72-82, 325-331), keys or queries.
__global__ void __launch_bounds__(256) kv8_heads_kernel(const __grid_constant__ Kv8HeadsParams p) {
  const int item = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (item >= p.rows * p.heads) return;
  const int r = item / p.heads, h = item % p.heads, b = r / p.T, t = r % p.T;
  const int position = p.pos[b] + p.offset + t;
  const float* x = p.proj + ((int64_t)b * p.src_T + t) * p.ldp + h * p.hd;
  float ss = 0.0f;
  for (int j = lane; j < p.hd; j += 32) ss += x[j] * x[j];
  const float rn = rsqrtf(warp_sum(ss) / (float)p.hd + p.eps);
  for (int j = lane; j < p.hd / 2; j += 32) {
    float x1 = x[2 * j] * rn * p.norm[2 * j], x2 = x[2 * j + 1] * rn * p.norm[2 * j + 1];
    if (j < p.rot2) rope_pair(x1, x2, position, p.inv_freq[j]);
    reinterpret_cast<float2*>(p.out + (int64_t)item * p.hd)[j] = make_float2(x1, x2);
  }
}

// out[r][h][d] = o[r][h][d] * sigmoid(gate[r][h]) (layers.py:243)
__global__ void __launch_bounds__(256) kv8_gate_kernel(const float* __restrict__ o, const float* __restrict__ gate, int ldg,
                                                       int rows, int heads, int hd, float* __restrict__ out, int ldo) {
  const int i = blockIdx.x * 256 + threadIdx.x, width = heads * hd;
  if (i >= rows * width) return;
  const int r = i / width, c = i % width;
  out[(int64_t)r * ldo + c] = o[i] * sigmoid(gate[(int64_t)r * ldg + c / hd]);
}

// at[b] = slots[b] + offset
__global__ void kv8_slots_kernel(const int32_t* slots, int batch, int offset, int32_t* at) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b < batch) at[b] = slots[b] + offset;
}

}  // namespace

int launch_kv8_heads(const Kv8HeadsParams& p, cudaStream_t st) {
  kv8_heads_kernel<<<ceil_div(p.rows * p.heads, 8), 256, 0, st>>>(p);
  count_launch();
  return cudaGetLastError() == cudaSuccess ? CB_OK : CB_ERR_CUDA;
}

int launch_kv8_gate(const float* o, const float* gate, int ldg, int rows, int heads, int hd, float* out, int ldo,
                    cudaStream_t st) {
  kv8_gate_kernel<<<ceil_div(rows * heads * hd, 256), 256, 0, st>>>(o, gate, ldg, rows, heads, hd, out, ldo);
  count_launch();
  return cudaGetLastError() == cudaSuccess ? CB_OK : CB_ERR_CUDA;
}

int launch_kv8_slots(const int32_t* slots, int batch, int offset, int32_t* at, cudaStream_t st) {
  kv8_slots_kernel<<<ceil_div(batch, 128), 128, 0, st>>>(slots, batch, offset, at);
  count_launch();
  return cudaGetLastError() == cudaSuccess ? CB_OK : CB_ERR_CUDA;
}

}  // namespace cb
