// Internal interface of the 8-bit cache inside the forward (kv8_model.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "cirrus_b200.h"

namespace cb {

struct Kv8HeadsParams {
  const float* proj;      // row b * src_T + t, heads from column 0
  int ldp, src_T;
  int rows, T;            // rows b * T + t
  int heads, hd, rot2;
  const int32_t* pos;     // position pos[b] + offset + t
  int offset;
  const float* norm;
  const float* inv_freq;
  float eps;
  float* out;             // [rows][heads][hd]
};

int launch_kv8_heads(const Kv8HeadsParams& p, cudaStream_t st);
int launch_kv8_gate(const float* o, const float* gate, int ldg, int rows, int heads, int hd, float* out, int ldo,
                    cudaStream_t st);
int launch_kv8_slots(const int32_t* slots, int batch, int offset, int32_t* at, cudaStream_t st);
int kv8_check(const CbKv8* c);

}  // namespace cb
