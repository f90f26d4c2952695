// Internal interface of the attention over the 8-bit K/V cache.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "cirrus_b200.h"

namespace cb {

struct Sum;

struct AttendParams {
  CbKv8 c;
  const void* q;
  int dtype;
  int64_t qs[3];        // element strides between sequences, tokens, heads
  bool q_wide;          // q and its strides are multiples of 16 bytes
  int G, T, rows;       // query heads per KV head; rows = T * G of a KV head
  const int32_t* pos;
  const int32_t* counts;
  int limit;            // slots from here on are not seen
  float scale;
  bool add_mass;
  void* out;            // [batch][T][heads][dim], the queries' type
  float* lse;           // [batch][T][heads]
  float* lse2;          // [head][rows], log2 units: for the weights
  int block0;           // decode form: the launch's first block of query rows
  int splits;           // runs: of all heads' blocks (decode form), of each row tile's keys (prompt form)
  // parts: sums (Sum), and values against the same m'.  Decode form: [row block][run + head][row],
  // part_rows of them for each block (the 8, 16 or 32 query rows of a CTA); prompt form:
  // [head][rows][splits].
  int64_t part_rows;
  Sum* part_ml;         // [part]
  float* part_o;        // [part][dim]
  int* arrived;         // [row block of a launch][head]: parts finished; zero between calls
  float* scores;        // [head][rows][ld_scores] in log2 units, or null
  int64_t ld_scores;
  // the prompt form: query rows prepared in 128-row operand tiles, and the factors that undo their scaling
  int row_tiles;
  uint8_t* q16;         // [batch * kv heads][row_tiles][128 * dim * 2 bytes, float32: twice, head and tail]
  float* q_back;        // [batch * kv heads][row_tiles * 128]
  int32_t* status;
};

// A row's sum is taken from P against one value exponent e_ref as long as the blocks'
// exponents lie within kNear of it; what is left of float32's range then holds every P that
// matters to the sum.  A larger exponent becomes e_ref, what was summed so far is put aside
// (shared memory: it is rarely needed); blocks of smaller ones are summed there key by key, since their P may vanish
// beside the others' although their keys weigh as much (zeros have the exponent -100).
constexpr int kNear = 28;

// From here on what the rounding of m' leaves of x + e - m' (up to half its last bit, 2^-4
// here, the same for all keys) would pass f16's range: x + e is rounded before m' is taken
// off, and P ends at 2^kFarMost where the score's last bit is larger than the lags of m'.
// Scores beyond 2^24 are coarser than the value exponents.
constexpr float kFarScore = 1048576.0f, kFarMost = 15.0f;

// Many query rows, head_dim 64 or 128, queries of any type (kv8_prompt.cu).  Writes out
// and lse where splits is 1, parts otherwise.
int kv8_prompt_launch(const AttendParams& p, int bh, cudaStream_t st);
// The rows' attention weights into mass, after lse is complete.
int kv8_prompt_mass_launch(const AttendParams& p, int bh, int longest, cudaStream_t st);

int kv8_check(const CbKv8* c);
bool kv8_dtype_ok(int dtype);

}  // namespace cb
