// What the 8-bit integer kernels share: launch parameters (int8.cu) and the scale of a quantized row.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace gguf_b200 {

// Rows of floats -> int8 codes and one scale a row.  scatter != null: row r goes to the output rows scatter[r * copies + j], j < copies
// (negative: nowhere).  n_used != null: only the first *n_used rows count.
struct I8Quantize {
  const void* x;             // element type dtype, ldx elements between rows
  int dtype;
  int64_t ldx;
  int8_t* q;                 // ldq bytes between rows, a multiple of 16
  int64_t ldq;
  float* scale;
  int64_t rows, k;
  const int32_t* scatter;
  int copies;
  const int32_t* n_used;
};
int launch_i8_quantize(const I8Quantize& a, cudaStream_t stream);

// D[n, t] = sum over k of w[n, k] * q[t, k], with one scale a row on both sides.
struct I8Product {
  const int8_t* w;           // rows ldw bytes apart; experts: one matrix behind the other
  int64_t ldw;
  const float* w_scale;      // one for every row of w
  const int8_t* q;           // [m][ldq]
  int64_t ldq;
  const float* q_scale;      // [m]
  void* y;                   // element type dtype, ldy elements between rows
  int64_t ldy;
  int dtype;
  int64_t m, n, k;           // rows of q, results a row, values
  const void* bias;          // [n] in dtype, or null
  bool settled;              // w is complete: it may be read while the kernel ahead is still running
  // experts (null passes: dense): work list of launch_i8_plan; w was complete before the kernel ahead triggered
  const void* passes;
  const int32_t* n_passes;
  int64_t experts, max_passes, pass_rows;
  // ... gate and up product: w has n gate rows, then n up rows an expert; y[row] = act(gate) * up in fp32, in the order of q's rows
  int act;                   // 1 silu, 2 gelu; 0: down product
  // ... down product: y[sorted[row]], in fp32
  const int32_t* sorted;
  // ... tokens that are not quantized yet (null: q is used; see i8_few): [m][ldx] in dtype
  const void* x;
  int64_t ldx;
  int* status;
};
bool i8_few(const void* x, int dtype, int64_t ldx, int64_t m, int64_t n, int64_t k);
int launch_i8_product(const I8Product& a, cudaStream_t stream);

// The routed expert step around the products (int8_moe.cu)
int64_t i8_moe_pass_rows(int64_t slots, int64_t experts);
int64_t i8_moe_passes(int64_t slots, int64_t experts, int64_t pass_rows);   // room for passes
struct I8Plan {
  const int32_t* topk_ids;
  int64_t slots;
  int experts, pass_rows;
  int32_t* sorted;           // [slots] slots with a valid expert, sorted by it, in their order
  int32_t* place;            // [slots] where in that order a slot is; -1: it has no expert
  void* passes;              // int4 {expert, first row, rows, 0}: an expert's rows in passes of like size, at most pass_rows
  int32_t* n_passes;         // [0] passes, [1] rows
};
int launch_i8_plan(const I8Plan& a, cudaStream_t stream);
struct I8Sum {
  const float* y;            // [slots][h]
  void* out;                 // [tokens][h] in dtype
  const int32_t* place;      // [slots]; negative: the slot has no result
  const float* weights;      // [slots]
  int64_t tokens, top_k, h;
  int dtype;
};
int launch_i8_sum(const I8Sum& a, cudaStream_t stream);

constexpr int64_t I8_MAX_K = 131071;   // 128 * 128 * K < 2^31: no sum of products leaves 32 bits

}  // namespace gguf_b200
