// What the 8-bit integer kernels share: launch parameters (int8.cu) and the scale of a quantized row.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace gguf_b200 {

// Rows of floats -> int8 codes and one scale a row.  gather != null: output row r takes input row gather[r] / gather_div, and only the
// first *n_used rows (null: all) are written.
struct I8Quantize {
  const void* x;             // element type dtype, ldx elements between rows
  int dtype;
  int64_t ldx;
  int8_t* q;                 // ldq bytes between rows, a multiple of 16
  int64_t ldq;
  float* scale;
  int64_t rows, k;
  const int32_t* gather;
  int64_t gather_div;
  const int32_t* n_used;
};
int launch_i8_quantize(const I8Quantize& a, cudaStream_t stream);

// D[n, t] = sum over k of w[n, k] * q[t, k], with one scale a row on both sides.
struct I8Product {
  const int8_t* w;           // [experts * w_rows][ldw]
  int64_t ldw;
  const float* w_scale;      // [experts * w_rows]
  const int8_t* q;           // [m][ldq]
  int64_t ldq;
  const float* q_scale;      // [m]
  void* y;                   // element type dtype, ldy elements between rows
  int64_t ldy;
  int dtype;
  int64_t m, n, k;           // rows of q, rows of the result's other side, values
  const void* bias;          // [n] in dtype, or null
  bool settled;              // w is complete: it may be read while the kernel ahead is still running
  // experts (null passes: dense): work list of launch_moe_plan, pass = {expert, first row of q, rows}
  const void* passes;
  const int32_t* n_passes;
  int64_t experts, max_passes, pass_rows;
  // ... gate and up product: w has n gate rows, then n up rows an expert; y[row] = act(gate) * up in fp32, in the order of q's rows
  int act;                   // 1 silu, 2 gelu; 0: plain product
  // ... plain product: y[sorted[row]] = result * row_scale[sorted[row]]
  const int32_t* sorted;
  const float* row_scale;
  int* status;
};
int launch_i8_product(const I8Product& a, cudaStream_t stream);
int64_t i8_moe_pass_rows(int64_t slots, int64_t experts);

constexpr int64_t I8_MAX_K = 131071;   // 128 * 128 * K < 2^31: no sum of products leaves 32 bits

}  // namespace gguf_b200
