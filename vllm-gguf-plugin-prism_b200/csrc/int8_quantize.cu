// Rows of floats to 8-bit integers with one scale a row:  a = max |x|,  scale = a / 127,  code = x * 127 / a, halves to even.
// The same kernel serves a token's activations, an expert's hidden rows and, once, a weight matrix.
//
// How the codes are made exact: int8_codes.cuh.  A row with an infinity or a NaN has no scale: it gets NaN for one and codes of 0, so that
// every result it enters is NaN.
//
// Bound by memory: a row is read once, into registers (up to 64 values a thread), and written once (copies of it as often as asked).
// 28672x8192 fp16 in 106 us, 6.6 TB/s, the copy rate (two thirds of the bytes are read; 309 with codes by fp64 comparisons and 100 registers a
// thread); fp32 in 194, 6.1 TB/s.
#include "int8_codes.cuh"

namespace gguf_b200 {

__device__ __forceinline__ void i8q_store(uint4 c, int8_t* __restrict__ q, int64_t k, int64_t at) {
  if (at + I8Q_UNIT <= k) {
    *reinterpret_cast<uint4*>(q + at) = c;
  } else {
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int i = 0; i < I8Q_UNIT; ++i)
      if (at + i < k) q[at + i] = (int8_t)(w[i / 4] >> (8 * (i % 4)));
  }
}

// LANES threads a row, 256 / LANES rows a block; HOLD units of a thread stay in registers between the maximum and the codes, what is
// beyond is read again.  AHEAD: a block that walks over many rows asks for the next one while it makes this one's codes.  SCATTER:
// see I8Quantize::scatter.
template <typename T, bool VEC, int LANES, int HOLD, bool AHEAD, bool SCATTER>
__global__ void __launch_bounds__(256, VEC ? (HOLD * sizeof(T) <= 4 && !AHEAD ? 5 : HOLD * sizeof(T) <= 8 ? 4 : 2) : 2) i8_quantize_kernel(const I8Quantize p) {
  __shared__ uint32_t s_top[2][8];
  int turn = 0;
  const int lane = threadIdx.x % LANES;
  pdl_wait();
  pdl_trigger();
  const int64_t rows = p.n_used ? *p.n_used : p.rows;
  T next[AHEAD ? HOLD : 1][I8Q_UNIT];
  auto ask = [&](int64_t row) {
    const T* x = static_cast<const T*>(p.x) + (row < rows ? row : 0) * p.ldx;
    const int64_t k = row < rows ? p.k : 0;
#pragma unroll
    for (int h = 0; h < (AHEAD ? HOLD : 0); ++h) {
      const int64_t at = (int64_t)(h * LANES + lane) * I8Q_UNIT;
      if (at < k) i8q_load<T, VEC>(x, k, at, next[h]);
    }
  };
  ask((int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES);
  for (int64_t r0 = (int64_t)blockIdx.x * (256 / LANES); r0 < rows; r0 += (int64_t)gridDim.x * (256 / LANES)) {
    const int64_t r = r0 + threadIdx.x / LANES;
    const bool live = r < rows;
    const T* x = static_cast<const T*>(p.x) + (live ? r : 0) * p.ldx;
    const int64_t k = live ? p.k : 0;
    T v[HOLD][I8Q_UNIT];
    uint32_t top = 0;
#pragma unroll
    for (int h = 0; h < HOLD; ++h) {
      const int64_t at = (int64_t)(h * LANES + lane) * I8Q_UNIT;
      if (AHEAD) {
#pragma unroll
        for (int i = 0; i < I8Q_UNIT; ++i) v[h][i] = next[AHEAD ? h : 0][i];
      } else if (at < k) {
        i8q_load<T, VEC>(x, k, at, v[h]);
      }
    }
    ask(r + (int64_t)gridDim.x * (256 / LANES));
    const int copies = SCATTER ? p.copies : 1;
    int place = -1;   // of the first 32 copies, a lane each
    if (SCATTER && live && (int)(threadIdx.x & 31) < copies) place = __ldg(p.scatter + r * copies + (threadIdx.x & 31));
#pragma unroll
    for (int h = 0; h < HOLD; ++h)
      if ((int64_t)(h * LANES + lane) * I8Q_UNIT < k) top = i8q_top<T>(v[h], top);
    for (int64_t at = (int64_t)(HOLD * LANES + lane) * I8Q_UNIT; at < k; at += LANES * I8Q_UNIT) {
      T u[I8Q_UNIT];
      i8q_load<T, VEC>(x, k, at, u);
      top = i8q_top<T>(u, top);
    }
    top = __reduce_max_sync(0xffffffffu, i8q_top_bits<T>(top));
    if (LANES > 32) {
      uint32_t* st = s_top[turn];   // (in turn: whoever has passed this barrier is done with the last row's)
      turn ^= 1;
      if ((threadIdx.x & 31) == 0) st[threadIdx.x >> 5] = top;
      __syncthreads();
      const int w0 = (int)threadIdx.x / LANES * (LANES / 32);
      top = st[w0];
#pragma unroll
      for (int i = 1; i < LANES / 32; ++i) top = max(top, st[w0 + i]);
    }
    const bool finite = top < 0x7f800000u, zero = !finite || top == 0;
    const float a = __uint_as_float(top), scale = finite ? a / 127.f : __uint_as_float(0x7fc00000u);
    const I8Row w = i8q_row(zero ? 1.f : a);
    uint4 c[HOLD];
#pragma unroll
    for (int h = 0; h < HOLD; ++h) c[h] = zero ? make_uint4(0, 0, 0, 0) : i8q_unit<T>(v[h], w);
#pragma unroll 4
    for (int j = 0; j < copies; ++j) {
      const int64_t o = !live ? -1 : !SCATTER ? r : j < 32 ? __shfl_sync(0xffffffffu, place, j) : __ldg(p.scatter + r * copies + j);
      if (o < 0) continue;
      if (lane == 0) p.scale[o] = scale;
#pragma unroll
      for (int h = 0; h < HOLD; ++h) {
        const int64_t at = (int64_t)(h * LANES + lane) * I8Q_UNIT;
        if (at < k) i8q_store(c[h], p.q + o * p.ldq, k, at);
      }
    }
    for (int64_t at = (int64_t)(HOLD * LANES + lane) * I8Q_UNIT; at < k; at += LANES * I8Q_UNIT) {
      T u[I8Q_UNIT];
      i8q_load<T, VEC>(x, k, at, u);
      const uint4 c = zero ? make_uint4(0, 0, 0, 0) : i8q_unit<T>(u, w);
      for (int j = 0; j < copies; ++j) {
        const int64_t o = SCATTER ? (int64_t)__ldg(p.scatter + r * copies + j) : r;
        if (o >= 0) i8q_store(c, p.q + o * p.ldq, k, at);
      }
    }
  }
}

// Rows ahead cost a block of five on an SM, so they are for 16-bit rows that fill the GPU many times over: 28672x8192 110 us (122 without),
// 28672x4096 61.8 (64.8), 60000x1024 33.6 (33.1), all with one number to an instruction (int8_codes.cuh), but 4096x4096 12.2 (10.5); in fp32 28672x8192 279 (233).  At most 16 blocks an SM walk over the
// rest: rows that are read by single values, 100000x500, 84 us (95 with 64).  Rows that go to places have a kernel of their own: without it the
// others took longer (fp32 28672x8192 235, fp16 4096x4096 10.5 instead of 10.0), and so did a place looked up only when it is written to.
template <typename T, bool VEC, int LANES, int HOLD> static cudaError_t i8_quantize_form(const I8Quantize& a, cudaStream_t stream) {
  const int per = 256 / LANES;
  const int64_t blocks = (a.rows + per - 1) / per, most = 148 * 16;
  if (a.scatter) return launch_pdl(i8_quantize_kernel<T, VEC, LANES, HOLD, false, true>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, stream, a);
  if constexpr (VEC && sizeof(T) == 2 && HOLD == 2)
    if (blocks >= 148 * 32) return launch_pdl(i8_quantize_kernel<T, VEC, LANES, HOLD, true, false>, dim3(148 * 16), dim3(256), 0, stream, a);
  return launch_pdl(i8_quantize_kernel<T, VEC, LANES, HOLD, false, false>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, stream, a);
}
// Two units a thread where there are rows enough to fill the GPU; a block a row where there are not.  Rows that go to places, whose copies take
// longest, have a unit a thread (2048 rows of 2048 to eight places 9.6 us, 10.6 with two; hidden rows of 1024 in fp32 22.6, but 20.8 with two).
template <typename T, bool VEC> static cudaError_t i8_quantize_rows(const I8Quantize& a, cudaStream_t stream) {
  if (a.k > 512 * I8Q_UNIT) return i8_quantize_form<T, VEC, 256, 4>(a, stream);
  if (a.k > 256 * I8Q_UNIT) return i8_quantize_form<T, VEC, 256, 2>(a, stream);
  if (a.rows < 148 * 4) return i8_quantize_form<T, VEC, 256, 1>(a, stream);
  if (a.scatter && a.k > 128 * I8Q_UNIT) return i8_quantize_form<T, VEC, 256, 1>(a, stream);
  if (a.scatter && a.k > 64 * I8Q_UNIT) return i8_quantize_form<T, VEC, 128, 1>(a, stream);
  if (a.scatter) return i8_quantize_form<T, VEC, 64, 1>(a, stream);
  if (a.k > 128 * I8Q_UNIT) return i8_quantize_form<T, VEC, 128, 2>(a, stream);
  if (a.k > 64 * I8Q_UNIT) return i8_quantize_form<T, VEC, 64, 2>(a, stream);
  return i8_quantize_form<T, VEC, 32, 2>(a, stream);
}
template <typename T> static int i8_quantize_typed(const I8Quantize& a, cudaStream_t stream) {
  const bool vec = (reinterpret_cast<uintptr_t>(a.x) & 15) == 0 && a.ldx * (int64_t)sizeof(T) % 16 == 0;
  const cudaError_t e = vec ? i8_quantize_rows<T, true>(a, stream) : i8_quantize_rows<T, false>(a, stream);
  return e == cudaSuccess ? E_OK : E_CUDA;
}

int launch_i8_quantize(const I8Quantize& a, cudaStream_t stream) {
  if (a.rows == 0) return E_OK;
  switch (a.dtype) {
    case DT_F32: return i8_quantize_typed<float>(a, stream);
    case DT_F16: return i8_quantize_typed<__half>(a, stream);
    case DT_BF16: return i8_quantize_typed<__nv_bfloat16>(a, stream);
  }
  return E_BAD_DTYPE;
}

}  // namespace gguf_b200
