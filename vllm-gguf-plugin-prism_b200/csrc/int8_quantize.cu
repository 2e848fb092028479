// Rows of floats to 8-bit integers with one scale a row:  a = max |x|,  scale = a / 127,  code = x * 127 / a, halves to even.
// The same kernel serves a token's activations, an expert's hidden rows and, once, a weight matrix.
//
// The codes are those of exact arithmetic.  x * (127 / a) with the quotient in fp32 is off by less than 2^-17; within 2^-14 of a half
// the side is settled exactly (i8q_codes).  16-bit inputs hit halves all the time (x = a / 2 is code 63.5).  A row with an infinity or a NaN has no scale: it gets NaN for one and codes of 0,
// so that every result it enters is NaN.
//
// Bound by memory: a row is read once, into registers (up to 64 values a thread), and written once (copies of it as often as asked).
#include "common.cuh"
#include "int8.cuh"

namespace gguf_b200 {

constexpr int I8Q_UNIT = 16;   // values a thread handles at a time: one 16-byte store of codes

template <typename T, bool VEC>
__device__ __forceinline__ void i8q_load(const T* __restrict__ x, int64_t k, int64_t at, T (&v)[I8Q_UNIT]) {
  if (VEC && at + I8Q_UNIT <= k) {
#pragma unroll
    for (int i = 0; i < I8Q_UNIT * (int)sizeof(T) / 16; ++i) reinterpret_cast<uint4*>(v)[i] = __ldg(reinterpret_cast<const uint4*>(x + at) + i);
  } else {
#pragma unroll
    for (int i = 0; i < I8Q_UNIT; ++i) v[i] = at + i < k ? x[at + i] : from_float<T>(0.f);
  }
}
// Largest absolute value so far, as the bit pattern of T (of two values side by side for 16-bit types): infinity and NaN above all numbers
template <typename T> __device__ __forceinline__ uint32_t i8q_top(const T (&v)[I8Q_UNIT], uint32_t top) {
#pragma unroll
  for (int i = 0; i < I8Q_UNIT * (int)sizeof(T) / 4; ++i) {
    const uint32_t w = reinterpret_cast<const uint32_t*>(v)[i];
    top = sizeof(T) == 4 ? max(top, w & 0x7fffffffu) : __vmaxu2(top, w & 0x7fff7fffu);
  }
  return top;
}
template <typename T> __device__ __forceinline__ uint32_t i8q_top_bits(uint32_t top) {   // as the pattern of an fp32 number
  if (sizeof(T) == 4) return top;
  const unsigned short b = (unsigned short)max(top & 0xffffu, top >> 16);
  return __float_as_uint(to_float<T>(*reinterpret_cast<const T*>(&b))) & 0x7fffffffu;
}
// Four codes, a byte each.  1.5 * 2^23 added in one fused step rounds x / scale to an integer in the low bits; what was rounded away says
// whether a half is near, which is settled exactly: the sign of 254 |x| - (2 m + 1) a, m + 1/2 being the half, from two products and
// their rounding errors (the products are within a few ulp of one another, so their difference is exact).
__device__ __forceinline__ uint32_t i8q_codes(const float (&x)[4], float inv, float a) {
  constexpr float MAGIC = 12582912.f;
  float r[4], off = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[i] = fmaf(x[i], inv, MAGIC);
    off = fmaxf(off, fabsf(fmaf(x[i], inv, MAGIC - r[i])));
  }
  if (off > 0.5f - 0x1p-14f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float u = fabsf(x[i]), t = u * inv, m = floorf(t);
      if (fabsf(t - m - 0.5f) < 0x1p-13f) {
        const float h = 2.f * m + 1.f, p = 254.f * u, q = h * a;
        const float d = (p - q) + (fmaf(254.f, u, -p) - fmaf(h, a, -q));
        const float c = d > 0.f || (d == 0.f && ((int)m & 1)) ? m + 1.f : m;
        r[i] = MAGIC + copysignf(c, x[i]);
      }
    }
  }
  const uint32_t lo = __byte_perm(__float_as_uint(r[0]), __float_as_uint(r[1]), 0x0040), hi = __byte_perm(__float_as_uint(r[2]), __float_as_uint(r[3]), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}
// Sixteen codes; lift is 1 but for rows whose largest value is near the ends of fp32's range
template <typename T> __device__ __forceinline__ uint4 i8q_unit(const T (&v)[I8Q_UNIT], float lift, float inv, float a) {
  uint32_t w[4];
  if (lift == 1.f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x[4] = {to_float<T>(v[4 * i]), to_float<T>(v[4 * i + 1]), to_float<T>(v[4 * i + 2]), to_float<T>(v[4 * i + 3])};
      w[i] = i8q_codes(x, inv, a);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x[4] = {to_float<T>(v[4 * i]) * lift, to_float<T>(v[4 * i + 1]) * lift, to_float<T>(v[4 * i + 2]) * lift, to_float<T>(v[4 * i + 3]) * lift};
      w[i] = i8q_codes(x, inv, a);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
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
// beyond is read again
template <typename T, bool VEC, int LANES, int HOLD>
__global__ void __launch_bounds__(256, VEC ? (HOLD * sizeof(T) <= 4 ? 5 : HOLD * sizeof(T) <= 8 ? 4 : 2) : 2) i8_quantize_kernel(const I8Quantize p) {
  __shared__ uint32_t s_top[8];
  const int lane = threadIdx.x % LANES;
  pdl_wait();
  pdl_trigger();
  const int64_t rows = p.n_used ? *p.n_used : p.rows;
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
      if (at < k) i8q_load<T, VEC>(x, k, at, v[h]);
    }
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
      __syncthreads();
      if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
      __syncthreads();
      const int w0 = (int)threadIdx.x / LANES * (LANES / 32);
      top = s_top[w0];
#pragma unroll
      for (int i = 1; i < LANES / 32; ++i) top = max(top, s_top[w0 + i]);
    }
    const bool finite = top < 0x7f800000u;
    const float a0 = __uint_as_float(top), lift = a0 < 0x1p-90f ? 0x1p64f : a0 > 0x1p100f ? 0x1p-64f : 1.f;   // (so that 127 / a and 254 a stay in range)
    const float a = a0 * lift, inv = finite && top != 0 ? 127.f / a : 0.f, scale = finite ? a0 / 127.f : __uint_as_float(0x7fc00000u);
    const int copies = p.scatter ? p.copies : 1;
    uint4 c[HOLD];
#pragma unroll
    for (int h = 0; h < HOLD; ++h) c[h] = finite ? i8q_unit<T>(v[h], lift, inv, a) : make_uint4(0, 0, 0, 0);
#pragma unroll 4
    for (int j = 0; j < copies; ++j) {
      const int64_t o = !live ? -1 : p.scatter ? (int64_t)__ldg(p.scatter + r * copies + j) : r;
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
      const uint4 w = finite ? i8q_unit<T>(u, lift, inv, a) : make_uint4(0, 0, 0, 0);
      for (int j = 0; j < copies; ++j) {
        const int64_t o = p.scatter ? (int64_t)__ldg(p.scatter + r * copies + j) : r;
        if (o >= 0) i8q_store(w, p.q + o * p.ldq, k, at);
      }
    }
  }
}

template <typename T, bool VEC, int LANES, int HOLD> static cudaError_t i8_quantize_form(const I8Quantize& a, cudaStream_t stream) {
  const int per = 256 / LANES;
  const int64_t blocks = (a.rows + per - 1) / per, most = 148 * 64;
  return launch_pdl(i8_quantize_kernel<T, VEC, LANES, HOLD>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, stream, a);
}
template <typename T, bool VEC> static cudaError_t i8_quantize_rows(const I8Quantize& a, cudaStream_t stream) {
  if (a.k <= 32 * I8Q_UNIT) return i8_quantize_form<T, VEC, 32, 1>(a, stream);
  if (a.k <= 64 * I8Q_UNIT) return i8_quantize_form<T, VEC, 64, 1>(a, stream);
  if (a.k <= 128 * I8Q_UNIT) return i8_quantize_form<T, VEC, 128, 1>(a, stream);
  if (a.k <= 256 * I8Q_UNIT) return i8_quantize_form<T, VEC, 256, 1>(a, stream);
  if (a.k <= 512 * I8Q_UNIT) return i8_quantize_form<T, VEC, 256, 2>(a, stream);
  return i8_quantize_form<T, VEC, 256, 4>(a, stream);
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
