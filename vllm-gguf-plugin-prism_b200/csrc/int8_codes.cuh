// The codes of a row of floats (int8_quantize.cu, and the product of a few tokens, which makes them itself, int8.cu).
//
// Codes are those of exact arithmetic.  16-bit values: y = 127 x is exact in fp32, and a quotient y / a that is not a half is off by 2^-19 of
// itself at least (y has 18 bits, a 11), so the quotient with one correction step, right to 2^-23 and exact where it is a half, settles
// it; halves are common (x = a / 2 is code 63.5; of bf16 values one in three hundred).  fp32 values: within 2^-14 of a half the side is
// settled by exact products (i8q_exact).
#pragma once

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
__device__ __forceinline__ uint32_t i8q_pack(float r0, float r1, float r2, float r3) {   // the lowest bytes
  return __byte_perm(__byte_perm(__float_as_uint(r0), __float_as_uint(r1), 0x0040), __byte_perm(__float_as_uint(r2), __float_as_uint(r3), 0x0040), 0x5410);
}
// Two fp32 numbers side by side, rounded to nearest as one by one.  (With one to an instruction 28672x8192 fp16 had 83 % of the issue slots
// taken: 109 us; with two 105.7.  fp32 195 and 193.5.)
__device__ __forceinline__ uint64_t i8q_two(float a, float b) { return (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a); }
__device__ __forceinline__ uint64_t i8q_mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t i8q_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t i8q_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
constexpr float I8Q_MAGIC = 12582912.f;   // 1.5 * 2^23: added to a small number, it leaves its integer in the low bits
// The code of u = |x| (a lifted into fp32's middle): m or m + 1 by the sign of 254 u - (2 m + 1) a, from two products and their rounding
// errors (the products are within a few ulp of one another where it matters, so their difference is exact).
__device__ __forceinline__ float i8q_exact(float x, float inv, float a) {
  const float u = fabsf(x), t = u * inv, m = floorf(t);
  float c = rintf(t);
  if (fabsf(t - m - 0.5f) < 0x1p-13f) {
    const float h = 2.f * m + 1.f, p = 254.f * u, q = h * a;
    const float d = (p - q) + (fmaf(254.f, u, -p) - fmaf(h, a, -q));
    c = d > 0.f || (d == 0.f && ((int)m & 1)) ? m + 1.f : m;
  }
  return I8Q_MAGIC + copysignf(c, x);
}
// (one copy of the code that is hardly ever run: unrolled into every group of four, fetching it cost more than running it)
static __device__ __noinline__ uint32_t i8q_exact4(float x0, float x1, float x2, float x3, float lift, float inv, float a) {
  return i8q_pack(i8q_exact(x0 * lift, inv, a), i8q_exact(x1 * lift, inv, a), i8q_exact(x2 * lift, inv, a), i8q_exact(x3 * lift, inv, a));
}
// What the codes of a row go by; a is lifted (by a power of two, exactly) so that 127 / a and 254 a stay in range
struct I8Row {
  float a, inv, r, lift, y;   // 127 / a, 1 / a (both to a few units in the last place), 127 * lift
};
__device__ __forceinline__ I8Row i8q_row(float a) {
  I8Row w;
  w.lift = a < 0x1p-90f ? 0x1p64f : a > 0x1p100f ? 0x1p-64f : 1.f;
  w.a = a * w.lift;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(w.r) : "f"(w.a));
  w.inv = 127.f * w.r;
  w.y = 127.f * w.lift;
  return w;
}
// Sixteen codes, a byte each.  The number 1.5 * 2^23 added to a quotient rounds it to an integer; for fp32 in one fused step with the
// product, and what was rounded away says whether a half is near.
template <typename T> __device__ __forceinline__ uint4 i8q_unit(const T (&v)[I8Q_UNIT], const I8Row& p) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x[4], r[4];
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const uint64_t y = i8q_mul2(i8q_two(to_float<T>(v[4 * i + j]), to_float<T>(v[4 * i + j + 1])), i8q_two(p.y, p.y)), recip = i8q_two(p.r, p.r);
        const uint64_t q = i8q_mul2(y, recip), code = i8q_add2(i8q_fma2(i8q_fma2(q, i8q_two(-p.a, -p.a), y), recip, q), i8q_two(I8Q_MAGIC, I8Q_MAGIC));
        r[j] = __uint_as_float((uint32_t)code);
        r[j + 1] = __uint_as_float((uint32_t)(code >> 32));
      }
      w[i] = i8q_pack(r[0], r[1], r[2], r[3]);
    } else {
      float off = p.lift == 1.f ? 0.f : 1.f;
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        x[j] = to_float<T>(v[4 * i + j]);
        x[j + 1] = to_float<T>(v[4 * i + j + 1]);
        const uint64_t two = i8q_two(x[j], x[j + 1]), inv = i8q_two(p.inv, p.inv), magic = i8q_two(I8Q_MAGIC, I8Q_MAGIC), code = i8q_fma2(two, inv, magic);
        const uint64_t rest = i8q_fma2(two, inv, i8q_fma2(code, i8q_two(-1.f, -1.f), magic));
        r[j] = __uint_as_float((uint32_t)code);
        r[j + 1] = __uint_as_float((uint32_t)(code >> 32));
        off = fmaxf(off, fmaxf(fabsf(__uint_as_float((uint32_t)rest)), fabsf(__uint_as_float((uint32_t)(rest >> 32)))));
      }
      w[i] = off > 0.5f - 0x1p-14f ? i8q_exact4(x[0], x[1], x[2], x[3], p.lift, p.inv, p.a) : i8q_pack(r[0], r[1], r[2], r[3]);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

}  // namespace gguf_b200
