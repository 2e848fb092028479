// Products of 8-bit integers on the tensor cores:  D[n, t] = sum over k of W[n, k] * Q[t, k]  in 32-bit integers (exact, whatever the
// order), and y[t, n] = D * q_scale[t] * w_scale[n] (+ bias) rounded once.
//
// The scales sit on rows, so that nothing has to be done between the first and the last value of a sum: both operands go from memory
// to the tensor core as they are (TMA boxes of 128 rows x 128 bytes, 128-byte swizzle, tcgen05.mma kind::i8, four instructions a
// box).  Weight rows sit on the 128-row side of the instruction, tokens on its column side, any multiple of 16 up to 256; so one
// token costs no more tensor time than sixteen, and what bounds small batches is the weights' way from memory.
//
// A CTA: a loader, an MMA issuer, eight epilogue warps (lane = weight row = lane of tensor memory), over a ring of stages of 128
// values.  Three ways to deal out the work:
//   tiles    a CTA takes items (128 weight rows x up to 256 tokens) a grid apart, two accumulators in turn where they fit
//   split    fewer tiles than SMs: a cluster of 2, 4 or 8 CTAs shares the K of one tile.  Each sends its sums of every other's
//            rows into the other's shared memory, which then adds and stores its rows: no scratch in memory, nothing to clear, and
//            integer sums do not depend on the order
//   experts  items are (pass of an expert's tokens, 128 rows); for the gate and up product two boxes of weights, of the same rows of
//            gate and up, meet the same tokens in two accumulators, so that a thread has both and act(gate) * up never leaves it
//            but as the result
#include <cuda.h>

#include <math.h>

#include "int8.cuh"
#include "kernels.h"
#include "raw_stream.cuh"
#include "tcgen05.cuh"

namespace gguf_b200 {

constexpr int I8_ROWS = 128, I8_BK = 128;                 // weight rows of a box, values (= bytes) of a stage
constexpr int I8_A_BYTES = I8_ROWS * I8_BK;
constexpr int I8_EPI = 8;                                 // epilogue warps
constexpr int I8_THREADS = 128 + 32 * I8_EPI;             // warps 0 loader, 1 MMA issuer, 2 tensor memory, from 4 on epilogue
constexpr int I8_MAX_STAGES = 16;
constexpr int I8_SMS = 148;
constexpr int I8_AUX = 512 + 2 * 256 * 8 + I8_EPI * 1024; // barriers; scale and output row of every token, of two items; 16 tokens x 32 rows a warp

struct I8Params {
  int n, n_up;             // weight rows; distance of the up rows from the gate rows
  int w_rows;              // weight rows of an expert
  int k, nk;               // values, stages
  int m, rt, tt, tn, bh;   // tokens; row tiles, token tiles; tokens a tile; rows of a box of tokens
  int stages, stage_bytes, nbuf, aux_off;
  uint32_t tmem_cols;
  int split;
  void* y;
  int64_t ldy;
  int dtype;
  const float *w_scale, *q_scale;
  const void* bias;
  int settled;
  const int4* passes;
  const int32_t* n_passes;
  int act;
  const int32_t* sorted;
  const float* row_scale;
  int* status;
};

// Four times D[tmem] (+)= A[smem] * B[smem], 32 values (bytes) each: +2 in the descriptors' 16-byte units
__device__ __forceinline__ void umma_i8_ss4(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate, uint32_t lead) {
  asm volatile(
      "{\n\t.reg .pred p, q, t;\n\t.reg .b64 a, b;\n\t.reg .b32 al, bl;\n\t"
      "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
      "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::i8 [%0], a, b, %4, p;\n\t"
      "add.u32 al, %1, 2;\n\tadd.u32 bl, %2, 2;\n\tmov.b64 a, {al, %3};\n\tmov.b64 b, {bl, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::i8 [%0], a, b, %4, t;\n\t"
      "add.u32 al, %1, 4;\n\tadd.u32 bl, %2, 4;\n\tmov.b64 a, {al, %3};\n\tmov.b64 b, {bl, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::i8 [%0], a, b, %4, t;\n\t"
      "add.u32 al, %1, 6;\n\tadd.u32 bl, %2, 6;\n\tmov.b64 a, {al, %3};\n\tmov.b64 b, {bl, %3};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::i8 [%0], a, b, %4, t;\n\t}"
      ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate), "r"(lead)
      : "memory");
}
// kind::i8 instruction descriptor: 32-bit integer sums, both operands signed, K-major, 128 rows, n columns
__device__ __forceinline__ uint32_t i8_idesc(int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(I8_ROWS >> 4) << 24);
}
__device__ __forceinline__ void i8_box(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void i8_box_l2(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float i8_act(int act, float g) { return act == 1 ? g / (1.f + expf(-g)) : 0.5f * g * (1.f + erff(g * 0.70710678f)); }
__device__ __forceinline__ void i8_put(void* y, int dtype, int64_t at, float v) {
  if (dtype == DT_F32) static_cast<float*>(y)[at] = v;
  else if (dtype == DT_F16) static_cast<__half*>(y)[at] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(y)[at] = __float2bfloat16_rn(v);
}
__device__ __forceinline__ float i8_bias(const I8Params& p, int n) {
  if (!p.bias) return 0.f;
  return p.dtype == DT_F32 ? static_cast<const float*>(p.bias)[n]
         : p.dtype == DT_F16 ? __half2float(static_cast<const __half*>(p.bias)[n]) : __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[n]);
}

// Sixteen tokens (f[0 .. count)) of a warp's 32 rows, a lane's row being n: token j goes to row to[j] of y.  fp32 leaves as it is, 128 bytes
// an instruction.  16-bit results go through the warp's kilobyte of shared memory, and from there, where all 32 rows count and
// 16-byte stores are aligned (`wide`), eight tokens an instruction.
template <typename T>
__device__ __forceinline__ void i8_store16(T* __restrict__ y, int64_t ldy, const int* to, int count, const float (&f)[16], int n, int lane, int rows, bool wide,
                                           uint8_t* stage) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < count && lane < rows) y[to[j] * ldy + n] = f[j];
  } else {
    T* st = reinterpret_cast<T*>(stage);
#pragma unroll
    for (int j = 0; j < 16; ++j) st[j * 32 + lane] = from_float<T>(f[j]);
    __syncwarp();
    if (wide) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = 8 * h + (lane >> 2), part = lane & 3;
        const uint4 v = *reinterpret_cast<const uint4*>(stage + j * 64 + part * 16);
        if (j < count) *reinterpret_cast<uint4*>(y + to[j] * ldy + (n - lane + 8 * part)) = v;
      }
    } else if (lane < rows) {
      for (int j = 0; j < count; ++j) y[to[j] * ldy + n] = st[j * 32 + lane];
    }
    __syncwarp();
  }
}

struct I8Item {
  int n0, a_row;           // first row of the tile in its matrix, and in the weights
  int x0, rows;            // tokens
};
__device__ __forceinline__ I8Item i8_item(const I8Params& p, int i) {
  I8Item t;
  if (p.passes) {
    const int4 q = p.passes[i / p.rt];
    t.n0 = i % p.rt * I8_ROWS;
    t.a_row = q.x * p.w_rows + t.n0;
    t.x0 = q.y;
    t.rows = q.z;
  } else {   // the token tiles of a row tile are neighbours
    t.a_row = t.n0 = i / p.tt * I8_ROWS;
    t.x0 = i % p.tt * p.tn;
    t.rows = min(p.tn, p.m - t.x0);
  }
  return t;
}

// NA: boxes of weights a stage (2: gate and up)
template <int NA>
__global__ void __launch_bounds__(I8_THREADS, 2) i8_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap,
                                                           const __grid_constant__ I8Params p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // (from the shared-window address, so that the CTAs of a cluster agree about offsets)
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + p.aux_off);
  uint64_t *full = bars, *empty = bars + I8_MAX_STAGES, *accum = bars + 2 * I8_MAX_STAGES, *drained = accum + 2, *last = accum + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(accum + 5);
  volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* s_scale = reinterpret_cast<float*>(smem + p.aux_off + 512);   // [2][256]
  int* s_row = reinterpret_cast<int*>(s_scale + 512);                  // [2][256]
  uint8_t* s_stage = reinterpret_cast<uint8_t*>(s_row + 512);          // [I8_EPI][1024]
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&accum[s], 1);
      mbar_init(&drained[s], I8_EPI);
    }
    *gave_up = 0;
    fence_barrier_init();
  }
  if (warp == 2) {
    tmem_alloc(tmem_slot, p.tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t rank = p.split > 1 ? cluster_rank() : 0u;
  if (p.split > 1) cluster_sync();
  pdl_trigger();
  const uint32_t tmem = *tmem_slot, gave_up_s = smem_u32(const_cast<const int*>(gave_up)), full_s = smem_u32(full), empty_s = smem_u32(empty);
  const uint32_t accum_s = smem_u32(accum), drained_s = smem_u32(drained);
  const int first = p.split > 1 ? (int)blockIdx.x / p.split : (int)blockIdx.x, step = p.split > 1 ? 1 << 30 : (int)gridDim.x;
  const int kb0 = p.split > 1 ? (int)(p.nk * rank) / p.split : 0, kb1 = p.split > 1 ? (int)(p.nk * (rank + 1)) / p.split : p.nk;
  auto items = [&] { return p.passes ? *p.n_passes * p.rt : p.rt * p.tt; };   // (behind pdl_wait where there are passes)

  if (warp == 0) {
    // ---------------- loader ----------------
    const uint32_t lead = elect_one() ? 1u : 0u, ring = smem_u32(smem);
    int s = 0, ahead = 0;
    uint32_t ph = 0;
    if (!p.passes) {   // the first weights before the activations are there: into the ring, or, if they may still be written, into L2
      const I8Item t = i8_item(p, first);
      ahead = min(p.stages, kb1 - kb0);
      for (int j = 0; j < ahead; ++j)
        if (lead) {
          if (p.settled) {
            mbar_expect_tx(full_s + 8u * j, (uint32_t)(NA * I8_A_BYTES + (t.rows + p.bh - 1) / p.bh * p.bh * I8_BK));
            i8_box(ring + (uint32_t)(j * p.stage_bytes), &amap, (kb0 + j) * I8_BK, t.a_row, full_s + 8u * j);
          } else {
            i8_box_l2(&amap, (kb0 + j) * I8_BK, t.a_row);
          }
        }
      if (!p.settled) ahead = 0;
    }
    pdl_wait();
    const int n = items();
    for (int i = first; i < n; i += step) {
      const I8Item t = i8_item(p, i);
      const int boxes = (t.rows + p.bh - 1) / p.bh;
      for (int kb = kb0; kb < kb1; ++kb) {
        const uint32_t fb = full_s + 8u * s, at = ring + (uint32_t)(s * p.stage_bytes);
        if (ahead == 0) {
          mbar_wait_or(empty_s + 8u * s, ph ^ 1u, gave_up_s);
          if (lds32(gave_up_s) != 0u) goto loaded;   // (no copy into a slot that may be in use)
          __syncwarp();
          if (lead) {
            mbar_expect_tx(fb, (uint32_t)(NA * I8_A_BYTES + boxes * p.bh * I8_BK));
            i8_box(at, &amap, kb * I8_BK, t.a_row, fb);
            if (NA == 2) i8_box(at + I8_A_BYTES, &amap, kb * I8_BK, t.a_row + p.n_up, fb);
          }
        } else {
          --ahead;
        }
        if (lead)
          for (int b = 0; b < boxes; ++b) i8_box(at + (uint32_t)(NA * I8_A_BYTES + b * p.bh * I8_BK), &bmap, kb * I8_BK, t.x0 + b * p.bh, fb);
        if (++s == p.stages) { s = 0; ph ^= 1u; }
      }
    }
  loaded:;
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    const uint32_t lead = elect_one() ? 1u : 0u;
    const uint64_t d0 = umma_desc_sw128(smem_u32(smem));
    const uint32_t lo0 = (uint32_t)d0, hi = (uint32_t)(d0 >> 32), stage16 = (uint32_t)p.stage_bytes >> 4;
    int s = 0, buf = 0;
    uint32_t ph = 0, dph = 0;
    if (p.passes) pdl_wait();
    const int n = items();
    for (int i = first; i < n; i += step) {
      const int cols = (i8_item(p, i).rows + 15) & ~15;
      const uint32_t idesc = i8_idesc(cols), d = tmem + (uint32_t)(buf * NA * p.tn);
      mbar_wait_or(drained_s + 8u * buf, dph ^ 1u, gave_up_s);
      for (int kb = kb0; kb < kb1; ++kb) {
        mbar_wait_or(full_s + 8u * s, ph, gave_up_s);
        __syncwarp();
        tc_fence_after();
        const uint32_t a = lo0 + (uint32_t)s * stage16, b = a + (NA * I8_A_BYTES >> 4);
        umma_i8_ss4(d, a, b, hi, idesc, kb > kb0, lead);
        if (NA == 2) umma_i8_ss4(d + (uint32_t)p.tn, a + (I8_A_BYTES >> 4), b, hi, idesc, kb > kb0, lead);
        umma_commit(empty_s + 8u * s, lead);
        if (++s == p.stages) { s = 0; ph ^= 1u; }
      }
      umma_commit(accum_s + 8u * buf, lead);
      if (++buf == p.nbuf) { buf = 0; dph ^= 1u; }
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ---------------- epilogue ----------------
    // (a warp reaches the 32 lanes of tensor memory of its number modulo 4; two warps share them, taking 16 columns in turn)
    const int quad = (warp & 3) * 32, row = quad + lane, half = (warp - 4) >> 2, tid = threadIdx.x - 128;
    const uint32_t t_lane = tmem + ((uint32_t)quad << 16);
    uint8_t* stage = s_stage + (warp - 4) * 1024;
    const bool wide_y = p.dtype != DT_F32 && p.ldy % 8 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0;
    int buf = 0, turn = 0;
    uint32_t aph = 0;
    pdl_wait();
    const int n_items = items();
    for (int i = first; i < n_items; i += step) {
      const I8Item t = i8_item(p, i);
      float* xs = s_scale + turn * 256;   // (in turn: whoever has passed the last item's barrier is done with those of the item before it)
      int* xr = s_row + turn * 256;
      turn ^= 1;
      for (int c = tid; c < p.tn; c += 32 * I8_EPI) {
        float f = 0.f;
        int o = t.x0 + c;
        if (c < t.rows) {
          f = p.q_scale[o];
          if (p.passes && NA == 1) {
            o = p.sorted[o];
            f *= p.row_scale[o];
          }
        }
        xs[c] = f;
        xr[c] = o;
      }
      const int n = t.n0 + row, rows = min(32, p.n - (t.n0 + quad));   // (of this warp's 32; not positive: none)
      const bool live = lane < rows;
      const float ws = live ? p.w_scale[t.a_row + row] : 0.f, wu = NA == 2 && live ? p.w_scale[t.a_row + p.n_up + row] : 0.f;
      asm volatile("bar.sync 1, %0;" ::"n"(32 * I8_EPI) : "memory");
      mbar_wait_or(accum_s + 8u * buf, aph, gave_up_s);
      __syncwarp();
      tc_fence_after();
      if (p.split == 1) {
        const uint32_t d = t_lane + (uint32_t)(buf * NA * p.tn);
        const float bias = live ? i8_bias(p, n) : 0.f;
        for (int c0 = 16 * half; c0 < t.rows; c0 += 32) {
          uint32_t v[16], u[16];
          tmem_ld16(d + (uint32_t)c0, v);
          if (NA == 2) tmem_ld16(d + (uint32_t)(p.tn + c0), u);
          float f[16];
          float4 x[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = reinterpret_cast<const float4*>(xs + c0)[j];
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float xj = reinterpret_cast<const float*>(x)[j];
            f[j] = (float)(int)v[j] * (xj * ws);
            if (NA == 2) f[j] = i8_act(p.act, f[j]) * ((float)(int)u[j] * (xj * wu));
            else f[j] += bias;
          }
          const int count = min(16, t.rows - c0);
          if (NA == 2 || p.dtype == DT_F32) i8_store16<float>(static_cast<float*>(p.y), p.ldy, xr + c0, count, f, n, lane, rows, false, stage);
          else if (p.dtype == DT_F16) i8_store16<__half>(static_cast<__half*>(p.y), p.ldy, xr + c0, count, f, n, lane, rows, wide_y && rows == 32, stage);
          else i8_store16<__nv_bfloat16>(static_cast<__nv_bfloat16*>(p.y), p.ldy, xr + c0, count, f, n, lane, rows, wide_y && rows == 32, stage);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(drained_s + 8u * buf);
      }
      if (++buf == p.nbuf) { buf = 0; aph ^= 1u; }
    }
  }
  __syncwarp();
  if (NA == 1 && p.split > 1) {
    // ---------------- split: the sums of rows [per * rank, per * (rank + 1)) of the tile are this CTA's to add and store ----------------
    cluster_sync();   // every CTA's products are complete, its ring is free: [from][token][row]
    const I8Item t = i8_item(p, first);
    const int per = I8_ROWS / p.split, shift = 31 - __clz(per);
    const uint32_t ring = smem_u32(smem);
    if (warp >= 4) {
      const int quad = (warp & 3) * 32, row = quad + lane;
      const uint32_t d = tmem + ((uint32_t)quad << 16);
      uint32_t peer;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(ring + 4u * (uint32_t)((int)rank * p.tn * per + (row & (per - 1)))), "r"(row >> shift));
      for (int c0 = 16 * ((warp - 4) >> 2); c0 < t.rows; c0 += 32) {
        uint32_t v[16];
        tmem_ld16(d + (uint32_t)c0, v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer + 4u * (uint32_t)((c0 + j) * per)), "r"(v[j]) : "memory");
      }
    }
    cluster_sync();
    if (warp >= 4) {
      const int tid = threadIdx.x - 128, r = tid & (per - 1), row = (int)rank * per + r, n = t.n0 + row;
      if (n < p.n) {
        const float ws = p.w_scale[t.a_row + row], bias = i8_bias(p, n);
        for (int c = tid >> shift; c < t.rows; c += 32 * I8_EPI >> shift) {
          int sum = 0;
#pragma unroll 4
          for (int from = 0; from < p.split; ++from) sum += (int)lds32(ring + 4u * (uint32_t)((from * p.tn + c) * per + r));
          i8_put(p.y, p.dtype, (int64_t)(t.x0 + c) * p.ldy + n, (float)sum * (s_scale[c] * ws) + bias);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*gave_up) {
    if (threadIdx.x == 0) atomicExch(p.status, E_TIMEOUT);
    // A bounded wait ran out in this CTA.  What it started has to finish before its tensor memory is given up: the commit covers the
    // tensor pipe, and the copies in flight land within microseconds.
    if (warp == 1) {
      if (lane == 0) mbar_init(last, 1);
      __syncwarp();
      if (elect_one()) umma_commit(last);
      __syncwarp();
      mbar_wait_bounded(last, 0);
    }
    drain_pause();
    tc_fence_before();
    __syncthreads();
  }
  if (warp == 2) tmem_dealloc(tmem, p.tmem_cols);
}

static bool i8_map(CUtensorMap& map, const void* base, int64_t k, int64_t rows, int64_t pitch, int box_rows) {
  EncodeTiledFn enc = tensor_map_encoder();
  if (!enc) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch};
  const cuuint32_t box[2] = {I8_BK, (cuuint32_t)box_rows}, one[2] = {1, 1};
  return enc(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int NA> static int i8_launch(const CUtensorMap& amap, const CUtensorMap& bmap, const I8Params& p, int grid, size_t smem, cudaStream_t stream) {
  static bool configured[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return E_CUDA;
  if (!configured[dev & 63]) {
    if (cudaFuncSetAttribute(i8_kernel<NA>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess) return E_CUDA;
    configured[dev & 63] = true;
  }
  return launch_pdl_cluster(i8_kernel<NA>, dim3((unsigned)grid), dim3(I8_THREADS), (unsigned)p.split, smem, stream, amap, bmap, p) == cudaSuccess ? E_OK : E_CUDA;
}

// Tokens of an expert's pass: its average share of the slots and three standard deviations, up to 128
int64_t i8_moe_pass_rows(int64_t slots, int64_t experts) {
  const double mean = (double)slots / (double)experts;
  const int64_t rows = round_up((int64_t)(mean + 3.0 * sqrt(mean)) + 1, 16);
  return rows <= 64 ? rows : 128;
}

int launch_i8_product(const I8Product& a, cudaStream_t stream) {
  const int na = a.act ? 2 : 1;
  I8Params p{};
  p.n = (int)a.n;
  p.n_up = (int)a.n;
  p.w_rows = (int)(a.n * na);
  p.k = (int)a.k;
  p.nk = (int)((a.k + I8_BK - 1) / I8_BK);
  p.m = (int)a.m;
  p.rt = (int)((a.n + I8_ROWS - 1) / I8_ROWS);
  if (a.passes) {
    p.tn = (int)a.pass_rows;
    p.tt = 1;
  } else {
    p.tt = (int)((a.m + 255) / 256);
    p.tn = (int)round_up((a.m + p.tt - 1) / p.tt, 16);
  }
  p.bh = !a.passes || p.tn <= 64 ? p.tn : 64;
  p.stage_bytes = na * I8_A_BYTES + p.tn * I8_BK;
  const int per_sm = p.tn <= 64 ? 2 : 1;
  const int64_t tiles = a.passes ? a.max_passes * p.rt : (int64_t)p.rt * p.tt;
  if (tiles > 1 << 29) return E_TOO_LARGE;
  p.split = 1;
  if (!a.passes)
    while (p.split < 8 && tiles * p.split * 2 <= I8_SMS * per_sm && p.nk >= 8 * p.split) p.split *= 2;
  const int room = (per_sm == 2 ? 113 : 227) * 1024 - 1024 - I8_AUX - (per_sm == 2 ? 1024 : 0);
  p.stages = room / p.stage_bytes;
  if (p.stages > I8_MAX_STAGES) p.stages = I8_MAX_STAGES;
  p.aux_off = p.stages * p.stage_bytes;
  const int cols = na * p.tn, most = 512 / per_sm;
  p.nbuf = p.split == 1 && 2 * cols <= most ? 2 : 1;
  p.tmem_cols = 32;
  while ((int)p.tmem_cols < p.nbuf * cols) p.tmem_cols *= 2;
  p.y = a.y;
  p.ldy = a.ldy;
  p.dtype = a.dtype;
  p.w_scale = a.w_scale;
  p.q_scale = a.q_scale;
  p.bias = a.bias;
  p.settled = a.settled;
  p.passes = static_cast<const int4*>(a.passes);
  p.n_passes = a.n_passes;
  p.act = a.act;
  p.sorted = a.sorted;
  p.row_scale = a.row_scale;
  p.status = a.status;
  const int64_t slots = I8_SMS * per_sm, grid = p.split > 1 ? tiles * p.split : tiles < slots ? tiles : slots;
  CUtensorMap amap, bmap;
  if (!i8_map(amap, a.w, a.k, a.experts * p.w_rows, a.ldw, I8_ROWS) || !i8_map(bmap, a.q, a.k, a.m, a.ldq, p.bh)) return E_CUDA;
  const size_t smem = 1024 + (size_t)p.aux_off + I8_AUX;
  return na == 2 ? i8_launch<2>(amap, bmap, p, (int)grid, smem, stream) : i8_launch<1>(amap, bmap, p, (int)grid, smem, stream);
}

}  // namespace gguf_b200
