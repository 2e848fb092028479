// The routed expert step around its products of 8-bit integers: the order of the slots, and the sum over a token's experts.
//
//   i8_plan_kernel  slots (token * top_k + j) sorted by expert, in their order; every expert's rows in passes of like size.  Blocks take
//                   equal runs of slots; each counts all slots for itself (16 k of them are 64 KB, from L2), those ahead of its run apart,
//                   and places its own: no block waits for another.  More blocks, one an expert, look for the expert's largest scale.
//   i8_sum_kernel   out[t] = sum over j of y[t * top_k + j] * factor, in fp32, rounded once
//
// The experts' results y = D * w_scale travel from the down product to the sum in fp16 for 16-bit tokens (fp32 for fp32): half the bytes of
// the step's largest buffer.  They are divided by powers of two first, one above the expert's largest scale and one that brings the
// largest |D| there can be (128 * 127 * I) to 2^15 at most, so that nothing overflows whatever the scales.  It is one rounding of at most 2^-11
// of a result, an eighth of the sum's own for bf16, the same as the sum's own for fp16; of results below fp16's normal numbers, at
// most I * 2^-25 of one unit of D (at the expert's largest scale).
#include <math.h>

#include "common.cuh"
#include "int8.cuh"

namespace gguf_b200 {

constexpr int I8_MAX_EXPERTS = 256, I8_PLAN_BLOCKS = 32;

// An expert's c rows in passes of like size: whole groups of 16 tokens but for the last, at most pass_rows
__device__ __forceinline__ int i8_pass_size(int c, int pass_rows) {
  const int np = (c + pass_rows - 1) / pass_rows;
  return np > 0 ? ((c + np - 1) / np + 15) / 16 * 16 : 16;
}
__device__ __forceinline__ int i8_pass_count(int c, int pass_rows) {
  const int per = i8_pass_size(c, pass_rows);
  return (c + per - 1) / per;
}

__global__ void __launch_bounds__(1024) i8_plan_kernel(const I8Plan p, int blocks, int run) {
  pdl_wait();
  pdl_trigger();
  __shared__ int32_t s_cnt[32][I8_MAX_EXPERTS + 1];   // first: counts of all slots, by warp modulo 8; then a warp's slots of a step, and its first place
  __shared__ int32_t s_before[I8_MAX_EXPERTS], s_next[I8_MAX_EXPERTS], s_pass[I8_MAX_EXPERTS], s_total[I8_MAX_EXPERTS], s_order[I8_MAX_EXPERTS];
  __shared__ float s_top[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, E = p.experts;
  if ((int)blockIdx.x >= blocks) {   // largest scale of an expert (a scale that is not finite: as if it were not there)
    const int e = blockIdx.x - blocks;
    float top = 0.f;
    for (int64_t i = threadIdx.x; i < p.h; i += 1024) {
      const float v = fabsf(p.w2_scale[e * p.h + i]);
      if (v <= 3.402823466e+38f) top = fmaxf(top, v);
    }
    top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
    if (lane == 0) s_top[warp] = top;
    __syncthreads();
    if (warp == 0) {
      top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(s_top[lane])));
      if (lane == 0) {
        int x = 0;
        frexpf(top, &x);
        x = max(-126, min(127, x));
        p.w_top[e] = exp2f((float)x);
        p.w_unit[e] = exp2f((float)-x);
      }
    }
    return;
  }
  const int slots = (int)p.slots, s0 = min(slots, (int)blockIdx.x * run), s1 = min(slots, s0 + run);
  // Whether a slot has a valid expert, and how many lanes below this one have the same
  auto match = [&](int e, unsigned& below) {
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const bool valid = e >= 0 && e < E;
    below = __popc(same & ((1u << lane) - 1u));
    if (valid && below == 0) s_cnt[warp][e] = __popc(same);
    return valid;
  };
  // Of counts by warp: where a warp's first slot of the expert goes, from `at` on; returns where the next would
  auto spread = [&](int e, int at, int warps) {
    for (int w0 = 0; w0 < warps; w0 += 8) {   // (eight loads in flight)
      int v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = s_cnt[w0 + i][e];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s_cnt[w0 + i][e] = at;
        at += v[i];
      }
    }
    return at;
  };
  // One block for all slots counts them and places them in one go.
  const bool alone = blocks == 1;
  const int my_slot = threadIdx.x, warps = alone ? ((slots + 31) / 32 + 7) / 8 * 8 : 32;
  const int my_e = alone && my_slot < slots ? p.topk_ids[my_slot] : -1;
  unsigned my_below = 0;
  bool my_valid = false;
  for (int i = threadIdx.x; i < (alone ? warps : 16) * (I8_MAX_EXPERTS + 1); i += 1024) (&s_cnt[0][0])[i] = 0;
  __syncthreads();
  if (alone) {
    my_valid = match(my_e, my_below);
  } else {
    for (int b = threadIdx.x; b < slots; b += 8 * 1024) {   // (eight loads in flight)
      int e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = b + i * 1024 < slots ? p.topk_ids[b + i * 1024] : -1;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (e[i] >= 0 && e[i] < E) atomicAdd(&s_cnt[(warp & 7) + (b + i * 1024 < s0 ? 0 : 8)][e[i]], 1);
    }
  }
  __syncthreads();
  const bool by_size = p.pass_rows > 64 && blockIdx.x == 0;
  if ((int)threadIdx.x < E) {
    const int e = threadIdx.x;
    int before = 0, total = 0;
    if (alone) {
      total = spread(e, 0, warps);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        before += s_cnt[i][e];
        total += s_cnt[8 + i][e];
      }
      total += before;
    }
    s_before[e] = before;
    s_total[e] = total;
    if (by_size) s_pass[e] = i8_pass_size(total, p.pass_rows);
  }
  __syncthreads();
  // Large passes are dealt out by size, the largest first: CTAs that take them in turn then get like shares.
  if (by_size) {
    const int e = threadIdx.x >> 2, size = e < E ? s_pass[e] : 0;
    int rank = 0;
    for (int o = threadIdx.x & 3; o < E; o += 4) {
      const int other = s_pass[o];
      rank += other > size || (other == size && o < e);
    }
    rank += __shfl_xor_sync(0xffffffffu, rank, 1);
    rank += __shfl_xor_sync(0xffffffffu, rank, 2);
    if (e < E && (threadIdx.x & 3) == 0) s_order[rank] = e;
    __syncthreads();
  }
  if (warp == 0) {   // prefix sums over the experts: rows, and passes in that order
    int rows = 0, ps = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int e = e0 + lane, c = e < E ? s_total[e] : 0, o = by_size && e < E ? s_order[e] : e;
      const int np = e < E && blockIdx.x == 0 ? i8_pass_count(s_total[o], p.pass_rows) : 0;
      int a = c, b = np;
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, a, m), v = __shfl_up_sync(0xffffffffu, b, m);
        if (lane >= m) { a += u; b += v; }
      }
      if (e < E) {
        s_next[e] = rows + a - c + s_before[e];
        s_pass[o] = ps + b - np;
      }
      rows += __shfl_sync(0xffffffffu, a, 31);
      ps += __shfl_sync(0xffffffffu, b, 31);
    }
    if (lane == 0 && blockIdx.x == 0) {
      p.n_passes[0] = ps;
      p.n_passes[1] = rows;
    }
  }
  __syncthreads();
  if (blockIdx.x == 0)
    for (int e = warp; e < E; e += 32) {
      const int c = s_total[e], per = i8_pass_size(c, p.pass_rows);
      for (int i = lane; i * per < c; i += 32) static_cast<int4*>(p.passes)[s_pass[e] + i] = make_int4(e, s_next[e] + i * per, min(per, c - i * per), 0);
    }
  auto put = [&](int s, int at) {
    if (at >= 0) p.sorted[at] = s;
    p.place[s] = at;
  };
  if (alone) {
    if (my_slot < slots) put(my_slot, my_valid ? s_next[my_e] + s_cnt[warp][my_e] + (int)my_below : -1);
    return;
  }
  __syncthreads();   // (s_next moves on below)
  for (int b = s0; b < s1; b += 1024) {
    for (int i = threadIdx.x; i < 32 * (I8_MAX_EXPERTS + 1); i += 1024) (&s_cnt[0][0])[i] = 0;
    __syncthreads();
    const int s = b + threadIdx.x, e = s < s1 ? p.topk_ids[s] : -1;
    unsigned below;
    const bool valid = match(e, below);
    __syncthreads();
    if ((int)threadIdx.x < E) s_next[threadIdx.x] = spread(threadIdx.x, s_next[threadIdx.x], 32);
    __syncthreads();
    if (s < s1) put(s, valid ? s_cnt[warp][e] + (int)below : -1);
    __syncthreads();
  }
}

// Tokens of an expert's pass, at most 256: its average share of the slots and three standard deviations
int64_t i8_moe_pass_rows(int64_t slots, int64_t experts) {
  const double mean = (double)slots / (double)experts;
  const int64_t rows = round_up((int64_t)(mean + 3.0 * sqrt(mean)) + 1, 16);
  return rows < 256 ? rows : 256;
}
int64_t i8_moe_passes(int64_t slots, int64_t experts, int64_t pass_rows) {
  const int64_t worst = slots / pass_rows + experts;
  return slots < worst ? slots : worst;
}
int launch_i8_plan(const I8Plan& a, cudaStream_t stream) {
  if (a.experts < 1 || a.experts > I8_MAX_EXPERTS || a.slots > 1 << 24) return E_BAD_SHAPE;
  const int64_t steps = (a.slots + 1023) / 1024, per = (steps + I8_PLAN_BLOCKS - 1) / I8_PLAN_BLOCKS;
  const int run = (int)per * 1024, blocks = (int)((a.slots + run - 1) / run);
  return launch_pdl(i8_plan_kernel, dim3((unsigned)(blocks + a.experts)), dim3(1024), 0, stream, a, blocks, run) == cudaSuccess ? E_OK : E_CUDA;
}

// Eight columns a thread, ROWS experts' rows in flight: four of fp32, eight of fp16, four of fp16 where a token has no more experts (150 blocks of
// 1536 columns 3.0 us and 3.5).  2048 tokens of 2048 columns, eight experts, from L2 and memory: 16.5 us (19.2 when a row was asked for only
// once its place was known).
template <typename Y, typename T, int ROWS> __global__ void __launch_bounds__(128) i8_sum_kernel(const I8Sum p) {
  pdl_wait();
  pdl_trigger();
  constexpr int WI = sizeof(Y) / 2, WO = sizeof(T) / 2;   // 16-byte words of eight values
  const unsigned per_row = (unsigned)(p.h / 8), top_k = (unsigned)p.top_k;
  const unsigned i = blockIdx.x * 128 + threadIdx.x;
  if (i >= (unsigned)p.tokens * per_row) return;
  const unsigned t = i / per_row, c = 8 * (i - t * per_row), slot0 = t * top_k;
  const Y* in = static_cast<const Y*>(p.y) + (int64_t)slot0 * p.h + c;
  float s[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) s[k] = 0.f;
  for (unsigned j0 = 0; j0 < top_k; j0 += ROWS, in += ROWS * p.h) {
    uint4 v[ROWS][WI];
    float f[ROWS];
#pragma unroll
    for (unsigned j = 0; j < ROWS; ++j)   // (a row that nothing was written to is read as well, and left out below: none waits for its place)
#pragma unroll
      for (int k = 0; k < WI; ++k) v[j][k] = j0 + j < top_k ? reinterpret_cast<const uint4*>(in + j * p.h)[k] : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (unsigned j = 0; j < ROWS; ++j) {
      const bool live = j0 + j < top_k && __ldg(p.place + slot0 + j0 + j) >= 0;   // (a slot without a valid expert contributes nothing)
      f[j] = j0 + j < top_k ? __ldg(p.factor + slot0 + j0 + j) : 0.f;
      if (!live) {
        f[j] = 0.f;
#pragma unroll
        for (int k = 0; k < WI; ++k) v[j][k] = make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j)
#pragma unroll
      for (int k = 0; k < 8; ++k) s[k] = fmaf(to_float<Y>(reinterpret_cast<const Y*>(v[j])[k]), f[j], s[k]);
  }
  uint4 o[WO];
#pragma unroll
  for (int k = 0; k < 8; ++k) reinterpret_cast<T*>(o)[k] = from_float<T>(s[k]);
#pragma unroll
  for (int k = 0; k < WO; ++k) reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (int64_t)t * p.h + c)[k] = o[k];
}

int launch_i8_sum(const I8Sum& a, cudaStream_t stream) {
  const int64_t total = a.tokens * (a.h / 8);
  if (a.h % 8 != 0 || total >= (int64_t)1 << 31) return E_TOO_LARGE;
  const dim3 grid((unsigned)((total + 127) / 128));
  cudaError_t e;
  switch (a.dtype) {
    case DT_F32: e = launch_pdl(i8_sum_kernel<float, float, 4>, grid, dim3(128), 0, stream, a); break;
    case DT_F16: e = a.top_k <= 4 ? launch_pdl(i8_sum_kernel<__half, __half, 4>, grid, dim3(128), 0, stream, a) : launch_pdl(i8_sum_kernel<__half, __half, 8>, grid, dim3(128), 0, stream, a); break;
    case DT_BF16: e = a.top_k <= 4 ? launch_pdl(i8_sum_kernel<__half, __nv_bfloat16, 4>, grid, dim3(128), 0, stream, a) : launch_pdl(i8_sum_kernel<__half, __nv_bfloat16, 8>, grid, dim3(128), 0, stream, a); break;
    default: return E_BAD_DTYPE;
  }
  return e == cudaSuccess ? E_OK : E_CUDA;
}

}  // namespace gguf_b200
