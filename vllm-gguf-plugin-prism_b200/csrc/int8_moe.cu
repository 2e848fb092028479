// The routed expert step around its products of 8-bit integers: the order of the slots, and the sum over a token's experts.
//
//   i8_plan_kernel  slots (token * top_k + j) sorted by expert, in their order; every expert's rows in passes of like size.  One block
//                   takes up to 1024 slots; of more, a cluster of eight blocks takes equal runs, which learn of one another's counts
//                   through shared memory.  A warp counts its share of the run and, once the sums over warps, blocks and experts are
//                   there, places it, 32 slots at a time.
//                   Latencies bound it: 16384 slots of 64 experts 9 us behind the kernel ahead, 11 alone with cold caches; 64 slots 6.5 so.  (16 blocks
//                   that each counted all slots and summed over their warps for every 1024 of them took 2 us more, divisions between the sums 1.4.)
//   i8_sum_kernel   out[t] = sum over j of y[t * top_k + j] * weight, in fp32, rounded once.  Bound by memory: 2048 tokens of 2048 columns, eight
//                   experts, 134 MB in 27 to 28 us (20.8 at the copy rate, beside what L2 still has to write of them).
//
// The experts' results travel from the down product to the sum in fp32, whatever the tokens' type: the step's largest buffer, 134 MB for 2048 tokens
// of 2048 columns with eight experts each, written and read again.  (In fp16, with powers of two taken out, the same step took 196 us instead of
// 221, but an fp16 result was off by 2.9e-4 instead of 2.0e-4, and rows of W2 whose scale is far below the expert's largest lost their bits.
// The product and the sum in two halves of the columns, so that the buffer stays in L2: level.)
#include <math.h>

#include "common.cuh"
#include "int8.cuh"

namespace gguf_b200 {

constexpr int I8_MAX_EXPERTS = 256, I8_PLAN_BLOCKS = 8;

// An expert's c rows in passes of like size: whole groups of 16 tokens but for the last, at most pass_rows
__device__ __forceinline__ int i8_pass_size(int c, int pass_rows) {
  const int np = (c + pass_rows - 1) / pass_rows;
  return np > 0 ? ((c + np - 1) / np + 15) / 16 * 16 : 16;
}

__global__ void __launch_bounds__(1024, 1) i8_plan_kernel(const I8Plan p, int blocks, int run) {
  __shared__ int32_t s_cnt[32][I8_MAX_EXPERTS + 1];   // a warp's slots of an expert; then where its next one goes, from the block's first
  __shared__ int32_t s_run[I8_MAX_EXPERTS], s_total[I8_MAX_EXPERTS], s_next[I8_MAX_EXPERTS];   // the block's slots, all, the block's first place
  __shared__ int32_t s_size[I8_MAX_EXPERTS], s_passes[I8_MAX_EXPERTS], s_order[I8_MAX_EXPERTS], s_pass[I8_MAX_EXPERTS];   // block 0: passes
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, E = p.experts, slots = (int)p.slots;
  // One block for all slots has one for every thread.
  const bool alone = blocks == 1;
  const int warps = alone ? ((slots + 31) / 32 + 7) / 8 * 8 : 32;
  for (int i = threadIdx.x; i < warps * (I8_MAX_EXPERTS + 1); i += 1024) (&s_cnt[0][0])[i] = 0;
  pdl_wait();
  pdl_trigger();
  // A warp's slots: a 32nd of the block's, in their order, 32 at a time
  const int own = run / 32, s0 = min(slots, (int)blockIdx.x * run + warp * own), s1 = min(slots, s0 + own);
  // Lanes with this one's expert, and how many of them are below it
  auto match = [&](int e, unsigned& same) {
    same = __match_any_sync(0xffffffffu, e);
    return __popc(same & ((1u << lane) - 1u));
  };
  auto valid = [&](int e) { return e >= 0 && e < E; };
  int my_e = -1, my_below = 0;
  if (alone && s0 + lane < s1) my_e = p.topk_ids[s0 + lane];
  __syncthreads();
  if (alone) {
    unsigned same;
    my_below = match(my_e, same);
    if (valid(my_e) && my_below == 0) s_cnt[warp][my_e] = __popc(same);
  } else {
    for (int b = s0 + lane; b < s1; b += 8 * 32) {   // (eight loads in flight)
      int e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = b + i * 32 < s1 ? p.topk_ids[b + i * 32] : -1;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (valid(e[i])) atomicAdd(&s_cnt[warp][e[i]], 1);
    }
  }
  __syncthreads();
  int total = 0, before = 0;   // of expert threadIdx.x: in all blocks, in those ahead
  if ((int)threadIdx.x < E) {
    for (int w0 = 0; w0 < warps; w0 += 8) {   // (eight loads in flight)
      int v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = s_cnt[w0 + i][threadIdx.x];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s_cnt[w0 + i][threadIdx.x] = total;
        total += v[i];
      }
    }
    s_run[threadIdx.x] = total;
  }
  if (!alone) {
    cluster_arrive();
    cluster_wait();
    if ((int)threadIdx.x < E) {
      int c[I8_PLAN_BLOCKS];
#pragma unroll
      for (int i = 0; i < I8_PLAN_BLOCKS; ++i) {
        uint32_t at;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(&s_run[threadIdx.x])), "r"(i));
        asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(c[i]) : "r"(at) : "memory");
      }
      total = 0;
#pragma unroll
      for (int i = 0; i < I8_PLAN_BLOCKS; ++i) {
        if (i < (int)blockIdx.x) before += c[i];
        total += c[i];
      }
    }
    cluster_arrive();   // (the others' counts are not read again; waited for before the end)
  }
  const bool by_size = p.pass_rows > 64;
  if ((int)threadIdx.x < E) {
    const int e = threadIdx.x;
    s_total[e] = total;
    s_next[e] = before;
    if (blockIdx.x == 0) {
      s_size[e] = i8_pass_size(total, p.pass_rows);
      s_passes[e] = (total + s_size[e] - 1) / s_size[e];
      s_order[e] = e;
    }
  }
  __syncthreads();
  // Large passes are dealt out by size, the largest first: CTAs that take them in turn then get like shares.
  if (blockIdx.x == 0 && by_size) {
    const int team = E <= 64 ? 16 : 4, e = threadIdx.x / team, size = e < E ? s_size[e] : 0;
    int rank = 0;
    for (int o = threadIdx.x % team; o < E; o += team) {
      const int other = s_size[o];
      rank += other > size || (other == size && o < e);
    }
    for (int m = 1; m < team; m <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, m);
    if (e < E && threadIdx.x % team == 0) s_order[rank] = e;
    __syncthreads();
  }
  // Prefix sums over the experts: rows (warp 0), and passes in that order (block 0's warp 1).  A lane takes neighbours.
  if (warp == 0 || (warp == 1 && blockIdx.x == 0)) {
    const int per = (E + 31) / 32, e0 = min(E, lane * per), e1 = min(E, e0 + per);
    int sum = 0;
    for (int e = e0; e < e1; ++e) sum += warp == 0 ? s_total[e] : s_passes[s_order[e]];
    int a = sum;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, a, m);
      if (lane >= m) a += u;
    }
    if (lane == 31 && blockIdx.x == 0) p.n_passes[warp == 0 ? 1 : 0] = a;
    a -= sum;
    for (int e = e0; e < e1; ++e) {
      if (warp == 0) {
        s_next[e] += a;
        a += s_total[e];
      } else {
        s_pass[s_order[e]] = a;
        a += s_passes[s_order[e]];
      }
    }
  }
  __syncthreads();
  auto put = [&](int s, int at) {
    if (at >= 0) p.sorted[at] = s;
    p.place[s] = at;
  };
  if (alone) {
    if (s0 + lane < s1) put(s0 + lane, valid(my_e) ? s_next[my_e] + s_cnt[warp][my_e] + my_below : -1);
  } else {
    for (int b = s0; b < s1; b += 8 * 32) {
      int e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = b + i * 32 + lane < s1 ? p.topk_ids[b + i * 32 + lane] : -1;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (b + i * 32 >= s1) break;
        unsigned same;
        const int below = match(e[i], same);
        const int at = valid(e[i]) ? s_cnt[warp][e[i]] + below : -1;
        __syncwarp();
        if (valid(e[i]) && below == 0) s_cnt[warp][e[i]] += __popc(same);
        __syncwarp();
        if (b + i * 32 + lane < s1) put(b + i * 32 + lane, at < 0 ? -1 : s_next[e[i]] + at);
      }
    }
  }
  if (blockIdx.x == 0) {   // four threads an expert
    const int e = threadIdx.x >> 2;
    if (e < E) {
      const int c = s_total[e], per = s_size[e];
      for (int i = threadIdx.x & 3; i < s_passes[e]; i += 4) static_cast<int4*>(p.passes)[s_pass[e] + i] = make_int4(e, s_next[e] + i * per, min(per, c - i * per), 0);
    }
  }
  if (!alone) cluster_wait();
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
  const int blocks = a.slots <= 1024 ? 1 : I8_PLAN_BLOCKS, run = (int)((a.slots + blocks - 1) / blocks + 1023) / 1024 * 1024;
  return launch_pdl_cluster(i8_plan_kernel, dim3((unsigned)blocks), dim3(1024), (unsigned)blocks, 0, stream, a, blocks, run) == cudaSuccess ? E_OK : E_CUDA;
}

// Four columns a thread, ROWS experts' rows in flight: of eight tokens 1 us less than eight columns and four rows, of 2048 tokens 2 us less.
template <typename T, int ROWS> __global__ void __launch_bounds__(128) i8_sum_kernel(const I8Sum p) {
  pdl_wait();
  pdl_trigger();
  const unsigned per_row = (unsigned)(p.h / 4), top_k = (unsigned)p.top_k;
  const uint64_t at = (uint64_t)blockIdx.x * 128 + threadIdx.x;
  if (at >= (uint64_t)p.tokens * per_row) return;
  const unsigned i = (unsigned)at, t = i / per_row, c = 4 * (i - t * per_row), slot0 = t * top_k;   // (fewer than 2^32)
  const float* in = p.y + (int64_t)slot0 * p.h + c;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  for (unsigned j0 = 0; j0 < top_k; j0 += ROWS, in += ROWS * p.h) {
    float4 v[ROWS];
    float f[ROWS];
#pragma unroll
    for (unsigned j = 0; j < ROWS; ++j)   // (a row that nothing was written to is read as well, and left out below: none waits for its place)
      v[j] = j0 + j < top_k ? __ldcs(reinterpret_cast<const float4*>(in + j * p.h)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (unsigned j = 0; j < ROWS; ++j) {
      const bool live = j0 + j < top_k && __ldg(p.place + slot0 + j0 + j) >= 0;   // (a slot without a valid expert contributes nothing)
      f[j] = live ? __ldg(p.weights + slot0 + j0 + j) : 0.f;
      if (!live) v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k] = fmaf(reinterpret_cast<const float*>(&v[j])[k], f[j], s[k]);
  }
  alignas(16) T o[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) o[k] = from_float<T>(s[k]);
  T* out = static_cast<T*>(p.out) + (int64_t)t * p.h + c;
  if (sizeof(T) == 4) *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(o);
  else *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(o);
}

template <typename T> static cudaError_t i8_sum_typed(const I8Sum& a, dim3 grid, cudaStream_t stream) {
  return a.top_k <= 4 ? launch_pdl(i8_sum_kernel<T, 4>, grid, dim3(128), 0, stream, a) : launch_pdl(i8_sum_kernel<T, 8>, grid, dim3(128), 0, stream, a);
}
int launch_i8_sum(const I8Sum& a, cudaStream_t stream) {
  const int64_t total = a.tokens * (a.h / 4);
  if (a.h % 8 != 0 || total >= (int64_t)1 << 32) return E_TOO_LARGE;
  const dim3 grid((unsigned)((total + 127) / 128));
  cudaError_t e;
  switch (a.dtype) {
    case DT_F32: e = i8_sum_typed<float>(a, grid, stream); break;
    case DT_F16: e = i8_sum_typed<__half>(a, grid, stream); break;
    case DT_BF16: e = i8_sum_typed<__nv_bfloat16>(a, grid, stream); break;
    default: return E_BAD_DTYPE;
  }
  return e == cudaSuccess ? E_OK : E_CUDA;
}

}  // namespace gguf_b200
