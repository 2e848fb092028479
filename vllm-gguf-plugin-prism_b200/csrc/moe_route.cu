// The router of a mixture of experts: logits -> ids and weights of the top_k experts of every token.
//
//   s = softmax or sigmoid of the row's logits (fp64 where a choice hangs on it); an expert whose logit is -inf or NaN is masked
//   choice = s + bias; without a bias the order of s is the order of the logits, which are compared as they are
//   groups: only the experts of the topk_group best groups remain, by the sum of a group's two best choices (with a bias) or by
//   its best one (without)
//   the top_k best remaining, the best first, equals by the lower index; weight = s, divided by their sum, times scale
//   a place for which nothing is left: id -1, weight 0
//
// One warp a token, expert 32 j + l in lane l.  A choice becomes an unsigned key of the same order, 0 for "out", and the maximum
// over the warp is a hardware reduction.
#include "common.cuh"
#include "kernels.h"

namespace gguf_b200 {

struct RouteParams {
  const void* logits;
  int64_t ld;
  const float* bias;
  float* weights;
  int32_t* ids;
  int64_t tokens;
  int experts, top_k, groups, topk_group, sigmoid, renormalize;
  float scale;
};

// keys of the same order as the numbers they come from; 0 is below all of them
__device__ __forceinline__ uint32_t route_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return v == -INFINITY || v != v ? 0u : v == 0.f ? 0x80000000u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t route_key(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v);
  return v == -INFINITY || v != v ? 0ull : v == 0.0 ? 1ull << 63 : (b >> 63) ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ double route_value(uint64_t key) {
  return __longlong_as_double((long long)(key >> 63 ? key & ~(1ull << 63) : ~key));
}
__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ uint64_t warp_max(uint64_t v) {
  const uint32_t hi = warp_max((uint32_t)(v >> 32));
  return (uint64_t)hi << 32 | warp_max((uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

// Key: uint32_t, the logits themselves are compared (no bias); uint64_t, scores in fp64 (bias)
template <typename T, typename Key, int V>
__global__ void __launch_bounds__(128) moe_route_kernel(const RouteParams p) {
  pdl_trigger();
  pdl_wait();
  constexpr bool SCORES = sizeof(Key) == 8;
  const int lane = threadIdx.x & 31;
  for (int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5); t < p.tokens; t += (int64_t)gridDim.x * 4) {
    const T* row = static_cast<const T*>(p.logits) + t * p.ld;
    auto logit = [&](int e) {
      const float v = to_float<T>(row[e]);
      return v != v ? -INFINITY : fminf(v, 3.402823466e+38f);
    };
    float x[V];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = 32 * j + lane;
      x[j] = e < p.experts ? logit(e) : -INFINITY;
      top = max(top, route_key(x[j]));
    }
    top = warp_max(top);
    const float high = top == 0 ? 0.f : __uint_as_float(top >> 31 ? top & 0x7fffffffu : ~top);
    double total = 0.0;
    if (!p.sigmoid && (SCORES || !p.renormalize)) {
#pragma unroll
      for (int j = 0; j < V; ++j) total += x[j] == -INFINITY ? 0.0 : exp((double)x[j] - (double)high);
      total = warp_sum(total);
    }
    auto score = [&](float v) {   // of an unmasked expert; softmax without `total`: up to a factor
      if (p.sigmoid) return 1.0 / (1.0 + exp(-(double)v));
      const double e = exp((double)v - (double)high);
      return total > 0.0 ? e / total : e;
    };
    Key key[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if constexpr (SCORES)
        key[j] = x[j] == -INFINITY ? 0 : route_key(score(x[j]) + (double)p.bias[32 * j + lane]);
      else
        key[j] = route_key(x[j]);
    }
    if (p.groups > 1) {
      const int per = p.experts / p.groups;
      Key mine = 0;   // lane g: score of group g
      for (int g = 0; g < p.groups; ++g) {
        Key a = 0;
        int at = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int e = 32 * j + lane;
          if (e / per == g && key[j] > a) { a = key[j]; at = j; }
        }
        const Key best = warp_max(a);
        Key score_g = best;
        if constexpr (SCORES) {
          const int owner = __ffs(__ballot_sync(0xffffffffu, a == best)) - 1;
          Key b = 0;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int e = 32 * j + lane;
            if (e / per == g && !(lane == owner && j == at)) b = max(b, key[j]);
          }
          const Key second = warp_max(b);
          if (second != 0) score_g = route_key(route_value(best) + route_value(second));
        }
        if (lane == g) mine = score_g;
      }
      // (a group without an expert is picked when nothing else is left, which changes nothing)
      uint32_t taken = 0;
      for (int i = 0; i < p.topk_group; ++i) {
        const bool free = lane < p.groups && !(taken >> lane & 1u);
        const Key best = warp_max(free ? mine : Key(0));
        const int g = __ffs(__ballot_sync(0xffffffffu, free && mine == best)) - 1;
        taken |= 1u << g;
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int e = 32 * j + lane;
        if (e < p.experts && !(taken >> (e / per) & 1u)) key[j] = 0;
      }
    }
    int id = -1;   // lane i: the i-th choice
    for (int i = 0; i < p.top_k; ++i) {
      Key a = 0;
      int at = 0;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (key[j] > a) { a = key[j]; at = j; }
      const Key best = warp_max(a);
      if (best == 0) break;
      const int e = (int)__reduce_min_sync(0xffffffffu, a == best ? (unsigned)(32 * at + lane) : 0xffffffffu);
      if (lane == i) id = e;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (32 * j + lane == e) key[j] = 0;
    }
    double w = id >= 0 ? score(logit(id)) : 0.0;
    if (p.renormalize) {
      const double sum = warp_sum(w);
      w = sum > 0.0 ? w / sum : 0.0;
    }
    if (lane < p.top_k) {
      p.weights[t * p.top_k + lane] = (float)(w * (double)p.scale);
      p.ids[t * p.top_k + lane] = id;
    }
  }
}

template <typename T, typename Key> static cudaError_t route_launch(const RouteParams& p, cudaStream_t stream) {
  const int64_t blocks = (p.tokens + 3) / 4, most = 148 * 16;
  const dim3 grid((unsigned)(blocks < most ? blocks : most));
  if (p.experts <= 64) return launch_pdl(moe_route_kernel<T, Key, 2>, grid, dim3(128), 0, stream, p);
  if (p.experts <= 128) return launch_pdl(moe_route_kernel<T, Key, 4>, grid, dim3(128), 0, stream, p);
  if (p.experts <= 256) return launch_pdl(moe_route_kernel<T, Key, 8>, grid, dim3(128), 0, stream, p);
  return launch_pdl(moe_route_kernel<T, Key, 16>, grid, dim3(128), 0, stream, p);
}
template <typename T> static cudaError_t route_typed(const RouteParams& p, cudaStream_t stream) {
  return p.bias ? route_launch<T, uint64_t>(p, stream) : route_launch<T, uint32_t>(p, stream);
}

int launch_moe_route(const void* logits, int dtype, int64_t ld, const float* bias, float* weights, int32_t* ids, int64_t tokens, int experts, int top_k,
                     int groups, int topk_group, int sigmoid, int renormalize, float scale, cudaStream_t stream) {
  const RouteParams p{logits, ld, bias, weights, ids, tokens, experts, top_k, groups, topk_group, sigmoid, renormalize, scale};
  if (tokens == 0) return E_OK;
  cudaError_t e;
  switch (dtype) {
    case DT_F32: e = route_typed<float>(p, stream); break;
    case DT_F16: e = route_typed<__half>(p, stream); break;
    case DT_BF16: e = route_typed<__nv_bfloat16>(p, stream); break;
    default: return E_BAD_DTYPE;
  }
  return e == cudaSuccess ? E_OK : E_CUDA;
}

}  // namespace gguf_b200
