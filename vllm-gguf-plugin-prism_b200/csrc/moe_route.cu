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
// over the warp is a hardware reduction.  Choices by scores are made in fp32 first, with an error bound: where two of them that decide
// about something are nearer than that (one row in a thousand), the row is done again in fp64.  (8192 tokens, 256 experts in eight
// groups: 45 us with all scores in fp64.)
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
__device__ __forceinline__ float route_value(uint32_t key) { return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key); }
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
// Whether a choice `a` is above another, `b`, for certain.  An fp32 score (at most 1) is off by less than 2^-19: the approximate
// exponential by (|x| + 2) 2^-23 of itself, which the score's derivative brings below 2^-22; a softmax' sum of up to 512 terms by 21 roundings of
// 2^-24; the quotient by 2^-22.  The sum with the bias adds 2^-24 of itself, a sum of two choices twice all that.  (NaN: not certain.)
__device__ __forceinline__ bool route_above(float a, float b, float times) { return a - b > times * (0x1p-18f + 0x1p-22f * (fabsf(a) + fabsf(b))); }

// Keys of a token's experts -> lane i's id is the i-th choice, -1 where there is none.  False: the fp32 choices do not settle it.
template <typename Key, int V, bool SCORES>
__device__ __forceinline__ bool route_choose(const RouteParams& p, Key (&key)[V], int lane, int& id) {
  constexpr bool CHECK = SCORES && sizeof(Key) == 4;
  bool sure = true;
  if (p.groups > 1) {
    const int per = p.experts / p.groups;
    const float inv_per = 1.f / (float)per;
    int group[V];
#pragma unroll
    for (int j = 0; j < V; ++j) group[j] = (int)(((float)(32 * j + lane) + 0.5f) * inv_per);
    Key mine = 0;   // lane g: score of group g
    auto close = [&](int g, Key a, Key b) {   // a, b: this lane's two best of group g
      const Key best = warp_max(a);
      Key score = best;
      if constexpr (SCORES) {
        const int owner = __ffs(__ballot_sync(0xffffffffu, a == best)) - 1;
        const Key second = warp_max(lane == owner ? b : a);
        if (second != 0) score = route_key(route_value(best) + route_value(second));
      }
      if (lane == g) mine = score;
    };
    if (per % 32 == 0) {   // a group is whole registers
      Key a = 0, b = 0;
      int left = per / 32, g = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        b = max(b, min(a, key[j]));
        a = max(a, key[j]);
        if (--left == 0) {
          if (g < p.groups) close(g, a, b);
          a = b = 0;
          left = per / 32;
          ++g;
        }
      }
    } else {
      for (int g = 0; g < p.groups; ++g) {
        Key a = 0, b = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const Key x = group[j] == g ? key[j] : Key(0);
          b = max(b, min(a, x));
          a = max(a, x);
        }
        close(g, a, b);
      }
    }
    // (a group without an expert is picked when nothing else is left, which changes nothing)
    uint32_t taken = 0;
    Key last = 0;
    for (int i = 0; i < p.topk_group; ++i) {
      last = warp_max(mine);
      const int g = __ffs(__ballot_sync(0xffffffffu, mine == last && lane < p.groups && !(taken >> lane & 1u))) - 1;
      taken |= 1u << g;
      if (lane == g) mine = 0;
    }
    if (CHECK) {
      const Key next = warp_max(mine);
      sure = next == 0 || route_above((float)route_value(last), (float)route_value(next), 2.f);
    }
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (!(taken >> (group[j] & 31) & 1u)) key[j] = 0;   // (places behind the last expert are out already)
  }
  Key a = 0;
  int at = 0;
  auto nearest = [&] {
    a = 0;
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (key[j] > a) { a = key[j]; at = j; }
  };
  nearest();
  id = -1;
  Key before = 0;
  for (int i = 0; i < p.top_k + (CHECK ? 1 : 0); ++i) {
    const Key best = warp_max(a);
    if (best == 0) break;
    if (CHECK) {
      if (i > 0) sure = sure && route_above((float)route_value(before), (float)route_value(best), 1.f);
      before = best;
      if (i == p.top_k) break;
    }
    const int e = (int)__reduce_min_sync(0xffffffffu, a == best ? (unsigned)(32 * at + lane) : 0xffffffffu);
    if (lane == i) id = e;
    if (lane == (e & 31)) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (32 * j + lane == e) key[j] = 0;
      nearest();
    }
    __syncwarp();
  }
  return sure;
}

// SCORES: choices are scores and a bias; without, the logits themselves are compared
template <typename T, bool SCORES, int V>
__global__ void __launch_bounds__(128) moe_route_kernel(const RouteParams p) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  for (int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5); t < p.tokens; t += (int64_t)gridDim.x * 4) {
    const T* row = static_cast<const T*>(p.logits) + t * p.ld;
    auto logit = [&](int e) {
      const float v = to_float<T>(row[e]);
      return v != v ? -INFINITY : fminf(v, 3.402823466e+38f);
    };
    float x[V];
    uint32_t key[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = 32 * j + lane;
      x[j] = e < p.experts ? logit(e) : -INFINITY;
    }
    float high = 0.f;
    if (!p.sigmoid) {
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) top = max(top, route_key(x[j]));
      top = warp_max(top);
      if (top != 0) high = route_value(top);
    }
    double total = 0.0;   // of a softmax; 0 where the weights are divided by their own sum
    if (!p.sigmoid && !p.renormalize) {   // (terms off by 2^-21 of themselves at most)
#pragma unroll
      for (int j = 0; j < V; ++j) total += (double)expf(x[j] - high);
      total = warp_sum(total);
    }
    int id;
    bool sure;
    if constexpr (SCORES) {
      float e[V], sum = 1.f;
      if (!p.sigmoid) {
        sum = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          e[j] = __expf(x[j] - high);
          sum += e[j];
        }
        sum = __frcp_rn(fmaxf(warp_sum(sum), 1e-30f));
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float s = p.sigmoid ? __fdividef(1.f, 1.f + __expf(-x[j])) : e[j] * sum;
        key[j] = x[j] == -INFINITY ? 0u : route_key(s + p.bias[32 * j + lane]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) key[j] = route_key(x[j]);
    }
    sure = route_choose<uint32_t, V, SCORES>(p, key, lane, id);
    auto score = [&](float v) {   // of an unmasked expert; softmax without `total`: up to a factor
      if (p.sigmoid) return 1.0 / (1.0 + exp(-(double)v));
      const double e = exp((double)v - (double)high);
      return total > 0.0 ? e / total : e;
    };
    if constexpr (SCORES) {
      if (!p.sigmoid && !sure) {
        total = 0.0;
#pragma unroll 1
        for (int e = lane; e < p.experts; e += 32) {
          const float v = logit(e);
          total += v == -INFINITY ? 0.0 : exp((double)v - (double)high);
        }
        total = warp_sum(total);
      }
      if (!sure) {
        uint64_t wide[V];
#pragma unroll
        for (int j = 0; j < V; ++j) wide[j] = x[j] == -INFINITY ? 0 : route_key(score(x[j]) + (double)p.bias[32 * j + lane]);
        route_choose<uint64_t, V, true>(p, wide, lane, id);
      }
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

template <typename T, bool SCORES> static cudaError_t route_launch(const RouteParams& p, cudaStream_t stream) {
  const int64_t blocks = (p.tokens + 3) / 4, most = 148 * 16;
  const dim3 grid((unsigned)(blocks < most ? blocks : most));
  if (p.experts <= 64) return launch_pdl(moe_route_kernel<T, SCORES, 2>, grid, dim3(128), 0, stream, p);
  if (p.experts <= 128) return launch_pdl(moe_route_kernel<T, SCORES, 4>, grid, dim3(128), 0, stream, p);
  if (p.experts <= 256) return launch_pdl(moe_route_kernel<T, SCORES, 8>, grid, dim3(128), 0, stream, p);
  return launch_pdl(moe_route_kernel<T, SCORES, 16>, grid, dim3(128), 0, stream, p);
}
template <typename T> static cudaError_t route_typed(const RouteParams& p, cudaStream_t stream) {
  return p.bias ? route_launch<T, true>(p, stream) : route_launch<T, false>(p, stream);
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
