// The router of a mixture of experts: logits -> ids and weights of the top_k experts of every token.
//
//   s = softmax or sigmoid of the row's logits (fp64 where a choice hangs on it, fp32 in the weights); an expert whose logit is -inf or NaN is masked
//   choice = s + bias; without a bias the order of s is the order of the logits, which are compared as they are
//   groups: only the experts of the topk_group best groups remain, by the sum of a group's two best choices (with a bias) or by
//   its best one (without)
//   the top_k best remaining, the best first, equals by the lower index; weight = s, divided by their sum, times scale
//   a place for which nothing is left: id -1, weight 0
//
// One warp a token, expert 32 j + l in lane l.  A choice becomes an unsigned key of the same order, and the maximum over the warp is a
// hardware reduction.  In the first pass a key is 32 bits, the lowest of which say which of a lane's experts it is; where what is left of the
// numbers (in fp32, scores with an error bound) does not settle an order that matters, keys are taken until the next one is out of
// question, and these candidates, a lane each, are ordered by 64-bit keys: of scores one row in some hundred, of fp32 logits those with equals.
// More than 32 candidates, an order of groups that is not settled and a softmax with a bias (which wants its sum in fp64) do the whole row again.
//
// Bound by the integer pipe, which runs at half the issue rate, and by the last row that is done again: 8192 tokens, 256 experts in eight
// groups with a bias, 15.2 us (up to 19.3 where rows are among them whose groups are not settled; 45 with 64-bit keys throughout, 24 with keys that
// kept 0 for "out", exact maxima for every row and fp64 in the weights, 19 to 20 with whole rows done again); fp32 logits with equals, no groups,
// 11.1 (16.2 with whole rows, though 6.8 and not 6.6 for 64 experts without equals).  A token alone 2.5, of which the launch is most.
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
  int per, group_of;   // experts a group; (e * group_of) >> 20 is e's group (e < 512: off by less than 2^-11 from e / per)
};

// Keys of the same order as the numbers they come from (no NaN).  Those of -infinity, and 0, are below ROUTE_LEAST: "out".
constexpr uint32_t ROUTE_LEAST = 0x00800000u;
__device__ __forceinline__ uint32_t route_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);   // (zeros of both signs are equal)
  return b ^ (uint32_t)((int)b >> 31 | (int)0x80000000);
}
__device__ __forceinline__ uint64_t route_key(double v) {   // (and 0 for -infinity and NaN)
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
  return v > -INFINITY ? b ^ (uint64_t)((long long)b >> 63 | (long long)(1ull << 63)) : 0ull;
}
__device__ __forceinline__ float route_value(uint32_t key) { return __uint_as_float(key ^ (uint32_t)(~((int)key >> 31) | (int)0x80000000)); }
__device__ __forceinline__ double route_value(uint64_t key) { return __longlong_as_double((long long)(key ^ (uint64_t)(~((long long)key >> 63) | (long long)(1ull << 63)))); }
__device__ __forceinline__ bool route_out(uint32_t key) { return key < ROUTE_LEAST; }
__device__ __forceinline__ bool route_out(uint64_t key) { return key == 0; }
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
__device__ __forceinline__ float route_exp(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.44269504f));
  return r;
}
__device__ __forceinline__ float route_rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Whether a choice `a` is above another, `b`, for certain.  off: what two scores can be off by together.  e^x above is off by (|x| + 2) 2^-23 of
// itself; a sigmoid by s (1 - s) times that, at most 2^-23, and 2^-24 + 2^-23 for the sum and the reciprocal: two of them by less than 2^-20.
// A softmax' sum of up to 512 terms adds 21 roundings of 2^-24: two by less than 2^-18.  The sum with the bias is rounded by 2^-24 of
// itself, and a key leaves out less than V 2^-23 of it.  size: what has been rounded so, |a| + |b|.  (NaN: not certain.)
template <int V> __device__ __forceinline__ bool route_above(float a, float b, float off, float size) {
  return a - b > off * (1.f + (float)(V + 1) * 0x1p-3f * size);   // ((V + 1) 2^-23 size, off being 2^-20 at least)
}
template <int V> __device__ __forceinline__ bool route_above(float a, float b, float off) { return route_above<V>(a, b, off, fabsf(a) + fabsf(b)); }

// The groups that remain, a bit each.  sure: false where the order of two groups that decides is not certain.
template <typename Key, int V, bool SCORES>
__device__ __forceinline__ uint32_t route_groups(const RouteParams& p, const Key (&key)[V], int lane, float off, bool& sure) {
  Key first = 0, second = 0;   // lane g: the two best choices of group g
  auto close = [&](int g, Key a, Key b) {   // a, b: this lane's two best of group g
    const Key best = warp_max(a);
    Key next = 0;
    if constexpr (SCORES) {
      const int owner = __ffs(__ballot_sync(0xffffffffu, a == best)) - 1;
      next = warp_max(lane == owner ? b : a);
    }
    if (lane == g) {
      first = best;
      second = next;
    }
  };
  if (p.per % 32 == 0) {   // a group is whole registers
    const int n = p.per / 32;
    Key a = 0, b = 0;
    int left = n, g = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      b = max(b, min(a, key[j]));
      a = max(a, key[j]);
      if (--left == 0) {
        if (g < p.groups) close(g, a, b);
        a = b = 0;
        left = n;
        ++g;
      }
    }
  } else {
#pragma unroll 1
    for (int g = 0; g < p.groups; ++g) {
      Key a = 0, b = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const Key x = (32 * j + lane) * p.group_of >> 20 == g ? key[j] : Key(0);
        b = max(b, min(a, x));
        a = max(a, x);
      }
      close(g, a, b);
    }
  }
  // Lane g: score of group g, and what its error goes by, |best| + |second|, of which little may be left in their sum
  const bool two = SCORES && !route_out(second);
  Key mine = route_out(first) ? Key(0) : two ? route_key(route_value(first) + route_value(second)) : first;
  const float size = fabsf((float)route_value(first)) + (two ? fabsf((float)route_value(second)) : 0.f);
  // (a group without an expert is picked when nothing else is left, which changes nothing)
  uint32_t taken = 0;
  Key last = 0;
#pragma unroll 1
  for (int i = 0; i < p.topk_group; ++i) {
    last = warp_max(mine);
    const int g = __ffs(__ballot_sync(0xffffffffu, mine == last && lane < p.groups && !(taken >> lane & 1u))) - 1;
    taken |= 1u << g;
    if (lane == g) mine = 0;
  }
  if constexpr (sizeof(Key) == 4 && SCORES) {   // every group that is left against the last one taken, as if that were off by as much as the one of the largest size
    const float most = __uint_as_float(warp_max(taken >> lane & 1u ? __float_as_uint(size) : 0u));
    sure = __all_sync(0xffffffffu, mine == 0 || route_above<V>(route_value(last), route_value(mine), 2.f * off, most + size));
  } else if constexpr (sizeof(Key) == 4) {
    const Key next = warp_max(mine);
    sure = next == 0 || (last / V) > (next / V);   // (equal up to the index)
  }
  return taken;
}
template <typename Key, int V> __device__ __forceinline__ void route_keep(const RouteParams& p, Key (&key)[V], int lane, uint32_t taken) {
  if (p.per % 32 == 0) {
    const int n = p.per / 32;
    int left = n;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (!(taken & 1u)) key[j] = 0;
      if (--left == 0) {
        left = n;
        taken >>= 1;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (!(taken >> ((32 * j + lane) * p.group_of >> 20 & 31) & 1u)) key[j] = 0;   // (places behind the last expert are out already)
  }
}

// 64-bit keys (exact, equals by the lower index) -> lane i's id is the i-th choice, -1 where there is none
template <int V, bool SCORES> __device__ __forceinline__ int route_exact(const RouteParams& p, uint64_t (&key)[V], int lane) {
  if (p.groups > 1) {
    bool sure;
    route_keep<uint64_t, V>(p, key, lane, route_groups<uint64_t, V, SCORES>(p, key, lane, 0.f, sure));
  }
  int id = -1;
#pragma unroll 1
  for (int i = 0; i < p.top_k; ++i) {
    uint64_t a = 0;
    int at = 0;
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (key[j] > a) { a = key[j]; at = j; }
    const uint64_t best = warp_max(a);
    if (best == 0) break;
    const int e = (int)__reduce_min_sync(0xffffffffu, a == best ? (unsigned)(32 * at + lane) : 0xffffffffu);
    if (lane == i) id = e;
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (32 * j + lane == e) key[j] = 0;
  }
  return id;
}

// SCORES: choices are scores and a bias; without, the logits themselves are compared
template <typename T, bool SCORES, int V>
__global__ void __launch_bounds__(128) moe_route_kernel(const RouteParams p) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  for (int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5); t < p.tokens; t += (int64_t)gridDim.x * 4) {
    const T* row = static_cast<const T*>(p.logits) + t * p.ld;
    auto least = [](float v) { return fmaxf(v, -INFINITY); };              // (a NaN becomes -infinity)
    auto logit = [&](int e) { return fminf(least(to_float<T>(row[e])), 3.402823466e+38f); };   // (+infinity is the largest number)
    float x[V];
    uint32_t key[V];   // V is a power of two: the lowest bits hold V - 1 - j
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = 32 * j + lane;
      x[j] = e < p.experts ? logit(e) : -INFINITY;
    }
    // A softmax: the largest logit and the sum, where they are needed.  (Weights that are divided by their own sum, of experts chosen by
    // their logits, go by the first choice.)
    float high = 0.f, total = 0.f;
    if (!p.sigmoid && (SCORES || !p.renormalize)) {
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) top = max(top, route_key(x[j]));
      top = warp_max(top);
      if (!route_out(top)) high = route_value(top);
      if (!p.renormalize) {
#pragma unroll
        for (int j = 0; j < V; ++j) total += expf(x[j] - high);
        total = warp_sum(total);
      }
    }
    if constexpr (SCORES) {
      float s[V];
      if (p.sigmoid) {
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = route_rcp(1.f + route_exp(-x[j]));
      } else {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          s[j] = route_exp(x[j] - high);
          sum += s[j];
        }
        sum = route_rcp(fmaxf(warp_sum(sum), 1e-30f));
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] *= sum;
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {   // (0 * x: a masked expert's choice is a NaN, and out, like that of a bias which is one)
        const float bias = 32 * j + lane < p.experts ? p.bias[32 * j + lane] : 0.f;
        key[j] = route_key(least(s[j] + fmaf(0.f, x[j], bias)));
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) key[j] = route_key(x[j]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) key[j] = (key[j] & ~(uint32_t)(V - 1)) | (uint32_t)(V - 1 - j);
    bool sure = true;
    const float off = p.sigmoid ? 0x1p-20f : 0x1p-18f;
    if (p.groups > 1) {
      const uint32_t taken = route_groups<uint32_t, V, SCORES>(p, key, lane, off, sure);
      route_keep<uint32_t, V>(p, key, lane, taken);
    }
    // A lane's keys in descending order (odd-even merge sort), so that taking one is a shift.
#pragma unroll
    for (int n = 1; n < V; n *= 2)
#pragma unroll
      for (int d = n; d > 0; d /= 2)
#pragma unroll
        for (int j = d % n; j + d < V; j += 2 * d)
#pragma unroll
          for (int i = 0; i < d; ++i)
            if (i + j + d < V && (i + j) / (2 * n) == (i + j + d) / (2 * n)) {
              const uint32_t u = key[i + j], v = key[i + j + d];
              key[i + j] = max(u, v);
              key[i + j + d] = min(u, v);
            }
    // Of equal keys the one in the lowest lane is taken: the same j, so the lowest expert.  16-bit logits lose nothing in their keys.
    // Where they may have, keys are taken until the next one is below the last for certain: these and no others can be the top_k best.
    constexpr bool CHECK = SCORES || sizeof(T) == 4;
    const bool grouped = sure;
    int id = -1, i = 0;
    uint32_t before = 0;
#pragma unroll 1
    for (; i < (CHECK ? 33 : p.top_k); ++i) {
      const uint32_t best = warp_max(key[0]);
      if (route_out(best)) break;
      if (CHECK && i > 0) {
        const bool above = SCORES ? route_above<V>(route_value(before), route_value(best), off) : (before / V) > (best / V);
        sure = sure && above;
        if (i >= p.top_k && above) break;
      }
      before = best;
      const int owner = __ffs(__ballot_sync(0xffffffffu, key[0] == best)) - 1;
      if (lane == i) id = 32 * (V - 1 - (int)(best & (V - 1))) + owner;
      if (lane == owner) {
#pragma unroll
        for (int j = 0; j + 1 < V; ++j) key[j] = key[j + 1];
        key[V - 1] = 0;
      }
    }
    if (CHECK && __builtin_expect(!sure, 0) && grouped && i < 33 && (!SCORES || p.sigmoid)) {   // (a softmax wants its sum in fp64 too)
      uint64_t mine = 0;
      if (id >= 0) {
        const double d = (double)logit(id);
        mine = route_key(SCORES ? 1.0 / (1.0 + exp(-d)) + (double)p.bias[id] : d);
      }
      int e = -1;
#pragma unroll 1
      for (int i = 0; i < p.top_k; ++i) {
        const uint64_t best = warp_max(mine);
        if (best == 0) break;
        const unsigned first = __reduce_min_sync(0xffffffffu, mine == best ? (unsigned)id : 0xffffffffu);
        if (lane == i) e = (int)first;
        if ((unsigned)id == first) mine = 0;
      }
      id = e;
    } else if (CHECK && __builtin_expect(!sure, 0)) {
      uint64_t wide[V];
      if constexpr (SCORES) {
        double s[V], all = 0.0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          s[j] = x[j] == -INFINITY ? 0.0 : exp(p.sigmoid ? -(double)x[j] : (double)x[j] - (double)high);
          all += s[j];
        }
        if (!p.sigmoid) all = warp_sum(all);
#pragma unroll
        for (int j = 0; j < V; ++j)
          wide[j] = x[j] == -INFINITY ? 0 : route_key((p.sigmoid ? 1.0 / (1.0 + s[j]) : s[j] / all) + (double)p.bias[32 * j + lane]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) wide[j] = route_key((double)x[j]);
      }
      id = route_exact<V, SCORES>(p, wide, lane);
    } else if (CHECK && lane >= p.top_k) {
      id = -1;
    }
    const float v = id >= 0 ? logit(id) : 0.f;
    if (!SCORES && p.renormalize && !p.sigmoid) high = __shfl_sync(0xffffffffu, v, 0);
    float w = 0.f;
    if (id >= 0) {
      const float d = p.sigmoid ? -fabsf(v) : v - high, b = d - v;
      float z = expf(d);
      if (!p.sigmoid && d > -200.f) z += z * ((v - (d - b)) - (high + b));   // (what the difference lost: |d| 2^-25 of z)
      w = p.sigmoid ? (v >= 0.f ? 1.f : z) / (1.f + z) : total > 0.f ? z / total : z;
    }
    if (p.renormalize) {
      const float sum = warp_sum(w);
      if (sum >= 0x1p-20f) {
        w = w / sum;
      } else {   // (sigmoids of logits around -14 and less; a softmax with a bias that chose experts so far below the row's largest: scores may leave fp32's range)
        const double d = id < 0 ? 0.0 : p.sigmoid ? 1.0 / (1.0 + exp(-(double)v)) : exp((double)v - (double)high), all = warp_sum(d);
        w = all > 0.0 ? (float)(d / all) : 0.f;
      }
    }
    if (lane < p.top_k) {
      p.weights[t * p.top_k + lane] = w * p.scale;
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
  const RouteParams p{logits, ld, bias, weights, ids, tokens, experts, top_k, groups, topk_group, sigmoid, renormalize, scale, experts / groups,
                      ((1 << 20) + experts / groups - 1) / (experts / groups)};
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
