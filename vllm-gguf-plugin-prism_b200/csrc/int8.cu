// Products of 8-bit integers on the tensor cores:  D[n, t] = sum over k of W[n, k] * Q[t, k]  in 32-bit integers (exact, whatever the
// order), and y[t, n] = D * q_scale[t] * w_scale[n] (+ bias) rounded once.
//
// The scales sit on rows, so that nothing has to be done between the first and the last value of a sum: both operands go from memory
// to the tensor core as they are (TMA boxes of 128 rows x 128 bytes, 128-byte swizzle, tcgen05.mma kind::i8, four instructions a
// box).  Weight rows sit on the 128-row side of the instruction, tokens on its column side, any multiple of 16 up to 256; so one
// token costs no more tensor time than sixteen, and what bounds small batches is the weights' way from memory.
//
// A CTA: three loaders, an MMA issuer, sixteen epilogue warps (lane = weight row = lane of tensor memory), over a ring of stages of 128
// values.  Four ways to deal out the work:
//   tiles    a CTA takes items (128 weight rows x up to 256 tokens) a grid apart, two accumulators in turn
//   pairs    two CTAs take 256 rows together (cta_group::2): each brings its 128 rows and half of the tokens, and the tensor cores of both
//            read both halves, so that a CTA's copies and shared memory carry a third less for the same product
//   split    fewer tiles than SMs: a cluster of 2, 4 or 8 CTAs shares the K of one tile.  Each sends its sums of every other's
//            rows into the other's shared memory, which then adds and stores its rows: no scratch in memory, nothing to clear, and
//            integer sums do not depend on the order
//   experts  items are (pass of an expert's tokens, 128 rows).  For the gate and up product a box holds the same 64 rows of both, 8 and
//            8 in turn: the two meet in one warp, so that act(gate) * up is formed on the way out and nothing else is stored
//
// A few tokens come as they are (FEW): the epilogue warps make their codes, each CTA the ones of its K, in shared memory while the
// weights arrive.  One launch instead of two; every CTA repeats the search for a token's largest value.
//
// What bounds it (B200): one to 64 tokens, the weights from memory and 4 to 5 us of start and end (27 tokens of 14336x4096: 59 MB in 11.9 us,
// 9.1 at the copy rate); large batches, the tensor core and the power limit (4096 tokens of 14336x4096: 149 to 155 us, 3.1 to 3.2 P operations a
// second, the tensor pipe active 93 % of the time; single CTAs 173); experts of some 250 tokens, L2 and memory (2048 tokens over 64 experts
// of 2048x1024, caches cold: 81 us for gate and up, 62 us for down, which writes 134 MB; the tensor pipe at 41 and 26 %).  Without 16-byte stores from sixteen warps and with one
// loader the same 4096 tokens took 260 us.
#include <cuda.h>
#include <math.h>

#include "int8_codes.cuh"
#include "kernels.h"
#include "raw_stream.cuh"
#include "tcgen05.cuh"

namespace gguf_b200 {

constexpr int I8_ROWS = 128, I8_BK = 128;                 // weight rows of a box, values (= bytes) of a stage
constexpr int I8_A_BYTES = I8_ROWS * I8_BK;
constexpr int I8_EPI = 16;                                // epilogue warps
constexpr int I8_THREADS = 128 + 32 * I8_EPI;             // warps 0, 2, 3 loaders, 1 MMA issuer, from 4 on epilogue
constexpr int I8_MAX_STAGES = 16;
constexpr int I8_SMS = 148;
constexpr int I8_AUX = 512 + 2 * 256 * 8 + I8_EPI * 1024 + 128 * 16;   // barriers; scale and output row of every token, of two items; 16 tokens x 32 rows a warp; work list

struct I8Params {
  int n;                   // results a token
  int w_rows;              // weight rows of an expert
  int k, nk;               // values, stages
  int m, rt, tt, tn;       // tokens; row tiles, token tiles; tokens a tile
  int stages, stage_bytes, nbuf, aux_off;
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
  const void* x;           // FEW: [m][ldx], behind the ring the codes of this CTA's K (2 KB a stage)
  int64_t ldx;
  int codes_off, recv_off; // recv_off: room for other CTAs' sums, 0: in the ring
  int* status;
};

// Four times D[tmem] (+)= A[smem] * B[smem], 32 values (bytes) each: +2 in the descriptors' 16-byte units.  PAIR: by two SMs, each with its half
// of A's rows and of B's in its own shared memory, at the same place, and its rows' sums in its own tensor memory.
template <bool PAIR> __device__ __forceinline__ void umma_i8_ss4(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate, uint32_t lead) {
#define I8_MMA4(GROUP)                                                                          \
  asm volatile(                                                                                 \
      "{\n\t.reg .pred p, q, t;\n\t.reg .b64 a, b;\n\t.reg .b32 al, bl;\n\t"                   \
      "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"             \
      "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"                                       \
      "@q tcgen05.mma.cta_group::" GROUP ".kind::i8 [%0], a, b, %4, p;\n\t"                     \
      "add.u32 al, %1, 2;\n\tadd.u32 bl, %2, 2;\n\tmov.b64 a, {al, %3};\n\tmov.b64 b, {bl, %3};\n\t" \
      "@q tcgen05.mma.cta_group::" GROUP ".kind::i8 [%0], a, b, %4, t;\n\t"                     \
      "add.u32 al, %1, 4;\n\tadd.u32 bl, %2, 4;\n\tmov.b64 a, {al, %3};\n\tmov.b64 b, {bl, %3};\n\t" \
      "@q tcgen05.mma.cta_group::" GROUP ".kind::i8 [%0], a, b, %4, t;\n\t"                     \
      "add.u32 al, %1, 6;\n\tadd.u32 bl, %2, 6;\n\tmov.b64 a, {al, %3};\n\tmov.b64 b, {bl, %3};\n\t" \
      "@q tcgen05.mma.cta_group::" GROUP ".kind::i8 [%0], a, b, %4, t;\n\t}"                    \
      ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate), "r"(lead) : "memory")
  if (PAIR) I8_MMA4("2");
  else I8_MMA4("1");
#undef I8_MMA4
}
// kind::i8 instruction descriptor: 32-bit integer sums, both operands signed, K-major, 128 rows (or a pair's 256), n columns
__device__ __forceinline__ uint32_t i8_idesc(bool pair, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)((pair ? 2 : 1) * I8_ROWS >> 4) << 24);
}
// The MMAs so far are done: tells the barrier, of a pair both CTAs'
template <bool PAIR> __device__ __forceinline__ void i8_commit(uint32_t bar, uint32_t lead) {
  if (PAIR)
    asm volatile("{\n\t.reg .pred q;\n\t.reg .b16 both;\n\tsetp.ne.b32 q, %1, 0;\n\tmov.b16 both, 3;\n\t"
                 "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], both;\n\t}" ::"r"(bar), "r"(lead) : "memory");
  else
    umma_commit(bar, lead);
}
template <bool PAIR> __device__ __forceinline__ void i8_tmem_alloc(uint32_t* slot, uint32_t cols) {
  if (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tmem_alloc(slot, cols);
    tmem_relinquish();
  }
}
template <bool PAIR> __device__ __forceinline__ void i8_tmem_dealloc(uint32_t at, uint32_t cols) {
  if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(cols) : "memory");
  else tmem_dealloc(at, cols);
}
constexpr uint32_t I8_LEADER = 0xFEFFFFFFu;   // of a shared-memory address in a cluster of two: the same place in the first CTA
// (A pair's copies go each into its own shared memory and count on the first CTA's barrier.)
template <bool PAIR> __device__ __forceinline__ void i8_box(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar, uint64_t keep) {
  if (PAIR)
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;"
                 ::"r"(dst), "l"(map), "r"(bar & I8_LEADER), "r"(x), "r"(y), "l"(keep) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "l"(keep) : "memory");
}
template <bool PAIR> __device__ __forceinline__ void i8_box5(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar, uint64_t keep) {
  if (PAIR)
    asm volatile("cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, %4, %5, %6}], [%2], %7;"
                 ::"r"(dst), "l"(map), "r"(bar & I8_LEADER), "r"(x), "r"(0), "r"(y), "r"(z), "l"(keep) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, %4, %5, %6}], [%2], %7;"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(0), "r"(y), "r"(z), "l"(keep) : "memory");
}
// How long L2 should keep what a copy brings: weights that no other tile asks for leave first, so that what the next kernel reads stays (an
// expert step of 2048 tokens moves 130 MB of hidden rows and results through L2 between its kernels)
__device__ __forceinline__ uint64_t i8_policy(bool once) {
  uint64_t p;
  if (once) asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  else asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ void i8_box_l2(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y) : "memory");
}
// mbar_wait_or, and whether it was for nothing
__device__ __forceinline__ bool i8_wait(uint32_t bar, uint32_t parity, uint32_t gave_up) {
  if (mbar_try_wait(bar, parity)) return true;
  mbar_wait_or(bar, parity, gave_up);
  return lds32(gave_up) == 0u;
}
// g sigmoid(g) by z = e^-|g|: g / (1 + z), or g z / (1 + z), relative to itself to 2^-21 for gates above -87, where z leaves the normal numbers (the fast
// exponential loses 1.4 |g| 2^-24).  1 + z is between 1 and 2, where the approximate reciprocal is off by 2^-23.
__device__ __forceinline__ float i8_silu(float g) {
  const float z = expf(-fabsf(g));
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + z));
  return (g < 0.f ? g * z : g) * r;
}
// g Phi(g) = g / 2 erfc(-g / sqrt 2), relative to itself to 2^-20 for gates of both signs (1 + erf would cancel: nothing is left of it at -6).  What
// -g / sqrt 2 lost is put back by the derivative, erfc(x + d) = erfc(x) (1 - 2 x d) for x > 0 up to a few 2^-24: at -8 it would be 64 roundings.
// (One copy: in line, eight times over, a step of 200 tokens over 32 experts took 41.3 us instead of 39.5, one of 2048 with SiLU 201 instead of 199.5.)
static __device__ __noinline__ float i8_gelu(float g) {
  constexpr float HI = 0.70710678f, LO = 1.2101617e-8f;   // 1 / sqrt 2 in two parts
  const float x = -g * HI, lost = fmaf(-g, LO, fmaf(-g, HI, -x)), y = 0.5f * g * erfcf(x);
  return x > 0.f ? fmaf(y * -2.f * x, lost, y) : y;
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
__device__ __forceinline__ void i8_store16(T* __restrict__ y, int64_t ldy, const int* to, int count, const float (&f)[16], int n, int lane, bool live, bool wide,
                                           uint8_t* stage) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < count && live) y[to[j] * ldy + n] = f[j];
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
    } else if (live) {
      for (int j = 0; j < count; ++j) y[to[j] * ldy + n] = st[j * 32 + lane];
    }
    __syncwarp();
  }
}
__device__ __forceinline__ void i8_store16(const I8Params& p, const int* to, int count, const float (&f)[16], int n, int lane, bool live, bool wide, uint8_t* stage) {
  if (p.dtype == DT_F32) i8_store16<float>(static_cast<float*>(p.y), p.ldy, to, count, f, n, lane, live, wide, stage);
  else if (p.dtype == DT_F16) i8_store16<__half>(static_cast<__half*>(p.y), p.ldy, to, count, f, n, lane, live, wide, stage);
  else i8_store16<__nv_bfloat16>(static_cast<__nv_bfloat16*>(p.y), p.ldy, to, count, f, n, lane, live, wide, stage);
}

struct I8Item {
  int n0, a_row, e;        // this CTA's first result, first row in the weights (gate and up: of the gate), expert
  int x0, rows;            // tokens
};
// Item i.  (waited: behind this thread's pdl_wait.)
template <bool GLU, bool PAIR> __device__ __forceinline__ I8Item i8_item(const I8Params& p, int i, int rank, bool waited) {
  constexpr int PER = GLU ? I8_ROWS / 2 : I8_ROWS;
  I8Item t;
  int tile;
  if (p.passes) {
    const int pass = (int)((unsigned)i / (unsigned)p.rt);
    const int4 q = waited ? p.passes[pass] : ld_older(p.passes + pass);
    tile = i - pass * p.rt;
    t.e = q.x;
    t.x0 = q.y;
    t.rows = q.z;
  } else {   // the token tiles of a row tile are neighbours
    tile = (int)((unsigned)i / (unsigned)p.tt);
    t.e = 0;
    t.x0 = (i - tile * p.tt) * p.tn;
    t.rows = min(p.tn, p.m - t.x0);
  }
  t.n0 = PAIR ? (2 * tile + rank) * PER : tile * PER;
  t.a_row = t.e * p.w_rows + t.n0;
  return t;
}
constexpr int I8_LIST = 128;   // items of a CTA that are worked out ahead, in shared memory: {a_row, x0, rows, e}
template <bool GLU, bool PAIR> __device__ __forceinline__ I8Item i8_item(const I8Params& p, const int4* list, int i, int j, int rank, bool waited) {
  if (j >= I8_LIST) return i8_item<GLU, PAIR>(p, i, rank, waited);
  const int4 q = list[j];
  I8Item t;
  t.a_row = q.x;
  t.x0 = q.y;
  t.rows = q.z;
  t.e = q.w;
  t.n0 = q.x - q.w * p.w_rows;
  return t;
}

// A copy is one box wherever it can be.  (The weights of a stage in two / four / eight boxes instead of one cost one loader 22 / 68 / 158 ns more.)
struct I8Maps {
  CUtensorMap w, q[5];   // tokens: boxes of 256, 128, 64, 32, 16 rows for experts; dense: q[0], tn rows
};
// The weights of a stage: 128 rows, or eight times 8 gate rows and the 8 up rows that go with them
template <bool GLU, bool PAIR> __device__ __forceinline__ void i8_weights(const I8Maps& maps, uint32_t at, int kb, const I8Item& t, uint32_t bar, uint64_t keep) {
  if (GLU) i8_box5<PAIR>(at, &maps.w, kb * I8_BK, t.n0 / 8, t.e, bar, keep);
  else i8_box<PAIR>(at, &maps.w, kb * I8_BK, t.a_row, bar, keep);
}
// Columns of an item's instructions, and the copies of a stage's tokens: all of them, or (dense) a pair's half
__device__ __forceinline__ int i8_columns(const I8Params& p, const I8Item& t) { return p.passes ? (t.rows + 15) & ~15 : p.tn; }
template <bool PAIR> __device__ __forceinline__ void i8_tokens(const I8Params& p, const I8Maps& maps, uint32_t at, int kb, const I8Item& t, int rank, uint32_t bar, uint64_t keep) {
  if (!p.passes) {
    i8_box<PAIR>(at, &maps.q[0], kb * I8_BK, t.x0 + (PAIR ? rank * p.tn / 2 : 0), bar, keep);
    return;
  }
  const int rows = i8_columns(p, t);
  int y = 0;
#pragma unroll
  for (int i = 0; i < 5; ++i)
    if (rows & 256 >> i) {
      i8_box<PAIR>(at + (uint32_t)(y * I8_BK), &maps.q[i], kb * I8_BK, t.x0 + y, bar, keep);
      y += 256 >> i;
    }
}

// Codes of the tokens and their scales, by the 512 threads of the epilogue: a token's threads (all of them for one token, two warps each for
// five to eight) read its row once, up to two units each (I8_FEW_VALUES), and those that have units of [k0, k1) put the codes where a TMA box of
// 16 rows with the 128-byte swizzle would have.  (Behind K the weights are zeros, whatever the codes.)
constexpr int64_t I8_FEW = 8, I8_FEW_VALUES = 32 * I8_EPI * 2 * I8Q_UNIT;
__host__ __device__ constexpr int i8_few_rows(int m) { return m <= 2 ? m : m <= 4 ? 4 : 8; }
template <typename T> __device__ __forceinline__ void i8_few_codes(const I8Params& p, int k0, int k1, uint32_t codes, float* scale, uint32_t* top_of, int tid) {
  const int lanes = 32 * I8_EPI / i8_few_rows(p.m), warps = lanes / 32, tok = tid / lanes, lane = tid % lanes;
  const bool live = tok < p.m;
  const T* x = static_cast<const T*>(p.x) + (live ? tok : 0) * p.ldx;
  const int k = live ? p.k : 0;
  T v[2][I8Q_UNIT];
  uint32_t top = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if ((h * lanes + lane) * I8Q_UNIT < k) i8q_load<T, true>(x, k, (h * lanes + lane) * I8Q_UNIT, v[h]);
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if ((h * lanes + lane) * I8Q_UNIT < k) top = i8q_top<T>(v[h], top);
  top = __reduce_max_sync(0xffffffffu, i8q_top_bits<T>(top));
  if ((tid & 31) == 0) top_of[tid >> 5] = top;
  asm volatile("bar.sync 1, %0;" ::"n"(32 * I8_EPI) : "memory");
  top = __reduce_max_sync(0xffffffffu, (tid & 31) < warps ? top_of[tok * warps + (tid & 31)] : 0u);
  const bool finite = top < 0x7f800000u, zero = !finite || top == 0;
  const float a = __uint_as_float(top);
  const I8Row w = i8q_row(zero ? 1.f : a);
  if (live && lane == 0) scale[tok] = finite ? a / 127.f : __uint_as_float(0x7fc00000u);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int at = (h * lanes + lane) * I8Q_UNIT;
    if (at < k && at >= k0 && at < k1) {
      const uint4 c = zero ? make_uint4(0, 0, 0, 0) : i8q_unit<T>(v[h], w);
      const uint32_t to = codes + (uint32_t)((at - k0) / I8_BK * 2048 + tok * 128 + ((at / 16 ^ tok) & 7) * 16);
      asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(c.x), "r"(c.y), "r"(c.z), "r"(c.w) : "memory");
    }
  }
}

// GLU: gate and up product of experts.  FewT: float, __half, __nv_bfloat16: up to eight tokens of that type (void: not so).  PAIR: by pairs of CTAs
template <bool GLU, bool PAIR, typename FewT>
__global__ void __launch_bounds__(I8_THREADS, 1) i8_kernel(const __grid_constant__ I8Maps maps, const __grid_constant__ I8Params p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // (from the shared-window address, so that the CTAs of a cluster agree about offsets)
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + p.aux_off);
  uint64_t *full = bars, *empty = bars + I8_MAX_STAGES, *accum = bars + 2 * I8_MAX_STAGES, *drained = accum + 2, *last = accum + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(accum + 7);
  volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* s_scale = reinterpret_cast<float*>(smem + p.aux_off + 512);   // [2][256]
  int* s_row = reinterpret_cast<int*>(s_scale + 512);                  // [2][256]
  uint8_t* s_stage = reinterpret_cast<uint8_t*>(s_row + 512);          // [I8_EPI][1024]
  int4* s_list = reinterpret_cast<int4*>(s_stage + I8_EPI * 1024);     // [I8_LIST]
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  constexpr bool FEW = !std::is_void<FewT>::value;
  uint64_t* coded = accum + 6;   // FEW: the codes are there

  if (threadIdx.x == 0) {
    mbar_init(coded, I8_EPI);
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&accum[s], 1);
      mbar_init(&drained[s], PAIR ? 2 * I8_EPI : I8_EPI);
    }
    *gave_up = 0;
    fence_barrier_init();
  }
  if (!PAIR && p.split > 1) cluster_arrive();   // (waited for before anything is sent)
  if (warp == 2) i8_tmem_alloc<PAIR>(tmem_slot, 512);
  // (The MMA issuer's control flow and operands are known to be the same for all lanes and stay in uniform registers -- the rank from the block's
  // number, a warp's maximum of what comes from memory, all of the tensor memory, which starts at 0 --: a stage takes 50 clocks to issue.)
  const uint32_t rank = blockIdx.x & (uint32_t)(PAIR ? 1 : p.split - 1);
  constexpr int CTAS = PAIR ? 2 : 1;
  const int first = !PAIR && p.split > 1 ? (int)blockIdx.x / p.split : (int)blockIdx.x / CTAS, step = !PAIR && p.split > 1 ? 1 << 30 : (int)gridDim.x / CTAS;
  const int kb0 = !PAIR && p.split > 1 ? (int)(p.nk * rank) / p.split : 0, kb1 = !PAIR && p.split > 1 ? (int)(p.nk * (rank + 1)) / p.split : p.nk;
  // (the work list is older than the trigger of the kernel ahead: see pdl_wait)
  const int n_items = (int)__reduce_max_sync(0xffffffffu, (unsigned)(p.passes ? ld_older(p.n_passes) * p.rt : p.rt * p.tt));
  if (p.passes && warp == 3)
    for (int j = lane; j < I8_LIST && first + j * step < n_items; j += 32) {
      const I8Item t = i8_item<GLU, PAIR>(p, first + j * step, (int)rank, false);
      s_list[j] = make_int4(t.a_row, t.x0, t.rows, t.e);
    }
  tc_fence_before();
  __syncthreads();
  if (PAIR) {   // (the partner's barriers and tensor memory are there)
    cluster_arrive();
    cluster_wait();
  }
  tc_fence_after();
  pdl_trigger();
  constexpr uint32_t tmem = 0;
  const uint32_t gave_up_s = smem_u32(const_cast<const int*>(gave_up)), full_s = smem_u32(full), empty_s = smem_u32(empty);
  const uint32_t accum_s = smem_u32(accum), drained_s = smem_u32(drained);
  auto item = [&](int i, int j, bool waited) { return p.passes ? i8_item<GLU, PAIR>(p, s_list, i, j, (int)rank, waited) : i8_item<GLU, PAIR>(p, i, (int)rank, waited); };

  float ws = 0.f, bias = 0.f, scale = 1.f, next_ws = 0.f, next_bias = 0.f;   // epilogue: of this lane's row and (scale, to) this thread's token
  int to = 0;
  if (warp == 0 || warp == 2 || warp == 3) {
    // ---------------- loaders ----------------
    // Three warps take the stages in turn: a stage's wait, announcement and two copies take one warp 440 clocks to issue, most of the 512
    // that the tensor core takes for 256 tokens.  (One loader: 470 clocks a stage from one token to 128.)
    constexpr int LOADERS = 3;
    const uint32_t lead = elect_one() ? 1u : 0u, ring = smem_u32(smem);
    const int nkb = kb1 - kb0;
    const uint64_t weights_stay = i8_policy(p.tt == 1), tokens_stay = i8_policy(false);
    int k = warp == 0 ? 0 : warp - 1, s = k, i = first, j = 0;   // stage of the item, slot, item, its number
    uint32_t ph = 0;
    auto next_item = [&] {
      while (k >= nkb && i < n_items) {
        k -= nkb;
        i += step;
        ++j;
      }
    };
    // The first weights before the activations are there: into the ring, or, if they may still be written, into L2.
    int ahead = 0;
    if (first < n_items) {
      const I8Item t = item(first, 0, false);
      const uint32_t bytes = (uint32_t)(CTAS * I8_A_BYTES + (FEW ? 0 : i8_columns(p, t) * I8_BK));   // (a pair's, on the first CTA's barrier)
      ahead = FEW && !p.settled ? nkb : min(p.stages, nkb);
      for (int g = k; g < ahead; g += LOADERS)
        if (lead) {
          if (p.settled) {
            if (rank == 0 || !PAIR) mbar_expect_tx(full_s + 8u * g, bytes);
            i8_weights<GLU, PAIR>(maps, ring + (uint32_t)(g * p.stage_bytes), kb0 + g, t, full_s + 8u * g, weights_stay);
          } else {
            i8_box_l2(&maps.w, (kb0 + g) * I8_BK, t.a_row);
          }
        }
      if (!p.settled) ahead = 0;
    }
    pdl_wait();
    next_item();
    while (i < n_items) {
      const I8Item t = item(i, j, true);
      const uint32_t bytes = (uint32_t)(CTAS * I8_A_BYTES + (FEW ? 0 : i8_columns(p, t) * I8_BK));
      for (; k < nkb; k += LOADERS) {
        const uint32_t fb = full_s + 8u * s, at = ring + (uint32_t)(s * p.stage_bytes);
        const bool weights = j > 0 || k >= ahead;
        if (weights) {
          if (!i8_wait(empty_s + 8u * s, ph ^ 1u, gave_up_s)) goto loaded;   // (no copy into a slot that may be in use)
          __syncwarp();
        }
        if (lead) {
          if (weights) {
            if (rank == 0 || !PAIR) mbar_expect_tx(fb, bytes);
            i8_weights<GLU, PAIR>(maps, at, kb0 + k, t, fb, weights_stay);
          }
          if (!FEW) i8_tokens<PAIR>(p, maps, at + I8_A_BYTES, kb0 + k, t, (int)rank, fb, tokens_stay);
        }
        s += LOADERS;
        if (s >= p.stages) { s -= p.stages; ph ^= 1u; }
      }
      next_item();
    }
  loaded:;
  } else if (warp == 1 && (rank == 0 || !PAIR)) {
    // ---------------- MMA issuer (of a pair, the first CTA's) ----------------
    const uint32_t lead = elect_one() ? 1u : 0u;
    const uint64_t d0 = umma_desc_sw128(smem_u32(smem));
    const uint32_t lo0 = (uint32_t)d0, hi = (uint32_t)(d0 >> 32), stage16 = (uint32_t)p.stage_bytes >> 4;
    int s = 0, buf = 0;
    uint32_t ph = 0, dph = 0;
    for (int i = first, j = 0; i < n_items; i += step, ++j) {
      const int cols = (int)__reduce_max_sync(0xffffffffu, (unsigned)i8_columns(p, item(i, j, false)));
      const uint32_t idesc = i8_idesc(PAIR, cols), d = tmem + (uint32_t)(buf * p.tn);
      const uint32_t codes0 = (uint32_t)umma_desc_sw128(smem_u32(smem + p.codes_off));
      if (FEW) mbar_wait_or(smem_u32(coded), 0u, gave_up_s);
      mbar_wait_or(drained_s + 8u * buf, dph ^ 1u, gave_up_s);
      for (int kb = kb0; kb < kb1; ++kb) {
        mbar_wait_or(full_s + 8u * s, ph, gave_up_s);
        __syncwarp();
        tc_fence_after();
        const uint32_t a = lo0 + (uint32_t)s * stage16;
        umma_i8_ss4<PAIR>(d, a, FEW ? codes0 + (uint32_t)(kb - kb0) * (2048 >> 4) : a + (I8_A_BYTES >> 4), hi, idesc, kb > kb0, lead);
        i8_commit<PAIR>(empty_s + 8u * s, lead);
        if (++s == p.stages) { s = 0; ph ^= 1u; }
      }
      i8_commit<PAIR>(accum_s + 8u * buf, lead);
      if (++buf == p.nbuf) { buf = 0; dph ^= 1u; }
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ---------------- epilogue ----------------
    // (a warp reaches the 32 lanes of tensor memory of its number modulo 4; four warps share them, taking 16 columns in turn)
    const int quad = (warp & 3) * 32, row = quad + lane, turn16 = 16 * ((warp - 4) >> 2), tid = threadIdx.x - 128;
    const uint32_t t_lane = tmem + ((uint32_t)quad << 16);
    uint8_t* stage = s_stage + (warp - 4) * 1024;
    const bool wide_y = p.dtype != DT_F32 && p.ldy % 8 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0;
    int buf = 0, turn = 0;
    uint32_t aph = 0;
    // this lane's row: of 128, or, gate and up, of 64 gate rows or (lanes with bit 3) their up rows
    const int r = GLU ? quad / 2 + (lane >> 4) * 8 + (lane & 7) : row;
    const bool down = !GLU && p.passes;
    // What an item's end looks up in memory, a token a thread and a row a lane: asked for while the item before it is on its way out.
    auto older = [](const float* q) { return __int_as_float(ld_older(reinterpret_cast<const int32_t*>(q))); };
    // (a token's scale is written by the kernel ahead: behind the wait only)
    auto look_up = [&](const I8Item& t, bool waited) {
      const int at = t.x0 + tid, n = t.n0 + r;
      const bool mine = tid < t.rows, live = n < p.n;
      scale = !FEW && waited && mine ? p.q_scale[at] : 1.f;
      to = !(down && mine) ? at : waited ? p.sorted[at] : ld_older(p.sorted + at);
      const float* w = p.w_scale + t.a_row + r + (GLU && (lane & 8) ? p.n : 0);
      next_ws = !live ? 0.f : waited ? *w : older(w);
      next_bias = !GLU && live ? i8_bias(p, n) : 0.f;
    };
    if (down && first < n_items) look_up(item(first, 0, false), false);
    pdl_wait();
    if (!FEW && !down && first < n_items) look_up(item(first, 0, true), true);
    if (down && first < n_items) {
      const I8Item t = item(first, 0, true);
      if (tid < t.rows) scale = p.q_scale[t.x0 + tid];
    }
    for (int i = first, j = 0; i < n_items; i += step, ++j) {
      const I8Item t = item(i, j, true);
      float* xs = s_scale + (FEW ? 0 : turn * 256);   // (in turn: whoever has passed the last item's barrier is done with those of the item before it)
      int* xr = s_row + turn * 256;
      turn ^= 1;
      if (tid < p.tn) {
        if (!FEW) xs[tid] = scale;
        xr[tid] = FEW ? t.x0 + tid : to;
      }
      if constexpr (FEW) if (i == first) {   // (the same for all of a CTA's items)
        i8_few_codes<FewT>(p, kb0 * I8_BK, kb1 * I8_BK, smem_u32(smem + p.codes_off), xs, reinterpret_cast<uint32_t*>(s_stage), tid);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(coded);
        look_up(t, true);   // (not ahead of the codes: they would wait for it)
      }
      const int n = t.n0 + r;
      const bool live = n < p.n, wide = wide_y && t.n0 + quad + 32 <= p.n;
      ws = next_ws;
      bias = next_bias;
      asm volatile("bar.sync 1, %0;" ::"n"(32 * I8_EPI) : "memory");
      if (i + step < n_items) look_up(item(i + step, j + 1, true), true);
      mbar_wait_or(accum_s + 8u * buf, aph, gave_up_s);
      __syncwarp();
      tc_fence_after();
      if (p.split == 1) {
        const uint32_t d = t_lane + (uint32_t)(buf * p.tn);
        for (int c0 = turn16; c0 < t.rows; c0 += 4 * I8_EPI) {
          uint32_t v[16];
          tmem_ld16(d + (uint32_t)c0, v);
          float f[16];
          float4 x[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] = reinterpret_cast<const float4*>(xs + c0)[j];
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) f[j] = (float)(int)v[j] * (reinterpret_cast<const float*>(x)[j] * ws) + bias;
          const int count = min(16, t.rows - c0);
          if (GLU) {   // of two tokens, the lanes of the gate take the first and those of up the second
            const bool up = (lane & 8) != 0;
            float g[8], u[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float got = __shfl_xor_sync(0xffffffffu, up ? f[2 * j] : f[2 * j + 1], 8);
              g[j] = up ? got : f[2 * j];
              u[j] = up ? f[2 * j + 1] : got;
            }
            if (p.act == 1) {
#pragma unroll
              for (int j = 0; j < 8; ++j) u[j] *= i8_silu(g[j]);
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j) u[j] *= i8_gelu(g[j]);
            }
            float* y = static_cast<float*>(p.y) + (t.x0 + c0 + (up ? 1 : 0)) * p.ldy + n;
            const int left = live ? count - (up ? 1 : 0) : 0;
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (2 * j < left) y[2 * j * p.ldy] = u[j];
          } else {
            i8_store16(p, xr + c0, count, f, n, lane, live, wide, stage);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (PAIR)
            asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"((drained_s + 8u * buf) & I8_LEADER) : "memory");
          else
            mbar_arrive(drained_s + 8u * buf);
        }
      }
      if (++buf == p.nbuf) { buf = 0; aph ^= 1u; }
    }
  }
  __syncwarp();
  if (!GLU && !PAIR && p.split > 1) {
    // ---------------- split: the sums of rows [per * rank, per * (rank + 1)) of the tile are this CTA's to add and store ----------------
    // The rows of another CTA go into its shared memory, [sender][row][token], rows 16 bytes more than tn words apart (eight lanes' 16 bytes then
    // lie in different banks).  A lane keeps its row to the end.
    cluster_wait();
    if (p.recv_off == 0) {   // every CTA's products have to be complete, so that its ring is free
      cluster_arrive();
      cluster_wait();
    }
    const I8Item t = i8_item<false, false>(p, first, 0, true);
    const int per = I8_ROWS / p.split, shift = 31 - __clz(per), quad = (warp & 3) * 32, row = quad + lane, owner = row >> shift;
    const int turn16 = 16 * ((warp - 4) >> 2);
    const uint32_t d = tmem + ((uint32_t)quad << 16), pitch = 4u * (uint32_t)p.tn + 16u, ring = smem_u32(smem + p.recv_off);
    const bool mine = owner == (int)rank;
    if (warp >= 4 && !(p.split <= 4 && mine)) {   // (whole warps of a quad, unless 16 rows are a CTA's)
      const uint32_t slot = rank - (owner < (int)rank ? 1u : 0u);   // (senders in order, without the owner)
      uint32_t peer;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(ring + (slot * (uint32_t)per + (uint32_t)(row & (per - 1))) * pitch), "r"(owner));
      for (int c0 = turn16; c0 < t.rows; c0 += 4 * I8_EPI) {
        uint32_t v[16];
        tmem_ld16(d + (uint32_t)c0, v);
        tmem_ld_wait();
        if (!mine) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(peer + 4u * (uint32_t)(c0 + 4 * j)), "r"(v[4 * j]), "r"(v[4 * j + 1]), "r"(v[4 * j + 2]),
                         "r"(v[4 * j + 3]) : "memory");
        }
      }
    }
    cluster_arrive();
    cluster_wait();
    if (warp >= 4 && (p.split == 8 ? quad >> 5 == (int)rank >> 1 : mine)) {
      const int n = t.n0 + row;
      const bool live = mine && n < p.n, wide = p.split <= 4 && p.dtype != DT_F32 && p.ldy % 8 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0 && t.n0 + quad + 32 <= p.n;
      const uint32_t from0 = ring + (uint32_t)(row & (per - 1)) * pitch;
      for (int c0 = turn16; c0 < t.rows; c0 += 4 * I8_EPI) {
        uint32_t v[16];
        tmem_ld16(d + (uint32_t)c0, v);
        tmem_ld_wait();
        for (int from = 0; from < p.split - 1; ++from) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 w = lds128s(from0 + (uint32_t)(from * per) * pitch + 4u * (uint32_t)(c0 + 4 * j));
            v[4 * j] += w.x;
            v[4 * j + 1] += w.y;
            v[4 * j + 2] += w.z;
            v[4 * j + 3] += w.w;
          }
        }
        float f[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) f[j] = (float)(int)v[j] * (s_scale[c0 + j] * ws) + bias;
        i8_store16(p, s_row + c0, min(16, t.rows - c0), f, n, lane, live, wide, s_stage + (warp - 4) * 1024);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*gave_up) {
    if (threadIdx.x == 0) atomicExch(p.status, E_TIMEOUT);
    // A bounded wait ran out in this CTA.  What it started has to finish before its tensor memory is given up: the commit covers the
    // tensor pipe, and the copies in flight land within microseconds.
    if (warp == 1 && (rank == 0 || !PAIR)) {
      if (lane == 0) mbar_init(last, 1);
      __syncwarp();
      if (PAIR) {
        if (elect_one()) asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(last)) : "memory");
      } else if (elect_one()) umma_commit(last);
      __syncwarp();
      mbar_wait_bounded(last, 0);
    }
    drain_pause();
    tc_fence_before();
    __syncthreads();
  }
  if (PAIR) {   // (the partner's shared memory and tensor memory are in use until here)
    cluster_arrive();
    cluster_wait();
  }
  if (warp == 2) i8_tmem_dealloc<PAIR>(tmem, 512);
}

// rows of k bytes in boxes of box_rows; experts > 0: [experts][gate, up][rows / 8][8] in boxes of eight times 8 gate and 8 up rows
static bool i8_map(CUtensorMap& map, const void* base, int64_t k, int64_t rows, int64_t pitch, int box_rows, int64_t experts = 0) {
  EncodeTiledFn enc = tensor_map_encoder();
  if (!enc) return false;
  const cuuint32_t one[5] = {1, 1, 1, 1, 1};
  auto encode = [&](int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
    return enc(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  if (experts) {
    const cuuint64_t dims[5] = {(cuuint64_t)k, 8, 2, (cuuint64_t)rows / 8, (cuuint64_t)experts};
    const cuuint64_t strides[4] = {(cuuint64_t)pitch, (cuuint64_t)(rows * pitch), (cuuint64_t)(8 * pitch), (cuuint64_t)(2 * rows * pitch)};
    const cuuint32_t box[5] = {I8_BK, 8, 2, 8, 1};
    return encode(5, dims, strides, box);
  }
  const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch};
  const cuuint32_t box[2] = {I8_BK, (cuuint32_t)box_rows};
  return encode(2, dims, strides, box);
}

template <bool GLU, bool PAIR, typename FewT> static int i8_launch(const I8Maps& maps, const I8Params& p, int grid, size_t smem, cudaStream_t stream) {
  static bool configured[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return E_CUDA;
  if (!configured[dev & 63]) {
    if (cudaFuncSetAttribute(i8_kernel<GLU, PAIR, FewT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess) return E_CUDA;
    configured[dev & 63] = true;
  }
  return launch_pdl_cluster(i8_kernel<GLU, PAIR, FewT>, dim3((unsigned)grid), dim3(I8_THREADS), PAIR ? 2u : (unsigned)p.split, smem, stream, maps, p) == cudaSuccess ? E_OK : E_CUDA;
}

// How a dense product is dealt out: tokens a tile, whether pairs of CTAs take 256 rows together, how many CTAs share a tile's K.  What takes
// the least time by this model, in us on a chip that is not held back by its power limit: a stage 0.09 + 0.00088 a token (a pair: 0.065 +
// 0.00092), 5 for start and end (a pair 0.8 more), 0.012 a token for the last tile's way out, 2.8 + 0.012 a token for an exchange of sums
// (1 more by four or eight), and no less than its copies take from L2 at 17.5 TB/s.
// Measured, single / pair / shared by two: 500 tokens of 4096x14336 27.5 (tiles of 128) / 25.9 (128) / 30.4 (256); of 4096x4096 10.7 / 11.5 /
// 17.1; of 14336x4096 28.7 (256) / 26.1 (256); 1000 tokens of 4096x4096 16.3 (256) / 16.6 (128); 4096 tokens of 14336x4096 173 / 149.  Whole / by
// two / by four: 1 token of 4096x4096 6.6 / 7.7 / 7.9, of 4096x14336 15.3 / 13.6 / 12.3; 128 tokens of 4096x4096 9.7 / 11.1 / 12.1.
struct I8Deal {
  int tn, tt, split;
  bool pair;
};
// A few tokens (their product begins when the codes are made): a stage 0.127, an exchange 1.65 / 2.1 / 2.7 by two / four / eight, and no less than
// the weights at 9 TB/s.  (Whole / by two / by four / by eight: 1 token of 1024x4096 6.5 / 6.2 / 5.6 / 5.7, of 4096x4096 7.1 / 6.8 / 7.1, of 2048x2048 4.8 /
// 5.4 / 5.2.)
static I8Deal i8_deal_few(int64_t n, int nk) {
  const int64_t tiles = (n + I8_ROWS - 1) / I8_ROWS;
  const float exchange[4] = {0.f, 1.65f, 2.1f, 2.7f}, weights = (float)tiles * (float)nk * (float)I8_A_BYTES / 9e6f;
  I8Deal best{16, 1, 1, false};
  float least = INFINITY;
  for (int i = 0; i < 4 && (i == 0 || (tiles << i <= I8_SMS && nk >= 4 << i)); ++i) {
    const float t = fmaxf((float)((nk + (1 << i) - 1) >> i) * 0.127f, weights) + exchange[i];
    if (t < least) {
      least = t;
      best.split = 1 << i;
    }
  }
  return best;
}
static I8Deal i8_deal(int64_t m, int64_t n, int nk) {
  I8Deal best{};
  float least = INFINITY;
  for (int most = 256; most >= 32; most -= 32) {
    const int64_t tt = (m + most - 1) / most, each = (m + tt - 1) / tt;
    if (tt > 1 && most < 256 && tt == (m + most + 31) / (most + 32)) continue;   // (as the tile size before)
    for (int pair = 0; pair < 2; ++pair) {
      const int tn = (int)round_up(each, pair ? 32 : 16), rows = pair ? 2 * I8_ROWS : I8_ROWS;
      const int64_t tiles = (n + rows - 1) / rows * tt, slots = pair ? I8_SMS / 2 : I8_SMS;
      for (int split = 1; split <= (pair ? 1 : 8) && (split == 1 || (tiles * split <= slots && nk >= 4 * split)); split *= 2) {
        const float stage = pair ? 0.065f + 0.00092f * tn : 0.09f + 0.00088f * tn;
        const int64_t waves = split > 1 ? 1 : (tiles + slots - 1) / slots;
        const float copied = (float)tiles * (float)nk * (float)(rows + tn) * (float)I8_BK / 17.5e6f;
        const float t = fmaxf(waves * ((nk + split - 1) / split) * stage, copied) + (pair ? 0.8f : 0.f) + 0.012f * tn + (split > 1 ? 2.8f + 0.012f * tn : 0.f) + (split > 2 ? 1.f : 0.f);
        if (t < least) {
          least = t;
          best = I8Deal{tn, (int)tt, split, pair != 0};
        }
      }
    }
    if (each <= 32) break;
  }
  return best;
}
// Whether a product of m tokens is one launch: rows that 16-byte loads can start at, the codes of a CTA's K (2 KB a stage) leave half of its
// shared memory to the weights, and finding the tokens' largest values, which every CTA repeats, takes less than a launch.  (One / two
// launches in us, 4096x4096: 1 token 6.8 / 8.6, 4 tokens 7.4 / 8.6, 8 tokens 9.4 / 8.6; 4096x14336, 1 token 13.6 / 15.5, 8 tokens 27 / 15.5.)
bool i8_few(const void* x, int dtype, int64_t ldx, int64_t m, int64_t n, int64_t k) {
  const int64_t size = dtype == DT_F32 ? 4 : 2, nk = (k + I8_BK - 1) / I8_BK;
  if (m > I8_FEW || i8_few_rows((int)m) * k > I8_FEW_VALUES || (reinterpret_cast<uintptr_t>(x) & 15) != 0 || (m > 1 && ldx * size % 16 != 0)) return false;
  const int split = i8_deal_few(n, (int)nk).split;
  return (nk + split - 1) / split <= 48;
}

int launch_i8_product(const I8Product& a, cudaStream_t stream) {
  const bool glu = a.act != 0, few = a.x != nullptr;
  const int per_tile = glu ? I8_ROWS / 2 : I8_ROWS;   // results a row tile
  I8Params p{};
  p.n = (int)a.n;
  p.w_rows = (int)(a.n * (glu ? 2 : 1));
  p.k = (int)a.k;
  p.nk = (int)((a.k + I8_BK - 1) / I8_BK);
  p.m = (int)a.m;
  // (experts: pairs, and passes of 144 to 256 tokens, make no difference: 2048 tokens over 64 experts 177 to 181 us throughout)
  const I8Deal deal = a.passes ? I8Deal{(int)a.pass_rows, 1, 1, false} : few ? i8_deal_few(a.n, p.nk) : i8_deal(a.m, a.n, p.nk);
  const bool pair = deal.pair;
  p.rt = (int)((a.n + per_tile * (pair ? 2 : 1) - 1) / (per_tile * (pair ? 2 : 1)));
  p.tn = deal.tn;
  p.tt = deal.tt;
  p.split = deal.split;
  p.stage_bytes = I8_A_BYTES + (few ? 0 : p.tn * I8_BK / (pair ? 2 : 1));
  const int64_t tiles = a.passes ? a.max_passes * p.rt : (int64_t)p.rt * p.tt;
  if (tiles > 1 << 29) return E_TOO_LARGE;
  // shared memory: ring, barriers and scales, codes of a few tokens, sums of other CTAs where they are small
  const int recv = p.split > 1 ? I8_ROWS / p.split * (p.split - 1) * (4 * p.tn + 16) : 0;
  const int codes = few ? (p.nk + p.split - 1) / p.split * 2048 : 0;
  const int extra = I8_AUX + codes + (recv <= 32768 ? (int)round_up(recv, 1024) : 0);
  p.stages = (226 * 1024 - extra) / p.stage_bytes;
  if (p.stages > I8_MAX_STAGES) p.stages = I8_MAX_STAGES;
  const int ring = p.stages * p.stage_bytes;
  p.codes_off = ring;
  p.recv_off = recv > 0 && recv <= 32768 ? ring + codes : 0;
  p.aux_off = ring + extra - I8_AUX;
  p.nbuf = p.split == 1 && 2 * p.tn <= 512 ? 2 : 1;
  p.y = a.y;
  p.ldy = a.ldy;
  p.dtype = a.dtype;
  p.w_scale = a.w_scale;
  p.q_scale = a.q_scale;
  p.bias = a.bias;
  p.settled = a.settled || a.passes;
  p.passes = static_cast<const int4*>(a.passes);
  p.n_passes = a.n_passes;
  p.act = a.act;
  p.sorted = a.sorted;
  p.x = a.x;
  p.ldx = a.ldx;
  p.status = a.status;
  const int64_t slots = pair ? I8_SMS / 2 : I8_SMS, grid = p.split > 1 ? tiles * p.split : (tiles < slots ? tiles : slots) * (pair ? 2 : 1);
  I8Maps maps;
  if (!i8_map(maps.w, a.w, a.k, glu ? a.n : a.experts * p.w_rows, a.ldw, I8_ROWS, glu ? a.experts : 0)) return E_CUDA;
  for (int i = 0; i < (few ? 0 : a.passes ? 5 : 1); ++i)
    if (!i8_map(maps.q[i], a.q, a.k, a.m, a.ldq, a.passes ? 256 >> i : p.tn / (pair ? 2 : 1))) return E_CUDA;
  const size_t smem = 1024 + (size_t)p.aux_off + I8_AUX;
  if (glu) return i8_launch<true, false, void>(maps, p, (int)grid, smem, stream);
  if (pair) return i8_launch<false, true, void>(maps, p, (int)grid, smem, stream);
  if (!few) return i8_launch<false, false, void>(maps, p, (int)grid, smem, stream);
  switch (a.dtype) {
    case DT_F32: return i8_launch<false, false, float>(maps, p, (int)grid, smem, stream);
    case DT_F16: return i8_launch<false, false, __half>(maps, p, (int)grid, smem, stream);
    default: return i8_launch<false, false, __nv_bfloat16>(maps, p, (int)grid, smem, stream);
  }
}

}  // namespace gguf_b200
