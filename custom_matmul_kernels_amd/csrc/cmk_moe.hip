// A mixture-of-experts layer for a few tokens.
//
//   g[t][e] = sum_h x[t][h] R[e][h]          the k largest per token are chosen
//   w       = softmax over the chosen (or over all) g
//   a       = act(x G_e^T) * (x U_e^T)       G_e, U_e: rows 0..I-1, I..2I-1 of gate_up[e]
//   y[t]    = sum_j w_j (a D_e^T)            e the j-th choice of t
//
// For a few tokens the time is that of reading the chosen experts' weights once;
// everything here is laid out around that stream.
#include <algorithm>
#include <type_traits>

#include "cmk_mx4.hpp"

namespace cmk {

constexpr int kMoeTokens = 256;    // of one call
constexpr int kMoeExperts = 1024;
constexpr int kMoeChoices = 32;
constexpr int kRouterWaves = 4;
constexpr int kMoeWaves = 4;  // of the experts' kernels

// act(gate) * up goes to the down product as the sum of three bf16, which holds all 24
// bits of fp32 and its range.  Of the bf16 results of 64 tokens x 2048 x 1024 x 128
// experts 0.03 % then differ from the formula's rounded ones; with two (16 bits) it was
// 0.26 %.
constexpr int kInnerPlanes = 3;

typedef double f64x4 __attribute__((ext_vector_type(4)));

// Pieces of the workspace, each 256-byte aligned.
struct MoePlan {
  size_t logits, chosen, x, h, y, bytes;
  int Hp, Ip;      // H and I rounded up to whole slabs
  int splits;      // partial sums a logit comes in
  int x_planes;    // 16-bit planes of x
};

static MoePlan moe_plan(int T, int H, int I, int E, int k, int x_dtype, int w_dtype) {
  MoePlan p;
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  p.Hp = (int)(mx4_slabs(H) * kSlab);
  p.Ip = (int)(mx4_slabs(I) * kSlab);
  p.x_planes = x_dtype == CMK_F16 && w_dtype == CMK_MX4 ? 2 : 1;
  // a wave of the router's kernel sums 128 elements where that takes no more than
  // 16 work-groups a tile
  p.splits = std::min(16, (p.Hp / kSlab + kRouterWaves - 1) / kRouterWaves);
  size_t at = 0;
  p.logits = at; at += up((size_t)p.splits * T * E * 8);
  p.chosen = at; at += up((size_t)T * k * 4);
  p.x = at; at += up((size_t)p.x_planes * T * p.Hp * 2);
  p.h = at; at += up((size_t)kInnerPlanes * T * k * p.Ip * 2);
  p.y = at; at += up((size_t)T * k * H * 4);
  p.bytes = at;
  return p;
}

struct MoeArgs {
  const void *x, *router, *gate_up, *down;
  const uint8_t *gate_up_scales, *down_scales;
  void* y;
  float* weights;
  long long* experts;
  long long ld_x, ld_router, ld_gate_up, stride_gate_up, ld_down, stride_down;
  int T, H, I, E, k, Hp, Ip, splits;
  int act, renormalize;
  double* logits;
  int* chosen;     // [T*k]
  u16* xp;         // planes [planes][T][Hp]
  void* hp;        // fp32 [T*k][Ip], or planes [kInnerPlanes][T*k][Ip] (direct loads take them)
  float* yp;       // [T*k][H]
};

// ------------------------------------------------------------------- the router

// The planes of activations in front of 4-bit weights hold the 128 elements of a
// slab in the order in which the products take them: element q*32 + s*8 + i (block
// q of the weights, step s) at s*32 + q*8 + i.  Then a step's loads are contiguous
// for the four lanes of a row.  In front of 16-bit weights the order is natural.
template <bool four_bit>
__device__ __forceinline__ int plane_position(int k) {
  return four_bit ? (k & ~127) | (k & 24) << 2 | (k & 96) >> 2 | (k & 7) : k;
}

// Adds one slab of 16 experts x 16 tokens to the logits; `write`: this lane also
// writes its elements of x to the planes.
template <class TX, class TR, bool FOUR, int PLANES>
__device__ __forceinline__ void moe_router_slab(const MoeArgs& a, f64x4 (&acc)[2], const TX* x, const TR* w, int t, int slab, int q, bool write) {
  Octet<TX> ox[4];
  Octet<TR> ow[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int h = slab * kSlab + s * 32 + q * 8;
    ox[s] = load_octet(x + h, a.H - h);
    ow[s] = load_octet(w + h, a.H - h);
  }
  if (write) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      u16 hi[8], lo[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (PLANES == 1) {
          hi[i] = ox[s].bits(i);
        } else {
          const float f = ox[s].get(i);
          const __bf16 b = (__bf16)f;
          hi[i] = __builtin_bit_cast(u16, b);
          // an infinity or a NaN stays in the first plane alone
          lo[i] = __builtin_bit_cast(u16, (__bf16)(__builtin_isfinite(f) ? f - (float)b : 0.0f));
        }
      }
      const long long at = (long long)t * a.Hp + plane_position<FOUR>(slab * kSlab + s * 32 + q * 8);
      __builtin_memcpy(a.xp + at, hi, 16);
      if constexpr (PLANES == 2) __builtin_memcpy(a.xp + (long long)a.T * a.Hp + at, lo, 16);
    }
  }
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      acc[i & 1] = __builtin_amdgcn_mfma_f64_16x16x4f64((double)ow[s].get(i), (double)ox[s].get(i), acc[i & 1], 0, 0, 0);
}

// Logits by fp64 matrix instructions: the products of the operands are exact in
// fp64 and the sums off by 2^-53 a step, so that the order of the choice does not
// hang on the order of the sums; equal rows of the router give equal bits.  A
// work-group takes 16 experts x 16 tokens x a range of H, its waves split the
// range, and the choice adds the ranges up.  The work-groups of the first experts
// also write x as zero-padded planes for the products: its own bits, or (fp16 in
// front of 4-bit weights) the two bf16 that sum to it exactly.
template <class TX, class TR, bool FOUR, int PLANES>
__global__ __launch_bounds__(64 * kRouterWaves) void moe_logits_kernel(MoeArgs a) {
  __shared__ double part[kRouterWaves][64][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, q = lane >> 4;
  const int e0 = blockIdx.x * 16, t0 = blockIdx.y * 16;
  const int t = min(t0 + r, a.T - 1), e = min(e0 + r, a.E - 1);
  const TX* x = (const TX*)a.x + t * a.ld_x;
  const TR* w = (const TR*)a.router + e * a.ld_router;
  f64x4 acc[2] = {};
  for (int slab = blockIdx.z * kRouterWaves + wave; slab < a.Hp / kSlab; slab += a.splits * kRouterWaves)
    moe_router_slab<TX, TR, FOUR, PLANES>(a, acc, x, w, t, slab, q, blockIdx.x == 0 && t0 + r < a.T);
#pragma unroll
  for (int i = 0; i < 4; ++i) part[wave][lane][i] = acc[0][i] + acc[1][i];
  __syncthreads();
  const int l = threadIdx.x & 63, i = threadIdx.x >> 6;
  double s = 0;
#pragma unroll
  for (int v = 0; v < kRouterWaves; ++v) s += part[v][l][i];
  const int ee = e0 + (l >> 4) + 4 * i, tt = t0 + (l & 15);
  if (ee < a.E && tt < a.T) a.logits[((long long)blockIdx.z * a.T + tt) * a.E + ee] = s;
}

// Larger keys for larger logits, NaN above all; never 0.
__device__ __forceinline__ unsigned long long order_key(double v) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(v);
  if (v != v) return ~0ull;
  if (v == 0) return 0x8000000000000000ull;  // -0 equals +0
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

constexpr int kRankedExperts = 256;

// The choice of a token, by a work-group of 256 threads.
struct MoeChoice {
  unsigned long long key[kMoeExperts];
  double logit[kMoeExperts];
  int pick[kMoeChoices];
  float raised[kMoeChoices];
  float sum;
};

// pick[0..k-1] of token t, valid after the barrier at the end.  Up to 256 experts
// each is ranked by counting those in front of it, by one, two or four neighbouring
// lanes; beyond, k rounds look for the largest that is left.
__device__ __forceinline__ void moe_choose(const MoeArgs& a, int t, MoeChoice& c) {
  const int tid = threadIdx.x;
  for (int e = tid; e < a.E; e += 256) {
    double v = 0, part[4];
    for (int s0 = 0; s0 < a.splits; s0 += 4) {
#pragma unroll
      for (int s = 0; s < 4; ++s) part[s] = s0 + s < a.splits ? a.logits[((long long)(s0 + s) * a.T + t) * a.E + e] : 0.0;
#pragma unroll
      for (int s = 0; s < 4; ++s) v += part[s];
    }
    c.logit[e] = v;
    c.key[e] = order_key(v);
  }
  __syncthreads();
  if (a.E <= kRankedExperts) {
    const int shift = a.E <= 64 ? 2 : a.E <= 128 ? 1 : 0;  // lanes per expert: 1 << shift
    const int e = tid >> shift, share = tid & ((1 << shift) - 1);
    int before = 0;
    if (e < a.E) {
      const unsigned long long mine = c.key[e];
#pragma unroll 8
      for (int o = share; o < a.E; o += 1 << shift) {
        const unsigned long long other = c.key[o];
        before += other > mine || (other == mine && o < e);
      }
    }
    if (shift > 0) before += __shfl_xor(before, 1);
    if (shift > 1) before += __shfl_xor(before, 2);
    if (e < a.E && share == 0 && before < a.k) c.pick[before] = e;
    __syncthreads();
  } else {
    for (int j = 0; j < a.k; ++j) {
      if (tid < 64) {
        unsigned long long best = 0;
        int at = 0x7fffffff;
        for (int e = tid; e < a.E; e += 64)
          if (c.key[e] > best) { best = c.key[e]; at = e; }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const unsigned long long ob = __shfl_xor(best, d);
          const int oa = __shfl_xor(at, d);
          if (ob > best || (ob == best && oa < at)) { best = ob; at = oa; }
        }
        if (tid == 0) { c.pick[j] = at; c.key[at] = 0; }
      }
      __syncthreads();
    }
  }
}

// What the weights are made of: exp of the chosen logits and, where the softmax is
// over all, its sum.  After moe_choose; valid after the barrier at the end.
__device__ __forceinline__ void moe_raise(const MoeArgs& a, MoeChoice& c) {
  const int tid = threadIdx.x;
  const double top = c.logit[c.pick[0]];
  if (tid < a.k) c.raised[tid] = expf((float)(c.logit[c.pick[tid]] - top));
  if (!a.renormalize && tid < 64) {
    float sum = 0;
    for (int e = tid; e < a.E; e += 64) sum += expf((float)(c.logit[e] - top));
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
    if (tid == 0) c.sum = sum;
  }
  __syncthreads();
}

__device__ __forceinline__ float moe_weight(const MoeArgs& a, const MoeChoice& c, int j) {
  float sum = 0;
  if (a.renormalize)
    for (int i = 0; i < a.k; ++i) sum += c.raised[i];
  else sum = c.sum;
  return c.raised[j] / sum;
}

__global__ __launch_bounds__(256) void moe_select_kernel(MoeArgs a) {
  __shared__ MoeChoice c;
  moe_choose(a, blockIdx.x, c);
  moe_raise(a, c);
  if ((int)threadIdx.x < a.k) {
    const int s = blockIdx.x * a.k + threadIdx.x;
    a.chosen[s] = c.pick[threadIdx.x];
    a.experts[s] = c.pick[threadIdx.x];
    a.weights[s] = moe_weight(a, c, threadIdx.x);
  }
}

// Router and choice in one launch, for a router of few tiles: a work-group takes 16
// tokens, a wave one of the units of 16 experts x one slab, then a token.  (7 tokens,
// 10 experts, H = 1000, 8 units: 6.4 us, as two launches 4.2 + 3.6 and one more call on
// the host; a whole layer of 4 tokens and 64 inner features in two launches and in one: 8
// units 19.9 and 19.9 us, 10 units 21.0 and 22.4, 12 units 21.6 and 23.0, 16 units 22.8 and
// 25.6.)
constexpr int kSmallUnits = 8, kSmallExperts = 128;

static bool small_router(int E, int Hp) { return E <= kSmallExperts && (E + 15) / 16 * (Hp / kSlab) <= kSmallUnits; }

template <class TX, class TR, bool FOUR, int PLANES>
__global__ __launch_bounds__(1024) void moe_router_small_kernel(MoeArgs a) {
  __shared__ double part[kSmallUnits][64][4];
  __shared__ double logit[16][kSmallExperts];
  __shared__ unsigned long long key[16][kSmallExperts];
  __shared__ int pick[16][kMoeChoices];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int t0 = blockIdx.x * 16, slabs = a.Hp / kSlab, units = (a.E + 15) / 16 * slabs;
  {
    const int t = min(t0 + r, a.T - 1);
    const TX* x = (const TX*)a.x + t * a.ld_x;
    for (int u = wave; u < units; u += 16) {
      const int tile = u / slabs;
      const TR* w = (const TR*)a.router + min(tile * 16 + r, a.E - 1) * a.ld_router;
      f64x4 acc[2] = {};
      moe_router_slab<TX, TR, FOUR, PLANES>(a, acc, x, w, t, u - tile * slabs, q, tile == 0 && t0 + r < a.T);
#pragma unroll
      for (int i = 0; i < 4; ++i) part[u][lane][i] = acc[0][i] + acc[1][i];
    }
  }
  __syncthreads();
  for (int v = threadIdx.x; v < a.E * 16; v += 1024) {
    const int e = v >> 4, t = v & 15, in = e & 15;
    double sum = 0;
    for (int s = 0; s < slabs; ++s) sum += part[(e >> 4) * slabs + s][(in & 3) * 16 + t][in >> 2];
    logit[t][e] = sum;
    key[t][e] = order_key(sum);
  }
  __syncthreads();
  const int t = t0 + wave;
  if (t < a.T) {
    for (int e = lane; e < a.E; e += 64) {
      const unsigned long long mine = key[wave][e];
      int before = 0;
#pragma unroll 8
      for (int o = 0; o < a.E; ++o) {
        const unsigned long long other = key[wave][o];
        before += other > mine || (other == mine && o < e);
      }
      if (before < a.k) pick[wave][before] = e;
    }
  }
  __syncthreads();
  if (t >= a.T) return;
  const double top = logit[wave][pick[wave][0]];
  float sum = 0;
  const int count = a.renormalize ? a.k : a.E;
  for (int e = lane; e < count; e += 64) sum += expf((float)(logit[wave][a.renormalize ? pick[wave][e] : e] - top));
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
  if (lane < a.k) {
    const int s = t * a.k + lane, e = pick[wave][lane];
    a.chosen[s] = e;
    a.experts[s] = e;
    a.weights[s] = expf((float)(logit[wave][e] - top)) / sum;
  }
}

// ------------------------------------------------------------ experts' products

// What a lane reads of 16 rows x one slab of weights, row (lane & 15), as it feeds
// four steps of the 16x16x32 matrix instruction, 8 elements each: of 16-bit
// weights 16 bytes per step (64 contiguous bytes of a row per instruction), of
// 4-bit weights one block of 32, whose quarter s belongs to step s.  A sum over k
// does not mind the order as long as both operands use the same one.
template <int WF>
struct WeightSlab {  // 16-bit weights
  u32x4v v[4];
  __device__ __forceinline__ void load(const void* base, const uint8_t*, long long, long long row, long long ld, int slab, int K) {
    const int k = slab * kSlab + ((threadIdx.x & 63) >> 4) * 8;
    const u16* p = (const u16*)base + row * ld + k;
    if (slab * kSlab + kSlab <= K) {
#pragma unroll
      for (int s = 0; s < 4; ++s) __builtin_memcpy(&v[s], p + s * 32, 16);
    } else {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const Octet<__bf16> o = load_octet((const __bf16*)p + s * 32, K - k - s * 32);
        __builtin_memcpy(&v[s], o.v, 16);
      }
    }
  }
  __device__ __forceinline__ u32x4v step(int s) const { return v[s]; }
  __device__ __forceinline__ unsigned worst(unsigned w) const { return w; }
};

template <>
struct WeightSlab<CMK_MX4> {
  u32x4v v;
  unsigned scale;
  // base: codes of the expert, rows: rows a slab
  __device__ __forceinline__ void load(const void* base, const uint8_t* scales, long long rows, long long row, long long, int slab, int) {
    const int q = (threadIdx.x & 63) >> 4;
    const long long at = slab * rows + row;
    v = *(const u32x4v*)((const uint8_t*)base + at * kSlabBytes + q * 16);
    scale = scales[at * kSlabScales + q];
  }
  __device__ __forceinline__ u32x4v step(int s) const {  // as bf16, exactly
    const float f = scale_float(scale);
    const unsigned w = v[s];
    u32x4v o;
    o[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 0));
    o[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 1));
    o[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 2));
    o[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 3));
    return o;
  }
  __device__ __forceinline__ unsigned worst(unsigned w) const { return max(w, scale); }
};

// A block that stands for NaN (scale 255) makes its row's sums NaN whatever it is
// multiplied by: the largest scale a lane has seen tells it in one instruction a slab,
// where writing NaN over the elements took more than the conversion itself (68 of 118
// vector instructions a slab; gate and up of 64 experts x 4096 x 1280, 16 tokens: 51
// and now 46 us).
__device__ __forceinline__ void raise_nan(f32x4& acc, unsigned worst) {
  if (!__any(worst == 255u)) return;
  const int lane = threadIdx.x & 63;
  worst = max(worst, (unsigned)__shfl_xor((int)worst, 16));
  worst = max(worst, (unsigned)__shfl_xor((int)worst, 32));  // of row lane % 16
#pragma unroll
  for (int i = 0; i < 4; ++i)  // a lane holds rows 4 (lane / 16) + i
    if (__shfl((int)worst, (lane >> 4) * 4 + i) == 255) acc[i] = __builtin_nanf("");
}

__device__ __forceinline__ f32x4 mfma_bf16(u32x4v a, u32x4v b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_f16(u32x4v a, u32x4v b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// fp32 as the sum of three bf16, exactly (but for bits below 2^-133).  The first is cut,
// not rounded: a value that is finite in fp32 stays so up to the end of the range.  An
// infinity or a NaN stays in the first alone.
__device__ __forceinline__ void split_f32(float v, u16& a, u16& b, u16& c) {
  const bool finite = __builtin_isfinite(v);
  const float hi = finite ? __uint_as_float(__float_as_uint(v) & 0xffff0000u) : v;
  const float rest = finite ? v - hi : 0.0f;
  const __bf16 mid = (__bf16)rest;
  a = __builtin_bit_cast(u16, (__bf16)hi);
  b = __builtin_bit_cast(u16, mid);
  c = __builtin_bit_cast(u16, (__bf16)(rest - (float)mid));
}

// The parts of eight values to LDS, `apart` bytes from each other.
__device__ __forceinline__ void stage_parts(const Octet<float>& o, char* to, int apart) {
  u16 part[kInnerPlanes][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) split_f32(o.v[i], part[0][i], part[1][i], part[2][i]);
#pragma unroll
  for (int p = 0; p < kInnerPlanes; ++p) __builtin_memcpy(to + p * apart, part[p], 16);
}

// Eight fp16 as the sum of two times eight bf16, exactly (11 bits = 8 + 3).  The
// products with activations need it that may not fit fp16.  The second is 2^-9 of the
// weight at most, and its product with the third plane of an activation (2^-16 of that)
// is below fp32's last bit: it is left out where the planes are products of their own.  An
// infinite weight comes out as NaN.
__device__ __forceinline__ void split_f16(u32x4v w, u32x4v& hi, u32x4v& lo) {
  const f16x8 f = __builtin_bit_cast(f16x8, w);
  bf16x8 h, l;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = (float)f[i];
    h[i] = (__bf16)v;
    l[i] = (__bf16)(v - (float)h[i]);
  }
  hi = __builtin_bit_cast(u32x4v, h);
  lo = __builtin_bit_cast(u32x4v, l);
}

// The expert a work-group serves and the slots t*k+j that chose it.  Returns their
// count, 0 if there is nothing to do.  The order of the list may differ from run to
// run and does not matter: a slot's column is computed by itself.
template <int W>
__device__ __forceinline__ int moe_slots(const MoeArgs& a, int unit, int* list, int& expert) {
  const int n = a.T * a.k;
  __shared__ int count, taken;
  if (threadIdx.x == 0) count = taken = 0;
  const bool by_slot = n <= a.E;  // a unit is a slot: the first one that chose an expert serves it
  expert = by_slot ? a.chosen[unit] : unit;
  __syncthreads();
  for (int s0 = threadIdx.x; s0 < n; s0 += 4 * 64 * W) {
    int c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = s0 + i * 64 * W < n ? a.chosen[s0 + i * 64 * W] : -1;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c[i] == expert) {
        list[atomicAdd(&count, 1)] = s0 + i * 64 * W;
        if (by_slot && s0 + i * 64 * W < unit) taken = 1;
      }
  }
  __syncthreads();
  return taken ? 0 : count;
}

__device__ __forceinline__ float activate(float g, int act) {
  if (act == CMK_ACT_SILU) return g / (1.0f + expf(-g));
  return 0.5f * g * (1.0f + erff(g * 0.70710678118654752f));
}

// Activations of one pass in LDS: rows of 16-bit elements, plane by plane, a row
// 16 bytes longer than what it holds so that the 16 rows of a fragment spread over
// the banks.  Where the rows do not fit whole, the pass goes through k in pieces.
constexpr int kActBytes = 36 * 1024;       // gate and up
// Down: four work-groups a compute unit where a wave takes rows of its own, one group of
// them (64 tokens x 2048 x 1024 x 128 experts, from planes: 306 us, 309 with three); three
// elsewhere.
constexpr int inner_bytes(int KS, int RG) { return (KS == 1 && RG == 1 ? 36 : 51) * 1024; }

// The products of RG groups of 16 rows of one expert's matrix with the `count`
// activation rows (at most NB * 16) that `source` gives, over the slabs of one wave
// of the KS that split them; M products (gate and up, or one) share the activations.
//
// A ring of U slabs of weights is under way in registers.  The activations come
// through LDS: vector-memory loads are awaited in the order of their issue, so that
// activations loaded between the weights would wait for weights of later slabs (and
// they are read by four waves).
//
// PACK (for few rows, PLANES * count <= NB * 16): the planes are columns of the NB
// fragments, plane p of row c at p * count + c, instead of products of their own; the
// caller adds them (add_planes).  A third (half) of the matrix instructions and LDS reads.
// Whether that is done hangs on the expert's slots alone, not on a pass's, whose members
// may differ from run to run.
//
// `source` gives rows of planes, or of fp32 that become planes on the way to LDS (two
// thirds of the bytes: 64 tokens x 2048 x 1024 x 128 experts 307 us from planes, 297 from
// fp32; 16 x 4096 x 4096 x 8 experts in 4 bits 84 and 75).
template <int WF, int PLANES, int M, int RG, int NB, int U, int KS, bool SPLIT, bool PACK, int BYTES, class Source>
__device__ __forceinline__ void moe_products(f32x4 (&acc)[M][RG][NB], const void* base, const uint8_t* scales, long long rows,
                                             const long long (&row)[M][RG], long long ld, int K, int count, Source source,
                                             long long plane, int share, bool idle, char* lds) {
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int slabs = (K + kSlab - 1) / kSlab;
  constexpr int kFragments = PACK ? 1 : PLANES;  // of a block of columns
  static_assert((BYTES / (kFragments * NB * 16) - 16) / (2 * kSlab) >= KS, "a slab for each wave");
  // slabs of all rows that LDS holds; a multiple of KS, so that a slab is summed by the
  // same wave in a pass of any size
  const int fit = (BYTES / (PLANES * count) - 16) / (2 * kSlab) / KS * KS;
  const int piece = slabs <= fit ? slabs : fit;
  const int pitch = piece * 2 * kSlab + 16;
  const int columns = PACK ? PLANES * count : count;
  const char* mine[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) mine[b] = lds + min(b * 16 + r, columns - 1) * pitch + q * 16;
  const int plane_bytes = count * pitch;
  unsigned worst[M][RG] = {};
  for (int first = 0; first < slabs; first += piece) {
    const int end = min(slabs, first + piece);
    WeightSlab<WF> w[U][M][RG];
    auto request = [&](int u, int slab) {
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int g = 0; g < RG; ++g) w[u][m][g].load(base, scales, rows, row[m][g], ld, slab, K);
    };
    if (!idle)
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (first + share + u * KS < end) request(u, first + share + u * KS);
    if (first > 0) __syncthreads();
    const int units = (end - first) * 16;  // 16-byte units of a row
    constexpr bool kFloats = std::is_same_v<decltype(source(0)), const float*>;
    for (int v = threadIdx.x; v < (kFloats ? 1 : PLANES) * count * units; v += 64 * kMoeWaves) {
      const int line = v / units, at = v - line * units;
      if constexpr (kFloats) {
        static_assert(PLANES == kInnerPlanes, "the parts of an fp32");
        Octet<float> o;
        __builtin_memcpy(o.v, source(line) + first * kSlab + at * 8, 32);
        stage_parts(o, lds + line * pitch + at * 16, plane_bytes);
      } else {
        const int c = line % count, p = line / count;
        *(u32x4v*)(lds + p * plane_bytes + c * pitch + at * 16) = *(const u32x4v*)(source(c) + p * plane + first * kSlab + at * 8);
      }
    }
    __syncthreads();
    if (!idle)
      for (int s0 = first + share; s0 < end; s0 += KS * U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int slab = s0 + u * KS;
          if (slab >= end) break;
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            // reads of four steps at a time would not fit the registers
            if constexpr (RG * NB * kFragments > 16) __builtin_amdgcn_sched_barrier(0);
            u32x4v x[NB][kFragments];
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
              for (int p = 0; p < kFragments; ++p)
                x[b][p] = *(const u32x4v*)(mine[b] + p * plane_bytes + (slab - first) * 2 * kSlab + s * 64);
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
              for (int g = 0; g < RG; ++g) {
                u32x4v f = w[u][m][g].step(s), f2;
                if constexpr (SPLIT) split_f16(w[u][m][g].step(s), f, f2);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
#pragma unroll
                  for (int p = 0; p < kFragments; ++p)
                    acc[m][g][b] = WF == CMK_F16 && !SPLIT ? mfma_f16(f, x[b][p], acc[m][g][b]) : mfma_bf16(f, x[b][p], acc[m][g][b]);
                  if constexpr (SPLIT)
#pragma unroll
                    for (int p = 0; p < std::max(1, kFragments - 1); ++p) acc[m][g][b] = mfma_bf16(f2, x[b][p], acc[m][g][b]);
                }
              }
          }
#pragma unroll
          for (int m = 0; m < M; ++m)
#pragma unroll
            for (int g = 0; g < RG; ++g) worst[m][g] = w[u][m][g].worst(worst[m][g]);
          if (slab + U * KS < end) request(u, slab + U * KS);
        }
      }
  }
  if constexpr (WF == CMK_MX4)
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int g = 0; g < RG; ++g)
#pragma unroll
        for (int b = 0; b < NB; ++b) raise_nan(acc[m][g][b], worst[m][g]);
}

// The sum of the planes that PACK left in columns of their own, in the first `count`.
template <int PLANES, int N, int NB>
__device__ __forceinline__ void add_planes(f32x4 (&acc)[N][NB], int count) {
  static_assert(NB <= 2, "columns of one or two fragments");
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float lower = 0;
#pragma unroll
      for (int p = PLANES - 1; p > 0; --p) {
        const int column = (lane & 15) + p * count, from = (lane & 48) | (column & 15);
        float v = __shfl(acc[n][0][i], from);
        if constexpr (NB == 2) {
          const float w = __shfl(acc[n][1][i], from);
          if (column >= 16) v = w;
        }
        lower += v;
      }
      acc[n][0][i] += lower;
    }
}

// Stores four values to consecutive addresses, of which `left` exist.
template <class T>
__device__ __forceinline__ void store4(T* p, const T (&v)[4], int left, bool aligned) {
  if (left >= 4 && aligned) {
    __builtin_memcpy(p, v, sizeof(v));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) p[i] = v[i];
  }
}

// Sums of the KS waves that share rows, in the order of the waves; the first of
// them gets the result.  Every wave of the work-group takes part; the LDS is the
// activations'.
template <int KS, int N, int BYTES>
__device__ __forceinline__ void join_waves(f32x4 (&acc)[N], f32x4 (*part)[N][64], int share) {
  static_assert((size_t)kMoeWaves / KS * (KS - 1) * N * 64 * 16 <= BYTES, "the partial sums fit");
  const int lane = threadIdx.x & 63;
  __syncthreads();  // the activations have been read
  if constexpr (KS > 1) {
    part += (threadIdx.x >> 6) / KS * (KS - 1);
    if (share > 0)
#pragma unroll
      for (int n = 0; n < N; ++n) part[share - 1][n][lane] = acc[n];
    __syncthreads();
    if (share == 0)
#pragma unroll
      for (int w = 0; w < KS - 1; ++w)
#pragma unroll
        for (int n = 0; n < N; ++n) acc[n] += part[w][n][lane];
    __syncthreads();
  }
}

// Where an expert's matrices lie, and which rows a lane reads; rows beyond the last
// are replaced by it.
template <int WF>
__device__ __forceinline__ const char* moe_gate_up_base(const MoeArgs& a, int expert) {
  return (const char*)a.gate_up + (WF == CMK_MX4 ? (long long)expert * (a.Hp / 2) * (2 * a.I) : expert * a.stride_gate_up * 2);
}
template <int WF>
__device__ __forceinline__ const uint8_t* moe_gate_up_scales(const MoeArgs& a, int expert) {
  return WF == CMK_MX4 ? a.gate_up_scales + (long long)expert * (a.Hp / 32) * (2 * a.I) : nullptr;
}
template <int WF>
__device__ __forceinline__ const char* moe_down_base(const MoeArgs& a, int expert) {
  return (const char*)a.down + (WF == CMK_MX4 ? (long long)expert * (a.Ip / 2) * a.H : expert * a.stride_down * 2);
}
template <int WF>
__device__ __forceinline__ const uint8_t* moe_down_scales(const MoeArgs& a, int expert) {
  return WF == CMK_MX4 ? a.down_scales + (long long)expert * (a.Ip / 32) * a.H : nullptr;
}
template <int RG>
__device__ __forceinline__ void moe_gate_up_rows(const MoeArgs& a, int i0, long long (&row)[2][RG]) {
#pragma unroll
  for (int g = 0; g < RG; ++g) {
    row[0][g] = min(i0 + g * 16 + ((int)threadIdx.x & 15), a.I - 1);
    row[1][g] = a.I + row[0][g];
  }
}
template <int RG>
__device__ __forceinline__ void moe_down_rows(const MoeArgs& a, int n0, long long (&row)[1][RG]) {
#pragma unroll
  for (int g = 0; g < RG; ++g) row[0][g] = min(n0 + g * 16 + ((int)threadIdx.x & 15), a.H - 1);
}

// act(gate) * up of a wave's rows to the inner activations, as fp32 or as planes.
template <int WF, bool PLANES, int RG, int NB>
__device__ __forceinline__ void moe_store_inner(const MoeArgs& a, const f32x4 (&acc)[2][RG][NB], const int* list, int c0, int count, int i0) {
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int c = c0 + b * 16 + r;
    if (c >= count) continue;
    const long long row = (long long)list[c] * a.Ip;
#pragma unroll
    for (int g = 0; g < RG; ++g) {
      const int i1 = i0 + g * 16 + q * 4;  // four consecutive inner features of one token
      if (i1 >= a.Ip) continue;
      const long long at = row + plane_position<WF == CMK_MX4>(i1);
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = i1 + i < a.I ? activate(acc[0][g][b][i], a.act) * acc[1][g][b][i] : 0.0f;
      if constexpr (PLANES) {
        u16 part[kInnerPlanes][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) split_f32(v[i], part[0][i], part[1][i], part[2][i]);
#pragma unroll
        for (int p = 0; p < kInnerPlanes; ++p) __builtin_memcpy((u16*)a.hp + at + (long long)p * a.T * a.k * a.Ip, part[p], 8);
      } else {
        __builtin_memcpy((float*)a.hp + at, v, 16);
      }
    }
  }
}

// A wave's rows of the slots' outputs.
template <int RG, int NB>
__device__ __forceinline__ void moe_store_outer(const MoeArgs& a, const f32x4 (&acc)[1][RG][NB], const int* list, int c0, int count, int n0) {
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int c = c0 + b * 16 + r;
    if (c >= count) continue;
    float* y = a.yp + (long long)list[c] * a.H;
#pragma unroll
    for (int g = 0; g < RG; ++g) {
      const int n = n0 + g * 16 + q * 4;
      const float v[4] = {acc[0][g][b][0], acc[0][g][b][1], acc[0][g][b][2], acc[0][g][b][3]};
      store4(y + n, v, a.H - n, (a.H & 3) == 0);
    }
  }
}

// RG * 16 gate rows and the up rows that go with them, against NB * 16 tokens of
// one expert.  KS waves split H between them; the other waves of the work-group
// take the next rows.
template <int WF, int PLANES, int KS, int RG, int NB, int U, bool PACK>
__device__ __forceinline__ void moe_gate_up_tokens(const MoeArgs& a, int expert, const int* list, int c0, int count, char* lds) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int share = wave % KS;
  const int i0 = (blockIdx.x * (kMoeWaves / KS) + wave / KS) * 16 * RG;
  long long row[2][RG];
  moe_gate_up_rows<RG>(a, i0, row);
  f32x4 acc[2][RG][NB] = {};
  auto source = [&](int c) { return a.xp + (long long)(list[c0 + c] / a.k) * a.Hp; };
  moe_products<WF, PLANES, 2, RG, NB, U, KS, false, PACK, kActBytes>(acc, moe_gate_up_base<WF>(a, expert), moe_gate_up_scales<WF>(a, expert), 2 * a.I, row, a.ld_gate_up, a.H, min(count - c0, NB * 16),
                                                    source, (long long)a.T * a.Hp, share, i0 >= a.I, lds);
  join_waves<KS, 2 * RG * NB, kActBytes>((f32x4(&)[2 * RG * NB])acc, (f32x4(*)[2 * RG * NB][64])lds, share);
  if (share == 0) {
    if constexpr (PACK) add_planes<PLANES>((f32x4(&)[2 * RG][NB])acc, count - c0);
    moe_store_inner<WF, false, RG, NB>(a, acc, list, c0, count, i0);
  }
}

template <int WF, int PLANES, int KS, int RG, int U>
__global__ __launch_bounds__(64 * kMoeWaves) void moe_gate_up_kernel(MoeArgs a) {
  __shared__ int list[kMoeTokens];
  __shared__ __attribute__((aligned(16))) char lds[kActBytes];
  int expert;
  const int count = moe_slots<kMoeWaves>(a, blockIdx.y, list, expert);
  for (int c0 = 0; c0 < count; c0 += 32) {
    if (PLANES == 2 && count <= 8) moe_gate_up_tokens<WF, PLANES, KS, RG, 1, U, PLANES == 2>(a, expert, list, c0, count, lds);
    else if (count - c0 <= 16) moe_gate_up_tokens<WF, PLANES, KS, RG, 1, U, false>(a, expert, list, c0, count, lds);
    else moe_gate_up_tokens<WF, PLANES, KS, RG, 2, U, false>(a, expert, list, c0, count, lds);
  }
}

// The same for a single token, with the choice made on the way: every work-group
// makes it for itself (one L2 read of the logits; a kernel of its own took 4 us of
// 32 at 64 experts x 2048 x 1024), the first one writes it down.
template <int WF, int PLANES, int KS, int RG, int U>
__global__ __launch_bounds__(64 * kMoeWaves) void moe_gate_up_single_kernel(MoeArgs a) {
  static_assert(sizeof(MoeChoice) <= kActBytes && kMoeWaves == 4, "the choice takes 256 threads");
  __shared__ __attribute__((aligned(16))) char lds[kActBytes];
  __shared__ int list[1];
  MoeChoice& c = *(MoeChoice*)lds;
  moe_choose(a, 0, c);
  const int expert = __builtin_amdgcn_readfirstlane(c.pick[blockIdx.y]);
  if (blockIdx.x == 0 && blockIdx.y == 0) {
    moe_raise(a, c);
    if ((int)threadIdx.x < a.k) {
      a.chosen[threadIdx.x] = c.pick[threadIdx.x];
      a.experts[threadIdx.x] = c.pick[threadIdx.x];
      a.weights[threadIdx.x] = moe_weight(a, c, threadIdx.x);
    }
  }
  if (threadIdx.x == 0) list[0] = blockIdx.y;
  __syncthreads();  // list is there and the choice has been read
  moe_gate_up_tokens<WF, PLANES, KS, RG, 1, U, PLANES == 2>(a, expert, list, 0, 1, lds);
}

// RG * 16 rows of an expert's down matrix against its slots' activations.
template <int WF, int KS, int RG, int NB, int U, bool PACK>
__device__ __forceinline__ void moe_down_tokens(const MoeArgs& a, int expert, const int* list, int c0, int count, char* lds) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int share = wave % KS;
  const int n0 = (blockIdx.x * (kMoeWaves / KS) + wave / KS) * 16 * RG;
  long long row[1][RG];
  moe_down_rows<RG>(a, n0, row);
  f32x4 acc[1][RG][NB] = {};
  auto source = [&](int c) { return (const float*)a.hp + (long long)list[c0 + c] * a.Ip; };
  moe_products<WF, kInnerPlanes, 1, RG, NB, U, KS, WF == CMK_F16, PACK, inner_bytes(KS, RG)>(
      acc, moe_down_base<WF>(a, expert), moe_down_scales<WF>(a, expert), a.H, row, a.ld_down, a.I, min(count - c0, NB * 16), source, 0,
      share, n0 >= a.H, lds);
  join_waves<KS, RG * NB, inner_bytes(KS, RG)>((f32x4(&)[RG * NB])acc, (f32x4(*)[RG * NB][64])lds, share);
  if (share == 0) {
    if constexpr (PACK) add_planes<kInnerPlanes>((f32x4(&)[RG][NB])acc, count - c0);
    moe_store_outer<RG, NB>(a, acc, list, c0, count, n0);
  }
}

// (Three work-groups a compute unit.  Four groups of rows a wave read 4 KB of codes at a
// time, with no slab ahead: 24 us at 16 tokens x 4096 x 1280 x 64 experts in 4 bits; a
// slab ahead takes 29, with fewer rows 26.)
template <int WF, int KS, int RG, int U>
__global__ __launch_bounds__(64 * kMoeWaves, 3) void moe_down_kernel(MoeArgs a) {
  __shared__ int list[kMoeTokens];
  __shared__ __attribute__((aligned(16))) char lds[inner_bytes(KS, RG)];
  int expert;
  const int count = moe_slots<kMoeWaves>(a, blockIdx.y, list, expert);
  for (int c0 = 0; c0 < count; c0 += 32) {
    if (count * kInnerPlanes <= 16) moe_down_tokens<WF, KS, RG, 1, U, true>(a, expert, list, c0, count, lds);
    else if (count * kInnerPlanes <= 32) moe_down_tokens<WF, KS, RG, 2, U, true>(a, expert, list, c0, count, lds);
    else if (count - c0 <= 16) moe_down_tokens<WF, KS, RG, 1, U, false>(a, expert, list, c0, count, lds);
    else moe_down_tokens<WF, KS, RG, 2, U, false>(a, expert, list, c0, count, lds);
  }
}

// Where experts have many tokens each, the activations of a pass do not fit LDS and
// staging them in pieces leaves the memory idle between them (8 experts of 4096 x
// 4096, 64 tokens: 230 us in bf16, 121 in 4 bits; as here 195 and 86).  These kernels
// walk k with a ring of S slabs of activations in LDS, fetched by direct loads, and the
// weights in the register ring as before; the four waves take rows of their own.  Within a
// row the 16 blocks of 16 bytes of a slab are stored at position block ^ (row & 15), so
// that the 16 rows of a fragment spread over the banks.
constexpr int kGateUpStages = 4, kDownStages = 3;
constexpr int kDenseBlocks = 2;  // blocks of 16 slots of a pass (four would leave a compute unit one work-group)

template <int WF, int PLANES, int M, int RG, int NB, int U, int S, bool SPLIT, class Source>
__device__ __forceinline__ void moe_dense_products(f32x4 (&acc)[M][RG][NB], const void* base, const uint8_t* scales, long long rows,
                                                   const long long (&row)[M][RG], long long ld, int K, int count, Source source,
                                                   long long plane, uint8_t* lds) {
  constexpr int kStage = NB * 16 * PLANES * 2 * kSlab;
  constexpr int kActs = NB * PLANES;                               // requests of a wave per slab of activations,
  constexpr int kWeights = M * RG * (WF == CMK_MX4 ? 2 : 4);       // and of weights
  // What has been requested behind a slab's activations when they are awaited: those of S
  // - 2 more slabs, and weights in the S - 1 slabs of the loop since (at first, of U slabs).
  constexpr int kBehind = (S - 2) * kActs + std::min(U, S - 1) * kWeights;
  static_assert(kBehind < 64, "the count of requests under way");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int slabs = (K + kSlab - 1) / kSlab;
  // an instruction fetches four rows of one plane; rows beyond the slots repeat the last
  const char* from[kActs];
#pragma unroll
  for (int j = 0; j < kActs; ++j) {
    const int line = (wave * kActs + j) * 4 + (lane >> 4), in = line % (NB * 16), p = line / (NB * 16);
    from[j] = (const char*)(source(min(in, count - 1)) + p * plane) + ((lane & 15) ^ (in & 15)) * 16;
  }
  auto fetch = [&](int slab) {
    uint8_t* stage = lds + slab % S * kStage;
#pragma unroll
    for (int j = 0; j < kActs; ++j)
      __builtin_amdgcn_global_load_lds((gptr)(from[j] + slab * (2LL * kSlab)), (lptr)(stage + (wave * kActs + j) * 1024), 16, 0, 0);
  };
  WeightSlab<WF> w[U][M][RG];
  auto request = [&](int u, int slab) {
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int g = 0; g < RG; ++g) w[u][m][g].load(base, scales, rows, row[m][g], ld, slab, K);
  };
  unsigned worst[M][RG] = {};
  for (int s = 0; s < S - 1 && s < slabs; ++s) fetch(s);
  asm volatile("" ::: "memory");
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (u < slabs) request(u, u);
  for (int s0 = 0; s0 < slabs; s0 += U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u;
      if (s >= slabs) break;
      // Requests are awaited in the order of their issue.  Near the end, where fewer are
      // behind (or the last, shorter slab of weights takes fewer instructions), everything
      // is awaited.
      asm volatile("" ::: "memory");
      if (s + std::max(U, S - 1) < slabs) wait_loads<kBehind>();
      else wait_loads<0>();
      wait_lds();
      meet();
      if (s + S - 1 < slabs) fetch(s + S - 1);  // into the slab before's place
      asm volatile("" ::: "memory");
      const uint8_t* stage = lds + s % S * kStage;
#pragma unroll
      for (int step = 0; step < 4; ++step) {
        u32x4v x[NB][PLANES];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int p = 0; p < PLANES; ++p)
            x[b][p] = *(const u32x4v*)(stage + ((p * NB + b) * 16 + r) * (2 * kSlab) + ((step * 4 + q) ^ r) * 16);
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int g = 0; g < RG; ++g) {
            u32x4v f = w[u][m][g].step(step), f2;
            if constexpr (SPLIT) split_f16(w[u][m][g].step(step), f, f2);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
#pragma unroll
              for (int p = 0; p < PLANES; ++p)
                acc[m][g][b] = WF == CMK_F16 && !SPLIT ? mfma_f16(f, x[b][p], acc[m][g][b]) : mfma_bf16(f, x[b][p], acc[m][g][b]);
              if constexpr (SPLIT)
#pragma unroll
                for (int p = 0; p < PLANES - 1; ++p) acc[m][g][b] = mfma_bf16(f2, x[b][p], acc[m][g][b]);
            }
          }
      }
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int g = 0; g < RG; ++g) worst[m][g] = w[u][m][g].worst(worst[m][g]);
      asm volatile("" ::: "memory");
      if (s + U < slabs) request(u, s + U);
    }
  }
  if constexpr (WF == CMK_MX4)
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int g = 0; g < RG; ++g)
#pragma unroll
        for (int b = 0; b < NB; ++b) raise_nan(acc[m][g][b], worst[m][g]);
  wait_lds();
  meet();  // the ring is free for the next pass
}

template <int WF, int PLANES, int RG, int NB, int U>
__device__ __forceinline__ void moe_gate_up_dense(const MoeArgs& a, int expert, const int* list, int c0, int count, uint8_t* lds) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i0 = (blockIdx.x * kMoeWaves + wave) * 16 * RG;
  long long row[2][RG];
  f32x4 acc[2][RG][NB] = {};
  moe_gate_up_rows<RG>(a, i0, row);
  auto source = [&](int c) { return a.xp + (long long)(list[c0 + c] / a.k) * a.Hp; };
  moe_dense_products<WF, PLANES, 2, RG, NB, U, kGateUpStages, false>(acc, moe_gate_up_base<WF>(a, expert), moe_gate_up_scales<WF>(a, expert), 2 * a.I, row,
                                                      a.ld_gate_up, a.H, min(count - c0, NB * 16), source, (long long)a.T * a.Hp, lds);
  moe_store_inner<WF, true, RG, NB>(a, acc, list, c0, count, i0);
}

template <int WF, int RG, int NB, int U>
__device__ __forceinline__ void moe_down_dense(const MoeArgs& a, int expert, const int* list, int c0, int count, uint8_t* lds) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = (blockIdx.x * kMoeWaves + wave) * 16 * RG;
  long long row[1][RG];
  f32x4 acc[1][RG][NB] = {};
  moe_down_rows<RG>(a, n0, row);
  auto source = [&](int c) { return (const u16*)a.hp + (long long)list[c0 + c] * a.Ip; };
  moe_dense_products<WF, kInnerPlanes, 1, RG, NB, U, kDownStages, WF == CMK_F16>(acc, moe_down_base<WF>(a, expert), moe_down_scales<WF>(a, expert), a.H, row,
                                                         a.ld_down, a.I, min(count - c0, NB * 16), source, (long long)a.T * a.k * a.Ip, lds);
  moe_store_outer<RG, NB>(a, acc, list, c0, count, n0);
}

template <int WF, int PLANES, int RG, int U>
__global__ __launch_bounds__(64 * kMoeWaves) void moe_gate_up_dense_kernel(MoeArgs a) {
  __shared__ int list[kMoeTokens];
  __shared__ __attribute__((aligned(16))) uint8_t lds[kGateUpStages * kDenseBlocks * 16 * PLANES * 2 * kSlab];
  int expert;
  const int count = moe_slots<kMoeWaves>(a, blockIdx.y, list, expert);
  for (int c0 = 0; c0 < count; c0 += 16 * kDenseBlocks) {
    if (count - c0 <= 16) moe_gate_up_dense<WF, PLANES, RG, 1, U>(a, expert, list, c0, count, lds);
    else moe_gate_up_dense<WF, PLANES, RG, 2, U>(a, expert, list, c0, count, lds);
  }
}

template <int WF, int RG, int U>
__global__ __launch_bounds__(64 * kMoeWaves) void moe_down_dense_kernel(MoeArgs a) {
  __shared__ int list[kMoeTokens];
  __shared__ __attribute__((aligned(16))) uint8_t lds[kDownStages * kDenseBlocks * 16 * kInnerPlanes * 2 * kSlab];
  int expert;
  const int count = moe_slots<kMoeWaves>(a, blockIdx.y, list, expert);
  for (int c0 = 0; c0 < count; c0 += 16 * kDenseBlocks) {
    if (count - c0 <= 16) moe_down_dense<WF, RG, 1, U>(a, expert, list, c0, count, lds);
    else moe_down_dense<WF, RG, 2, U>(a, expert, list, c0, count, lds);
  }
}

// y[t] = sum_j w_j y_j in the order of j; four columns a thread, the loads of eight
// choices under way at a time.
template <class T>
__global__ __launch_bounds__(256) void moe_combine_kernel(MoeArgs a) {
  const int n = (blockIdx.x * 256 + threadIdx.x) * 4, t = blockIdx.y;
  if (n >= a.H) return;
  const bool aligned = (a.H & 3) == 0;
  const float* from = a.yp + (long long)t * a.k * a.H + n;
  f32x4 sum = {};
  for (int j0 = 0; j0 < a.k; j0 += 8) {
    f32x4 v[8];
    float w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j0 + j >= a.k) break;
      const float* p = from + (long long)(j0 + j) * a.H;
      w[j] = a.weights[t * a.k + j0 + j];
      if (aligned) {
        v[j] = *(const f32x4*)p;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[j][i] = n + i < a.H ? p[i] : 0.0f;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j0 + j >= a.k) break;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] = fmaf(w[j], v[j][i], sum[i]);
    }
  }
  const T o[4] = {from_f32<T>(sum[0]), from_f32<T>(sum[1]), from_f32<T>(sum[2]), from_f32<T>(sum[3])};
  store4((T*)a.y + (long long)t * a.H + n, o, a.H - n, aligned);
}

// The down products of a single token and their weighted sum: a work-group takes 16
// rows and all the chosen experts.  A unit is one slab of one of them; the W waves
// take units in turn, a ring of U under way each, and their sums meet in LDS in the
// order of the waves.  The activations are multiplied by the weights as they are
// staged and split.
constexpr int kSingleUnits = 80;  // staged at a time: two work-groups a compute unit

template <int WF, class T, int W, int U>
__global__ __launch_bounds__(64 * W) void moe_down_single_kernel(MoeArgs a) {
  constexpr int kUnit = kInnerPlanes * 2 * kSlab;
  __shared__ __attribute__((aligned(16))) char lds[kSingleUnits * kUnit];
  __shared__ f32x4 part[W][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int row = min(n0 + r, a.H - 1);
  const int slabs = a.Ip / kSlab, units = a.k * slabs;
  f32x4 acc = {};
  unsigned worst = 0;
  for (int first = 0; first < units; first += kSingleUnits) {
    const int end = min(units, first + kSingleUnits);
    WeightSlab<WF> w[U];
    auto request = [&](int u, int unit) {
      const int j = unit / slabs, expert = a.chosen[j];
      const char* base = (const char*)a.down + (WF == CMK_MX4 ? (long long)expert * (a.Ip / 2) * a.H : expert * a.stride_down * 2);
      const uint8_t* scales = WF == CMK_MX4 ? a.down_scales + (long long)expert * (a.Ip / 32) * a.H : nullptr;
      w[u].load(base, scales, a.H, row, a.ld_down, unit - j * slabs, a.I);
    };
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (first + wave + u * W < end) request(u, first + wave + u * W);
    if (first > 0) __syncthreads();
    for (int v = threadIdx.x; v < (end - first) * (kSlab / 8); v += 64 * W) {
      const int unit = v / (kSlab / 8), at = v % (kSlab / 8) * 8;
      const long long from = (long long)(first + unit) * kSlab + at;  // units are consecutive in memory
      const float weight = a.weights[(first + unit) / slabs];
      Octet<float> o;
      __builtin_memcpy(o.v, (const float*)a.hp + from, 32);
#pragma unroll
      for (int i = 0; i < 8; ++i) o.v[i] *= weight;
      stage_parts(o, lds + unit * kUnit + at * 2, 2 * kSlab);
    }
    __syncthreads();
    for (int s0 = first + wave; s0 < end; s0 += W * U) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int unit = s0 + u * W;
        if (unit >= end) break;
        const char* x = lds + (unit - first) * kUnit + min(r >> 2, kInnerPlanes - 1) * 2 * kSlab + q * 16;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const u32x4v h = *(const u32x4v*)(x + s * 64);
          u32x4v f = w[u].step(s), f2;
          if constexpr (WF == CMK_F16) split_f16(w[u].step(s), f, f2);
          acc = mfma_bf16(f, h, acc);
          if constexpr (WF == CMK_F16) acc = mfma_bf16(f2, h, acc);
        }
        worst = w[u].worst(worst);
        if (unit + U * W < end) request(u, unit + U * W);
      }
    }
  }
  if constexpr (WF == CMK_MX4) raise_nan(acc, worst);
  part[wave][lane] = acc;
  __syncthreads();
  // four columns each hold the sums of a plane, the last four repeat one: row 4 q + i of
  // plane p in component i of lane 16 q + 4 p
  if (threadIdx.x < 16 && n0 + (int)threadIdx.x < a.H) {
    float sum = 0;
#pragma unroll
    for (int v = 0; v < W; ++v) {
      float one = 0;
#pragma unroll
      for (int p = kInnerPlanes - 1; p >= 0; --p) one += part[v][(threadIdx.x >> 2 << 4) + 4 * p][threadIdx.x & 3];
      sum += one;
    }
    ((T*)a.y)[n0 + threadIdx.x] = from_f32<T>(sum);
  }
}

static int check_moe(const cmk_moe_desc* d) {
  if (!d) return fail(CMK_ERR_INVALID_ARG, "cmk_moe: null descriptor");
  if (d->T < 0 || d->H < 1 || d->I < 1 || d->E < 1 || d->k < 1 || d->k > d->E)
    return fail(CMK_ERR_INVALID_ARG, "cmk_moe: bad extents (T=%d H=%d I=%d E=%d k=%d)", d->T, d->H, d->I, d->E, d->k);
  if (d->T > kMoeTokens || d->E > kMoeExperts || d->k > kMoeChoices)
    return fail(CMK_ERR_UNSUPPORTED, "cmk_moe: at most %d tokens, %d experts and %d choices (T=%d E=%d k=%d)", kMoeTokens,
                kMoeExperts, kMoeChoices, d->T, d->E, d->k);
  if (d->H > (1 << 20) || d->I > (1 << 20))
    return fail(CMK_ERR_UNSUPPORTED, "cmk_moe: H and I are at most %d (H=%d I=%d)", 1 << 20, d->H, d->I);
  if (d->x_dtype != CMK_BF16 && d->x_dtype != CMK_F16)
    return fail(CMK_ERR_INVALID_ARG, "cmk_moe: x must be CMK_BF16 or CMK_F16 (got %d)", d->x_dtype);
  if (d->router_dtype != CMK_F32 && d->router_dtype != d->x_dtype)
    return fail(CMK_ERR_INVALID_ARG, "cmk_moe: the router must be CMK_F32 or of x's type (got %d)", d->router_dtype);
  if (d->w_dtype != CMK_MX4 && d->w_dtype != d->x_dtype)
    return fail(CMK_ERR_INVALID_ARG, "cmk_moe: the experts must be CMK_MX4 or of x's type (got %d)", d->w_dtype);
  if (d->activation != CMK_ACT_SILU && d->activation != CMK_ACT_GELU)
    return fail(CMK_ERR_INVALID_ARG, "cmk_moe: unknown activation %d", d->activation);
  if (d->ld_x < d->H || d->ld_router < d->H)
    return fail(CMK_ERR_INVALID_ARG, "cmk_moe: leading dimension too small (ld_x=%lld ld_router=%lld)", d->ld_x, d->ld_router);
  if (d->w_dtype != CMK_MX4 && (d->ld_gate_up < d->H || d->ld_down < d->I || d->stride_gate_up < 0 || d->stride_down < 0))
    return fail(CMK_ERR_INVALID_ARG, "cmk_moe: strides of the experts too small");
  return CMK_OK;
}

}  // namespace cmk

using namespace cmk;

extern "C" size_t cmk_moe_workspace_bytes(const cmk_moe_desc* d) {
  if (check_moe(d)) return 0;
  return moe_plan(d->T, d->H, d->I, d->E, d->k, d->x_dtype, d->w_dtype).bytes;
}

extern "C" int cmk_moe(const void* x, const void* router, const void* gate_up, const uint8_t* gate_up_scales,
                       const void* down, const uint8_t* down_scales, void* y, float* weights, long long* experts,
                       const cmk_moe_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
  if (int e = check_moe(d)) return e;
  if (d->T == 0) return CMK_OK;
  if (!x || !router || !gate_up || !down || !y || !weights || !experts)
    return fail(CMK_ERR_INVALID_ARG, "cmk_moe: null pointer");
  if (d->w_dtype == CMK_MX4) {
    if (!gate_up_scales || !down_scales) return fail(CMK_ERR_INVALID_ARG, "cmk_moe: null pointer to scales");
    if (((reinterpret_cast<uintptr_t>(gate_up) | reinterpret_cast<uintptr_t>(down)) & 15) ||
        ((reinterpret_cast<uintptr_t>(gate_up_scales) | reinterpret_cast<uintptr_t>(down_scales)) & 3))
      return fail(CMK_ERR_INVALID_ARG, "cmk_moe: codes need 16-byte alignment, scales 4-byte alignment");
  }
  const MoePlan p = moe_plan(d->T, d->H, d->I, d->E, d->k, d->x_dtype, d->w_dtype);
  if (!workspace || workspace_bytes < p.bytes || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return fail(CMK_ERR_WORKSPACE, "cmk_moe: needs a 256-byte aligned workspace of %zu bytes, got %zu", p.bytes, workspace_bytes);
  char* ws = (char*)workspace;
  MoeArgs a{x, router, gate_up, down, gate_up_scales, down_scales, y, weights, experts,
            d->ld_x, d->ld_router, d->ld_gate_up, d->stride_gate_up, d->ld_down, d->stride_down,
            d->T, d->H, d->I, d->E, d->k, p.Hp, p.Ip, p.splits, d->activation, d->renormalize,
            (double*)(ws + p.logits), (int*)(ws + p.chosen), (u16*)(ws + p.x), ws + p.h, (float*)(ws + p.y)};
  hipStream_t st = (hipStream_t)stream;
  const bool r32 = d->router_dtype == CMK_F32, four = d->w_dtype == CMK_MX4;
  const bool small = d->T > 1 && small_router(d->E, p.Hp);
  auto run_router = [&](auto split_kernel, auto small_kernel) {
    if (small) {
      hipLaunchKernelGGL(small_kernel, dim3(ceil_div(d->T, 16)), dim3(1024), 0, st, a);
      return;
    }
    hipLaunchKernelGGL(split_kernel, dim3(ceil_div(d->E, 16), ceil_div(d->T, 16), p.splits), dim3(64 * kRouterWaves), 0, st, a);
    if (d->T > 1) hipLaunchKernelGGL(moe_select_kernel, dim3(d->T), dim3(256), 0, st, a);
  };
#define ROUTER(...) run_router(moe_logits_kernel<__VA_ARGS__>, moe_router_small_kernel<__VA_ARGS__>)
  if (d->x_dtype == CMK_BF16) {
    if (four) r32 ? ROUTER(__bf16, float, true, 1) : ROUTER(__bf16, __bf16, true, 1);
    else r32 ? ROUTER(__bf16, float, false, 1) : ROUTER(__bf16, __bf16, false, 1);
  } else {
    if (four) r32 ? ROUTER(_Float16, float, true, 2) : ROUTER(_Float16, _Float16, true, 2);
    else r32 ? ROUTER(_Float16, float, false, 1) : ROUTER(_Float16, _Float16, false, 1);
  }
#undef ROUTER
  if (d->T == 1) {
    auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(ceil_div(p.Ip, 16), d->k), dim3(64 * kMoeWaves), 0, st, a); };
    if (d->w_dtype == CMK_BF16) run(moe_gate_up_single_kernel<CMK_BF16, 1, 4, 1, 4>);
    else if (d->w_dtype == CMK_F16) run(moe_gate_up_single_kernel<CMK_F16, 1, 4, 1, 4>);
    else if (d->x_dtype == CMK_BF16) run(moe_gate_up_single_kernel<CMK_MX4, 1, 4, 1, 4>);
    else run(moe_gate_up_single_kernel<CMK_MX4, 2, 4, 1, 4>);
    auto down = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(ceil_div(d->H, 16)), dim3(1024), 0, st, a); };
    if (d->w_dtype == CMK_BF16) down(moe_down_single_kernel<CMK_BF16, __bf16, 16, 2>);
    else if (d->w_dtype == CMK_F16) down(moe_down_single_kernel<CMK_F16, _Float16, 16, 2>);
    else if (d->x_dtype == CMK_BF16) down(moe_down_single_kernel<CMK_MX4, __bf16, 16, 4>);
    else down(moe_down_single_kernel<CMK_MX4, _Float16, 16, 4>);
    return hip_status(hipGetLastError(), "cmk_moe launch");
  }
  const int units = d->T * d->k <= d->E ? d->T * d->k : d->E;
  // rows a work-group: 16 * rg for each of the kMoeWaves / ks groups of waves
  auto experts_kernel = [&](auto kernel, int rows, int rg, int ks) {
    hipLaunchKernelGGL(kernel, dim3(ceil_div(rows, 16 * rg * kMoeWaves / ks), units), dim3(64 * kMoeWaves), 0, st, a);
  };
  // Whether waves take rows of their own, or share k (gate and up in 16 bits always do).
  // Shared and own, us: 4 bits, 2048 x 1024, 16 units 30 and 36, 32 units 37 and 40 with
  // one slot each, 51 and 48 with four, 64 units 53 and 51; 4096 x 1280, 16 units 57 and
  // 59, 32 units 60 and 60, 86 and 77; 16 bits, 2048 x 1024, 16 units 47 and 47, 32 units
  // 72 and 72, 64 units 113 and 111.
  const bool many = units >= 32;
  // Whether k is walked with the activations in a ring (no and yes, us; slots an expert in
  // brackets).  4 bits: 64 experts x 2048 x 1024 (4) 68 and 74, (6) 72 and 75, (8) 76 and
  // 76, (12) 90 and 85; 32 x 1024 x 1024 (6) 43 and 37; 8 x 4096 x 4096 (4) 75 and 80, (6)
  // 82 and 81, (8) 88 and 81, (16) 121 and 91; 8 x 512 x 2048 (6) 30 and 33, (10) 34 and
  // 33; 4 x 512 x 512 (16) 25 and 24.
  // 16 bits read four times as much and lose more to the barrier of a slab, most where
  // rows are few: 8 x 4096 x 4096 (8) 184 and 192, (12) 199 and 199, (16) 230 and 198; 64 x
  // 2048 x 1024 (8) 172 and 189, (16) 202 and 199; 32 x 1024 x 1024 (8) 63 and 61, (12) 69
  // and 64; but 32 x 512 x 512 (16) 43 and 44, 8 x 2048 x 2048 (16) 77 and 78, (32) 111 and
  // 120, 4 x 1024 x 1024 (32) 46 and 62.
  const bool dense = four ? d->T * d->k >= (many ? 6 : 8) * d->E
                          : d->T * d->k >= 12 * d->E && (long long)d->E * std::min(d->H, d->I) >= 128LL * compute_units();
  auto dense_kernel = [&](auto kernel, int rows, int rg) {
    hipLaunchKernelGGL(kernel, dim3(ceil_div(rows, 16 * rg * kMoeWaves), units), dim3(64 * kMoeWaves), 0, st, a);
  };
  // The down products take as few groups of 16 rows a wave as let all work-groups run at
  // once, two a compute unit, and then ask for weights as far ahead as registers hold (4
  // bits, one group: four slabs 86 us, two 91).  One, two and four groups of two, two and
  // one slabs: 4 bits, 8 experts x 4096 x 4096, 64 tokens 91, 95, 126 us; 8 x 5000 x 5000, 48 tokens 149, 125, 152; 16 x 6144 x 2048,
  // 128 tokens 130, 120, 116; 64 x 2048 x 1024, 256 tokens 158, 142, 139.  One and two,
  // 16 bits: 8 x 4096 x 4096, 64 tokens 197 and 199; 64 x 2048 x 1024, 256 tokens 306 and 296.
  auto all_at_once = [&](int rg) { return d->E * ceil_div(d->H, 16 * rg * kMoeWaves) <= 2 * compute_units(); };
  if (dense) {
    if (d->w_dtype == CMK_MX4) {
      if (p.x_planes == 1) dense_kernel(moe_gate_up_dense_kernel<CMK_MX4, 1, 1, 3>, p.Ip, 1);
      else dense_kernel(moe_gate_up_dense_kernel<CMK_MX4, 2, 1, 3>, p.Ip, 1);
      if (all_at_once(1)) dense_kernel(moe_down_dense_kernel<CMK_MX4, 1, 4>, d->H, 1);
      else if (all_at_once(2)) dense_kernel(moe_down_dense_kernel<CMK_MX4, 2, 4>, d->H, 2);
      else dense_kernel(moe_down_dense_kernel<CMK_MX4, 4, 1>, d->H, 4);
    } else if (d->w_dtype == CMK_BF16) {
      dense_kernel(moe_gate_up_dense_kernel<CMK_BF16, 1, 1, 2>, p.Ip, 1);
      if (all_at_once(1)) dense_kernel(moe_down_dense_kernel<CMK_BF16, 1, 3>, d->H, 1);
      else dense_kernel(moe_down_dense_kernel<CMK_BF16, 2, 1>, d->H, 2);
    } else {
      dense_kernel(moe_gate_up_dense_kernel<CMK_F16, 1, 1, 2>, p.Ip, 1);
      if (all_at_once(1)) dense_kernel(moe_down_dense_kernel<CMK_F16, 1, 3>, d->H, 1);
      else dense_kernel(moe_down_dense_kernel<CMK_F16, 2, 1>, d->H, 2);
    }
  } else if (d->w_dtype == CMK_MX4) {
    if (p.x_planes == 1) {
      if (many) experts_kernel(moe_gate_up_kernel<CMK_MX4, 1, 1, 1, 4>, p.Ip, 1, 1);
      else experts_kernel(moe_gate_up_kernel<CMK_MX4, 1, 2, 1, 3>, p.Ip, 1, 2);
    } else {
      if (many) experts_kernel(moe_gate_up_kernel<CMK_MX4, 2, 1, 1, 3>, p.Ip, 1, 1);
      else experts_kernel(moe_gate_up_kernel<CMK_MX4, 2, 2, 1, 3>, p.Ip, 1, 2);
    }
    if (many) experts_kernel(moe_down_kernel<CMK_MX4, 1, 4, 1>, d->H, 4, 1);
    else experts_kernel(moe_down_kernel<CMK_MX4, 2, 2, 3>, d->H, 2, 2);
  } else if (d->w_dtype == CMK_BF16) {
    if (many) experts_kernel(moe_gate_up_kernel<CMK_BF16, 1, 4, 1, 1>, p.Ip, 1, 4);
    else experts_kernel(moe_gate_up_kernel<CMK_BF16, 1, 4, 1, 2>, p.Ip, 1, 4);
    if (many) experts_kernel(moe_down_kernel<CMK_BF16, 1, 1, 4>, d->H, 1, 1);
    else experts_kernel(moe_down_kernel<CMK_BF16, 2, 1, 3>, d->H, 1, 2);
  } else {
    if (many) experts_kernel(moe_gate_up_kernel<CMK_F16, 1, 4, 1, 1>, p.Ip, 1, 4);
    else experts_kernel(moe_gate_up_kernel<CMK_F16, 1, 4, 1, 2>, p.Ip, 1, 4);
    if (many) experts_kernel(moe_down_kernel<CMK_F16, 1, 1, 4>, d->H, 1, 1);
    else experts_kernel(moe_down_kernel<CMK_F16, 2, 1, 3>, d->H, 1, 2);
  }
  const dim3 out_grid(ceil_div(d->H, 1024), d->T);
  if (d->x_dtype == CMK_BF16) hipLaunchKernelGGL(moe_combine_kernel<__bf16>, out_grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(moe_combine_kernel<_Float16>, out_grid, dim3(256), 0, st, a);
  return hip_status(hipGetLastError(), "cmk_moe launch");
}
