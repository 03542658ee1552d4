// A mixture-of-experts layer for a few tokens.
//
//   g[t][e] = sum_h x[t][h] R[e][h]          the k largest per token are chosen
//   w       = softmax over the chosen (or over all) g
//   a       = act(x G_e^T) * (x U_e^T)       G_e, U_e: rows 0..I-1, I..2I-1 of gate_up[e]
//   y[t]    = sum_j w_j (a D_e^T)            e the j-th choice of t
//
// For a few tokens the time is that of reading the chosen experts' weights once;
// everything here is laid out around that stream.
#include "cmk_mx4.hpp"

namespace cmk {

constexpr int kMoeTokens = 256;    // of one call
constexpr int kMoeExperts = 1024;
constexpr int kMoeChoices = 32;

typedef double f64x4 __attribute__((ext_vector_type(4)));

// Pieces of the workspace, each 256-byte aligned.
struct MoePlan {
  size_t logits, chosen, x, h, y, bytes;
  int Hp, Ip;      // H and I rounded up to whole slabs
  int x_planes;    // 16-bit planes of x
};

static MoePlan moe_plan(int T, int H, int I, int E, int k, int x_dtype, int w_dtype) {
  MoePlan p;
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  p.Hp = (int)(mx4_slabs(H) * kSlab);
  p.Ip = (int)(mx4_slabs(I) * kSlab);
  p.x_planes = x_dtype == CMK_F16 && w_dtype == CMK_MX4 ? 2 : 1;
  size_t at = 0;
  p.logits = at; at += up((size_t)T * E * 8);
  p.chosen = at; at += up((size_t)T * k * 4);
  p.x = at; at += up((size_t)p.x_planes * T * p.Hp * 2);
  p.h = at; at += up((size_t)2 * T * k * p.Ip * 2);
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
  int T, H, I, E, k, Hp, Ip;
  int act, renormalize;
  double* logits;
  int* chosen;     // [T*k]
  u16 *xp, *hp;    // planes [planes][T][Hp], [2][T*k][Ip]
  float* yp;       // [T*k][H]
};

// ------------------------------------------------------------------- the router

// Logits by fp64 matrix instructions: the products of the operands are exact in
// fp64 and the sums off by 2^-53 a step, so that the order of the choice does not
// hang on the order of the sums; equal rows of the router give equal bits.  A
// work-group takes 16 experts x 16 tokens, its waves split H; the work-groups of
// the first experts also write x as zero-padded planes for the products: its own
// bits, or (fp16 in front of 4-bit weights) the two bf16 that sum to it exactly.
template <class TX, class TR, int PLANES>
__global__ __launch_bounds__(512) void moe_logits_kernel(MoeArgs a) {
  __shared__ double part[8][64][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, q = lane >> 4;
  const int e0 = blockIdx.x * 16, t0 = blockIdx.y * 16;
  const int t = min(t0 + r, a.T - 1), e = min(e0 + r, a.E - 1);
  const TX* x = (const TX*)a.x + t * a.ld_x;
  const TR* w = (const TR*)a.router + e * a.ld_router;
  f64x4 acc = {0, 0, 0, 0};
  for (int h0 = wave * 32; h0 < a.Hp; h0 += 8 * 32) {
    const int h = h0 + q * 8;
    const Octet<TX> ox = load_octet(x + h, a.H - h);
    const Octet<TR> ow = load_octet(w + h, a.H - h);
    if (blockIdx.x == 0 && t0 + r < a.T) {
      u16 hi[8], lo[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (PLANES == 1) {
          hi[i] = ox.bits(i);
        } else {
          const float f = ox.get(i);
          const __bf16 b = (__bf16)f;
          hi[i] = __builtin_bit_cast(u16, b);
          // an infinity or a NaN stays in the first plane alone
          lo[i] = __builtin_bit_cast(u16, (__bf16)(__builtin_isfinite(f) ? f - (float)b : 0.0f));
        }
      }
      __builtin_memcpy(a.xp + (long long)t * a.Hp + h, hi, 16);
      if constexpr (PLANES == 2) __builtin_memcpy(a.xp + ((long long)a.T + t) * a.Hp + h, lo, 16);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)ow.get(i), (double)ox.get(i), acc, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) part[wave][lane][i] = acc[i];
  __syncthreads();
  if (threadIdx.x < 256) {
    const int l = threadIdx.x & 63, i = threadIdx.x >> 6;
    double s = 0;
#pragma unroll
    for (int v = 0; v < 8; ++v) s += part[v][l][i];
    const int ee = e0 + (l >> 4) + 4 * i, tt = t0 + (l & 15);
    if (ee < a.E && tt < a.T) a.logits[(long long)tt * a.E + ee] = s;
  }
}

// Larger keys for larger logits, NaN above all; never 0.
__device__ __forceinline__ unsigned long long order_key(double v) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(v);
  if (v != v) return ~0ull;
  if (v == 0) return 0x8000000000000000ull;  // -0 equals +0
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

// A wave per token: k rounds of the largest key that is left, the lowest index of
// equal ones.
__global__ __launch_bounds__(64) void moe_select_kernel(MoeArgs a) {
  __shared__ unsigned long long key[kMoeExperts];
  __shared__ int pick[kMoeChoices];
  const int t = blockIdx.x, lane = threadIdx.x;
  const double* logits = a.logits + (long long)t * a.E;
  for (int e = lane; e < a.E; e += 64) key[e] = order_key(logits[e]);
  __syncthreads();
  for (int j = 0; j < a.k; ++j) {
    unsigned long long best = 0;
    int at = 0x7fffffff;
    for (int e = lane; e < a.E; e += 64)
      if (key[e] > best) { best = key[e]; at = e; }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const unsigned long long ob = __shfl_xor(best, d);
      const int oa = __shfl_xor(at, d);
      if (ob > best || (ob == best && oa < at)) { best = ob; at = oa; }
    }
    if (lane == 0) { pick[j] = at; key[at] = 0; }
    __syncthreads();
  }
  const double top = logits[pick[0]];
  float sum = 0;
  if (a.renormalize) {
    for (int j = 0; j < a.k; ++j) sum += expf((float)(logits[pick[j]] - top));
  } else {
    for (int e = lane; e < a.E; e += 64) sum += expf((float)(logits[e] - top));
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
  }
  if (lane < a.k) {
    const int s = t * a.k + lane;
    a.chosen[s] = pick[lane];
    a.experts[s] = pick[lane];
    a.weights[s] = expf((float)(logits[pick[lane]] - top)) / sum;
  }
}

// ------------------------------------------------------------ experts' products

// What a lane reads of 16 rows x one slab of weights: its row (lane & 15) at the
// 32 elements (lane >> 4) * 32 of the slab, the 64 (16) bytes of which feed four
// steps of the 16x16x32 matrix instruction, 8 elements each.  The other operand
// reads its elements the same way: a sum over k does not mind the order.
template <int WF>
struct WeightSlab {  // 16-bit weights
  u32x4v v[4];
  __device__ __forceinline__ void load(const void* base, const uint8_t*, long long, long long row, long long ld, int slab, int K) {
    const int q = (threadIdx.x & 63) >> 4;
    const int k = slab * kSlab + q * 32;
    const u16* p = (const u16*)base + row * ld + k;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int left = K - k - s * 8;
      if (left >= 8) {
        __builtin_memcpy(&v[s], p + s * 8, 16);
      } else {
        u16 e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = i < left ? p[s * 8 + i] : (u16)0;
        __builtin_memcpy(&v[s], e, 16);
      }
    }
  }
  __device__ __forceinline__ u32x4v step(int s) const { return v[s]; }
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
    const unsigned nan = scale == 255u ? 0x7fff7fffu : 0u;
    const unsigned w = v[s];
    u32x4v o;
    o[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 0)) | nan;
    o[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 1)) | nan;
    o[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 2)) | nan;
    o[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 3)) | nan;
    return o;
  }
};

__device__ __forceinline__ f32x4 mfma_bf16(u32x4v a, u32x4v b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_f16(u32x4v a, u32x4v b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Eight fp16 as the sum of two times eight bf16, exactly (11 bits = 8 + 3).  The
// products with activations need it that may not fit fp16.  An infinite weight
// comes out as NaN.
__device__ __forceinline__ void split_f16(u32x4v w, u32x4v& hi, u32x4v& lo) {
  const f16x8 f = __builtin_bit_cast(f16x8, w);
  bf16x8 h, l;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = (float)f[i];
    const float top = __uint_as_float(__float_as_uint(v) & 0xffff0000u);
    h[i] = __builtin_bit_cast(__bf16, (u16)(__float_as_uint(v) >> 16));
    l[i] = __builtin_bit_cast(__bf16, (u16)(__float_as_uint(v - top) >> 16));
  }
  hi = __builtin_bit_cast(u32x4v, h);
  lo = __builtin_bit_cast(u32x4v, l);
}

constexpr int kMoeWaves = 4;
constexpr int kMoeBlocks = 4;  // column blocks of 16 tokens at a time

// The expert a work-group serves and the slots t*k+j that chose it, in order.
// Returns their count, 0 if there is nothing to do.
__device__ __forceinline__ int moe_slots(const MoeArgs& a, int unit, int* list, int& expert) {
  const int n = a.T * a.k;
  __shared__ int count;
  if (n <= a.E) {  // a unit is a slot: the first one that chose the expert serves it
    expert = a.chosen[unit];
    for (int s = 0; s < unit; ++s)
      if (a.chosen[s] == expert) return 0;
  } else {
    expert = unit;
  }
  if (threadIdx.x < 64) {
    int found = 0;
    for (int s0 = 0; s0 < n; s0 += 64) {
      const int s = s0 + (int)threadIdx.x;
      const bool mine = s < n && a.chosen[s] == expert;
      const unsigned long long m = __ballot(mine);
      if (mine) list[found + __popcll(m & ((1ull << threadIdx.x) - 1))] = s;
      found += __popcll(m);
    }
    if (threadIdx.x == 0) count = found;
  }
  __syncthreads();
  return count;
}

__device__ __forceinline__ float activate(float g, int act) {
  if (act == CMK_ACT_SILU) return g / (1.0f + expf(-g));
  return 0.5f * g * (1.0f + erff(g * 0.70710678118654752f));
}

// 16 gate rows and the 16 up rows that go with them, against the tokens of one
// expert; the waves split H and their sums meet in LDS, in order.
template <int WF, int PLANES>
__global__ __launch_bounds__(64 * kMoeWaves) void moe_gate_up_kernel(MoeArgs a) {
  __shared__ int list[kMoeTokens];
  __shared__ float part[kMoeWaves][2][kMoeBlocks][64][4];
  int expert;
  const int count = moe_slots(a, blockIdx.y, list, expert);
  if (count == 0) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, q = lane >> 4;
  const int i0 = blockIdx.x * 16;
  const int row = min(i0 + r, a.I - 1);
  const char* base = (const char*)a.gate_up + (WF == CMK_MX4 ? (long long)expert * (a.Hp / 2) * (2 * a.I) : expert * a.stride_gate_up * 2);
  const uint8_t* scales = WF == CMK_MX4 ? a.gate_up_scales + (long long)expert * (a.Hp / 32) * (2 * a.I) : nullptr;
  const int slabs = a.Hp / kSlab;
  for (int c0 = 0; c0 < count; c0 += 16 * kMoeBlocks) {
    const int blocks = min(kMoeBlocks, (count - c0 + 15) / 16);
    f32x4 g[kMoeBlocks] = {}, u[kMoeBlocks] = {};
    const u16* xs[kMoeBlocks];
#pragma unroll
    for (int b = 0; b < kMoeBlocks; ++b) {
      const int t = list[min(c0 + b * 16 + r, count - 1)] / a.k;
      xs[b] = a.xp + (long long)t * a.Hp + q * 32;
    }
    for (int slab = wave; slab < slabs; slab += kMoeWaves) {
      WeightSlab<WF> wg, wu;
      wg.load(base, scales, 2 * a.I, row, a.ld_gate_up, slab, a.H);
      wu.load(base, scales, 2 * a.I, a.I + row, a.ld_gate_up, slab, a.H);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const u32x4v fg = wg.step(s), fu = wu.step(s);
#pragma unroll
        for (int b = 0; b < kMoeBlocks; ++b) {
          if (b >= blocks) break;
#pragma unroll
          for (int p = 0; p < PLANES; ++p) {
            const u32x4v x = *(const u32x4v*)(xs[b] + (long long)p * a.T * a.Hp + slab * kSlab + s * 8);
            if (WF == CMK_F16) { g[b] = mfma_f16(fg, x, g[b]); u[b] = mfma_f16(fu, x, u[b]); }
            else { g[b] = mfma_bf16(fg, x, g[b]); u[b] = mfma_bf16(fu, x, u[b]); }
          }
        }
      }
    }
#pragma unroll
    for (int b = 0; b < kMoeBlocks; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) { part[wave][0][b][lane][i] = g[b][i]; part[wave][1][b][lane][i] = u[b][i]; }
    __syncthreads();
    for (int v = threadIdx.x; v < blocks * 256; v += 64 * kMoeWaves) {
      // 16 rows of one token next to each other
      const int row_in = v & 15, col = v >> 4 & 15, b = v >> 8;
      const int l = (row_in >> 2) * 16 + col, i = row_in & 3;
      float sg = 0, su = 0;
#pragma unroll
      for (int w = 0; w < kMoeWaves; ++w) { sg += part[w][0][b][l][i]; su += part[w][1][b][l][i]; }
      const int c = c0 + b * 16 + col;
      if (c < count) {
        const float h = i0 + row_in < a.I ? activate(sg, a.act) * su : 0.0f;
        // two bf16: 16 bits of mantissa and fp32's range
        const __bf16 hi = (__bf16)h;
        const __bf16 lo = (__bf16)(__builtin_isfinite(h) ? h - (float)hi : 0.0f);
        const long long at = (long long)list[c] * a.Ip + i0 + row_in;
        a.hp[at] = __builtin_bit_cast(u16, hi);
        a.hp[at + (long long)a.T * a.k * a.Ip] = __builtin_bit_cast(u16, lo);
      }
    }
    __syncthreads();
  }
}

// 16 rows of an expert's down matrix against its slots' activations.
template <int WF>
__global__ __launch_bounds__(64 * kMoeWaves) void moe_down_kernel(MoeArgs a) {
  __shared__ int list[kMoeTokens];
  __shared__ float part[kMoeWaves][kMoeBlocks][64][4];
  int expert;
  const int count = moe_slots(a, blockIdx.y, list, expert);
  if (count == 0) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int row = min(n0 + r, a.H - 1);
  const char* base = (const char*)a.down + (WF == CMK_MX4 ? (long long)expert * (a.Ip / 2) * a.H : expert * a.stride_down * 2);
  const uint8_t* scales = WF == CMK_MX4 ? a.down_scales + (long long)expert * (a.Ip / 32) * a.H : nullptr;
  const int slabs = a.Ip / kSlab;
  const long long plane = (long long)a.T * a.k * a.Ip;
  for (int c0 = 0; c0 < count; c0 += 16 * kMoeBlocks) {
    const int blocks = min(kMoeBlocks, (count - c0 + 15) / 16);
    f32x4 y[kMoeBlocks] = {};
    const u16* hs[kMoeBlocks];
#pragma unroll
    for (int b = 0; b < kMoeBlocks; ++b)
      hs[b] = a.hp + (long long)list[min(c0 + b * 16 + r, count - 1)] * a.Ip + q * 32;
    for (int slab = wave; slab < slabs; slab += kMoeWaves) {
      WeightSlab<WF> w;
      w.load(base, scales, a.H, row, a.ld_down, slab, a.I);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        u32x4v f = w.step(s), f2 = f;
        if (WF == CMK_F16) split_f16(w.step(s), f, f2);
#pragma unroll
        for (int b = 0; b < kMoeBlocks; ++b) {
          if (b >= blocks) break;
          const u32x4v hi = *(const u32x4v*)(hs[b] + slab * kSlab + s * 8);
          const u32x4v lo = *(const u32x4v*)(hs[b] + plane + slab * kSlab + s * 8);
          y[b] = mfma_bf16(f, hi, y[b]);
          y[b] = mfma_bf16(f, lo, y[b]);
          if (WF == CMK_F16) y[b] = mfma_bf16(f2, hi, y[b]);
        }
      }
    }
#pragma unroll
    for (int b = 0; b < kMoeBlocks; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[wave][b][lane][i] = y[b][i];
    __syncthreads();
    for (int v = threadIdx.x; v < blocks * 256; v += 64 * kMoeWaves) {
      const int row_in = v & 15, col = v >> 4 & 15, b = v >> 8;
      const int l = (row_in >> 2) * 16 + col, i = row_in & 3;
      float s = 0;
#pragma unroll
      for (int w = 0; w < kMoeWaves; ++w) s += part[w][b][l][i];
      const int c = c0 + b * 16 + col;
      if (c < count && n0 + row_in < a.H) a.yp[(long long)list[c] * a.H + n0 + row_in] = s;
    }
    __syncthreads();
  }
}

template <class T>
__global__ __launch_bounds__(256) void moe_combine_kernel(MoeArgs a) {
  const int n = blockIdx.x * 256 + threadIdx.x, t = blockIdx.y;
  if (n >= a.H) return;
  float s = 0;
  for (int j = 0; j < a.k; ++j) s = fmaf(a.weights[t * a.k + j], a.yp[((long long)t * a.k + j) * a.H + n], s);
  ((T*)a.y)[(long long)t * a.H + n] = from_f32<T>(s);
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
            d->T, d->H, d->I, d->E, d->k, p.Hp, p.Ip, d->activation, d->renormalize,
            (double*)(ws + p.logits), (int*)(ws + p.chosen), (u16*)(ws + p.x), (u16*)(ws + p.h), (float*)(ws + p.y)};
  hipStream_t st = (hipStream_t)stream;
  const dim3 router_grid(ceil_div(d->E, 16), ceil_div(d->T, 16));
  const bool r32 = d->router_dtype == CMK_F32;
  if (d->x_dtype == CMK_BF16) {
    if (r32) hipLaunchKernelGGL((moe_logits_kernel<__bf16, float, 1>), router_grid, dim3(512), 0, st, a);
    else hipLaunchKernelGGL((moe_logits_kernel<__bf16, __bf16, 1>), router_grid, dim3(512), 0, st, a);
  } else if (p.x_planes == 1) {
    if (r32) hipLaunchKernelGGL((moe_logits_kernel<_Float16, float, 1>), router_grid, dim3(512), 0, st, a);
    else hipLaunchKernelGGL((moe_logits_kernel<_Float16, _Float16, 1>), router_grid, dim3(512), 0, st, a);
  } else {
    if (r32) hipLaunchKernelGGL((moe_logits_kernel<_Float16, float, 2>), router_grid, dim3(512), 0, st, a);
    else hipLaunchKernelGGL((moe_logits_kernel<_Float16, _Float16, 2>), router_grid, dim3(512), 0, st, a);
  }
  hipLaunchKernelGGL(moe_select_kernel, dim3(d->T), dim3(64), 0, st, a);
  const int units = d->T * d->k <= d->E ? d->T * d->k : d->E;
  const dim3 up_grid(p.Ip / 16, units), down_grid(ceil_div(d->H, 16), units), b(64 * kMoeWaves);
  if (d->w_dtype == CMK_MX4) {
    if (p.x_planes == 1) hipLaunchKernelGGL((moe_gate_up_kernel<CMK_MX4, 1>), up_grid, b, 0, st, a);
    else hipLaunchKernelGGL((moe_gate_up_kernel<CMK_MX4, 2>), up_grid, b, 0, st, a);
    hipLaunchKernelGGL(moe_down_kernel<CMK_MX4>, down_grid, b, 0, st, a);
  } else if (d->w_dtype == CMK_BF16) {
    hipLaunchKernelGGL((moe_gate_up_kernel<CMK_BF16, 1>), up_grid, b, 0, st, a);
    hipLaunchKernelGGL(moe_down_kernel<CMK_BF16>, down_grid, b, 0, st, a);
  } else {
    hipLaunchKernelGGL((moe_gate_up_kernel<CMK_F16, 1>), up_grid, b, 0, st, a);
    hipLaunchKernelGGL(moe_down_kernel<CMK_F16>, down_grid, b, 0, st, a);
  }
  const dim3 out_grid(ceil_div(d->H, 256), d->T);
  if (d->x_dtype == CMK_BF16) hipLaunchKernelGGL(moe_combine_kernel<__bf16>, out_grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(moe_combine_kernel<_Float16>, out_grid, dim3(256), 0, st, a);
  return hip_status(hipGetLastError(), "cmk_moe launch");
}
