// 4-bit microscaled matrices: quantisation, its inverse, and the batched product.
#include "cmk_mx4.hpp"

namespace cmk {

// ---------------------------------------------------------------- quantisation

struct QuantArgs {
  const void* x;
  uint8_t* codes;
  uint8_t* scales;
  int L, R, K;
  long long slabs, row_groups, groups;
  long long sl, sr, sk;  // element strides of x
};

// k contiguous.  Four lanes share a block (8 elements each), 16 lanes a row's
// slab, a wave 16 rows x one slab in four steps: it reads 256 (512) contiguous
// bytes of a row per step and writes one contiguous KB of codes.
template <class T>
__global__ __launch_bounds__(256) void mx4_quantize_rows_kernel(QuantArgs a) {
  const int lane = threadIdx.x & 63;
  const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= a.groups) return;
  const long long rg = unit % a.row_groups;
  const long long ls = unit / a.row_groups;  // l * slabs + slab
  const int l = (int)(ls / a.slabs), slab = (int)(ls % a.slabs);
  const int k0 = slab * kSlab + (lane & 15) * 8;
  const T* x = (const T*)a.x + l * a.sl + k0;
  Octet<T> o[4];
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const long long row = rg * 16 + p * 4 + (lane >> 4);
    o[p] = load_octet(x + row * a.sr, row < a.R ? a.K - k0 : 0);
  }
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const long long row = rg * 16 + p * 4 + (lane >> 4);
    unsigned top = o[p].top();
    top = max(top, (unsigned)__shfl_xor((int)top, 1));
    top = max(top, (unsigned)__shfl_xor((int)top, 2));
    const unsigned s = scale_byte(top);
    const unsigned w = s == 255u ? 0u : o[p].codes(scale_float(s));
    if (row < a.R) {
      const long long at = ls * a.R + row;
      *(unsigned*)(a.codes + at * kSlabBytes + (lane & 15) * 4) = w;
      if ((lane & 3) == 0) a.scales[at * kSlabScales + ((lane & 15) >> 2)] = (uint8_t)s;
    }
  }
}

// Any strides: a lane takes one row's slab, neighbouring lanes neighbouring rows
// (contiguous where the matrix is stored with its rows' axis innermost).
template <class T>
__global__ __launch_bounds__(256) void mx4_quantize_columns_kernel(QuantArgs a) {
  const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= a.groups) return;
  const long long rg = unit % a.row_groups;
  const long long ls = unit / a.row_groups;
  const int l = (int)(ls / a.slabs), slab = (int)(ls % a.slabs);
  const long long row = rg * 64 + (threadIdx.x & 63);
  if (row >= a.R) return;
  const T* x = (const T*)a.x + l * a.sl + row * a.sr;
  unsigned scales = 0;
  u32x4v codes[4];
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const int k0 = slab * kSlab + b * 32;
    Octet<T> o[4];
#pragma unroll
    for (int i = 0; i < 32; ++i)
      o[i >> 3].v[i & 7] = k0 + i < a.K ? x[(k0 + i) * a.sk] : (T)0.0f;
    const unsigned top = max(max(o[0].top(), o[1].top()), max(o[2].top(), o[3].top()));
    const unsigned s = scale_byte(top);
    const float f = scale_float(s);
#pragma unroll
    for (int i = 0; i < 4; ++i) codes[b][i] = s == 255u ? 0u : o[i].codes(f);
    scales |= s << (8 * b);
  }
  const long long at = ls * a.R + row;
#pragma unroll
  for (int b = 0; b < 4; ++b) *(u32x4v*)(a.codes + at * kSlabBytes + b * 16) = codes[b];
  *(unsigned*)(a.scales + at * kSlabScales) = scales;
}

// ------------------------------------------------------------------ its inverse

struct DequantArgs {
  const uint8_t* codes;
  const uint8_t* scales;
  void* out;  // dense: [L][R][K], or [L][K][R]
  int L, R, K;
  long long slabs, row_groups, groups;
};

// Eight values of a word of codes, in fp32.  The conversion is exact: a code times
// a power of two.  A scale byte of 255 is NaN.
__device__ __forceinline__ void decode_octet(unsigned w, unsigned s, float* v) {
  const float f = scale_float(s);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    f32x2 p;
    switch (i) {
      case 0: p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 0); break;
      case 1: p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 1); break;
      case 2: p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 2); break;
      default: p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 3); break;
    }
    v[2 * i] = s == 255u ? __uint_as_float(0x7fc00000u) : p[0];
    v[2 * i + 1] = s == 255u ? __uint_as_float(0x7fc00000u) : p[1];
  }
}

template <class T>
__global__ __launch_bounds__(256) void mx4_dequantize_rows_kernel(DequantArgs a) {
  const int lane = threadIdx.x & 63;
  const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= a.groups) return;
  const long long rg = unit % a.row_groups;
  const long long ls = unit / a.row_groups;
  const int l = (int)(ls / a.slabs), slab = (int)(ls % a.slabs);
  const int k0 = slab * kSlab + (lane & 15) * 8;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const long long row = rg * 16 + p * 4 + (lane >> 4);
    if (row >= a.R) continue;
    const long long at = ls * a.R + row;
    const unsigned w = *(const unsigned*)(a.codes + at * kSlabBytes + (lane & 15) * 4);
    const unsigned s = a.scales[at * kSlabScales + ((lane & 15) >> 2)];
    float v[8];
    decode_octet(w, s, v);
    T o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = from_f32<T>(v[i]);
    T* out = (T*)a.out + ((long long)l * a.R + row) * a.K + k0;
    if (k0 + 8 <= a.K) {
      __builtin_memcpy(out, o, sizeof(o));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k0 + i < a.K) out[i] = o[i];
    }
  }
}

template <class T>
__global__ __launch_bounds__(256) void mx4_dequantize_columns_kernel(DequantArgs a) {
  const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= a.groups) return;
  const long long rg = unit % a.row_groups;
  const long long ls = unit / a.row_groups;
  const int l = (int)(ls / a.slabs), slab = (int)(ls % a.slabs);
  const long long row = rg * 64 + (threadIdx.x & 63);
  if (row >= a.R) return;
  const long long at = ls * a.R + row;
  const unsigned scales = *(const unsigned*)(a.scales + at * kSlabScales);
  T* out = (T*)a.out + (long long)l * a.K * a.R + row;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const u32x4v w = *(const u32x4v*)(a.codes + at * kSlabBytes + b * 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float v[8];
      decode_octet(w[i], scales >> (8 * b) & 255u, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int k = slab * kSlab + b * 32 + i * 8 + j;
        if (k < a.K) out[(long long)k * a.R] = from_f32<T>(v[j]);
      }
    }
  }
}

// -------------------------------------------------------------------- product

struct Mx4GemmArgs {
  const uint8_t *a_codes, *a_scales, *b_codes, *b_scales;
  void* c;  // dense [L][M][N]
  int L, M, N;
  int slabs;
  int tiles_m, tiles_n;
};

// One work-group of four waves computes a 128 x 128 tile; a wave 64 x 64 of it.
// The matrix instruction's first operand are the columns n of C, so that a lane
// ends up with runs of four consecutive n of one row m.
template <class T>
__global__ __launch_bounds__(256) void mx4_gemm_kernel(Mx4GemmArgs a) {
  constexpr int TM = 128, TN = 128;
  __shared__ __attribute__((aligned(16))) uint8_t sa[TM * kSlabBytes], sb[TN * kSlabBytes];
  __shared__ unsigned ssa[TM], ssb[TN];
  const int per_batch = a.tiles_m * a.tiles_n;
  const int l = blockIdx.x / per_batch;
  const int t = blockIdx.x - l * per_batch;
  const int m0 = t / a.tiles_n * TM, n0 = t % a.tiles_n * TN;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  const int r = lane & 31, h = lane >> 5;
  f32x16 acc[2][2] = {};
  for (int s = 0; s < a.slabs; ++s) {
    const long long arow = ((long long)l * a.slabs + s) * a.M, brow = ((long long)l * a.slabs + s) * a.N;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = threadIdx.x + 256 * i, row = c >> 2, part = c & 3;
      const long long ra = arow + min(m0 + row, a.M - 1), rb = brow + min(n0 + row, a.N - 1);
      *(u32x4v*)(sa + c * 16) = *(const u32x4v*)(a.a_codes + ra * kSlabBytes + part * 16);
      *(u32x4v*)(sb + c * 16) = *(const u32x4v*)(a.b_codes + rb * kSlabBytes + part * 16);
    }
    if (threadIdx.x < 128) ssa[threadIdx.x] = *(const unsigned*)(a.a_scales + (arow + min(m0 + (int)threadIdx.x, a.M - 1)) * kSlabScales);
    else ssb[threadIdx.x - 128] = *(const unsigned*)(a.b_scales + (brow + min(n0 + (int)threadIdx.x - 128, a.N - 1)) * kSlabScales);
    __syncthreads();
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      i32x8 fm[2] = {}, fn[2] = {};
      int cm[2], cn[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const u32x4v vm = *(const u32x4v*)(sa + (wm + b * 32 + r) * kSlabBytes + (2 * h + g) * 16);
        const u32x4v vn = *(const u32x4v*)(sb + (wn + b * 32 + r) * kSlabBytes + (2 * h + g) * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) { fm[b][i] = vm[i]; fn[b][i] = vn[i]; }
        cm[b] = ssa[wm + b * 32 + r] >> (16 * h + 8 * g);
        cn[b] = ssb[wn + b * 32 + r] >> (16 * h + 8 * g);
      }
#pragma unroll
      for (int bn = 0; bn < 2; ++bn)
#pragma unroll
        for (int bm = 0; bm < 2; ++bm)
          acc[bn][bm] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fn[bn], fm[bm], acc[bn][bm], 4, 4, 0, cn[bn], 0, cm[bm]);
    }
  }
  T* c = (T*)a.c + (long long)l * a.M * a.N;
#pragma unroll
  for (int bm = 0; bm < 2; ++bm) {
    const int m = m0 + wm + bm * 32 + r;
    if (m >= a.M) continue;
#pragma unroll
    for (int bn = 0; bn < 2; ++bn)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int n = n0 + wn + bn * 32 + 8 * (i >> 2) + 4 * h + (i & 3);
        if (n < a.N) c[(long long)m * a.N + n] = from_f32<T>(acc[bn][bm][i]);
      }
  }
}

static int check_mx4(const char* who, int L, int R, int K) {
  if (L < 0 || R < 0 || K < 0) return fail(CMK_ERR_INVALID_ARG, "%s: negative extent (L=%d R=%d K=%d)", who, L, R, K);
  return CMK_OK;
}

static int check_dtype(const char* who, int dtype) {
  if (dtype != CMK_F32 && dtype != CMK_BF16 && dtype != CMK_F16)
    return fail(CMK_ERR_INVALID_ARG, "%s: unknown element type %d", who, dtype);
  return CMK_OK;
}

// Calls f with a value of the element type.
template <class F>
static void by_dtype(int dtype, F f) {
  if (dtype == CMK_F32) f(0.0f);
  else if (dtype == CMK_BF16) f((__bf16)0.0f);
  else f((_Float16)0.0f);
}

}  // namespace cmk

using namespace cmk;

extern "C" int cmk_mx4_quantize(const void* x, int dtype, uint8_t* codes, uint8_t* scales, int L, int R, int K,
                                long long stride_l, long long stride_r, long long stride_k, void* stream) {
  if (int e = check_mx4("cmk_mx4_quantize", L, R, K)) return e;
  if (int e = check_dtype("cmk_mx4_quantize", dtype)) return e;
  if (L == 0 || R == 0 || K == 0) return CMK_OK;
  if (!x || !codes || !scales) return fail(CMK_ERR_INVALID_ARG, "cmk_mx4_quantize: null pointer");
  if ((reinterpret_cast<uintptr_t>(codes) & 15) || (reinterpret_cast<uintptr_t>(scales) & 3))
    return fail(CMK_ERR_INVALID_ARG, "cmk_mx4_quantize: codes need 16-byte alignment, scales 4-byte alignment");
  QuantArgs a{x, codes, scales, L, R, K, mx4_slabs(K), 0, 0, stride_l, stride_r, stride_k};
  const bool rows = stride_k == 1 || K == 1;
  a.row_groups = rows ? ((long long)R + 15) / 16 : ((long long)R + 63) / 64;
  a.groups = a.row_groups * a.slabs * L;
  const long long grid = (a.groups + 3) / 4;
  if (int e = check_grid(grid)) return e;
  hipStream_t st = (hipStream_t)stream;
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (rows) hipLaunchKernelGGL(mx4_quantize_rows_kernel<T>, dim3((unsigned)grid), dim3(256), 0, st, a);
    else hipLaunchKernelGGL(mx4_quantize_columns_kernel<T>, dim3((unsigned)grid), dim3(256), 0, st, a);
  });
  return hip_status(hipGetLastError(), "cmk_mx4_quantize launch");
}

extern "C" int cmk_mx4_dequantize(const uint8_t* codes, const uint8_t* scales, void* out, int dtype, int L, int R,
                                  int K, int rows_innermost, void* stream) {
  if (int e = check_mx4("cmk_mx4_dequantize", L, R, K)) return e;
  if (int e = check_dtype("cmk_mx4_dequantize", dtype)) return e;
  if (L == 0 || R == 0 || K == 0) return CMK_OK;
  if (!out || !codes || !scales) return fail(CMK_ERR_INVALID_ARG, "cmk_mx4_dequantize: null pointer");
  if ((reinterpret_cast<uintptr_t>(codes) & 15) || (reinterpret_cast<uintptr_t>(scales) & 3))
    return fail(CMK_ERR_INVALID_ARG, "cmk_mx4_dequantize: codes need 16-byte alignment, scales 4-byte alignment");
  DequantArgs a{codes, scales, out, L, R, K, mx4_slabs(K), 0, 0};
  a.row_groups = rows_innermost ? ((long long)R + 63) / 64 : ((long long)R + 15) / 16;
  a.groups = a.row_groups * a.slabs * L;
  const long long grid = (a.groups + 3) / 4;
  if (int e = check_grid(grid)) return e;
  hipStream_t st = (hipStream_t)stream;
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (rows_innermost) hipLaunchKernelGGL(mx4_dequantize_columns_kernel<T>, dim3((unsigned)grid), dim3(256), 0, st, a);
    else hipLaunchKernelGGL(mx4_dequantize_rows_kernel<T>, dim3((unsigned)grid), dim3(256), 0, st, a);
  });
  return hip_status(hipGetLastError(), "cmk_mx4_dequantize launch");
}

extern "C" int cmk_mx4_bmm(const uint8_t* a_codes, const uint8_t* a_scales, const uint8_t* b_codes,
                           const uint8_t* b_scales, void* C, int dtype, int L, int M, int N, int K, void* stream) {
  if (L < 0 || M < 0 || N < 0 || K < 0)
    return fail(CMK_ERR_INVALID_ARG, "cmk_mx4_bmm: negative extent (L=%d M=%d N=%d K=%d)", L, M, N, K);
  if (int e = check_dtype("cmk_mx4_bmm", dtype)) return e;
  if (L == 0 || M == 0 || N == 0) return CMK_OK;
  if (!C || (K > 0 && (!a_codes || !a_scales || !b_codes || !b_scales)))
    return fail(CMK_ERR_INVALID_ARG, "cmk_mx4_bmm: null pointer");
  if (((reinterpret_cast<uintptr_t>(a_codes) | reinterpret_cast<uintptr_t>(b_codes)) & 15) ||
      ((reinterpret_cast<uintptr_t>(a_scales) | reinterpret_cast<uintptr_t>(b_scales)) & 3))
    return fail(CMK_ERR_INVALID_ARG, "cmk_mx4_bmm: codes need 16-byte alignment, scales 4-byte alignment");
  Mx4GemmArgs a{a_codes, a_scales, b_codes, b_scales, C, L, M, N, (int)mx4_slabs(K), ceil_div(M, 128), ceil_div(N, 128)};
  const long long grid = (long long)L * a.tiles_m * a.tiles_n;
  if (int e = check_grid(grid)) return e;
  hipStream_t st = (hipStream_t)stream;
  const dim3 g((unsigned)grid), b(256);
  by_dtype(dtype, [&](auto t) { hipLaunchKernelGGL(mx4_gemm_kernel<decltype(t)>, g, b, 0, st, a); });
  return hip_status(hipGetLastError(), "cmk_mx4_bmm launch");
}
