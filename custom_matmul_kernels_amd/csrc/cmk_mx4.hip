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
      o[i >> 3].set(i & 7, k0 + i < a.K ? x[(k0 + i) * a.sk] : (T)0.0f);
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

// A work-group of four waves computes a TM x TN tile of C, a wave a quarter of it
// in blocks of 32 x 32 (v_mfma_scale_f32_32x32x64_f8f6f4: 64 elements of k, each
// lane holding one whole 32-element block of one row, so that the lane's scale is
// one byte).
//
// Slabs of both operands (codes and scales) travel by direct global-to-LDS loads
// into a ring of kStages buffers, two slabs ahead of the products.  Half a slab's
// fragments are in registers at a time; those of the next half are read while the
// matrix pipe works on them.  The one barrier of a slab sits between its halves:
// it follows the wait for the next slab, whose first half is read behind it, and
// frees the buffer of the slab before.  Within a row the four 16-byte blocks are
// stored at position block ^ ((row >> 2) & 3), so that the 16 rows that the LDS
// serves at a time spread over all banks; the swizzle is produced by choosing
// which block each lane of a load asks for.
constexpr int kStages = 4;

template <int TM, int TN>
struct Mx4Tile {
  static constexpr int BM = TM / 64, BN = TN / 64;  // 32 x 32 blocks of a wave
  static constexpr int kCodesA = TM * kSlabBytes, kCodesB = TN * kSlabBytes;
  static constexpr int kStageBytes = kCodesA + kCodesB + (TM + TN) * kSlabScales;
  static constexpr int kLoads = TM / 64 + TN / 64 + 2;  // vector-memory instructions of a wave per slab
};

typedef const __attribute__((address_space(1))) void* gptr;
typedef __attribute__((address_space(3))) void* lptr;

// Waits until at most `left` of the wave's vector-memory instructions are under way.
template <int left>
__device__ __forceinline__ void wait_loads() {
  static_assert(left < 64, "the counter has six bits");
  __builtin_amdgcn_s_waitcnt(0x0f70 | (left & 15) | (left >> 4 << 14));
}

template <int v>
struct Int {
  static constexpr int value = v;
};

// The barrier of the work-group's waves; memory operations stay on their side of it.
__device__ __forceinline__ void meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Work-groups go round the eight XCDs in turn, each with an L2 of its own: an XCD
// gets a contiguous run of the tiles of all batches, in strips of eight tile rows,
// so that what runs on it at a time shares few panels of both operands.
__device__ __forceinline__ void place_tile(const Mx4GemmArgs& a, int& l, int& tile_m, int& tile_n) {
  const int total = gridDim.x, xcd = blockIdx.x & 7, turn = blockIdx.x >> 3;
  const int each = total >> 3, extra = total & 7;
  const int id = xcd * each + min(xcd, extra) + turn;
  const int per_batch = a.tiles_m * a.tiles_n;
  l = id / per_batch;
  const int t = id - l * per_batch;
  const int strip = t / (8 * a.tiles_n), in = t - strip * 8 * a.tiles_n;
  const int height = min(8, a.tiles_m - strip * 8);
  tile_m = strip * 8 + in % height;
  tile_n = in / height;
}

template <class T, int TM, int TN>
__global__ __launch_bounds__(256, 1) void mx4_gemm_kernel(Mx4GemmArgs a) {
  using Tile = Mx4Tile<TM, TN>;
  constexpr int BM = Tile::BM, BN = Tile::BN;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kStages * Tile::kStageBytes];
  int l, tile_m, tile_n;
  place_tile(a, l, tile_m, tile_n);
  const int m0 = tile_m * TM, n0 = tile_n * TN;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = (wave >> 1) * (TM / 2), wn = (wave & 1) * (TN / 2);
  const int r = lane & 31, h = lane >> 5;

  // what this lane asks for: 16 rows x 64 bytes per instruction, rows beyond the
  // matrix replaced by its last one
  unsigned oa[TM / 64], ob[TN / 64];
#pragma unroll
  for (int i = 0; i < TM / 64; ++i) {
    const int row = (wave * (TM / 64) + i) * 16 + (lane >> 2);
    oa[i] = min(row, a.M - 1 - m0) * kSlabBytes + ((lane & 3) ^ ((row >> 2) & 3)) * 16;
  }
#pragma unroll
  for (int i = 0; i < TN / 64; ++i) {
    const int row = (wave * (TN / 64) + i) * 16 + (lane >> 2);
    ob[i] = min(row, a.N - 1 - n0) * kSlabBytes + ((lane & 3) ^ ((row >> 2) & 3)) * 16;
  }
  unsigned osa = min(wave * (TM / 4) + (lane & (TM / 4 - 1)), a.M - 1 - m0) * kSlabScales;
  unsigned osb = min(wave * (TN / 4) + (lane & (TN / 4 - 1)), a.N - 1 - n0) * kSlabScales;
  // The next slab to be requested.  Beyond the last one the requests repeat it, so
  // that every slab of the loop issues and awaits the same number of loads.
  const uint8_t* pa = a.a_codes + ((long long)l * a.slabs * a.M + m0) * kSlabBytes;
  const uint8_t* pb = a.b_codes + ((long long)l * a.slabs * a.N + n0) * kSlabBytes;
  const uint8_t* psa = a.a_scales + ((long long)l * a.slabs * a.M + m0) * kSlabScales;
  const uint8_t* psb = a.b_scales + ((long long)l * a.slabs * a.N + n0) * kSlabScales;
  const long long step_a = (long long)a.M * kSlabBytes, step_b = (long long)a.N * kSlabBytes;
  int requested = 0;
  // scalar base + 32-bit lane offset, no vector addition
  auto load16 = [&](const uint8_t* base, unsigned& off, uint8_t* to) {
    asm volatile("" : "+s"(base));
    asm volatile("" : "+v"(off));
    __builtin_amdgcn_global_load_lds((gptr)(base + off), (lptr)to, 16, 0, 0);
  };
  auto load4 = [&](const uint8_t* base, unsigned& off, uint8_t* to) {
    asm volatile("" : "+s"(base));
    asm volatile("" : "+v"(off));
    __builtin_amdgcn_global_load_lds((gptr)(base + off), (lptr)to, 4, 0, 0);
  };
  auto fetch = [&](int stage) {
    uint8_t* at = lds + stage * Tile::kStageBytes;
#pragma unroll
    for (int i = 0; i < TM / 64; ++i) load16(pa, oa[i], at + (wave * (TM / 64) + i) * 1024);
#pragma unroll
    for (int i = 0; i < TN / 64; ++i) load16(pb, ob[i], at + Tile::kCodesA + (wave * (TN / 64) + i) * 1024);
    uint8_t* scales = at + Tile::kCodesA + Tile::kCodesB;
    if (TM == 256 || lane < TM / 4) load4(psa, osa, scales + wave * TM);
    if (TN == 256 || lane < TN / 4) load4(psb, osb, scales + TM * kSlabScales + wave * TN);
    const long long more = ++requested < a.slabs ? 1 : 0;
    pa += more * step_a; pb += more * step_b;
    psa += more * (step_a / (kSlabBytes / kSlabScales)); psb += more * (step_b / (kSlabBytes / kSlabScales));
  };

  // Where this lane reads: one register per half of a slab, operand and pair of
  // stages, the rest of an address is the instruction's offset (vector
  // instructions in the loop cost matrix-pipe time).
  const unsigned lds0 = (unsigned)(uintptr_t)(lptr)lds;
  unsigned at_m[2][2], at_n[2][2], at_cm[2], at_cn[2];
#pragma unroll
  for (int pair = 0; pair < 2; ++pair) {
    const unsigned base = lds0 + pair * 2 * Tile::kStageBytes;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const unsigned part = ((2 * h + g) ^ ((r >> 2) & 3)) * 16;
      at_m[pair][g] = base + (wm + r) * kSlabBytes + part;
      at_n[pair][g] = base + Tile::kCodesA + (wn + r) * kSlabBytes + part;
      asm("" : "+v"(at_m[pair][g]), "+v"(at_n[pair][g]));
    }
    at_cm[pair] = base + Tile::kCodesA + Tile::kCodesB + (wm + r) * kSlabScales + 2 * h;
    at_cn[pair] = base + Tile::kCodesA + Tile::kCodesB + (TM + wn + r) * kSlabScales + 2 * h;
    asm("" : "+v"(at_cm[pair]), "+v"(at_cn[pair]));
  }
  struct Half {
    u32x4v m[BM], n[BN];
  };
  struct Scales {
    int m[BM], n[BN];  // a lane's two blocks of the slab in the low bytes
  };
  typedef const __attribute__((address_space(3))) u32x4v* l16;
  typedef const __attribute__((address_space(3))) unsigned short* l2;
  auto read = [&](int stage, int g, Half& f) {
    const unsigned off = (stage & 1) * Tile::kStageBytes;
#pragma unroll
    for (int b = 0; b < BM; ++b) f.m[b] = *(l16)(lptr)(uintptr_t)(at_m[stage >> 1][g] + off + b * 32 * kSlabBytes);
#pragma unroll
    for (int b = 0; b < BN; ++b) f.n[b] = *(l16)(lptr)(uintptr_t)(at_n[stage >> 1][g] + off + b * 32 * kSlabBytes);
  };
  auto read_scales = [&](int stage, Scales& c) {
    const unsigned off = (stage & 1) * Tile::kStageBytes;
#pragma unroll
    for (int b = 0; b < BM; ++b) c.m[b] = *(l2)(lptr)(uintptr_t)(at_cm[stage >> 1] + off + b * 32 * kSlabScales);
#pragma unroll
    for (int b = 0; b < BN; ++b) c.n[b] = *(l2)(lptr)(uintptr_t)(at_cn[stage >> 1] + off + b * 32 * kSlabScales);
  };
  f32x16 acc[BM][BN] = {};
  auto wide = [](u32x4v v) { return i32x8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0}; };

  // One slab of ring position `stage`, c its scales, d the next one's.
  Half f0, f1;
  auto slab = [&](auto stage, Scales& c, Scales& d) {
    constexpr int Stage = decltype(stage)::value;
    constexpr int Next = (Stage + 1) % kStages;
    read(Stage, 1, f1);
#pragma unroll
    for (int bm = 0; bm < BM; ++bm)
#pragma unroll
      for (int bn = 0; bn < BN; ++bn)
        acc[bm][bn] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(f0.m[bm]), wide(f0.n[bn]), acc[bm][bn], 4, 4, 0, c.m[bm], 0, c.n[bn]);
    // a read, then as many products as keep the matrix pipe busy until the next
#pragma unroll
    for (int i = 0; i < BM + BN; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, BM * BN / (BM + BN), 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    wait_loads<Tile::kLoads>();
    meet();
    read_scales(Next, d);
    read(Next, 0, f0);
    fetch((Stage + kStages - 1) % kStages);
#pragma unroll
    for (int bm = 0; bm < BM; ++bm)
#pragma unroll
      for (int bn = 0; bn < BN; ++bn)
        acc[bm][bn] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(f1.m[bm]), wide(f1.n[bn]), acc[bm][bn], 4, 4, 1, c.m[bm], 1, c.n[bn]);
    // what the next slab starts with first, the requests behind it
#pragma unroll
    for (int i = 0; i < BM + BN; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, BM * BN / 2 / (BM + BN), 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
#pragma unroll
    for (int i = 0; i < Tile::kLoads; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  if (a.slabs > 0) {
    Scales c0, c1;
    fetch(0);
    fetch(1);
    fetch(2);
    wait_loads<2 * Tile::kLoads>();
    meet();
    read_scales(0, c0);
    read(0, 0, f0);
    int left = a.slabs;
    for (; left >= 4; left -= 4) {
      slab(Int<0>{}, c0, c1);
      slab(Int<1>{}, c1, c0);
      slab(Int<2>{}, c0, c1);
      slab(Int<3>{}, c1, c0);
    }
    if (left > 0) slab(Int<0>{}, c0, c1);
    if (left > 1) slab(Int<1>{}, c1, c0);
    if (left > 2) slab(Int<2>{}, c0, c1);
    wait_loads<0>();  // no load may land after the work-group has ended
  }

  // lane: column n = lane & 31, rows 8 * (i / 4) + 4 * h + i % 4: a store covers two
  // runs of 32 columns
  T* c = (T*)a.c + (long long)l * a.M * a.N;
#pragma unroll
  for (int bm = 0; bm < BM; ++bm)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int m = m0 + wm + bm * 32 + 8 * (i >> 2) + 4 * h + (i & 3);
      if (m >= a.M) continue;
      T* row = c + (long long)m * a.N;
#pragma unroll
      for (int bn = 0; bn < BN; ++bn) {
        const int n = n0 + wn + bn * 32 + r;
        if (n < a.N) row[n] = from_f32<T>(acc[bm][bn][i]);
      }
    }
}

// ------------------------------------------------------- product with few rows

struct Mx4RowsArgs {
  const void* x;  // the left operand: codes, or elements with k contiguous
  const uint8_t *x_scales, *b_codes, *b_scales;
  void* c;
  int M, N, K, slabs;
  long long sl, sm;  // strides of x in elements
};

// A lane's share of one slab of 16 rows: 32 elements of row lane & 15, those of
// block lane >> 4, as the 16x16x128 instruction takes them.
struct Mx4Fragment {
  u32x4v codes;
  int scale;
};

__device__ __forceinline__ void load_fragment(Mx4Fragment& f, const uint8_t* codes, const uint8_t* scales, long long at, int q) {
  f.codes = *(const u32x4v*)(codes + at * kSlabBytes + q * 16);
  f.scale = scales[at * kSlabScales + q];
}

// Quantises 32 elements in one lane.
template <class T>
__device__ __forceinline__ void quantize_fragment(Mx4Fragment& f, const Octet<T> (&o)[4]) {
  const unsigned s = scale_byte(max(max(o[0].top(), o[1].top()), max(o[2].top(), o[3].top())));
  const float scale = scale_float(s);
#pragma unroll
  for (int i = 0; i < 4; ++i) f.codes[i] = s == 255u ? 0u : o[i].codes(scale);
  f.scale = (int)s;
}

// A work-group takes 16 * RG columns of C and all its rows (up to 16 * MB); its
// waves split the slabs and their sums meet in LDS, in the order of the waves.
// There is nothing to gain but the stream of the right operand: its fragments
// (1 KB of contiguous codes per instruction) go straight to registers, U slabs at
// a time.  TX: the left operand's elements, quantised on the way, or uint8_t for
// codes.
template <class TX, class T, int W, int RG, int MB, int U>
__global__ __launch_bounds__(64 * W) void mx4_rows_kernel(Mx4RowsArgs a) {
  constexpr bool kCodes = sizeof(TX) == 1;
  __shared__ float part[W][RG][MB][64][4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int l = blockIdx.y, n0 = blockIdx.x * 16 * RG;
  const long long batch_b = (long long)l * a.slabs * a.N;
  int row[RG];
#pragma unroll
  for (int g = 0; g < RG; ++g) row[g] = min(n0 + g * 16 + r, a.N - 1);
  f32x4 acc[RG][MB] = {};
  auto wide = [](u32x4v v) { return i32x8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0}; };
  for (int s0 = wave; s0 < a.slabs; s0 += W * U) {
    Mx4Fragment fb[U][RG], fx[U][MB];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u * W;
      if (s >= a.slabs) break;
#pragma unroll
      for (int g = 0; g < RG; ++g) load_fragment(fb[u][g], a.b_codes, a.b_scales, batch_b + (long long)s * a.N + row[g], q);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u * W;
      if (s >= a.slabs) break;
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        if constexpr (kCodes) {
          const int m = min(b * 16 + r, a.M - 1);
          load_fragment(fx[u][b], (const uint8_t*)a.x, a.x_scales, ((long long)l * a.slabs + s) * a.M + m, q);
        } else {
          const int m = b * 16 + r, k = s * kSlab + q * 32;
          const TX* x = (const TX*)a.x + l * a.sl + m * a.sm + k;
          Octet<TX> o[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = load_octet(x + i * 8, m < a.M ? a.K - k - i * 8 : 0);
          quantize_fragment(fx[u][b], o);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u * W >= a.slabs) break;
#pragma unroll
      for (int g = 0; g < RG; ++g)
#pragma unroll
        for (int b = 0; b < MB; ++b)
          acc[g][b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(fb[u][g].codes), wide(fx[u][b].codes), acc[g][b], 4, 4, 0,
                                                                      fb[u][g].scale, 0, fx[u][b].scale);
    }
  }
#pragma unroll
  for (int g = 0; g < RG; ++g)
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[wave][g][b][lane][i] = acc[g][b][i];
  __syncthreads();
  T* c = (T*)a.c + (long long)l * a.M * a.N;
  for (int v = threadIdx.x; v < RG * MB * 256; v += 64 * W) {
    // neighbouring threads take neighbouring columns of one row
    const int n = v % (16 * RG), m = v / (16 * RG);
    const int g = n >> 4, i = n & 3, from = ((n & 15) >> 2) * 16 + (m & 15), b = m >> 4;
    if (m < a.M && n0 + n < a.N) {
      float sum = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) sum += part[w][g][b][from][i];
      c[(long long)m * a.N + n0 + n] = from_f32<T>(sum);
    }
  }
}

// Rows up to this many are served by mx4_rows_kernel.
constexpr int kMx4Rows = 64;
// and up to this many with the left operand quantised on the way
constexpr int kMx4RowsFloat = 16;

// TX: uint8_t or the element type of the left operand.
template <class TX, class T>
static void launch_rows(const Mx4RowsArgs& a, int L, hipStream_t st) {
  const long long groups = (long long)ceil_div(a.N, 16) * L;
  // Four row groups a wave share one fragment of the left operand; one each where
  // that would leave compute units without work.
  const bool many = groups >= 4LL * compute_units();
  auto grid = [&](int rg) { return dim3(ceil_div(a.N, 16 * rg), L); };
  if (a.M <= 16) {
    if (many) hipLaunchKernelGGL((mx4_rows_kernel<TX, T, 8, 4, 1, 2>), grid(4), dim3(512), 0, st, a);
    else if (a.slabs > 32) hipLaunchKernelGGL((mx4_rows_kernel<TX, T, 16, 1, 1, 4>), grid(1), dim3(1024), 0, st, a);
    else hipLaunchKernelGGL((mx4_rows_kernel<TX, T, 8, 1, 1, 4>), grid(1), dim3(512), 0, st, a);
  } else if constexpr (sizeof(TX) == 1) {
    if (a.M <= 32) {
      if (many) hipLaunchKernelGGL((mx4_rows_kernel<TX, T, 8, 4, 2, 2>), grid(4), dim3(512), 0, st, a);
      else hipLaunchKernelGGL((mx4_rows_kernel<TX, T, 8, 1, 2, 4>), grid(1), dim3(512), 0, st, a);
    } else {
      if (many) hipLaunchKernelGGL((mx4_rows_kernel<TX, T, 8, 2, 4, 2>), grid(2), dim3(512), 0, st, a);
      else hipLaunchKernelGGL((mx4_rows_kernel<TX, T, 8, 1, 4, 2>), grid(1), dim3(512), 0, st, a);
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
  if (M <= kMx4Rows && L <= 65535) {
    const Mx4RowsArgs r{a_codes, a_scales, b_codes, b_scales, C, M, N, K, (int)mx4_slabs(K), 0, 0};
    by_dtype(dtype, [&](auto t) { launch_rows<uint8_t, decltype(t)>(r, L, (hipStream_t)stream); });
    return hip_status(hipGetLastError(), "cmk_mx4_bmm launch");
  }
  const bool large = (long long)L * ceil_div(M, 256) * ceil_div(N, 256) >= compute_units();
  const int tile = large ? 256 : 128;
  Mx4GemmArgs a{a_codes, a_scales, b_codes, b_scales, C, L, M, N, (int)mx4_slabs(K), ceil_div(M, tile), ceil_div(N, tile)};
  const long long grid = (long long)L * a.tiles_m * a.tiles_n;
  if (int e = check_grid(grid)) return e;
  hipStream_t st = (hipStream_t)stream;
  const dim3 g((unsigned)grid), b(256);
  by_dtype(dtype, [&](auto t) {
    if (large) hipLaunchKernelGGL((mx4_gemm_kernel<decltype(t), 256, 256>), g, b, 0, st, a);
    else hipLaunchKernelGGL((mx4_gemm_kernel<decltype(t), 128, 128>), g, b, 0, st, a);
  });
  return hip_status(hipGetLastError(), "cmk_mx4_bmm launch");
}

extern "C" int cmk_mx4_bmm_rows(const void* x, int x_dtype, long long stride_l, long long stride_m, const uint8_t* b_codes,
                                const uint8_t* b_scales, void* C, int dtype, int L, int M, int N, int K, void* stream) {
  if (L < 0 || M < 0 || N < 0 || K < 0)
    return fail(CMK_ERR_INVALID_ARG, "cmk_mx4_bmm_rows: negative extent (L=%d M=%d N=%d K=%d)", L, M, N, K);
  if (int e = check_dtype("cmk_mx4_bmm_rows", dtype)) return e;
  if (int e = check_dtype("cmk_mx4_bmm_rows", x_dtype)) return e;
  if (M > kMx4RowsFloat || L > 65535)
    return fail(CMK_ERR_UNSUPPORTED, "cmk_mx4_bmm_rows: at most %d rows and 65535 batches (M=%d L=%d)", kMx4RowsFloat, M, L);
  if (L == 0 || M == 0 || N == 0) return CMK_OK;
  if (!C || (K > 0 && (!x || !b_codes || !b_scales))) return fail(CMK_ERR_INVALID_ARG, "cmk_mx4_bmm_rows: null pointer");
  if ((reinterpret_cast<uintptr_t>(b_codes) & 15) || (reinterpret_cast<uintptr_t>(b_scales) & 3))
    return fail(CMK_ERR_INVALID_ARG, "cmk_mx4_bmm_rows: codes need 16-byte alignment, scales 4-byte alignment");
  const Mx4RowsArgs a{x, nullptr, b_codes, b_scales, C, M, N, K, (int)mx4_slabs(K), stride_l, stride_m};
  by_dtype(x_dtype, [&](auto tx) {
    by_dtype(dtype, [&](auto t) { launch_rows<decltype(tx), decltype(t)>(a, L, (hipStream_t)stream); });
  });
  return hip_status(hipGetLastError(), "cmk_mx4_bmm_rows launch");
}
