// 4-bit microscaled matrices: quantisation, its inverse, and the batched product.
#include <algorithm>
#include <type_traits>

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

// Two matrices of one type for one launch; the second may be empty.
struct QuantPair {
  QuantArgs of[2];
};

// k contiguous.  Four lanes share a block (8 elements each), 16 lanes a row's
// slab, a wave 16 rows x one slab in four steps: it reads 256 (512) contiguous
// bytes of a row per step and writes one contiguous KB of codes.
template <class T>
__global__ __launch_bounds__(256) void mx4_quantize_rows_kernel(QuantPair both) {
  const int lane = threadIdx.x & 63;
  long long unit = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool second = unit >= both.of[0].groups;
  const QuantArgs& a = both.of[second ? 1 : 0];
  if (second) unit -= both.of[0].groups;
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
    const unsigned s = scale_byte(quad_max(o[p].top()));
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

// Large results are stored past the caches: they would not stay there, and what ran
// before and what runs next keep their lines (dequantisation of 8192 x 8192 to bf16
// 40 -> 34 us and the quantisation in front of it 38 -> 33; a product with 512 MB of
// results 116 -> 119 us, the quantisation of the next call's operands 62 -> 24).  Only
// where rows are whole cache lines: partial lines are merged by the L2 alone.  (The
// inverse down columns stores 1 KB of a row at a time in fp32 and gains at any width: 3 x
// 4096 x 4095 there and back 111 -> 98 us; in 16 bits 8192 x 8192 92 -> 89, 8192 x 8190
// would lose, 100 -> 106.)
constexpr size_t kStreamBytes = 32u << 20;

static int streams(const void* out, long long rows, long long row_bytes) {
  return (size_t)rows * row_bytes >= kStreamBytes && row_bytes % 128 == 0 && (reinterpret_cast<uintptr_t>(out) & 127) == 0;
}

template <bool STREAM, class V>
__device__ __forceinline__ void store_as(V* p, V v) {
  if constexpr (STREAM) __builtin_nontemporal_store(v, p);
  else *p = v;
}

template <bool STREAM, class T>
__device__ __forceinline__ void store_one(T* p, T v) {
  if constexpr (sizeof(T) == 4) store_as<STREAM>((unsigned*)p, __builtin_bit_cast(unsigned, v));
  else store_as<STREAM>((u16*)p, __builtin_bit_cast(u16, v));
}

// N elements, 16 (8) bytes at a time, at any element's address.
template <bool STREAM, class T, int N>
__device__ __forceinline__ void store_run(T* p, const T (&v)[N]) {
  if constexpr (!STREAM) {
    __builtin_memcpy(p, v, sizeof(v));
  } else if constexpr (sizeof(v) % 16 == 0) {
    typedef u32x4v __attribute__((aligned(2))) any16;
#pragma unroll
    for (int i = 0; i < (int)sizeof(v) / 16; ++i) {
      u32x4v w;
      __builtin_memcpy(&w, (const char*)v + 16 * i, 16);
      __builtin_nontemporal_store(w, (any16*)((char*)p + 16 * i));
    }
  } else {
    typedef u32x2 __attribute__((aligned(2))) any8;
    u32x2 w;
    __builtin_memcpy(&w, v, 8);
    __builtin_nontemporal_store(w, (any8*)p);
  }
}

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

template <class T, bool STREAM>
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
      store_run<STREAM>(out, o);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k0 + i < a.K) out[i] = o[i];
    }
  }
}

// Rows innermost: a lane takes one slab of V neighbouring rows, so that it stores V
// values side by side.
template <class T, int V, bool STREAM>
__global__ __launch_bounds__(256) void mx4_dequantize_columns_kernel(DequantArgs a) {
  const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= a.groups) return;
  const long long rg = unit % a.row_groups;
  const long long ls = unit / a.row_groups;
  const int l = (int)(ls / a.slabs), slab = (int)(ls % a.slabs);
  const long long row = (rg * 64 + (threadIdx.x & 63)) * V;
  if (row >= a.R) return;
  const int have = (int)min((long long)V, a.R - row);
  unsigned scales[V];
  u32x4v w[V][4];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const long long at = ls * a.R + row + min(v, have - 1);
    scales[v] = *(const unsigned*)(a.scales + at * kSlabScales);
#pragma unroll
    for (int b = 0; b < 4; ++b) w[v][b] = *(const u32x4v*)(a.codes + at * kSlabBytes + b * 16);
  }
  T* out = (T*)a.out + (long long)l * a.K * a.R + row;
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x[V][8];
#pragma unroll
      for (int v = 0; v < V; ++v) decode_octet(w[v][b][i], scales[v] >> (8 * b) & 255u, x[v]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int k = slab * kSlab + b * 32 + i * 8 + j;
        if (k >= a.K) continue;
        T* p = out + (long long)k * a.R;
        T o[V];
#pragma unroll
        for (int v = 0; v < V; ++v) o[v] = from_f32<T>(x[v][j]);
        if constexpr (V == 1) {
          store_one<STREAM>(p, o[0]);
        } else if (have == V) {
          store_run<STREAM>(p, o);
        } else {
#pragma unroll
          for (int v = 0; v < V; ++v)
            if (v < have) p[v] = o[v];
        }
      }
    }
}

// -------------------------------------------------------------------- product

struct Mx4GemmArgs {
  const uint8_t *a_codes, *a_scales, *b_codes, *b_scales;
  void* c;  // dense [L][M][N]; of several splits: one such after another
  int L, M, N;
  int slabs;
  int tiles_m, tiles_n;
  int splits;  // ranges of slabs
  int stream;  // c is stored past the caches
  int wide;    // rows of c start on 16-byte boundaries and hold whole multiples of them
};

// A work-group of four waves computes a TM x TN tile of C, a wave a quarter of it
// in blocks of 32 x 32 (v_mfma_scale_f32_32x32x64_f8f6f4: 64 elements of k, each
// lane holding one whole 32-element block of one row, so that the lane's scale is
// one byte).
//
// Slabs of both operands (codes and scales) travel by direct global-to-LDS loads
// into a ring of S buffers, S - 2 slabs ahead of the products.  Half a slab's
// fragments are in registers at a time; those of the next half are read while the
// matrix pipe works on them.  The one barrier of a slab sits between its halves:
// it follows the wait for the next slab, whose first half is read behind it, and
// frees the buffer of the slab before.  Within a row the four 16-byte blocks are
// stored at position block ^ ((row >> 2) & 3), so that the 16 rows that the LDS
// serves at a time spread over all banks; the swizzle is produced by choosing
// which block each lane of a load asks for.
template <int TM, int TN, int S>
struct Mx4Tile {
  static constexpr int BM = TM / 64, BN = TN / 64;  // 32 x 32 blocks of a wave
  static constexpr int kCodesA = TM * kSlabBytes, kCodesB = TN * kSlabBytes;
  static constexpr int kStageBytes = kCodesA + kCodesB + (TM + TN) * kSlabScales;
  static constexpr int kLoads = TM / 64 + TN / 64 + 2;  // vector-memory instructions of a wave per slab
  // stages that one address register reaches with the 16-bit offset of an LDS read
  static constexpr int kReach = (65535 - (BM > BN ? BM : BN) * 32 * kSlabBytes) / kStageBytes + 1;
  static constexpr int kBases = (S + kReach - 1) / kReach;
};

// Work-groups go round the eight XCDs in turn, each with an L2 of its own: an XCD
// gets a contiguous run of the tiles of all batches, in strips of eight tile rows,
// so that what runs on it at a time shares few panels of both operands.
__device__ __forceinline__ void place_tile(const Mx4GemmArgs& a, int& split, int& l, int& tile_m, int& tile_n) {
  const int total = gridDim.x, xcd = blockIdx.x & 7, turn = blockIdx.x >> 3;
  const int each = total >> 3, extra = total & 7;
  const int id = xcd * each + min(xcd, extra) + turn;
  const int per_batch = a.tiles_m * a.tiles_n;
  split = id / (per_batch * a.L);
  const int in_split = id - split * per_batch * a.L;
  l = in_split / per_batch;
  const int t = in_split - l * per_batch;
  const int strip = t / (8 * a.tiles_n), in = t - strip * 8 * a.tiles_n;
  const int height = min(8, a.tiles_m - strip * 8);
  tile_m = strip * 8 + in % height;
  tile_n = in / height;
}

template <class T, int TM, int TN, int S>
__global__ __launch_bounds__(256, 1) void mx4_gemm_kernel(Mx4GemmArgs a) {
  using Tile = Mx4Tile<TM, TN, S>;
  constexpr int BM = Tile::BM, BN = Tile::BN;
  static_assert((S & 1) == 0, "the slabs' scales alternate between two sets of registers");
  __shared__ __attribute__((aligned(16))) uint8_t lds[S * Tile::kStageBytes];
  int split, l, tile_m, tile_n;
  place_tile(a, split, l, tile_m, tile_n);
  const int slab0 = (int)((long long)a.slabs * split / a.splits), slabs = (int)((long long)a.slabs * (split + 1) / a.splits) - slab0;
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
  const uint8_t* pa = a.a_codes + (((long long)l * a.slabs + slab0) * a.M + m0) * kSlabBytes;
  const uint8_t* pb = a.b_codes + (((long long)l * a.slabs + slab0) * a.N + n0) * kSlabBytes;
  const uint8_t* psa = a.a_scales + (((long long)l * a.slabs + slab0) * a.M + m0) * kSlabScales;
  const uint8_t* psb = a.b_scales + (((long long)l * a.slabs + slab0) * a.N + n0) * kSlabScales;
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
    const long long more = ++requested < slabs ? 1 : 0;
    pa += more * step_a; pb += more * step_b;
    psa += more * (step_a / (kSlabBytes / kSlabScales)); psb += more * (step_b / (kSlabBytes / kSlabScales));
  };

  // Where this lane reads: one register per half of a slab, operand and group of
  // stages, the rest of an address is the instruction's offset (vector
  // instructions in the loop cost matrix-pipe time).
  constexpr int kReach = Tile::kReach;
  const unsigned lds0 = (unsigned)(uintptr_t)(lptr)lds;
  unsigned at_m[Tile::kBases][2], at_n[Tile::kBases][2], at_cm[Tile::kBases], at_cn[Tile::kBases];
#pragma unroll
  for (int p = 0; p < Tile::kBases; ++p) {
    const unsigned base = lds0 + p * kReach * Tile::kStageBytes;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const unsigned part = ((2 * h + g) ^ ((r >> 2) & 3)) * 16;
      at_m[p][g] = base + (wm + r) * kSlabBytes + part;
      at_n[p][g] = base + Tile::kCodesA + (wn + r) * kSlabBytes + part;
      asm("" : "+v"(at_m[p][g]), "+v"(at_n[p][g]));
    }
    at_cm[p] = base + Tile::kCodesA + Tile::kCodesB + (wm + r) * kSlabScales + 2 * h;
    at_cn[p] = base + Tile::kCodesA + Tile::kCodesB + (TM + wn + r) * kSlabScales + 2 * h;
    asm("" : "+v"(at_cm[p]), "+v"(at_cn[p]));
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
    const unsigned off = stage % kReach * Tile::kStageBytes;
#pragma unroll
    for (int b = 0; b < BM; ++b) f.m[b] = *(l16)(lptr)(uintptr_t)(at_m[stage / kReach][g] + off + b * 32 * kSlabBytes);
#pragma unroll
    for (int b = 0; b < BN; ++b) f.n[b] = *(l16)(lptr)(uintptr_t)(at_n[stage / kReach][g] + off + b * 32 * kSlabBytes);
  };
  auto read_scales = [&](int stage, Scales& c) {
    const unsigned off = stage % kReach * Tile::kStageBytes;
#pragma unroll
    for (int b = 0; b < BM; ++b) c.m[b] = *(l2)(lptr)(uintptr_t)(at_cm[stage / kReach] + off + b * 32 * kSlabScales);
#pragma unroll
    for (int b = 0; b < BN; ++b) c.n[b] = *(l2)(lptr)(uintptr_t)(at_cn[stage / kReach] + off + b * 32 * kSlabScales);
  };
  f32x16 acc[BM][BN] = {};
  auto wide = [](u32x4v v) { return i32x8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0}; };

  // One slab of ring position `stage`, c its scales, d the next one's.
  Half f0, f1;
  auto slab = [&](auto stage, Scales& c, Scales& d) {
    constexpr int Stage = decltype(stage)::value;
    constexpr int Next = (Stage + 1) % S;
    read(Stage, 1, f1);
#pragma unroll
    for (int bm = 0; bm < BM; ++bm)
#pragma unroll
      for (int bn = 0; bn < BN; ++bn)
        acc[bm][bn] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(f0.m[bm]), wide(f0.n[bn]), acc[bm][bn], 4, 4, 0, c.m[bm], 0, c.n[bn]);
    // a read, then as many products as keep the matrix pipe busy until the next
    if constexpr (BM * BN >= 4) {
#pragma unroll
      for (int i = 0; i < BM + BN; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, BM * BN / (BM + BN), 0);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    wait_loads<(S - 3) * Tile::kLoads>();
    meet();
    read_scales(Next, d);
    read(Next, 0, f0);
    fetch((Stage + S - 1) % S);
#pragma unroll
    for (int bm = 0; bm < BM; ++bm)
#pragma unroll
      for (int bn = 0; bn < BN; ++bn)
        acc[bm][bn] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(f1.m[bm]), wide(f1.n[bn]), acc[bm][bn], 4, 4, 1, c.m[bm], 1, c.n[bn]);
    // what the next slab starts with first, the requests behind it
    if constexpr (BM * BN >= 4) {
#pragma unroll
      for (int i = 0; i < BM + BN; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, std::max(1, BM * BN / 2 / (BM + BN)), 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      }
#pragma unroll
      for (int i = 0; i < Tile::kLoads; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  if (slabs > 0) {
    Scales c0, c1;
#pragma unroll
    for (int s = 0; s < S - 1; ++s) fetch(s);
    wait_loads<(S - 2) * Tile::kLoads>();
    meet();
    read_scales(0, c0);
    read(0, 0, f0);
    int left = slabs;
    for (; left >= S; left -= S) {
      slab(Int<0>{}, c0, c1);
      slab(Int<1>{}, c1, c0);
      slab(Int<2>{}, c0, c1);
      slab(Int<3>{}, c1, c0);
      if constexpr (S == 8) {
        slab(Int<4>{}, c0, c1);
        slab(Int<5>{}, c1, c0);
        slab(Int<6>{}, c0, c1);
        slab(Int<7>{}, c1, c0);
      }
    }
    if (left > 0) slab(Int<0>{}, c0, c1);
    if (left > 1) slab(Int<1>{}, c1, c0);
    if (left > 2) slab(Int<2>{}, c0, c1);
    if constexpr (S == 8) {
      if (left > 3) slab(Int<3>{}, c1, c0);
      if (left > 4) slab(Int<4>{}, c0, c1);
      if (left > 5) slab(Int<5>{}, c1, c0);
      if (left > 6) slab(Int<6>{}, c0, c1);
    }
    wait_loads<0>();  // no load may land after the work-group has ended
  }

  // lane: column n = lane & 31, rows 8 * (i / 4) + 4 * h + i % 4: a store covers two
  // runs of 32 columns.  16-bit results would be runs of 64 bytes, two at a time; they
  // go through the wave's share of LDS and out 16 bytes a lane (stores of pairs of
  // columns, exchanged between neighbouring lanes, took 380 instead of 275 us at
  // 8192^3).
  T* c = (T*)a.c + ((long long)split * a.L + l) * a.M * a.N;
  auto store_tile = [&](auto past) {
    constexpr bool STREAM = decltype(past)::value;
    if constexpr (sizeof(T) == 2) {
      if (a.wide) {
        constexpr int WM = TM / 2, WN = TN / 2, kPitch = WN * 2 + 16, kLanes = WN / 8, kRows = 64 / kLanes;
        static_assert(4 * WM * kPitch <= S * Tile::kStageBytes, "the tile fits into the ring");
        meet();  // every wave has read its last slab
        uint8_t* mine = lds + wave * (WM * kPitch);
#pragma unroll
        for (int bm = 0; bm < BM; ++bm)
#pragma unroll
          for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int bn = 0; bn < BN; ++bn)
              *(T*)(mine + (bm * 32 + 8 * (i >> 2) + 4 * h + (i & 3)) * kPitch + (bn * 32 + r) * 2) = from_f32<T>(acc[bm][bn][i]);
        const int col = lane % kLanes * 8, n = n0 + wn + col;
        for (int i = lane / kLanes; i < WM; i += kRows) {
          const u32x4v v = *(const u32x4v*)(mine + i * kPitch + col * 2);
          const int m = m0 + wm + i;
          if (m < a.M && n < a.N) store_as<STREAM>((u32x4v*)(c + (long long)m * a.N + n), v);
        }
        return;
      }
    }
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
          if (n < a.N) store_one<STREAM>(row + n, from_f32<T>(acc[bm][bn][i]));
        }
      }
  };
  if (a.stream) store_tile(Int<1>{});
  else store_tile(Int<0>{});
}

// The sum of the splits, in their order.
template <class T>
__global__ __launch_bounds__(256) void mx4_join_kernel(const float* part, T* c, long long n, int splits) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    float sum = 0;
    for (int s0 = 0; s0 < splits; s0 += 8) {
      float v[8];
#pragma unroll
      for (int s = 0; s < 8; ++s) v[s] = s0 + s < splits ? part[(s0 + s) * n + i] : 0.0f;
#pragma unroll
      for (int s = 0; s < 8; ++s) sum += v[s];
    }
    c[i] = from_f32<T>(sum);
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

constexpr int kRowsLds = 72 * 1024;

// A work-group takes 16 * RG columns of C and all its rows (up to 16 * MB); its W
// waves split the slabs and their sums meet in LDS, in the order of the waves.
// There is nothing to gain but the stream of the right operand: its fragments
// (1 KB of contiguous codes per instruction) go straight to registers, a ring of U
// slabs under way.  The left operand's codes wait in LDS, as many slabs of all rows
// at a time as fit, quantised on the way there if TX is an element type; uint8_t
// stands for codes.
template <class TX, class T, int W, int RG, int MB, int U>
__global__ __launch_bounds__(64 * W) void mx4_rows_kernel(Mx4RowsArgs a) {
  constexpr bool kCodes = sizeof(TX) == 1;
  constexpr int kSteps = sizeof(TX) == 4 ? 2 : 4;
  static_assert(W == 8 && W * RG * MB * 1024 <= kRowsLds, "the partial sums fit");
  __shared__ __attribute__((aligned(16))) char lds[kRowsLds];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int l = blockIdx.y, n0 = blockIdx.x * 16 * RG;
  // a row of `piece` slabs: codes and scales, each 16 (4) bytes longer so that the
  // rows of a fragment spread over the banks
  const int fit = (kRowsLds / a.M - 20) / (kSlabBytes + kSlabScales);
  const int piece = min(a.slabs, fit);
  const int pitch = piece * kSlabBytes + 16, spitch = piece * kSlabScales + 4;
  char* const scales = lds + a.M * pitch;
  const int together = a.M > 4 ? 8 : a.M > 2 ? 4 : a.M > 1 ? 2 : 1;  // rows that the waves stage at a time
  const uint8_t* bc[RG];
  const uint8_t* bs[RG];
#pragma unroll
  for (int g = 0; g < RG; ++g) {
    const long long at = (long long)l * a.slabs * a.N + min(n0 + g * 16 + r, a.N - 1);
    bc[g] = a.b_codes + at * kSlabBytes + q * 16;
    bs[g] = a.b_scales + at * kSlabScales + q;
  }
  const long long step_codes = (long long)a.N * kSlabBytes, step_scales = (long long)a.N * kSlabScales;
  f32x4 acc[RG][MB] = {};
  auto wide = [](u32x4v v) { return i32x8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0}; };
  for (int first = 0; first < a.slabs; first += piece) {
    const int end = min(a.slabs, first + piece);
    Mx4Fragment fb[U][RG];
    auto request = [&](int u, int s) {
#pragma unroll
      for (int g = 0; g < RG; ++g) {
        fb[u][g].codes = __builtin_nontemporal_load((const u32x4v*)(bc[g] + s * step_codes));
        fb[u][g].scale = bs[g][s * step_scales];
      }
    };
    // A wave takes 16 slabs of one row at a time (a step); with few rows several waves
    // share one.  Four lanes share a block, so that a load reads 1 KB in one run.
    // Loads are awaited in the order of their issue: the first steps are requested
    // ahead of the right operand's ring, so that they are quantised while that is on
    // its way.
    const int start = first + wave / together * 16, each = W / together * 16;
    const int whole = min(end, a.K / kSlab);  // slabs up to here hold 128 elements
    int m = start < end ? wave & (together - 1) : a.M, s0 = start;  // the next step
    int step_m[kSteps], step_s[kSteps];                             // those under way
    Octet<std::conditional_t<kCodes, float, TX>> o[kSteps][kCodes ? 1 : 4];
    Mx4Fragment f[kSteps];
    auto load_steps = [&]() {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        step_m[i] = m;
        step_s[i] = s0;
        if (m < a.M) {
          if constexpr (kCodes) {
            const long long at = ((long long)l * a.slabs + min(s0 + (lane >> 2), end - 1)) * a.M + m;
            f[i].codes = *(const u32x4v*)((const uint8_t*)a.x + at * kSlabBytes + (lane & 3) * 16);
            f[i].scale = a.x_scales[at * kSlabScales + (lane & 3)];
          } else {
            const TX* x = (const TX*)a.x + l * a.sl + m * a.sm + (long long)s0 * kSlab + lane * 8;
            if (s0 + 16 <= whole) {  // no lane is beyond the end
#pragma unroll
              for (int e = 0; e < 4; ++e) __builtin_memcpy(o[i][e].v, x + 4 * e * kSlab, sizeof(o[i][e].v));
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int s = s0 + 4 * e + (lane >> 4);
                o[i][e] = load_octet(x + 4 * e * kSlab, s < end ? a.K - s * kSlab - (lane & 15) * 8 : 0);
              }
            }
          }
          s0 += each;
          if (s0 >= end) { s0 = start; m += together; }
        }
      }
    };
    load_steps();
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (first + wave + u * W < end) request(u, first + wave + u * W);
    if (first > 0) __syncthreads();
    while (step_m[0] < a.M) {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        if (step_m[i] >= a.M) break;
        char* codes = lds + step_m[i] * pitch;
        char* bytes = scales + step_m[i] * spitch;
        if constexpr (kCodes) {
          const int s = step_s[i] + (lane >> 2);
          if (s < end) {
            *(u32x4v*)(codes + (s - first) * kSlabBytes + (lane & 3) * 16) = f[i].codes;
            bytes[(s - first) * kSlabScales + (lane & 3)] = (char)f[i].scale;
          }
        } else {
          // a step's codes and scales are contiguous: 4 bytes a lane and one of four lanes
          codes += (step_s[i] - first) * kSlabBytes + lane * 4;
          bytes += (step_s[i] - first) * kSlabScales + (lane >> 2);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const unsigned scale = scale_byte(quad_max(o[i][e].top()));
            const unsigned w = scale == 255u ? 0u : o[i][e].codes(scale_float(scale));
            if (step_s[i] + 16 <= end || step_s[i] + 4 * e + (lane >> 4) < end) {
              *(unsigned*)(codes + 4 * e * kSlabBytes) = w;
              if ((lane & 3) == 0) bytes[4 * e * kSlabScales] = (char)scale;
            }
          }
        }
      }
      load_steps();
    }
    __syncthreads();
    for (int s0 = first + wave; s0 < end; s0 += W * U) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int s = s0 + u * W;
        if (s >= end) break;
        Mx4Fragment fx[MB];
#pragma unroll
        for (int b = 0; b < MB; ++b) {
          const int m = min(b * 16 + r, a.M - 1);
          fx[b].codes = *(const u32x4v*)(lds + m * pitch + (s - first) * kSlabBytes + q * 16);
          fx[b].scale = (unsigned char)scales[m * spitch + (s - first) * kSlabScales + q];
        }
#pragma unroll
        for (int g = 0; g < RG; ++g)
#pragma unroll
          for (int b = 0; b < MB; ++b)
            acc[g][b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(fb[u][g].codes), wide(fx[b].codes), acc[g][b], 4, 4, 0,
                                                                        fb[u][g].scale, 0, fx[b].scale);
        if (s + U * W < end) request(u, s + U * W);
      }
    }
  }
  f32x4(*part)[RG][MB][64] = (f32x4(*)[RG][MB][64])lds;
  __syncthreads();
#pragma unroll
  for (int g = 0; g < RG; ++g)
#pragma unroll
    for (int b = 0; b < MB; ++b) part[wave][g][b][lane] = acc[g][b];
  __syncthreads();
  T* c = (T*)a.c + (long long)l * a.M * a.N;
  for (int v = threadIdx.x; v < RG * 16 * min(a.M, MB * 16); v += 64 * W) {
    // neighbouring threads take neighbouring columns of one row
    const int n = v % (16 * RG), m = v / (16 * RG);
    const int g = n >> 4, i = n & 3, from = ((n & 15) >> 2) * 16 + (m & 15), b = m >> 4;
    if (n0 + n < a.N) {
      float sum = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) sum += part[w][g][b][from][i];
      c[(long long)m * a.N + n0 + n] = from_f32<T>(sum);
    }
  }
}

// Rows up to this many are served by mx4_rows_kernel.
constexpr int kMx4Rows = 32;

// TX: uint8_t or the element type of the left operand.
template <class TX, class T>
static void launch_rows(const Mx4RowsArgs& a, int L, hipStream_t st) {
  const long long groups = (long long)ceil_div(a.N, 16) * L;
  const int cus = compute_units();
  // Row groups of a wave share the left operand's fragments and its quantisation;
  // fewer where that would leave compute units without work.
  auto run = [&](auto kernel, int rg) { hipLaunchKernelGGL(kernel, dim3(ceil_div(a.N, 16 * rg), L), dim3(512), 0, st, a); };
  if (a.M <= 16) {
    if (groups >= 4LL * cus) run(mx4_rows_kernel<TX, T, 8, 4, 1, 4>, 4);
    else if (groups >= 2LL * cus) run(mx4_rows_kernel<TX, T, 8, 2, 1, 4>, 2);
    else run(mx4_rows_kernel<TX, T, 8, 1, 1, 4>, 1);
  } else if constexpr (sizeof(TX) == 1) {
    if (groups >= 2LL * cus) run(mx4_rows_kernel<TX, T, 8, 2, 2, 4>, 2);
    else run(mx4_rows_kernel<TX, T, 8, 1, 2, 4>, 1);
  }
}

static bool use_rows(int L, int M, int N, int K) {
  // What one launch holds: 65535 batches, and along N work-groups of 512 threads for 64
  // columns.
  if (M > kMx4Rows || L > 65535 || !fits_launch(ceil_div(N, 64), 512)) return false;
  // From 17 rows on the tiles win where there are enough of them (32 rows against
  // 16384 x 8192: 24 us by rows, 14 by tiles; 4096 x 4096: 5.4 and 7.6) or k is long
  // enough to be cut (1024 x 16384: 16 and 8).
  return M <= 16 || ((long long)L * ceil_div(N, 64) < compute_units() && mx4_slabs(K) <= 64);
}

struct Mx4Plan {
  int tile, splits;
  size_t bytes;
};

// Microseconds that `tiles` tiles of `slabs` slabs take, as measured on 256 compute
// units: a fixed part and one per slab, for a compute unit that holds one or two
// work-groups (the largest tile fills its LDS).  One tile each, 64 slabs: 61, 28, 13
// us; two each: 45 (of 128), 21 (of 64).
static double tile_cost(int tile, long long tiles, int slabs, int cus) {
  const double one = tile == 256 ? 9 + 0.85 * slabs : tile == 128 ? 4.5 + 0.37 * slabs : 3.5 + 0.145 * slabs;
  const double two = tile == 256 ? 2 * one : tile == 128 ? 5 + 0.63 * slabs : 3.5 + 0.28 * slabs;
  const long long rest = tiles % (2LL * cus);
  return tiles / (2LL * cus) * two + (rest == 0 ? 0 : rest <= cus ? one : two);
}

// The tile, and for the smallest the number of ranges of k, that cost least.  Ranges
// pay for a second kernel that reads what they wrote (1024 x 1024 with 64 slabs: 13 us
// whole, 19 in two ranges; 128 x 1024 with 128 slabs: 40 whole, 13 in eight).
static Mx4Plan mx4_plan(int L, int M, int N, int K) {
  const int cus = compute_units(), slabs = (int)mx4_slabs(K);
  auto tiles = [&](int t) { return (long long)L * ceil_div(M, t) * ceil_div(N, t); };
  Mx4Plan p{64, 1, 0};
  if (use_rows(L, M, N, K)) return p;
  double best = tile_cost(64, tiles(64), slabs, cus);
  for (int tile : {128, 256}) {
    const double cost = tile_cost(tile, tiles(tile), slabs, cus);
    if (cost < best) { best = cost; p.tile = tile; }
  }
  for (int s = 2; s <= 16 && s * 4 <= slabs && s * tiles(64) <= 2LL * cus; ++s) {
    const double cost = tile_cost(64, s * tiles(64), ceil_div(slabs, s), cus) + 4 + 8e-6 / 4.9 * s * L * M * N;
    if (cost < best) { best = cost; p.tile = 64; p.splits = s; }
  }
  if (p.splits > 1) p.bytes = (size_t)p.splits * L * M * N * 4;
  return p;
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

constexpr int kThreads = 256;

static int check_launch(const char* who, long long groups) {
  if (!fits_launch(groups, kThreads))
    return fail(CMK_ERR_UNSUPPORTED, "%s: needs %lld work-groups, more than a launch holds", who, groups);
  return CMK_OK;
}

// Calls f with a value of the element type.
template <class F>
static void by_dtype(int dtype, F f) {
  if (dtype == CMK_F32) f(0.0f);
  else if (dtype == CMK_BF16) f((__bf16)0.0f);
  else f((_Float16)0.0f);
}

// Whether the kernel that reads along k takes the matrix.
static bool along_k(int K, long long stride_k) { return stride_k == 1 || K == 1; }

static QuantArgs quant_args(const void* x, uint8_t* codes, uint8_t* scales, int L, int R, int K, long long sl, long long sr, long long sk) {
  QuantArgs a{x, codes, scales, L, R, K, mx4_slabs(K), 0, 0, sl, sr, sk};
  a.row_groups = along_k(K, sk) ? ((long long)R + 15) / 16 : ((long long)R + 63) / 64;
  a.groups = a.row_groups * a.slabs * L;
  return a;
}

// Quantises one matrix, or two of one type that are both read along k (b then).
static int launch_quantize(int dtype, const QuantArgs& a, const QuantArgs* b, hipStream_t st) {
  const long long grid = (a.groups + (b ? b->groups : 0) + 3) / 4;
  if (grid == 0) return CMK_OK;
  if (int e = check_launch("quantisation", grid)) return e;
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (along_k(a.K, a.sk)) {
      const QuantPair both{{a, b ? *b : QuantArgs{}}};
      hipLaunchKernelGGL(mx4_quantize_rows_kernel<T>, dim3((unsigned)grid), dim3(256), 0, st, both);
    } else {
      hipLaunchKernelGGL(mx4_quantize_columns_kernel<T>, dim3((unsigned)grid), dim3(256), 0, st, a);
    }
  });
  return hip_status(hipGetLastError(), "quantisation launch");
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
  return launch_quantize(dtype, quant_args(x, codes, scales, L, R, K, stride_l, stride_r, stride_k), nullptr, (hipStream_t)stream);
}

extern "C" int cmk_mx4_dequantize(const uint8_t* codes, const uint8_t* scales, void* out, int dtype, int L, int R,
                                  int K, int rows_innermost, void* stream) {
  if (int e = check_mx4("cmk_mx4_dequantize", L, R, K)) return e;
  if (int e = check_dtype("cmk_mx4_dequantize", dtype)) return e;
  if (L == 0 || R == 0 || K == 0) return CMK_OK;
  if (!out || !codes || !scales) return fail(CMK_ERR_INVALID_ARG, "cmk_mx4_dequantize: null pointer");
  if ((reinterpret_cast<uintptr_t>(codes) & 15) || (reinterpret_cast<uintptr_t>(scales) & 3))
    return fail(CMK_ERR_INVALID_ARG, "cmk_mx4_dequantize: codes need 16-byte alignment, scales 4-byte alignment");
  const int size = dtype == CMK_F32 ? 4 : 2;
  DequantArgs a{codes, scales, out, L, R, K, mx4_slabs(K), 0, 0};
  // four rows a lane where a wave's 256 rows are there
  const int v = rows_innermost && R >= 256 ? 4 : 1;
  const bool large = (size_t)L * R * K * size >= kStreamBytes;
  const bool past = !rows_innermost ? streams(out, (long long)L * R, (long long)K * size)
                                    : v == 4 && (size == 4 ? large : streams(out, (long long)L * K, (long long)R * size));
  a.row_groups = rows_innermost ? ((long long)R + 64 * v - 1) / (64 * v) : ((long long)R + 15) / 16;
  a.groups = a.row_groups * a.slabs * L;
  const long long grid = (a.groups + 3) / 4;
  if (int e = check_launch("cmk_mx4_dequantize", grid)) return e;
  hipStream_t st = (hipStream_t)stream;
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const dim3 g((unsigned)grid), b(256);
    auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, g, b, 0, st, a); };
    if (!rows_innermost) past ? run(mx4_dequantize_rows_kernel<T, true>) : run(mx4_dequantize_rows_kernel<T, false>);
    else if (v == 4) past ? run(mx4_dequantize_columns_kernel<T, 4, true>) : run(mx4_dequantize_columns_kernel<T, 4, false>);
    else run(mx4_dequantize_columns_kernel<T, 1, false>);
  });
  return hip_status(hipGetLastError(), "cmk_mx4_dequantize launch");
}

// Where the pieces of a product's workspace lie: codes and scales of the operands
// that are quantised in the call, sums of the ranges of k.
struct Mx4Work {
  bool on_the_way;  // the left operand is quantised by the product itself
  size_t codes[2], scales[2], sums, bytes;
};

// Up to this many rows of a float left operand the product quantises by itself (16
// rows against 16384 x 8192: 19.0 us that way, 17.1 in a launch before; 4 rows: 13.8
// and 15.1).
constexpr int kMx4RowsFloat = 8;

static Mx4Work mx4_work(int a_dtype, int b_dtype, bool a_along_k, int L, int M, int N, int K) {
  Mx4Work w{};
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  size_t at = 0;
  w.on_the_way = a_dtype != CMK_MX4 && a_along_k && M <= kMx4RowsFloat && use_rows(L, M, N, K);
  const int rows[2] = {M, N};
  const bool apart[2] = {a_dtype != CMK_MX4 && !w.on_the_way, b_dtype != CMK_MX4};
  for (int i = 0; i < 2; ++i)
    if (apart[i]) {
      const size_t units = (size_t)L * mx4_slabs(K) * rows[i];
      w.codes[i] = at; at += up(units * kSlabBytes);
      w.scales[i] = at; at += up(units * kSlabScales);
    }
  w.sums = at; at += up(mx4_plan(L, M, N, K).bytes);
  w.bytes = at;
  return w;
}

static int check_product(const char* who, const cmk_mx4_operand* A, const cmk_mx4_operand* B, int dtype, int L, int M, int N, int K) {
  if (!A || !B) return fail(CMK_ERR_INVALID_ARG, "%s: null operand", who);
  if (L < 0 || M < 0 || N < 0 || K < 0)
    return fail(CMK_ERR_INVALID_ARG, "%s: negative extent (L=%d M=%d N=%d K=%d)", who, L, M, N, K);
  if (M > (1 << 30) || N > (1 << 30))
    return fail(CMK_ERR_UNSUPPORTED, "%s: M and N are at most %d (M=%d N=%d)", who, 1 << 30, M, N);
  if (int e = check_dtype(who, dtype)) return e;
  for (const cmk_mx4_operand* o : {A, B})
    if (o->dtype != CMK_MX4)
      if (int e = check_dtype(who, o->dtype)) return e;
  return CMK_OK;
}

extern "C" size_t cmk_mx4_workspace_bytes(const cmk_mx4_operand* A, const cmk_mx4_operand* B, int L, int M, int N, int K) {
  if (check_product("cmk_mx4_workspace_bytes", A, B, CMK_F32, L, M, N, K) || L == 0 || M == 0 || N == 0) return 0;
  return mx4_work(A->dtype, B->dtype, along_k(K, A->stride_k), L, M, N, K).bytes;
}

extern "C" int cmk_mx4_bmm(const cmk_mx4_operand* A, const cmk_mx4_operand* B, void* C, int dtype, int L, int M, int N, int K,
                           void* workspace, size_t workspace_bytes, void* stream) {
  if (int e = check_product("cmk_mx4_bmm", A, B, dtype, L, M, N, K)) return e;
  if (L == 0 || M == 0 || N == 0) return CMK_OK;
  if (!C) return fail(CMK_ERR_INVALID_ARG, "cmk_mx4_bmm: null pointer");
  if (K > 0)
    for (const cmk_mx4_operand* o : {A, B}) {
      if (!o->data || (o->dtype == CMK_MX4 && !o->scales)) return fail(CMK_ERR_INVALID_ARG, "cmk_mx4_bmm: null pointer");
      if (o->dtype == CMK_MX4 && ((reinterpret_cast<uintptr_t>(o->data) & 15) || (reinterpret_cast<uintptr_t>(o->scales) & 3)))
        return fail(CMK_ERR_INVALID_ARG, "cmk_mx4_bmm: codes need 16-byte alignment, scales 4-byte alignment");
    }
  const Mx4Work w = mx4_work(A->dtype, B->dtype, along_k(K, A->stride_k), L, M, N, K);
  if (w.bytes > 0 && (!workspace || workspace_bytes < w.bytes || (reinterpret_cast<uintptr_t>(workspace) & 255)))
    return fail(CMK_ERR_WORKSPACE, "cmk_mx4_bmm: needs a 256-byte aligned workspace of %zu bytes, got %zu", w.bytes, workspace_bytes);
  const Mx4Plan p = mx4_plan(L, M, N, K);
  const long long grid = (long long)L * ceil_div(M, p.tile) * ceil_div(N, p.tile) * p.splits;
  if (!use_rows(L, M, N, K))
    if (int e = check_launch("cmk_mx4_bmm", grid)) return e;
  uint8_t* ws = (uint8_t*)workspace;
  hipStream_t st = (hipStream_t)stream;

  const uint8_t* codes[2] = {(const uint8_t*)A->data, (const uint8_t*)B->data};
  const uint8_t* scales[2] = {A->scales, B->scales};
  QuantArgs q[2];
  const cmk_mx4_operand* pending[2];
  int count = 0;
  for (int i = 0; i < 2; ++i) {
    const cmk_mx4_operand* o = i == 0 ? A : B;
    if (o->dtype == CMK_MX4 || (i == 0 && w.on_the_way)) continue;
    codes[i] = ws + w.codes[i];
    scales[i] = ws + w.scales[i];
    q[count] = quant_args(o->data, ws + w.codes[i], ws + w.scales[i], L, i == 0 ? M : N, K, o->stride_l, o->stride_r, o->stride_k);
    pending[count++] = o;
  }
  if (count == 2 && pending[0]->dtype == pending[1]->dtype && along_k(K, pending[0]->stride_k) && along_k(K, pending[1]->stride_k)) {
    if (int e = launch_quantize(pending[0]->dtype, q[0], &q[1], st)) return e;
  } else {
    for (int i = 0; i < count; ++i)
      if (int e = launch_quantize(pending[i]->dtype, q[i], nullptr, st)) return e;
  }

  if (use_rows(L, M, N, K)) {
    if (w.on_the_way) {
      const Mx4RowsArgs r{A->data, nullptr, codes[1], scales[1], C, M, N, K, (int)mx4_slabs(K), A->stride_l, A->stride_r};
      by_dtype(A->dtype, [&](auto tx) {
        by_dtype(dtype, [&](auto t) { launch_rows<decltype(tx), decltype(t)>(r, L, st); });
      });
    } else {
      const Mx4RowsArgs r{codes[0], scales[0], codes[1], scales[1], C, M, N, K, (int)mx4_slabs(K), 0, 0};
      by_dtype(dtype, [&](auto t) { launch_rows<uint8_t, decltype(t)>(r, L, st); });
    }
    return hip_status(hipGetLastError(), "cmk_mx4_bmm launch");
  }
  Mx4GemmArgs a{codes[0], scales[0], codes[1], scales[1], C, L, M, N, (int)mx4_slabs(K), ceil_div(M, p.tile), ceil_div(N, p.tile), p.splits,
                p.splits == 1 && streams(C, (long long)L * M, (long long)N * (dtype == CMK_F32 ? 4 : 2)),
                (N & 7) == 0 && (reinterpret_cast<uintptr_t>(C) & 15) == 0};
  const dim3 g((unsigned)grid), b(kThreads);
  auto gemm = [&](auto t) {
    using T = decltype(t);
    if (p.tile == 256) hipLaunchKernelGGL((mx4_gemm_kernel<T, 256, 256, 4>), g, b, 0, st, a);
    else if (p.tile == 128) hipLaunchKernelGGL((mx4_gemm_kernel<T, 128, 128, 4>), g, b, 0, st, a);
    else hipLaunchKernelGGL((mx4_gemm_kernel<T, 64, 64, 8>), g, b, 0, st, a);
  };
  if (p.splits == 1) {
    by_dtype(dtype, gemm);
  } else {
    float* sums = (float*)(ws + w.sums);
    a.c = sums;
    gemm(0.0f);
    const long long n = (long long)L * M * N;
    const dim3 joins((unsigned)std::min<long long>((n + 255) / 256, 16LL * compute_units()));
    by_dtype(dtype, [&](auto t) {
      hipLaunchKernelGGL(mx4_join_kernel<decltype(t)>, joins, b, 0, st, sums, (decltype(t)*)C, n, p.splits);
    });
  }
  return hip_status(hipGetLastError(), "cmk_mx4_bmm launch");
}
