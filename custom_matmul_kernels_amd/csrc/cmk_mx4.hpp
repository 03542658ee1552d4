// The 4-bit microscaled form of a matrix, and the device code that reads and
// writes it.
//
// A block is 32 consecutive elements along the contraction axis k.  With
// a = max |x| of the block the scale is 2^(s-127), s = max(exponent field of a
// - 2, 0), so that the largest magnitude lands in [4, 8); an element becomes the
// nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 times the scale (ties to the even code,
// beyond 6 to 6) with its sign.  A block that holds an infinity or a NaN gets
// s = 255 and stands for NaN.
//
// Storage of a matrix of R rows and K elements a row, batch by batch:
//   codes  [slabs][R][64] bytes, a slab being 128 elements of k: 4 blocks of 16
//          bytes, the element of even index in the low half of a byte;
//   scales [slabs][R][4] bytes.
// The slab comes first so that a tile of rows x 128 elements is one contiguous
// piece for the direct global-to-LDS loads, for few rows as for many.  k is
// padded with zero codes of scale 0 to whole slabs: no product needs an edge
// case along k.
#pragma once
#include "cmk_launch.hpp"

namespace cmk {

constexpr int kSlab = 128;       // elements of k per slab
constexpr int kSlabBytes = 64;   // of one row
constexpr int kSlabScales = 4;

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4v __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

static inline long long mx4_slabs(int K) { return ((long long)K + kSlab - 1) / kSlab; }

typedef unsigned short u16;
typedef u16 u16x2 __attribute__((ext_vector_type(2)));

// Eight consecutive elements of one type; addresses need the element's alignment
// only (the hardware takes unaligned 16-byte loads).
template <class T>
struct Octet;

template <>
struct Octet<float> {
  float v[8];
  __device__ __forceinline__ void set(int i, float x) { v[i] = x; }
  __device__ __forceinline__ float get(int i) const { return v[i]; }
  __device__ __forceinline__ unsigned top() const {  // largest |x| as fp32 bits
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m;
  }
  __device__ __forceinline__ unsigned codes(float scale) const {
    unsigned w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
  }
};

// 16-bit elements, two to a register: the largest magnitude takes one mask and one
// packed 16-bit maximum per pair.
struct Octet16 {
  unsigned v[4];
  __device__ __forceinline__ unsigned top16() const {
    u16x2 m = __builtin_bit_cast(u16x2, v[0] & 0x7fff7fffu);
#pragma unroll
    for (int i = 1; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, v[i] & 0x7fff7fffu));
    return max((unsigned)m[0], (unsigned)m[1]);
  }
  __device__ __forceinline__ u16 bits(int i) const { return (u16)(v[i >> 1] >> (16 * (i & 1))); }
  __device__ __forceinline__ void set_bits(int i, u16 b) {
    v[i >> 1] = i & 1 ? (v[i >> 1] & 0xffffu) | (unsigned)b << 16 : (v[i >> 1] & 0xffff0000u) | b;
  }
};

template <>
struct Octet<__bf16> : Octet16 {
  __device__ __forceinline__ void set(int i, __bf16 x) { set_bits(i, __builtin_bit_cast(u16, x)); }
  __device__ __forceinline__ float get(int i) const { return __uint_as_float((unsigned)bits(i) << 16); }
  __device__ __forceinline__ unsigned top() const { return top16() << 16; }
  __device__ __forceinline__ unsigned codes(float scale) const {
    unsigned w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, v[0]), scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, v[1]), scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, v[2]), scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, v[3]), scale, 3);
  }
};

template <>
struct Octet<_Float16> : Octet16 {
  __device__ __forceinline__ void set(int i, _Float16 x) { set_bits(i, __builtin_bit_cast(u16, x)); }
  __device__ __forceinline__ float get(int i) const { return (float)__builtin_bit_cast(_Float16, bits(i)); }
  // as fp32: infinities and NaN keep the top exponent
  __device__ __forceinline__ unsigned top() const {
    return __float_as_uint((float)__builtin_bit_cast(_Float16, (u16)top16()));
  }
  __device__ __forceinline__ unsigned codes(float scale) const {
    unsigned w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(f16x2, v[0]), scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(f16x2, v[1]), scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(f16x2, v[2]), scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(f16x2, v[3]), scale, 3);
  }
};

// `left` of the eight elements exist (all, if it is 8 or more; none, if it is
// not positive); the others are zeros and are not touched.
template <class T>
__device__ __forceinline__ Octet<T> load_octet(const T* p, int left) {
  Octet<T> o;
  if (left >= 8) {
    __builtin_memcpy(o.v, p, sizeof(o.v));
  } else {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(o.v) / 4); ++i) o.v[i] = 0;
    if (left > 0) {
#pragma unroll
      for (int i = 0; i < 7; ++i)
        if (i < left) o.set(i, p[i]);
    }
  }
  return o;
}

// The largest value of four neighbouring lanes, in each of them.
__device__ __forceinline__ unsigned quad_max(unsigned v) {
  v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true));  // lanes 1 0 3 2
  return max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true));  // lanes 2 3 0 1
}

// Scale byte of a block whose largest magnitude has these fp32 bits.
__device__ __forceinline__ unsigned scale_byte(unsigned top) {
  const unsigned e = top >> 23;
  return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}

// The scale as the conversion instructions take it: its exponent field counts.
__device__ __forceinline__ float scale_float(unsigned s) { return __uint_as_float(s ? s << 23 : 0x00400000u); }

// Rounds to nearest, ties to even.
template <class T>
__device__ __forceinline__ T from_f32(float x) { return (T)x; }

typedef const __attribute__((address_space(1))) void* gptr;
typedef __attribute__((address_space(3))) void* lptr;

// Waits until at most `left` of the wave's vector-memory instructions are under way.
template <int left>
__device__ __forceinline__ void wait_loads() {
  static_assert(left < 64, "the counter has six bits");
  __builtin_amdgcn_s_waitcnt(0x0f70 | (left & 15) | (left >> 4 << 14));
}

// Waits until the wave's LDS reads have returned.
__device__ __forceinline__ void wait_lds() { __builtin_amdgcn_s_waitcnt(0xc07f); }

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

}  // namespace cmk
