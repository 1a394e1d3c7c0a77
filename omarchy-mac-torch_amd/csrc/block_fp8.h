// Tensors of 16 and 32 bits as vectors of eight floats, and the 8-bit format of the feed-forward operators: e4m3 values
// with a float32 scale for each block of 128 along the row, scale = max(largest magnitude, 1e-30) / 448, so that the
// block's largest value is e4m3's largest, 448. Shared by the norm, quantization and matrix-product kernels.
#pragma once

#include "omt_internal.h"

namespace omt {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kFp8Block = 128;
constexpr float kFp8Max = 448.f;      // e4m3's largest value
constexpr float kFp8Floor = 1e-30f;   // a block of smaller values is scaled as if this were its largest

// ---- eight consecutive elements of a row, as floats; those from `cols` on read as 0 and are not written -------------
// VEC: every row starts on 16 bytes and holds a multiple of eight elements, so the eight are in range together. Without it
// they are read and written together where all are in range, at their type's alignment, and one by one at a row's end.

template <bool VEC>
__device__ __forceinline__ f32x8 load8(const float* p, int64_t c, int64_t cols) {
  f32x8 v = {};
  if constexpr (VEC) {
    if (c < cols) {
      const f32x4 a = *(const f32x4*)(p + c), b = *(const f32x4*)(p + c + 4);
      v = f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
  } else if (c + 8 <= cols) {
    __builtin_memcpy(&v, p + c, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < cols) v[e] = p[c + e];
  }
  return v;
}
template <bool VEC>
__device__ __forceinline__ f32x8 load8(const __bf16* p, int64_t c, int64_t cols) {
  f32x8 v = {};
  if constexpr (VEC) {
    if (c < cols) v = __builtin_convertvector(*(const bf16x8*)(p + c), f32x8);
  } else if (c + 8 <= cols) {
    bf16x8 b;
    __builtin_memcpy(&b, p + c, sizeof(b));
    v = __builtin_convertvector(b, f32x8);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < cols) v[e] = (float)p[c + e];
  }
  return v;
}
// e4m3, without its scale
__device__ __forceinline__ f32x8 widen_fp8x8(uint2 w) {
  f32x8 v;
  v[0] = __builtin_amdgcn_cvt_f32_fp8((int)w.x, 0), v[1] = __builtin_amdgcn_cvt_f32_fp8((int)w.x, 1);
  v[2] = __builtin_amdgcn_cvt_f32_fp8((int)w.x, 2), v[3] = __builtin_amdgcn_cvt_f32_fp8((int)w.x, 3);
  v[4] = __builtin_amdgcn_cvt_f32_fp8((int)w.y, 0), v[5] = __builtin_amdgcn_cvt_f32_fp8((int)w.y, 1);
  v[6] = __builtin_amdgcn_cvt_f32_fp8((int)w.y, 2), v[7] = __builtin_amdgcn_cvt_f32_fp8((int)w.y, 3);
  return v;
}
template <bool VEC>
__device__ __forceinline__ f32x8 load8(const uint8_t* p, int64_t c, int64_t cols) {
  uint2 w = make_uint2(0, 0);
  if constexpr (VEC) {
    if (c < cols) w = *(const uint2*)(p + c);
  } else if (c + 8 <= cols) {
    __builtin_memcpy(&w, p + c, sizeof(w));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < cols) (e < 4 ? w.x : w.y) |= (uint32_t)p[c + e] << (8 * (e & 3));
  }
  return widen_fp8x8(w);
}
template <bool VEC>
__device__ __forceinline__ void store8(float* p, int64_t c, int64_t cols, f32x8 v) {
  if constexpr (VEC) {
    if (c < cols) {
      *(f32x4*)(p + c) = f32x4{v[0], v[1], v[2], v[3]};
      *(f32x4*)(p + c + 4) = f32x4{v[4], v[5], v[6], v[7]};
    }
  } else if (c + 8 <= cols) {
    __builtin_memcpy(p + c, &v, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < cols) p[c + e] = v[e];
  }
}
template <bool VEC>
__device__ __forceinline__ void store8(__bf16* p, int64_t c, int64_t cols, f32x8 v) {
  if constexpr (VEC) {
    if (c < cols) *(bf16x8*)(p + c) = __builtin_convertvector(v, bf16x8);
  } else if (c + 8 <= cols) {
    const bf16x8 b = __builtin_convertvector(v, bf16x8);
    __builtin_memcpy(p + c, &b, sizeof(b));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < cols) p[c + e] = (__bf16)v[e];
  }
}
// v as it reads back from memory of type T
__device__ __forceinline__ f32x8 rounded8(f32x8 v, const float*) { return v; }
__device__ __forceinline__ f32x8 rounded8(f32x8 v, const __bf16*) {
  return __builtin_convertvector(__builtin_convertvector(v, bf16x8), f32x8);
}

// ---- scales ---------------------------------------------------------------------------------------------------------
// Magnitudes are compared as bits: finite < infinity < NaN, so that a block holding either gets a scale that is not
// finite, and every value it stands for is NaN.

__device__ __forceinline__ uint32_t abs_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t max_u32(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t abs_bits8(f32x8 v) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max_u32(m, abs_bits(v[e]));
  return m;
}
// the largest over each row of 16 lanes, in every lane of the row (all lanes of the row active)
__device__ __forceinline__ uint32_t row16_max(uint32_t m) {
  m = max_u32(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, false));   // quad_perm [1,0,3,2]
  m = max_u32(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, false));   // quad_perm [2,3,0,1]
  m = max_u32(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xF, 0xF, false));  // row_half_mirror
  return max_u32(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x140, 0xF, 0xF, false));  // row_mirror
}
__device__ __forceinline__ float block_scale(uint32_t amax_bits) {
  return __builtin_bit_cast(float, max_u32(amax_bits, __builtin_bit_cast(uint32_t, kFp8Floor))) / kFp8Max;
}
// The next power of two from that scale on: amax = 1.m * 2^E with 448 = 1.75 * 2^8 gives 2^(E - 8), or 2^(E - 7) where
// the mantissa is over .75. Values divided by it and multiplied back are exact, and so are e4m3 values times it in
// bfloat16.
__device__ __forceinline__ float block_scale_pow2(uint32_t amax_bits) {
  const uint32_t b = max_u32(amax_bits, __builtin_bit_cast(uint32_t, kFp8Floor));
  if (b >= 0x7f800000u) return __builtin_bit_cast(float, b);
  return __builtin_bit_cast(float, ((b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1u : 0u)) << 23);
}

// ---- e4m3 ------------------------------------------------------------------------------------------------------------
// Rounded to nearest even; magnitudes are at most 448 times 1 + 2^-22 here (464 and less round to 448).

__device__ __forceinline__ uint32_t pack_fp8(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
__device__ __forceinline__ uint2 pack_fp8x8(f32x8 v, float inv) {
  return make_uint2(pack_fp8(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                    pack_fp8(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
}
template <bool VEC>
__device__ __forceinline__ void store_fp8x8(uint8_t* p, int64_t c, int64_t cols, uint2 w) {
  if constexpr (VEC) {
    if (c < cols) *(uint2*)(p + c) = w;
  } else if (c + 8 <= cols) {
    __builtin_memcpy(p + c, &w, sizeof(w));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < cols) p[c + e] = (uint8_t)((e < 4 ? w.x : w.y) >> (8 * (e & 3)));
  }
}

}  // namespace omt
