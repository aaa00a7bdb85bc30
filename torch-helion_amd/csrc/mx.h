// Blocks of the OCP microscaling format, as the kernels of mx.hip and mx_gemm.hip
// make them: 32 values that share a scale 2^(s - 127).
#pragma once

#include "common.h"

#include <algorithm>

namespace th {

constexpr int kMxEmaxE4M3 = 8, kMxEmaxE2M1 = 2;  // exponent of a format's largest value

// The bits of |v|: as unsigned numbers they are ordered as the values are, infinity and NaN last.
__device__ __forceinline__ uint32_t mx_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// A block's scale byte by its largest magnitude: floor(log2) of that is its exponent field - 127
// (of a subnormal below -126, where the byte is 0 in any case).
__device__ __forceinline__ int mx_scale(uint32_t top, bool e2m1) {
  return top >= 0x7f800000u ? 255 : max((int)(top >> 23) - (e2m1 ? kMxEmaxE2M1 : kMxEmaxE4M3), 0);
}

// The conversions below take the scale as a float of which they use the exponent field (0: 2^-127).
__device__ __forceinline__ float mx_scale_operand(int s) { return __uint_as_float((uint32_t)s << 23); }

// The largest e4m3 value of a block: past 464 the conversion gives NaN, so values are held to it
// before. (e2m1's conversion saturates by itself.)
__device__ __forceinline__ float mx_limit(int s) {
  return 448.f * __uint_as_float(s ? (uint32_t)s << 23 : 0x00400000u);
}

// 4 values to 4 e4m3 bytes / 8 values to 8 e2m1 nibbles, to nearest even.
__device__ __forceinline__ uint32_t mx_e4m3x4(const float* v, float scale, float limit) {
  typedef short s2_t __attribute__((ext_vector_type(2)));
  float x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = __builtin_amdgcn_fmed3f(v[i], -limit, limit);
  s2_t w = {0, 0};
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x[0], x[1], scale, false);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x[2], x[3], scale, true);
  return __builtin_bit_cast(uint32_t, w);
}
__device__ __forceinline__ uint32_t mx_e2m1x8(const float* v, float scale) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
  return w;
}

// The maximum over the four lanes of a quad (lane ids 4 q .. 4 q + 3).
__device__ __forceinline__ uint32_t mx_quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true));  // lanes 1 0 3 2
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true));  // lanes 2 3 0 1
}

// One lane's 8 of a quad's 32 values into the row's codes and scales: chunk c of the row (the
// lanes of a quad have the chunks 4 b .. 4 b + 3 of block b and all take part).
__device__ __forceinline__ void mx_put8(float (&v)[8], bool e2m1, uint8_t* codes, uint8_t* scales, int c, bool live) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, mx_bits(v[i]));
  top = mx_quad_max(top);
  const int s = mx_scale(top, e2m1);
  const float scale = mx_scale_operand(s == 255 ? 127 : s);
  if (s == 255) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
  }
  if (!live) return;
  if ((c & 3) == 0) scales[c >> 2] = (uint8_t)s;
  if (e2m1) {
    *(uint32_t*)(codes + 4 * (int64_t)c) = mx_e2m1x8(v, scale);
  } else {
    const float limit = mx_limit(s == 255 ? 127 : s);
    *(uint2*)(codes + 8 * (int64_t)c) = make_uint2(mx_e4m3x4(v, scale, limit), mx_e4m3x4(v + 4, scale, limit));
  }
}

// 16 and 8 bytes at any address of whole elements: gfx950 loads and stores them in one instruction (for rows of 4096
// that lie 4097 apart th_mx_rmsnorm of 16384 took 321 us with an instruction an element, and takes 103).
typedef uint32_t mx_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t mx_u4at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t mx_u4at4 __attribute__((ext_vector_type(4), aligned(4)));
#define TH_GLOBAL __attribute__((address_space(1)))  // whichever pointer a lane chose
__device__ __forceinline__ mx_u4 mx_load16(const uint16_t* p) { return *(const TH_GLOBAL mx_u4at2*)p; }
__device__ __forceinline__ mx_u4 mx_load16(const float* p) { return *(const TH_GLOBAL mx_u4at4*)p; }
__device__ __forceinline__ void mx_store16(uint16_t* p, mx_u4 v) { *(TH_GLOBAL mx_u4at2*)p = v; }
__device__ __forceinline__ void mx_store16(float* p, mx_u4 v) { *(TH_GLOBAL mx_u4at4*)p = v; }
__device__ __forceinline__ uint2 mx_load8b(const uint16_t* p) {
  typedef uint32_t u2 __attribute__((ext_vector_type(2), aligned(2)));
  const u2 v = *(const TH_GLOBAL u2*)p;
  return make_uint2(v[0], v[1]);
}
__device__ __forceinline__ void mx_store8b(uint16_t* p, uint2 v) {
  typedef uint32_t u2 __attribute__((ext_vector_type(2), aligned(2)));
  *(TH_GLOBAL u2*)p = u2{v.x, v.y};
}
#undef TH_GLOBAL

// ------------------------------------------------------------ host side
// The bytes that a tensor of rows stands for (none without a pointer).
struct MxSpan {
  const void* p;
  int64_t rows, stride, width;  // bytes; a stride is no less than the width
};

// Whether two tensors share a byte. Rows of one may lie between those of the other.
inline bool mx_meet(const MxSpan& a, const MxSpan& b) {
  typedef __int128 wide;  // (strides are the caller's: their products may pass 64 bits)
  if (!a.p || !b.p || a.rows <= 0 || b.rows <= 0) return false;
  const wide at = (wide)(uintptr_t)b.p - (wide)(uintptr_t)a.p;  // of b's first row, from a's
  const wide sa = a.rows > 1 ? a.stride : a.width, sb = b.rows > 1 ? b.stride : b.width;
  if (at >= (a.rows - 1) * sa + a.width || -at >= (b.rows - 1) * sb + b.width) return false;
  auto down = [](wide x, wide y) { return x >= 0 ? x / y : -((y - 1 - x) / y); };  // floor
  // Rows i of a and j of b meet where -b.width < at + j sb - i sa < a.width.
  if (sa == sb)  // by i - j
    return std::max<wide>(down(at - a.width, sa) + 1, 1 - b.rows) <= std::min<wide>(-down(-(at + b.width), sa) - 1, a.rows - 1);
  if (a.rows > b.rows) return mx_meet(b, a);
  const wide first = std::max<wide>(0, down(at - a.width, sa) + 1);
  const wide last = std::min<wide>(a.rows - 1, -down(-(at + (b.rows - 1) * sb + b.width), sa) - 1);
  for (wide i = first; i <= last; ++i)
    if (std::max<wide>(0, down(i * sa - at - b.width, sb) + 1) <= std::min<wide>(b.rows - 1, -down(-(i * sa - at + a.width), sb) - 1))
      return true;
  return false;
}

// The same memory altogether, rows at the same places (in place), or none in common.
inline bool mx_same_or_apart(const MxSpan& a, const MxSpan& b) {
  return (a.p == b.p && (a.stride == b.stride || a.rows <= 1)) || !mx_meet(a, b);
}

}  // namespace th
