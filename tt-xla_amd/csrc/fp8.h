// The 8-bit cache with a scale for each block of tokens and head: shared device pieces.
//
// An element is e4m3 (OCP, largest value 448, no infinity) and stands for itself times its block's scale of that head, a
// power of two.  A floating-point element keeps its three mantissa bits whatever the scale's mantissa would be, so a
// power of two costs nothing but a share of a binade of the element's range; and it makes every step exact but the one
// rounding to e4m3: scaling in, scaling out (the product is a bfloat16 value), and a change of a block's scale for
// all elements but those that fall among the subnormals.
//
// The scale of values with the largest magnitude `most` is the smallest power of two with most <= 448 scale, its exponent
// kept in [-110, 119], where every value of an element is a normal bfloat16 number; 448 * 2^119 is what larger values
// become.  NaN and infinities become NaN and have no part in the scale.
#pragma once

#include "common.h"

namespace ttpa {
namespace fp8 {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// The magnitude that counts for a scale, of two packed bfloat16 values: bits as whole numbers, 0 for NaN and infinities.
__device__ __forceinline__ uint32_t finite_magnitude(uint32_t pair) {
  const uint32_t lo = pair & 0x7fffu, hi = (pair >> 16) & 0x7fffu;
  return max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u);
}
// The scale for bfloat16 values of at most this magnitude (its bits): 448 = 1.75 * 2^8.
__device__ __forceinline__ float scale_for(uint32_t most_bits) {
  const int e = (int)(most_bits >> 7) - (127 + 8) + ((most_bits & 0x7fu) > 0x60u ? 1 : 0);
  return __builtin_bit_cast(float, (uint32_t)(min(max(e, -110), 119) + 127) << 23);
}
// 1 / scale for a power of two in the range above.
__device__ __forceinline__ float inverse_scale(float scale) {
  return __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(uint32_t, scale));
}
// A value already divided by its scale, brought to e4m3's range: beyond it the largest value; infinities as NaN.
__device__ __forceinline__ float in_range(float x) {
  const float c = __builtin_amdgcn_fmed3f(x, -448.f, 448.f);
  return fabsf(x) < INFINITY ? c : __builtin_bit_cast(float, 0x7fc00000u);
}
// Four values in e4m3's range -> four elements, each rounded to nearest even.
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
// Eight packed bfloat16 values, times `inv`, -> eight elements.
__device__ __forceinline__ u32x2 encode8(const u32x4 &w, float inv) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) f[2 * i] = in_range(bf16_lo(w[i]) * inv), f[2 * i + 1] = in_range(bf16_hi(w[i]) * inv);
  return u32x2{encode4(f[0], f[1], f[2], f[3]), encode4(f[4], f[5], f[6], f[7])};
}
// Four elements times a power of two of at most 1, rounded to e4m3 again.
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float ratio) {
  typedef float float2_t __attribute__((ext_vector_type(2)));
  const float2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return encode4(lo.x * ratio, lo.y * ratio, hi.x * ratio, hi.y * ratio);
}
// Eight elements (two dwords) -> eight bfloat16 values times `scale` (a power of two; exact).
__device__ __forceinline__ u32x4 decode8(uint32_t w0, uint32_t w1, float scale) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, true)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, true))};
}

// The caches of a layer, and where rows go in them.
struct Caches {
  uint8_t *k, *v;            // [num_blocks, kv_heads, block_size, head_size] e4m3
  float *k_scales, *v_scales;  // [num_blocks, kv_heads]
  uint16_t *bounds;          // bfloat16 [num_blocks, kv_heads, 2, head_size]: least and largest key per feature; or null
  const int32_t *pt;
  int64_t pt_rs;
  int hkv, bs, w, nb;
  uint32_t bs_inv;  // floor((2^32 - 1) / bs)
};
inline uint32_t block_inverse(int bs) { return bs > 0 ? 0xffffffffu / (uint32_t)bs : 0u; }

// Column and row of position `pos` of a table row; false: negative or outside the table.  (A table row holds less than 2^31 tokens.)
__device__ __forceinline__ bool place_of(const Caches &c, int64_t pos, int &col, int &row) {
  const uint32_t p = (uint32_t)pos;
  uint32_t q = __umulhi(p, c.bs_inv), r = p - q * (uint32_t)c.bs;  // one too few at most
  if (r >= (uint32_t)c.bs) ++q, r -= (uint32_t)c.bs;
  col = (int)q, row = (int)r;
  return pos >= 0 && pos < (int64_t)c.w * c.bs;
}

}  // namespace fp8
}  // namespace ttpa
