// kv4.cuh — the paged cache in 4 bits: where a page holds what, and the conversions.
//
// Sixteen neighbouring values of a head share a scale byte: five bits of exponent and three of mantissa, the upper byte of a half without its
// sign (value = the half with bits b << 7; no scale per tensor is needed for values from 4.6e-5 to 61440).  A value is a code of four bits,
// sign, two of exponent, one of mantissa: 0, .5, 1, 1.5, 2, 3, 4, 6 times the scale; codes times scales have six bits and are exact in bf16
// and fp16.  A layer is [num_blocks][n_kv] pages of 18 D bytes each: keys' codes (8 D), their scales (D), values' codes, their scales, so
// that a bulk copy of 18 D bytes brings all that one head has of 16 tokens.
//
// Inside its part everything lies as the tensor-core products of single-token attention (kv4_attn.cu) read it.  Lane 4 g + t of a warp:
//   keys    rows of a 16 x 16 tile are tokens: row r = 2 t + (j & 1) + 8 (j >> 1) is token t + 4 j (t, j = 0 .. 3).  A row's D / 2 bytes are
//           cut into four parts (D = 256: twice four), one per t; a lane reads 16 bytes of rows g and g + 8 without bank conflicts.
//   values  rows are tokens, D / 2 bytes each, cut into eight parts, one per g; a lane reads those of tokens t, t + 4, t + 8, t + 12.
//   scales  in the order in which lanes use them: one load of D / 32 bytes per lane for the keys', D = 64, 128: four, D = 256: eight for the values'.
// kv4_key_code and the functions behind it say the same as byte offsets.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace b200q {

template <int D>
struct Kv4 {
  static constexpr int KS = 8 * D, V = 9 * D, VS = 17 * D, BYTES = 18 * D;  // offsets inside a head's page, its size
};

// bytes inside a head's page.  `piece`: where the codes of values 16 p .. 16 p + 15 of a token begin (8 bytes)
template <int D>
__device__ __forceinline__ int kv4_key_row(int token) {
  const int t = token & 3, j = token >> 2;
  return 2 * t + (j & 1) + 8 * (j >> 1);
}
template <int D>
__device__ __forceinline__ int kv4_key_code(int row, int p) {
  if constexpr (D == 256) return row * 128 + (((p >> 1) ^ ((row & 1) * 4)) << 4) + (p & 1) * 8;
  return row * (D / 2) + p * 8;
}
template <int D>
__device__ __forceinline__ int kv4_key_scale(int row, int p) {
  const int lane = (row & 7) * 4, deep = row >> 3;
  if constexpr (D == 64) return Kv4<D>::KS + (lane + p) * 2 + deep;
  if constexpr (D == 128) return Kv4<D>::KS + (lane + (p >> 1)) * 4 + deep * 2 + (p & 1);
  return Kv4<D>::KS + (lane + ((p & 7) >> 1)) * 8 + deep * 4 + (p >> 3) * 2 + (p & 1);
}
template <int D>
__device__ __forceinline__ int kv4_value_code(int token, int p) {
  if constexpr (D == 256) return Kv4<D>::V + token * 128 + (((p >> 1) ^ ((token & 3) * 2)) << 4) + (p & 1) * 8;
  if constexpr (D == 128) return Kv4<D>::V + token * 64 + ((p ^ (((token >> 1) & 1) * 4)) << 3);
  return Kv4<D>::V + token * 32 + p * 8;
}
template <int D>
__device__ __forceinline__ int kv4_value_scale(int token, int p) {
  const int t = token & 3, j = token >> 2;
  if constexpr (D == 256) return Kv4<D>::VS + ((p >> 1) * 4 + t) * 8 + (p & 1) * 4 + j;
  return Kv4<D>::VS + (p * 4 + t) * 4 + j;
}

// four bytes of codes as eight halves in pairs: values 2 i and 2 i + 1 (lower and upper half) of byte i
__device__ __forceinline__ void kv4_halves(uint32_t codes, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
}
__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// bytes `lo` and `hi` of w as a pair of scales
template <int lo, int hi>
__device__ __forceinline__ uint32_t kv4_scales(uint32_t w) {
  return __byte_perm(w, 0, 0x4040 | lo | (hi << 8)) << 7;
}

// The scale byte of a group by its largest magnitude: a sixth of it, to nearest (even), from 2^-17 to 10240.  Rounded twice, but a 16-bit
// float's sixth in fp32 lies on a border only if it does exactly: borders times 6 have seven bits.
__device__ __forceinline__ uint32_t kv4_scale_of(float most, bool nan) {
  const float want = fminf(__fdiv_rn(most, 6.f), 10240.f);
  const uint32_t u = __float_as_uint(want);
  const uint32_t normal = ((u + 0x7ffffu + ((u >> 20) & 1u)) >> 20) - ((127u - 15u) << 3);
  const uint32_t small = (uint32_t)max(__float2int_rn(want * 131072.f), 1);
  return nan ? 0xffu : want < 6.103515625e-5f ? small : normal;
}
__device__ __forceinline__ float kv4_scale_value(uint32_t b) { return __half2float(__ushort_as_half((unsigned short)(b << 7))); }

// Sixteen bf16 values to their codes and scale byte.  Quotients that are not on a border between two codes are 2^-11 and more away from it
// (both have few bits): to multiples of 2^-13 they fall onto it exactly where they are on it, whatever the reciprocal rounds.
__device__ __forceinline__ uint2 kv4_quantise(const uint4& x0, const uint4& x1, uint32_t& scale) {
  const uint32_t x[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(most) : "r"(x[i] & 0x7fff7fffu));
  const float lo = bf16_lo(most), hi = bf16_hi(most);
  const bool nan = lo != lo || hi != hi;
  scale = kv4_scale_of(fmaxf(lo, hi), nan);
  const float r = __frcp_rn(kv4_scale_value(nan ? 1u : scale));
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float y[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t v = x[4 * i + k / 2];
      const float f = k & 1 ? bf16_hi(v) : bf16_lo(v);
      y[k] = copysignf(__fsub_rn(__fadd_rn(__fmul_rn(fabsf(f), r), 1536.f), 1536.f), f);  // (a zero keeps its sign)
    }
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(w[i])
        : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
  }
  return make_uint2(w[0], w[1]);
}

}  // namespace b200q
