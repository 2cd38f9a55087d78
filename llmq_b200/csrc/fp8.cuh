// fp8.cuh — values in 8 bits with a scale for each block of 128 (fp8_ops.cu, gemm_fp8.cu).
//
// A value is an e4m3 code times an fp32 scale, a 448th of the largest magnitude of its block: of 128 neighbours of a row of activations, of a
// square of 128 x 128 weights.  Codes are rounded to nearest (even).  Magnitudes are compared as bits, so that a NaN is the largest: its block's
// scale, and with it all of the block, is NaN.  A block with an infinity has an infinite scale and reads back as NaN throughout.  Blocks whose
// magnitudes are all below 2^-100 (zeros, say) have the scale of one of 2^-100, so that a scale's reciprocal is finite.
#pragma once
#include "layered_common.cuh"

namespace b200q {

constexpr int FP8_BLOCK = 128;

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ float fp8_scale(uint32_t largest) { return __uint_as_float(max(largest, 0x0d800000u)) / 448.f; }  // 0x0d800000: 2^-100
// two codes, the first in the lower byte
__device__ __forceinline__ uint32_t fp8_pair(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t fp8_four(float a, float b, float c, float d) { return fp8_pair(a, b) | fp8_pair(c, d) << 16; }

// eight values of a row of bf16 or fp32
template <typename T>
struct Eight;
template <>
struct Eight<bf16> {
  uint4 v;
  __device__ __forceinline__ void load(const bf16* p) { v = ld_once_v4(p); }
  __device__ __forceinline__ void zero() { v = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = bf16_lo(w[i]);
      f[2 * i + 1] = bf16_hi(w[i]);
    }
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    v = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
  __device__ __forceinline__ void store(bf16* p) const { st_v4(p, v); }
};
template <>
struct Eight<float> {
  uint4 v, u;
  __device__ __forceinline__ void load(const float* p) {
    v = ld_once_v4(p);
    u = ld_once_v4(p + 4);
  }
  __device__ __forceinline__ void zero() { v = u = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t w[8] = {v.x, v.y, v.z, v.w, u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    v = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    u = make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7]));
  }
  __device__ __forceinline__ void store(float* p) const {
    st_v4(p, v);
    st_v4(p + 4, u);
  }
};
__device__ __forceinline__ uint32_t largest_of(const float (&f)[8]) {
  uint32_t m = abs_bits(f[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = max(m, abs_bits(f[i]));
  return m;
}
__device__ __forceinline__ uint2 fp8_eight(const float (&f)[8], float by) {
  return make_uint2(fp8_four(f[0] * by, f[1] * by, f[2] * by, f[3] * by), fp8_four(f[4] * by, f[5] * by, f[6] * by, f[7] * by));
}

}  // namespace b200q
