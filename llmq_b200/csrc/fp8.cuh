// fp8.cuh — values in 8 bits with a scale for each block of 128 (fp8_ops.cu, gemm_fp8.cu).
//
// A value is an e4m3 code times an fp32 scale, a 448th of the largest magnitude of its block: of 128 neighbours of a row of activations, of a
// square of 128 x 128 weights.  Codes are rounded to nearest (even).  Maxima hand NaN on, so that a block with a NaN has a NaN for its scale and
// reads back as NaN throughout; so does one with an infinity, whose scale is infinite.  Blocks whose magnitudes are all below 2^-100 (zeros, say)
// have the scale of one of 2^-100, so that a scale's reciprocal is finite.
#pragma once
#include "layered_common.cuh"

namespace b200q {

constexpr int FP8_BLOCK = 128;
constexpr int FP8_MOST = 2147483647 - 1023;  // rows, columns, lengths at most: rounded up to whole tiles they are still 32-bit numbers

__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// (the product with 1 / 448, itself off by 0.38 x 2^-23, is off by 0.88 x 2^-23 of the quotient at most)
__device__ __forceinline__ float fp8_scale(float largest) { return max_or_nan(largest, 7.888609052210118e-31f) * (1.f / 448.f); }
__device__ __forceinline__ float fp8_inverse(float scale) {  // (2^-109 <= scale < 2^120, infinite or NaN; off by 2^-23)
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(scale));
  return r;
}
// four codes, the first in the lowest byte
__device__ __forceinline__ uint32_t fp8_four(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n\t"
      ".reg .b16 lo, hi;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
      "mov.b32 %0, {lo, hi};\n\t"
      "}\n"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
// the largest over eight neighbouring lanes
__device__ __forceinline__ float max_of_8_lanes(float m) {
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) m = max_or_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

// eight values of a row of bf16 or fp32
template <typename T>
struct Eight;
template <>
struct Eight<bf16> {
  uint32_t w[4];
  __device__ __forceinline__ void load(const bf16* p) {
    const uint4 v = ld_once_v4(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  }
  __device__ __forceinline__ void zero() { w[0] = w[1] = w[2] = w[3] = 0u; }
  __device__ __forceinline__ void store(bf16* p) const { st_v4(p, make_uint4(w[0], w[1], w[2], w[3])); }
  __device__ __forceinline__ float get(int i) const { return i & 1 ? bf16_hi(w[i >> 1]) : bf16_lo(w[i >> 1]); }
  // (one rounding; a fp32 sum rounded to bf16 is the same: where it is not exact the smaller number is below 2^-16 of the other, far from any tie)
  __device__ __forceinline__ void add(const Eight& o) {
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("add.rn.bf16x2 %0, %0, %1;" : "+r"(w[i]) : "r"(o.w[i]));
  }
  // magnitudes are compared as whole numbers, two at once
  __device__ __forceinline__ float largest() const {
    uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
    for (int i = 1; i < 4; ++i) asm("max.u16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i] & 0x7fff7fffu));
    return __uint_as_float(max(m & 0xffff0000u, m << 16));
  }
};
template <>
struct Eight<float> {
  float w[8];
  __device__ __forceinline__ void load(const float* p) {
    const uint4 v = ld_once_v4(p), u = ld_once_v4(p + 4);
    w[0] = __uint_as_float(v.x); w[1] = __uint_as_float(v.y); w[2] = __uint_as_float(v.z); w[3] = __uint_as_float(v.w);
    w[4] = __uint_as_float(u.x); w[5] = __uint_as_float(u.y); w[6] = __uint_as_float(u.z); w[7] = __uint_as_float(u.w);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 0.f;
  }
  __device__ __forceinline__ void store(float* p) const {
    *reinterpret_cast<float4*>(p) = make_float4(w[0], w[1], w[2], w[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(w[4], w[5], w[6], w[7]);
  }
  __device__ __forceinline__ float get(int i) const { return w[i]; }
  __device__ __forceinline__ void add(const Eight& o) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] += o.w[i];
  }
  __device__ __forceinline__ float largest() const {
    float m = fabsf(w[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) m = max_or_nan(m, fabsf(w[i]));
    return m;
  }
};
template <typename T>
__device__ __forceinline__ uint2 fp8_eight(const Eight<T>& v, float by) {
  return make_uint2(fp8_four(v.get(0) * by, v.get(1) * by, v.get(2) * by, v.get(3) * by),
                    fp8_four(v.get(4) * by, v.get(5) * by, v.get(6) * by, v.get(7) * by));
}

}  // namespace b200q
