// fp8_ops.cu — rows and weights in 8 bits (format: fp8.cuh): RMS norm with the residual's addition, rows as they are or gathered, weights.
// All three are bound by memory: every value is read once and leaves as one byte.  Next to that bound are their instructions, so that eight lanes
// have a block of 128 (two pieces of eight values each: three exchanges for the largest), and pairs of bf16 are added and compared at once.  (The
// norm's factor is multiplied in on its own: its product with a scale's reciprocal, up to 2^109, can pass fp32's range where a row is next to zero,
// and 0 times that is no zero.  4608 x 4096 24.2 us for 24.0.)
#include "fp8.cuh"

namespace b200q {

constexpr int F8_MAX_H = 16384;

// r <- x + r;  y = r / sqrt(mean(r^2) + eps) * w in 8 bits.  A CTA to a row, CH blocks of 128 values to eight lanes, held in registers between the
// sum of squares and the products with w, whose largest magnitude is known before the norm's factor is.
template <typename T, int CH>
__global__ void __launch_bounds__(256)
    rmsnorm_fp8_kernel(const T* __restrict__ x, T* __restrict__ residual, const T* __restrict__ w, uint2* __restrict__ y,
                       float* __restrict__ scales, int ld_scales, int H, float inv_h, float eps) {
  follow_previous(x, residual, w, y, scales);
  const long long row = blockIdx.x;
  const int groups = blockDim.x / 8, lane = threadIdx.x & 7;
  auto place = [&](int j, int p) { return (j * groups + (int)(threadIdx.x >> 3)) * FP8_BLOCK + p * 64 + lane * 8; };
  Eight<T> v[CH][2], u[CH][2];
#pragma unroll
  for (int j = 0; j < CH; ++j)
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      v[j][p].zero();
      u[j][p].zero();
      if (place(j, p) < H) {
        v[j][p].load(x + row * H + place(j, p));
        if (residual) u[j][p].load(residual + row * H + place(j, p));
      }
    }
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < CH; ++j)
#pragma unroll
    for (int p = 0; p < 2; ++p)
      if (place(j, p) < H) {
        if (residual) {  // (the residual stream is held in its own type: the sum is rounded before it is normalised)
          v[j][p].add(u[j][p]);
          v[j][p].store(residual + row * H + place(j, p));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += v[j][p].get(i) * v[j][p].get(i);
        u[j][p].load(w + place(j, p));
      }
  __shared__ float red[8];
  ss = warp_sum(ss);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
  __syncthreads();
  float total = 0.f;
  for (int i = 0; i < (int)blockDim.x / 32; ++i) total += red[i];
  const float inv = rsqrtf(total * inv_h + eps);
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    Eight<float> n[2];
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int i = 0; i < 8; ++i) n[p].w[i] = v[j][p].get(i) * inv * u[j][p].get(i);
    const float scale = fp8_scale(max_of_8_lanes(max_or_nan(n[0].largest(), n[1].largest()))), by = fp8_inverse(scale);
#pragma unroll
    for (int p = 0; p < 2; ++p)
      if (place(j, p) < H) y[(row * H + place(j, p)) >> 3] = fp8_eight(n[p], by);
    if (lane == 0 && place(j, 0) < H) scales[(long long)(place(j, 0) / FP8_BLOCK) * ld_scales + row] = scale;
  }
}

// y[i] = row rows[i] (NULL: i) of x in 8 bits.  Eight lanes to a block of 128 values, and no more than one block: many short CTAs keep more reads
// under way than longer ones (one measurement: 4608 x 4096 10.3 us, two blocks 11.8, four 12.3; 4004 gathered rows of 2048 4.7 / 5.9 / 5.9.  Others, inputs
// from HBM: 10.5 to 10.8 and 5.2 to 5.3).
template <typename T>
__global__ void __launch_bounds__(256)
    quantize_fp8_kernel(const T* __restrict__ x, long long ld_x, const int32_t* __restrict__ rows, uint2* __restrict__ y,
                        float* __restrict__ scales, int ld_scales, int K, uint32_t blocks, uint32_t by_blocks, int shift, uint32_t total) {
  follow_previous(x, rows, y, scales);
  // item / blocks (by_blocks: 2^shift / blocks and less than 2^(shift - 31) more, so exact for items below 2^31)
  const uint32_t item = blockIdx.x * 32 + (threadIdx.x >> 3), row = (uint32_t)((uint64_t)item * by_blocks >> shift), block = item - row * blocks;
  const int lane = threadIdx.x & 7, k = (int)block * FP8_BLOCK + lane * 8;
  const bool live = item < total;
  const T* from = x + (live ? (rows ? (long long)rows[row] : (long long)row) : 0ll) * ld_x + k;
  Eight<T> v[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    v[p].zero();
    if (live && k + p * 64 < K) v[p].load(from + p * 64);
  }
  const float scale = fp8_scale(max_of_8_lanes(max_or_nan(v[0].largest(), v[1].largest()))), by = fp8_inverse(scale);
#pragma unroll
  for (int p = 0; p < 2; ++p)
    if (live && k + p * 64 < K) y[((long long)row * K + k + p * 64) >> 3] = fp8_eight(v[p], by);
  if (live && lane == 0) scales[(long long)block * ld_scales + row] = scale;
}

// A square of 128 x 128 weights to a CTA: eight rows x eight columns to a thread, held in registers between the largest and the codes.
template <typename T>
__global__ void __launch_bounds__(256)
    quantize_fp8_weight_kernel(const T* __restrict__ w, uint2* __restrict__ q, float* __restrict__ scales, int N, int K) {
  follow_previous(w, q, scales);
  const int k = blockIdx.x * FP8_BLOCK + (threadIdx.x & 15) * 8, n0 = blockIdx.y * FP8_BLOCK + (threadIdx.x >> 4);
  const long long first = (long long)blockIdx.z * N;
  Eight<T> v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i].zero();
    if (k < K && n0 + 16 * i < N) v[i].load(w + (first + n0 + 16 * i) * K + k);
  }
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max_or_nan(m, v[i].largest());
  const uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(m));  // (no sign: NaN is the largest as a whole number too)
  __shared__ uint32_t red[8];
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = most;
  __syncthreads();
  uint32_t all = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) all = max(all, red[i]);
  const float scale = fp8_scale(__uint_as_float(all)), by = fp8_inverse(scale);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (k < K && n0 + 16 * i < N) q[((first + n0 + 16 * i) * K + k) >> 3] = fp8_eight(v[i], by);
  if (threadIdx.x == 0) scales[((long long)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x] = scale;
}

static bool aligned16(const void* a, const void* b = nullptr, const void* c = nullptr, const void* d = nullptr) {
  return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c) | reinterpret_cast<uintptr_t>(d)) & 15) == 0;
}

}  // namespace b200q

using namespace b200q;

extern "C" {

int b200q_rmsnorm_fp8(const void* x, void* residual, const void* w, void* y, float* scales, int ld_scales, int T_, int H, float eps, int dtype,
                      void* stream) {
  B200Q_CHECK_ARG(T_ >= 0 && H > 0 && H % 16 == 0 && H <= F8_MAX_H && is_dtype(dtype), "rmsnorm_fp8: bad shape T=%d H=%d or dtype=%d", T_, H, dtype);
  B200Q_CHECK_ARG(ld_scales >= T_, "rmsnorm_fp8: ld_scales=%d is less than T=%d", ld_scales, T_);
  if (T_ == 0) return B200Q_OK;
  B200Q_CHECK_ARG(x && w && y && scales, "rmsnorm_fp8: null argument");
  B200Q_CHECK_ARG(aligned16(x, residual, w, y), "rmsnorm_fp8: x, residual, w and y must be 16-byte aligned");
  const int blocks = (H + FP8_BLOCK - 1) / FP8_BLOCK, threads = blocks < 32 ? (blocks * 8 + 31) / 32 * 32 : 256, each = (blocks + threads / 8 - 1) / (threads / 8);
  auto launch = [&](auto type, auto ch) -> int {
    using T = decltype(type);
    B200Q_CUDA(launch_early(rmsnorm_fp8_kernel<T, decltype(ch)::value>, T_, threads, 0, as_stream(stream), 1, (const T*)x, (T*)residual, (const T*)w,
                            (uint2*)y, scales, ld_scales, H, 1.f / (float)H, eps));
    count_launch();
    return B200Q_OK;
  };
  auto pieces = [&](auto type) -> int {
    return each <= 1   ? launch(type, std::integral_constant<int, 1>{})
           : each <= 2 ? launch(type, std::integral_constant<int, 2>{})
                       : launch(type, std::integral_constant<int, 4>{});
  };
  return dtype == B200Q_DTYPE_F32 ? pieces(float{}) : pieces(bf16{});
}

int b200q_quantize_fp8(const void* x, int64_t ld_x, const int32_t* rows, void* y, float* scales, int ld_scales, int T_, int K, int dtype,
                       void* stream) {
  B200Q_CHECK_ARG(T_ >= 0 && K > 0 && K <= FP8_MOST && K % 16 == 0 && is_dtype(dtype), "quantize_fp8: bad shape T=%d K=%d or dtype=%d", T_, K, dtype);
  B200Q_CHECK_ARG(ld_scales >= T_ && ld_x >= K && ld_x % 8 == 0, "quantize_fp8: ld_scales=%d or ld_x=%lld does not fit", ld_scales, (long long)ld_x);
  if (T_ == 0) return B200Q_OK;
  B200Q_CHECK_ARG(x && y && scales, "quantize_fp8: null argument");
  B200Q_CHECK_ARG(aligned16(x, y), "quantize_fp8: x and y must be 16-byte aligned");
  const int blocks = (K + FP8_BLOCK - 1) / FP8_BLOCK;
  const long long total = (long long)T_ * blocks;
  B200Q_CHECK_ARG(total < (1ll << 31), "quantize_fp8: too much at once (T=%d K=%d)", T_, K);
  int up = 0;  // 2^up >= blocks
  while ((1 << up) < blocks) ++up;
  const uint32_t by_blocks = (uint32_t)((1ull << (31 + up)) / (uint32_t)blocks + 1);
  auto launch = [&](auto type) -> int {
    using T = decltype(type);
    B200Q_CUDA(launch_early(quantize_fp8_kernel<T>, dim3((unsigned)((total + 31) / 32)), 256, 0, as_stream(stream), 1, (const T*)x, (long long)ld_x, rows,
                            (uint2*)y, scales, ld_scales, K, (uint32_t)blocks, by_blocks, 31 + up, (uint32_t)total));
    count_launch();
    return B200Q_OK;
  };
  return dtype == B200Q_DTYPE_F32 ? launch(float{}) : launch(bf16{});
}

int b200q_quantize_fp8_weight(const void* w, void* q, float* scales, int groups, int N, int K, int dtype, void* stream) {
  B200Q_CHECK_ARG(groups >= 0 && groups <= 65535 && N > 0 && N <= 65535 * 128 && K > 0 && K <= FP8_MOST && K % 16 == 0 && is_dtype(dtype),
                  "quantize_fp8_weight: bad shape groups=%d N=%d K=%d or dtype=%d", groups, N, K, dtype);
  if (groups == 0) return B200Q_OK;
  B200Q_CHECK_ARG(w && q && scales, "quantize_fp8_weight: null argument");
  B200Q_CHECK_ARG(aligned16(w, q), "quantize_fp8_weight: w and q must be 16-byte aligned");
  auto launch = [&](auto type) -> int {
    using T = decltype(type);
    B200Q_CUDA(launch_early(quantize_fp8_weight_kernel<T>, dim3((K + 127) / 128, (N + 127) / 128, groups), 256, 0, as_stream(stream), 1, (const T*)w,
                            (uint2*)q, scales, N, K));
    count_launch();
    return B200Q_OK;
  };
  return dtype == B200Q_DTYPE_F32 ? launch(float{}) : launch(bf16{});
}

}  // extern "C"
