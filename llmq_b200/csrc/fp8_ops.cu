// fp8_ops.cu — rows and weights in 8 bits (format: fp8.cuh): RMS norm with the residual's addition, rows as they are or gathered, weights.
// All three are bound by memory: every value is read once and leaves as one byte; what they compute between is some ten instructions a value.
#include "fp8.cuh"

namespace b200q {

constexpr int F8_MAX_H = 16384;

// r <- x + r;  y = r / sqrt(mean(r^2) + eps) * w in 8 bits.  A block to a row, CH pieces of eight values to a thread, held in registers between
// the sum and the product; sixteen lanes are a block of 128 values, whose largest magnitude crosses them in four exchanges.
template <typename T, int CH>
__global__ void __launch_bounds__(256)
    rmsnorm_fp8_kernel(const T* __restrict__ x, T* __restrict__ residual, const T* __restrict__ w, uint2* __restrict__ y,
                       float* __restrict__ scales, int ld_scales, int H, float inv_h, float eps) {
  follow_previous(x, residual, w, y, scales);
  const long long row = blockIdx.x;
  const int threads = blockDim.x, chunks = H / 8;
  Eight<T> v[CH], weight[CH];
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    const int c = threadIdx.x + j * threads;
    if (c < chunks) v[j].load(x + row * H + c * 8);
  }
  if (residual) {
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int c = threadIdx.x + j * threads;
      if (c < chunks) weight[j].load(residual + row * H + c * 8);
    }
  }
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    const int c = threadIdx.x + j * threads;
    if (c < chunks) {
      float f[8];
      v[j].get(f);
      if (residual) {
        float r[8];
        weight[j].get(r);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] += r[i];
        v[j].set(f);  // (the residual stream is held in its own type: the sum is rounded before it is normalised)
        v[j].store(residual + row * H + c * 8);
        v[j].get(f);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += f[i] * f[i];
      weight[j].load(w + c * 8);
    }
  }
  __shared__ float red[8];
  ss = warp_sum(ss);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
  __syncthreads();
  float total = 0.f;
  for (int i = 0; i < threads / 32; ++i) total += red[i];
  const float inv = rsqrtf(total * inv_h + eps);
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    const int c = threadIdx.x + j * threads;
    if (j * threads >= chunks) break;  // (a whole warp takes part in the exchanges)
    float f[8] = {};
    if (c < chunks) {
      float g[8];
      v[j].get(f);
      weight[j].get(g);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = f[i] * inv * g[i];
    }
    uint32_t m = largest_of(f);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float scale = fp8_scale(m);
    if (c < chunks) {
      y[row * chunks + c] = fp8_eight(f, 1.f / scale);
      if (c % 16 == 0) scales[(long long)(c / 16) * ld_scales + row] = scale;
    }
  }
}

// y[i] = row rows[i] (NULL: i) of x in 8 bits.  Sixteen lanes to a block of 128 values.
template <typename T>
__global__ void __launch_bounds__(256)
    quantize_fp8_kernel(const T* __restrict__ x, long long ld_x, const int32_t* __restrict__ rows, uint2* __restrict__ y,
                        float* __restrict__ scales, int ld_scales, int K, int blocks, long long total) {
  follow_previous(x, rows, y, scales);
  const long long item = ((long long)blockIdx.x * 256 + threadIdx.x) >> 4;
  const int at = (threadIdx.x & 15) * 8;
  const long long row = item / blocks;
  const int block = (int)(item - row * blocks), k = block * FP8_BLOCK + at;
  const bool live = item < total && k < K;
  Eight<T> v;
  v.zero();
  if (live) v.load(x + (rows ? (long long)rows[row] : row) * ld_x + k);
  float f[8];
  v.get(f);
  uint32_t m = largest_of(f);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float scale = fp8_scale(m);
  if (live) {
    y[(row * K + k) >> 3] = fp8_eight(f, 1.f / scale);
    if (at == 0) scales[(long long)block * ld_scales + row] = scale;
  }
}

// A square of 128 x 128 weights to a block: eight rows x eight columns to a thread, held in registers between the largest and the codes.
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
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float f[8];
    v[i].get(f);
    m = max(m, largest_of(f));
  }
  m = __reduce_max_sync(0xffffffffu, m);
  __shared__ uint32_t red[8];
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, red[i]);
  const float scale = fp8_scale(m), by = 1.f / scale;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (k < K && n0 + 16 * i < N) {
      float f[8];
      v[i].get(f);
      q[((first + n0 + 16 * i) * K + k) >> 3] = fp8_eight(f, by);
    }
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
  const int chunks = H / 8, threads = chunks < 256 ? (chunks + 31) / 32 * 32 : 256, each = (chunks + threads - 1) / threads;
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
           : each <= 4 ? launch(type, std::integral_constant<int, 4>{})
                       : launch(type, std::integral_constant<int, 8>{});
  };
  return dtype == B200Q_DTYPE_F32 ? pieces(float{}) : pieces(bf16{});
}

int b200q_quantize_fp8(const void* x, int64_t ld_x, const int32_t* rows, void* y, float* scales, int ld_scales, int T_, int K, int dtype,
                       void* stream) {
  B200Q_CHECK_ARG(T_ >= 0 && K > 0 && K % 16 == 0 && is_dtype(dtype), "quantize_fp8: bad shape T=%d K=%d or dtype=%d", T_, K, dtype);
  B200Q_CHECK_ARG(ld_scales >= T_ && ld_x >= K && ld_x % 8 == 0, "quantize_fp8: ld_scales=%d or ld_x=%lld does not fit", ld_scales, (long long)ld_x);
  if (T_ == 0) return B200Q_OK;
  B200Q_CHECK_ARG(x && y && scales, "quantize_fp8: null argument");
  B200Q_CHECK_ARG(aligned16(x, y), "quantize_fp8: x and y must be 16-byte aligned");
  const int blocks = (K + FP8_BLOCK - 1) / FP8_BLOCK;
  const long long total = (long long)T_ * blocks, grid = (total + 15) / 16;
  B200Q_CHECK_ARG(grid < (1ll << 31), "quantize_fp8: too much at once (T=%d K=%d)", T_, K);
  auto launch = [&](auto type) -> int {
    using T = decltype(type);
    B200Q_CUDA(launch_early(quantize_fp8_kernel<T>, dim3((unsigned)grid), 256, 0, as_stream(stream), 1, (const T*)x, (long long)ld_x, rows, (uint2*)y, scales,
                            ld_scales, K, blocks, total));
    count_launch();
    return B200Q_OK;
  };
  return dtype == B200Q_DTYPE_F32 ? launch(float{}) : launch(bf16{});
}

int b200q_quantize_fp8_weight(const void* w, void* q, float* scales, int groups, int N, int K, int dtype, void* stream) {
  B200Q_CHECK_ARG(groups >= 0 && groups <= 65535 && N > 0 && K > 0 && K % 16 == 0 && is_dtype(dtype) && (N + 127) / 128 <= 65535,
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
