// kv4_ops.cu — writing the 4-bit cache (rotation and quantisation), reading its pages back as 16-bit ones, and prompt attention over it.
// The page's layout and the conversions: kv4.cuh.
#include "kv4.cuh"

namespace b200q {

__device__ __forceinline__ void floats_of(const uint4& v, float* x) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16_lo(w[i]);
    x[2 * i + 1] = bf16_hi(w[i]);
  }
}

// ------------------------------------------------------------------------------------------------------------------------
// Rotation of q and k (pairs i, i + D/2; a bf16 rounding behind every operation, as in elementwise.cu) and the write into 4-bit pages.
// Items of a token: groups of 16 values of k with those they are paired with (two groups), groups of v, 8 + 8 values of q.  A thread has
// its groups whole, so that no maximum crosses threads; rotated keys exist in registers only.
// Bound: the rows' bytes (a cached token is 9/16 of a byte per value, a quarter of what the 16-bit write stores).
// ------------------------------------------------------------------------------------------------------------------------
template <int D>
__global__ void __launch_bounds__(256) rope_kvwrite_q4_kernel(uint4* qkv, const uint4* cos_sin, const int32_t* positions, const int32_t* slot_mapping,
                                                              uint8_t* kv_layer, int n_q, int n_kv) {
  follow_previous(qkv, cos_sin, positions, slot_mapping, kv_layer);
  constexpr int CPR = D / 8, HALF = CPR / 2;  // 16-byte pieces of a head's row, of half of it
  const long long t = blockIdx.x;
  uint4* row = qkv + t * (n_q + 2 * n_kv) * CPR;
  const int slot = slot_mapping[t];
  const uint4* cs_row = cos_sin + (long long)positions[t] * CPR;
  const int token = slot & 15;
  uint8_t* page = kv_layer + (long long)(slot >> 4) * n_kv * Kv4<D>::BYTES;
  const int k_items = slot >= 0 ? n_kv * (D / 32) : 0, v_items = slot >= 0 ? n_kv * (D / 16) : 0;
  const int n_items = k_items + v_items + n_q * HALF;
  auto turn = [](float x1, float x2, float c, float s, float& o1, float& o2) {
    o1 = round_bf16(round_bf16(x1 * c) - round_bf16(x2 * s));
    o2 = round_bf16(round_bf16(x2 * c) + round_bf16(x1 * s));
  };
  for (int it = blockIdx.y * blockDim.x + threadIdx.x; it < n_items; it += gridDim.y * blockDim.x) {
    if (it < k_items) {
      const int h = it / (D / 32), p = it % (D / 32);  // groups p and p + D/32
      const uint4* src = row + (n_q + h) * CPR + 2 * p;
      float a[16], b[16], c[16], s[16];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        floats_of(ld_v4(src + i), a + 8 * i);
        floats_of(ld_v4(src + HALF + i), b + 8 * i);
        floats_of(ld_v4(cs_row + 2 * p + i), c + 8 * i);
        floats_of(ld_v4(cs_row + HALF + 2 * p + i), s + 8 * i);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) turn(a[i], b[i], c[i], s[i], a[i], b[i]);
      uint8_t* to = page + h * Kv4<D>::BYTES;
      const int r = kv4_key_row<D>(token);
      uint32_t scale;
      *reinterpret_cast<uint2*>(to + kv4_key_code<D>(r, p)) = kv4_quantise(a, scale);
      to[kv4_key_scale<D>(r, p)] = (uint8_t)scale;
      *reinterpret_cast<uint2*>(to + kv4_key_code<D>(r, p + D / 32)) = kv4_quantise(b, scale);
      to[kv4_key_scale<D>(r, p + D / 32)] = (uint8_t)scale;
    } else if (it < k_items + v_items) {
      const int h = (it - k_items) / (D / 16), p = (it - k_items) % (D / 16);
      const uint4* src = row + (n_q + n_kv + h) * CPR + 2 * p;
      float a[16];
      floats_of(ld_v4(src), a);
      floats_of(ld_v4(src + 1), a + 8);
      uint8_t* to = page + h * Kv4<D>::BYTES;
      uint32_t scale;
      *reinterpret_cast<uint2*>(to + kv4_value_code<D>(token, p)) = kv4_quantise(a, scale);
      to[kv4_value_scale<D>(token, p)] = (uint8_t)scale;
    } else {
      const int h = (it - k_items - v_items) / HALF, c0 = (it - k_items - v_items) % HALF;
      uint4* at = row + h * CPR + c0;
      float a[8], b[8], c[8], s[8];
      floats_of(ld_v4(at), a);
      floats_of(ld_v4(at + HALF), b);
      floats_of(ld_v4(cs_row + c0), c);
      floats_of(ld_v4(cs_row + HALF + c0), s);
#pragma unroll
      for (int i = 0; i < 8; ++i) turn(a[i], b[i], c[i], s[i], a[i], b[i]);
      st_v4(at, make_uint4(pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]), pack_bf16x2(a[4], a[5]), pack_bf16x2(a[6], a[7])));
      st_v4(at + HALF, make_uint4(pack_bf16x2(b[0], b[1]), pack_bf16x2(b[2], b[3]), pack_bf16x2(b[4], b[5]), pack_bf16x2(b[6], b[7])));
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------------
// 4-bit pages as 16-bit ones (the layout of attn.cu: [2][n_kv][16][D], the 16-byte piece c of a row at c ^ (token & 7)).  Exact.
// ------------------------------------------------------------------------------------------------------------------------
// one head's page by the threads of a warp: an item is 8 values
template <int D>
__device__ __forceinline__ void kv4_spread_head(const uint8_t* head, uint4* keys, uint4* values, int lane) {
  constexpr int CPR = D / 8;
#pragma unroll 4
  for (int it = lane; it < 32 * CPR; it += 32) {
    const int which = it / (16 * CPR), token = it / CPR % 16, c = it % CPR, p = c >> 1;
    const int r = kv4_key_row<D>(token);
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(head + (which ? kv4_value_code<D>(token, p) : kv4_key_code<D>(r, p)) + (c & 1) * 4);
    const uint32_t b = head[which ? kv4_value_scale<D>(token, p) : kv4_key_scale<D>(r, p)];
    uint32_t h[4];
    kv4_halves(codes, h);
    const float s = kv4_scale_value(b);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
      w[i] = pack_bf16x2(f.x * s, f.y * s);
    }
    (which ? values : keys)[token * CPR + (c ^ (token & 7))] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <int D>
__global__ void __launch_bounds__(128) kv4_unpack_kernel(const uint8_t* kv4, const int32_t* pages, int n_pages, uint4* out, int n_kv) {
  follow_previous(kv4, pages, out);
  const long long items = (long long)n_pages * n_kv;
  for (long long it = (long long)blockIdx.x * 4 + (threadIdx.x >> 5); it < items; it += (long long)gridDim.x * 4) {
    const long long i = it / n_kv;
    const int h = (int)(it % n_kv);
    constexpr int ROWS = 16 * D / 8;
    uint4* keys = out + ((i * 2) * n_kv + h) * ROWS;
    kv4_spread_head<D>(kv4 + ((long long)pages[i] * n_kv + h) * Kv4<D>::BYTES, keys, keys + (long long)n_kv * ROWS, threadIdx.x & 31);
  }
}

// The pages that a step's portions see, spread out to a workspace in which column c of row r of the block table is page r * bt_stride + c.
// A block has SPREAD_COLUMNS columns of one row; what a row needs it finds from the tiles (their first visible and their last key).
constexpr int SPREAD_COLUMNS = 4;
template <int D>
__global__ void __launch_bounds__(256) kv4_spread_kernel(const uint8_t* kv4, const int32_t* block_table, int bt_stride, const int4* tiles, int n_tiles,
                                                         int n_kv, int window, uint4* out, int32_t* table) {
  follow_previous(kv4, block_table, tiles, out, table);
  const int row = blockIdx.y, c0 = blockIdx.x * SPREAD_COLUMNS;
  int lo = 0x7fffffff, hi = 0;
  for (int i = threadIdx.x; i < n_tiles; i += blockDim.x) {
    const int4 t = tiles[i];
    if (t.x == row && t.z > 0) {
      lo = min(lo, window > 0 ? max(t.w + 1 - window, 0) : 0);
      hi = max(hi, t.w + min(t.z, 16));
    }
  }
  __shared__ int s_lo, s_hi;
  if (threadIdx.x == 0) {
    s_lo = 0x7fffffff;
    s_hi = 0;
  }
  __syncthreads();
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if ((threadIdx.x & 31) == 0) {
    atomicMin(&s_lo, lo);
    atomicMax(&s_hi, hi);
  }
  __syncthreads();
  // (where a portion follows another of the same row, both are in [lo, hi))
  const int first = max(s_lo / 16, c0), last = min(min((s_hi + 15) / 16, bt_stride), c0 + SPREAD_COLUMNS);
  const int n = (last - first) * n_kv;
  for (int it = threadIdx.x >> 5; it < n; it += 8) {
    const int c = first + it / n_kv, h = it % n_kv;
    const long long to = (long long)row * bt_stride + c;
    constexpr int ROWS = 16 * D / 8;
    uint4* keys = out + ((to * 2) * n_kv + h) * ROWS;
    kv4_spread_head<D>(kv4 + ((long long)block_table[to] * n_kv + h) * Kv4<D>::BYTES, keys, keys + (long long)n_kv * ROWS, threadIdx.x & 31);
    if (h == 0 && (threadIdx.x & 31) == 0) table[to] = (int32_t)to;
  }
}

static inline int64_t spread_pages_bytes(int64_t pages, int n_kv, int D) { return pages * (4LL * n_kv * 16 * D); }

}  // namespace b200q

using namespace b200q;

#define B200Q_KV4_DIMS(what, D, call) \
  do {                                \
    if ((D) == 64) {                  \
      constexpr int kD = 64;          \
      call;                           \
    } else if ((D) == 128) {          \
      constexpr int kD = 128;         \
      call;                           \
    } else {                          \
      constexpr int kD = 256;         \
      call;                           \
    }                                 \
  } while (0)

extern "C" {

int64_t b200q_kv4_page_bytes(int n_kv, int D) {
  if (n_kv <= 0 || (D != 64 && D != 128 && D != 256)) {
    set_error("kv4_page_bytes: unsupported n_kv=%d D=%d (D in {64,128,256})", n_kv, D);
    return B200Q_EINVAL;
  }
  return 18LL * D * n_kv;
}

int b200q_rope_kvwrite_q4(void* qkv, const void* cos_sin, const int32_t* positions, const int32_t* slot_mapping, void* kv4_layer, int T, int n_q,
                          int n_kv, int D, int block_size, void* stream) {
  B200Q_CHECK_ARG(T >= 0 && (D == 64 || D == 128 || D == 256) && n_q >= 0 && n_kv > 0 && block_size == 16,
                  "rope_kvwrite_q4: bad shape T=%d n_q=%d n_kv=%d D=%d bs=%d (D in {64,128,256}, block 16)", T, n_q, n_kv, D, block_size);
  if (T == 0) return B200Q_OK;
  B200Q_CHECK_ARG(qkv && cos_sin && positions && slot_mapping && kv4_layer, "rope_kvwrite_q4: null argument");
  B200Q_CHECK_ARG(((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(cos_sin) | reinterpret_cast<uintptr_t>(kv4_layer)) & 15) == 0,
                  "rope_kvwrite_q4: qkv, cos_sin and the cache must be 16-byte aligned");
  const int items = n_kv * (D / 32) + n_kv * (D / 16) + n_q * (D / 16), blocks = T <= 320 ? (items + 127) / 128 : 1;
  const int threads = blocks > 1 ? 128 : 256;
  B200Q_KV4_DIMS("rope_kvwrite_q4", D,
                 B200Q_CUDA(launch_early(rope_kvwrite_q4_kernel<kD>, dim3(T, blocks), threads, 0, as_stream(stream), 1, (uint4*)qkv,
                                         (const uint4*)cos_sin, positions, slot_mapping, (uint8_t*)kv4_layer, n_q, n_kv)));
  count_launch();
  return B200Q_OK;
}

int b200q_kv4_unpack(const void* kv4_layer, const int32_t* pages, int n_pages, void* kv_out, int n_kv, int D, int block_size, void* stream) {
  B200Q_CHECK_ARG(n_pages >= 0 && n_kv > 0 && (D == 64 || D == 128 || D == 256) && block_size == 16,
                  "kv4_unpack: bad shape n_pages=%d n_kv=%d D=%d bs=%d (D in {64,128,256}, block 16)", n_pages, n_kv, D, block_size);
  if (n_pages == 0) return B200Q_OK;
  B200Q_CHECK_ARG(kv4_layer && pages && kv_out, "kv4_unpack: null argument");
  B200Q_CHECK_ARG(((reinterpret_cast<uintptr_t>(kv4_layer) | reinterpret_cast<uintptr_t>(kv_out)) & 15) == 0, "kv4_unpack: caches must be 16-byte aligned");
  const long long items = (long long)n_pages * n_kv, blocks = (items + 3) / 4;
  B200Q_KV4_DIMS("kv4_unpack", D,
                 B200Q_CUDA(launch_early(kv4_unpack_kernel<kD>, dim3((unsigned)(blocks < 1 << 20 ? blocks : 1 << 20)), 128, 0, as_stream(stream), 1,
                                         (const uint8_t*)kv4_layer, pages, n_pages, (uint4*)kv_out, n_kv)));
  count_launch();
  return B200Q_OK;
}

int64_t b200q_prefill_attn_q4_workspace(int n_seqs, int bt_stride, int n_kv, int D) {
  if (n_seqs < 0 || bt_stride < 0 || n_kv <= 0 || (D != 64 && D != 128 && D != 256)) {
    set_error("prefill_attn_q4_workspace: bad shape n_seqs=%d bt_stride=%d n_kv=%d D=%d", n_seqs, bt_stride, n_kv, D);
    return B200Q_EINVAL;
  }
  const int64_t pages = (int64_t)n_seqs * bt_stride;
  return spread_pages_bytes(pages, n_kv, D) + (pages * 4 + 255) / 256 * 256;
}

int b200q_prefill_attn_q4(const void* q, int q_stride, void* out, const void* kv4_layer, const int32_t* block_table, int bt_stride, int n_seqs,
                          const int32_t* tiles, int n_tiles, int n_q, int n_kv, int D, int block_size, float scale, float softcap, int window,
                          void* workspace, int64_t workspace_bytes, void* stream) {
  B200Q_CHECK_ARG(n_tiles >= 0 && n_kv > 0 && n_q >= n_kv && n_q % n_kv == 0 && n_q / n_kv <= (D == 256 ? 4 : 8),
                  "prefill_attn_q4: unsupported heads n_q=%d n_kv=%d (GQA group <= 8; <= 4 at head_dim 256)", n_q, n_kv);
  B200Q_CHECK_ARG(block_size == 16 && (D == 64 || D == 128 || D == 256), "prefill_attn_q4: unsupported D=%d block_size=%d (D in {64,128,256}, block 16)",
                  D, block_size);
  B200Q_CHECK_ARG(n_seqs >= 0 && n_seqs <= 65535 && bt_stride >= 0 && (int64_t)n_seqs * bt_stride < (1ll << 30),
                  "prefill_attn_q4: bad block table [%d, %d] (up to 65535 rows and 2^30 entries)", n_seqs, bt_stride);
  if (n_tiles == 0 || n_seqs == 0 || bt_stride == 0) return B200Q_OK;
  B200Q_CHECK_ARG(q && out && kv4_layer && block_table && tiles && workspace, "prefill_attn_q4: null argument");
  const int64_t need = b200q_prefill_attn_q4_workspace(n_seqs, bt_stride, n_kv, D);
  B200Q_CHECK_ARG(workspace_bytes >= need, "prefill_attn_q4: workspace too small: %lld < %lld", (long long)workspace_bytes, (long long)need);
  B200Q_CHECK_ARG(((reinterpret_cast<uintptr_t>(workspace) & 255) | (reinterpret_cast<uintptr_t>(kv4_layer) & 15) |
                   (reinterpret_cast<uintptr_t>(tiles) & 15)) == 0,
                  "prefill_attn_q4: the workspace must be 256-byte aligned, cache and tiles 16-byte aligned");
  const int64_t pages = (int64_t)n_seqs * bt_stride;
  int32_t* table = (int32_t*)((uint8_t*)workspace + spread_pages_bytes(pages, n_kv, D));
  B200Q_KV4_DIMS("prefill_attn_q4", D,
                 B200Q_CUDA(launch_early(kv4_spread_kernel<kD>, dim3((bt_stride + SPREAD_COLUMNS - 1) / SPREAD_COLUMNS, n_seqs), 256, 0, as_stream(stream),
                                         1, (const uint8_t*)kv4_layer, block_table, bt_stride, (const int4*)tiles, n_tiles, n_kv, window,
                                         (uint4*)workspace, table)));
  count_launch();
  return b200q_prefill_attn_seqs(q, q_stride, out, workspace, table, bt_stride, n_seqs, tiles, n_tiles, n_q, n_kv, D, block_size, scale, softcap,
                                 window, stream);
}

}  // extern "C"
