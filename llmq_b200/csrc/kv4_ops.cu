// kv4_ops.cu — writing the 4-bit cache (rotation and quantisation), reading its pages back as 16-bit ones, and prompt attention over it.
// The page's layout and the conversions: kv4.cuh.
#include <type_traits>

#include "kv4.cuh"

namespace b200q {

// Two bf16 at once.  A product, a sum or a difference of two bf16 rounded to bf16 once is what fp32 arithmetic and a rounding behind it give
// (products are exact in fp32; sums either are, or their fp32 rounding lies far below bf16's).
__device__ __forceinline__ uint32_t mul_bf2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t add_bf2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t sub_bf2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// x1, x2 <- x1 cos - x2 sin, x2 cos + x1 sin, a rounding behind every operation
__device__ __forceinline__ void turn_bf2(uint32_t& x1, uint32_t& x2, uint32_t c, uint32_t s) {
  const uint32_t o1 = sub_bf2(mul_bf2(x1, c), mul_bf2(x2, s));
  x2 = add_bf2(mul_bf2(x2, c), mul_bf2(x1, s));
  x1 = o1;
}
__device__ __forceinline__ void turn_bf8(uint4& x1, uint4& x2, const uint4& c, const uint4& s) {
  turn_bf2(x1.x, x2.x, c.x, s.x);
  turn_bf2(x1.y, x2.y, c.y, s.y);
  turn_bf2(x1.z, x2.z, c.z, s.z);
  turn_bf2(x1.w, x2.w, c.w, s.w);
}

// ------------------------------------------------------------------------------------------------------------------------
// Rotation of q and k (pairs i, i + D/2; a bf16 rounding behind every operation, as in elementwise.cu) and the write into 4-bit pages.
// Items of a token: groups of 16 values of k with those they are paired with (two groups), groups of v, 8 + 8 values of q; a thread to an item,
// so that no maximum crosses threads; rotated keys exist in registers only.
// Bound: the rows' bytes (a cached token is 9/16 of a byte per value, a quarter of what the 16-bit write stores).  4608 / 1000 / 7 rows of 32 + 8 + 8
// heads of 128 that lie in L2: 15.3 / 4.2 / 1.7 us (their bytes from memory 15.6 / 3.4 / 0).  48 registers keep an item's loads together: with 60 (8 blocks of 128 per SM) 16.4 /
// 4.9 / 1.7, with 32 16.4 / 5.1 / 2.1.  CTAs that go on to the next rows, whose places are known by then: 17.4 to 20.5.
// ------------------------------------------------------------------------------------------------------------------------
template <int D>
__global__ void __launch_bounds__(128, 10) rope_kvwrite_q4_kernel(uint4* qkv, const uint4* cos_sin, const int32_t* positions, const int32_t* slot_mapping,
                                                              uint8_t* kv_layer, int n_q, int n_kv) {
  follow_previous(qkv, cos_sin, positions, slot_mapping, kv_layer);
  constexpr int CPR = D / 8, HALF = CPR / 2;  // 16-byte pieces of a head's row, of half of it
  const long long t = blockIdx.x;
  uint4* row = qkv + t * (n_q + 2 * n_kv) * CPR;
  const int slot = slot_mapping[t];
  const uint4* cs_row = cos_sin + (long long)positions[t] * CPR;
  const int token = slot & 15;
  uint8_t* page = kv_layer + (long long)(slot >> 4) * n_kv * Kv4<D>::BYTES;
  const int k_items = n_kv * (D / 32), v_items = n_kv * (D / 16);
  const int n_items = k_items + v_items + n_q * HALF;
  for (int it = blockIdx.y * blockDim.x + threadIdx.x; it < n_items; it += gridDim.y * blockDim.x) {
    if (it < k_items) {
      if (slot < 0) continue;
      const int h = it / (D / 32), p = it % (D / 32);  // groups p and p + D/32
      const uint4* src = row + (n_q + h) * CPR + 2 * p;
      const uint4* cs = cs_row + 2 * p;
      uint4 a[2], b[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        a[i] = ld_v4(src + i);
        b[i] = ld_v4(src + HALF + i);
        turn_bf8(a[i], b[i], ld_v4(cs + i), ld_v4(cs + HALF + i));
      }
      uint8_t* to = page + h * Kv4<D>::BYTES;
      const int r = kv4_key_row<D>(token);
      uint32_t scale;
      *reinterpret_cast<uint2*>(to + kv4_key_code<D>(r, p)) = kv4_quantise(a[0], a[1], scale);
      to[kv4_key_scale<D>(r, p)] = (uint8_t)scale;
      *reinterpret_cast<uint2*>(to + kv4_key_code<D>(r, p + D / 32)) = kv4_quantise(b[0], b[1], scale);
      to[kv4_key_scale<D>(r, p + D / 32)] = (uint8_t)scale;
    } else if (it < k_items + v_items) {
      if (slot < 0) continue;
      const int h = (it - k_items) / (D / 16), p = (it - k_items) % (D / 16);
      const uint4* src = row + (n_q + n_kv + h) * CPR + 2 * p;
      uint8_t* to = page + h * Kv4<D>::BYTES;
      uint32_t scale;
      *reinterpret_cast<uint2*>(to + kv4_value_code<D>(token, p)) = kv4_quantise(ld_v4(src), ld_v4(src + 1), scale);
      to[kv4_value_scale<D>(token, p)] = (uint8_t)scale;
    } else {
      const int h = (it - k_items - v_items) / HALF, c0 = (it - k_items - v_items) % HALF;
      uint4* at = row + h * CPR + c0;
      uint4 a = ld_v4(at), b = ld_v4(at + HALF);
      turn_bf8(a, b, ld_v4(cs_row + c0), ld_v4(cs_row + HALF + c0));
      st_v4(at, a);
      st_v4(at + HALF, b);
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------------
// 4-bit pages as 16-bit ones (the layout of attn.cu: [2][n_kv][16][D], the 16-byte piece c of a row at c ^ (token & 7)).  Exact.
// ------------------------------------------------------------------------------------------------------------------------
// Keys or values of one head's page by a warp, through its own place in shared memory (their bytes, 16 a lane): then an item is 8 values, 16 bytes
// out, and a warp's stores are whole rows.
template <int D>
constexpr int SPREAD_BYTES = Kv4<D>::BYTES / 2;
template <int D, bool kValue>
__device__ __forceinline__ void kv4_spread_half(const uint8_t* half, uint4* out, uint8_t* stage, int lane) {
  constexpr int CPR = D / 8, PIECES = SPREAD_BYTES<D> / 16, FROM = kValue ? SPREAD_BYTES<D> : 0;
  __syncwarp();
  uint4 v[(PIECES + 31) / 32];
#pragma unroll
  for (int i = 0; i < (PIECES + 31) / 32; ++i)
    if (i * 32 + lane < PIECES) v[i] = ld_once_v4(half + (i * 32 + lane) * 16);
#pragma unroll
  for (int i = 0; i < (PIECES + 31) / 32; ++i)
    if (i * 32 + lane < PIECES) st_v4(stage + (i * 32 + lane) * 16, v[i]);
  __syncwarp();
#pragma unroll 4
  for (int it = lane; it < 16 * CPR; it += 32) {
    const int token = it / CPR, c = it % CPR, p = c >> 1, r = kv4_key_row<D>(token);
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(stage + (kValue ? kv4_value_code<D>(token, p) : kv4_key_code<D>(r, p)) - FROM + (c & 1) * 4);
    const uint32_t b = stage[(kValue ? kv4_value_scale<D>(token, p) : kv4_key_scale<D>(r, p)) - FROM];
    uint32_t h[4];
    kv4_halves(codes, h);
    const float s = kv4_scale_value(b);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
      w[i] = pack_bf16x2(f.x * s, f.y * s);
    }
    st_v4(out + token * CPR + (c ^ (token & 7)), make_uint4(w[0], w[1], w[2], w[3]));
  }
}
// keys (which = 0) or values of head h of page `from` to page `to`
template <int D>
__device__ __forceinline__ void kv4_spread_part(const uint8_t* kv4, long long from, uint4* out, long long to, int n_kv, int h, int which, uint8_t* stage, int lane) {
  const uint8_t* half = kv4 + (from * n_kv + h) * Kv4<D>::BYTES + which * SPREAD_BYTES<D>;
  uint4* at = out + ((to * 2 + which) * n_kv + h) * (16 * D / 8);
  if (which)
    kv4_spread_half<D, true>(half, at, stage, lane);
  else
    kv4_spread_half<D, false>(half, at, stage, lane);
}

constexpr int SPREAD_WARPS = 8;
template <int D>
__global__ void __launch_bounds__(SPREAD_WARPS * 32) kv4_unpack_kernel(const uint8_t* kv4, const int32_t* pages, int n_pages, uint4* out, int n_kv) {
  follow_previous(kv4, pages, out);
  __shared__ __align__(16) uint8_t stage[SPREAD_WARPS][SPREAD_BYTES<D>];
  const int warp = threadIdx.x >> 5;
  const long long items = 2LL * n_pages * n_kv;
  for (long long it = (long long)blockIdx.x * SPREAD_WARPS + warp; it < items; it += (long long)gridDim.x * SPREAD_WARPS) {
    const long long i = it / (2 * n_kv);
    const int part = (int)(it - i * (2 * n_kv));
    kv4_spread_part<D>(kv4, pages[i], out, i, n_kv, part >> 1, part & 1, stage[warp], threadIdx.x & 31);
  }
}

// The pages that a step's portions see, spread out to a workspace in which column c of row r of the block table is page r * bt_stride + c.
// A warp has the keys or the values of one head of one page; what a row needs it finds from the tiles (their first visible and their last key).
template <int D>
__global__ void __launch_bounds__(SPREAD_WARPS * 32) kv4_spread_kernel(const uint8_t* kv4, const int32_t* block_table, int bt_stride, const int4* tiles,
                                                                       int n_tiles, int n_kv, int window, uint4* out, int32_t* table) {
  follow_previous(kv4, block_table, tiles, out, table);
  __shared__ __align__(16) uint8_t stage[SPREAD_WARPS][SPREAD_BYTES<D>];
  const int row = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = (blockIdx.x * SPREAD_WARPS + warp) / (2 * n_kv), part = (blockIdx.x * SPREAD_WARPS + warp) % (2 * n_kv);
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
  if (c < s_lo / 16 || c >= min((s_hi + 15) / 16, bt_stride)) return;
  const long long to = (long long)row * bt_stride + c;
  kv4_spread_part<D>(kv4, block_table[to], out, to, n_kv, part >> 1, part & 1, stage[warp], lane);
  if (part == 0 && lane == 0) table[to] = (int32_t)to;
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
  // A thread to an item, in blocks of up to 128 (at 32 registers 4608 rows of 32 + 8 + 8 heads of 128 and reading them back: 26.7 us, in blocks of 192
  // 27.3, of 384 31.3; 512 of heads of 64 3.3 / 4.5 / 4.4)
  const int items = n_kv * (D / 32) + n_kv * (D / 16) + n_q * (D / 16), blocks = (items + 127) / 128;
  const int threads = ((items + blocks - 1) / blocks + 31) / 32 * 32;
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
  const long long items = 2LL * n_pages * n_kv, blocks = (items + SPREAD_WARPS - 1) / SPREAD_WARPS;
  B200Q_KV4_DIMS("kv4_unpack", D,
                 B200Q_CUDA(launch_early(kv4_unpack_kernel<kD>, dim3((unsigned)(blocks < 1 << 20 ? blocks : 1 << 20)), SPREAD_WARPS * 32, 0, as_stream(stream), 1,
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
                 B200Q_CUDA(launch_early(kv4_spread_kernel<kD>, dim3((unsigned)((2LL * bt_stride * n_kv + SPREAD_WARPS - 1) / SPREAD_WARPS), n_seqs), SPREAD_WARPS * 32, 0, as_stream(stream),
                                         1, (const uint8_t*)kv4_layer, block_table, bt_stride, (const int4*)tiles, n_tiles, n_kv, window,
                                         (uint4*)workspace, table)));
  count_launch();
  return b200q_prefill_attn_seqs(q, q_stride, out, workspace, table, bt_stride, n_seqs, tiles, n_tiles, n_q, n_kv, D, block_size, scale, softcap,
                                 window, stream);
}

}  // extern "C"
