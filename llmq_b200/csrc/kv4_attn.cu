// kv4_attn.cu — single-token attention over the 4-bit paged cache (layout: kv4.cuh).
//
//   out[s, h] = sum_j softmax_j(x(scale q . k_j)) v_j,  max(0, ctx - window) <= j < ctx,  x(y) = y or cap tanh(y / cap)
//
// Bound: 18 D bytes of a head's 16 tokens, and next to them the instructions that turn codes into operands: at the memory's rate an SM
// meets 42 codes a clock.  So a code is touched by few instructions:
//   * A page's part of one head arrives by one bulk copy in a ring that each warp has for itself; nobody waits for another warp.
//   * Scores are S^T = K Q^T: tokens are the rows of the 16 x 16 operand tile and heads of the group its 8 columns (a group of up to 8 fills
//     them; with heads as rows half the tile would be zeros).  The page is laid out so that a lane's operand registers are the codes of 16
//     consecutive bytes: one conversion and one multiplication by the scale (both exact) for two values, no shuffles, no transposes.
//   * Outputs are O^T = V^T P^T: the values' operand wants two tokens in one register; two words of different tokens are merged by nibbles
//     before the conversion (half an instruction for two values).  P^T is S^T after movmatrix.
//   * The running maximum moves only when a score is 2^4 above it, which a vote finds out; otherwise no lane asks another one for anything.
//     Probabilities are fp16 with 2^8 for the maximum's place (up to 2^12), so that a probability of 2^-32 of the largest still counts.
// Queries are divided by the power of two in their largest magnitude before they become fp16, which costs nothing that fp32 sums would keep.
#include <type_traits>

#include "kv4.cuh"
#include "layered_common.cuh"
#include "tcgen05.cuh"

namespace b200q {

bool batch_invariant();
int num_sms();

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t transposed8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float q4_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// tanh(x) = 1 - 2 / (1 + e^2x); x comes as 2 log2(e) x.  Off by 2^-22 at most, times the cap: as much as the score's own rounding
__device__ __forceinline__ float q4_tanh(float x2) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + q4_ex2(x2)));
  return fmaf(-2.f, r, 1.f);
}

struct Kv4Args {
  const bf16* q;
  bf16* out;
  const uint8_t* kv;
  const int32_t* block_table;
  const int32_t* ctx_lens;
  int* failed;  // set when a bounded wait runs out
  int q_stride, bt_stride, n_seqs, n_q, n_kv, G, window;
  float c0, c1;  // of a product: plain c0 = scale log2(e); capped c0 = 2 log2(e) scale / cap, c1 = cap log2(e)
};

// pages that a warp works on at once (one chain of scores, exponentials and outputs for 256 keys' values of D = 16), turns of them in flight
template <int D>
struct Q4Cfg {
  static constexpr int PAGES = 256 / D, STAGES = 3;
  static constexpr int TURN = PAGES * Kv4<D>::BYTES, RING = STAGES * TURN;  // 4608, 13824
};

// what a warp knows of the keys that it has seen: outputs times sums, per lane heads 2 t and 2 t + 1 (t = lane % 4)
template <int D>
struct Q4State {
  float o[D / 16][4];  // [tile i]: values 2 i (o[0], o[1]) and 2 i + 1 (o[2], o[3]) of lane / 4's part of a row
  float m[2], l[2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
  }
};

// queries of one group as the product's second operand: lane (g, t) has those values of head g that lane (., t) reads of a key
template <int D>
struct Q4Query {
  uint32_t b[D / 16][2];
  float c[2];  // c0 times what heads 2 t, 2 t + 1 were divided by
  __device__ __forceinline__ void load(const bf16* rows, int G, float c0, int lane) {
    const int g = lane >> 2, t = lane & 3;
    constexpr int PART = D == 256 ? 32 : D / 4, PARTS = D == 256 ? 2 : 1;  // consecutive values
    float x[PARTS][PART];
    float most = 0.f;
#pragma unroll
    for (int h = 0; h < PARTS; ++h)
#pragma unroll
      for (int i = 0; i < PART / 8; ++i) {
        const uint4 v = g < G ? ld_v4(rows + (long long)g * D + h * 128 + t * PART + i * 8) : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[h][8 * i + 2 * k] = bf16_lo(w[k]);
          x[h][8 * i + 2 * k + 1] = bf16_hi(w[k]);
          most = fmaxf(most, fmaxf(fabsf(bf16_lo(w[k])), fabsf(bf16_hi(w[k]))));
        }
      }
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const int e = min(max((int)(__float_as_uint(most) >> 23) - 127, -126), 126);
    const float down = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
    for (int h = 0; h < PARTS; ++h)
#pragma unroll
      for (int s = 0; s < PART / 4; ++s) {
        b[h * (PART / 4) + s][0] = pack_half2(x[h][4 * s] * down, x[h][4 * s + 1] * down);
        b[h * (PART / 4) + s][1] = pack_half2(x[h][4 * s + 2] * down, x[h][4 * s + 3] * down);
      }
#pragma unroll
    for (int i = 0; i < 2; ++i) c[i] = c0 * __uint_as_float((uint32_t)(127 + __shfl_sync(0xffffffffu, e, 8 * t + 4 * i)) << 23);
  }
};

__device__ __forceinline__ uint4 lds_v4(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ uint2 lds_v2(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
  return v;
}
__device__ __forceinline__ uint32_t lds_u32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at));
  return v;
}
__device__ __forceinline__ uint32_t lds_u16(uint32_t at) {
  unsigned short v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at));
  return v;
}

// four k-steps' worth: 8 values of rows g (w0) and g + 8 (w1) are two k-steps
__device__ __forceinline__ void q4_score_steps(float (&s)[4], uint32_t w0, uint32_t w1, uint32_t s0, uint32_t s1, const uint32_t (&b0)[2],
                                               const uint32_t (&b1)[2]) {
  uint32_t x[4], y[4];
  kv4_halves(w0, x);
  kv4_halves(w1, y);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = mul_half2(x[i], s0);
    y[i] = mul_half2(y[i], s1);
  }
  mma_f16_16816(s, x[0], y[0], x[1], y[1], b0[0], b0[1]);
  mma_f16_16816(s, x[2], y[2], x[3], y[3], b1[0], b1[1]);
}

// s = S^T of one page: rows are tokens (lane / 4 and + 8, in the page's order), columns heads 2 t, 2 t + 1
template <int D>
__device__ __forceinline__ void q4_scores(uint32_t page, const Q4Query<D>& q, float (&s)[4], int lane) {
  const int g = lane >> 2, t = lane & 3;
  s[0] = s[1] = s[2] = s[3] = 0.f;
  if constexpr (D == 64) {
    const uint2 a = lds_v2(page + g * 32 + t * 8), b = lds_v2(page + (g + 8) * 32 + t * 8);
    const uint32_t w = lds_u16(page + Kv4<D>::KS + lane * 2);
    const uint32_t s0 = kv4_scales<0, 0>(w), s1 = kv4_scales<1, 1>(w);
    q4_score_steps(s, a.x, b.x, s0, s1, q.b[0], q.b[1]);
    q4_score_steps(s, a.y, b.y, s0, s1, q.b[2], q.b[3]);
  } else if constexpr (D == 128) {
    const uint4 a = lds_v4(page + g * 64 + t * 16), b = lds_v4(page + (g + 8) * 64 + t * 16);
    const uint32_t w = lds_u32(page + Kv4<D>::KS + lane * 4);
    const uint32_t s0 = kv4_scales<0, 0>(w), s1 = kv4_scales<2, 2>(w), s2 = kv4_scales<1, 1>(w), s3 = kv4_scales<3, 3>(w);
    q4_score_steps(s, a.x, b.x, s0, s1, q.b[0], q.b[1]);
    q4_score_steps(s, a.y, b.y, s0, s1, q.b[2], q.b[3]);
    q4_score_steps(s, a.z, b.z, s2, s3, q.b[4], q.b[5]);
    q4_score_steps(s, a.w, b.w, s2, s3, q.b[6], q.b[7]);
  } else {
    const uint2 w = lds_v2(page + Kv4<D>::KS + lane * 8);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t at = page + g * 128 + ((t + 4 * h) ^ ((g & 1) * 4)) * 16;  // (rows g and g + 8 are turned alike)
      const uint4 a = lds_v4(at), b = lds_v4(at + 8 * 128);
      const uint32_t w0 = h ? w.x >> 16 : w.x, w1 = h ? w.y >> 16 : w.y;
      const uint32_t s0 = kv4_scales<0, 0>(w0), s1 = kv4_scales<0, 0>(w1), s2 = kv4_scales<1, 1>(w0), s3 = kv4_scales<1, 1>(w1);
      q4_score_steps(s, a.x, b.x, s0, s1, q.b[8 * h], q.b[8 * h + 1]);
      q4_score_steps(s, a.y, b.y, s0, s1, q.b[8 * h + 2], q.b[8 * h + 3]);
      q4_score_steps(s, a.z, b.z, s2, s3, q.b[8 * h + 4], q.b[8 * h + 5]);
      q4_score_steps(s, a.w, b.w, s2, s3, q.b[8 * h + 6], q.b[8 * h + 7]);
    }
  }
}

// 8 values of four tokens (one word each): four tiles of outputs.  s01, s23: the tokens' scales
__device__ __forceinline__ void q4_value_steps(float (*o)[4], uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, uint32_t s01, uint32_t s23,
                                               uint32_t p0, uint32_t p1) {
  constexpr uint32_t LOW = 0x0f0f0f0fu;
  uint32_t a[4], b[4], c[4], d[4];
  kv4_halves((w0 & LOW) | ((w1 << 4) & ~LOW), a);  // even values of tokens 0 and 1
  kv4_halves(((w0 >> 4) & LOW) | (w1 & ~LOW), b);  // odd ones
  kv4_halves((w2 & LOW) | ((w3 << 4) & ~LOW), c);
  kv4_halves(((w2 >> 4) & LOW) | (w3 & ~LOW), d);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    mma_f16_16816(o[i], mul_half2(a[i], s01), mul_half2(b[i], s01), mul_half2(c[i], s23), mul_half2(d[i], s23), p0, p1);
}

// outputs of one page's values.  keep (kEdge): scale bytes of tokens t, t + 4, t + 8, t + 12 that do not count become 0, because what lies
// there may be anything, NaN too
template <int D, bool kEdge>
__device__ __forceinline__ void q4_outputs(uint32_t page, uint32_t p0, uint32_t p1, float (*o)[4], uint32_t keep, int lane) {
  const int g = lane >> 2, t = lane & 3;
  if constexpr (D == 64) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = lds_u32(page + Kv4<D>::V + (t + 4 * j) * 32 + g * 4);
    uint32_t sc = lds_u32(page + Kv4<D>::VS + ((g >> 1) * 4 + t) * 4);
    if (kEdge) sc &= keep;
    q4_value_steps(o, w[0], w[1], w[2], w[3], kv4_scales<0, 1>(sc), kv4_scales<2, 3>(sc), p0, p1);
  } else if constexpr (D == 128) {
    uint2 w[4];
    const uint32_t at = page + Kv4<D>::V + t * 64 + (g ^ ((t >> 1) * 4)) * 8;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = lds_v2(at + j * 256);
    uint32_t sc = lds_u32(page + Kv4<D>::VS + lane * 4);
    if (kEdge) sc &= keep;
    const uint32_t s01 = kv4_scales<0, 1>(sc), s23 = kv4_scales<2, 3>(sc);
    q4_value_steps(o, w[0].x, w[1].x, w[2].x, w[3].x, s01, s23, p0, p1);
    q4_value_steps(o + 4, w[0].y, w[1].y, w[2].y, w[3].y, s01, s23, p0, p1);
  } else {
    uint4 w[4];
    const uint32_t at = page + Kv4<D>::V + t * 128 + (g ^ (t * 2)) * 16;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = lds_v4(at + j * 512);
    uint2 sc = lds_v2(page + Kv4<D>::VS + lane * 8);
    if (kEdge) {
      sc.x &= keep;
      sc.y &= keep;
    }
    const uint32_t s01 = kv4_scales<0, 1>(sc.x), s23 = kv4_scales<2, 3>(sc.x), r01 = kv4_scales<0, 1>(sc.y), r23 = kv4_scales<2, 3>(sc.y);
    q4_value_steps(o, w[0].x, w[1].x, w[2].x, w[3].x, s01, s23, p0, p1);
    q4_value_steps(o + 4, w[0].y, w[1].y, w[2].y, w[3].y, s01, s23, p0, p1);
    q4_value_steps(o + 8, w[0].z, w[1].z, w[2].z, w[3].z, r01, r23, p0, p1);
    q4_value_steps(o + 12, w[0].w, w[1].w, w[2].w, w[3].w, r01, r23, p0, p1);
  }
}

// One turn: up to PAGES pages at `at`, of which page x begins at key first[x] (kEdge: keys outside [lo, ctx) do not count, a page behind the
// last one lies outside whole).
template <int D, bool kCap, bool kEdge>
__device__ __forceinline__ void q4_turn(uint32_t at, const Q4Query<D>& q, Q4State<D>& st, float c1, const int* first, int lo, int ctx, int lane) {
  constexpr int P = Q4Cfg<D>::PAGES;
  const int g = lane >> 2, t = lane & 3;
  float s[P][4];
#pragma unroll
  for (int x = 0; x < P; ++x) q4_scores<D>(at + x * Kv4<D>::BYTES, q, s[x], lane);
  float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int x = 0; x < P; ++x)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float v = s[x][i] * q.c[i & 1];
      if (kCap) v = q4_tanh(v) * c1;
      if (kEdge) {
        const int j = first[x] + (g >> 1) + 4 * (g & 1) + 8 * (i >> 1);
        v = j >= lo && j < ctx ? v : -INFINITY;
      }
      s[x][i] = v;
      top[i & 1] = fmaxf(top[i & 1], v);
    }
  if (__any_sync(0xffffffffu, top[0] > st.m[0] + 4.f || top[1] > st.m[1] + 4.f)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 4));
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 8));
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 16));
    }
    float a[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float m = fmaxf(st.m[i], top[i]);
      a[i] = st.m[i] == -INFINITY ? 0.f : q4_ex2(st.m[i] - m);  // (nothing seen so far: outputs and sums are 0)
      st.m[i] = m;
      st.l[i] *= a[i];
    }
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      st.o[i][0] *= a[0];
      st.o[i][1] *= a[1];
      st.o[i][2] *= a[0];
      st.o[i][3] *= a[1];
    }
  }
  float base[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) base[i] = st.m[i] == -INFINITY ? 0.f : st.m[i] - 8.f;
#pragma unroll
  for (int x = 0; x < P; ++x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) s[x][i] = q4_ex2(s[x][i] - base[i & 1]);
    st.l[0] += s[x][0] + s[x][2];
    st.l[1] += s[x][1] + s[x][3];
  }
#pragma unroll
  for (int x = 0; x < P; ++x) {
    const uint32_t p0 = transposed8x8(pack_half2(s[x][0], s[x][1])), p1 = transposed8x8(pack_half2(s[x][2], s[x][3]));
    uint32_t keep = 0;
    if (kEdge) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = first[x] + t + 4 * j;
        keep |= key >= lo && key < ctx ? 0xffu << (8 * j) : 0u;
      }
    }
    q4_outputs<D, kEdge>(at + x * Kv4<D>::BYTES, p0, p1, st.o, keep, lane);
  }
}

// a warp's share of one sequence and head: pages wg, wg + n_warps, ... of those that hold visible keys, through the warp's own ring
template <int D>
struct Q4Share {
  static constexpr int P = Q4Cfg<D>::PAGES, STAGES = Q4Cfg<D>::STAGES;
  const int32_t* bt;
  const uint8_t* kv;  // this head's page of block 0
  int ctx, lo, page0, n, turns, wg, n_warps, ids_base, ids;
  long long page_stride;
  __device__ __forceinline__ void begin(const Kv4Args& a, int seq, int kvh, int wg_, int n_warps_, int lane) {
    ctx = a.ctx_lens[seq];
    wg = wg_;
    n_warps = n_warps_;
    ctx = min(max(ctx, 0), a.bt_stride * 16);
    lo = a.window > 0 && ctx > a.window ? ctx - a.window : 0;
    page0 = lo / 16;
    const int pages = (ctx + 15) / 16 - page0;
    n = pages > wg ? (pages - wg + n_warps - 1) / n_warps : 0;
    turns = (n + P - 1) / P;
    page_stride = (long long)a.n_kv * Kv4<D>::BYTES;
    kv = a.kv + (long long)kvh * Kv4<D>::BYTES;
    bt = a.block_table + (long long)seq * a.bt_stride + page0 + wg;
    ids_base = 0;
    ids = lane < n ? bt[n_warps * lane] : 0;
  }
  // whole warp; the pages of turn k into its place of the ring
  __device__ __forceinline__ void fetch(int k, uint8_t* ring, uint64_t* bars, int lane) {
    const int k0 = k * P;
    if (k0 - ids_base >= 32) {
      ids_base += 32;
      ids = ids_base + lane < n ? bt[n_warps * (ids_base + lane)] : 0;
    }
    const int st = k % STAGES, count = min(P, n - k0);
    int blk[P];
#pragma unroll
    for (int x = 0; x < P; ++x) blk[x] = __shfl_sync(0xffffffffu, ids, (k0 - ids_base + x) & 31);
    if (lane == 0) {
      mbar_expect_tx(bars + st, (uint32_t)(count * Kv4<D>::BYTES));
#pragma unroll
      for (int x = 0; x < P; ++x)
        if (x < count) tma_bulk_g2s(ring + st * Q4Cfg<D>::TURN + x * Kv4<D>::BYTES, kv + blk[x] * page_stride, Kv4<D>::BYTES, bars + st);
    }
  }
  __device__ __forceinline__ int first_key(int i) const { return (page0 + wg + n_warps * i) * 16; }
};

// WARPS warps of a CTA, and the gridDim.x CTAs of a cluster, share one sequence and head.
constexpr int Q4_WARPS = 4, Q4_MOST_CTAS = 16;
template <int D>
struct Q4Smem {
  static constexpr int TOTAL = Q4_WARPS * Q4Cfg<D>::RING + Q4_WARPS * Q4Cfg<D>::STAGES * 8;
};
template <int D, bool kCap>
__global__ void __launch_bounds__(Q4_WARPS * 32, D == 256 ? 3 : 4) kv4_decode_kernel(Kv4Args a) {
  follow_previous(a.q, a.out, a.kv, a.block_table, a.ctx_lens);
  using C = Q4Cfg<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int splits = gridDim.x, split = blockIdx.x, seq = blockIdx.y, kvh = blockIdx.z;
  uint8_t* ring = smem + warp * C::RING;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Q4_WARPS * C::RING) + warp * C::STAGES;
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < C::STAGES; ++s) mbar_init(bars + s, 1);
    mbar_fence_init();
  }
  __shared__ int dead;
  if (threadIdx.x == 0) dead = 0;
  __syncthreads();
  Q4Share<D> w;
  w.begin(a, seq, kvh, split * Q4_WARPS + warp, splits * Q4_WARPS, lane);
  for (int k = 0; k < min(w.turns, C::STAGES); ++k) w.fetch(k, ring, bars, lane);
  Q4Query<D> q;
  q.load(a.q + (long long)seq * a.q_stride + (long long)kvh * a.G * D, a.G, a.c0, lane);
  Q4State<D> st;
  st.clear();
  for (int k = 0; k < w.turns; ++k) {
    const int stage = k % C::STAGES;
    if (!__all_sync(0xffffffffu, mbar_wait_or_fail(bars + stage, (uint32_t)(k / C::STAGES) & 1u, &dead, a.failed))) break;
    const uint32_t at = smem_u32(ring + stage * C::TURN);
    int first[C::PAGES];
#pragma unroll
    for (int x = 0; x < C::PAGES; ++x) first[x] = w.first_key(k * C::PAGES + x);
    if (first[0] < w.lo || first[C::PAGES - 1] + 16 > w.ctx)
      q4_turn<D, kCap, true>(at, q, st, a.c1, first, w.lo, w.ctx, lane);
    else
      q4_turn<D, kCap, false>(at, q, st, a.c1, first, w.lo, w.ctx, lane);
    __syncwarp();
    if (k + C::STAGES < w.turns) w.fetch(k + C::STAGES, ring, bars, lane);
  }
  // ---- this warp's state into its ring (all its copies have come): [head][D] | maxima [8] | sums [8]
  float* mine = reinterpret_cast<float*>(ring);
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    st.l[i] += __shfl_xor_sync(0xffffffffu, st.l[i], 4);
    st.l[i] += __shfl_xor_sync(0xffffffffu, st.l[i], 8);
    st.l[i] += __shfl_xor_sync(0xffffffffu, st.l[i], 16);
    const int head = 2 * t + i;
    if (head < a.G) {
      float* to = mine + head * D + g * (D / 8);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) *reinterpret_cast<float2*>(to + 2 * k) = make_float2(st.o[k][i], st.o[k][2 + i]);
      if (g == 0) {
        mine[8 * D + head] = st.m[i];
        mine[8 * D + 8 + head] = st.l[i];
      }
    }
  }
  __syncthreads();
  // ---- one state per CTA, in the first warp's place (an item is two values, which one thread reads and writes)
  constexpr int RING_F = C::RING / 4;
  float* all = reinterpret_cast<float*>(smem);
  bf16* out = a.out + ((long long)seq * a.n_q + (long long)kvh * a.G) * D;
  for (int idx = threadIdx.x * 2; idx < a.G * D; idx += Q4_WARPS * 64) {
    const int r = idx / D;
    float M = -INFINITY, den = 0.f;
    float2 num = make_float2(0.f, 0.f);
#pragma unroll
    for (int x = 0; x < Q4_WARPS; ++x) M = fmaxf(M, all[x * RING_F + 8 * D + r]);
#pragma unroll
    for (int x = 0; x < Q4_WARPS; ++x) {
      const float mx = all[x * RING_F + 8 * D + r], wgt = mx == -INFINITY ? 0.f : q4_ex2(mx - M);
      const float2 v = *reinterpret_cast<const float2*>(all + x * RING_F + idx);
      num.x += wgt * v.x;
      num.y += wgt * v.y;
      den += wgt * all[x * RING_F + 8 * D + 8 + r];
    }
    if (splits > 1) {
      *reinterpret_cast<float2*>(all + idx) = num;
      if (idx % D == 0) {  // (the first warp's maxima and sums are still read: these go behind them)
        all[8 * D + 16 + r] = M;
        all[8 * D + 24 + r] = den;
      }
    } else {
      const float inv = den > 0.f ? 1.f / den : den == 0.f ? 0.f : den;  // (NaN stays)
      *reinterpret_cast<uint32_t*>(out + idx) = pack_bf16x2(num.x * inv, num.y * inv);
    }
  }
  if (splits > 1) {
    cluster_sync_all();
    const int per = (a.G * D / 2 + splits - 1) / splits * 2;
    for (int idx = split * per + threadIdx.x * 2; idx < min((split + 1) * per, a.G * D); idx += Q4_WARPS * 64) {
      const int r = idx / D;
      float M = -INFINITY, den = 0.f;
      float2 num = make_float2(0.f, 0.f);
      for (int x = 0; x < splits; ++x) M = fmaxf(M, ld_cluster_f32(mapa_shared(all + 8 * D + 16 + r, x)));
      for (int x = 0; x < splits; ++x) {
        const float mx = ld_cluster_f32(mapa_shared(all + 8 * D + 16 + r, x)), wgt = mx == -INFINITY ? 0.f : q4_ex2(mx - M);
        const uint32_t from = mapa_shared(all + idx, x);
        num.x += wgt * ld_cluster_f32(from);
        num.y += wgt * ld_cluster_f32(from + 4);
        den += wgt * ld_cluster_f32(mapa_shared(all + 8 * D + 24 + r, x));
      }
      const float inv = den > 0.f ? 1.f / den : den == 0.f ? 0.f : den;
      *reinterpret_cast<uint32_t*>(out + idx) = pack_bf16x2(num.x * inv, num.y * inv);
    }
    cluster_sync_all();  // nobody leaves while a peer still reads
  }
}

int g_q4_splits = 0;  // test hook: > 0 forces the number of CTAs per sequence and head

template <int D, bool kCap>
static int launch_kv4_decode(const Kv4Args& a, cudaStream_t st) {
  auto kern = kv4_decode_kernel<D, kCap>;
  static bool ready[64];
  int dev = 0;
  B200Q_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !ready[dev]) {
    B200Q_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Q4Smem<D>::TOTAL));
    B200Q_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    if (dev < 64) ready[dev] = true;
  }
  const int pages = a.window > 0 && (a.window + 15) / 16 + 1 < a.bt_stride ? (a.window + 15) / 16 + 1 : a.bt_stride;
  const long long items = (long long)a.n_seqs * a.n_kv;
  int splits = 1;
  while (!batch_invariant() && splits < Q4_MOST_CTAS && items * splits * 2 <= 4 * 148 && pages >= 2 * splits * Q4_WARPS * Q4Cfg<D>::PAGES) splits *= 2;
  if (g_q4_splits > 0) splits = g_q4_splits;
  for (int s0 = 0; s0 < a.n_seqs; s0 += 65535) {  // (a grid's second dimension ends there)
    Kv4Args b = a;
    b.n_seqs = a.n_seqs - s0 < 65535 ? a.n_seqs - s0 : 65535;
    b.q += (long long)s0 * a.q_stride;
    b.out += (long long)s0 * a.n_q * D;
    b.block_table += (long long)s0 * a.bt_stride;
    b.ctx_lens += s0;
    B200Q_CUDA(launch_early(kern, dim3(splits, b.n_seqs, b.n_kv), Q4_WARPS * 32, Q4Smem<D>::TOTAL, st, splits, b));
    count_launch();
  }
  return B200Q_OK;
}

}  // namespace b200q

using namespace b200q;

extern "C" {

int b200q_decode_attn_q4_set_splits(int splits) {
  B200Q_CHECK_ARG(splits >= 0 && splits <= Q4_MOST_CTAS, "decode_attn_q4: splits must be 0..%d", Q4_MOST_CTAS);
  g_q4_splits = splits;
  bump_tuning_epoch();
  return B200Q_OK;
}

int b200q_decode_attn_q4(const void* q, int q_stride, void* out, const void* kv4_layer, const int32_t* block_table, int bt_stride,
                         const int32_t* ctx_lens, int n_seqs, int n_q, int n_kv, int D, int block_size, float scale, float softcap, int window,
                         void* stream) {
  B200Q_CHECK_ARG(n_seqs >= 0 && n_kv > 0 && n_kv <= 65535 && n_q >= n_kv && n_q % n_kv == 0 && n_q / n_kv <= 8,
                  "decode_attn_q4: unsupported heads n_q=%d n_kv=%d (GQA group must be <= 8)", n_q, n_kv);
  B200Q_CHECK_ARG(block_size == 16 && (D == 64 || D == 128 || D == 256), "decode_attn_q4: unsupported D=%d block_size=%d (D in {64,128,256}, block 16)",
                  D, block_size);
  B200Q_CHECK_ARG(bt_stride >= 0 && bt_stride <= (1 << 26), "decode_attn_q4: bad bt_stride=%d", bt_stride);
  if (n_seqs == 0) return B200Q_OK;
  B200Q_CHECK_ARG(q && out && kv4_layer && block_table && ctx_lens, "decode_attn_q4: null argument");
  B200Q_CHECK_ARG(q_stride % 8 == 0 && q_stride >= n_q * D && ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kv4_layer)) & 15) == 0,
                  "decode_attn_q4: q (rows of q_stride=%d, a multiple of 8) and the cache must be 16-byte aligned", q_stride);
  B200Q_CHECK_ARG((reinterpret_cast<uintptr_t>(out) & 3) == 0, "decode_attn_q4: out must be 4-byte aligned");
  const float log2e = 1.4426950408889634f;
  Kv4Args a{};
  a.q = (const bf16*)q;
  a.out = (bf16*)out;
  a.kv = (const uint8_t*)kv4_layer;
  a.block_table = block_table;
  a.ctx_lens = ctx_lens;
  a.q_stride = q_stride;
  a.bt_stride = bt_stride;
  a.n_seqs = n_seqs;
  a.n_q = n_q;
  a.n_kv = n_kv;
  a.G = n_q / n_kv;
  a.window = window;
  a.c0 = softcap > 0.f ? 2.f * log2e * scale / softcap : scale * log2e;
  a.c1 = softcap * log2e;
  if (!wait_flag(&a.failed)) {
    set_error("decode_attn_q4: no host memory for the wait flag");
    return B200Q_ENOMEM;
  }
  cudaStream_t st = as_stream(stream);
  auto run = [&](auto cap) {
    constexpr bool c = decltype(cap)::value;
    if (D == 64) return launch_kv4_decode<64, c>(a, st);
    if (D == 128) return launch_kv4_decode<128, c>(a, st);
    return launch_kv4_decode<256, c>(a, st);
  };
  return softcap > 0.f ? run(std::true_type{}) : run(std::false_type{});
}

}  // extern "C"
