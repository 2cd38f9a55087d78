// kv4_attn.cu — single-token attention over the 4-bit paged cache (layout: kv4.cuh).
//
//   out[s, h] = sum_j softmax_j(x(scale q . k_j)) v_j,  max(0, ctx - window) <= j < ctx,  x(y) = y or cap tanh(y / cap)
//
// Bound: 18 D bytes of a head's 16 tokens from memory, and as long as that takes the instructions that turn codes into operands: from shared
// memory alone the loop below goes through 7.3 TB/s of pages (8 to 24 warps per SM alike; without the scales' multiplications 9.7, without
// the conversions 8.0, without the matrix products 7.6), the memory gives 6.5.  So a code is touched by few instructions:
//   * Scores are S^T = K Q^T: tokens are the rows of the 16 x 16 operand tile and heads of the group its 8 columns (a group of up to 8 fills
//     them; with heads as rows half the tile would be zeros).  The page is laid out so that a lane's operand registers are the codes of 16
//     consecutive bytes: one conversion and one multiplication by the scale (both exact) for two values, no shuffles, no transposes.
//   * Outputs are O^T = V^T P^T: the values' operand wants two tokens in one register; two words of different tokens are merged by nibbles
//     before the conversion (half an instruction for two values).  P^T is S^T after movmatrix.
//   * The running maximum moves only when a score is 2^4 above it, which a vote finds out; otherwise no lane asks another one for anything.
//     Probabilities are fp16 with 2^8 for the maximum's place (up to 2^12), so that a probability of 2^-32 of the largest still counts.
//   * A warp has its own pages on their way, by asynchronous copies; nobody waits for another warp.
// Queries are divided by the power of two in their largest magnitude before they become fp16, which costs nothing that fp32 sums would keep.
// Many sequences are streamed through by all warps (kv4_stream_kernel), few get a cluster of CTAs for each head (kv4_cluster_kernel).
// 700 sequences of 33 to 1000 tokens, 32 / 8 heads of 128: 95.1 us, 4.5 TB/s (the memory's share 66 us); 22 of 16000: 84, its copies alone 70 and
// its arithmetic alone 75; 16 of 1000 9.6; 3 of 9000 to 16000, heads of 64: 13.5 (3.4); 64 of 100 to 1500, 16 / 8 heads of 256, cap: 33.9 (17.5).
#include <algorithm>
#include <mutex>
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
  int q_stride, bt_stride, n_seqs, n_q, n_kv, G, window;
  float c0, c1;  // of a product: plain c0 = scale log2(e); capped c0 = 2 log2(e) scale / cap, c1 = cap log2(e)
};

// pages that a warp works on at once: a turn
template <int D>
struct Q4Cfg {
  static constexpr int PAGES = 256 / D, TURN = PAGES * Kv4<D>::BYTES;  // 4608 bytes
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

// queries of one group as the product's second operand: lane (g, t) has those values of head g that lane (., t) reads of a key
template <int D>
struct Q4Query {
  uint32_t b[D / 16][2];
  float c[2];  // c0 times what heads 2 t, 2 t + 1 were divided by
  template <typename F>
  __device__ __forceinline__ void load(F&& values, int G, float c0, int lane) {  // (values i .. i + 7 of the group's [G][D])
    const int g = lane >> 2, t = lane & 3;
    constexpr int PART = D == 256 ? 32 : D / 4, PARTS = D == 256 ? 2 : 1;  // consecutive values
    float x[PARTS][PART];
    float most = 0.f;
#pragma unroll
    for (int h = 0; h < PARTS; ++h)
#pragma unroll
      for (int i = 0; i < PART / 8; ++i) {
        const uint4 v = g < G ? values(g * D + h * 128 + t * PART + i * 8) : make_uint4(0, 0, 0, 0);
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
    const uint32_t p0 = movmatrix_trans(pack_half2(s[x][0], s[x][1])), p1 = movmatrix_trans(pack_half2(s[x][2], s[x][3]));
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

// ------------------------------------------------------------------------------------------------------------------------
// All pages of all sequences and heads in one row (units: sequence, head, page; an item's begin and end count as two pages more, about what
// they cost), and every warp of the chip a piece of it of the same length.  A warp streams through its piece as it comes, the next item's
// pages and queries on their way while the last one's are worked on; items that lie in it whole are finished there, of those that go on in
// the next warp's piece the states go to scratch, where the second kernel adds them up.  Ragged contexts, few long ones and many short ones
// then take the same time per page.
// ------------------------------------------------------------------------------------------------------------------------
constexpr int Q4_BEGIN = 2;        // units of an item beside its pages
constexpr int Q4_LEAST_SHARE = 8;  // units of a piece at least
template <int D>
struct Q4Stream {
  static constexpr int WARPS = 4 /* the join kernel's too */, STAGES = 2 /* turns change them with ^ 1 */, CTAS = D == 256 ? 3 : 4;
  static constexpr int TURN = Q4Cfg<D>::TURN;
  // bytes of a stage: a turn's pages, and the group's queries for an item that begins with it
  static int stage_bytes(int G) { return TURN + G * D * 2; }
  static int smem(int G) { return WARPS * STAGES * stage_bytes(G); }
};
// an item's chain of pieces: warps from .. from + n - 1 of them; n = 0: none
struct __align__(16) Q4Chain {
  int seq, head, from, n;
};
struct Q4Item {
  int seq, head, ctx, lo, page0, pages;
};
// scratch (none for whole items): two chains per warp (of the piece at its beginning, of the one at its end), then two pieces per warp, [G][D] outputs, [G] maxima, [G] sums
__host__ __device__ inline long long q4_piece_floats(int G, int D) { return ((long long)G * (D + 2) + 3) / 4 * 4; }
__host__ __device__ inline long long q4_chain_floats(int warps) { return 8LL * warps; }

// sequence s: keys that count and the pages that hold them
struct Q4Span {
  int ctx, lo, page0, pages;
  __device__ __forceinline__ Q4Span(const Kv4Args& a, int n) {
    ctx = min(max(n, 0), a.bt_stride * 16);
    lo = a.window > 0 && ctx > a.window ? ctx - a.window : 0;
    page0 = lo / 16;
    pages = (ctx + 15) / 16 - page0;
  }
  __device__ __forceinline__ int units() const { return pages > 0 ? pages + Q4_BEGIN : 0; }  // of a head
};

template <int D, bool kCap>
__global__ void __launch_bounds__(Q4Stream<D>::WARPS * 32, Q4Stream<D>::CTAS) kv4_stream_kernel(Kv4Args a, int stage_bytes, int whole_items, int least_share, float* scratch) {
  follow_previous(a.q, a.out, a.kv, a.block_table, a.ctx_lens, scratch);
  using C = Q4Stream<D>;
  constexpr int P = Q4Cfg<D>::PAGES, STAGES = C::STAGES, THREADS = C::WARPS * 32;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint32_t before[THREADS + 1];  // units of a head of the sequences before each thread's
  __shared__ uint32_t warp_sum[C::WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(smem + warp * STAGES * stage_bytes);
  // ---- where every thread's share of the sequences begins
  const int per = (a.n_seqs + THREADS - 1) / THREADS;
  {
    uint32_t mine = 0;
    const int s0 = threadIdx.x * per, s1 = min(a.n_seqs, s0 + per);
#pragma unroll 8
    for (int s = s0; s < s1; ++s) mine += Q4Span(a, a.ctx_lens[s]).units();
    uint32_t sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += y;
    }
    if (lane == 31) warp_sum[warp] = sum;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < C::WARPS; ++w)
      if (w < warp) sum += warp_sum[w];
    before[threadIdx.x + 1] = sum;
    if (threadIdx.x == 0) before[0] = 0;
    __syncthreads();
  }
  // ---- sequences of no keys
  for (int s = blockIdx.x; s < a.n_seqs; s += gridDim.x)
    if (a.ctx_lens[s] <= 0 || a.bt_stride == 0)
      for (int i = threadIdx.x; i < a.n_q * D / 2; i += THREADS) reinterpret_cast<uint32_t*>(a.out + (long long)s * a.n_q * D)[i] = 0;
  const long long units = (long long)before[THREADS] * a.n_kv;
  const int w_at = blockIdx.x * C::WARPS + warp, n_warps = gridDim.x * C::WARPS;
  // (a division of 64 bits is some 100 instructions: only where 32 do not hold the units)
  const int share = max(units >> 32 ? (int)((units + n_warps - 1) / n_warps) : (int)(((uint32_t)units + (uint32_t)n_warps - 1u) / (uint32_t)n_warps), least_share);
  const long long piece0 = (long long)w_at * share;
  long long u0 = piece0, u1 = min(u0 + share, units);
  Q4Chain* chains = reinterpret_cast<Q4Chain*>(scratch) + 2 * w_at;
  float* pieces = scratch + q4_chain_floats(n_warps) + 2 * w_at * q4_piece_floats(a.G, D);
  if (!whole_items && lane < 2) chains[lane] = {0, 0, 0, 0};  // (whole items have no pieces, and no scratch)
  __syncwarp();
  if (u0 >= u1) return;
  // ---- the sequence that has unit u, and its first unit
  auto find = [&](long long u, long long& first) {
    int c = 0;
#pragma unroll
    for (int k = 0; k < THREADS / 32; ++k) c += __popc(__ballot_sync(0xffffffffu, (long long)before[32 * k + lane + 1] * a.n_kv <= u));
    uint32_t at = before[c];
    for (int s = c * per;; s += 32) {
      uint32_t sum = per > 1 && s + lane < a.n_seqs ? Q4Span(a, a.ctx_lens[s + lane]).units() : 0;
      if (per == 1) {
        first = (long long)at * a.n_kv;
        return s;
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += y;
      }
      const int k = __popc(__ballot_sync(0xffffffffu, (long long)(at + sum) * a.n_kv <= u));
      const uint32_t all = __shfl_sync(0xffffffffu, sum, 31), here = __shfl_sync(0xffffffffu, sum, max(k - 1, 0));
      if (k < 32) {
        first = (long long)(at + (k ? here : 0)) * a.n_kv;
        return s + k;
      }
      at += all;
    }
  };
  long long seq_unit;
  int seq = find(u0, seq_unit);
  if (whole_items) {  // (B200Q_BATCH_INVARIANT: the items that begin in the piece, whole)
    auto up = [&](long long u, int s, long long first) {
      const uint32_t n = Q4Span(a, a.ctx_lens[s]).units();
      return first + ((uint32_t)(u - first) + n - 1) / n * n;
    };
    long long first;
    u0 = up(u0, seq, seq_unit);
    if (u1 < units) {
      const int s = find(u1, first);
      u1 = up(u1, s, first);
    }
    if (u0 >= u1) return;
    seq = find(u0, seq_unit);
  }
  // ---- pages on their way: of item (f_seq, f_head) from page f_page on; `left` units are not asked for yet.  What the other side has to know
  // of an item goes through a small ring (the items of the turns in flight, and one more)
  constexpr int ITEMS = 4;
  static_assert(ITEMS > STAGES, "an item for every turn in flight");
  __shared__ Q4Item items[C::WARPS][ITEMS];
  int f_seq = seq, f_ctx = a.ctx_lens[seq], f_item = 0;
  Q4Span f(a, f_ctx);
  const uint32_t into = (uint32_t)(u0 - seq_unit);
  int f_head = (int)(into / (uint32_t)f.units()), f_page = (int)(into - f_head * f.units()) - Q4_BEGIN, left = (int)(u1 - u0);
  long long unit = u0 - (f_page + Q4_BEGIN);  // the item's first
  if (f_page < 0) {  // (a piece that begins before the item's first page)
    left += f_page;
    f_page = 0;
  }
  if (left <= 0) return;  // (an item's begin and none of its pages)
  bool fresh = true;      // the next turn is the first one of its item here
  int f_stop = 0;
  const int page_stride = a.n_kv * Kv4<D>::BYTES;
  const uint8_t* f_kv = a.kv + (long long)f_head * Kv4<D>::BYTES;
  const int32_t* f_row = a.block_table + (long long)f_seq * a.bt_stride + f.page0;
  // numbers of the item's pages: 32 of them from ids_at on, the next 32, the first 32 of the sequence, and of the next sequence
  auto ids_of = [&](const int32_t* row, int pages, int from) { return from + lane < pages ? row[from + lane] : 0; };
  int ids_at = f_page;
  int ids0 = ids_of(f_row, f.pages, 0), ids = ids_at ? ids_of(f_row, f.pages, ids_at) : ids0, ids_ahead = ids_of(f_row, f.pages, ids_at + 32);
  int n_seq = 0, n_ctx = 0, n_ids = 0;  // the next sequence that has keys, once the last head of this one has begun
  auto look_ahead = [&]() {
    n_seq = f_seq;
    do n_ctx = ++n_seq < a.n_seqs ? a.ctx_lens[n_seq] : 1; while (n_ctx <= 0);
    if (n_seq < a.n_seqs) {
      const Q4Span x(a, n_ctx);
      n_ids = ids_of(a.block_table + (long long)n_seq * a.bt_stride + x.page0, x.pages, 0);
    }
  };
  auto begin_item = [&]() {
    fresh = true;
    if (lane == 0) items[warp][f_item % ITEMS] = {f_seq, f_head, f.ctx, f.lo, f.page0, f.pages};
    ++f_item;
    if (f_head == a.n_kv - 1) look_ahead();
  };
  auto next_item = [&]() {
    f_page = 0;
    f_kv += Kv4<D>::BYTES;
    if (++f_head == a.n_kv) {
      f_head = 0;
      f_seq = n_seq;
      f = Q4Span(a, n_ctx);
      f_kv = a.kv;
      f_row = a.block_table + (long long)f_seq * a.bt_stride + f.page0;
      ids0 = n_ids;
    }
    ids_at = 0;
    ids = ids0;
    ids_ahead = ids_of(f_row, f.pages, 32);
    begin_item();
  };
  // The next turn's pages into their stage: those of the item that are left, up to P of them.  Sixteen bytes per lane and copy, 512 in a row;
  // a turn is nine copies.  (A bulk copy has to be told its addresses by one lane for all, some 40 instructions a page.)
  constexpr int PIECES = Kv4<D>::BYTES / 16;  // of a page
  auto copy_pages = [&](uint32_t to, int count) {
    const uint8_t* from[P];
#pragma unroll
    for (int x = 0; x < P; ++x) from[x] = f_kv + lane * 16 + (long long)__shfl_sync(0xffffffffu, ids, f_page - ids_at + x) * page_stride;
#pragma unroll
    for (int k = 0; k < C::TURN / 512; ++k) {
      const int x0 = 32 * k / PIECES, x1 = (32 * k + 31) / PIECES;  // the pages in which a copy's lanes lie
      const bool second = x0 != x1 && lane >= x1 * PIECES - 32 * k;
      const uint8_t* src = second ? from[x1] + 16 * (32 * k - x1 * PIECES) : from[x0] + 16 * (32 * k - x0 * PIECES);
      if (count == P || (second ? x1 : x0) < count) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 512 * k), "l"(src) : "memory");
    }
  };
  auto fetch_edge = [&](uint32_t to) {  // behind the last page, at an item's beginning and end, where the numbers are used up
    if (left <= 0) return;
    if (f_page - ids_at >= 32) {
      ids_at += 32;
      ids = ids_ahead;
      ids_ahead = ids_of(f_row, f.pages, ids_at + 32);
    }
    const int count = min(P, min(f.pages - f_page, left));
    copy_pages(to, count);
    if (fresh) {
      const uint8_t* q_rows = reinterpret_cast<const uint8_t*>(a.q + (long long)f_seq * a.q_stride + (long long)f_head * a.G * D);
      for (int i = lane * 16; i < a.G * D * 2; i += 512)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to - lane * 16 + C::TURN + i), "l"(q_rows + i) : "memory");
      fresh = false;
    }
    left -= count;
    f_page += count;
    if (f_page == f.pages) {
      left -= Q4_BEGIN;  // (of the next item)
      if (left > 0) next_item();
    }
    // up to here a turn is P pages of the same item whose numbers are there, and the next one begins behind it
    f_stop = left > 0 && !fresh ? min(min(f.pages, f_page + left) - P, ids_at + 32 - P + 1) : 0;
  };
  auto fetch = [&](int stage) {
    const uint32_t to = ring + stage * stage_bytes + lane * 16;
    if (f_page < f_stop) {
      copy_pages(to, P);
      f_page += P;
      left -= P;
    } else {
      fetch_edge(to);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  begin_item();
  int page = f_page, to_do = left;  // the first item's pages begin here; units that have not been worked on, less the item's begin
#pragma unroll
  for (int s = 0; s < STAGES; ++s) fetch(s);
  Q4Query<D> q;
  Q4State<D> st;
  int stage = 0, item = 0;
  while (to_do > 0) {
    __syncwarp();
    const Q4Item it = items[warp][item++ % ITEMS];
    const bool whole = page == 0;  // the item began in this piece
    const int end = min(it.pages, page + to_do);
    to_do -= end - page + Q4_BEGIN;
    // turns whose keys all count begin from page `inner` up to `outer`
    const int inner = it.lo > (it.page0 + page) * 16 ? page + 1 : page, outer = min(end - P, it.pages - P - 1);
    for (bool first_turn = true; page < end; first_turn = false) {
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
      __syncwarp();
      const uint32_t at = ring + stage * stage_bytes;
      if (first_turn) {
        q.load([&](int i) { return lds_v4(at + C::TURN + 2 * i); }, a.G, a.c0, lane);
        st.clear();
      }
      if (page >= inner && page <= outer) {
        q4_turn<D, kCap, false>(at, q, st, a.c1, nullptr, 0, 0, lane);
      } else {
        int first[P];
#pragma unroll
        for (int x = 0; x < P; ++x) first[x] = page + x < end ? (it.page0 + page + x) * 16 : it.ctx;
        q4_turn<D, kCap, true>(at, q, st, a.c1, first, it.lo, it.ctx, lane);
      }
      __syncwarp();
      fetch(stage);
      stage ^= 1;
      page += P;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      st.l[i] += __shfl_xor_sync(0xffffffffu, st.l[i], 4);
      st.l[i] += __shfl_xor_sync(0xffffffffu, st.l[i], 8);
      st.l[i] += __shfl_xor_sync(0xffffffffu, st.l[i], 16);
    }
    if (whole && end == it.pages) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int head = 2 * t + i;
        const float inv = st.l[i] > 0.f ? 1.f / st.l[i] : st.l[i];  // (NaN stays)
        uint32_t* to = reinterpret_cast<uint32_t*>(a.out + ((long long)it.seq * a.n_q + (long long)it.head * a.G + head) * D) + g * (D / 16);
        if (head < a.G)
#pragma unroll
          for (int k = 0; k < D / 16; ++k) to[k] = pack_bf16x2(st.o[k][i] * inv, st.o[k][2 + i] * inv);
      }
    } else {
      const int slot = whole ? 1 : 0;  // (an item that ends in the next piece, or one that began in an earlier one)
      float* to = pieces + slot * q4_piece_floats(a.G, D);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int head = 2 * t + i;
        if (head < a.G) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) *reinterpret_cast<float2*>(to + head * D + g * (D / 8) + 2 * k) = make_float2(st.o[k][i], st.o[k][2 + i]);
          if (g == 0) {
            to[a.G * D + head] = st.m[i];
            to[a.G * D + a.G + head] = st.l[i];
          }
        }
      }
      if (lane == 0) {
        // pages of the item before this warp's piece and behind it, and so the warps that have the first and the last one
        const int ahead = max((int)(piece0 - (unit + Q4_BEGIN)), 0), behind = (int)(unit + Q4_BEGIN + it.pages - 1 - piece0);
        const int from = w_at - (ahead + share - 1) / share;
        chains[slot] = {it.seq, it.head, from, w_at + behind / share - from + 1};
      }
    }
    unit += it.pages + Q4_BEGIN;
    page = 0;
  }
}

// The pieces of one item's chain: every warp of it has 64 threads here, and as many groups of them share the outputs, four of them to a thread; threads
// that have no outputs of their own take a share of the pieces instead.
constexpr int Q4_JOIN = 64;
struct Q4Part {
  float m = -INFINITY, l = 0.f;
  float4 o = {0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ void add(const Q4Part& x) {
    if (x.m == -INFINITY && x.l == 0.f) return;
    const float top = fmaxf(m, x.m), old = m == -INFINITY ? 0.f : q4_ex2(m - top), now = x.m == -INFINITY ? 1.f : q4_ex2(x.m - top);
    m = top;
    l = l * old + x.l * now;
    o = make_float4(o.x * old + x.o.x * now, o.y * old + x.o.y * now, o.z * old + x.o.z * now, o.w * old + x.o.w * now);
  }
};
template <int D>
__global__ void __launch_bounds__(4 * Q4_JOIN) kv4_join_kernel(const float* scratch, bf16* out, int n_q, int G) {
  follow_previous(scratch, out);
  // two warps' chains to a block, 64 threads to each of a warp's two
  const int n_warps = gridDim.x * 2, tid = threadIdx.x % Q4_JOIN, w_at = blockIdx.x * 2 + threadIdx.x / (2 * Q4_JOIN), slot = threadIdx.x / Q4_JOIN % 2;
  __shared__ Q4Part shared[4 * Q4_JOIN];
  const Q4Chain c = reinterpret_cast<const Q4Chain*>(scratch)[2 * w_at + slot];
  if (c.n < 2) return;
  const float* pieces = scratch + q4_chain_floats(n_warps);
  const int size = (int)q4_piece_floats(G, D);
  const int rank = w_at - c.from, quads = G * D / 4, per = (quads + c.n - 1) / c.n, q_end = min(quads, (rank + 1) * per);
  const int here = max(min(Q4_JOIN, q_end - rank * per), 0);
  // threads side by side; the others go through the pieces beside them
  const int width = here > 1 ? 1 << (32 - __clz(here - 1)) : 1, parts = Q4_JOIN / width, part = tid / width;
  for (int q0 = rank * per; q0 < q_end; q0 += Q4_JOIN) {
    const int quad = q0 + tid % width, head = quad * 4 / D;
    const bool mine = tid % width < here && quad < q_end;
    Q4Part x;
    if (mine)
      for (int p0 = part; p0 < c.n; p0 += 4 * parts) {
        Q4Part y[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int p = p0 + u * parts;
          const float* from = pieces + (2LL * (c.from + p) + (p == 0)) * size;
          if (p < c.n) {
            y[u].m = from[G * D + head];
            y[u].l = from[G * D + G + head];
            y[u].o = *reinterpret_cast<const float4*>(from + 4 * quad);
          }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) x.add(y[u]);
      }
    auto other = [&](int o) {  // of the thread o lanes away
      Q4Part y;
      y.m = __shfl_xor_sync(0xffffffffu, x.m, o);
      y.l = __shfl_xor_sync(0xffffffffu, x.l, o);
      y.o = make_float4(__shfl_xor_sync(0xffffffffu, x.o.x, o), __shfl_xor_sync(0xffffffffu, x.o.y, o), __shfl_xor_sync(0xffffffffu, x.o.z, o),
                        __shfl_xor_sync(0xffffffffu, x.o.w, o));
      return y;
    };
    for (int o = 16; o >= width; o /= 2) x.add(other(o));
    if (parts > 1) {  // (two warps)
      shared[threadIdx.x] = x;
      asm volatile("bar.sync %0, 64;" ::"r"(1 + (int)threadIdx.x / Q4_JOIN) : "memory");
      if (tid < 32) x.add(shared[threadIdx.x + 32]);
      asm volatile("bar.sync %0, 64;" ::"r"(1 + (int)threadIdx.x / Q4_JOIN) : "memory");
    }
    if (mine && tid < width) {
      const float inv = x.l > 0.f ? 1.f / x.l : x.l;
      bf16* to = out + ((long long)c.seq * n_q + (long long)c.head * G) * D + 4 * quad;
      *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(x.o.x * inv, x.o.y * inv), pack_bf16x2(x.o.z * inv, x.o.w * inv));
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------------
// Few sequences: a cluster of CTAs to a sequence and head, each warp of it with every n-th page; no lists to make before the first page can be
// asked for and no second kernel, but whatever the lengths, every sequence gets the same warps.
// ------------------------------------------------------------------------------------------------------------------------
constexpr int Q4_MOST_CTAS = 16;
template <int D>
struct Q4Cluster {
  static constexpr int WARPS = 4, STAGES = 3, CTAS = Q4Stream<D>::CTAS, TURN = Q4Cfg<D>::TURN, RING = STAGES * TURN, SMEM = WARPS * RING;
  static_assert((8 * D + 32) * 4 <= RING, "a warp's outputs, maxima and sums");
};
template <int D, bool kCap>
__global__ void __launch_bounds__(Q4Cluster<D>::WARPS * 32, Q4Cluster<D>::CTAS) kv4_cluster_kernel(Kv4Args a) {
  follow_previous(a.q, a.out, a.kv, a.block_table, a.ctx_lens);
  using C = Q4Cluster<D>;
  constexpr int P = Q4Cfg<D>::PAGES, STAGES = C::STAGES, WARPS = C::WARPS, PIECES = Kv4<D>::BYTES / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int splits = gridDim.x, split = blockIdx.x, seq = blockIdx.y, kvh = blockIdx.z;
  const uint32_t ring = smem_u32(smem + warp * C::RING);
  // pages wg, wg + n_warps, ... of those that hold visible keys
  const int wg = split * WARPS + warp, n_warps = splits * WARPS;
  const Q4Span f(a, a.ctx_lens[seq]);
  const int n = f.pages > wg ? (f.pages - wg + n_warps - 1) / n_warps : 0, turns = (n + P - 1) / P;
  const int32_t* row = a.block_table + (long long)seq * a.bt_stride + f.page0 + wg;
  const uint8_t* kv = a.kv + (long long)kvh * Kv4<D>::BYTES + lane * 16;
  const long long page_stride = (long long)a.n_kv * Kv4<D>::BYTES;
  int ids_at = 0, ids = lane < n ? row[n_warps * lane] : 0;  // numbers of 32 pages
  auto fetch = [&](int k) {
    if (k < turns) {
      const int k0 = k * P, count = min(P, n - k0);
      if (k0 - ids_at >= 32) {
        ids_at += 32;
        ids = ids_at + lane < n ? row[n_warps * (ids_at + lane)] : 0;
      }
      const uint8_t* from[P];
#pragma unroll
      for (int x = 0; x < P; ++x) from[x] = kv + (long long)__shfl_sync(0xffffffffu, ids, k0 - ids_at + x) * page_stride;
      const uint32_t to = ring + k % STAGES * C::TURN + lane * 16;
#pragma unroll
      for (int i = 0; i < C::TURN / 512; ++i) {
        const int x0 = 32 * i / PIECES, x1 = (32 * i + 31) / PIECES;  // the pages in which a copy's lanes lie
        const bool second = x0 != x1 && lane >= x1 * PIECES - 32 * i;
        const uint8_t* src = second ? from[x1] + 16 * (32 * i - x1 * PIECES) : from[x0] + 16 * (32 * i - x0 * PIECES);
        if ((second ? x1 : x0) < count) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 512 * i), "l"(src) : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int k = 0; k < STAGES; ++k) fetch(k);
  Q4Query<D> q;
  const bf16* q_rows = a.q + (long long)seq * a.q_stride + (long long)kvh * a.G * D;
  q.load([&](int i) { return ld_v4(q_rows + i); }, a.G, a.c0, lane);
  Q4State<D> st;
  st.clear();
  for (int k = 0; k < turns; ++k) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
    __syncwarp();
    const uint32_t at = ring + k % STAGES * C::TURN;
    int first[P];
#pragma unroll
    for (int x = 0; x < P; ++x) first[x] = (f.page0 + wg + n_warps * (k * P + x)) * 16;
    if (first[0] < f.lo || first[P - 1] + 16 > f.ctx)
      q4_turn<D, kCap, true>(at, q, st, a.c1, first, f.lo, f.ctx, lane);
    else
      q4_turn<D, kCap, false>(at, q, st, a.c1, nullptr, 0, 0, lane);
    __syncwarp();
    fetch(k + STAGES);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncwarp();
  // ---- this warp's state into its ring: [head][D] | maxima [8] | sums [8]
  float* mine = reinterpret_cast<float*>(smem + warp * C::RING);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    st.l[i] += __shfl_xor_sync(0xffffffffu, st.l[i], 4);
    st.l[i] += __shfl_xor_sync(0xffffffffu, st.l[i], 8);
    st.l[i] += __shfl_xor_sync(0xffffffffu, st.l[i], 16);
    const int head = 2 * t + i;
    if (head < a.G) {
#pragma unroll
      for (int k = 0; k < D / 16; ++k) *reinterpret_cast<float2*>(mine + head * D + g * (D / 8) + 2 * k) = make_float2(st.o[k][i], st.o[k][2 + i]);
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
  auto write = [&](int i, float2 num, float den) {
    const float inv = den > 0.f ? 1.f / den : den;  // (NaN stays)
    *reinterpret_cast<uint32_t*>(out + i) = pack_bf16x2(num.x * inv, num.y * inv);
  };
  for (int i = threadIdx.x * 2; i < a.G * D; i += WARPS * 64) {
    const int r = i / D;
    float M = -INFINITY, den = 0.f;
    float2 num = make_float2(0.f, 0.f);
#pragma unroll
    for (int x = 0; x < WARPS; ++x) M = fmaxf(M, all[x * RING_F + 8 * D + r]);
#pragma unroll
    for (int x = 0; x < WARPS; ++x) {
      const float m = all[x * RING_F + 8 * D + r], l = all[x * RING_F + 8 * D + 8 + r];
      const float weight = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : q4_ex2(m - M);  // (no maximum and a sum: NaN)
      const float2 v = *reinterpret_cast<const float2*>(all + x * RING_F + i);
      num.x += weight * v.x;
      num.y += weight * v.y;
      den += weight * l;
    }
    if (splits > 1) {
      *reinterpret_cast<float2*>(all + i) = num;
      if (i % D == 0) {  // (the first warp's maxima and sums are still read: these go behind them)
        all[8 * D + 16 + r] = M;
        all[8 * D + 24 + r] = den;
      }
    } else {
      write(i, num, den);
    }
  }
  if (splits > 1) {
    cluster_sync_all();
    const int per = (a.G * D / 2 + splits - 1) / splits * 2;
    for (int i = split * per + threadIdx.x * 2; i < min((split + 1) * per, a.G * D); i += WARPS * 64) {
      const int r = i / D;
      float M = -INFINITY, den = 0.f;
      float2 num = make_float2(0.f, 0.f);
      for (int x = 0; x < splits; ++x) M = fmaxf(M, ld_cluster_f32(mapa_shared(all + 8 * D + 16 + r, x)));
      for (int x = 0; x < splits; ++x) {
        const float m = ld_cluster_f32(mapa_shared(all + 8 * D + 16 + r, x)), l = ld_cluster_f32(mapa_shared(all + 8 * D + 24 + r, x));
        const float weight = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : q4_ex2(m - M);
        const uint32_t from = mapa_shared(all + i, x);
        num.x += weight * ld_cluster_f32(from);
        num.y += weight * ld_cluster_f32(from + 4);
        den += weight * l;
      }
      write(i, num, den);
    }
    cluster_sync_all();  // nobody leaves while a peer still reads
  }
}

// test hook: 1 / 0 give items to warps whole or not, -2 to clusters, -3 as 0 but that the pieces ask for more memory than any GPU has (-1: by size,
// and as B200Q_BATCH_INVARIANT says)
int g_q4_whole = -1;
static std::mutex g_q4_pair;  // no other thread's pieces on the same stream between a stream kernel and its join

// CTAs of a cluster for each of these items of up to `pages` pages, or 0: the kernel above.  Times in us, fitted to 1 to 450 sequences of 16 to 16000
// tokens, 8 heads.  Clusters: 4 and what a CTA's pages take (beside three others on an SM; alone half; 16 CTAs to a cluster 2.5 more), or several
// rounds of CTAs; the kernel above: `start`, or where items are whole what the pages of one take a warp, and `slope` times what all pages take from
// memory.  us above / with clusters, D = 128: one sequence of 64 tokens 5.9 / 3.4, of 300 10.8 / 5.6, 16 of 1000 15.1 / 9.6, 16 of 4000 24.4 / 20.5, 24 of
// 4000 33.9 / 34.5, 150 of 300 22.5 / 18.1, 250 of 128 14.1 / 15.8; D = 256: 6 of 4000 22.0 / 17.1, 8 of 4000 25.4 / 26.6.  Lengths below the table's width:
// 48 of 200 to 2000 23.8 / 30.2, 700 of 33 to 1000 95 / 105.
template <int D>
static int kv4_clusters(long long items, int pages, bool forced) {
  constexpr double page = D == 64 ? 0.15 : D == 128 ? 0.27 : 0.44, start = D == 64 ? 9.5 : D == 128 ? 10.0 : 14.0,
                   slope = D == 64 ? 1.5 : D == 128 ? 1.33 : 1.05;
  const long long places = (long long)num_sms() * Q4Cluster<D>::CTAS;
  if (items > 8 * places) return 0;
  int n = 1;  // (clusters of 16 leave places that none fits into: where they fill two thirds)
  while (n < Q4_MOST_CTAS && items * n * 2 <= (n == 8 ? places * 13 / 20 : places) && pages >= 2 * n * Q4Cluster<D>::WARPS * Q4Cfg<D>::PAGES) n *= 2;
  const double all = (double)items * pages * Kv4<D>::BYTES / 6.45e6, per_sm = (double)(items * n) / num_sms(),
               full = std::min(1.0, D == 256 ? 0.5 + 0.2 * per_sm : 0.3 + 0.25 * per_sm), rounds = (double)items / places,
               clusters = rounds <= 1.0 ? 4.0 + full * page * pages / n + (n == 16 ? 2.5 : 0.0) : 3.0 + rounds * (2.8 + page * pages),
               above = pages <= 8 ? 4.5 + 2.0 * page * pages + 1.33 * all : start + slope * all;
  return forced || clusters < above ? n : 0;
}

template <int D, bool kCap>
static int launch_kv4_stream(const Kv4Args& a, cudaStream_t st) {
  using C = Q4Stream<D>;
  auto kern = kv4_stream_kernel<D, kCap>;
  static bool ready[64];
  int dev = 0;
  B200Q_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !ready[dev]) {
    B200Q_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::smem(8)));
    B200Q_CUDA(cudaFuncSetAttribute(kv4_cluster_kernel<D, kCap>, cudaFuncAttributeMaxDynamicSharedMemorySize, Q4Cluster<D>::SMEM));
    B200Q_CUDA(cudaFuncSetAttribute(kv4_cluster_kernel<D, kCap>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    if (dev < 64) ready[dev] = true;
  }
  const int ctas = C::CTAS * num_sms(), warps = ctas * C::WARPS;
  // Items of up to 8 pages go to warps whole: adding up pieces costs as much as they do (one sequence of 64 tokens, 8 kv heads, 5.6 us, in
  // pieces 9.5; 2800 of 128 tokens 96.5, in pieces 103.9).
  const int width = a.window > 0 && a.window / 16 + 2 < a.bt_stride ? a.window / 16 + 2 : a.bt_stride;  // pages of an item at most
  if (g_q4_whole == -2 || (g_q4_whole == -1 && !batch_invariant()))
    if (const int n = kv4_clusters<D>((long long)a.n_seqs * a.n_kv, width, g_q4_whole == -2)) {
      B200Q_CUDA(launch_early(kv4_cluster_kernel<D, kCap>, dim3(n, a.n_seqs, a.n_kv), Q4Cluster<D>::WARPS * 32, Q4Cluster<D>::SMEM, st, n, a));
      count_launch();
      return B200Q_OK;
    }
  bool whole = g_q4_whole == -1 || g_q4_whole == -2 ? batch_invariant() || width <= 8 : g_q4_whole == 1;
  float* scratch = nullptr;
  // (where there is no memory for pieces, items go to warps whole)
  const size_t bytes = g_q4_whole == -3 ? (size_t)1 << 60 : (size_t)(q4_chain_floats(warps) + 2 * warps * q4_piece_floats(a.G, D)) * sizeof(float);
  if (!whole && stream_scratch(1, bytes, st, &scratch)) {
    cudaGetLastError();
    whole = true;
  }
  std::lock_guard<std::mutex> together(g_q4_pair);
  B200Q_CUDA(launch_early(kern, dim3(ctas), C::WARPS * 32, C::smem(a.G), st, 1, a, C::stage_bytes(a.G), (int)whole, whole ? 1 : Q4_LEAST_SHARE, scratch));
  count_launch();
  if (whole) return B200Q_OK;
  B200Q_CUDA(launch_early(kv4_join_kernel<D>, dim3(warps / 2), 4 * Q4_JOIN, 0, st, 1, (const float*)scratch, a.out, a.n_q, a.G));
  count_launch();
  return B200Q_OK;
}

}  // namespace b200q

using namespace b200q;

extern "C" {

int b200q_decode_attn_q4_set_whole(int whole) {
  B200Q_CHECK_ARG(whole >= -3 && whole <= 1, "decode_attn_q4: whole must be -3..1");
  g_q4_whole = whole;
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
  // (what the kernel counts in 32 bits: units of a head, of a sequence, of a warp's piece)
  const long long units = bt_stride + Q4_BEGIN;
  B200Q_CHECK_ARG(units * n_seqs < 1ll << 32 && units * n_kv < 1ll << 31 && units * n_seqs < (1ll << 40) / n_kv,
                  "decode_attn_q4: too much at once: n_seqs=%d bt_stride=%d n_kv=%d (2^32 pages of a head, 2^31 of a sequence, 2^40 in all)", n_seqs,
                  bt_stride, n_kv);
  if (n_seqs == 0) return B200Q_OK;
  // (a table of no columns need not exist)
  B200Q_CHECK_ARG(q && out && ctx_lens && (bt_stride == 0 || (kv4_layer && block_table)), "decode_attn_q4: null argument");
  B200Q_CHECK_ARG(q_stride % 8 == 0 && q_stride >= n_q * D && ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kv4_layer)) & 15) == 0,
                  "decode_attn_q4: q (rows of q_stride=%d, a multiple of 8) and the cache must be 16-byte aligned", q_stride);
  B200Q_CHECK_ARG((reinterpret_cast<uintptr_t>(out) & 7) == 0, "decode_attn_q4: out must be 8-byte aligned");
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
  cudaStream_t st = as_stream(stream);
  auto run = [&](auto cap) {
    constexpr bool c = decltype(cap)::value;
    if (D == 64) return launch_kv4_stream<64, c>(a, st);
    if (D == 128) return launch_kv4_stream<128, c>(a, st);
    return launch_kv4_stream<256, c>(a, st);
  };
  return softcap > 0.f ? run(std::true_type{}) : run(std::false_type{});
}

}  // extern "C"
