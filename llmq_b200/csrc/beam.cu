// beam.cu — the best continuations of beams: for every group of W rows of logits, of t(w, v) = score_w + logit_wv - log sum_v exp(logit_wv)
// the K largest of W V, of equal ones those with the lowest w V + v first; and the first W of them that do not end.
//
// Two kernels.  The first has a piece of a row per CTA and goes through it once: the sum of its exponentials and its K best logits (a row's
// order needs no logarithm).  The largest logits of groups of threads give a bound that K of the first tile reach; vectors in which something
// reaches it are collected, and once they are many their logits are ranked by counting: the K-th best so far is the bound from there on.  The
// second kernel has a group per CTA: sums to logarithms, best logits to scores, and again a bound (the K-th best of the pieces' first entries),
// what reaches it, and ranks.
// Scores that are compared across rows are 64 bits; a row's logarithm comes from sums whose terms are off by 2^-22 (the exponential) and 1.5 x 2^-24
// (its exponent's rounding) at most, whatever the logits' size, and go through five additions in fp32 before those in 64 bits.
// Bound: the logits, 2 bytes each, once; next to it the exponentials (16 a cycle and SM: two thirds of the memory's
// time) and some nine instructions a logit.  Logits come by asynchronous copies two tiles ahead (in registers a tile ahead 2.7 us more).
// 48 groups of 8 beams over 256000 tokens, 16 candidates: 54.4 us (the memory's share 30; 46.5 for one candidate of each row, so that looking for
// the 16 best and the second kernel's ranks are 8; with 4 or 3 CTAs per SM in place of 5 55.3 and 60.0), one group of 4 over 128256: 10.4.
#include "common.cuh"

namespace b200q {

bool batch_invariant();

constexpr int BEAM_THREADS = 256, BEAM_MOST_K = 64, BEAM_MOST_W = 32, BEAM_FOUND = 512, BEAM_VECTORS = 256;

__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// either of two numbers >= that of `bound` (NaN is not)
__device__ __forceinline__ bool reaches_bf16x2(uint32_t m, uint32_t bound) {
  int r;
  asm("{ .reg .pred p, q;\n setp.ge.bf16x2 p|q, %1, %2;\n or.pred p, p, q;\n selp.s32 %0, 1, 0, p; }" : "=r"(r) : "r"(m), "r"(bound));
  return r;
}
// unsigned integers of the same order as the numbers (bf16 bits); NaN counts as -infinity, -0 as 0
__device__ __forceinline__ uint32_t beam_order(uint32_t h) {
  if ((h & 0x7fffu) > 0x7f80u) h = 0xff80u;
  if (h == 0x8000u) h = 0u;
  return (h & 0x8000u) ? 0xffffu ^ h : h | 0x8000u;
}
// Sums of a row are those of 2^(L x - c), L the fp32 number next to log2(e) and c a whole number near L times the largest logit so far: L x - c is
// rounded once, so that it is off by 2^-24 of itself, not of x, and by more than 1.5 x 2^-24 only where the term is small beside the largest.  What L is
// off by makes e^x of 2^(L x) by a factor e^(BEAM_LOW x), for which that of the largest logit stands.
constexpr float BEAM_L = 1.44269504088896341f;
constexpr double BEAM_LOW = (1.44269504088896340736 - 1.44269502162933349609) * 0.69314718055994530942;
__device__ __forceinline__ float beam_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^(L w + minus_c) of two logits, and of eight (a pair of sums)
__device__ __forceinline__ f32x2 beam_exps(uint32_t w, float minus_c) {
  const float2 h = halves_of(fma2(pair_of(bf16_lo(w), bf16_hi(w)), pair_of(BEAM_L, BEAM_L), pair_of(minus_c, minus_c)));
  return pair_of(beam_ex2(h.x), beam_ex2(h.y));
}
__device__ __forceinline__ f32x2 beam_exps(const uint4& v, float minus_c) {
  return add2(add2(beam_exps(v.x, minus_c), beam_exps(v.y, minus_c)), add2(beam_exps(v.z, minus_c), beam_exps(v.w, minus_c)));
}
// 2^e of a whole number e (0 below the smallest)
__device__ __forceinline__ float power_of_two(float e) { return e < -126.f ? 0.f : __int_as_float((127 + (int)e) << 23); }

// logits 8 i .. 8 i + 7 of a row, those behind its end as -infinity.  Rows of a V that is no multiple of 8 begin anywhere: they are cut at the
// same places all the same, so that equal rows give equal sums, and a vector is put together from the two aligned ones that it lies in.
template <bool kAligned>
struct BeamRow {
  const bf16* x;
  long long V;
  const uint4* base;  // the aligned vector in which the row begins
  int shift;          // logits of that vector that are another row's
  long long left;     // whole aligned vectors from `base` to the end of the last row
  __device__ __forceinline__ BeamRow(const bf16* logits, long long V_, long long row, long long rows) : x(logits + row * V_), V(V_) {
    const long long at = row * V;
    shift = kAligned ? 0 : (int)(at & 7);
    base = reinterpret_cast<const uint4*>(logits + (at - shift));
    left = (rows * V - (at - shift)) / 8;
  }
  __device__ __forceinline__ uint4 operator()(long long i) const {
    if constexpr (kAligned) return ld_once_v4(base + i);
    if (8 * i + 8 > V || i + 2 > left) {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const long long e = 8 * i + 2 * k;
        const uint32_t lo = e < V ? *reinterpret_cast<const uint16_t*>(x + e) : 0xff80u, hi = e + 1 < V ? *reinterpret_cast<const uint16_t*>(x + e + 1) : 0xff80u;
        w[k] = lo | hi << 16;
      }
      return make_uint4(w[0], w[1], w[2], w[3]);
    }
    const uint4 p = ld_v4(base + i), q = ld_v4(base + i + 1);
    uint32_t w[7] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z}, v[5];
    if (shift & 4) {
      w[0] = w[2];
      w[1] = w[3];
      w[2] = w[4];
      w[3] = w[5];
      w[4] = w[6];
      w[5] = q.w;
    }
#pragma unroll
    for (int k = 0; k < 5; ++k) v[k] = (shift & 2) ? w[k + 1] : w[k];
    const int bits = (shift & 1) * 16;
    return make_uint4(__funnelshift_r(v[0], v[1], bits), __funnelshift_r(v[1], v[2], bits), __funnelshift_r(v[2], v[3], bits),
                      __funnelshift_r(v[3], v[4], bits));
  }
};

// the next place in a list in shared memory (few lanes at a time ask for one: no need to ask for all of them together)
__device__ __forceinline__ int next_place(int* count) {
  int at;
  asm volatile("atom.shared.add.s32 %0, [%1], 1;" : "=r"(at) : "r"(smem_u32(count)) : "memory");
  return at;
}

// A piece of a row, in tiles of TILE vectors; the next ones are on their way while one is looked at.  Vectors collected from which on they are
// ranked: 24 / 48 / 96 cost 384 rows of 256000 logits 54.9 / 54.4 / 60.0 us.
constexpr int BEAM_NV = 4, TILE = BEAM_NV * BEAM_THREADS, BEAM_MANY = 48, BEAM_RING = 2;
template <bool kAligned>
__global__ void __launch_bounds__(BEAM_THREADS, 5) beam_rows_kernel(const bf16* logits, long long V, int K, long long row0, long long rows,
                                                                    int2* entries, double2* piece_sums) {
  follow_previous(logits, entries, piece_sums);
  const int tid = threadIdx.x, piece = blockIdx.x, n_pieces = gridDim.x;
  const long long row = row0 + blockIdx.y;
  const BeamRow<kAligned> x(logits, V, row, rows);
  const int vecs = (int)((V + 7) / 8), per = (vecs + n_pieces - 1) / n_pieces, v0 = min(vecs, piece * per), v1 = min(vecs, v0 + per);
  const uint4 none = make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
  __shared__ float tops[BEAM_THREADS];
  __shared__ uint64_t found[BEAM_FOUND], best[BEAM_MOST_K];
  __shared__ double sums[BEAM_THREADS / 32];
  __shared__ uint4 vectors[BEAM_VECTORS];  // that hold a logit that reaches the bound, and which they are
  __shared__ int vector_at[BEAM_VECTORS], n_vectors, n_found, bound_s, top_s;
  __shared__ uint64_t best_s[BEAM_THREADS / 32];
  // Rows of aligned vectors come through a ring of BEAM_RING tiles, every thread's vectors in places of its own (no waiting for others); of
  // other rows the next tile's are in registers.
  extern __shared__ uint4 ring[];
  const uint32_t place = smem_u32(ring + tid);
  const uint4* source = x.base + v0 + tid;
  const int whole = (v1 - v0) / TILE;
  auto ask = [&](int tile, int stage) {
    const uint32_t to = place + 16 * stage * TILE;
    if (tile < whole) {
#pragma unroll
      for (int u = 0; u < BEAM_NV; ++u)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 16 * u * BEAM_THREADS), "l"(source + u * BEAM_THREADS) : "memory");
    } else {
      const int left = v1 - v0 - tile * TILE - tid;
#pragma unroll
      for (int u = 0; u < BEAM_NV; ++u)
        if (u * BEAM_THREADS < left)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 16 * u * BEAM_THREADS), "l"(source + u * BEAM_THREADS) : "memory");
    }
    source += TILE;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  uint4 a[BEAM_NV];
  if constexpr (kAligned) {
#pragma unroll
    for (int s = 0; s < BEAM_RING; ++s) ask(s, s);
    asm volatile("cp.async.wait_group %0;" ::"n"(BEAM_RING - 1) : "memory");
#pragma unroll
    for (int u = 0; u < BEAM_NV; ++u) a[u] = v0 + u * BEAM_THREADS + tid < v1 ? lds_v4(place + 16 * u * BEAM_THREADS) : none;
  } else {
#pragma unroll
    for (int u = 0; u < BEAM_NV; ++u) a[u] = v0 + u * BEAM_THREADS + tid < v1 ? x(v0 + u * BEAM_THREADS + tid) : none;
  }
  if (tid == 0) n_found = n_vectors = 0;
  float bound = -INFINITY;
  uint32_t bound2 = 0xff80ff80u;  // twice the same as bf16
  double sum = 0.0;  // (an fp32 sum swallows the small terms behind a large one: only a tile's meet there)
  // the logits of the collected vectors that reach the bound, and the k0 in best: the K best of them into best, in order.  How many there are;
  // -1: too many to look at
  auto prune = [&](int k0) {
    __syncthreads();
    const int nv = n_vectors;
    if (nv > 0 && nv <= BEAM_VECTORS)
      for (int i = tid; i < 8 * nv; i += BEAM_THREADS) {
        const uint32_t w = reinterpret_cast<const uint32_t*>(vectors)[i >> 1], h = i & 1 ? w >> 16 : w & 0xffffu;
        const long long token = 8LL * vector_at[i >> 3] + (i & 7);
        if (__uint_as_float(h << 16) >= bound && token < V) {
          const int at = next_place(&n_found);
          if (at < BEAM_FOUND) found[at] = ((uint64_t)beam_order(h) << 32) | (0xffffffffu - (uint32_t)token);
        }
      }
    __syncthreads();
    const int n = n_found;
    if (nv == 0) return k0;
    if (nv > BEAM_VECTORS || n > BEAM_FOUND) return -1;
    uint64_t key[BEAM_FOUND / BEAM_THREADS + 1];
    int rank[BEAM_FOUND / BEAM_THREADS + 1];
#pragma unroll
    for (int i = 0; i < BEAM_FOUND / BEAM_THREADS + 1; ++i) {
      const int at = i * BEAM_THREADS + tid;
      rank[i] = K;
      if (at >= k0 + n) continue;
      key[i] = at < k0 ? best[at] : found[at - k0];
      rank[i] = at < k0 ? at : 0;
#pragma unroll 4
      for (int k = 0; k < n; ++k) rank[i] += found[k] > key[i];
      if (at >= k0)
#pragma unroll 4
        for (int k = 0; k < k0; ++k) rank[i] += best[k] > key[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < BEAM_FOUND / BEAM_THREADS + 1; ++i)
      if (rank[i] < K) best[rank[i]] = key[i];
    if (tid == 0) n_found = n_vectors = 0;
    __syncthreads();
    return min(k0 + n, K);
  };
  auto value_of = [](uint64_t key) {  // the logit of a key
    const uint32_t o = (uint32_t)(key >> 32), h = (o & 0x8000u) ? o & 0x7fffu : 0xffffu ^ o;
    return __uint_as_float(h << 16);
  };
  // a bound that K of the first tile reach: the K-th of the largest logits of groups of threads, at least twice as many as are wanted.  Where
  // fewer are above -infinity, the lowest number there is
  {
    uint32_t m = 0xff80ff80u;
#pragma unroll
    for (int u = 0; u < BEAM_NV; ++u) m = max_bf16x2(m, max_bf16x2(max_bf16x2(a[u].x, a[u].y), max_bf16x2(a[u].z, a[u].w)));
    const int deep = K <= 32 ? 2 : 1, groups = BEAM_THREADS >> deep;
    float mine = fmaxf(bf16_lo(m), bf16_hi(m));  // (max of a number and NaN is the number; -infinity was among them)
    for (int o = 1; o < 1 << deep; o <<= 1) mine = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, o));
    if ((tid & ((1 << deep) - 1)) == 0) tops[tid >> deep] = mine;
    __syncthreads();
    if (tid < groups) {
      const float y = tops[tid];
      int rank = 0;
#pragma unroll 16
      for (int i = 0; i < groups; ++i) rank += tops[i] > y || (tops[i] == y && i < tid);
      if (rank == K - 1) bound_s = __float_as_int(y);
      if (rank == 0) top_s = __float_as_int(y);
    }
    __syncthreads();
    bound = fmaxf(__int_as_float(bound_s), __uint_as_float(0xff7f0000u));
    bound2 = __float_as_uint(bound) >> 16 | __float_as_uint(bound);
  }
  // minus c of this thread's sum.  No logit above -infinity so far: one comes to `raise` before it is added, as it reaches the bound
  float minus_c = __int_as_float(top_s) > -INFINITY ? -rintf(__int_as_float(top_s) * BEAM_L) : 3e38f;
  auto raise = [&](float to) {
    if (!(to > 1.f - minus_c)) return;
    const float c = rintf(to), down = power_of_two(-minus_c - c);
    sum *= (double)down;
    minus_c = -c;
  };
  auto most_of = [](const uint4& v) { return max_bf16x2(max_bf16x2(v.x, v.y), max_bf16x2(v.z, v.w)); };
  auto collect = [&](const uint4& v, int c) {
    const int at = next_place(&n_vectors);
    if (at < BEAM_VECTORS) {
      vectors[at] = v;
      vector_at[at] = c;
    }
  };
  auto add = [&](f32x2 exps) {
    const float2 h = halves_of(exps);
    sum += (double)(h.x + h.y);
  };
  auto look = [&](const uint4& v, int c) {
    const uint32_t m = most_of(v);
    if (reaches_bf16x2(m, bound2)) {
      collect(v, c);
      raise(fmaxf(bf16_lo(m), bf16_hi(m)) * BEAM_L);
    }
    add(beam_exps(v, minus_c));
  };
  int c = v0 + tid;
  auto look_at_tile = [&]() {
    uint32_t m[BEAM_NV];
#pragma unroll
    for (int u = 0; u < BEAM_NV; ++u) m[u] = most_of(a[u]);
    const uint32_t top = max_bf16x2(max_bf16x2(m[0], m[1]), max_bf16x2(m[2], m[3]));
    if (reaches_bf16x2(top, bound2)) {  // (seldom)
#pragma unroll
      for (int u = 0; u < BEAM_NV; ++u)
        if (reaches_bf16x2(m[u], bound2)) collect(a[u], c + u * BEAM_THREADS);
      raise(fmaxf(bf16_lo(top), bf16_hi(top)) * BEAM_L);
    }
    add(add2(add2(beam_exps(a[0], minus_c), beam_exps(a[1], minus_c)), add2(beam_exps(a[2], minus_c), beam_exps(a[3], minus_c))));
  };
  // Whole tiles; what comes next is asked for as soon as a place is free.  Behind tiles 0, 1, 3, 7, ... it is looked at whether enough has been found for only the K best so far to matter from there on (the ranks cost the square of it).
  int kept = 0;
  bool overflow = false;
  auto settle = [&]() {
    const int k = prune(kept);
    overflow |= k < 0;
    if (!overflow) kept = k;
    if (overflow) {  // (whatever is found from here on does not matter, but for logits that c has to follow: the bf16 number below c's reach)
      const uint32_t b = __float_as_uint((1.f - minus_c) * (1.f / BEAM_L));
      bound = __uint_as_float((b + (b >> 31 ? 0xffffu : 0u)) & 0xffff0000u);
    } else {
      if (kept == K) bound = value_of(best[K - 1]);
      raise(bound * BEAM_L);  // (logits below the bound are not looked at: c is not below it)
    }
    bound2 = __float_as_uint(bound) >> 16 | __float_as_uint(bound);
  };
  int stage = 0;
  for (int t = 0, end = 1; t < whole; end *= 2) {
    for (; t < min(end, whole); ++t) {
      if constexpr (kAligned) {
        asm volatile("cp.async.wait_group %0;" ::"n"(BEAM_RING - 1) : "memory");
#pragma unroll
        for (int u = 0; u < BEAM_NV; ++u) a[u] = lds_v4(place + 16 * (stage * TILE + u * BEAM_THREADS));
        look_at_tile();
        ask(t + BEAM_RING, stage);
        stage = stage + 1 < BEAM_RING ? stage + 1 : 0;
        c += TILE;
      } else {
        look_at_tile();
#pragma unroll
        for (int u = 0; u < BEAM_NV; ++u, c += BEAM_THREADS)
          if (c + TILE < v1) a[u] = x(c + TILE);
      }
    }
    // (the count that a thread sees holds its own vectors, so that the last one to add any sees them all)
    if (t < whole && __syncthreads_or(*(volatile int*)&n_vectors > BEAM_MANY)) settle();
  }
  // what is behind the last whole tile
  if constexpr (kAligned) asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int u = 0; u < BEAM_NV; ++u, c += BEAM_THREADS)
    if (c < v1) look(kAligned ? lds_v4(place + 16 * (stage * TILE + u * BEAM_THREADS)) : a[u], c);
  settle();
  // the largest logit: where the sum would leave what 64 bits hold once more by differences to it; where a thread met NaN once more without
  float top = -INFINITY;
  if (!overflow) {
    if (kept > 0) top = value_of(best[0]);
  } else {
    uint32_t m = 0xff80ff80u;
    for (int c = v0 + tid; c < v1; c += BEAM_THREADS) m = max_bf16x2(m, most_of(x(c)));
    top = fmaxf(bf16_lo(m), bf16_hi(m));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((tid & 31) == 0) tops[tid >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < BEAM_THREADS / 32; ++w) top = fmaxf(top, tops[w]);
  }
  const bool far = fabsf(top) > 600.f;
  if (far || sum != sum) {
    sum = 0.0;
    for (int c = v0 + tid; c < v1; c += BEAM_THREADS) {
      const uint4 v = x(c);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      float part[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float y = k & 1 ? bf16_hi(w[k >> 1]) : bf16_lo(w[k >> 1]);
        if (y == y) part[k & 1] += far ? (y == top ? 1.f : expf(y - top)) : beam_ex2(fmaf(y, BEAM_L, minus_c));
      }
      sum += (double)(part[0] + part[1]);
    }
  }
  // (far below the largest logit, if there is one: 0)
  const double unit = far ? 1.0 : minus_c > 1000.f ? 0.0 : __hiloint2double((1023 - (int)minus_c) << 20, 0);
  double d = sum * unit;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
  if ((tid & 31) == 0) sums[tid >> 5] = d;
  __syncthreads();
  const long long out = row * n_pieces + piece;
  if (tid == 0) {
    double s = 0.0;
    for (int w = 0; w < BEAM_THREADS / 32; ++w) s += sums[w];
    const double low = (double)top * BEAM_LOW;  // (up to 8e-6)
    if (!far) s *= 1.0 + low * (1.0 + 0.5 * low);
    // s e^base; base +infinity: a logit is, -infinity: there are none
    piece_sums[out] = make_double2(far ? (double)top : 0.0, s);
  }
  int2* to = entries + out * K;
  auto tell = [&](int rank, uint64_t key) { to[rank] = make_int2(__float_as_int(value_of(key)), (int)(0xffffffffu - (uint32_t)key)); };
  // Too many reached the bound (logits in some order, a mask over the row's first part): tile by tile once more, each with a bound of its own, the
  // K-th of the threads' largest logits.  384 rows of 256000 logits whose first half is hidden: 178 us (one after the other, as below, 1160).
  if (overflow) {
    overflow = false;
    kept = 0;
    bound = __uint_as_float(0xff7f0000u);
    for (int from = v0; from < v1 && !overflow; from += TILE) {
      __syncthreads();
      uint32_t m = 0xff80ff80u;
#pragma unroll
      for (int u = 0; u < BEAM_NV; ++u) {
        a[u] = from + u * BEAM_THREADS + tid < v1 ? x(from + u * BEAM_THREADS + tid) : none;
        m = max_bf16x2(m, most_of(a[u]));
      }
      const float mine = fmaxf(bf16_lo(m), bf16_hi(m));
      tops[tid] = mine;
      if (tid == 0) n_found = n_vectors = 0;
      __syncthreads();
      int rank = 0;
#pragma unroll 16
      for (int i = 0; i < BEAM_THREADS; ++i) rank += tops[i] > mine || (tops[i] == mine && i < tid);
      if (rank == K - 1) bound_s = __float_as_int(mine);
      __syncthreads();
      bound = fmaxf(bound, __int_as_float(bound_s));
      bound2 = __float_as_uint(bound) >> 16 | __float_as_uint(bound);
#pragma unroll
      for (int u = 0; u < BEAM_NV; ++u)
        if (reaches_bf16x2(most_of(a[u]), bound2)) collect(a[u], from + u * BEAM_THREADS + tid);
      const int k = prune(kept);
      overflow = k < 0;
      kept = max(k, 0);
      if (kept == K) bound = value_of(best[K - 1]);
    }
  }
  if (!overflow) {
    if (tid < kept) tell(tid, best[tid]);
    // Fewer than K above -infinity: the first tokens at -infinity follow (NaN counts as that).  They are among the piece's first K.
    if (kept < K && tid < 32)
      for (int k0 = 0, at = kept; at < K; k0 += 32) {
        const long long token = 8LL * v0 + k0 + tid, end = min(8LL * v1, V);
        const bool low = k0 + tid < K && token < end && !(__bfloat162float(x.x[token]) > -INFINITY);
        const uint32_t votes = __ballot_sync(0xffffffffu, low || k0 >= K);  // (fewer than K tokens: none)
        const int place = at + __popc(votes & ((1u << tid) - 1u));
        if ((votes >> tid & 1u) && place < K) to[place] = make_int2((int)0xff800000u, low ? (int)token : -1);
        at += __popc(votes);
      }
    return;
  }
  // Hundreds of equal or ever larger logits: one after the other.
  uint64_t last = ~0ull;
  for (int k = 0; k < K; ++k) {
    uint64_t most = 0;
    for (int c = v0 + tid; c < v1; c += BEAM_THREADS) {
      const uint4 v = x(c);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint64_t key = ((uint64_t)beam_order(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu) << 32) | (0xffffffffu - (uint32_t)(8 * c + i));
        if (8LL * c + i < V && key < last && key > most) most = key;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = max(most, (uint64_t)__shfl_xor_sync(0xffffffffu, (unsigned long long)most, o));
    if ((tid & 31) == 0) best_s[tid >> 5] = most;
    __syncthreads();
    for (int w = 0; w < BEAM_THREADS / 32; ++w) most = max(most, best_s[w]);
    __syncthreads();
    if (tid == 0) {
      if (most)
        tell(k, most);
      else
        to[k] = make_int2((int)0xff800000u, -1);
    }
    last = most;  // (0: nothing is below it, so the rest is told to be none too)
  }
}

struct BeamArgs {
  const float* scores;
  const int32_t* stops;
  const int2* entries;
  const double2* piece_sums;  // of exponentials: y e^x
  float *cand_scores, *next_scores;
  int32_t *cand_tokens, *cand_rows, *next_tokens, *next_rows;
  int W, K, n_pieces, n_stops;
  long long V;
};
// unsigned 64-bit integers of the same order as the numbers (-0 is 0)
__device__ __forceinline__ uint64_t order_double(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

constexpr int MERGE_THREADS = 512, HEADS = 128, MERGE_KEYS = 2048, MERGE_OWN = MERGE_KEYS / MERGE_THREADS;
__global__ void __launch_bounds__(MERGE_THREADS) beam_groups_kernel(BeamArgs a) {
  follow_previous(a.scores, a.stops, a.entries, a.piece_sums, a.cand_scores, a.next_scores, a.cand_tokens, a.cand_rows, a.next_tokens, a.next_rows);
  const int tid = threadIdx.x, W = a.W, K = a.K;
  const long long group = blockIdx.x, row0 = group * W;
  const int lists = W * a.n_pieces, n = lists * K;
  __shared__ double shift[BEAM_MOST_W];  // score - log of the sum; -infinity: the row has no candidates
  __shared__ float score[BEAM_MOST_W];
  __shared__ uint64_t bound_s;
  __shared__ int n_found;
  constexpr int FOUND = 1024;
  __shared__ uint64_t found_key[FOUND];
  __shared__ int found_place[FOUND];  // place among the group's n entries
  __shared__ uint64_t heads[HEADS], keys[MERGE_KEYS];
  __shared__ double out_t[BEAM_MOST_K];
  __shared__ int out_token[BEAM_MOST_K], out_row[BEAM_MOST_K];
  const int2* entries = a.entries + row0 * a.n_pieces * K;
  const double2* piece_sums = a.piece_sums + row0 * a.n_pieces;
  const bool held = n <= MERGE_KEYS;  // every thread has its entries, asked for before the rows' logarithms are known
  int2 mine[MERGE_OWN];
#pragma unroll
  for (int i = 0; i < MERGE_OWN; ++i)
    if (held && i * MERGE_THREADS + tid < n) mine[i] = entries[i * MERGE_THREADS + tid];
  for (int w = tid >> 5; w < W; w += MERGE_THREADS / 32) {
    const int lane = tid & 31;
    const double s = (double)a.scores[row0 + w];
    // (up to 64 pieces are read once)
    const double2 none = make_double2(-INFINITY, 0.0);
    const double2 p0 = lane < a.n_pieces ? piece_sums[w * a.n_pieces + lane] : none,
                  p1 = lane + 32 < a.n_pieces ? piece_sums[w * a.n_pieces + lane + 32] : none;
    double top = fmax(p0.x, p1.x);
    for (int p = lane + 64; p < a.n_pieces; p += 32) top = fmax(top, piece_sums[w * a.n_pieces + p].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
    const bool finite = top > -INFINITY && top < INFINITY;
    auto part = [&](double2 v) { return v.x == top ? v.y : v.x > -INFINITY ? v.y * exp(v.x - top) : 0.0; };  // (mostly the same base: 0)
    double sum = finite ? part(p0) + part(p1) : 0.0;
    for (int p = lane + 64; p < a.n_pieces && finite; p += 32) sum += part(piece_sums[w * a.n_pieces + p]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) score[w] = a.scores[row0 + w];
    if (lane == 0) shift[w] = finite && s > -INFINITY && s < INFINITY ? s - (top + log(sum)) : -INFINITY;
  }
  if (tid == 0) {
    n_found = 0;
    bound_s = 0;
  }
  __syncthreads();
  // entry e at place i: its score; of rows without candidates the first list stands for tokens 0 .. K - 1 at -infinity
  auto score_of = [&](int2 e, int i, int& w, int& token) -> double {
    const int list = i / K;
    w = list / a.n_pieces;
    token = e.y;
    if (shift[w] == -INFINITY) token = list % a.n_pieces == 0 ? i % K : -1;
    const float x = __int_as_float(e.x);
    // (no token is more than certain)
    return shift[w] == -INFINITY || !(x > -INFINITY) ? -INFINITY : fmin(shift[w] + (double)x, (double)score[w]);
  };
  auto entry = [&](int i, int& w, int& token) { return score_of(entries[i], i, w, token); };
  auto key_of = [&](int2 e, int i) -> uint64_t {
    int w, token;
    const double t = score_of(e, i, w, token);
    return token >= 0 ? order_double(t) : 0;
  };
#pragma unroll
  for (int i = 0; i < MERGE_OWN; ++i)
    if (held && i * MERGE_THREADS + tid < n) keys[i * MERGE_THREADS + tid] = key_of(mine[i], i * MERGE_THREADS + tid);
  __syncthreads();
  // ---- a bound that K candidates reach: the K-th best of the first entries of each list, so many that they are up to 128 together; of more
  // lists, the K-th of the largest first entries of 128 classes of lists
  {
    const int deep = min(K, max(1, HEADS / lists)), heads_n = min(lists * deep, HEADS);
    uint64_t best = 0;
    if (tid < heads_n) {
      const int first = tid / deep * K + tid % deep, step = heads_n / deep * K;
      for (int i = first; i < n; i += step) best = max(best, held ? keys[i] : key_of(entries[i], i));
    }
    if (tid < HEADS) heads[tid] = best;
    __syncthreads();
    if (tid < heads_n) {
      int rank = 0;
#pragma unroll 8
      for (int i = 0; i < heads_n; ++i) rank += heads[i] > best || (heads[i] == best && i < tid);
      if (rank == min(K, heads_n) - 1) bound_s = best;
    }
    __syncthreads();
  }
  const uint64_t bound = max(bound_s, (uint64_t)1);
  for (int i = tid; i < n; i += MERGE_THREADS) {
    const uint64_t key = held ? keys[i] : key_of(entries[i], i);
    if (key >= bound) {
      const int at = next_place(&n_found);
      if (at < FOUND) {
        found_key[at] = key;
        found_place[at] = i;
      }
    }
  }
  __syncthreads();
  auto token_of = [&](int i, int& w) {
    int token;
    entry(i, w, token);
    return token;
  };
  // equal scores: the lower row, then the lower token
  auto before = [&](int i, int j) {
    int wi, wj;
    const int ti = token_of(i, wi), tj = token_of(j, wj);
    return wi != wj ? wi < wj : ti < tj;
  };
  if (n_found <= FOUND) {
    const int m = n_found;
    for (int i = tid; i < m; i += MERGE_THREADS) {
      const uint64_t key = found_key[i];
      int rank = 0;
      for (int k = 0; k < m; ++k) rank += found_key[k] > key || (found_key[k] == key && k != i && before(found_place[k], found_place[i]));
      if (rank < K) {
        int w, token;
        out_t[rank] = entry(found_place[i], w, token);
        out_token[rank] = token;
        out_row[rank] = w;
      }
    }
  } else {  // hundreds of equal scores: one after the other, each the best behind the one before
    __shared__ int best_s[MERGE_THREADS / 32];
    int last = -1;
    for (int k = 0; k < K; ++k) {
      int best = -1;
      auto better = [&](int i, int j) {  // entry i before entry j (-1: none)
        if (j < 0) return i >= 0;
        if (i < 0) return false;
        int w, token;
        const uint64_t x = order_double(entry(i, w, token)), y = order_double(entry(j, w, token));
        return x != y ? x > y : i != j && before(i, j);
      };
      for (int i = tid; i < n; i += MERGE_THREADS) {
        int w;
        if (token_of(i, w) >= 0 && (last < 0 || better(last, i)) && better(i, best)) best = i;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const int other = __shfl_xor_sync(0xffffffffu, best, o);
        if (better(other, best)) best = other;
      }
      if ((tid & 31) == 0) best_s[tid >> 5] = best;
      __syncthreads();
      for (int w = 0; w < MERGE_THREADS / 32; ++w)
        if (better(best_s[w], best)) best = best_s[w];
      __syncthreads();
      if (tid == 0) {
        int w, token;
        out_t[k] = entry(best, w, token);
        out_token[k] = token;
        out_row[k] = w;
      }
      last = best;
    }
  }
  __syncthreads();
  if (tid < K) {
    a.cand_scores[group * K + tid] = (float)out_t[tid];
    a.cand_tokens[group * K + tid] = out_token[tid];
    a.cand_rows[group * K + tid] = (int)(row0 + out_row[tid]);
  }
  // ---- the first W that go on (a warp finds them; candidates beyond the 32nd with its second round)
  if (tid < 32) {
    int kept = 0;
    for (int k0 = 0; k0 < K; k0 += 32) {
      const int k = k0 + tid;
      bool on = k < K;
      for (int s = 0; s < a.n_stops && on; ++s) on = a.stops[s] != out_token[k];
      const uint32_t votes = __ballot_sync(0xffffffffu, on);
      const int at = kept + __popc(votes & ((1u << tid) - 1u));
      if (on && at < W) {
        a.next_scores[row0 + at] = (float)out_t[k];
        a.next_tokens[row0 + at] = out_token[k];
        a.next_rows[row0 + at] = (int)(row0 + out_row[k]);
      }
      kept += __popc(votes);
    }
    for (int at = kept + tid; at < W; at += 32) {  // all others end here: beams that have no candidates from now on
      a.next_scores[row0 + at] = -INFINITY;
      a.next_tokens[row0 + at] = 0;
      a.next_rows[row0 + at] = (int)row0;
    }
  }
}

// Pieces of a row: the least time of the SM that has most CTAs, each its logits (five CTAs at once are as fast as an SM gets) and 11000 logits'
// worth beside them, and of the lists that the second kernel has to look at.  384 rows of 256000 logits: 1 / 2 / 3 / 4 / 6 / 8 pieces 71.3 /
// 56.2 / 54.6 / 57.8 / 64.6 / 67.2 us; 4 rows of 128256: 8 / 16 / 32 / 48 / 64 pieces 11.1 / 10.5 / 10.5 / 11.4 / 12.4 us.
// B200Q_BATCH_INVARIANT=1: as for 64 rows whatever their number, since a row's sum is that of its pieces' sums.
static int beam_pieces(long long rows, long long V) {
  if (batch_invariant()) rows = 64;
  int best = 1;
  double least = 1e30;
  for (int p = 1; p <= 256 && (p == 1 || V / p >= 2048); ++p) {
    const long long deep = (rows * p + 147) / 148;
    const double t = (double)(deep > 5 ? deep : 5) * ((double)V / p) + deep * 11000.0 + 500.0 * p;
    if (t < 0.98 * least) {
      least = t;
      best = p;
    }
  }
  return best;
}

}  // namespace b200q

using namespace b200q;

extern "C" {

int64_t b200q_beam_select_workspace(int groups, int beams, int64_t V, int K) {
  if (groups < 0 || beams <= 0 || beams > BEAM_MOST_W || V <= 0 || V > 0x7fffffff || K <= 0 || K > BEAM_MOST_K) {
    set_error("beam_select_workspace: bad shape groups=%d beams=%d (up to %d) V=%lld K=%d (up to %d)", groups, beams, BEAM_MOST_W, (long long)V, K,
              BEAM_MOST_K);
    return B200Q_EINVAL;
  }
  const int64_t pieces = (int64_t)groups * beams * beam_pieces((int64_t)groups * beams, V);
  return pieces * (int64_t)(sizeof(double2) + K * sizeof(int2));
}

int b200q_beam_select(const void* logits, const float* scores, int groups, int beams, int64_t V, const int32_t* stops, int n_stops, int K,
                      float* cand_scores, int32_t* cand_tokens, int32_t* cand_rows, float* next_scores, int32_t* next_tokens, int32_t* next_rows,
                      void* workspace, int64_t workspace_bytes, void* stream) {
  B200Q_CHECK_ARG(groups >= 0 && beams > 0 && beams <= BEAM_MOST_W && K >= beams && K <= BEAM_MOST_K && V >= K && V <= 0x7fffffff - 64 && n_stops >= 0,
                  "beam_select: bad shape groups=%d beams=%d (up to %d) V=%lld K=%d (from beams to %d and V) n_stops=%d", groups, beams, BEAM_MOST_W,
                  (long long)V, K, BEAM_MOST_K, n_stops);
  if (groups == 0) return B200Q_OK;
  const int64_t rows = (int64_t)groups * beams;
  B200Q_CHECK_ARG(rows <= 0x7fffffff, "beam_select: too many rows (%lld)", (long long)rows);
  B200Q_CHECK_ARG(logits && scores && (stops || n_stops == 0) && cand_scores && cand_tokens && cand_rows && next_scores && next_tokens && next_rows &&
                      workspace,
                  "beam_select: null argument");
  const int64_t need = b200q_beam_select_workspace(groups, beams, V, K);
  B200Q_CHECK_ARG(workspace_bytes >= need, "beam_select: workspace too small: %lld < %lld", (long long)workspace_bytes, (long long)need);
  B200Q_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 15) == 0 && (reinterpret_cast<uintptr_t>(logits) & 15) == 0,
                  "beam_select: logits and workspace must be 16-byte aligned");
  const int pieces = beam_pieces(rows, V);
  double2* piece_sums = (double2*)workspace;
  int2* entries = (int2*)(piece_sums + rows * pieces);
  cudaStream_t st = as_stream(stream);
  for (int64_t r0 = 0; r0 < rows; r0 += 65535) {  // (a grid's second dimension ends there)
    const unsigned n = (unsigned)(rows - r0 < 65535 ? rows - r0 : 65535);
    auto kern = V % 8 ? beam_rows_kernel<false> : beam_rows_kernel<true>;
    B200Q_CUDA(launch_early(kern, dim3(pieces, n), BEAM_THREADS, V % 8 ? 0 : BEAM_RING * TILE * 16, st, 1, (const bf16*)logits, (long long)V, K, (long long)r0, (long long)rows, entries, piece_sums));
    count_launch();
  }
  const BeamArgs a{scores, stops, entries, piece_sums, cand_scores, next_scores, cand_tokens, cand_rows, next_tokens, next_rows, beams, K, pieces, n_stops,
                   (long long)V};
  B200Q_CUDA(launch_early(beam_groups_kernel, dim3(groups), MERGE_THREADS, 0, st, 1, a));
  count_launch();
  return B200Q_OK;
}

}  // extern "C"
