// beam.cu — the best continuations of beams: for every group of W rows of logits, of t(w, v) = score_w + logit_wv - log sum_v exp(logit_wv)
// the K largest of W V, of equal ones those with the lowest w V + v first; and the first W of them that do not end.
//
// Two kernels.  The first has a piece of a row per CTA, in registers: its maximum, the sum of its exponentials and its K best logits (a row's
// order needs no logarithm).  The largest logit of each pair of threads gives a bound that K of the piece reach; what reaches it, K or a
// few more, is ranked by counting.  The second has a group per CTA: sums to logarithms, best logits to scores, and again a bound (the K-th
// best of the pieces' first entries), what reaches it, and ranks.
// Scores that are compared across rows are 64 bits, and a row's sum of exponentials keeps about 2^-26: rows whose candidates are that close
// would come in an order of rounding errors otherwise.
// Bound: the logits, 2 bytes each, once; next to it the exponentials, some nine instructions a logit.
#include "common.cuh"

namespace b200q {

constexpr int BEAM_THREADS = 256, BEAM_PAIRS = BEAM_THREADS / 2, BEAM_MOST_K = 64, BEAM_MOST_W = 32, BEAM_FOUND = 512;

// what a piece tells the second kernel: beside `entries` [K] {logit as fp32 bits, token; -1: there is none}
struct BeamPiece {
  double sum;
  float top;
  int pad;
};

__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// unsigned integers of the same order as the numbers (bf16 bits); NaN counts as -infinity
__device__ __forceinline__ uint32_t beam_order(uint32_t h) {
  if ((h & 0x7fffu) > 0x7f80u) h = 0xff80u;
  return (h & 0x8000u) ? 0xffffu ^ h : h | 0x8000u;
}
// e^d for d <= 0 (0 below e^-160, and for NaN): the product with log2(e) in two parts, so that the exponent's rounding does not show
__device__ __forceinline__ float beam_exp(float d) {
  d = fmaxf(d, -160.f);
  const float hi = d * 1.44269504088896341f;
  const float lo = fmaf(d, 1.44269504088896341f, -hi) + d * 1.925963033500e-8f;  // log2(e) - float(log2(e)) = 1.926e-8
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(hi));
  return fmaf(e, lo * 0.693147180559945309f, e);
}

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

// NV: vectors per thread; a piece is up to 8 * NV * 256 logits
template <int NV, bool kAligned>
__global__ void __launch_bounds__(BEAM_THREADS, NV == 8 ? 3 : 4) beam_rows_kernel(const bf16* logits, long long V, int K, long long row0, long long rows,
                                                                                  int2* entries, BeamPiece* pieces) {
  follow_previous(logits, entries, pieces);
  const int tid = threadIdx.x, piece = blockIdx.x, n_pieces = gridDim.x;
  const long long row = row0 + blockIdx.y;
  const BeamRow<kAligned> x(logits, V, row, rows);
  const int vecs = (int)((V + 7) / 8), per = (vecs + n_pieces - 1) / n_pieces, v0 = min(vecs, piece * per), v1 = min(vecs, v0 + per);
  const uint4 none = make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
  uint4 a[NV];
#pragma unroll
  for (int u = 0; u < NV; ++u) a[u] = v0 + u * BEAM_THREADS + tid < v1 ? x(v0 + u * BEAM_THREADS + tid) : none;

  __shared__ float tops[BEAM_PAIRS];
  __shared__ uint64_t found[BEAM_FOUND];
  __shared__ double sums[BEAM_THREADS / 32];
  __shared__ int n_found, bound_s;
  __shared__ float top_s;
  __shared__ uint64_t best_s[BEAM_THREADS / 32];
  uint32_t m2 = 0xff80ff80u;
#pragma unroll
  for (int u = 0; u < NV; ++u) m2 = max_bf16x2(m2, max_bf16x2(max_bf16x2(a[u].x, a[u].y), max_bf16x2(a[u].z, a[u].w)));
  float mine = fmaxf(bf16_lo(m2), bf16_hi(m2));  // (max of a number and NaN is the number; -infinity was among them)
  mine = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, 1));
  if ((tid & 1) == 0) tops[tid >> 1] = mine;
  if (tid == 0) n_found = 0;
  __syncthreads();
  if (tid < BEAM_PAIRS) {  // the K-th of the pairs' maxima, and the first
    const float t = tops[tid];
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < BEAM_PAIRS; ++i) rank += tops[i] > t || (tops[i] == t && i < tid);
    if (rank == 0) top_s = t;
    if (rank == K - 1) bound_s = __float_as_int(t);
  }
  __syncthreads();
  const float top = top_s, bound = __int_as_float(bound_s);
  // ---- the sum, and what reaches the bound
  float sum = 0.f;
  const bool finite = top > -INFINITY && top < INFINITY;
  uint32_t reached = 0;  // bit u: vector u has a logit that reaches the bound
  auto keep = [&](uint32_t h, int token) {
    const int at = atomicAdd(&n_found, 1);
    if (at < BEAM_FOUND) found[at] = ((uint64_t)beam_order(h) << 32) | (0xffffffffu - (uint32_t)token);
  };
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const uint32_t w[4] = {a[u].x, a[u].y, a[u].z, a[u].w};
    bool any = false;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      any |= bf16_lo(w[k]) >= bound || bf16_hi(w[k]) >= bound;
      sum += beam_exp(bf16_lo(w[k]) - top);
      sum += beam_exp(bf16_hi(w[k]) - top);
    }
    reached |= any ? 1u << u : 0u;
  }
  // (seldom: the vector once more, so that this is no code for every register)
  for (; reached; reached &= reached - 1) {
    const int c = v0 + (__ffs(reached) - 1) * BEAM_THREADS + tid;
    if (c >= v1) break;
    const uint4 v = x(c);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t h = k & 1 ? w[k >> 1] >> 16 : w[k >> 1] & 0xffffu;
      if (__uint_as_float(h << 16) >= bound && 8LL * c + k < V) keep(h, 8 * c + k);
    }
  }
  double d = finite ? (double)sum : 0.0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
  if ((tid & 31) == 0) sums[tid >> 5] = d;
  __syncthreads();
  const long long out = row * n_pieces + piece;
  if (tid == 0) {
    double s = 0.0;
    for (int w = 0; w < BEAM_THREADS / 32; ++w) s += sums[w];
    pieces[out] = {s, top, 0};
  }
  int2* to = entries + out * K;
  const int n = n_found;
  auto tell = [&](int rank, uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32), h = (o & 0x8000u) ? o & 0x7fffu : 0xffffu ^ o;
    to[rank] = make_int2((int)(h << 16), (int)(0xffffffffu - (uint32_t)key));
  };
  if (bound > -INFINITY && n <= BEAM_FOUND) {  // (K and more reach the bound; the keys are all different)
    for (int i = tid; i < n; i += BEAM_THREADS) {
      const uint64_t key = found[i];
      int rank = 0;
      for (int k = 0; k < n; ++k) rank += found[k] > key;
      if (rank < K) tell(rank, key);
    }
    return;
  }
  // Fewer than K pairs with a number above -infinity, or hundreds of equal logits: one after the other.
  uint64_t last = ~0ull;
  for (int k = 0; k < K; ++k) {
    uint64_t best = 0;
    auto look = [&](uint32_t h, int token) {
      const uint64_t key = ((uint64_t)beam_order(h) << 32) | (0xffffffffu - (uint32_t)token);
      if (key < last && key > best) best = key;
    };
    for (int c = v0 + tid; c < v1; c += BEAM_THREADS) {
      const uint4 v = x(c);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (8LL * c + i < V) look(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu, 8 * c + i);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, (uint64_t)__shfl_xor_sync(0xffffffffu, (unsigned long long)best, o));
    if ((tid & 31) == 0) best_s[tid >> 5] = best;
    __syncthreads();
    for (int w = 0; w < BEAM_THREADS / 32; ++w) best = max(best, best_s[w]);
    __syncthreads();
    if (tid == 0) {
      if (best)
        tell(k, best);
      else
        to[k] = make_int2((int)0xff800000u, -1);
    }
    last = best;  // (0: nothing is below it, so the rest is told to be none too)
  }
}

struct BeamArgs {
  const float* scores;
  const int32_t* stops;
  const int2* entries;
  const BeamPiece* pieces;
  float *cand_scores, *next_scores;
  int32_t *cand_tokens, *cand_rows, *next_tokens, *next_rows;
  int W, K, n_pieces, n_stops;
  long long V;
};
// unsigned 64-bit integers of the same order as the numbers
__device__ __forceinline__ uint64_t order_double(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v);
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

constexpr int MERGE_THREADS = 512, HEADS = 256;
__global__ void __launch_bounds__(MERGE_THREADS) beam_groups_kernel(BeamArgs a) {
  follow_previous(a.scores, a.stops, a.entries, a.pieces, a.cand_scores, a.next_scores, a.cand_tokens, a.cand_rows, a.next_tokens, a.next_rows);
  const int tid = threadIdx.x, W = a.W, K = a.K;
  const long long group = blockIdx.x, row0 = group * W;
  const int lists = W * a.n_pieces, n = lists * K;
  __shared__ double shift[BEAM_MOST_W];  // score - log of the sum; -infinity: the row has no candidates
  __shared__ uint64_t bound_s;
  __shared__ int n_found;
  constexpr int FOUND = 1024;
  __shared__ uint64_t found_key[FOUND];
  __shared__ int found_place[FOUND];  // place among the group's n entries
  __shared__ uint64_t heads[HEADS];
  __shared__ double out_t[BEAM_MOST_K];
  __shared__ int out_token[BEAM_MOST_K], out_row[BEAM_MOST_K];
  const int2* entries = a.entries + row0 * a.n_pieces * K;
  const BeamPiece* pieces = a.pieces + row0 * a.n_pieces;
  for (int w = tid >> 5; w < W; w += MERGE_THREADS / 32) {
    const int lane = tid & 31;
    float top = -INFINITY;
    for (int p = lane; p < a.n_pieces; p += 32) top = fmaxf(top, pieces[w * a.n_pieces + p].top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    double sum = 0.0;
    const bool finite = top > -INFINITY && top < INFINITY;
    for (int p = lane; p < a.n_pieces && finite; p += 32) {
      const BeamPiece b = pieces[w * a.n_pieces + p];
      if (b.top > -INFINITY) sum += b.sum * exp((double)b.top - (double)top);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      const double s = (double)a.scores[row0 + w];
      const double t = finite && s > -INFINITY && s < INFINITY ? s - ((double)top + log(sum)) : -INFINITY;
      shift[w] = t;
    }
  }
  if (tid == 0) {
    n_found = 0;
    bound_s = 0;
  }
  __syncthreads();
  // an entry's score; of rows without candidates the first list stands for tokens 0 .. K - 1 at -infinity
  auto entry = [&](int i, int& w, int& token) -> double {
    const int list = i / K;
    w = list / a.n_pieces;
    const int2 e = entries[i];
    token = e.y;
    if (shift[w] == -INFINITY) token = list % a.n_pieces == 0 ? i % K : -1;
    const float x = __int_as_float(e.x);
    return shift[w] == -INFINITY || !(x > -INFINITY) ? -INFINITY : shift[w] + (double)x;
  };
  // ---- a bound that K candidates reach.  Of K lists and more: the K-th of the largest first entries of up to 256 classes of lists; of
  // fewer: the least of the entries that are K together.
  {
    const int classes = min(lists, HEADS), deep = lists >= K ? 0 : (K + lists - 1) / lists - 1;
    uint64_t mine = 0;
    if (tid < classes)
      for (int l = tid; l < lists; l += classes) {
        int w, token;
        const double t = entry(l * K + deep, w, token);
        mine = max(mine, token >= 0 ? order_double(t) : 0);
      }
    if (tid < HEADS) heads[tid] = mine;
    __syncthreads();
    if (tid < classes) {
      int rank = 0;
      for (int i = 0; i < classes; ++i) rank += heads[i] > mine || (heads[i] == mine && i < tid);
      if (rank == min(K, classes) - 1) bound_s = mine;
    }
    __syncthreads();
  }
  const uint64_t bound = bound_s;
  for (int i = tid; i < n; i += MERGE_THREADS) {
    int w, token;
    const double t = entry(i, w, token);
    if (token >= 0 && order_double(t) >= bound) {
      const int at = atomicAdd(&n_found, 1);
      if (at < FOUND) {
        found_key[at] = order_double(t);
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

// Pieces of a row: of 16384 logits where the rows alone fill the chip, else of 4096
static int beam_vectors(long long rows, long long V) { return rows * ((V + 16383) / 16384) >= 2 * 148 ? 8 : 2; }
static int beam_pieces(long long rows, long long V) {
  const long long most = beam_vectors(rows, V) * 8LL * BEAM_THREADS;
  return (int)((V + most - 1) / most);
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
  return pieces * (int64_t)(sizeof(BeamPiece) + K * sizeof(int2));
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
  BeamPiece* piece = (BeamPiece*)workspace;
  int2* entries = (int2*)(piece + rows * pieces);
  cudaStream_t st = as_stream(stream);
  for (int64_t r0 = 0; r0 < rows; r0 += 65535) {  // (a grid's second dimension ends there)
    const unsigned n = (unsigned)(rows - r0 < 65535 ? rows - r0 : 65535);
    const bool wide = beam_vectors(rows, V) == 8;
    auto kern = V % 8 ? (wide ? beam_rows_kernel<8, false> : beam_rows_kernel<2, false>) : wide ? beam_rows_kernel<8, true> : beam_rows_kernel<2, true>;
    B200Q_CUDA(launch_early(kern, dim3(pieces, n), BEAM_THREADS, 0, st, 1, (const bf16*)logits, (long long)V, K, (long long)r0, (long long)rows, entries, piece));
    count_launch();
  }
  const BeamArgs a{scores, stops, entries, piece, cand_scores, next_scores, cand_tokens, cand_rows, next_tokens, next_rows, beams, K, pieces, n_stops,
                   (long long)V};
  B200Q_CUDA(launch_early(beam_groups_kernel, dim3(groups), MERGE_THREADS, 0, st, 1, a));
  count_launch();
  return B200Q_OK;
}

}  // extern "C"
