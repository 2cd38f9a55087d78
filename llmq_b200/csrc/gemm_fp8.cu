// gemm_fp8.cu — C[m,n] = sum_b as[b,m] ws[n/128,b] sum_{k in block b} A[m,k] W[n,k]: products of e4m3 codes with a scale for each block of 128 of
// the reduction (fp8.cuh), fp32 sums; dense, gated (the unit's values leave in 8 bits again) and by expert.
//
// A block of 128 codes is one swizzle span, one stage of the ring and four tcgen05.mma (kind::f8f6f4, 32 codes each) whose fp32 sums start from
// zero; the block's scales are then multiplied in while the sums leave tensor memory for the registers that hold the running total ("promoted").
// Two accumulators in tensor memory let the tensor core work on block b + 1 meanwhile.  Bounds: the weight stream (N K bytes) for few rows; for many
// the tensor core at twice the bf16 rate, and, close behind it, the promotion, which reads 4 bytes of tensor memory and does one multiply-add
// for every 128 products.
//
//   * large: rows of A are the tensor core's M side (a lane has a row, so that its scale is one number to a thread), 256 columns to a CTA, eight
//     warps that promote 128 columns each in 128 registers a thread.  Persistent.  One CTA to 128 rows, or a pair (cta_group::2) to 256, each of
//     which fetches half of the weights.
//   * small, up to 128 rows to a tile: the weights are the M side and the rows, padded to 16, the N side; the reduction is split over a
//     cluster whose partial sums meet in distributed shared memory in the order of the splits.
#include <type_traits>

#include "fp8.cuh"
#include "tcgen05.cuh"

namespace b200q {

constexpr int F8_STAGE_W = 128 * FP8_BLOCK;  // bytes of 128 rows of one block

struct Fp8Args {
  const float* as;   // [blocks][ld_as]
  const float* ws;   // [groups][n_blocks][blocks]
  void* C;           // bf16 or fp32 [M][N], or codes [M][N / 2]
  float* ys;         // [N / 256][ld_ys], gated
  const int4* tab;   // [*n_mt] {group, first row, end of its rows, 0}, or NULL: the rows are one group
  const int32_t* n_mt;
  int* failed;
  int ld_as, ld_ys, M, N, K, blocks, n_blocks, max_mt, groups, out_f32, gelu;
  // small tiles
  int rows, box_rows, stages, cols, splits;
};

__device__ __forceinline__ void umma_fp8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
      "}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(add)
      : "memory");
}
__device__ __forceinline__ void umma_fp8_2sm(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
      "}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(add)
      : "memory");
}
// D = f32, A = B = e4m3, both K-major
__host__ __device__ constexpr uint32_t fp8_idesc(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }
// the loads into v have come (tied to v, so that nothing reads it before)
__device__ __forceinline__ void tmem_ld_wait_for(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]),
                 "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]),
                 "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]),
                 "+r"(v[31])::"memory");
}
__device__ __forceinline__ void f8_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void f8_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cluster.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void f8_load_2sm(void* to, const void* tmap, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(to)),
      "l"(tmap), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void f8_store(const void* tmap, int c0, int c1, uint32_t from) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(tmap), "r"(c0), "r"(c1), "r"(from) : "memory");
}
__device__ __forceinline__ void f8_commit_2sm(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
               "h"((uint16_t)3)
               : "memory");
}
// the unit of a gate and what it gates, fp32 from the sums on: g sigmoid(g) u, or tanh GELU, 0.5 g (1 + tanh t) = g sigmoid(2 t)
__device__ __forceinline__ float fp8_unit(float g, float u, int gelu) {
  const float t = gelu ? 1.5957691216057308f * (g + 0.044715f * (g * g * g)) : g;
  return __fdividef(g, 1.f + __expf(-t)) * u;
}
// (dead: another role of the CTA has given up; flag and clock are looked at every 64 tries)
__device__ __forceinline__ void f8_wait(uint64_t* bar, uint32_t parity, volatile int* dead, int* failed) {
  long long t0 = 0;
  for (int n = 0; !mbar_try_wait(bar, parity); ++n) {
    if (n % 64 != 63) continue;
    if (n == 63) t0 = clock64();
    if (*dead) return;
    if (clock64() - t0 > WAIT_CYCLES) {
      *dead = 1;
      __threadfence_block();
      *(volatile int*)failed = 1;
      return;
    }
  }
}
// copies in flight end before a block that gave up returns its memory
__device__ __noinline__ void f8_let_copies_end() {
  const long long t0 = clock64();
  while (clock64() - t0 < 4000000ll) {
  }
  __syncthreads();
}

// ---- large ---------------------------------------------------------------------------------------------------------------------
constexpr int FL_THREADS = 384, FL_BN = 256, FL_PATCH = 4096;
// registers: 384 threads begin with 168; four warps give back 128 each and eight take 64 more (40 x 128 + 232 x 256 = 168 x 384)
constexpr int FL_REGS_FEW = 40, FL_REGS_MANY = 232;
// The products of a block are two to 128 columns, whose accumulators are filled and emptied on their own: a half's next product waits for four
// warps and not for eight, and the tensor core has the other half's to do meanwhile.  Rows of W come in boxes, so that the columns of a half
// are 128 neighbours, or (gated) 64 gates and the 64 that they gate; of a pair each CTA has 64 of them.
template <bool PAIR, bool GATED>
struct LargeCfg {
  static constexpr int STAGE = F8_STAGE_W + (PAIR ? F8_STAGE_W : 2 * F8_STAGE_W);  // 128 rows of A, 256 (the pair: 128) of W
  static constexpr int STAGES = PAIR ? 6 : 4;
  static constexpr int BOX = PAIR || GATED ? 64 : 256, BOXES = (PAIR ? 128 : 256) / BOX;  // rows of W, boxes of a stage
  static constexpr int SMEM = STAGES * STAGE + 8 * FL_PATCH + 1024;
};

// 64 sums to a thread (its row, columns in turn) += scale * 32 of them that have come from tensor memory
__device__ __forceinline__ void promote(f32x2* acc, const uint32_t (&v)[32], f32x2 scale) {
#pragma unroll
  for (int j = 0; j < 16; ++j) acc[j] = fma2(pair_of(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), scale, acc[j]);
}

template <bool PAIR, bool GATED, bool GROUPED>
__global__ void __launch_bounds__(FL_THREADS, 1)
    gemm_fp8_large_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                          const __grid_constant__ CUtensorMap tmap_c, const __grid_constant__ Fp8Args a) {
  using Cfg = LargeCfg<PAIR, GATED>;
  constexpr int STAGES = Cfg::STAGES, BM = PAIR ? 256 : 128;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* patches = smem + STAGES * Cfg::STAGE;
  __shared__ __align__(8) uint64_t full[STAGES], empty[STAGES], acc_full[2][2], acc_empty[2][2];  // of accumulators: [half of the columns][turn]
  __shared__ uint32_t tmem_slot;
  __shared__ int dead;
  __shared__ float most[2][128];  // gated: the largest of a half row's 64 values
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = PAIR ? (int)cluster_ctarank() : 0;
  const int unit = PAIR ? blockIdx.x >> 1 : blockIdx.x, units = PAIR ? gridDim.x >> 1 : gridDim.x;
  const int n_tiles = (a.N + FL_BN - 1) / FL_BN, blocks = a.blocks;
  // the i-th box of a stage begins so many rows of W behind the tile's first
  auto w_box = [&](int i) { return PAIR ? (GATED ? rank * 128 + i * 64 : i * 128 + rank * 64) : GATED ? (i & 1) * 128 + (i >> 1) * 64 : 0; };

  if (warp == 0 && lane == 0) {
    dead = 0;
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_w);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full + s, PAIR ? 2 : 1);
      mbar_init(empty + s, 2);  // both halves' products
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(acc_full[s >> 1] + (s & 1), 1);
      mbar_init(acc_empty[s >> 1] + (s & 1), PAIR ? 8 : 4);  // (the leader's) the warps that promote
    }
    mbar_fence_init();
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_slot)) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      tmem_alloc(&tmem_slot, 512);
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
  if (!GROUPED && warp == 0 && lane == 0) {  // the first weights into L2 while the kernel before this one ends
    const int m_tiles = (a.M + BM - 1) / BM, n0 = unit / m_tiles * FL_BN;
    for (int b = 0; b < min(STAGES, blocks); ++b)
      for (int i = 0; i < Cfg::BOXES; ++i) tma_prefetch_2d(&tmap_w, b * 64, n0 + w_box(i));
  }
  __syncwarp();
  const float *as = a.as, *ws = a.ws;
  const int4* tab = a.tab;
  const int32_t* n_mt = a.n_mt;
  follow_previous(as, ws, tab, n_mt);
  const int m_tiles = GROUPED ? min(*n_mt, a.max_mt) : (a.M + BM - 1) / BM;
  const int num_tiles = m_tiles * n_tiles;
  // a tile: columns n0 .., rows row0 .. row_end of a group
  auto tile_of = [&](int tile, int& g, int& row0, int& row_end, int& n0) {
    const int mt = tile % m_tiles;
    n0 = tile / m_tiles * FL_BN;
    if constexpr (GROUPED) {
      const int4 e = tab[mt];  // (kept within the matrices, whatever the table says)
      g = min(max(e.x, 0), a.groups - 1);
      row0 = max(e.y, 0);
      row_end = min(e.z, a.M);
    } else {
      g = 0;
      row0 = mt * BM + rank * 128;
      row_end = a.M;
    }
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(FL_REGS_FEW));
    if (warp == 0) {
      if (lane == 0) {
        int stage = 0;
        uint32_t phase = 0;
        for (int tile = unit; tile < num_tiles; tile += units) {
          int g, row0, row_end, n0;
          tile_of(tile, g, row0, row_end, n0);
          const int wrow = g * a.N + n0;
          for (int b = 0; b < blocks; ++b) {
            uint8_t* to = smem + stage * Cfg::STAGE;
            f8_wait(empty + stage, phase ^ 1u, &dead, a.failed);
            if constexpr (PAIR) {
              const uint32_t bar = mapa_shared(full + stage, 0);
              f8_expect_tx(bar, Cfg::STAGE);
#pragma unroll
              for (int i = 0; i < Cfg::BOXES; ++i) f8_load_2sm(to + F8_STAGE_W + i * Cfg::BOX * 128, &tmap_w, b * 64, wrow + w_box(i), bar);
              f8_load_2sm(to, &tmap_a, b * 64, row0, bar);
            } else {
              mbar_expect_tx(full + stage, Cfg::STAGE);
#pragma unroll
              for (int i = 0; i < Cfg::BOXES; ++i) tma_load_2d(to + F8_STAGE_W + i * Cfg::BOX * 128, &tmap_w, b * 64, wrow + w_box(i), full + stage);
              tma_load_2d(to, &tmap_a, b * 64, row0, full + stage);
            }
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (*(volatile int*)&dead) break;
        }
      }
      __syncwarp();
    } else if (warp < 3 && rank == 0) {  // a warp to the products of each half
      const int h = warp - 1;
      constexpr uint32_t idesc = fp8_idesc(BM, 128);
      const uint32_t ring = __shfl_sync(0xffffffffu, smem_u32(smem), 0);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      if (elect_one())
        for (int tile = unit; tile < num_tiles; tile += units) {
          for (int b = 0; b < blocks; ++b) {
            f8_wait(full + stage, phase, &dead, a.failed);
            f8_wait(acc_empty[h] + acc, acc_phase ^ 1u, &dead, a.failed);
            tc_fence_after();
            const uint32_t sa = ring + (uint32_t)(stage * Cfg::STAGE), sw = sa + F8_STAGE_W + h * (PAIR ? 64 : 128) * 128;
            const uint32_t d = tmem + (uint32_t)(acc * FL_BN + h * 128);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if constexpr (PAIR)
                umma_fp8_2sm(d, make_smem_desc(sa + k * 32), make_smem_desc(sw + k * 32), idesc, k > 0);
              else
                umma_fp8(d, make_smem_desc(sa + k * 32), make_smem_desc(sw + k * 32), idesc, k > 0);
            }
            if constexpr (PAIR) {
              f8_commit_2sm(acc_full[h] + acc);
              f8_commit_2sm(empty + stage);
            } else {
              umma_commit(acc_full[h] + acc);
              umma_commit(empty + stage);
            }
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
            acc ^= 1;
            if (acc == 0) acc_phase ^= 1u;
          }
          if (*(volatile int*)&dead) break;
        }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(FL_REGS_MANY));
    // rows quarter * 32 + lane; columns: plain half * 128 + 0 .. 127, gated half * 64 + 0 .. 63 of the gates and of what they gate
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * 128);
    uint8_t* const patch = patches + (warp - 4) * FL_PATCH;
    const uint32_t patch_s = smem_u32(patch);
    const uint32_t empty0 = PAIR ? mapa_shared(acc_empty[half], 0) : smem_u32(acc_empty[half]);
    int acc = 0, parity = 0;
    uint32_t acc_phase = 0;
    for (int tile = unit; tile < num_tiles; tile += units) {
      int g, row0, row_end, n0;
      tile_of(tile, g, row0, row_end, n0);
      const int row = row0 + quarter * 32 + lane;
      const bool live = row < row_end;
      // weights' scales: this lane's of 32 blocks, handed round by shuffles; gated: of the gates and of what they gate
      const int nb0 = GATED ? n0 / 128 : min(n0 / 128 + half, a.n_blocks - 1);
      const float* w0 = ws + ((long long)g * a.n_blocks + nb0) * blocks;
      float sw[2] = {0.f, 0.f}, sa[4], sa_next[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) sa_next[i] = live && i < blocks ? as[(long long)i * a.ld_as + row] : 0.f;
      f32x2 sum[4][16];
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int j = 0; j < 16; ++j) sum[c][j] = 0ull;
      uint32_t v[2][32];
      f8_wait(acc_full[half] + acc, acc_phase, &dead, a.failed);
      __syncwarp();
      tc_fence_after();
      tmem_ld32(lanes + (uint32_t)(acc * FL_BN), v[0]);
      for (int b0 = 0; b0 < blocks; b0 += 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sa[i] = sa_next[i];
          sa_next[i] = live && b0 + 4 + i < blocks ? as[(long long)(b0 + 4 + i) * a.ld_as + row] : 0.f;
        }
        if (b0 % 32 == 0 && b0 + lane < blocks) {
          sw[0] = w0[b0 + lane];
          if constexpr (GATED) sw[1] = w0[blocks + b0 + lane];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (b0 + i < blocks) {
            f32x2 s[2];
#pragma unroll
            for (int h = 0; h < (GATED ? 2 : 1); ++h) {
              const float x = sa[i] * __shfl_sync(0xffffffffu, sw[h], (b0 + i) & 31);
              s[h] = pair_of(x, x);
            }
            const uint32_t from = lanes + (uint32_t)(acc * FL_BN);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              tmem_ld_wait_for(v[c & 1]);
              if (c < 3) {
                tmem_ld32(from + (uint32_t)(c * 32 + 32), v[(c + 1) & 1]);
              } else {  // the accumulator is free; the next one's first columns while the last of this are added
                tc_fence_before();
                __syncwarp();
                if (lane == 0) f8_arrive(empty0 + acc * 8);
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1u;
                if (b0 + i + 1 < blocks) {
                  f8_wait(acc_full[half] + acc, acc_phase, &dead, a.failed);
                  __syncwarp();
                  tc_fence_after();
                  tmem_ld32(lanes + (uint32_t)(acc * FL_BN), v[0]);
                }
              }
              promote(sum[c], v[c & 1], s[GATED ? c >> 1 : 0]);
            }
          }
        }
      }
      // ---- the sums leave ----
      if constexpr (GATED) {
        float y[64];
        float m = 0.f;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float2 gate = halves_of(sum[c][j]), up = halves_of(sum[c + 2][j]);
            y[c * 32 + 2 * j] = fp8_unit(gate.x, up.x, a.gelu);
            y[c * 32 + 2 * j + 1] = fp8_unit(gate.y, up.y, a.gelu);
          }
#pragma unroll
        for (int j = 0; j < 64; ++j) m = max_or_nan(m, fabsf(y[j]));
        most[half][quarter * 32 + lane] = m;
        // (two warps share a quarter's rows, and a patch of 32 rows x 128 codes for each parity of the tile)
        uint8_t* const out = patches + (2 * quarter + parity) * FL_PATCH;
        const bool copies = !GROUPED && half == 0 && lane == 0;
        if (copies) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
        asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
        const float scale = fp8_scale(max_or_nan(m, most[half ^ 1][quarter * 32 + lane])), by = fp8_inverse(scale);
        if (half == 0 && live) a.ys[(long long)(n0 / 256) * a.ld_ys + row] = scale;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float* f = y + 16 * j + 4 * i;
            w[i] = fp8_four(f[0] * by, f[1] * by, f[2] * by, f[3] * by);
          }
          st_v4(out + lane * 128 + (((half * 4 + j) ^ (lane & 7)) << 4), make_uint4(w[0], w[1], w[2], w[3]));
        }
        if constexpr (!GROUPED) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
        if (copies) {  // (rows that do not exist leave an empty group, as the wait counts turns)
          if (row0 + quarter * 32 < a.M) f8_store(&tmap_c, n0 / 4, row0 + quarter * 32, smem_u32(out));
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
        if constexpr (GROUPED) {
          uint8_t* to = (uint8_t*)a.C + (long long)(row0 + quarter * 32) * (a.N / 2) + n0 / 2;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = half * 16 + i * 4 + (lane >> 3), c = lane & 7;
            if (row0 + quarter * 32 + r < row_end) st_v4(to + (long long)r * (a.N / 2) + c * 16, ld_v4(out + r * 128 + ((c ^ (r & 7)) << 4)));
          }
        }
        parity ^= 1;
      } else if (a.out_f32) {
        float* to = (float*)a.C + (long long)row * a.N + n0 + half * 128;
        const int cols = a.N - n0 - half * 128;
        if (live) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (c * 32 + j * 4 < cols) {
                const float2 x = halves_of(sum[c][2 * j]), y = halves_of(sum[c][2 * j + 1]);
                *reinterpret_cast<float4*>(to + c * 32 + j * 4) = make_float4(x.x, x.y, y.x, y.y);
              }
        }
      } else {
        const int r0 = row0 + quarter * 32, n = n0 + half * 128;
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // 64 columns at a time
          if (!GROUPED && lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const f32x2* x = sum[2 * h + j / 4] + 4 * (j & 3);
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 f = halves_of(x[i]);
              w[i] = pack_bf16x2(f.x, f.y);
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(patch_s + lane * 128 + ((j ^ (lane & 7)) << 4)), "r"(w[0]), "r"(w[1]),
                         "r"(w[2]), "r"(w[3])
                         : "memory");
          }
          if constexpr (!GROUPED) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0 && n + 64 * h < a.N && r0 < a.M) {
              f8_store(&tmap_c, n + 64 * h, r0, patch_s);
              asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
          } else {
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int r = i * 4 + (lane >> 3), c = lane & 7, col = n + 64 * h + c * 8;
              if (r0 + r < row_end && col < a.N) st_v4((bf16*)a.C + (long long)(r0 + r) * a.N + col, lds_v4(patch_s + r * 128 + ((c ^ (r & 7)) << 4)));
            }
            __syncwarp();
          }
        }
      }
    }
    if (!GROUPED && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }

  tc_fence_before();
  __syncthreads();
  if (dead) f8_let_copies_end();
  if constexpr (PAIR) cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    else
      tmem_dealloc(tmem, 512);
  }
}

// ---- small ---------------------------------------------------------------------------------------------------------------------
constexpr int FS_MAX_STAGES = 8, FS_MAX_SPLITS = 8, FS_SCALES = 576;  // bytes of a stage's scales of rows: up to 132, from a multiple of four on
constexpr int FS_RING_ALONE = 208 * 1024, FS_RING_SHARED = 106 * 1024;

// CTAs of a tile to an SM: registers for the sums and the loads, tensor memory and the ring allow two where the rows are few
template <bool GATED>
constexpr int small_resident(int most_rows) { return most_rows <= (GATED ? 32 : 64) ? 2 : 1; }

// GATED: 128 gates and the 128 that they gate, else 128 rows of W; MOST: rows of A at most (a thread's sums)
template <bool GATED, int MOST, bool GROUPED>
__global__ void __launch_bounds__(GATED ? 320 : 192, small_resident<GATED>(MOST))
    gemm_fp8_small_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                          const __grid_constant__ Fp8Args a) {
  constexpr int WT = GATED ? 2 : 1, NT = WT * 128, EPI = 4 * WT, THREADS = 64 + 32 * EPI;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t full[FS_MAX_STAGES], empty[FS_MAX_STAGES], acc_full[2], acc_empty[2];
  __shared__ __align__(16) float scales[FS_MAX_STAGES][FS_SCALES / 4];
  __shared__ uint32_t tmem_slot;
  __shared__ int dead;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int splits = a.splits, split = blockIdx.x, n0 = blockIdx.y * NT;
  const float *as = a.as, *ws = a.ws;
  int g = 0, row0 = blockIdx.z * a.rows, row_end = a.M;
  if constexpr (GROUPED) {
    wait_for_previous();
    if ((int)blockIdx.z >= min(*a.n_mt, a.max_mt)) return;
    const int4 e = a.tab[blockIdx.z];
    g = min(max(e.x, 0), a.groups - 1);
    row0 = max(e.y, 0);
    row_end = min(e.z, a.M);
    if (row0 >= row_end) return;
  }
  const int rows = min(row_end - row0, a.rows), mp = (rows + 15) & ~15, stride = (rows + 31) & ~31;  // stride: columns of an accumulator
  const int boxes = GROUPED ? (rows + a.box_rows - 1) / a.box_rows : 1;
  const int b0 = split * a.blocks / splits, b1 = (split + 1) * a.blocks / splits;
  const int a_room = (a.rows + 31) / 32 * 32 * FP8_BLOCK, stage_bytes = WT * F8_STAGE_W + a_room;

  if (warp == 0 && lane == 0) {
    dead = 0;
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_w);
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1 + EPI);  // the products', and the warps that have read the scales
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(acc_full + s, 1);
      mbar_init(acc_empty + s, EPI);
    }
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc(&tmem_slot, a.cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
  const int w_row = g * a.N + n0;
  if (!GROUPED && warp == 0 && lane == 0)  // the first weights into L2 while the kernel before this one ends
    for (int i = 0; i < min(a.stages, b1 - b0); ++i) tma_prefetch_2d(&tmap_w, (b0 + i) * 64, w_row);
  __syncwarp();
  follow_previous(as, ws);

  if (warp == 0) {
    if (lane == 0) {
      // scales of the rows: from a multiple of four on, no further than their line goes
      const int s0 = row0 & ~3, n_scales = min((row0 - s0 + mp + 3) & ~3, a.ld_as - s0);
      const uint32_t bytes = (uint32_t)(WT * F8_STAGE_W + boxes * a.box_rows * FP8_BLOCK + n_scales * 4);
      int stage = 0;
      uint32_t phase = 0;
      for (int b = b0; b < b1; ++b) {
        uint8_t* to = smem + stage * stage_bytes;
        f8_wait(empty + stage, phase ^ 1u, &dead, a.failed);
        if (*(volatile int*)&dead) break;
        mbar_expect_tx(full + stage, bytes);
        tma_load_2d(to, &tmap_w, b * 64, w_row, full + stage);
        for (int x = 0; x < boxes; ++x)
          tma_load_2d(to + WT * F8_STAGE_W + x * a.box_rows * FP8_BLOCK, &tmap_a, b * 64, row0 + x * a.box_rows, full + stage);
        tma_bulk_g2s(scales[stage], as + (long long)b * a.ld_as + s0, n_scales * 4, full + stage);
        if (++stage == a.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    const uint32_t idesc = fp8_idesc(128, mp);
    const uint32_t ring = __shfl_sync(0xffffffffu, smem_u32(smem), 0);
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    for (int b = b0; b < b1; ++b) {
      if (!mbar_wait_warp(acc_empty + acc, acc_phase ^ 1u, &dead, a.failed, WAIT_CYCLES)) break;
      if (!mbar_wait_warp(full + stage, phase, &dead, a.failed, WAIT_CYCLES)) break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t sw = ring + (uint32_t)(stage * stage_bytes), sa = sw + WT * F8_STAGE_W, d = tmem + (uint32_t)(acc * WT * stride);
#pragma unroll
        for (int h = 0; h < WT; ++h)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_fp8(d + (uint32_t)(h * stride), make_smem_desc(sw + h * F8_STAGE_W + k * 32), make_smem_desc(sa + k * 32), idesc, k > 0);
        umma_commit(empty + stage);
        umma_commit(acc_full + acc);
      }
      __syncwarp();
      if (++stage == a.stages) {
        stage = 0;
        phase ^= 1u;
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    }
    __syncwarp();
  }

  // ---- lane = row of W, column = row of A ----
  float* red = reinterpret_cast<float*>(smem);
  if (warp >= 2) {
    const int quarter = warp & 3, which = (warp - 2) >> 2;  // which: gates, or what they gate
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(which * stride);
    const float* w0 = ws + ((long long)g * a.n_blocks + blockIdx.y * WT + which) * a.blocks;
    f32x2 sum[MOST / 32][16];
#pragma unroll
    for (int c = 0; c < MOST / 32; ++c)
#pragma unroll
      for (int j = 0; j < 16; ++j) sum[c][j] = 0ull;
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    const int shift = row0 & 3;
    float sw = 0.f;
    for (int b = b0; b < b1; ++b) {
      if ((b - b0) % 32 == 0 && b + lane < b1) sw = w0[b + lane];
      const float x = __shfl_sync(0xffffffffu, sw, (b - b0) & 31);
      const f32x2 by = pair_of(x, x);
      f8_wait(full + stage, phase, &dead, a.failed);  // (the scales)
      f8_wait(acc_full + acc, acc_phase, &dead, a.failed);
      __syncwarp();
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < MOST / 32; ++c)
        if (c * 32 < rows) {
          uint32_t v[32];
          tmem_ld32(lanes + (uint32_t)(acc * WT * stride + c * 32), v);
          tmem_ld_wait_for(v);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float4 s;
            if constexpr (GROUPED) {
              const float* p = scales[stage] + shift + c * 32 + j * 4;
              s = make_float4(p[0], p[1], p[2], p[3]);
            } else {
              s = *reinterpret_cast<const float4*>(scales[stage] + c * 32 + j * 4);
            }
            sum[c][2 * j] = fma2(pair_of(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1])), mul2(pair_of(s.x, s.y), by), sum[c][2 * j]);
            sum[c][2 * j + 1] =
                fma2(pair_of(__uint_as_float(v[4 * j + 2]), __uint_as_float(v[4 * j + 3])), mul2(pair_of(s.z, s.w), by), sum[c][2 * j + 1]);
          }
        }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(acc_empty + acc);
        mbar_arrive(empty + stage);
      }
      if (++stage == a.stages) {
        stage = 0;
        phase ^= 1u;
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    }
    // (every warp has seen the last products, which have read the ring; a CTA that gave up leaves the ring alone)
    asm volatile("bar.sync 1, %0;" ::"n"(32 * EPI) : "memory");
    if (*(volatile int*)&dead == 0) {
      const int at = which * 128 + quarter * 32 + lane;
#pragma unroll
      for (int c = 0; c < MOST / 32; ++c)
        if (c * 32 < rows) {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float2 f = halves_of(sum[c][j]);
            red[(c * 32 + 2 * j) * NT + at] = f.x;
            red[(c * 32 + 2 * j + 1) * NT + at] = f.y;
          }
        }
    }
  }
  if (splits > 1)
    cluster_sync_all();
  else
    __syncthreads();
  // rows split, split + splits, ... are this CTA's to add and store, a row to a warp, four columns to a lane
  for (int r = warp * splits + split; r < rows; r += THREADS / 32 * splits) {
    const float* src = red + r * NT + lane * 4;
    float4 p[FS_MAX_SPLITS], q[GATED ? FS_MAX_SPLITS : 1];
    if (splits > 1) {
#pragma unroll
      for (int s = 0; s < FS_MAX_SPLITS; ++s)
        if (s < splits) {
          const uint32_t at = mapa_shared(src, s);
          p[s] = ld_cluster_v4(at);
          if constexpr (GATED) q[s] = ld_cluster_v4(at + 512);
        }
    } else {
      p[0] = *reinterpret_cast<const float4*>(src);
      if constexpr (GATED) q[0] = *reinterpret_cast<const float4*>(src + 128);
    }
    float4 x = p[0], u = x;
    if constexpr (GATED) u = q[0];
#pragma unroll
    for (int s = 1; s < FS_MAX_SPLITS; ++s)
      if (s < splits) {
        x.x += p[s].x; x.y += p[s].y; x.z += p[s].z; x.w += p[s].w;
        if constexpr (GATED) { u.x += q[s].x; u.y += q[s].y; u.z += q[s].z; u.w += q[s].w; }
      }
    const long long row = row0 + r;
    if constexpr (GATED) {
      x.x = fp8_unit(x.x, u.x, a.gelu);
      x.y = fp8_unit(x.y, u.y, a.gelu);
      x.z = fp8_unit(x.z, u.z, a.gelu);
      x.w = fp8_unit(x.w, u.w, a.gelu);
      const float m = max_or_nan(max_or_nan(fabsf(x.x), fabsf(x.y)), max_or_nan(fabsf(x.z), fabsf(x.w)));
      const float scale = fp8_scale(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)))), by = fp8_inverse(scale);
      *reinterpret_cast<uint32_t*>((uint8_t*)a.C + row * (a.N / 2) + n0 / 2 + lane * 4) = fp8_four(x.x * by, x.y * by, x.z * by, x.w * by);
      if (lane == 0) a.ys[(long long)blockIdx.y * a.ld_ys + row] = scale;
    } else if (n0 + lane * 4 < a.N) {
      if (a.out_f32)
        *reinterpret_cast<float4*>((float*)a.C + row * a.N + n0 + lane * 4) = x;
      else
        *reinterpret_cast<uint2*>((bf16*)a.C + row * a.N + n0 + lane * 4) = make_uint2(pack_bf16x2(x.x, x.y), pack_bf16x2(x.z, x.w));
    }
  }
  if (splits > 1) cluster_sync_all();  // nobody leaves with what a peer still reads
  tc_fence_before();
  __syncthreads();
  if (dead) f8_let_copies_end();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, a.cols);
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------
// once for each device that a kernel runs on
template <typename F>
static int once_per_device(uint64_t (&seen)[2], F&& f) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 128 && (seen[dev / 64] >> (dev % 64) & 1)) return B200Q_OK;
  const int rc = f();
  if (!rc && dev >= 0 && dev < 128) seen[dev / 64] |= 1ull << (dev % 64);
  return rc;
}

// as many clusters as can be resident at once, one CTA to an SM
template <typename K>
static int clusters_that_fit(K kern, int cluster, int threads, int smem) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cluster, 148);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    n = num_sms() / cluster;
  }
  return n < num_sms() / cluster ? n : num_sms() / cluster;
}

template <bool PAIR, bool GATED, bool GROUPED>
static int launch_large(const void* A, long long a_rows, const void* W, long long w_rows, Fp8Args a, cudaStream_t st) {
  using Cfg = LargeCfg<PAIR, GATED>;
  auto kern = gemm_fp8_large_kernel<PAIR, GATED, GROUPED>;
  static uint64_t seen[2];
  int rc = once_per_device(seen, [&]() -> int {
    B200Q_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
    return B200Q_OK;
  });
  CUtensorMap ta, tw, tc = {};
  // (two codes are one element of the maps; a box is 128 codes wide)
  if (!rc) rc = get_tmap(A, a_rows, a.K / 2, 128, &ta);
  if (!rc) rc = get_tmap(W, w_rows, a.K / 2, Cfg::BOX, &tw);
  if (!rc && !GROUPED && GATED) rc = get_tmap(a.C, a.M, a.N / 4, 32, &tc);
  if (!rc && !GROUPED && !GATED && !a.out_f32) rc = get_tmap(a.C, a.M, a.N, 32, &tc);
  if (rc) return rc;
  const long long n_tiles = (a.N + FL_BN - 1) / FL_BN, m_tiles = GROUPED ? a.max_mt : (a.M + (PAIR ? 255 : 127)) / (PAIR ? 256 : 128);
  B200Q_CHECK_ARG(n_tiles * m_tiles < (1ll << 31), "gemm_fp8: too many tiles (M=%d N=%d)", a.M, a.N);
  static int pairs = 0;
  if (PAIR && pairs == 0) pairs = clusters_that_fit(kern, 2, FL_THREADS, Cfg::SMEM);
  const long long units = PAIR ? pairs : num_sms(), grid = (n_tiles * m_tiles < units ? n_tiles * m_tiles : units) * (PAIR ? 2 : 1);
  B200Q_CUDA(launch_early(kern, (int)grid, FL_THREADS, Cfg::SMEM, st, PAIR ? 2 : 1, ta, tw, tc, a));
  count_launch();
  return B200Q_OK;
}

template <bool GATED, int MOST, bool GROUPED>
static int launch_small(const void* A, long long a_rows, const void* W, long long w_rows, Fp8Args a, cudaStream_t st) {
  constexpr int NT = GATED ? 256 : 128, THREADS = GATED ? 320 : 192, RESIDENT = small_resident<GATED>(MOST);
  constexpr int RING = RESIDENT == 2 ? FS_RING_SHARED : FS_RING_ALONE;
  auto kern = gemm_fp8_small_kernel<GATED, MOST, GROUPED>;
  static uint64_t seen[2];
  static int fit[FS_MAX_SPLITS + 1];
  int rc = once_per_device(seen, [&]() -> int {
    B200Q_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, RING + 1024));
    return B200Q_OK;
  });
  if (rc) return rc;
  const int n_tiles = (a.N + NT - 1) / NT, m_tiles = GROUPED ? a.max_mt : (a.M + a.rows - 1) / a.rows;
  B200Q_CHECK_ARG(n_tiles <= 65535 && m_tiles <= 65535, "gemm_fp8: too many tiles (M=%d N=%d)", a.M, a.N);
  a.box_rows = GROUPED ? 32 : (a.rows + 7) & ~7;
  if (!GROUPED && a.M < a.box_rows) a.box_rows = (a.M + 7) & ~7;
  const int stage = (GATED ? 2 : 1) * F8_STAGE_W + (a.rows + 31) / 32 * 32 * FP8_BLOCK;
  a.stages = RING / stage < FS_MAX_STAGES ? RING / stage : FS_MAX_STAGES;
  a.cols = 32;
  while (a.cols < 2 * (GATED ? 2 : 1) * ((a.rows + 31) / 32 * 32)) a.cols *= 2;
  // splits: as many as leave every cluster resident, three blocks each at least
  a.splits = 1;
  if (!batch_invariant())
    for (int s = 2; s <= FS_MAX_SPLITS && a.blocks / s >= 3; ++s) {
      if (fit[s] == 0) fit[s] = clusters_that_fit(kern, s, THREADS, FS_RING_ALONE + 1024 < RING + 1024 ? FS_RING_ALONE + 1024 : RING + 1024);
      if ((long long)n_tiles * m_tiles <= (long long)fit[s] * RESIDENT) a.splits = s;
    }
  CUtensorMap ta, tw;
  rc = get_tmap(A, a_rows, a.K / 2, a.box_rows, &ta);
  if (!rc) rc = get_tmap(W, w_rows, a.K / 2, NT, &tw);
  if (rc) return rc;
  B200Q_CUDA(launch_early(kern, dim3(a.splits, n_tiles, m_tiles), THREADS, RING + 1024, st, a.splits, ta, tw, a));
  count_launch();
  return B200Q_OK;
}

template <bool GATED, bool GROUPED>
static int launch_small(const void* A, long long a_rows, const void* W, long long w_rows, const Fp8Args& a, cudaStream_t st) {
  if (a.rows <= 32) return launch_small<GATED, 32, GROUPED>(A, a_rows, W, w_rows, a, st);
  if (a.rows <= 64) return launch_small<GATED, 64, GROUPED>(A, a_rows, W, w_rows, a, st);
  return launch_small<GATED, 128, GROUPED>(A, a_rows, W, w_rows, a, st);
}

int g_fp8_mode = 0;  // test hook: 1 = small tiles, 2 = large ones of one CTA, 3 = of a pair

static int finish_args(Fp8Args& a) {
  a.blocks = (a.K + FP8_BLOCK - 1) / FP8_BLOCK;
  a.n_blocks = (a.N + 127) / 128;
  if (!wait_flag(&a.failed)) {
    set_error("gemm_fp8: no host-visible flag for bounded waits");
    return B200Q_ECUDA;
  }
  return B200Q_OK;
}

template <bool GATED>
static int dense(const void* A, const void* W, Fp8Args a, cudaStream_t st) {
  int rc = finish_args(a);
  if (rc) return rc;
  int mode = g_fp8_mode;
  if (mode == 0) mode = a.M <= 128 ? 1 : a.M <= 256 ? 2 : 3;
  if (mode == 1) {
    const int tiles = (a.M + 127) / 128;
    a.rows = ((a.M + tiles - 1) / tiles + 15) / 16 * 16;
    return launch_small<GATED, false>(A, a.M, W, a.N, a, st);
  }
  return mode == 2 ? launch_large<false, GATED, false>(A, a.M, W, a.N, a, st) : launch_large<true, GATED, false>(A, a.M, W, a.N, a, st);
}

template <bool GATED>
static int grouped(const void* A, long long a_rows, const void* W, int groups, Fp8Args a, cudaStream_t st) {
  int rc = finish_args(a);
  if (rc) return rc;
  a.groups = groups;
  int mode = g_fp8_mode;
  if (mode == 0) mode = a_rows <= 64ll * groups ? 1 : 2;
  if (mode == 1) {
    a.rows = 128;
    return launch_small<GATED, true>(A, a_rows, W, (long long)groups * a.N, a, st);
  }
  return launch_large<false, GATED, true>(A, a_rows, W, (long long)groups * a.N, a, st);
}

static bool fp8_aligned(const void* a, const void* b, const void* c, const void* d) {
  return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c) | reinterpret_cast<uintptr_t>(d)) & 15) == 0;
}

// what all products ask of their arguments
static int check_product(const char* what, const void* A, const float* as, int ld_as, const void* W, const float* ws, const void* C, int M, int N,
                         int K, bool gated) {
  B200Q_CHECK_ARG(M >= 0 && N > 0 && K > 0 && K % 16 == 0 && N % (gated ? 256 : 8) == 0, "%s: unsupported shape M=%d N=%d K=%d (K%%16==0, N%%%d==0)", what,
                  M, N, K, gated ? 256 : 8);
  B200Q_CHECK_ARG(ld_as >= M && ld_as % 4 == 0, "%s: ld_a_scales=%d is less than M=%d or no multiple of 4", what, ld_as, M);
  if (M == 0) return B200Q_OK;
  B200Q_CHECK_ARG(A && as && W && ws && C, "%s: null argument", what);
  B200Q_CHECK_ARG(fp8_aligned(A, as, W, C), "%s: A, a_scales, W and the output must be 16-byte aligned", what);
  return B200Q_OK;
}

}  // namespace b200q

using namespace b200q;

extern "C" {

int b200q_gemm_fp8(const void* A, const float* a_scales, int ld_a_scales, const void* W, const float* w_scales, void* C, int M, int N, int K,
                   int out_f32, void* stream) {
  int rc = check_product("gemm_fp8", A, a_scales, ld_a_scales, W, w_scales, C, M, N, K, false);
  if (rc || M == 0) return rc;
  Fp8Args a{};
  a.as = a_scales;
  a.ld_as = ld_a_scales;
  a.ws = w_scales;
  a.C = C;
  a.M = M;
  a.N = N;
  a.K = K;
  a.out_f32 = out_f32 != 0;
  return dense<false>(A, W, a, as_stream(stream));
}

int b200q_gemm_gated_fp8(const void* A, const float* a_scales, int ld_a_scales, const void* W, const float* w_scales, void* Y, float* y_scales,
                         int ld_y_scales, int M, int N, int K, int act, void* stream) {
  int rc = check_product("gemm_gated_fp8", A, a_scales, ld_a_scales, W, w_scales, Y, M, N, K, true);
  if (rc) return rc;
  B200Q_CHECK_ARG((act == 0 || act == 1) && ld_y_scales >= M, "gemm_gated_fp8: act=%d or ld_y_scales=%d unknown or too small", act, ld_y_scales);
  if (M == 0) return B200Q_OK;
  B200Q_CHECK_ARG(y_scales, "gemm_gated_fp8: null argument");
  Fp8Args a{};
  a.as = a_scales;
  a.ld_as = ld_a_scales;
  a.ws = w_scales;
  a.C = Y;
  a.ys = y_scales;
  a.ld_ys = ld_y_scales;
  a.M = M;
  a.N = N;
  a.K = K;
  a.gelu = act;
  return dense<true>(A, W, a, as_stream(stream));
}

int b200q_gemm_grouped_fp8(const void* A, int a_rows, const float* a_scales, int ld_a_scales, const void* W, const float* w_scales, int groups, void* C,
                           int N, int K, const void* tab, const int32_t* n_mt, int max_mtiles, int out_f32, void* stream) {
  int rc = check_product("gemm_grouped_fp8", A, a_scales, ld_a_scales, W, w_scales, C, a_rows, N, K, false);
  if (rc) return rc;
  B200Q_CHECK_ARG(groups > 0 && max_mtiles >= 0 && (long long)groups * N < (1ll << 31), "gemm_grouped_fp8: groups=%d max_mtiles=%d", groups, max_mtiles);
  if (a_rows == 0 || max_mtiles == 0) return B200Q_OK;
  B200Q_CHECK_ARG(tab && n_mt && (reinterpret_cast<uintptr_t>(tab) & 15) == 0, "gemm_grouped_fp8: the table of tiles is missing or not aligned");
  Fp8Args a{};
  a.as = a_scales;
  a.ld_as = ld_a_scales;
  a.ws = w_scales;
  a.C = C;
  a.tab = (const int4*)tab;
  a.n_mt = n_mt;
  a.max_mt = max_mtiles;
  a.M = a_rows;
  a.N = N;
  a.K = K;
  a.out_f32 = out_f32 != 0;
  return grouped<false>(A, a_rows, W, groups, a, as_stream(stream));
}

int b200q_gemm_grouped_gated_fp8(const void* A, int a_rows, const float* a_scales, int ld_a_scales, const void* W, const float* w_scales, int groups,
                                 void* Y, float* y_scales, int ld_y_scales, int N, int K, const void* tab, const int32_t* n_mt, int max_mtiles, int act,
                                 void* stream) {
  int rc = check_product("gemm_grouped_gated_fp8", A, a_scales, ld_a_scales, W, w_scales, Y, a_rows, N, K, true);
  if (rc) return rc;
  B200Q_CHECK_ARG((act == 0 || act == 1) && ld_y_scales >= a_rows, "gemm_grouped_gated_fp8: act=%d or ld_y_scales=%d unknown or too small", act, ld_y_scales);
  B200Q_CHECK_ARG(groups > 0 && max_mtiles >= 0 && (long long)groups * N < (1ll << 31), "gemm_grouped_gated_fp8: groups=%d max_mtiles=%d", groups, max_mtiles);
  if (a_rows == 0 || max_mtiles == 0) return B200Q_OK;
  B200Q_CHECK_ARG(tab && n_mt && y_scales && (reinterpret_cast<uintptr_t>(tab) & 15) == 0,
                  "gemm_grouped_gated_fp8: the table of tiles or y_scales is missing or not aligned");
  Fp8Args a{};
  a.as = a_scales;
  a.ld_as = ld_a_scales;
  a.ws = w_scales;
  a.C = Y;
  a.ys = y_scales;
  a.ld_ys = ld_y_scales;
  a.tab = (const int4*)tab;
  a.n_mt = n_mt;
  a.max_mt = max_mtiles;
  a.M = a_rows;
  a.N = N;
  a.K = K;
  a.gelu = act;
  return grouped<true>(A, a_rows, W, groups, a, as_stream(stream));
}

// test hook: 0 = by size, 1 = small tiles, 2 = large tiles of one CTA, 3 = of a pair (dense products)
int b200q_gemm_fp8_set_mode(int mode) {
  B200Q_CHECK_ARG(mode >= 0 && mode <= 3, "gemm_fp8_set_mode: mode=%d", mode);
  g_fp8_mode = mode;
  bump_tuning_epoch();
  return B200Q_OK;
}

}  // extern "C"
