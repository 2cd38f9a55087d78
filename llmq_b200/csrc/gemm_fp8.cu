// gemm_fp8.cu — C[m,n] = sum_b as[b,m] ws[n/128,b] sum_{k in block b} A[m,k] W[n,k]: products of e4m3 codes with a scale for each block of 128 of
// the reduction (fp8.cuh), fp32 sums; dense, gated (the unit's values leave in 8 bits again) and by expert.
//
// A block of 128 codes is one swizzle span, one stage of the ring and four tcgen05.mma (kind::f8f6f4, 32 codes each) whose fp32 sums start from
// zero; the block's scales are then multiplied in while the sums leave tensor memory for the registers that hold the running total ("promoted").
// Two or four accumulators let the tensor core work on the next blocks meanwhile.
//
// Bounds: for few rows the weight stream (N K bytes); for many the tensor core at twice the bf16 rate and, as near, tensor memory, which products
// fill while the promotion reads it (32 columns: some 165 cycles beside products, 16 to 30 alone), two packed multiply-adds to four sums; over a second
// of them the clock, which the power limit holds at 1.2 to 1.5 GHz.  us, back to back in a graph, weights from HBM (the first milliseconds / over a
// second): 1 x 4096 x 4096 6.3, 48 x 4096 x 14336 14.7 (4.0 TB/s of weights; bf16 24), 1001 x 8192 x 3584 29.9 / 34.7 (1.97 / 1.70 PFLOP/s; bf16
// 44.9 / 51.7), 4608 x 4096 x 14336 231 / 265 (2.34 / 2.04 PFLOP/s; bf16 370 / 428; over a second the library's product of the same codes with one scale
// for all of them 196, of zeros 133); gated 7 x 16384 x 2048 9.3, 4608 x 28672 x 4096 463 / 529 (bf16 684 / 781); 16 experts of 2048 x 2048, 64
// tokens to four of them 16.1 / 17.2 (4.2 TB/s of weights).
//
//   * large: rows of A are the tensor core's M side (a lane has a row, so that its scale is one number to a thread), up to 256 columns to a CTA,
//     eight warps that promote half of them each in up to 128 registers a thread.  Persistent.  One CTA to 128 rows, or a pair (cta_group::2) to
//     256, each of which fetches half of the weights; or a cluster to a tile, with a part of the reduction to each CTA or pair.
//   * small, up to 128 rows to a tile (gated: 64): the weights are the M side and the rows, padded to 16, the N side; the reduction is split over
//     a cluster whose partial sums meet in distributed shared memory in the order of the splits.
#include <atomic>
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
  int ld_as, ld_ys, M, N, K, blocks, n_blocks, max_mt, groups, ahead, out_f32, gelu, a_bytes;
  // small tiles
  int rows, box_rows, stages, accs, cols, splits;
  // blocks that a warp of products makes before it gives up (a test's; else more than there are); large: cycles that a wait lasts (read from here the
  // small kernel's cost 48 x 4096 x 14336 0.4 us)
  long long patience;
  int give_up;
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
// arrive on the barrier at this place in both CTAs of the pair, `pair` (a bit to a CTA of the cluster)
__device__ __forceinline__ void f8_commit_2sm(uint64_t* bar, uint16_t pair) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"(pair)
               : "memory");
}
// the last barrier of a cluster whose CTAs only read each other's memory: what they have read they have used (an arrival that releases would
// wait for the outputs' stores: 128 x 4096 x 14336 in four parts 1.5 us)
__device__ __forceinline__ void f8_leave_cluster() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}
// the unit of a gate and what it gates, fp32 from the sums on: g sigmoid(g) u, or tanh GELU, 0.5 g (1 + tanh t) = g sigmoid(2 t)
// (the exponent is for base 2, its rounding 2^-24 of it; the two instructions are off by 2^-22 and 2^-23 at most; the same through __expf and
// __fdividef, which look at subnormal numbers: 4608 x 16384 x 2048 174 us for 170)
// The reciprocal is that of a quarter and is multiplied by a quarter of the gate: fp32 has it in full up to where the exponential passes its range,
// 2^128 (gates below -88.7, tanh GELU -10.06), and nothing is let through.  (That of 1 + e ends at 2^126: what gates from -87.3 on let through was 0.)
__device__ __forceinline__ float fp8_unit(float g, float u, int gelu) {
  const float q = 0.25f * g, t = gelu ? q * fmaf(64.f * -0.10294324f, q * q, 4.f * -2.3022082f) : q * (4.f * -1.4426950f);
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(e, 0.25f, 0.25f)));
  return q * r * u;
}
// A wait with a limit: false where it has run out, or another role of the CTA has given up (dead; flag and clock are looked at every 64 tries).  Who
// is told so issues nothing more: a load would come to a place that is still read, or arm a barrier that is armed, a product would read what has not
// come.
__device__ __forceinline__ bool f8_give_up(volatile int* dead, int* failed) {
  *dead = 1;
  __threadfence_block();
  *(volatile int*)failed = 1;
  return false;
}
[[nodiscard]] __device__ __forceinline__ bool f8_wait(uint64_t* bar, uint32_t parity, volatile int* dead, int* failed, long long limit = WAIT_CYCLES) {
  long long t0 = 0;
  for (int n = 0; !mbar_try_wait(bar, parity); ++n) {
    if (n % 64 != 63) continue;
    if (n == 63) t0 = clock64();
    if (*dead) return false;
    if (clock64() - t0 > limit) return f8_give_up(dead, failed);
  }
  return true;
}
// the same of who looks at `dead` itself before anything is issued, or issues nothing
__device__ __forceinline__ void f8_await(uint64_t* bar, uint32_t parity, volatile int* dead, int* failed, long long limit = WAIT_CYCLES) {
  (void)f8_wait(bar, parity, dead, failed, limit);
}
// copies in flight end before a block that gave up returns its memory
__device__ __noinline__ void f8_let_copies_end() {
  const long long t0 = clock64();
  while (clock64() - t0 < 4000000ll) {
  }
  __syncthreads();
}

// ---- large ---------------------------------------------------------------------------------------------------------------------
constexpr int FL_THREADS = 384, FL_MAX_SPLITS = 8;
// registers: 384 threads begin with 168; four warps give back 128 each and eight take 64 more (40 x 128 + 232 x 256 = 168 x 384)
constexpr int FL_REGS_FEW = 40, FL_REGS_MANY = 232;
// A tile has 64 CH columns.  The products of a block are two, to a half of them each, whose accumulators are filled and emptied on their own: a
// half's next product waits for four warps and not for eight, and the tensor core has the other half's to do meanwhile.  Rows of W come in boxes,
// so that the columns of a half are neighbours, or (gated) 64 gates and the 64 that they gate; of a pair each CTA has half of them.
template <bool PAIR, int CH, bool GATED>
struct LargeCfg {
  static constexpr int BN = 64 * CH, W_ROWS = PAIR ? BN / 2 : BN;                // columns of a tile; rows of W that a CTA fetches
  static constexpr int ACCS = 512 / BN < 4 ? 2 : 4;                              // accumulators of each half in tensor memory
  static constexpr int STAGE = F8_STAGE_W + W_ROWS * FP8_BLOCK;                  // behind 128 rows of A
  // a warp's columns of C on their way out: all of them where a wide tile of a pair leaves room, else 64 (gated: 128 codes of two tiles for two warps)
  static constexpr int PATCH = PAIR && CH == 4 && !GATED ? 8192 : 4096;
  static constexpr int STAGES = (229376 - 8 * PATCH) / STAGE < 8 ? (229376 - 8 * PATCH) / STAGE : 8;
  static constexpr int BOX = PAIR ? 16 * CH : GATED ? 64 : BN, BOXES = W_ROWS / BOX;
  static constexpr int SMEM = STAGES * STAGE + 8 * PATCH + 1024;
};

// 32 of a thread's sums (its row, columns in turn) += scale * what has come from tensor memory
__device__ __forceinline__ void promote(f32x2* acc, const uint32_t (&v)[32], f32x2 scale) {
#pragma unroll
  for (int j = 0; j < 16; ++j) acc[j] = fma2(pair_of(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), scale, acc[j]);
}

// SPLIT: a cluster to a tile, a part of the reduction to each of its CTAs, whose sums meet in distributed shared memory in the order of the parts
template <bool PAIR, int CH, bool GATED, bool GROUPED, bool SPLIT>
__global__ void __launch_bounds__(FL_THREADS, 1)
    gemm_fp8_large_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                          const __grid_constant__ CUtensorMap tmap_c, const __grid_constant__ Fp8Args a) {
  using Cfg = LargeCfg<PAIR, CH, GATED>;
  static_assert(!GATED || CH == 4, "a gated tile has 128 gates");
  static_assert(!SPLIT || !(GROUPED || GATED), "parts of dense products");
  constexpr int STAGES = Cfg::STAGES, BM = PAIR ? 256 : 128, BN = Cfg::BN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* patches = smem + STAGES * Cfg::STAGE;
  __shared__ __align__(8) uint64_t full[STAGES], empty[STAGES], acc_full[2][Cfg::ACCS], acc_empty[2][Cfg::ACCS];  // of accumulators: [half of the columns][turn]
  __shared__ uint32_t tmem_slot;
  __shared__ int dead;
  __shared__ float most[2][128];  // gated: the largest of a half row's 64 values
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  constexpr int CTAS = PAIR ? 2 : 1;  // that make a tile's products together
  const int in_cluster = PAIR || SPLIT ? (int)cluster_ctarank() : 0, rank = in_cluster % CTAS, leader = in_cluster - rank;
  const int split = in_cluster / CTAS, share = SPLIT ? CTAS * a.splits : CTAS;  // share: CTAs to a tile
  const int unit = blockIdx.x / share, units = gridDim.x / share;
  const int n_tiles = (a.N + BN - 1) / BN, blocks = a.blocks;
  const int b_begin = SPLIT ? split * blocks / a.splits : 0, b_end = SPLIT ? (split + 1) * blocks / a.splits : blocks;
  auto next_acc = [](int& acc, uint32_t& phase) {
    if (++acc == Cfg::ACCS) {
      acc = 0;
      phase ^= 1u;
    }
  };
  // the i-th box of a stage begins so many rows of W behind the tile's first
  auto w_box = [&](int i) { return PAIR ? (GATED ? rank * 128 + i * 64 : (i * 2 + rank) * Cfg::BOX) : GATED ? (i & 1) * 128 + (i >> 1) * 64 : 0; };

  if (warp == 0 && lane == 0) {
    dead = 0;
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_w);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full + s, PAIR ? 2 : 1);
      mbar_init(empty + s, 2);  // both halves' products
    }
    for (int s = 0; s < 2 * Cfg::ACCS; ++s) {
      mbar_init(acc_full[0] + s, 1);
      mbar_init(acc_empty[0] + s, PAIR ? 8 : 4);  // (the leader's) the warps that promote
    }
    mbar_fence_init();
  }
  if (warp == 3 && lane == 0 && (!GROUPED || unit < a.ahead)) {
    // the first weights into L2 while the kernel before this one ends and this one makes ready (behind that: 1 to 2 % more for few rows).  The table
    // is not known yet: as if every group had one tile
    const int m_tiles = GROUPED ? a.groups : (a.M + BM - 1) / BM, n0 = unit / m_tiles * BN + (GROUPED ? unit % m_tiles * a.N : 0);
    for (int b = 0; b < min(STAGES, b_end - b_begin); ++b)
      for (int i = 0; i < Cfg::BOXES; ++i) tma_prefetch_2d(&tmap_w, (b_begin + b) * 64, n0 + w_box(i));
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
  const float *as = a.as, *ws = a.ws;
  const int4* tab = a.tab;
  const int32_t* n_mt = a.n_mt;
  follow_previous(as, ws, tab, n_mt);
  const int m_tiles = GROUPED ? min(*n_mt, a.max_mt) : (a.M + BM - 1) / BM;
  const int num_tiles = m_tiles * n_tiles;
  // a tile: columns n0 .., rows row0 .. row_end of a group
  auto entry_of = [&](int tile) { return GROUPED ? tab[tile % m_tiles] : make_int4(0, 0, 0, 0); };
  auto tile_of = [&](int tile, int4 e, int& g, int& row0, int& row_end, int& n0) {
    const int mt = tile % m_tiles;
    n0 = tile / m_tiles * BN;
    if constexpr (GROUPED) {  // (kept within the matrices, whatever the table says)
      g = min(max(e.x, 0), a.groups - 1);
      row0 = min(max(e.y, 0), a.M);
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
        bool on = true;
        for (int tile = unit; on && tile < num_tiles; tile += units) {
          int g, row0, row_end, n0;
          tile_of(tile, entry_of(tile), g, row0, row_end, n0);
          const int wrow = g * a.N + n0;
          for (int b = b_begin; b < b_end; ++b) {
            uint8_t* to = smem + stage * Cfg::STAGE;
            on = f8_wait(empty + stage, phase ^ 1u, &dead, a.failed, a.patience);
            if (!on) break;
            if constexpr (PAIR) {
              const uint32_t bar = mapa_shared(full + stage, leader);
              f8_expect_tx(bar, Cfg::STAGE - F8_STAGE_W + a.a_bytes);
#pragma unroll
              for (int i = 0; i < Cfg::BOXES; ++i) f8_load_2sm(to + F8_STAGE_W + i * Cfg::BOX * 128, &tmap_w, b * 64, wrow + w_box(i), bar);
              f8_load_2sm(to, &tmap_a, b * 64, row0, bar);
            } else {
              mbar_expect_tx(full + stage, Cfg::STAGE - F8_STAGE_W + a.a_bytes);
#pragma unroll
              for (int i = 0; i < Cfg::BOXES; ++i) tma_load_2d(to + F8_STAGE_W + i * Cfg::BOX * 128, &tmap_w, b * 64, wrow + w_box(i), full + stage);
              tma_load_2d(to, &tmap_a, b * 64, row0, full + stage);
            }
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
      }
      __syncwarp();
    } else if (warp < 3 && rank == 0) {  // a warp to the products of each half
      const int h = warp - 1;
      constexpr uint32_t idesc = fp8_idesc(BM, BN / 2);
      const uint32_t ring = __shfl_sync(0xffffffffu, smem_u32(smem), 0);
      const uint64_t rows = make_smem_desc(ring), columns = make_smem_desc(ring + F8_STAGE_W + h * (Cfg::W_ROWS / 2) * FP8_BLOCK);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      int left = a.give_up;
      bool on = true;
      if (elect_one())
        for (int tile = unit; on && tile < num_tiles; tile += units) {
          const int b_stop = left < b_end - b_begin ? b_begin + left : b_end;
          left -= b_stop - b_begin;
          for (int b = b_begin; b < b_stop; ++b) {
            on = f8_wait(full + stage, phase, &dead, a.failed, a.patience) && f8_wait(acc_empty[h] + acc, acc_phase ^ 1u, &dead, a.failed, a.patience);
            if (!on) break;
            tc_fence_after();
            const uint64_t at = (uint64_t)(stage * (Cfg::STAGE / 16));  // (addresses in descriptors count 16 bytes)
            const uint32_t d = tmem + (uint32_t)(acc * BN + h * (BN / 2));
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if constexpr (PAIR)
                umma_fp8_2sm(d, rows + at + 2 * k, columns + at + 2 * k, idesc, k > 0);
              else
                umma_fp8(d, rows + at + 2 * k, columns + at + 2 * k, idesc, k > 0);
            }
            if constexpr (PAIR) {
              f8_commit_2sm(acc_full[h] + acc, (uint16_t)(3 << leader));
              f8_commit_2sm(empty + stage, (uint16_t)(3 << leader));
            } else {
              umma_commit(acc_full[h] + acc);
              umma_commit(empty + stage);
            }
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
            next_acc(acc, acc_phase);
          }
          if (b_stop < b_end) on = f8_give_up(&dead, a.failed);
        }
      __syncwarp();
    }
    if constexpr (SPLIT) cluster_sync_all();  // (as the other warps do where their sums are in shared memory)
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(FL_REGS_MANY));
    // rows quarter * 32 + lane; columns: half of the tile's, gated: half * 64 + 0 .. 63 of the gates and of what they gate
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * (BN / 2));
    uint8_t* const patch = patches + (warp - 4) * Cfg::PATCH;
    const uint32_t patch_s = smem_u32(patch);
    const uint32_t empty0 = PAIR ? mapa_shared(acc_empty[half], leader) : smem_u32(acc_empty[half]);
    int acc = 0, parity = 0;
    uint32_t acc_phase = 0;
    auto await_sums = [&]() {
      f8_await(acc_full[half] + acc, acc_phase, &dead, a.failed, a.patience);
      __syncwarp();
    };
    // Weights' scales: a lane's of 32 blocks of the reduction, handed round by shuffles.  A tile's columns lie in up to two blocks of 128 (gated:
    // the gates' and that of what they gate); 32 neighbouring columns lie in one.  Rows' scales: four blocks'.  A tile's first are asked for
    // while the one before it leaves.  (Without a condition: a load that may not be made is waited for where it is made.  Rows and blocks that do
    // not exist take the last ones', or the first.)
    constexpr int SCALES = GATED || CH == 3 ? 2 : 1;
    float sw[SCALES], sa[4];
    auto row_scales = [&](int row0, int row_end) { return as + max(min(row0 + quarter * 32 + lane, row_end - 1), 0); };
    auto row_scale = [&](const float* rows, int b) { return rows[(long long)min(b, b_end - 1) * a.ld_as]; };
    auto column_scales = [&](int g, int n0) {
      return ws + ((long long)g * a.n_blocks + min(n0 / 128 + (CH == 4 && !GATED ? half : 0), a.n_blocks - 1)) * blocks;
    };
    auto column_scale = [&](const float* columns, int n0, int b, int h) {
      return columns[(h && n0 / 128 + 1 < a.n_blocks ? blocks : 0) + min(b + lane, b_end - 1)];
    };
    auto first_scales = [&](int tile, int4 e) {
      int g, row0, row_end, n0;
      tile_of(tile, e, g, row0, row_end, n0);
#pragma unroll
      for (int h = 0; h < SCALES; ++h) sw[h] = column_scale(column_scales(g, n0), n0, b_begin, h);
#pragma unroll
      for (int i = 0; i < 4; ++i) sa[i] = row_scale(row_scales(row0, row_end), b_begin + i);
    };
    int4 entry = make_int4(0, 0, 0, 0), next_entry = entry;
    if (unit < num_tiles) {
      next_entry = entry_of(unit);
      first_scales(unit, next_entry);
    }
    for (int tile = unit; tile < num_tiles; tile += units) {
      int g, row0, row_end, n0;
      entry = next_entry;
      if (tile + units < num_tiles) next_entry = entry_of(tile + units);
      tile_of(tile, entry, g, row0, row_end, n0);
      const int row = row0 + quarter * 32 + lane;
      const bool live = row < row_end;
      if (!SPLIT && row0 + quarter * 32 >= row_end) {  // no rows: the accumulators only have to be passed on
        for (int b = b_begin; b < b_end; ++b) {
          await_sums();
          if (lane == 0) f8_arrive(empty0 + acc * 8);
          next_acc(acc, acc_phase);
        }
        if (tile + units < num_tiles) first_scales(tile + units, next_entry);
        continue;
      }
      const int col0 = GATED ? 0 : n0 % 128 + half * (BN / 2);
      auto scale_of = [&](int c) { return GATED ? c >> 1 : CH == 3 ? (col0 + 32 * c) >> 7 : 0; };
      const float *own_rows = row_scales(row0, row_end), *columns = column_scales(g, n0);
      f32x2 sum[CH][16];
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < 16; ++j) sum[c][j] = 0ull;
      uint32_t v[2][32];
      await_sums();
      tc_fence_after();
      tmem_ld32(lanes + (uint32_t)(acc * BN), v[0]);
      // (a block is an odd number of loads where CH is 3: its first goes to v[i & 1] there, four blocks to a round)
      for (int b0 = b_begin; b0 < b_end; b0 += 4) {
        // four blocks' factors, and only then the loads of the next four: a wait for a load is one for all that were issued before it
        float x[4][SCALES];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int h = 0; h < SCALES; ++h) x[i][h] = sa[i] * __shfl_sync(0xffffffffu, sw[h], (b0 + i - b_begin) & 31);
#pragma unroll
        for (int i = 0; i < 4; ++i) sa[i] = row_scale(own_rows, b0 + 4 + i);
        if ((b0 + 4 - b_begin) % 32 == 0) {
#pragma unroll
          for (int h = 0; h < SCALES; ++h) sw[h] = column_scale(columns, n0, b0 + 4, h);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (b0 + i < b_end) {
            f32x2 s[SCALES];
#pragma unroll
            for (int h = 0; h < SCALES; ++h) s[h] = pair_of(x[i][h], x[i][h]);
            const uint32_t from = lanes + (uint32_t)(acc * BN);
#pragma unroll
            for (int c = 0; c < CH; ++c) {
              constexpr int ODD = CH & 1;
              uint32_t(&now)[32] = v[(c + ODD * i) & 1];
              uint32_t(&next)[32] = v[(c + 1 + ODD * i) & 1];
              tmem_ld_wait_for(now);
              if (c < CH - 1) {
                tmem_ld32(from + (uint32_t)(c * 32 + 32), next);
              } else {  // the accumulator is free; the next one's first columns while the last of this are added
                tc_fence_before();
                __syncwarp();
                if (lane == 0) f8_arrive(empty0 + acc * 8);
                next_acc(acc, acc_phase);
                if (b0 + i + 1 < b_end) {
                  await_sums();
                  tc_fence_after();
                  tmem_ld32(lanes + (uint32_t)(acc * BN), next);
                }
              }
              promote(sum[c], now, SCALES == 2 && scale_of(c) ? s[SCALES - 1] : s[0]);
            }
          }
        }
      }
      if constexpr (SPLIT) {
        // [32 rows][column / 4][row][4] sums; of the tile's pieces of 32 rows x 16 columns a CTA adds up every `splits`-th, a warp to a piece
        float4* red = reinterpret_cast<float4*>(smem) + lane;
        asm volatile("bar.sync 5, 256;" ::: "memory");  // (both halves' products have read the ring)
        if (*(volatile int*)&dead == 0) {
#pragma unroll
          for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float2 x = halves_of(sum[c][2 * j]), y = halves_of(sum[c][2 * j + 1]);
              red[(((quarter * 2 + half) * CH + c) * 8 + j) * 32] = make_float4(x.x, x.y, y.x, y.y);
            }
        }
        cluster_sync_all();
        for (int piece = dead ? 16 * CH : split + (warp - 4) * a.splits; piece < 16 * CH; piece += 8 * a.splits) {
          const int r0 = row0 + piece / (4 * CH) * 32, n = n0 + piece % (4 * CH) * 16;
          if (r0 >= row_end) break;
          float4 total[4];
          constexpr int AT_ONCE = CH == 2 ? 4 : 1;  // parts whose reads are under way together (more registers than there are beside wider tiles)
#pragma unroll 1
          for (int p0 = 0; p0 < a.splits; p0 += AT_ONCE) {
            float4 x[AT_ONCE][4];
#pragma unroll
            for (int p = 0; p < AT_ONCE; ++p)
              if (p0 + p < a.splits) {
                const uint32_t at = mapa_shared(red + piece * 128, (p0 + p) * CTAS + rank);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[p][j] = ld_cluster_v4(at + j * 512);
              }
#pragma unroll
            for (int p = 0; p < AT_ONCE; ++p)
              if (p0 + p < a.splits) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  total[j] = p0 + p == 0 ? x[p][j]
                                         : make_float4(total[j].x + x[p][j].x, total[j].y + x[p][j].y, total[j].z + x[p][j].z, total[j].w + x[p][j].w);
              }
          }
          if (r0 + lane < row_end) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
              if (n + j * 8 < a.N) {
                const float4 lo = total[2 * j], hi = total[2 * j + 1];
                const long long to = (long long)(r0 + lane) * a.N + n + j * 8;
                if (a.out_f32) {
                  *reinterpret_cast<float4*>((float*)a.C + to) = lo;
                  *reinterpret_cast<float4*>((float*)a.C + to + 4) = hi;
                } else {
                  st_v4((bf16*)a.C + to, make_uint4(pack_bf16x2(lo.x, lo.y), pack_bf16x2(lo.z, lo.w), pack_bf16x2(hi.x, hi.y), pack_bf16x2(hi.z, hi.w)));
                }
              }
          }
        }
        continue;  // (a tile to a CTA: the loop ends)
      }
      if (tile + units < num_tiles) first_scales(tile + units, next_entry);
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
        uint8_t* const out = patches + (2 * quarter + parity) * Cfg::PATCH;
        const bool copies = half == 0 && lane == 0, engine = !GROUPED || row0 + quarter * 32 + 32 <= row_end;  // (no rows that are another group's)
        if (copies) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
        uint32_t gone = *(volatile int*)&dead;  // (for both warps, which meet again below)
        asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            "setp.ne.b32 p, %0, 0;\n\t"
            "bar.red.or.pred p, %1, 64, p;\n\t"
            "selp.b32 %0, 1, 0, p;\n\t"
            "}\n"
            : "+r"(gone)
            : "r"(1 + quarter)
            : "memory");
        if (gone) break;
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
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
        if (copies) {  // (rows that are not copied so leave an empty group, as the wait counts turns)
          if (engine && row0 + quarter * 32 < a.M) f8_store(&tmap_c, n0 / 4, row0 + quarter * 32, smem_u32(out));
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
        if (!engine) {
          uint8_t* to = (uint8_t*)a.C + (long long)(row0 + quarter * 32) * (a.N / 2) + n0 / 2;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = half * 16 + i * 4 + (lane >> 3), c = lane & 7;
            if (row0 + quarter * 32 + r < row_end) st_v4(to + (long long)r * (a.N / 2) + c * 16, ld_v4(out + r * 128 + ((c ^ (r & 7)) << 4)));
          }
        }
        parity ^= 1;
      } else if (__any_sync(0xffffffffu, *(volatile int*)&dead)) {
        break;
      } else if (a.out_f32) {
        float* to = (float*)a.C + (long long)row * a.N + n0 + half * (BN / 2);
        const int cols = a.N - n0 - half * (BN / 2);
        if (live) {
#pragma unroll
          for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (c * 32 + j * 4 < cols) {
                const float2 x = halves_of(sum[c][2 * j]), y = halves_of(sum[c][2 * j + 1]);
                *reinterpret_cast<float4*>(to + c * 32 + j * 4) = make_float4(x.x, x.y, y.x, y.y);
              }
        }
      } else {
        const int r0 = row0 + quarter * 32, n = n0 + half * (BN / 2);
        constexpr int WIDE = CH % 2 ? 32 : 64;  // columns at a time
        // by the copy engine, which takes 64 columns of 32 rows, and none that are another group's; else by this warp, as all but the last 64
        // where the patch has room for no more: the engine takes some 1000 cycles to read it (64 tokens, 16 experts of 2048 x 1024 9.0 -> 8.7 us)
        constexpr bool ENGINE = WIDE == 64, ROOM = Cfg::PATCH > 4096;
        constexpr int LAST = 32 * CH / WIDE - 1;
        const bool copies = ENGINE && (!GROUPED || r0 + 32 <= row_end);
        if (ENGINE) {  // (what the tile before left has been read)
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          __syncwarp();
        }
#pragma unroll
        for (int h = 0; h <= LAST; ++h) {
          const uint32_t to = patch_s + (ROOM ? h * 4096 : 0);
#pragma unroll
          for (int j = 0; j < WIDE / 8; ++j) {
            const f32x2* x = sum[h * (WIDE / 32) + j / 4] + 4 * (j & 3);
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 f = halves_of(x[i]);
              w[i] = pack_bf16x2(f.x, f.y);
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + lane * 128 + ((j ^ (lane & 7)) << 4)), "r"(w[0]), "r"(w[1]),
                         "r"(w[2]), "r"(w[3])
                         : "memory");
          }
          if (copies && (ROOM || h == LAST)) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0 && n + 64 * h < a.N && r0 < a.M) {
              f8_store(&tmap_c, n + 64 * h, r0, to);
              asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
          } else {
            __syncwarp();
#pragma unroll
            for (int i = 0; i < WIDE / 8; ++i) {
              constexpr int ACROSS = WIDE / 8;  // lanes to a row
              const int r = i * (32 / ACROSS) + lane / ACROSS, c = lane % ACROSS, col = n + WIDE * h + c * 8;
              if (r0 + r < row_end && col < a.N) st_v4((bf16*)a.C + (long long)(r0 + r) * a.N + col, lds_v4(to + r * 128 + ((c ^ (r & 7)) << 4)));
            }
            __syncwarp();
          }
        }
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }

  tc_fence_before();
  __syncthreads();
  if (dead) f8_let_copies_end();
  if constexpr (PAIR)
    cluster_sync_all();  // nobody leaves with what a peer still reads or signals
  else if constexpr (SPLIT)
    f8_leave_cluster();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    else
      tmem_dealloc(tmem, 512);
  }
}

// ---- small ---------------------------------------------------------------------------------------------------------------------
constexpr int FS_MAX_STAGES = 8, FS_MAX_SPLITS = 8, FS_MAX_ACCS = 4, FS_SCALES = 512;  // bytes of a stage's scales of rows
constexpr int FS_MAX_TILES = 65535;  // in each of the grid's directions
constexpr int FS_RING_ALONE = 208 * 1024, FS_RING_SHARED = 106 * 1024;

// CTAs of a tile to an SM: registers for the sums and the loads, tensor memory and the ring allow two where the rows are few
template <bool GATED>
constexpr int small_resident(int most_rows) { return most_rows <= (GATED ? 32 : 64) ? 2 : 1; }

// groups of four warps that share an accumulator's columns (rows of A), 64 each
constexpr int small_groups(int most_rows) { return most_rows > 64 ? 2 : 1; }
template <bool GATED>
constexpr int small_threads(int most_rows) { return 64 + 128 * (GATED ? 2 : 1) * small_groups(most_rows); }

// GATED: 128 gates and the 128 that they gate, else 128 rows of W; MOST: rows of A at most
template <bool GATED, int MOST>
__global__ void __launch_bounds__(small_threads<GATED>(MOST), small_resident<GATED>(MOST))
    gemm_fp8_small_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                          const __grid_constant__ Fp8Args a) {
  constexpr int WT = GATED ? 2 : 1, NT = WT * 128, CG = small_groups(MOST), EPI = 4 * WT * CG, THREADS = 64 + 32 * EPI;
  constexpr int CHUNKS = MOST / CG / 32;               // of 32 columns to a warp
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t full[FS_MAX_STAGES], empty[FS_MAX_STAGES], acc_full[FS_MAX_ACCS], acc_empty[FS_MAX_ACCS];
  __shared__ __align__(16) float scales[FS_MAX_STAGES][FS_SCALES / 4];
  __shared__ uint32_t tmem_slot;
  __shared__ int dead;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int splits = a.splits, split = blockIdx.x, n0 = blockIdx.y * NT;
  const float *as = a.as, *ws = a.ws;
  const int row0 = blockIdx.z * a.rows;
  const int rows = min(a.M - row0, a.rows), mp = (rows + 15) & ~15, stride = (rows + 31) & ~31;  // stride: columns of an accumulator
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
    for (int s = 0; s < a.accs; ++s) {
      mbar_init(acc_full + s, 1);
      mbar_init(acc_empty + s, EPI);
    }
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc(&tmem_slot, a.cols);
  if (warp == 2 && lane == 0)  // the first weights into L2 while the kernel before this one ends and this one makes ready
    for (int i = 0; i < min(a.stages, b1 - b0); ++i) tma_prefetch_2d(&tmap_w, (b0 + i) * 64, n0);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
  follow_previous(as, ws);

  if (warp == 0) {
    if (lane == 0) {
      const int n_scales = min(mp, a.ld_as - row0);  // (no further than their line goes: a multiple of four, as row0 is)
      const uint32_t bytes = (uint32_t)(WT * F8_STAGE_W + a.box_rows * FP8_BLOCK + n_scales * 4);
      int stage = 0;
      uint32_t phase = 0;
      for (int b = b0; b < b1; ++b) {
        uint8_t* to = smem + stage * stage_bytes;
        f8_await(empty + stage, phase ^ 1u, &dead, a.failed);
        if (*(volatile int*)&dead) break;  // (warps whose waits have run out arrive all the same, behind the flag)
        mbar_expect_tx(full + stage, bytes);
        tma_load_2d(to, &tmap_w, b * 64, n0, full + stage);
        tma_load_2d(to + WT * F8_STAGE_W, &tmap_a, b * 64, row0, full + stage);
        tma_bulk_g2s(scales[stage], as + (long long)b * a.ld_as + row0, n_scales * 4, full + stage);
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
    const uint64_t weights = make_smem_desc(ring), rows_of_a = make_smem_desc(ring + WT * F8_STAGE_W);
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    const int b_stop = a.give_up < b1 - b0 ? b0 + a.give_up : b1;
    if (elect_one()) {
      for (int b = b0; b < b_stop; ++b) {
        f8_await(acc_empty + acc, acc_phase ^ 1u, &dead, a.failed);
        f8_await(full + stage, phase, &dead, a.failed);
        if (*(volatile int*)&dead) break;
        tc_fence_after();
        const uint64_t at = (uint64_t)(uint32_t)(stage * (stage_bytes / 16));  // (addresses in descriptors count 16 bytes)
        const uint32_t d = tmem + (uint32_t)(acc * WT * stride);
#pragma unroll
        for (int h = 0; h < WT; ++h)
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_fp8(d + (uint32_t)(h * stride), weights + at + (h * (F8_STAGE_W / 16) + 2 * k), rows_of_a + at + 2 * k, idesc, k > 0);
        umma_commit(acc_full + acc);
        umma_commit(empty + stage);
        if (++stage == a.stages) {
          stage = 0;
          phase ^= 1u;
        }
        if (++acc == a.accs) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
      if (b_stop < b1) f8_give_up(&dead, a.failed);
    }
    __syncwarp();
  }

  // ---- lane = row of W, column = row of A ----
  float* red = reinterpret_cast<float*>(smem);
  if (warp >= 2) {
    const int quarter = warp & 3, which = (warp - 2) / 4 % WT, col0 = (warp - 2) / (4 * WT) * (MOST / CG);  // which: gates, or what they gate
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(which * stride + col0);
    const float* w0 = ws + (long long)(blockIdx.y * WT + which) * a.blocks;
    f32x2 sum[CHUNKS][16];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
      for (int j = 0; j < 16; ++j) sum[c][j] = 0ull;
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    float sw = 0.f;
    for (int b = b0; b < b1; ++b) {
      if ((b - b0) % 32 == 0 && b + lane < b1) sw = w0[b + lane];
      const float x = __shfl_sync(0xffffffffu, sw, (b - b0) & 31);
      const f32x2 by = pair_of(x, x);
      f8_await(full + stage, phase, &dead, a.failed);  // (the scales)
      f8_await(acc_full + acc, acc_phase, &dead, a.failed);
      __syncwarp();
      tc_fence_after();
      uint32_t v[CHUNKS][32];
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c)
        if (col0 + c * 32 < rows) tmem_ld32(lanes + (uint32_t)(acc * WT * stride + c * 32), v[c]);
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c)
        if (col0 + c * 32 < rows) {
          tmem_ld_wait_for(v[c]);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 s = *reinterpret_cast<const float4*>(scales[stage] + col0 + c * 32 + j * 4);
            sum[c][2 * j] = fma2(pair_of(__uint_as_float(v[c][4 * j]), __uint_as_float(v[c][4 * j + 1])), mul2(pair_of(s.x, s.y), by), sum[c][2 * j]);
            sum[c][2 * j + 1] =
                fma2(pair_of(__uint_as_float(v[c][4 * j + 2]), __uint_as_float(v[c][4 * j + 3])), mul2(pair_of(s.z, s.w), by), sum[c][2 * j + 1]);
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
      if (++acc == a.accs) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
    // (every warp has seen the last products, which have read the ring; a CTA that gave up leaves the ring alone)
    asm volatile("bar.sync 1, %0;" ::"n"(32 * EPI) : "memory");
    if (*(volatile int*)&dead == 0) {
      const int at = which * 128 + quarter * 32 + lane;
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c)
        if (col0 + c * 32 < rows) {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float2 f = halves_of(sum[c][j]);
            red[(col0 + c * 32 + 2 * j) * NT + at] = f.x;
            red[(col0 + c * 32 + 2 * j + 1) * NT + at] = f.y;
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
  if (splits > 1) f8_leave_cluster();  // nobody leaves with what a peer still reads
  tc_fence_before();
  __syncthreads();
  if (dead) f8_let_copies_end();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, a.cols);
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------
// once for each device that a kernel runs on (twice at most where two threads meet)
template <typename F>
static int once_per_device(std::atomic<uint64_t> (&seen)[2], F&& f) {
  int dev = 0;
  cudaGetDevice(&dev);
  const bool counted = dev >= 0 && dev < 128;
  if (counted && (seen[dev / 64].load() >> (dev % 64) & 1)) return B200Q_OK;
  const int rc = f();
  if (!rc && counted) seen[dev / 64].fetch_or(1ull << (dev % 64));
  return rc;
}

// As many clusters of so many CTAs as can be resident at once, by their shared memory (one of 225 KiB to an SM, or two of 107): asked of a
// kernel that is never launched, since the query knows one CTA to an SM for kernels that hold tensor memory.  Asked once on each device (which SMs a
// device has, and so how many clusters fit, is its own); where the query fails, by the number of SMs, and again the next time.
__global__ void fp8_probe_kernel() {}
constexpr int F8_WHOLE_SM = 230400, F8_HALF_SM = 109568;
static int clusters_that_fit(int cluster, int smem, int threads) {
  constexpr int DEVICES = 64;
  static std::atomic<int> known[DEVICES][2][FL_MAX_SPLITS + 1];
  int dev = -1;
  cudaGetDevice(&dev);
  std::atomic<int>* const kept = dev >= 0 && dev < DEVICES ? &known[dev][smem == F8_HALF_SM][cluster] : nullptr;
  if (kept)
    if (int n = kept->load()) return n;
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
  if (cudaFuncSetAttribute(fp8_probe_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, F8_WHOLE_SM) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, fp8_probe_kernel, &cfg) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    return num_sms() * (smem == F8_HALF_SM ? 2 : 1) / cluster;
  }
  if (kept) kept->store(n);
  return n;
}

// splits > 1 (SPLIT): CTAs to a tile
template <bool PAIR, int CH, bool GATED, bool GROUPED, bool SPLIT>
static int launch_large(const void* A, long long a_rows, const void* W, long long w_rows, Fp8Args a, cudaStream_t st) {
  using Cfg = LargeCfg<PAIR, CH, GATED>;
  auto kern = gemm_fp8_large_kernel<PAIR, CH, GATED, GROUPED, SPLIT>;
  static std::atomic<uint64_t> seen[2];
  int rc = once_per_device(seen, [&]() -> int {
    B200Q_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
    return B200Q_OK;
  });
  CUtensorMap ta, tw, tc = {};
  // (two codes are one element of the maps; a box is 128 codes wide)
  const int box = !GROUPED && a_rows < 128 ? ((int)a_rows + 7) & ~7 : 128;  // rows of A that travel
  a.a_bytes = box * FP8_BLOCK;
  if (!rc) rc = get_tmap(A, a_rows, a.K / 2, box, &ta);
  if (!rc) rc = get_tmap(W, w_rows, a.K / 2, Cfg::BOX, &tw);
  if (!rc && GATED) rc = get_tmap(a.C, a.M, a.N / 4, 32, &tc);
  if (!rc && !GATED && !a.out_f32) rc = get_tmap(a.C, a.M, a.N, 32, &tc);
  if (rc) return rc;
  const long long n_tiles = (a.N + Cfg::BN - 1) / Cfg::BN, m_tiles = GROUPED ? a.max_mt : (a.M + (PAIR ? 255 : 127)) / (PAIR ? 256 : 128);
  const long long tiles = n_tiles * m_tiles;
  B200Q_CHECK_ARG(tiles < (1ll << 27), "gemm_fp8: too many tiles (M=%d N=%d)", a.M, a.N);
  const long long units = PAIR ? clusters_that_fit(2, F8_WHOLE_SM, FL_THREADS) : num_sms(), at_once = SPLIT || tiles < units ? tiles : units;
  const int cluster = (PAIR ? 2 : 1) * (SPLIT ? a.splits : 1);
  B200Q_CUDA(launch_early(kern, (int)(at_once * cluster), FL_THREADS, Cfg::SMEM, st, cluster, ta, tw, tc, a));
  count_launch();
  return B200Q_OK;
}

// small tiles of a product: rows of each, parts of the reduction (as many as leave every cluster resident, three blocks each at least)
struct SmallPlan {
  int rows, m_tiles, n_tiles, splits, resident;
};
template <bool GATED>
static SmallPlan small_plan(int M, int N, int blocks) {
  const int most = GATED ? 64 : 128;
  SmallPlan p{};
  p.m_tiles = (M + most - 1) / most;
  p.rows = ((M + p.m_tiles - 1) / p.m_tiles + 15) / 16 * 16;
  p.m_tiles = (M + p.rows - 1) / p.rows;
  p.n_tiles = (N + (GATED ? 255 : 127)) / (GATED ? 256 : 128);
  p.resident = small_resident<GATED>(p.rows <= 32 ? 32 : p.rows <= 64 ? 64 : 128);
  p.splits = 1;
  if (!batch_invariant())
    for (int s = 2; s <= FS_MAX_SPLITS && blocks / s >= 3; ++s)
      if ((long long)p.n_tiles * p.m_tiles <= clusters_that_fit(s, p.resident == 2 ? F8_HALF_SM : F8_WHOLE_SM, 192)) p.splits = s;
  return p;
}

template <bool GATED, int MOST>
static int launch_small(const void* A, const void* W, const SmallPlan& p, Fp8Args a, cudaStream_t st) {
  constexpr int NT = GATED ? 256 : 128, THREADS = small_threads<GATED>(MOST), RESIDENT = small_resident<GATED>(MOST);
  constexpr int RING = RESIDENT == 2 ? FS_RING_SHARED : FS_RING_ALONE;
  auto kern = gemm_fp8_small_kernel<GATED, MOST>;
  static std::atomic<uint64_t> seen[2];
  int rc = once_per_device(seen, [&]() -> int {
    B200Q_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, RING + 1024));
    return B200Q_OK;
  });
  if (rc) return rc;
  B200Q_CHECK_ARG(p.n_tiles <= FS_MAX_TILES && p.m_tiles <= FS_MAX_TILES, "gemm_fp8: too many tiles (M=%d N=%d)", a.M, a.N);
  a.rows = p.rows;
  a.splits = p.splits;
  a.box_rows = a.M < a.rows ? (a.M + 7) & ~7 : a.rows;
  const int padded = (a.rows + 31) / 32 * 32, stage = (GATED ? 2 : 1) * F8_STAGE_W + padded * FP8_BLOCK;
  a.stages = RING / stage < FS_MAX_STAGES ? RING / stage : FS_MAX_STAGES;
  // accumulators: four where they fit the CTA's share of tensor memory, so that no role waits for the round through the others
  const int each = (GATED ? 2 : 1) * padded;
  a.accs = FS_MAX_ACCS * each <= 512 / RESIDENT ? FS_MAX_ACCS : 512 / RESIDENT / each;
  a.cols = 32;
  while (a.cols < a.accs * each) a.cols *= 2;
  CUtensorMap ta, tw;
  rc = get_tmap(A, a.M, a.K / 2, a.box_rows, &ta);
  if (!rc) rc = get_tmap(W, a.N, a.K / 2, NT, &tw);
  if (rc) return rc;
  B200Q_CUDA(launch_early(kern, dim3(a.splits, p.n_tiles, p.m_tiles), THREADS, RING + 1024, st, a.splits, ta, tw, a));
  count_launch();
  return B200Q_OK;
}

template <bool GATED>
static int launch_small(const void* A, const void* W, const Fp8Args& a, cudaStream_t st) {
  const SmallPlan p = small_plan<GATED>(a.M, a.N, a.blocks);
  if (p.rows <= 32) return launch_small<GATED, 32>(A, W, p, a, st);
  if constexpr (GATED) {
    return launch_small<GATED, 64>(A, W, p, a, st);
  } else {
    return p.rows <= 64 ? launch_small<GATED, 64>(A, W, p, a, st) : launch_small<GATED, 128>(A, W, p, a, st);
  }
}

int g_fp8_mode = 0;  // test hook: see b200q_gemm_fp8_set_mode
int g_fp8_give_up = 0;

// Which kernel and tile: the least of what each is expected to take, us.  A round of tiles (as many as are resident at once) costs so much for
// its start and end and so much a block; no kernel takes less than the weights do to come from memory; parts cost their exchange.  Fitted to
// 450 sizes (15 shapes of 1024 to 16384 columns x 1024 to 14336, 30 row counts from 1 to 4608, weights from HBM, bf16 outputs, back to back in a
// graph) and every kernel: what is taken is 0.5 % slower than the best on average, more than 5 % at 9 of them, and 10 % at 3000 x 2304 x 9216 (pairs
// of 192 columns 68.9 us, of 256 62.7).  us (of that measurement: one card, its large products at the power limit), the choice / others:
// 1 x 4096 x 4096 small 6.3 / four parts of 128 columns 8.3; 48 x 4096 x 14336 small 14.5 / four
// parts 15.9; 128 x 4096 x 14336 four parts of 128 columns 16.7 / small 22.5, whole tiles 43; 200 x 4096 x 14336 three parts of 192 columns
// 23.0 / two of 128 23.4, whole 43; 300 x 8192 x 3584 pairs of 256 columns 15.7 / single CTAs 16.3, of 128 columns 21.1; 450 x 4096 x 14336 pairs
// in two parts 35.1 / 128 columns 37.8; 768 x 4096 x 4096 pairs of 256 17.2 / of 192 17.4, 128 columns 23.1; 4608 x 4096 x 14336 pairs of 256
// 252 / single CTAs 251 to 277.
// Gated (184 sizes, 8 shapes; 0.2 % on average): 16 x 16384 x 2048 small 10.6 / 13.4 / pairs 13.5; 48 x 28672 x 4096 small 27.7 / 25.2 / 35.9;
// 200 x 28672 x 4096 99 / 42 / 37; 300 110 / 62 / 69; 4608 single CTAs 586 / pairs 507.
struct Fp8Tile {
  int kind, ch, splits;  // as the hook's
};
template <bool GATED>
static Fp8Tile choose_fp8_tile(int M, int N, int blocks) {
  const double weights = 1.6e-7 * N * FP8_BLOCK * blocks;
  Fp8Tile best{1, 4, 1};
  double least = 1e30;
  auto offer = [&](Fp8Tile t, double us) {
    if (us < least) {
      least = us;
      best = t;
    }
  };
  auto larger = [](double a, double b) { return a > b ? a : b; };
  if (M <= 512 && N <= FS_MAX_TILES * (GATED ? 256 : 128)) {
    const SmallPlan p = small_plan<GATED>(M, N, blocks);
    const int fit = p.splits > 1 ? clusters_that_fit(p.splits, p.resident == 2 ? F8_HALF_SM : F8_WHOLE_SM, 192) : num_sms() * p.resident;
    const int rounds = (p.n_tiles * p.m_tiles + fit - 1) / fit, each = (blocks + p.splits - 1) / p.splits;
    const double parts = p.splits - 1;
    if (GATED)
      offer({1, 4, 1}, p.resident == 2 ? 5.5 + larger(rounds * (0.29 + 0.093 * each), 1.05 * weights) : 2.5 + larger(rounds * (2.55 + 0.677 * each), 1.4 * weights));
    else if (p.rows <= 32)
      offer({1, 4, 1}, 2.9 + larger(rounds * 0.464 * each, 1.14 * weights) + 0.13 * parts);
    else if (p.rows <= 64)
      offer({1, 4, 1}, 2.4 + larger(rounds * 0.78 * each, weights) + 0.07 * parts + 0.025 * (M - 33));
    else if (rounds == 1 && each <= 16)
      offer({1, 4, 1}, 4.5 + larger(0.5 * each, weights) + 0.024 * parts);
  }
  const struct {
    Fp8Tile tile;  // splits: the most
    double fixed, round, block, part, weights;
  } plain[6] = {{{2, 2, 1}, 2.0, 1.45, 0.307, 0, 1.19}, {{2, 4, 1}, 0, 4.16, 0.406, 0, 1}, {{3, 3, 1}, 0, 4.4, 0.342, 0, 1}, {{3, 4, 1}, 0, 4.63, 0.359, 0, 1},
                {{4, 2, 6}, 0, 5.5, 0.325, 0.12, 1}, {{4, 3, 4}, 0, 6.9, 0.384, 0.1, 1.87}},
    pair_parts = {{5, 4, 3}, 0, 9.05, 0.429, 0, 1},
    gated[2] = {{{2, 4, 1}, 2.1, 2.72, 0.53, 0, 1.25}, {{3, 4, 1}, 2.4, 3.24, 0.435, 0, 1.06}};
  auto large = [&](const auto& c) {
    const bool pair = c.tile.kind == 3 || c.tile.kind == 5;
    const long long tiles = (long long)((M + (pair ? 255 : 127)) / (pair ? 256 : 128)) * ((N + 64 * c.tile.ch - 1) / (64 * c.tile.ch));
    for (int s = c.tile.splits > 1 ? 2 : 1; s <= c.tile.splits && (s == 1 || blocks / s >= 2); ++s) {
      const int ctas = s * (pair ? 2 : 1), fit = ctas > 1 ? clusters_that_fit(ctas, F8_WHOLE_SM, FL_THREADS) : num_sms();
      const double rounds = (double)((tiles + fit - 1) / fit);
      offer({c.tile.kind, c.tile.ch, s}, c.fixed + larger(rounds * (c.round + c.block * ((blocks + s - 1) / s)), c.weights * weights) + c.part * (s - 1));
    }
  };
  if (GATED) {
    for (const auto& c : gated) large(c);
  } else {
    for (int i = 0; i < (batch_invariant() ? 4 : 6); ++i) large(plain[i]);
    if (!batch_invariant()) large(pair_parts);
  }
  return best;
}

static int finish_args(Fp8Args& a) {
  a.blocks = (a.K + FP8_BLOCK - 1) / FP8_BLOCK;
  a.n_blocks = (a.N + 127) / 128;
  a.patience = g_fp8_give_up ? 200000 : WAIT_CYCLES;
  a.give_up = g_fp8_give_up ? g_fp8_give_up - 1 : 2147483647;
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
  Fp8Tile t{g_fp8_mode % 10, g_fp8_mode / 10 % 10, g_fp8_mode / 100};
  if (t.kind == 0) t = choose_fp8_tile<GATED>(a.M, a.N, a.blocks);
  if (t.kind == 1) return launch_small<GATED>(A, W, a, st);
  a.splits = t.splits < a.blocks ? t.splits : a.blocks;
  const bool pair = t.kind == 3 || t.kind == 5;
  auto large = [&](auto pair, auto columns, auto split) {
    return launch_large<decltype(pair)::value, decltype(columns)::value, GATED, false, decltype(split)::value>(A, a.M, W, a.N, a, st);
  };
  const std::integral_constant<int, 2> c128;
  const std::integral_constant<int, 3> c192;
  const std::integral_constant<int, 4> c256;
  const std::true_type yes;
  const std::false_type no;
  if constexpr (!GATED) {
    if (a.splits > 1 && t.kind >= 4) return pair ? large(yes, c256, yes) : t.ch == 2 ? large(no, c128, yes) : large(no, c192, yes);
    if (pair && t.ch == 3) return large(yes, c192, no);
    if (!pair && t.ch == 2) return large(no, c128, no);
  }
  return pair ? large(yes, c256, no) : large(no, c256, no);
}

template <bool GATED>
static int grouped(const void* A, long long a_rows, const void* W, int groups, Fp8Args a, cudaStream_t st) {
  int rc = finish_args(a);
  if (rc) return rc;
  a.groups = groups;
  // weights are asked for before the table is known where most groups have one tile: two rows or more to a group on average, one tile at most
  if (a_rows >= 2ll * groups && a_rows <= 128ll * groups) a.ahead = (int)((long long)groups * ((a.N + 255) / 256) < (1 << 30) ? groups * ((a.N + 255) / 256) : 1 << 30);
  return launch_large<false, 4, GATED, true, false>(A, a_rows, W, (long long)groups * a.N, a, st);
}

static bool fp8_aligned(const void* a, const void* b, const void* c, const void* d) {
  return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c) | reinterpret_cast<uintptr_t>(d)) & 15) == 0;
}

// what all products ask of their arguments
static int check_product(const char* what, const void* A, const float* as, int ld_as, const void* W, const float* ws, const void* C, int M, int N,
                         int K, bool gated) {
  B200Q_CHECK_ARG(M >= 0 && N > 0 && K > 0 && K % 16 == 0 && N % (gated ? 256 : 8) == 0 && M <= FP8_MOST && N <= FP8_MOST && K <= FP8_MOST,
                  "%s: unsupported shape M=%d N=%d K=%d (K%%16==0, N%%%d==0, each up to 2^31 - 1024)", what, M, N, K, gated ? 256 : 8);
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
  B200Q_CHECK_ARG(groups > 0 && max_mtiles >= 0 && (long long)groups * N <= FP8_MOST, "gemm_grouped_fp8: groups=%d max_mtiles=%d", groups, max_mtiles);
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
  B200Q_CHECK_ARG(groups > 0 && max_mtiles >= 0 && (long long)groups * N <= FP8_MOST, "gemm_grouped_gated_fp8: groups=%d max_mtiles=%d", groups, max_mtiles);
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

// test hook: 0 = by size, 1 = small tiles, 2 = large tiles of single CTAs, 3 = of pairs; 4 and 5 = these in mode / 100 parts of the reduction.
// mode / 10 % 10: 64 columns each to a dense product's tile, 0 and what there is no kernel of = 4 (2: single CTAs; 3: pairs; parts: 2 or 3 for
// single CTAs, 4 for pairs)
int b200q_gemm_fp8_set_mode(int mode) {
  const int kind = mode % 10, ch = mode / 10 % 10, splits = mode / 100;
  B200Q_CHECK_ARG(mode >= 0 && kind <= 5 && (ch == 0 || (ch >= 2 && ch <= 4)) && splits <= (kind == 5 ? FL_MAX_SPLITS / 2 : FL_MAX_SPLITS) && (splits > 0) == (kind >= 4),
                  "gemm_fp8_set_mode: mode=%d", mode);
  g_fp8_mode = mode;
  bump_tuning_epoch();
  return B200Q_OK;
}

// test hook: n > 0 = every warp of products gives up before its n-th block (b200q_wait_failures says so; what large
// tiles had no sums for is not stored, small ones are wrong) and waits of pairs last some 100 us, 0 = normal
int b200q_gemm_fp8_set_give_up(int n) {
  B200Q_CHECK_ARG(n >= 0, "gemm_fp8_set_give_up: n=%d", n);
  g_fp8_give_up = n;
  bump_tuning_epoch();
  return B200Q_OK;
}

// test hook: the mode that stands for what a dense product takes
int b200q_gemm_fp8_choice(int M, int N, int K, int gated) {
  const Fp8Tile t = gated ? choose_fp8_tile<true>(M, N, (K + FP8_BLOCK - 1) / FP8_BLOCK) : choose_fp8_tile<false>(M, N, (K + FP8_BLOCK - 1) / FP8_BLOCK);
  return t.kind == 1 ? 1 : t.kind + 10 * t.ch + (t.splits > 1 ? 100 * t.splits : 0);
}

}  // extern "C"
