// pages.cu — pages of a paged cache between sequences: forks, ends, copies and moves.
//
// A cache's pages are numbered; a sequence's row of the block table names its pages; refs[p] says how many rows hold page p, 0: it is free.
// That is all the state there is, so that a step's selection of beams needs no answer from the GPU before the next step can be enqueued.
//   fork     rows become continuations of other rows.  Pages are shared; the page that a row's next token goes to is its own: the lowest free
//            one where the old ones are full, the old last one for its first continuation if nobody else holds it, a copy for all others.
//   free     rows end.
//   copy     pages (all layers) as a list of pairs says.
//   compact  the pages in use move to the front of the pool, as few of them as that takes.
// Bound: fork and compact by latency (chains of a few dependent reads; a cluster of CTAs works on all rows and all pages at once, its
// barriers between the steps), copies by the pages' bytes.  Results follow from the arguments alone: page numbers are given out in order of
// rows and pages, counts change by atomic additions of whole numbers.
// 24 searches of 6 beams of 50 to 900 tokens, 16 layers of 8 heads of 128: fork 10 us, its copies 18 (their bytes 15); of 5 rows 5 and 2.5.
// 20000 pages moved: 10 us for the plan, 184 for the pages (171).
#include "layered_common.cuh"
#include "tcgen05.cuh"

namespace b200q {

constexpr int PG_THREADS = 1024, PG_CTAS = 8, PG_ROWS = 8192, PG_BLOCK = 16;

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// sum over the threads before this one, and over all (every thread of the CTA calls it)
__device__ __forceinline__ int block_prefix(int v, int* total, int* scratch /* 33 */) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) scratch[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int s = lane < (int)blockDim.x / 32 ? scratch[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    scratch[lane] = s;
  }
  __syncthreads();
  const int before = (warp ? scratch[warp - 1] : 0) + x - v;
  *total = scratch[31];
  __syncthreads();
  return before;
}

// pages of a row of len tokens (lengths beyond the table's width count as its width; len + 15 may pass 2^31)
__device__ __forceinline__ int pages_held(int len, int stride) {
  const int n = max(len, 0);
  return min(n / PG_BLOCK + (n % PG_BLOCK != 0), stride);
}

// the share of [0, n) of this CTA of the cluster, cut at multiples of 4 (refs is read four at a time)
struct PageShare {
  int from, to;
  __device__ __forceinline__ PageShare(int n) {
    const int per = ((n + (int)gridDim.x - 1) / (int)gridDim.x + 3) / 4 * 4;
    from = min(n, (int)blockIdx.x * per);
    to = min(n, from + per);
  }
};
// pages p .. p + 3 (those in [.., to)): their counts, others -1
__device__ __forceinline__ int4 counts_of(const int32_t* refs, int p, int to, bool vec) {
  if (vec && p + 4 <= to) return *reinterpret_cast<const int4*>(refs + p);
  return make_int4(p < to ? refs[p] : -1, p + 1 < to ? refs[p + 1] : -1, p + 2 < to ? refs[p + 2] : -1, p + 3 < to ? refs[p + 3] : -1);
}

// one number per CTA of the cluster: the sums of those before this CTA and of all (every thread calls it; box: two ints, `turn` 0, 1, ...)
__device__ __forceinline__ int cluster_prefix(int v, int* total, int* box, int turn) {
  if (gridDim.x == 1) {
    *total = v;
    return 0;
  }
  if (threadIdx.x == 0) box[turn & 1] = v;
  cluster_sync_all();
  int before = 0, all = 0;
  for (int c = 0; c < (int)gridDim.x; ++c) {
    const int x = (int)ld_cluster_u32(mapa_shared(box + (turn & 1), c));
    before += c < (int)blockIdx.x ? x : 0;
    all += x;
  }
  *total = all;
  return before;
}
__device__ __forceinline__ void rows_sync() {
  if (gridDim.x == 1)
    __syncthreads();
  else
    cluster_sync_all();
}

// entries 0 .. n - 1 of a table, eight of a thread at once: what `read` gives for those of (row, column) goes to `write`, unless it is NO_ENTRY
constexpr int NO_ENTRY = -0x7fffffff - 1;
template <typename R, typename W>
__device__ __forceinline__ void for_entries(int n, int stride, int at, int threads, R&& read, W&& write) {
  for (int e0 = at; e0 < n; e0 += 8 * threads) {
    int v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int e = e0 + u * threads, i = e / stride;
      v[u] = e < n ? read(i, e - i * stride) : NO_ENTRY;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (v[u] != NO_ENTRY) write(e0 + u * threads, v[u]);
  }
}

struct ForkArgs {
  const int32_t *table, *lens, *parents;
  int32_t *refs, *table_out, *slots;
  int2* pairs;
  int32_t* status;
  int n_old, n_new, stride, num_blocks;
};

__global__ void __launch_bounds__(PG_THREADS, 1) pages_fork_kernel(ForkArgs a) {
  follow_previous(a.table, a.lens, a.parents, a.refs, a.table_out, a.slots, a.pairs, a.status);
  extern __shared__ int32_t rows[];
  // per old row: its first continuation, how many, its length; per new row: its parent (-1: none); the new rows that need a page, in order
  int32_t *first = rows, *count = first + a.n_old, *lens = count + a.n_old, *parent = lens + a.n_old, *fresh = parent + a.n_new;
  __shared__ int scratch[33], box[2], no_column_s;
  const int tid = threadIdx.x, nt = blockDim.x;
  const int most = a.stride * PG_BLOCK;
  // counts of this CTA's share of the pages, asked for before anything else; of a share that is one round of the threads they stay in registers
  const PageShare share(a.num_blocks);
  const bool vec = (reinterpret_cast<uintptr_t>(a.refs) & 15) == 0, one_round = share.to - share.from <= 4 * nt;
  const int p_mine = share.from + 4 * tid;
  const int4 c_mine = one_round && p_mine < share.to ? counts_of(a.refs, p_mine, share.to, vec) : make_int4(-1, -1, -1, -1);
  for (int i = tid; i < a.n_old; i += nt) {
    first[i] = 0x7fffffff;
    count[i] = 0;
    lens[i] = min(max(a.lens[i], 0), most);
  }
  for (int i = tid; i < a.n_new; i += nt) {
    const int p = a.parents[i];
    parent[i] = p >= 0 && p < a.n_old ? p : -1;
  }
  if (tid == 0) no_column_s = 0;
  __syncthreads();
  for (int i = tid; i < a.n_new; i += nt)
    if (parent[i] >= 0) {
      atomicMin(first + parent[i], i);
      atomicAdd(count + parent[i], 1);
    }
  __syncthreads();
  // ---- who needs a page (every CTA finds this out for all rows: it is a few reads per row, and nobody has to be told)
  int n_fresh = 0;
  for (int i0 = 0; i0 < a.n_new; i0 += nt) {
    const int i = i0 + tid, p = i < a.n_new ? parent[i] : -1;
    bool need = false;
    if (p >= 0) {
      const int len = lens[p], last = len / PG_BLOCK;
      if (last >= a.stride) {
        if (blockIdx.x == 0) atomicAdd(&no_column_s, 1);
      } else if (len % PG_BLOCK == 0) {
        need = true;
      } else {
        const int page = a.table[p * a.stride + last];
        need = !(first[p] == i && page >= 0 && page < a.num_blocks && a.refs[page] == 1);
      }
    }
    int all;
    const int before = block_prefix(need, &all, scratch);
    if (need) fresh[n_fresh + before] = i;
    n_fresh += all;
  }
  // ---- the free pages of this CTA's share, and of all
  auto free_in = [](int4 c) { return (c.x == 0) + (c.y == 0) + (c.z == 0) + (c.w == 0); };
  int mine = free_in(c_mine);
  if (!one_round)
    for (int p = p_mine; p < share.to; p += 4 * nt) mine += free_in(counts_of(a.refs, p, share.to, vec));
  int here, free_all;
  const int before_mine = block_prefix(mine, &here, scratch);
  int rank = cluster_prefix(here, &free_all, box, 0);
  const bool enough = free_all >= n_fresh;
  if (blockIdx.x == 0 && tid == 0) {
    a.status[0] = enough ? 0 : n_fresh - free_all;
    a.status[1] = no_column_s;
  }
  if (!enough) {  // nothing changes, and nobody has a place to write to
    for (int i = blockIdx.x * nt + tid; i < a.n_new; i += gridDim.x * nt) {
      a.slots[i] = -1;
      a.pairs[i] = make_int2(-1, -1);
    }
    if (gridDim.x > 1) cluster_sync_all();  // (a peer may still read this CTA's number)
    return;
  }
  // ---- the k-th free page goes to the k-th row that needs one
  auto give = [&](int p, int4 c4, int k) {  // those of pages p .. p + 3 that are free, the first of them the k-th of all
    const int c[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (c[x] == 0) {
        if (k < n_fresh) {
          const int i = fresh[k], from = parent[i], len = lens[from], last = len / PG_BLOCK;
          a.refs[p + x] = 1;
          a.table_out[i * a.stride + last] = p + x;
          a.slots[i] = (p + x) * PG_BLOCK + len % PG_BLOCK;
          a.pairs[i] = len % PG_BLOCK ? make_int2(a.table[from * a.stride + last], p + x) : make_int2(-1, -1);
        }
        ++k;
      }
  };
  if (one_round) {
    if (rank < n_fresh) give(p_mine, c_mine, rank + before_mine);
  } else {
    for (int p0 = share.from; p0 < share.to && rank < n_fresh; p0 += 4 * nt) {
      const int p = p0 + 4 * tid;
      const int4 c = p < share.to ? counts_of(a.refs, p, share.to, vec) : make_int4(-1, -1, -1, -1);
      int all;
      const int k = block_prefix(free_in(c), &all, scratch);
      give(p, c, rank + k);
      rank += all;
    }
  }
  rows_sync();  // all free pages have been looked for: counts may change
  // ---- tables of the new rows, slots of those that keep a page; then what the old rows' pages gain and lose
  auto is_fresh = [&](int i) {  // (decided by counts that have changed since: the list of the rows that need a page says it)
    int lo = 0, hi = n_fresh;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (fresh[mid] < i)
        lo = mid + 1;
      else
        hi = mid;
    }
    return lo < n_fresh && fresh[lo] == i;
  };
  const int at = blockIdx.x * nt + tid, threads = gridDim.x * nt;
  for_entries(a.n_new * a.stride, a.stride, at, threads, [&](int i, int c) {
    const int p = parent[i];
    return p >= 0 && c < lens[p] / PG_BLOCK ? a.table[p * a.stride + c] : NO_ENTRY;
  }, [&](int e, int page) { a.table_out[e] = page; });
  for (int i = at; i < a.n_new; i += threads) {
    const int p = parent[i], len = p >= 0 ? lens[p] : 0, last = len / PG_BLOCK;
    if (p < 0 || last >= a.stride) {
      a.slots[i] = -1;
      a.pairs[i] = make_int2(-1, -1);
    } else if (len % PG_BLOCK && !is_fresh(i)) {
      const int page = a.table[p * a.stride + last];
      a.table_out[i * a.stride + last] = page;
      a.slots[i] = page * PG_BLOCK + len % PG_BLOCK;
      a.pairs[i] = make_int2(-1, -1);
    }
  }
  // (both loops go through the old table: an entry counts for how many rows more or fewer hold its page now)
  for_entries(a.n_old * a.stride, a.stride, at, threads, [&](int p, int c) {
    const bool counts = count[p] != 1 && c < lens[p] / PG_BLOCK;
    return counts ? a.table[p * a.stride + c] : NO_ENTRY;
  }, [&](int e, int page) {
    if (page >= 0 && page < a.num_blocks) atomicAdd(a.refs + page, count[e / a.stride] - 1);
  });
  for (int p = at; p < a.n_old; p += threads)
    if (lens[p] % PG_BLOCK && !(count[p] > 0 && !is_fresh(first[p]))) {
      const int page = a.table[p * a.stride + lens[p] / PG_BLOCK];
      if (page >= 0 && page < a.num_blocks) atomicAdd(a.refs + page, -1);
    }
  if (gridDim.x > 1) cluster_sync_all();  // (nobody leaves while a peer may read its number)
}

// A warp to a row.
__global__ void __launch_bounds__(256) pages_free_kernel(const int32_t* table, const int32_t* lens, const int32_t* ends, int n, int stride,
                                                         int32_t* refs, int num_blocks) {
  follow_previous(table, lens, ends, refs);
  const int lane = threadIdx.x & 31;
  for (int r = blockIdx.x * 8 + (threadIdx.x >> 5); r < n; r += gridDim.x * 8) {
    if (ends && ends[r] == 0) continue;
    const int pages = pages_held(lens[r], stride);
    for (int c = lane; c < pages; c += 32) {
      const int p = table[(long long)r * stride + c];
      if (p >= 0 && p < num_blocks) atomicAdd(refs + p, -1);
    }
  }
}

// An item is COPY_BYTES of one layer's page (the last one of a page may be shorter): eight pieces of 16 bytes per thread on their way at once.
constexpr int COPY_THREADS = 256, COPY_AT_ONCE = 8, COPY_BYTES = COPY_THREADS * COPY_AT_ONCE * 16;
__global__ void __launch_bounds__(COPY_THREADS) pages_copy_kernel(uint8_t* kv, const int2* pairs, const int32_t* count, int n, long long page_bytes,
                                                                  int n_layers, long long layer_stride, int num_blocks) {
  follow_previous(kv, pairs, count);
  const int parts = (int)((page_bytes + COPY_BYTES - 1) / COPY_BYTES);
  const long long items = (long long)(count ? min(max(count[0], 0), n) : n) * n_layers * parts;
  for (long long it = blockIdx.x; it < items; it += gridDim.x) {
    const int part = (int)(it % parts), layer = (int)(it / parts % n_layers);
    const int2 pr = pairs[it / parts / n_layers];
    if (pr.x < 0 || pr.y < 0 || pr.x >= num_blocks || pr.y >= num_blocks) continue;
    uint8_t* base = kv + layer * layer_stride + (long long)part * COPY_BYTES;
    const uint4* from = reinterpret_cast<const uint4*>(base + pr.x * page_bytes);
    uint4* to = reinterpret_cast<uint4*>(base + pr.y * page_bytes);
    const int pieces = (int)min((long long)COPY_BYTES, page_bytes - (long long)part * COPY_BYTES) / 16;
    uint4 v[COPY_AT_ONCE];
#pragma unroll
    for (int u = 0; u < COPY_AT_ONCE; ++u)
      if (u * COPY_THREADS + (int)threadIdx.x < pieces) v[u] = ld_once_v4(from + u * COPY_THREADS + threadIdx.x);
#pragma unroll
    for (int u = 0; u < COPY_AT_ONCE; ++u)
      if (u * COPY_THREADS + (int)threadIdx.x < pieces) st_v4(to + u * COPY_THREADS + threadIdx.x, v[u]);
  }
}

struct CompactArgs {
  const int32_t *table, *lens, *refs;
  int32_t *table_out, *refs_out, *map;
  int2* pairs;
  int32_t* status;
  int n_rows, stride, num_blocks;
};

// n pages are in use.  Of two counts of pages in use, before page p and before page n, follow the places: free page p < n is number
// p - before(p) of those that are filled, page p >= n in use is number before(p) - before(n) of those that fill them.
__global__ void __launch_bounds__(PG_THREADS, 1) pages_compact_kernel(CompactArgs a) {
  follow_previous(a.table, a.lens, a.refs, a.table_out, a.refs_out, a.map, a.pairs, a.status);
  __shared__ int scratch[33], box[2];
  const int tid = threadIdx.x, nt = blockDim.x;
  const PageShare share(a.num_blocks);
  const bool vec = (reinterpret_cast<uintptr_t>(a.refs) & 15) == 0;
  int mine = 0;
  for (int p = share.from + 4 * tid; p < share.to; p += 4 * nt) {
    const int4 c = counts_of(a.refs, p, share.to, vec);
    mine += (c.x > 0) + (c.y > 0) + (c.z > 0) + (c.w > 0);
  }
  int here, n, below_all;
  block_prefix(mine, &here, scratch);
  int before = cluster_prefix(here, &n, box, 0);
  int below = 0;
  for (int p = share.from + 4 * tid; p < min(share.to, n); p += 4 * nt) {
    const int4 c = counts_of(a.refs, p, min(share.to, n), vec);
    below += (c.x > 0) + (c.y > 0) + (c.z > 0) + (c.w > 0);
  }
  block_prefix(below, &here, scratch);
  cluster_prefix(here, &below_all, box, 1);
  const int moves = n - below_all;
  if (blockIdx.x == 0 && tid == 0) {
    a.status[0] = n;
    a.status[1] = moves;
  }
  for (int p0 = share.from; p0 < share.to; p0 += 4 * nt) {
    const int p = p0 + 4 * tid;
    const int4 c4 = p < share.to ? counts_of(a.refs, p, share.to, vec) : make_int4(-1, -1, -1, -1);
    const int c[4] = {c4.x, c4.y, c4.z, c4.w};
    int all;
    int k = before + block_prefix((c[0] > 0) + (c[1] > 0) + (c[2] > 0) + (c[3] > 0), &all, scratch);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int id = p + x;
      if (id >= share.to || p >= share.to) continue;
      if (c[x] > 0) {
        if (id < n) {
          a.map[id] = id;
          a.refs_out[id] = c[x];
        } else {
          a.pairs[k - below_all].x = id;
        }
        ++k;
      } else {
        a.map[id] = -1;
        if (id < n)
          a.pairs[id - k].y = id;
        else
          a.refs_out[id] = 0;
      }
    }
    before += all;
  }
  rows_sync();
  const int at = blockIdx.x * nt + tid, threads = gridDim.x * nt;
  for (int k = at; k < moves; k += threads) {
    const int2 pr = a.pairs[k];
    a.map[pr.x] = pr.y;
    a.refs_out[pr.y] = a.refs[pr.x];
    a.refs_out[pr.x] = 0;  // (refs_out may be refs)
  }
  rows_sync();
  for_entries(a.n_rows * a.stride, a.stride, at, threads, [&](int r, int c) {
    if (c >= pages_held(a.lens[r], a.stride)) return NO_ENTRY;
    const int p = a.table[r * a.stride + c];
    return p >= 0 && p < a.num_blocks ? a.map[p] : -1;
  }, [&](int e, int page) { a.table_out[e] = page; });
}

// CTAs and their threads: one where a thread has a few pages and a few entries, a cluster of 8 above that; a barrier of few warps is shorter, so
// 256 threads where there is about a page and an entry or so to each.  us for fork / compact with 1 x 256, 1 x 1024, 8 x 256, 8 x 1024:
//   538 pages, 148 entries     5.2 / 4.1     6.0 / 4.8     7.1 / 7.2     8.4 / 8.6
//   2304 pages, 1184 entries   7.6 / 7.7     7.3 / 6.1     8.1 / 7.4     9.9 / 9.0
//   3008 pages, 5328 entries   14.6 / 14.8   10.3 / 8.7    9.1 / 8.1     10.6 / 9.1
//   10432 pages, 9472 entries  23.5 / 31.3   16.3 / 17.7   11.5 / 11.1   11.4 / 10.7
//   32432 pages, 9472 entries  30.1 / 62.4   18.0 / 36.2   13.0 / 16.0   11.5 / 13.2
static int page_ctas(int num_blocks, long long entries) { return num_blocks <= 4096 && entries <= 2048 ? 1 : PG_CTAS; }
static int page_threads(int num_blocks, long long entries, int ctas) {
  return num_blocks <= 1024 * ctas && entries <= 1024 * ctas ? 256 : PG_THREADS;
}
constexpr long long PG_ENTRIES = 0x7fffffff - 8 * PG_CTAS * PG_THREADS;  // of a block table

}  // namespace b200q

using namespace b200q;

extern "C" {

int b200q_pages_fork(const int32_t* table, const int32_t* lens, int n_old, const int32_t* parents, int n_new, int bt_stride, int32_t* refs,
                     int num_blocks, int block_size, int32_t* table_out, int32_t* slots, int32_t* pairs, int32_t* status, void* stream) {
  B200Q_CHECK_ARG(n_old >= 0 && n_new >= 0 && n_old <= PG_ROWS && n_new <= PG_ROWS && bt_stride > 0 && bt_stride <= (1 << 26) && num_blocks > 0 &&
                      num_blocks <= (1 << 27) && block_size == PG_BLOCK,
                  "pages_fork: bad shape n_old=%d n_new=%d (up to %d) bt_stride=%d num_blocks=%d block_size=%d (16)", n_old, n_new, PG_ROWS, bt_stride,
                  num_blocks, block_size);
  B200Q_CHECK_ARG((long long)n_old * bt_stride <= PG_ENTRIES && (long long)n_new * bt_stride <= PG_ENTRIES, "pages_fork: tables of more than 2^31 entries");
  B200Q_CHECK_ARG(refs && status && (n_old == 0 || (table && lens)) && (n_new == 0 || (parents && table_out && slots && pairs)),
                  "pages_fork: null argument");
  B200Q_CHECK_ARG(n_old == 0 || n_new == 0 ||
                      !(table_out < table + (long long)n_old * bt_stride && table < table_out + (long long)n_new * bt_stride),
                  "pages_fork: the new table must not overlap the old one");
  B200Q_CHECK_ARG((reinterpret_cast<uintptr_t>(pairs) & 7) == 0, "pages_fork: pairs must be 8-byte aligned");
  const size_t smem = (3 * (size_t)n_old + 2 * (size_t)n_new) * 4;
  static bool ready[64];
  int dev = 0;
  B200Q_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !ready[dev]) {
    B200Q_CUDA(cudaFuncSetAttribute(pages_fork_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 5 * PG_ROWS * 4));
    if (dev < 64) ready[dev] = true;
  }
  const int ctas = page_ctas(num_blocks, (long long)(n_old > n_new ? n_old : n_new) * bt_stride);
  const ForkArgs a{table, lens, parents, refs, table_out, slots, (int2*)pairs, status, n_old, n_new, bt_stride, num_blocks};
  B200Q_CUDA(launch_early(pages_fork_kernel, dim3(ctas), page_threads(num_blocks, (long long)(n_old > n_new ? n_old : n_new) * bt_stride, ctas), smem, as_stream(stream), ctas, a));
  count_launch();
  return B200Q_OK;
}

int b200q_pages_free(const int32_t* table, const int32_t* lens, const int32_t* ends, int n_rows, int bt_stride, int32_t* refs, int num_blocks,
                     int block_size, void* stream) {
  B200Q_CHECK_ARG(n_rows >= 0 && bt_stride >= 0 && num_blocks > 0 && num_blocks <= (1 << 27) && block_size == PG_BLOCK,
                  "pages_free: bad shape n_rows=%d bt_stride=%d num_blocks=%d block_size=%d (16)", n_rows, bt_stride, num_blocks, block_size);
  if (n_rows == 0 || bt_stride == 0) return B200Q_OK;
  B200Q_CHECK_ARG(table && lens && refs, "pages_free: null argument");
  const int blocks = (n_rows + 7) / 8;
  B200Q_CUDA(launch_early(pages_free_kernel, dim3(blocks < 4096 ? blocks : 4096), 256, 0, as_stream(stream), 1, table, lens, ends, n_rows, bt_stride, refs,
                          num_blocks));
  count_launch();
  return B200Q_OK;
}

int b200q_pages_copy(void* kv, const int32_t* pairs, int n_pairs, const int32_t* count, int64_t page_bytes, int n_layers, int64_t layer_stride,
                     int num_blocks, void* stream) {
  B200Q_CHECK_ARG(n_pairs >= 0 && page_bytes > 0 && page_bytes % 16 == 0 && page_bytes < (1ll << 31) && n_layers >= 0 && layer_stride % 16 == 0 &&
                      num_blocks > 0,
                  "pages_copy: bad shape n_pairs=%d page_bytes=%lld n_layers=%d layer_stride=%lld num_blocks=%d (bytes in multiples of 16)", n_pairs,
                  (long long)page_bytes, n_layers, (long long)layer_stride, num_blocks);
  if (n_pairs == 0 || n_layers == 0) return B200Q_OK;
  B200Q_CHECK_ARG(kv && pairs, "pages_copy: null argument");
  B200Q_CHECK_ARG((reinterpret_cast<uintptr_t>(kv) & 15) == 0 && (reinterpret_cast<uintptr_t>(pairs) & 7) == 0,
                  "pages_copy: the cache must be 16-byte aligned, pairs 8-byte");
  const long long items = (long long)n_pairs * n_layers * ((page_bytes + COPY_BYTES - 1) / COPY_BYTES);
  const long long most = 8LL * num_sms();
  B200Q_CUDA(launch_early(pages_copy_kernel, dim3((unsigned)(items < most ? items : most)), COPY_THREADS, 0, as_stream(stream), 1, (uint8_t*)kv,
                          (const int2*)pairs, count, n_pairs, (long long)page_bytes, n_layers, (long long)layer_stride, num_blocks));
  count_launch();
  return B200Q_OK;
}

int b200q_pages_compact(const int32_t* table, const int32_t* lens, int n_rows, int bt_stride, const int32_t* refs, int num_blocks, int block_size,
                        int32_t* table_out, int32_t* refs_out, int32_t* map, int32_t* pairs, int32_t* status, void* stream) {
  B200Q_CHECK_ARG(n_rows >= 0 && bt_stride >= 0 && bt_stride <= (1 << 26) && num_blocks > 0 && num_blocks <= (1 << 27) && block_size == PG_BLOCK,
                  "pages_compact: bad shape n_rows=%d bt_stride=%d num_blocks=%d block_size=%d (16)", n_rows, bt_stride, num_blocks, block_size);
  B200Q_CHECK_ARG((long long)n_rows * bt_stride <= PG_ENTRIES, "pages_compact: a table of more than 2^31 entries");
  B200Q_CHECK_ARG(refs && refs_out && map && pairs && status && (n_rows == 0 || bt_stride == 0 || (table && lens && table_out)),
                  "pages_compact: null argument");
  B200Q_CHECK_ARG((reinterpret_cast<uintptr_t>(pairs) & 7) == 0, "pages_compact: pairs must be 8-byte aligned");
  const int ctas = page_ctas(num_blocks, (long long)n_rows * bt_stride);
  const CompactArgs a{table, lens, refs, table_out, refs_out, map, (int2*)pairs, status, bt_stride > 0 ? n_rows : 0, bt_stride, num_blocks};
  B200Q_CUDA(launch_early(pages_compact_kernel, dim3(ctas), page_threads(num_blocks, (long long)n_rows * bt_stride, ctas), 0, as_stream(stream), ctas, a));
  count_launch();
  return B200Q_OK;
}

}  // extern "C"
