// Page tables of a paged cache on the device: rows that take over other rows' pages, room for further tokens, pages that fall free, and pages that move to
// the front of the cache.  A page may be held by several rows; refs[page] counts them.  A page that is not full yet belongs to one row: when several rows
// take it over, the first keeps it and the others get copies of the tokens in it.
//
// Two launches: one cluster that works the tables out (its blocks meet three times; atomics on integers only, so that nothing hangs on their order), and a
// kernel that copies what it listed, in all layers of all caches.
//
// Free pages are given out lowest number first, to rows in their order, to a row first the page for a copy.  All or nothing: if pages or columns run short
// nothing changes and the status says so: that stays, and the pool as it is, until the caller has cleared those words, so that a loop that never asks cannot lose
// it.  Meanwhile `live` tells the kernels behind a step that its rows have no tokens: nothing is appended, nothing read.
//
// What bounds it: the tables a chain of dependent loads and meetings (a step of 64 rows 7 us, a chain of such steps; 16 continuations of a prompt of 8000 tokens 8),
// the contents HBM: tails of a step, 57 MB, 10 us beside a floor of 8.9; 140 pages of 2.1 MB
// that move, 587 MB read and written, 91 of 97.5 us in all (6.4 TB/s).
#include "../../include/vb_api.h"
#define VB_PDL_FAMILY 4
#include "rowmma.cuh"

namespace vb {

constexpr int PG_THREADS = 1024, PG_FEW_THREADS = 512, PG_FEW_CELLS = 16384, PG_MAX_CLUSTER = 8, PG_MAX_ROWS = 4096, PG_STAGE = 8192, PG_SMEM_PAGES = 8192;

// words of a pool's status
enum { PS_MISSING = 0, PS_LONG = 1, PS_COPIES = 2, PS_USED = 3 };

__device__ __forceinline__ int ldcg(const int32_t* p) { return __ldcg(p); }

// exclusive prefix over the block of two numbers a thread; totals in all threads.  `sums`: 33 words
template <int THREADS>
__device__ __forceinline__ int2 block_prefix(int2 mine, int2* sums, int2& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int2 inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, inc.x, o), y = __shfl_up_sync(0xffffffffu, inc.y, o);
    if (lane >= o) inc.x += x, inc.y += y;
  }
  __syncthreads();                                   // (the last call's sums have been read)
  if (lane == 31) sums[warp] = inc;
  __syncthreads();
  const int2 s = THREADS == 1024 || lane < THREADS / 32 ? sums[lane] : make_int2(0, 0);
  const int2 before = make_int2(__reduce_add_sync(0xffffffffu, lane < warp ? s.x : 0), __reduce_add_sync(0xffffffffu, lane < warp ? s.y : 0));
  total = make_int2(__reduce_add_sync(0xffffffffu, s.x), __reduce_add_sync(0xffffffffu, s.y));
  return make_int2(before.x + inc.x - mine.x, before.y + inc.y - mine.y);
}

struct ForkParams {
  const int32_t *table, *tokens, *refs;              // the pool as it is
  int32_t *out_table, *out_tokens, *out_refs;        // as it becomes (may be the same)
  int32_t *status, *copies, *work, *free;            // of the pool that is written: copies [rows][3]; scratch work / free [pages], where these are not in shared memory
  const int32_t* was;                                // status of the pool as it is
  int32_t* live;                                     // of the pool that is written, or null: tokens, 0 while it is short
  const int32_t *src, *grow;                         // row that every row continues (null: itself; < 0: none), tokens it gets room for (null: grow_all)
  int rows, columns, pages, page_size, group, grow_all, in_smem;
};

// the row that row i continues; -1: none
__device__ __forceinline__ int fork_source(const ForkParams& p, int i) {
  if (!p.src) return i;
  int s = p.src[i];
  if (s < 0) return -1;
  if (p.group > 0) {
    if (s >= p.group) return -1;
    s += i / p.group * p.group;
  }
  return s < p.rows ? s : -1;
}
__device__ __forceinline__ int fork_tokens(const ForkParams& p, int row) {
  const int n = ldcg(p.tokens + row);
  return n < 0 ? 0 : n < p.columns * p.page_size ? n : p.columns * p.page_size;
}
// (a page number of the table, or -1 where it names none: the tables are the caller's memory)
__device__ __forceinline__ int fork_page(const ForkParams& p, int row, int col) {
  const int g = ldcg(p.table + static_cast<long long>(row) * p.columns + col);
  return g >= 0 && g < p.pages ? g : -1;
}

// the same place in block 0's shared memory, as an ordinary address
template <typename T>
__device__ __forceinline__ T* in_block0(T* p) {
  T* r;
  asm("mapa.u64 %0, %1, 0;" : "=l"(r) : "l"(p));
  return r;
}

// What is known of a row stands in every block's shared memory.  A row that k rows continue adds k - 1 to the count of each of its pages, once a page and not
// once a row that takes it over.  Counts and free pages stand in block 0's shared memory for pools of up to PG_SMEM_PAGES pages (scratch in global memory
// beyond: a step of 64 rows took 13.0 us with it, 11.4 without, each launch by itself), and are volatile to every block.
template <int THREADS>
__global__ void __launch_bounds__(THREADS, 1) fork_pages_kernel(const __grid_constant__ ForkParams p) {
  constexpr int LOG_THREADS = THREADS == 1024 ? 10 : 9;
  static_assert(THREADS == 1 << LOG_THREADS, "rows of the cluster's threads are powers of two");
  extern __shared__ int32_t pg_smem[];
  int32_t* s_src = pg_smem;                          // [rows] the row that a row continues, -1: none
  int32_t* s_grow = s_src + p.rows;                  // [rows] tokens it gets room for
  int32_t* s_tok = s_grow + p.rows;                  // [rows] tokens before the step
  int32_t* s_held = s_tok + p.rows;                  // [rows] ... and pages
  int32_t* s_heirs = s_held + p.rows;                // [rows] rows that continue it
  int32_t* s_keeper = s_heirs + p.rows;              // [rows] ... the first of them
  int32_t* s_tail = s_keeper + p.rows;               // [rows] page that the row copies, -1: none
  int32_t* s_base = s_tail + p.rows;                 // [rows] its first of the free pages, times two; 1: that one is for a copy
  int32_t* stage = s_base + p.rows;                  // PG_STAGE: new values of a block of columns
  __shared__ int2 sums[32];
  __shared__ int s_ok, s_copies;
  const int tid = threadIdx.x, rank = cluster_ctarank(), blocks = cluster_nctarank(), P = p.page_size;
  const int all = blocks * THREADS, mine = rank * THREADS + tid;
  volatile int32_t* work = p.in_smem ? in_block0(stage + PG_STAGE) : p.work;                // [pages] holders
  volatile int32_t* free = p.in_smem ? in_block0(stage + PG_STAGE + p.pages) : p.free;      // [pages needed] the lowest free ones
  volatile int32_t* base = in_block0(s_base);
  pdl_sync();
  const int ref = mine < p.pages ? p.refs[mine] : 0;      // (all loads of the start at once)
  const int was_missing = p.was[PS_MISSING], was_long = p.was[PS_LONG];      // an earlier step's: the pool has stood still since
  for (int i = tid; i < p.rows; i += THREADS) {
    const int s = fork_source(p, i), n = fork_tokens(p, i), g = p.grow ? p.grow[i] : p.grow_all;
    s_src[i] = s, s_grow[i] = g > 0 ? g : 0, s_tok[i] = n, s_held[i] = (n + P - 1) / P, s_heirs[i] = 0, s_keeper[i] = 0x7fffffff, s_tail[i] = -1;
  }
  if (tid == 0) s_copies = 0;
  if (blocks > 1) cluster_sync_all();                // (block 0 runs: its shared memory may be written)
  if (mine < p.pages) work[mine] = ref;
  for (int g = mine + all; g < p.pages; g += all) work[g] = p.refs[g];
  __syncthreads();
  for (int i = tid; i < p.rows; i += THREADS)
    if (s_src[i] >= 0) atomicAdd(s_heirs + s_src[i], 1), atomicMin(s_keeper + s_src[i], i);
  cluster_sync_all();

  // holders of every page after the step, from those before it
  const int log_x = min(LOG_THREADS, 32 - __clz(p.columns - 1)), x = 1 << log_x;      // (x neighbouring threads of the cluster a row)
  for (int s = mine >> log_x; s < p.rows; s += all >> log_x) {
    const int more = s_heirs[s] - 1, held = more ? s_held[s] : 0;
#pragma unroll 1
    for (int c = mine & (x - 1); c < held; c += x) {
      const int g = fork_page(p, s, c);
      if (g >= 0) atomicAdd(const_cast<int32_t*>(work) + g, more);
    }
  }
  if (rank == 0)
    for (int i = tid; i < p.rows; i += THREADS) {
      const int s = s_src[i], n = s < 0 ? 0 : s_tok[s];
      if (n % P && s_keeper[s] != i) s_tail[i] = fork_page(p, s, n / P);
    }
  cluster_sync_all();

  // (tokens after the step fit 32 bits: at most 2^30 and what a row may grow by)
  auto pages_after = [&](int s, int i) { return (static_cast<uint32_t>(s_tok[s]) + static_cast<uint32_t>(s_grow[i]) + P - 1u) / static_cast<uint32_t>(P); };
  if (rank == 0) {
    // pages that every row needs: one for a copy, the others for tokens
    int need_all = 0, too_long = 0;
    for (int i0 = 0; i0 < p.rows; i0 += THREADS) {
      const int i = i0 + tid, s = i < p.rows ? s_src[i] : -1;
      int need = 0, longer = 0, copy = 0;
      if (s >= 0) {
        const uint32_t want = pages_after(s, i);
        copy = s_tail[i] >= 0;
        longer = want > static_cast<uint32_t>(p.columns);
        need = longer ? 0 : copy + static_cast<int>(want) - s_held[s];
      }
      int2 total;
      const int2 before = block_prefix<THREADS>(make_int2(need, longer), sums, total);
      if (i < p.rows) s_base[i] = (need_all + before.x) * 2 + copy;
      need_all += total.x;
      too_long += total.y;
    }
    // the lowest free pages
    int have = 0;
    for (int g0 = 0; g0 < p.pages && have < need_all; g0 += 4 * THREADS) {
      int n[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int g = g0 + 4 * tid + j;
        n[j] = g < p.pages ? work[g] : 1;
      }
      int2 total;
      int at = have + block_prefix<THREADS>(make_int2((n[0] == 0) + (n[1] == 0) + (n[2] == 0) + (n[3] == 0), 0), sums, total).x;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n[j] == 0) {
          if (at < need_all) free[at] = g0 + 4 * tid + j;
          ++at;
        }
      have += total.x;
    }
    const bool stands = was_missing != 0 || was_long != 0, ok = !stands && have >= need_all && too_long == 0;
    __syncthreads();
    if (ok) {
      for (int k = tid; k < need_all; k += THREADS) work[free[k]] = 1;
      for (int i = tid; i < p.rows; i += THREADS)
        if (s_tail[i] >= 0) {
          int32_t* c = p.copies + 3ll * atomicAdd(&s_copies, 1);
          c[0] = s_tail[i], c[1] = free[s_base[i] >> 1], c[2] = s_tok[s_src[i]] % P;
          atomicSub(const_cast<int32_t*>(work) + s_tail[i], 1);
        }
      __syncthreads();
    }
    if (tid == 0) {
      s_ok = ok;
      p.status[PS_MISSING] = stands ? was_missing : have >= need_all ? 0 : need_all - have;
      p.status[PS_LONG] = stands ? was_long : too_long;
      p.status[PS_COPIES] = ok ? s_copies : 0;
    }
  }
  cluster_sync_all();

  const bool ok = *static_cast<volatile int*>(in_block0(&s_ok)) != 0;
  int32_t* s_want = s_keeper;                        // [rows] pages after the step
  for (int i = tid; i < p.rows; i += THREADS) {
    if (rank != 0) s_base[i] = base[i];
    s_want[i] = s_src[i] < 0 ? 0 : static_cast<int>(min(pages_after(s_src[i], i), static_cast<uint32_t>(p.columns)));
  }
  __syncthreads();
  if (ok || p.out_table != p.table) {               // (in place, not ok: nothing has been written)
    for (int g = mine; g < p.pages; g += all) p.out_refs[g] = ok ? work[g] : ldcg(p.refs + g);
    // A block of columns in all rows at a time, read before it is written: rows may take over one another's pages in place.  `across` neighbouring threads a
    // row, without a division an entry.
    const int wide = min((p.columns + blocks - 1) / blocks, max(1, PG_STAGE / p.rows));
    const int log_across = min(LOG_THREADS, 32 - __clz(wide - 1)), across = 1 << log_across, tx = tid & (across - 1), ty = tid >> log_across, down = THREADS >> log_across;
    for (int c0 = rank * wide; c0 < p.columns; c0 += blocks * wide) {
      const int w = min(wide, p.columns - c0);
      for (int k = tx; k < w; k += across) {
        const int c = c0 + k;
#pragma unroll 4
        for (int i = ty; i < p.rows; i += down) {
          const int s = ok ? s_src[i] : i;
          int v = -1;
          if (s >= 0) {
            const int held = ok ? s_held[s] : p.columns, b = ok ? s_base[i] : 0, copy = b & 1;
            if (c < held - copy) v = ldcg(p.table + static_cast<long long>(s) * p.columns + c);
            else if (c < (ok ? s_want[i] : 0)) v = free[(b >> 1) + (c < held ? 0 : copy + c - held)];
          }
          stage[i * w + k] = v;
        }
      }
      __syncthreads();
      for (int k = tx; k < w; k += across)
#pragma unroll 4
        for (int i = ty; i < p.rows; i += down) p.out_table[static_cast<long long>(i) * p.columns + c0 + k] = stage[i * w + k];
      __syncthreads();
    }
    // (tokens last: every block has read what it needs of them only at the start)
    for (int i = mine; i < p.rows; i += all) {
      const int s = s_src[i];
      p.out_tokens[i] = !ok ? ldcg(p.tokens + i) : s < 0 ? 0 : s_tok[s] + s_grow[i];
    }
  }
  if (p.live)
    for (int i = mine; i < p.rows; i += all) {
      const int s = ok ? s_src[i] : -1;
      p.live[i] = s < 0 ? 0 : s_tok[s] + s_grow[i];
    }
  if (blocks > 1) cluster_sync_all();                // (block 0's shared memory is read to the end)
}

struct CompactParams {
  const int32_t *table, *tokens, *refs;
  int32_t *out_table, *out_tokens, *out_refs, *moved;        // moved [pages]: a page's new number, -1: not in use
  int32_t *status, *copies;                                  // copies [pages][3]
  const int32_t* was;                                        // status of the pool as it is
  int32_t* live;                                             // (as for ForkParams)
  int32_t *from, *to;                                        // scratch [pages]
  long long cells;
  int rows, pages, page_size;
};

// The pages in use that stand behind as many places as there are pages in use move into the holes in front, in their order.
template <int THREADS>
__global__ void __launch_bounds__(THREADS, 1) compact_pages_kernel(const __grid_constant__ CompactParams p) {
  __shared__ int2 sums[32];
  const int tid = threadIdx.x, rank = cluster_ctarank(), blocks = cluster_nctarank();
  pdl_sync();
  if (rank == 0) {
    int used = 0;
    for (int g0 = 0; g0 < p.pages; g0 += 4 * THREADS) {
      int mine = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int g = g0 + 4 * tid + j;
        mine += g < p.pages && p.refs[g] > 0;
      }
      int2 total;
      block_prefix<THREADS>(make_int2(mine, 0), sums, total);
      used += total.x;
    }
    int holes = 0, movers = 0;
    for (int g0 = 0; g0 < p.pages; g0 += 4 * THREADS) {
      int n[2] = {0, 0}, what[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int g = g0 + 4 * tid + j;
        const bool in = g < p.pages && p.refs[g] > 0;
        what[j] = g >= p.pages ? -1 : in ? (g >= used ? 1 : -1) : (g < used ? 0 : -1);
        if (what[j] >= 0) ++n[what[j]];
        if (g < p.pages) p.moved[g] = in && g < used ? g : -1;
      }
      int2 total;
      const int2 before = block_prefix<THREADS>(make_int2(n[0], n[1]), sums, total);
      int h = holes + before.x, m = movers + before.y;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (what[j] == 0) p.to[h++] = g0 + 4 * tid + j;
        if (what[j] == 1) p.from[m++] = g0 + 4 * tid + j;
      }
      holes += total.x;
      movers += total.y;
    }
    __syncthreads();
    for (int k = tid; k < movers; k += THREADS) {      // (as many holes as movers)
      const int from = p.from[k], to = p.to[k];
      p.moved[from] = to;
      int32_t* c = p.copies + 3ll * k;
      c[0] = from, c[1] = to, c[2] = p.page_size;
    }
    if (tid == 0) p.status[PS_COPIES] = movers, p.status[PS_USED] = used;
  }
  cluster_sync_all();
  const long long at = static_cast<long long>(rank) * THREADS + tid, step = static_cast<long long>(blocks) * THREADS;
  for (long long e = at; e < p.cells; e += step) {
    const int g = p.table[e];
    p.out_table[e] = g >= 0 && g < p.pages ? ldcg(p.moved + g) : g;
  }
  const int was_missing = p.was[PS_MISSING], was_long = p.was[PS_LONG];
  if (at == 0 && p.status != p.was) p.status[PS_MISSING] = was_missing, p.status[PS_LONG] = was_long;      // (a shortage stands until it is cleared)
  for (long long i = at; i < p.rows; i += step) {
    const int n = p.tokens[i];
    p.out_tokens[i] = n;
    if (p.live) p.live[i] = was_missing != 0 || was_long != 0 ? 0 : n;
  }
  const int movers = ldcg(p.status + PS_COPIES), used = ldcg(p.status + PS_USED);
  if (p.out_refs != p.refs)
    for (long long g = at; g < p.pages; g += step)
      if (g >= used || p.refs[g] > 0) p.out_refs[g] = g < used ? p.refs[g] : 0;
  cluster_sync_all();                                     // (in place: what moves is read before it is cleared)
  for (long long k = at; k < movers; k += step) {
    const int from = ldcg(p.from + k), to = ldcg(p.to + k), n = p.refs[from];
    p.out_refs[to] = n;
    p.out_refs[from] = 0;
  }
}

// ---- contents of pages ------------------------------------------------------------------------------------------------------------
// A cache is [layers][pages][parts][slots][slot bytes] (keys | values: two parts).  copies[k] = (page, page, tokens): the first tokens of every part of the
// one go to the other.  A unit of work is 16 KB of a part of a copy in a layer.
constexpr int PC_CACHES = 32, PC_THREADS = 256, PC_UNIT = 1024;      // (vectors of a unit)
struct CopyCaches {
  uint4* at[PC_CACHES];
  long long layer[PC_CACHES], page[PC_CACHES], part[PC_CACHES];      // strides in vectors
  int layers[PC_CACHES], parts[PC_CACHES], slot[PC_CACHES], slots[PC_CACHES], units[PC_CACHES];      // vectors and slots of a part, units of a part
  long long first[PC_CACHES + 1];                                    // units of a copy in front
  int n, page_size;
};

__global__ void __launch_bounds__(PC_THREADS) copy_listed_pages_kernel(const __grid_constant__ CopyCaches t, const int32_t* copies, const int32_t* status) {
  pdl_sync();
  const int n = status[PS_COPIES];
  const long long per = t.first[t.n], all = per * n;
  for (long long u = blockIdx.x; u < all; u += gridDim.x) {
    const int k = static_cast<int>(u / per);
    long long r = u - k * per;
    int c = 0;
    while (c + 1 < t.n && t.first[c + 1] <= r) ++c;
    r -= t.first[c];
    const int chunk = static_cast<int>(r % t.units[c]);
    r /= t.units[c];
    const int part = static_cast<int>(r % t.parts[c]), layer = static_cast<int>(r / t.parts[c]);
    const int32_t* e = copies + 3ll * k;
    // (a part with other slots than a page's tokens -- blocks of tokens, say -- goes as a whole)
    const int slots = t.slots[c] == t.page_size ? min(e[2], t.slots[c]) : t.slots[c];
    const int end = min(slots * t.slot[c], (chunk + 1) * PC_UNIT);
    const long long in_layer = layer * t.layer[c] + part * t.part[c];
    const uint4* from = t.at[c] + in_layer + e[0] * t.page[c];
    uint4* to = t.at[c] + in_layer + e[1] * t.page[c];
    uint4 v[4];
    const int i0 = chunk * PC_UNIT + threadIdx.x;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i0 + j * PC_THREADS < end) v[j] = from[i0 + j * PC_THREADS];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i0 + j * PC_THREADS < end) to[i0 + j * PC_THREADS] = v[j];
  }
}

// Blocks of 256 threads an SM: whole pages move best with three (587 MB: 97.7 us; four 106.8, six 107.0, eight 109.5, two 110.9), the few tokens of a step's tails
// with six (57 MB: 19.6 us the whole step; three 21.3, eight 19.7).
constexpr int PC_WHOLE = 3, PC_TAILS = 6;
static int copy_listed(const VbPageCache* caches, int n_caches, const VbPagePool* pool, const int32_t* copies, const int32_t* status, int blocks, void* stream) {
  for (int c0 = 0; c0 < n_caches; c0 += PC_CACHES) {
    CopyCaches t = {};
    t.n = n_caches - c0 < PC_CACHES ? n_caches - c0 : PC_CACHES;
    t.page_size = pool->page_size;
    for (int c = 0; c < t.n; ++c) {
      const VbPageCache& s = caches[c0 + c];
      t.at[c] = static_cast<uint4*>(s.data);
      t.layers[c] = s.layers, t.parts[c] = s.parts, t.slots[c] = s.slots;
      t.slot[c] = static_cast<int>(s.slot_bytes / 16);
      t.part[c] = static_cast<long long>(s.slots) * t.slot[c];
      t.page[c] = t.part[c] * s.parts;
      t.layer[c] = t.page[c] * pool->pages;
      t.units[c] = static_cast<int>((t.part[c] + PC_UNIT - 1) / PC_UNIT);
      t.first[c + 1] = t.first[c] + static_cast<long long>(s.layers) * s.parts * t.units[c];
    }
    VB_LAUNCH_PDL(copy_listed_pages_kernel, sm_count() * blocks, PC_THREADS, 0, stream, t, copies, status);
  }
  return 0;
}

// Small tables take half as many threads a block: what is done once costs its instructions and meetings.  A step, 512 / 1024 threads: 44 cells 6.5 / 7.4 us, 8000 11.6 /
// 12.9, 16000 17.1 / 17.3, 34000 26.4 / 21.4, 130000 33.4 / 27.3.
static bool pg_few(long long cells, int pages) { return cells <= PG_FEW_CELLS && pages <= PG_SMEM_PAGES; }
static int pg_cluster(long long cells, bool few) {
  const long long per = 4 * (few ? PG_FEW_THREADS : PG_THREADS), share = (cells + per - 1) / per;
  return share >= PG_MAX_CLUSTER ? PG_MAX_CLUSTER : share > 2 ? 4 : static_cast<int>(share);
}
static int check_pool(const char* who, const VbPagePool* a, const VbPagePool* out) {
  VB_CHECK_ARG(a && out, "%s: null pool", who);
  for (const VbPagePool* p : {a, out})
    VB_CHECK_ARG(p->d_table && p->d_tokens && p->d_refs && p->d_status && p->d_copies && p->d_moved && p->d_scratch, "%s: null pointer in a pool", who);
  VB_CHECK_ARG(a->pages > 0 && a->page_size > 0 && a->rows > 0 && a->rows <= PG_MAX_ROWS && a->columns > 0, "%s: a pool of %d pages of %d tokens, %d rows (1 to %d) of %d columns",
               who, a->pages, a->page_size, a->rows, PG_MAX_ROWS, a->columns);
  VB_CHECK_ARG(static_cast<int64_t>(a->columns) * a->page_size <= 0x3fffffff && static_cast<int64_t>(a->columns + 1) * a->rows <= 0x3fffffff,
               "%s: %d rows of %d pages of %d tokens", who, a->rows, a->columns, a->page_size);
  VB_CHECK_ARG(a->pages == out->pages && a->page_size == out->page_size && a->rows == out->rows && a->columns == out->columns,
               "%s: the pool that is written is of another size", who);
  VB_CHECK_ARG((a->d_table == out->d_table) == (a->d_refs == out->d_refs) && (a->d_table == out->d_table) == (a->d_tokens == out->d_tokens),
               "%s: two pools that share some of their buffers", who);
  return 0;
}
static int check_caches(const char* who, const VbPageCache* caches, int n) {
  VB_CHECK_ARG(n >= 0 && (n == 0 || caches), "%s: %d caches", who, n);
  for (int c = 0; c < n; ++c) {
    const VbPageCache& s = caches[c];
    VB_CHECK_ARG(s.data && s.layers > 0 && s.parts > 0 && s.slots > 0 && s.slot_bytes > 0, "%s: cache %d is empty", who, c);
    VB_CHECK_ARG(s.slot_bytes % 16 == 0 && reinterpret_cast<uintptr_t>(s.data) % 16 == 0, "%s: cache %d: %lld bytes a slot (a multiple of 16, aligned to 16)", who, c,
                 static_cast<long long>(s.slot_bytes));
    VB_CHECK_ARG(s.slot_bytes / 16 * s.slots <= 0x3fffffff, "%s: cache %d: %d slots of %lld bytes", who, c, s.slots, static_cast<long long>(s.slot_bytes));
  }
  return 0;
}

}  // namespace vb

using namespace vb;

extern "C" size_t vb_page_pool_scratch_bytes(int pages) {
  if (pages <= 0) return 0;
  return 8ull * pages;
}

extern "C" int vb_fork_pages(const VbPagePool* pool, const VbPagePool* out, const int32_t* d_src, int group, const int32_t* d_grow, int grow, const VbPageCache* caches,
                             int n_caches, void* stream) {
  if (int rc = check_pool("vb_fork_pages", pool, out)) return rc;
  if (int rc = check_caches("vb_fork_pages", caches, n_caches)) return rc;
  VB_CHECK_ARG(group >= 0 && (group == 0 || pool->rows % group == 0), "vb_fork_pages: %d rows in groups of %d", pool->rows, group);
  VB_CHECK_ARG(grow >= 0, "vb_fork_pages: room for %d more tokens", grow);
  ForkParams p = {};
  p.table = pool->d_table, p.tokens = pool->d_tokens, p.refs = pool->d_refs;
  p.out_table = out->d_table, p.out_tokens = out->d_tokens, p.out_refs = out->d_refs;
  p.status = out->d_status, p.copies = out->d_copies, p.was = pool->d_status, p.live = out->d_live;
  p.work = out->d_scratch, p.free = p.work + pool->pages, p.in_smem = pool->pages <= PG_SMEM_PAGES;
  p.src = d_src, p.grow = d_grow, p.grow_all = grow;
  p.rows = pool->rows, p.columns = pool->columns, p.pages = pool->pages, p.page_size = pool->page_size, p.group = group;
  const bool few = pg_few(static_cast<long long>(p.rows) * p.columns, p.pages);
  const int cluster = pg_cluster(static_cast<long long>(p.rows) * p.columns, few), most = (8 * PG_MAX_ROWS + PG_STAGE + 2 * PG_SMEM_PAGES) * 4;
  const int smem = (8 * p.rows + PG_STAGE + (p.in_smem ? 2 * p.pages : 0)) * 4;
  VB_CHECK_CUDA(few ? rm_smem<fork_pages_kernel<PG_FEW_THREADS>>(most) : rm_smem<fork_pages_kernel<PG_THREADS>>(most));
  if (few) VB_LAUNCH_PDL_CLUSTER(fork_pages_kernel<PG_FEW_THREADS>, cluster, PG_FEW_THREADS, smem, stream, cluster, p);
  else VB_LAUNCH_PDL_CLUSTER(fork_pages_kernel<PG_THREADS>, cluster, PG_THREADS, smem, stream, cluster, p);
  return copy_listed(caches, n_caches, pool, out->d_copies, out->d_status, PC_TAILS, stream);
}

extern "C" int vb_compact_pages(const VbPagePool* pool, const VbPagePool* out, const VbPageCache* caches, int n_caches, void* stream) {
  if (int rc = check_pool("vb_compact_pages", pool, out)) return rc;
  if (int rc = check_caches("vb_compact_pages", caches, n_caches)) return rc;
  CompactParams p = {};
  p.table = pool->d_table, p.tokens = pool->d_tokens, p.refs = pool->d_refs;
  p.out_table = out->d_table, p.out_tokens = out->d_tokens, p.out_refs = out->d_refs, p.moved = out->d_moved;
  p.status = out->d_status, p.copies = out->d_copies, p.was = pool->d_status, p.live = out->d_live;
  p.from = out->d_scratch, p.to = p.from + pool->pages;
  p.rows = pool->rows, p.pages = pool->pages, p.page_size = pool->page_size;
  p.cells = static_cast<long long>(pool->rows) * pool->columns;
  const bool few = pg_few(p.cells, p.pages);
  const int cluster = pg_cluster(p.cells, few);
  if (few) VB_LAUNCH_PDL_CLUSTER(compact_pages_kernel<PG_FEW_THREADS>, cluster, PG_FEW_THREADS, 0, stream, cluster, p);
  else VB_LAUNCH_PDL_CLUSTER(compact_pages_kernel<PG_THREADS>, cluster, PG_THREADS, 0, stream, cluster, p);
  return copy_listed(caches, n_caches, pool, out->d_copies, out->d_status, PC_WHOLE, stream);
}
