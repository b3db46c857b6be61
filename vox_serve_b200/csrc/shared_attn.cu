// Attention of one new token a row over a paged cache in which rows share pages: beams of one search, continuations of one prompt.
//
//   out[r] = sum_t softmax_t(q[r] . k[t] / sqrt d) v[t]     over row r's own tokens t
//
// What bounds it is the cache that is read.  Rows stand in groups (the rows of a request); of every column of their page table each DIFFERENT page is read
// once, with the set of rows that hold it, instead of once for every row.  A group's rows times the query heads of a key head, up to 128, are the accumulator
// rows of the tcgen05 core (attn_tc.cuh): a tile of 64 keys meets all of them while it is on chip.
//
//   plan (once a step)   a cluster a group lists its different pages in pieces of 16 tokens {place in the cache, position, rows, tokens}: first the tiles
//                        that all living rows see whole, then the rest; the tiles of every group and key head are cut into equal segments, as many as there are
//                        blocks (two an SM); where there are more groups and heads than blocks, a block gets an equal stretch of all of them
//   attention            a block walks its segments: maximum, denominator and unnormalised output of each one's rows
//   join                 the segments of a group and head meet, in their order
//
// Tiles that are seen whole need no masks.  In the others a row's probability is 0 where it does not see, and 0 times what is not finite is not 0.  So a block
// whose results are not finite, and that had such tiles, walks its segments again: values that are not finite are taken out on the way, and the rows that see
// them get them back at the end.  Caches that hold finite numbers everywhere, behind a row's last token too, never go there.
// Probabilities enter the second product as two bf16 parts (2^-17).
//
// What bounds it now: HBM while tiles arrive (6 to 7.6 TB/s), and around that 2.5 us to the first copy, 3 to 5 from a block's last scores to its results in memory,
// 4 for the join.  Measured, a call in a captured chain: 8 requests of 8 rows (7 alive) on prompts of 4050 tokens and 300 more, 16 heads on 8 of 128, pages of 128:
// 157 MB in 37.4 us (24.4 of HBM; blocks of a group and head end unevenly, up to 4 us); 2 of 5 on 61007 tokens, 32 heads on 2, pages of 48: 110 MB in 34.7 us (17.1;
// 80 rows of products put out 12 MB of partial results); 4 rows of 171 tokens, pages of 16: 7.7 us.  Read once for every row (paged_attn) the same take 112, 322 and 13.4.
// Against paged_attn without anything to share: 8 rows of 1100 tokens 15.2 us beside 18.0, 32 rows of 600 21.0 beside 17.4: a row alone keeps 126 of 128 accumulator
// rows idle, and that one fetches while the kernel in front still runs.
// At 128 registers, for two blocks an SM, heads of 128 spill 96 bytes a thread, heads of 64 spill 64.  mma.sync instead of the tcgen05 core took 104 us for the second case.
// Three to six blocks' worth of segments an SM instead of two: 54 to 58 for the first (43 then).
#include "../../include/vb_api.h"
#define VB_PDL_FAMILY 1
#include "attn_tc.cuh"
#include "rowmma.cuh"

namespace vb {

constexpr int SA_MAX_ROWS = 128;                 // rows of a group times query heads of a key head
// behind the operands: two sets of barriers, four tiles' pieces, results on their way out
template <int D>
constexpr int SA_OUT = PtcLayout<D>::BAR + 768;
template <int D>
constexpr int SA_SMEM = SA_OUT<D> + 128 * 64 + 1024;
// Pages are listed in pieces of 16 tokens, four to a tile.  Pieces of a tile that are neighbours in a page come with one copy of as many rows: one of 64 for most
// tiles of pages of 64 and more.
constexpr int SA_PIECE = 16, SA_TILE_PIECES = PTC_KT / SA_PIECE;

// ---- the plan -------------------------------------------------------------------------------------------------------------------
constexpr int SD_PART = 8;       // words of 16 bytes, a line: a block knows what to fetch first with one load
struct SharedPlanParams {
  int4* entries;                 // [groups][cap]: {token's place in a layer's pages, its position, rows that hold it, tokens}
  int4* parts;                   // [grid][SD_PART]: {group, head, first tile, tiles}, {pieces of the group, its tiles that are seen whole}, the first tile's pieces
  int32_t *counts, *whole, *len; // [groups] pieces and tiles that are seen whole, [rows]
  int32_t* tile0;                // [groups + 1] tiles in front of a group
  int2* blocks_of;               // [units] first and last block of a unit
  const int32_t *table, *tokens;
  int rows, width, sub, subs, groups, cap, columns, pages, page_size, heads, grid;
};

constexpr int SP_THREADS = 512, SP_WARPS = SP_THREADS / 32, SP_CHUNK = 128, SP_MAX_COLUMNS = 16384, SP_CLUSTER = 8;

// exclusive prefix over a block of WARPS warps of what its threads have, and the total; `sums`: a word a warp
template <int WARPS>
__device__ __forceinline__ int sp_prefix(int mine, int* sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  __syncthreads();                                     // (the last call's sums have been read)
  if (lane == 31) sums[warp] = inc;
  __syncthreads();
  const int all = WARPS == 32 || lane < WARPS ? sums[lane] : 0, before = __reduce_add_sync(0xffffffffu, lane < warp ? all : 0);
  total = __reduce_add_sync(0xffffffffu, all);
  return before + inc - mine;
}

__device__ __forceinline__ int shared_first_row(const SharedPlanParams& p, int g, int& n) {
  const int in = g % p.subs * p.sub;
  n = min(p.sub, p.width - in);
  return g / p.subs * p.width + in;
}

// One column as a warp sees it, lane: row.  A class of lanes holds the same page; its first lane speaks for it: pieces that all living rows see whole,
// pieces in all, tokens.
struct SharedColumn {
  int page, whole, pieces, tokens;
  uint32_t same;
};
__device__ __forceinline__ SharedColumn shared_column(const SharedPlanParams& p, int page, int tokens, uint32_t alive) {
  SharedColumn c;
  c.page = tokens > 0 && page >= 0 && page < p.pages ? page : -1;
  c.same = __match_any_sync(0xffffffffu, c.page);
  int most = tokens, least = tokens;
  if (!__all_sync(0xffffffffu, c.page < 0 || tokens >= p.page_size)) {      // (only a row's last column is not full)
    most = 0, least = p.page_size;
    for (uint32_t left = c.same; left; left &= left - 1) {
      const int v = __shfl_sync(c.same, tokens, __ffs(left) - 1);
      most = max(most, v), least = min(least, v);
    }
  }
  const bool leads = c.page >= 0 && static_cast<int>(threadIdx.x & 31) == __ffs(c.same) - 1;
  c.tokens = most = min(most, p.page_size);
  c.pieces = leads ? (most + SA_PIECE - 1) / SA_PIECE : 0;
  c.whole = leads && (c.same & alive) == alive ? min(least, p.page_size) / SA_PIECE : 0;
  return c;
}

// A cluster a group, its columns in chunks to the blocks in turn.  A column of which all living rows see one whole page is known by its largest and least page
// number: threads side by side read columns side by side, four of them the rows of one.  The others, where rows have parted, take a warp each, a lane a row.
// Counted first, then written behind what stands in front, block after block.  What bounds it is latency: the tables' and the code's own, which runs once; so no
// loop is unrolled but those of loads, and blocks have no more warps than load.  Both launches, one after the other in a graph (the first columns of the table in
// brackets): 2 requests of 5 rows [1273] 12.3 us, 8 of 8 [34] 11.5, one of 4 [11] 11.2; every column with a warp, four unrolled, took 36.5, 18.1 and 12.7.
__global__ void __launch_bounds__(SP_THREADS) shared_list_kernel(const __grid_constant__ SharedPlanParams p) {
  extern __shared__ int sp_smem[];                     // of the block's columns: whole pieces in front, others in front, the page that all see, those that have parted
  __shared__ int sums[SP_WARPS], n_parted;
  __shared__ int2 seen[SP_THREADS];
  __shared__ float totals[2];                          // (ints, read by the other blocks)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = cluster_ctarank(), blocks = cluster_nctarank(), g = blockIdx.x / blocks;
  const int at_c = tid % SP_CHUNK, at_r = tid / SP_CHUNK;
  constexpr int ACROSS = SP_THREADS / SP_CHUNK;
  if (tid == 0) n_parted = 0;
  pdl_sync();
  int n;
  const int r0 = shared_first_row(p, g, n);
  const int32_t* table = p.table + static_cast<long long>(r0) * p.columns;
  auto column = [&](int i) { return (i / SP_CHUNK * blocks + rank) * SP_CHUNK + i % SP_CHUNK; };
  int v[32 / ACROSS];
  auto ask = [&](int c) {
#pragma unroll
    for (int j = 0; j < 32 / ACROSS; ++j)
      if (at_r + j * ACROSS < n && c < p.columns) v[j] = table[static_cast<long long>(at_r + j * ACROSS) * p.columns + c];
  };
  ask(column(at_c));                                   // (on its way together with the tokens)
  int len = 0;
  if (lane < n) {
    len = p.tokens[r0 + lane];
    len = len < 0 ? 0 : min(len, p.columns * p.page_size);
    if (rank == 0 && warp == 0) p.len[r0 + lane] = len;
  }
  const uint32_t alive = __ballot_sync(0xffffffffu, len > 0);
  const int longest = __reduce_max_sync(0xffffffffu, len), shortest = __reduce_min_sync(0xffffffffu, len > 0 ? len : 0x7fffffff);
  const int columns = (longest + p.page_size - 1) / p.page_size, per_page = p.page_size / SA_PIECE;
  const int here = (columns + blocks * SP_CHUNK - 1) / (blocks * SP_CHUNK) * SP_CHUNK;      // (with places behind the last column)
  int *first_w = sp_smem, *first_o = first_w + here, *one = first_o + here, *parted = one + here;
  for (int c0 = 0; c0 < here; c0 += SP_CHUNK) {
    const int i = c0 + at_c, c = column(i);
    if (c0 > 0) ask(c);
    int2 m = make_int2(-1, 0x7fffffff);
#pragma unroll
    for (int j = 0; j < 32 / ACROSS; ++j)
      if (at_r + j * ACROSS < n && c < columns && (alive >> (at_r + j * ACROSS) & 1u)) m = make_int2(max(m.x, v[j]), min(m.y, v[j]));
    seen[tid] = m;
    __syncthreads();
    if (at_r == 0) {
#pragma unroll
      for (int k = 1; k < ACROSS; ++k) m = make_int2(max(m.x, seen[at_c + k * SP_CHUNK].x), min(m.y, seen[at_c + k * SP_CHUNK].y));
      const bool same = c < columns && (c + 1) * p.page_size <= shortest && m.x == m.y && m.x >= 0 && m.x < p.pages;
      first_w[i] = same ? per_page : 0, first_o[i] = 0, one[i] = same ? m.x : -1;
      if (!same && c < columns) parted[atomicAdd(&n_parted, 1)] = i;
    }
    __syncthreads();
  }
  const int n_warp = n_parted;
  auto parted_column = [&](int i) {
    const int c = column(i);
    return shared_column(p, c * p.page_size < len ? table[static_cast<long long>(lane) * p.columns + c] : -1, len - c * p.page_size, alive);
  };
#pragma unroll 1
  for (int k = warp; k < n_warp; k += SP_WARPS) {
    const SharedColumn c = parted_column(parted[k]);
    const int all = __reduce_add_sync(0xffffffffu, c.pieces), whole = __reduce_add_sync(0xffffffffu, c.whole);
    if (lane == 0) first_w[parted[k]] = whole, first_o[parted[k]] = all - whole;
  }
  __syncthreads();
  int carry_w = 0, carry_o = 0;
  for (int c0 = 0; c0 < here; c0 += SP_THREADS) {       // exclusive prefix over the block's columns
    const int c = c0 + tid;
    int all_w, all_o;
    const int w = sp_prefix<SP_WARPS>(c < here ? first_w[c] : 0, sums, all_w), o = sp_prefix<SP_WARPS>(c < here ? first_o[c] : 0, sums, all_o);
    if (c < here) first_w[c] = carry_w + w, first_o[c] = carry_o + o;
    carry_w += all_w, carry_o += all_o;
  }
  if (tid == 0) totals[0] = __int_as_float(carry_w), totals[1] = __int_as_float(carry_o);
  __syncthreads();
  int w0 = 0, o0 = 0, all_w = carry_w, all_o = carry_o; // pieces of the blocks in front, of all
  if (blocks > 1) {
    cluster_sync_all();
    all_w = all_o = 0;
    for (int b = 0; b < blocks; ++b) {
      const int w = __float_as_int(ld_dsmem_f32(&totals[0], b)), o = __float_as_int(ld_dsmem_f32(&totals[1], b));
      if (b < rank) w0 += w, o0 += o;
      all_w += w, all_o += o;
    }
  }
  const int tiles_w = all_w / SA_TILE_PIECES;            // (what is left of the whole ones fills the first of the others)
  if (rank == 0 && tid == 0) p.counts[g] = all_w + all_o, p.whole[g] = tiles_w;
  int4* out = p.entries + static_cast<long long>(g) * p.cap;
#pragma unroll 1
  for (int k = warp; k < n_warp; k += SP_WARPS) {
    const int at = parted[k], col = column(at);
    const SharedColumn c = parted_column(at);
    int inc_w = c.whole, inc_o = c.pieces - c.whole;
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, inc_w, o), y = __shfl_up_sync(0xffffffffu, inc_o, o);
      if (lane >= o) inc_w += x, inc_o += y;
    }
    int at_w = w0 + first_w[at] + inc_w - c.whole, at_o = all_w + o0 + first_o[at] + inc_o - (c.pieces - c.whole);
#pragma unroll 1
    for (int i = 0; i < c.pieces; ++i) {
      const int off = i * SA_PIECE;
      out[i < c.whole ? at_w++ : at_o++] = make_int4(c.page * p.page_size + off, col * p.page_size + off, static_cast<int>(c.same), min(SA_PIECE, c.tokens - off));
    }
  }
#pragma unroll 1
  for (int i = at_c; i < here; i += SP_CHUNK)
    if (one[i] >= 0)
      for (int k = at_r; k < per_page; k += ACROSS)
        out[w0 + first_w[i] + k] = make_int4(one[i] * p.page_size + k * SA_PIECE, column(i) * p.page_size + k * SA_PIECE, static_cast<int>(alive), SA_PIECE);
  if (blocks > 1) cluster_sync_all();                   // (totals have been read)
}

constexpr int SD_THREADS = 1024, SD_WARPS = SD_THREADS / 32, SD_MAX_GROUPS = 4096;
__global__ void __launch_bounds__(SD_THREADS) shared_deal_kernel(const __grid_constant__ SharedPlanParams p) {
  __shared__ int sums[SD_WARPS], tiles_s[SD_MAX_GROUPS], first_s[SD_MAX_GROUPS];      // tiles of a group, its first block
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_sync();
  const int units = p.groups * p.heads;
  auto write_part = [&](int i, const int4& part, const int4& of) {
    int4 *to = p.parts + i * SD_PART, e[4];
    const int first = part.z * SA_TILE_PIECES;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      e[k] = k < SA_TILE_PIECES && part.w > 0 && first + k < of.x ? __ldcg(p.entries + static_cast<long long>(part.x) * p.cap + first + k) : make_int4(0, 0, 0, 0);
    to[0] = part, to[1] = of;
#pragma unroll
    for (int k = 0; k < 4; ++k) to[2 + k] = e[k];
  };
  int total = 0;
  for (int g0 = 0; g0 < p.groups; g0 += SD_THREADS) {
    const int g = g0 + tid, mine = g < p.groups ? (__ldcg(p.counts + g) + SA_TILE_PIECES - 1) / SA_TILE_PIECES : 0;
    int all;
    const int before = sp_prefix<SD_WARPS>(mine, sums, all);
    if (units <= p.grid) {
      if (g < p.groups) tiles_s[g] = mine;
    } else if (g < p.groups) {
      p.tile0[g] = total + before;
    }
    total += all;
  }
  const long long work = static_cast<long long>(total) * p.heads;
  __syncthreads();
  if (units <= p.grid) {
    // Blocks of their own for every unit (one that goes on to another unit waits for it: 5 us): equal segments of at most q tiles, q the smallest with which
    // the blocks are enough: a unit of t tiles takes at most t / q + 1 of them, which bounds it from above.  A warp tries one, 32 at once.
    int lo = static_cast<int>(max(1ll, (work + p.grid - 1) / p.grid)), hi = max(lo, total);
    if (units < p.grid) hi = max(lo, min(hi, static_cast<int>((work + p.grid - units - 1) / (p.grid - units))));
    while (lo < hi) {
      const int step = (hi - lo + SD_WARPS - 1) / SD_WARPS, q = min(lo + warp * step, hi);
      int mine = 0;
      for (int g = lane; g < p.groups; g += 32) mine += (tiles_s[g] + q - 1) / q;
      mine = __reduce_add_sync(0xffffffffu, mine);
      if (lane == 0) sums[warp] = mine * p.heads <= p.grid;
      __syncthreads();
      const uint32_t enough = __ballot_sync(0xffffffffu, sums[lane] != 0);
      __syncthreads();
      const int i = enough ? __ffs(enough) - 1 : SD_WARPS;      // the first that is enough
      const int up = i < SD_WARPS ? min(lo + i * step, hi) : hi;
      if (i > 0) lo = min(lo + (i - 1) * step, hi) + 1;
      hi = max(lo, up);
    }
    const int q = lo;
    int used = 0;
    for (int g0 = 0; g0 < p.groups; g0 += SD_THREADS) {
      const int g = g0 + tid, n = g < p.groups ? (tiles_s[g] + q - 1) / q : 0;
      int all;
      const int before = sp_prefix<SD_WARPS>(n * p.heads, sums, all);
      if (g < p.groups) {
        first_s[g] = used + before;
        for (int h = 0; h < p.heads; ++h) p.blocks_of[g * p.heads + h] = make_int2(used + before + h * n, used + before + h * n + n - 1);
      }
      used += all;
    }
    __syncthreads();
    for (int i = tid; i < p.grid; i += SD_THREADS) {
      int4 part = make_int4(0, 0, 0, 0), of = part;
      if (i < used) {
        int g = 0, last = p.groups - 1;                  // the last group that begins at or before this block (of several the others are empty)
        while (g < last) {
          const int mid = (g + last + 1) >> 1;
          if (first_s[mid] <= i) g = mid;
          else last = mid - 1;
        }
        const int tiles = tiles_s[g], n = (tiles + q - 1) / q, h = (i - first_s[g]) / n, k = (i - first_s[g]) - h * n;
        const int from = static_cast<int>(static_cast<long long>(tiles) * k / n), to = static_cast<int>(static_cast<long long>(tiles) * (k + 1) / n);
        part = make_int4(g, h, from, to - from);
        of = make_int4(__ldcg(p.counts + g), __ldcg(p.whole + g), 0, 0);
      }
      write_part(i, part, of);
    }
    return;
  }
  if (tid == 0) p.tile0[p.groups] = total;
  __syncthreads();
  auto tile0 = [&](int g) { return __ldcg(p.tile0 + g); };
  // More units than blocks: equal stretches of all their tiles in a line
  const long long blocks = min(work, static_cast<long long>(p.grid));      // (none without a tile: the join counts on it)
  for (int i = tid; i < p.grid; i += SD_THREADS) {
    int4 part = make_int4(0, 0, 0, 0), of = part;
    if (i < blocks) {
      const long long start = work * i / blocks;
      int lo = 0, hi = p.groups - 1;                    // the last group that begins at or before the start (of several the others are empty)
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (static_cast<long long>(tile0(mid)) * p.heads <= start) lo = mid;
        else hi = mid - 1;
      }
      const int t0 = tile0(lo), tiles = tile0(lo + 1) - t0, in = static_cast<int>(start - static_cast<long long>(t0) * p.heads);
      part = make_int4(lo, in / tiles, in % tiles, static_cast<int>(work * (i + 1) / blocks - start));
      of = make_int4(__ldcg(p.counts + lo), __ldcg(p.whole + lo), 0, 0);
    }
    write_part(i, part, of);
  }
  for (int u = tid; u < units; u += SD_THREADS) {
    const int g = u / p.heads, t0 = tile0(g), tiles = tile0(g + 1) - t0;
    const long long first = static_cast<long long>(t0) * p.heads + static_cast<long long>(u - g * p.heads) * tiles;
    // (whose stretch holds a tile)
    if (tiles) p.blocks_of[u] = make_int2(static_cast<int>(((first + 1) * blocks - 1) / work), static_cast<int>(((first + tiles) * blocks - 1) / work));
    else p.blocks_of[u] = make_int2(0, -1);
  }
}

// ---- attention -------------------------------------------------------------------------------------------------------------------
struct SharedAttnParams {
  const __nv_bfloat16 *q, *kv;
  __nv_bfloat16* out;
  const int4 *entries, *parts;
  const int32_t *counts, *whole, *len;
  const int2* blocks_of;         // [units]
  float* acc;                    // [blocks + units][mpad][D]: the segment of block b on unit u stands at b + u
  float2* stat;                  // [blocks + units][mpad] maximum (base 2), denominator against it
  long long slab_base, slabs;
  unsigned char *wait_flag, *plan_flag;
  const int32_t* expect;         // tokens of the rows in the step that calls, or null: a plan of other ones is another step's
  int rows, width, sub, subs, groups, cap, page_size, n_q, heads, G, mpad, xt_tile;
  float scale_log2;
};

__device__ __forceinline__ int shared_group(const SharedAttnParams& p, int g, int& n) {
  const int in = g % p.subs * p.sub;
  n = min(p.sub, p.width - in);
  return g / p.subs * p.width + in;
}

// A block's stretch, segment by segment
struct SharedWalk {
  const SharedAttnParams& p;
  int g, h, t, left;             // group, key head, first tile; tiles of the stretch from here on
  int count, whole, tiles;       // of the group
  __device__ __forceinline__ SharedWalk(const SharedAttnParams& p_, const int4& part, const int4& of)
      : p(p_), g(part.x), h(part.y), t(part.z), left(part.w), count(of.x), whole(of.y), tiles((of.x + SA_TILE_PIECES - 1) / SA_TILE_PIECES) {}
  __device__ __forceinline__ int here() const { return min(left, tiles - t); }      // tiles of the segment
  __device__ __forceinline__ void step(int n) {                                     // n tiles on, within the segment
    t += n, left -= n;
    if (t < tiles || left <= 0) return;
    t = 0;
    if (++h < p.heads) return;
    h = 0;
    do {
      ++g;
      count = p.counts[g];
    } while (count == 0);        // (tiles are left, so there is one)
    whole = p.whole[g], tiles = (count + SA_TILE_PIECES - 1) / SA_TILE_PIECES;
  }
};

// Tokens of a tile that a row sees: it holds the page, and the token is not behind its last
__device__ __forceinline__ uint64_t shared_mask(const int4* pieces, int n_pieces, int bit, int len) {
  uint64_t m = 0ull;
#pragma unroll
  for (int i = 0; i < SA_TILE_PIECES; ++i) {
    if (i >= n_pieces) break;
    const int4 e = pieces[i];
    const int n = (static_cast<uint32_t>(e.z) >> bit & 1u) ? min(len - e.y, e.w) : 0;
    if (n > 0) m |= ((1ull << n) - 1ull) << (i * SA_PIECE);
  }
  return m;
}
// What is not finite among the values that a row sees in the segment's tiles with masks, where it was taken out: 32 dimensions from c0.  (Not a member: an
// object that is handed on lives in memory.)
template <int D>
__device__ __noinline__ void shared_give_back(const SharedAttnParams& p, const int4* entries, int count, int from, int to, int head, int bit, int len, int c0, float* v) {
  for (int t = from; t < to; ++t) {
    const int first = t * SA_TILE_PIECES;
    const uint64_t m = shared_mask(entries + first, min(SA_TILE_PIECES, count - first), bit, len);
    for (int k = 0; k < PTC_KT; ++k) {
      if (!(m >> k & 1ull)) continue;
      const int tok = entries[first + k / SA_PIECE].x + k % SA_PIECE, page = tok / p.page_size, slot = tok - page * p.page_size;
      if (p.slab_base + page >= p.slabs) continue;               // (behind the cache: the copies brought zeros)
      const uint32_t* src = reinterpret_cast<const uint32_t*>(p.kv + ((((p.slab_base + page) * 2 + 1) * p.page_size + slot) * p.heads + head) * D + c0);
      for (int i = 0; i < 16; ++i) {
        const uint32_t w = src[i];
        if ((w & 0x7f80u) == 0x7f80u) v[2 * i] += bf16_lo(w);
        if ((w & 0x7f800000u) == 0x7f800000u) v[2 * i + 1] += bf16_hi(w);
      }
    }
  }
}

// what this thread's row sees of a segment, and where its part goes
template <int D>
struct SharedRows {
  static constexpr bool HOLE = false, STAGED = false, CHAINED = true;
  static constexpr int hole0 = 0, hole1 = 0;
  const SharedAttnParams& p;
  uint8_t* smem;
  PtcShared* sh;
  const int4 *entries, *meta;    // of the group; of the block's last four tiles, as far as they have masks
  int base;                      // tiles of the block in front of the segment
  int count, whole, t0, n_tiles; // pieces; tiles that need no mask; the segment
  int row0, n_rows, head, group; // first row, rows, key head, query heads of it
  int len, bit;
  bool ok;
  float scale_log2;
  float2* stat;
  float* acc;                    // of the segment
  int next_g, next_h;            // the segment behind this one; -1: none
  bool careful;                  // values that are not finite have been taken out
  mutable bool bad;              // a result that is not finite
  mutable uint64_t seen;
  __device__ __forceinline__ int tile(int it) const { return t0 + it; }
  __device__ __forceinline__ bool full(int tok0) const {
    seen = ~0ull;
    const int t = tok0 / PTC_KT;
    if (t >= whole && ok) seen = shared_mask(meta + (base + t - t0 & 3) * 4, SA_TILE_PIECES, bit, len);      // (a row that is none may have anything)
    return seen == ~0ull;
  }
  __device__ __forceinline__ bool visible(int kj) const { return seen >> (kj & (PTC_KT - 1)) & 1ull; }
  __device__ __forceinline__ const __nv_bfloat16* q_row(int t, int g) const {
    return t < n_rows ? p.q + (static_cast<size_t>(row0 + t) * p.n_q + head * group + g) * D : nullptr;
  }
  struct Query {                 // of the segment behind this one
    const SharedAttnParams& p;
    int row0, n_rows, head, group;
    __device__ __forceinline__ const __nv_bfloat16* q_row(int t, int g) const {
      return t < n_rows ? p.q + (static_cast<size_t>(row0 + t) * p.n_q + head * group + g) * D : nullptr;
    }
  };
  __device__ __forceinline__ void next_q() const {
    if (next_g < 0) return;
    Query q{p, 0, 0, next_h, group};
    q.row0 = shared_group(p, next_g, q.n_rows);
    ptc_load_q<D>(smem, sh, q);
  }
  __device__ __forceinline__ uint4* out_at(int, int, int) const { return nullptr; }
  __device__ __forceinline__ float finish(float m_ref, float l) const {
    if (ok) *stat = make_float2(m_ref, l);
    return 1.f;
  }
  __device__ __forceinline__ void store(int c0, const uint32_t (&o)[32], float) const {
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(o[i]);
    if (careful && ok) {                                      // (a copy: an array that is handed on lives in memory)
      float w[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) w[i] = v[i];
      shared_give_back<D>(p, entries, count, max(t0, whole), t0 + n_tiles, head, bit, len, c0, w);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = w[i];
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) bad |= !isfinite(v[i]);
    // Up to 16 rows of the warp: 16 bytes a lane of its own row.  More: in whole sectors, 16 values of a row at a time through shared memory (16-byte chunk c of
    // row r at chunk c ^ (r / 2 & 3)).  Measured, own rows / sectors: 14 rows 39.1 / 39.9 us, 80 rows 37.1 / 36.0 (a call of the cases of 157 and 110 MB).
    const int lane = threadIdx.x & 31, row = threadIdx.x - lane, mine_rows = n_rows * group - row;
    if (mine_rows <= 16) {
      float4* y = reinterpret_cast<float4*>(acc + static_cast<int>(threadIdx.x) * D + c0);
      if (ok)
#pragma unroll
        for (int c = 0; c < 8; ++c) y[c] = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
      return;
    }
    float4* mine = reinterpret_cast<float4*>(smem + SA_OUT<D>) + row * 4;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      __syncwarp();
#pragma unroll
      for (int c = 0; c < 4; ++c)
        mine[lane * 4 + (c ^ (lane >> 1 & 3))] = make_float4(v[16 * half + 4 * c], v[16 * half + 4 * c + 1], v[16 * half + 4 * c + 2], v[16 * half + 4 * c + 3]);
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = i * 8 + (lane >> 2), c = lane & 3;
        if (r < mine_rows) *reinterpret_cast<float4*>(acc + (row + r) * D + c0 + 16 * half + c * 4) = mine[r * 4 + (c ^ (r >> 1 & 3))];
      }
    }
  }
};

// A lane a piece of the tile: the first of every run of neighbours copies them, K or V.  A place without a piece gets the tile's first one again: what stands there is
// multiplied by probability 0, and what an earlier kernel left in shared memory need not be finite.
struct SharedMaps {
  CUtensorMap rows[SA_TILE_PIECES];      // boxes of 16, 32, 48, 64 rows (as far as a page has so many)
};
template <int D>
__device__ __forceinline__ void shared_fetch(const SharedAttnParams& p, const SharedMaps& maps, const int4& e, int part, int head, uint32_t dst, uint64_t* bar) {
  const int lane = threadIdx.x & 31;
  const int first = __shfl_sync(0xffffffffu, e.x, 0), at = e.w > 0 ? e.x : first, before = __shfl_up_sync(0xffffffffu, at, 1);
  const int page = at / p.page_size, slot = at - page * p.page_size;
  const uint32_t starts = __ballot_sync(0xffffffffu, lane == 0 || at != before + SA_PIECE || slot == 0);
  __syncwarp();                          // (what the other lanes wrote of the tile's pieces is released by lane 0's arrival; shuffles order no memory)
  if (lane == 0) mbar_arrive_expect_tx(bar, PTC_KT * D * 2);
  __syncwarp();
  if (lane < SA_TILE_PIECES && (starts >> lane & 1u)) {
    const uint32_t behind = (starts | 1u << SA_TILE_PIECES) & ~((2u << lane) - 1u);
    const CUtensorMap* map = &maps.rows[__ffs(behind) - 2 - lane];
#pragma unroll
    for (int kb = 0; kb < D / 64; ++kb)
      ptc_tma_5d(dst + kb * (PTC_KT * 128) + lane * SA_PIECE * 128, map, smem_u32(bar), kb * 64, slot, head, part, static_cast<int>(p.slab_base + page));
  }
  __syncwarp();
}

template <int D>
__global__ void __launch_bounds__(PTC_THREADS, 2) shared_attn_kernel(const __grid_constant__ SharedMaps maps, const __grid_constant__ SharedAttnParams p) {
  using L = PtcLayout<D>;
  extern __shared__ uint8_t sa_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(sa_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  static_assert(sizeof(PtcShared) <= 256, "two of them and four tiles' pieces behind the operands");
  PtcShared *sh = reinterpret_cast<PtcShared*>(smem + L::BAR), *sh2 = reinterpret_cast<PtcShared*>(smem + L::BAR + 256);
  int4* meta = reinterpret_cast<int4*>(smem + L::BAR + 512);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  BoundedWait bw{p.wait_flag};
  if (tid == 0) {
    ptc_init(sh, 1);
    ptc_init(sh2, 1);
    prefetch_tmap(&maps.rows[0]);
    prefetch_tmap(&maps.rows[SA_TILE_PIECES - 1]);
  }
  if (warp == 4) {
    tmem_alloc(&sh->tmem, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = sh->tmem;
  if (tid == 0) sh2->tmem = tmem_base;
  pdl_wait();
  const int4 part = p.parts[SD_PART * blockIdx.x], of = p.parts[SD_PART * blockIdx.x + 1], head_piece = p.parts[SD_PART * blockIdx.x + 2 + (lane & 3)];
  pdl_trigger();
#pragma unroll 1
  for (int pass = 0; part.w > 0; ++pass) {
    bool bad = false;
    const bool careful = pass != 0;
    SharedWalk w(p, part, of);
    if (warp < 4) {
      for (int base = 0, walk = 0; w.left > 0 && !bw.dead; ++walk) {
        const int g = w.g, head = w.h, t0 = w.t, n_tiles = w.here(), whole = w.whole, count = w.count;
        w.step(n_tiles);                                      // (the next segment)
        int n_rows;
        const int row0 = shared_group(p, g, n_rows), t = tid / p.G;
        const bool ok = t < n_rows;
        const long long slot = (blockIdx.x + static_cast<long long>(g) * p.heads + head) * p.mpad;
        SharedRows<D> rows{p, smem, sh, p.entries + static_cast<long long>(g) * p.cap, meta, base, count, whole, t0, n_tiles, row0, n_rows, head, p.G,
                           ok ? p.len[row0 + t] : 0, ok ? t : 0, ok, p.scale_log2, p.stat + slot + tid, p.acc + slot * D, w.left > 0 ? w.g : -1, w.h, careful, false, ~0ull};
        if (walk == 0) ptc_load_q<D>(smem, sh, rows);
        if (warp * 32 < n_rows * p.G) ptc_softmax<D>(smem, sh, rows, bw, base, walk);
        else ptc_idle(sh, rows, bw, base, walk);
        bad |= rows.bad && rows.len > 0 && t0 + n_tiles > whole;
        base += n_tiles;
      }
    } else if (warp == 4) {
      for (int base = 0, walk = 0; w.left > 0 && !bw.dead; ++walk) {
        const int n_tiles = w.here();
        ptc_issue<D>(smem, sh, n_tiles, bw, base, walk);
        base += n_tiles;
        w.step(n_tiles);
      }
    } else {
      const bool values = warp == 6;
      uint64_t *full = values ? sh->v_full : sh->k_full, *empty = values ? sh->v_empty : sh->k_empty;
      const uint32_t ring = smem_u32(smem + (values ? L::V : L::K));
      auto find = [&]() {                                     // a lane a piece of the tile
        const int i = w.t * SA_TILE_PIECES + lane;
        return lane < SA_TILE_PIECES && w.left > 0 && i < w.count ? p.entries[static_cast<long long>(w.g) * p.cap + i] : make_int4(0, 0, 0, 0);
      };
      int4 next = lane < SA_TILE_PIECES ? head_piece : make_int4(0, 0, 0, 0);      // (the first tile's)
      uint32_t turn = 0;                                      // bit s: parity of stage s's next tile that is changed
      bool pending = false;                                   // the tile in front, if its values are still to be changed
      for (int j = 0; j <= part.w; ++j) {
        const int s = j & 1;
        const int4 e = next;
        bool change = false;
        if (j < part.w) {
          const int head = w.h;
          const bool masked = w.t >= w.whole;
          w.step(1);
          next = find();
          bw.wait(&empty[s], ((j >> 1) & 1) ^ 1);
          if (!__all_sync(0xffffffffu, !bw.dead)) {
            bw.dead = true;
            break;
          }
          // (tile j + 4's stands where tile j's was: its stage was empty, so tile j + 2's scores have been multiplied, and tile j's output with them)
          if (!values && masked && lane < SA_TILE_PIECES) meta[(j & 3) * 4 + lane] = e;
          change = values && masked && careful;
          shared_fetch<D>(p, maps, e, values ? 1 : 0, head, ring + s * L::TILE, change ? &sh->v_part[s] : &full[s]);
        }
        if (pending) {                                        // (behind the next tile's copies, which are on their way meanwhile)
          const int o = s ^ 1;
          bw.wait(&sh->v_part[o], turn >> o & 1u);
          if (!__all_sync(0xffffffffu, !bw.dead)) {
            bw.dead = true;
            break;
          }
          turn ^= 1u << o;
          uint4* v_tile = reinterpret_cast<uint4*>(smem + L::V + o * L::TILE);
          for (int i = lane; i < (D / 64) * PTC_KT * 8; i += 32) {
            uint4 v = v_tile[i];
            uint32_t* x = &v.x;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if ((x[k] & 0x7f80u) == 0x7f80u) x[k] &= 0xffff0000u;
              if ((x[k] & 0x7f800000u) == 0x7f800000u) x[k] &= 0xffffu;
            }
            v_tile[i] = v;
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[o]);
        }
        pending = change;
      }
      ptc_let_land(bw.dead);
      __syncwarp();
    }
    tc_fence_before();
    const bool again = __syncthreads_or(bad && !bw.dead);
    tc_fence_after();
    if (!again || pass) break;
    sh = sh2;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 256);
  }
}

// The segments of a group and head meet: WPR warps a row, each every WPR-th segment, a lane D / 32 neighbouring dimensions.
constexpr int SJ_WARPS = 8;
template <int D, int WPR>
__global__ void __launch_bounds__(32 * SJ_WARPS) shared_join_kernel(const __grid_constant__ SharedAttnParams p) {
  constexpr int E = D / 32;
  __shared__ float part[SJ_WARPS][32][E + 1], tops[SJ_WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, unit = blockIdx.x, g = unit / p.heads, h = unit - g * p.heads;
  const int m = blockIdx.y * (SJ_WARPS / WPR) + warp / WPR, sub = warp % WPR;
  pdl_sync();
  int n_rows;
  const int r0 = shared_group(p, g, n_rows);
  const bool on = m < n_rows * p.G;
  const int row = r0 + (on ? m / p.G : 0), k = (h * p.G + (on ? m % p.G : 0)) * D + lane * E;
  const int2 blocks = p.blocks_of[unit];
  const int len = p.len[row];
  const bool other = p.expect && max(0, p.expect[row]) != len;  // (zeros come out, and the host is told)
  if (other && on && lane == 0) {
    *reinterpret_cast<volatile unsigned char*>(p.plan_flag) = 1;
    __threadfence_system();
  }
  float acc[E], total = 0.f, top = -INFINITY;                   // against the largest maximum so far
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  if (on && len > 0 && !other) {
    const int s0 = blocks.x + unit, s1 = blocks.y + unit + 1;
    for (int s = s0 + sub; s < s1; s += 8 * WPR) {              // eight segments' maxima and outputs at once
      float2 st[8];
      float v[8][E];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const long long at = static_cast<long long>(s + i * WPR) * p.mpad + m;
        const bool in = s + i * WPR < s1;
        st[i] = in ? p.stat[at] : make_float2(-INFINITY, 0.f);
        if (E == 4) *reinterpret_cast<float4*>(v[i]) = in ? *reinterpret_cast<const float4*>(p.acc + at * D + lane * E) : make_float4(0.f, 0.f, 0.f, 0.f);
        else *reinterpret_cast<float2*>(v[i]) = in ? *reinterpret_cast<const float2*>(p.acc + at * D + lane * E) : make_float2(0.f, 0.f);
      }
      float most = top;
#pragma unroll
      for (int i = 0; i < 8; ++i) most = fmaxf(most, st[i].x);
      const float keep = top == -INFINITY ? 1.f : ptc_ex2(top - most);      // (nothing yet, or what is not a number)
      total *= keep;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] *= keep;
      top = most;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float f = st[i].x == -INFINITY ? (st[i].y == 0.f ? 0.f : 1.f) : ptc_ex2(st[i].x - top);      // (nothing seen; scores that are NaN)
        total += st[i].y * f;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += v[i][e] * f;
      }
    }
  }
  if (WPR > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) part[warp][lane][e] = acc[e];
    part[warp][lane][E] = total;
    if (lane == 0) tops[warp] = top;
    __syncthreads();
    if (sub == 0) {
      float most = top;
#pragma unroll
      for (int w = 1; w < WPR; ++w) most = fmaxf(most, tops[warp + w]);
      const float keep = top == -INFINITY ? 1.f : ptc_ex2(top - most);
      total *= keep;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] *= keep;
#pragma unroll
      for (int w = 1; w < WPR; ++w) {
        const float f = tops[warp + w] == -INFINITY ? 1.f : ptc_ex2(tops[warp + w] - most);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += part[warp + w][lane][e] * f;
        total += part[warp + w][lane][E] * f;
      }
    }
  }
  if (!on || sub != 0) return;
  const float by = total != 0.f ? 1.f / total : 0.f;
  const size_t at = p.xt_tile ? xt_index(row, k, p.xt_tile, p.n_q * D / 64) : static_cast<size_t>(row) * p.n_q * D + k;
#pragma unroll
  for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(p.out + at + e) = pack_bf16(acc[e] * by, acc[e + 1] * by);
}

template <int D>
static int launch_shared(const SharedMaps& maps, const SharedAttnParams& p, int grid, void* stream) {
  const int units = p.groups * p.heads, m = p.sub * p.G;
  VB_CHECK_CUDA(rm_smem<shared_attn_kernel<D>>(SA_SMEM<D>));
  VB_LAUNCH_PDL(shared_attn_kernel<D>, grid, PTC_THREADS, SA_SMEM<D>, stream, maps, p);
  // (eight warps a row where a unit has more than eight segments; one / eight warps: 4 units 51.2 / 35.5 us, 8 units 15.4 / 12.6, 64 38.5 / 40.5, 256 20.8 / 23.5)
  if (grid > 8 * units) VB_LAUNCH_PDL((shared_join_kernel<D, SJ_WARPS>), dim3(units, m), 32 * SJ_WARPS, 0, stream, p);
  else VB_LAUNCH_PDL((shared_join_kernel<D, 1>), dim3(units, (m + SJ_WARPS - 1) / SJ_WARPS), 32 * SJ_WARPS, 0, stream, p);
  return 0;
}

// rows of a group's products, group by group: the widest part of a request's rows whose products fit, requests cut evenly
static int shared_sub(int width, int G) {
  const int most = SA_MAX_ROWS / G < 32 ? SA_MAX_ROWS / G : 32, subs = (width + most - 1) / most;
  return (width + subs - 1) / subs;
}

static int check_shared(const char* who, const VbSharedPlan* s) {
  VB_CHECK_ARG(s && s->d_buffer, "%s: null pointer", who);
  VB_CHECK_ARG(s->rows > 0 && s->width > 0 && s->rows % s->width == 0, "%s: %d rows in requests of %d", who, s->rows, s->width);
  VB_CHECK_ARG(s->n_kv > 0 && s->n_q > 0 && s->n_q % s->n_kv == 0 && s->n_q / s->n_kv <= SA_MAX_ROWS, "%s: %d query heads on %d key heads (at most %d on one)", who, s->n_q,
               s->n_kv, SA_MAX_ROWS);
  VB_CHECK_ARG(s->head_dim == 64 || s->head_dim == 128, "%s: heads of %d (64 or 128)", who, s->head_dim);
  VB_CHECK_ARG(s->page_size > 0 && s->page_size % 16 == 0 && s->page_size <= 4096, "%s: pages of %d tokens (a multiple of 16, at most 4096)", who, s->page_size);
  VB_CHECK_ARG(s->columns > 0 && s->columns <= SP_MAX_COLUMNS && static_cast<int64_t>(s->columns) * s->page_size <= 0x3fffffff, "%s: %d pages a row (1 to %d)", who, s->columns,
               SP_MAX_COLUMNS);
  VB_CHECK_ARG(s->grid > 0 && s->grid <= 4096, "%s: %d blocks", who, s->grid);
  const int64_t pieces = static_cast<int64_t>(s->rows) * s->columns * (s->page_size / SA_PIECE);
  VB_CHECK_ARG(pieces * s->n_kv <= 0x3fffffff, "%s: %d rows of %d pages on %d heads", who, s->rows, s->columns, s->n_kv);
  return 0;
}

struct SharedLayout {
  int sub, subs, groups, cap, mpad;
  size_t parts, acc, stat, blocks_of, ints, bytes;      // entries first
};
static SharedLayout shared_layout(const VbSharedPlan* s) {
  SharedLayout l;
  const int G = s->n_q / s->n_kv;
  l.sub = shared_sub(s->width, G);
  l.subs = (s->width + l.sub - 1) / l.sub;
  l.groups = s->rows / s->width * l.subs;
  l.cap = l.sub * s->columns * (s->page_size / SA_PIECE);
  l.mpad = (l.sub * G + 15) / 16 * 16;
  const size_t units = static_cast<size_t>(l.groups) * s->n_kv, segments = s->grid + units;
  l.parts = 16ull * l.groups * l.cap;
  l.acc = l.parts + 16ull * SD_PART * s->grid;
  l.stat = l.acc + 4ull * segments * l.mpad * s->head_dim;
  l.blocks_of = l.stat + 8ull * segments * l.mpad;
  l.ints = l.blocks_of + 8ull * units;
  l.bytes = l.ints + 4ull * (3ull * l.groups + 1 + s->rows);
  return l;
}

}  // namespace vb

using namespace vb;

extern "C" size_t vb_shared_plan_bytes(const VbSharedPlan* plan) {
  VbSharedPlan s = plan ? *plan : VbSharedPlan{};
  s.d_buffer = &s;
  return check_shared("vb_shared_plan_bytes", &s) ? 0 : shared_layout(&s).bytes;
}

extern "C" int vb_shared_plan(const VbSharedPlan* plan, const int32_t* d_table, const int32_t* d_tokens, int pages, void* stream) {
  if (int rc = check_shared("vb_shared_plan", plan)) return rc;
  VB_CHECK_ARG(d_table && d_tokens, "vb_shared_plan: null pointer");
  VB_CHECK_ARG(pages > 0 && static_cast<int64_t>(pages) * plan->page_size <= 0x7fffffff, "vb_shared_plan: %d pages of %d tokens", pages, plan->page_size);
  const SharedLayout l = shared_layout(plan);
  uint8_t* at = static_cast<uint8_t*>(plan->d_buffer);
  SharedPlanParams p = {};
  p.entries = reinterpret_cast<int4*>(at);
  p.parts = reinterpret_cast<int4*>(at + l.parts);
  p.counts = reinterpret_cast<int32_t*>(at + l.ints);
  p.whole = p.counts + l.groups, p.tile0 = p.whole + l.groups, p.len = p.tile0 + l.groups + 1;
  p.blocks_of = reinterpret_cast<int2*>(at + l.blocks_of);
  p.table = d_table, p.tokens = d_tokens;
  p.rows = plan->rows, p.width = plan->width, p.sub = l.sub, p.subs = l.subs, p.groups = l.groups, p.cap = l.cap;
  p.columns = plan->columns, p.pages = pages, p.page_size = plan->page_size, p.heads = plan->n_kv, p.grid = plan->grid;
  const int chunks = (plan->columns + SP_CHUNK - 1) / SP_CHUNK, cluster = chunks > 4 ? SP_CLUSTER : chunks > 2 ? 4 : chunks;      // (a chunk a block, as far as they go)
  VB_LAUNCH_PDL_CLUSTER(shared_list_kernel, l.groups * cluster, SP_THREADS, (chunks + cluster - 1) / cluster * SP_CHUNK * 16, stream, cluster, p);
  VB_LAUNCH_PDL(shared_deal_kernel, 1, SD_THREADS, 0, stream, p);
  return 0;
}

extern "C" int vb_shared_attn(void* d_out, const void* d_q, const void* d_kv, int64_t slabs, int64_t slab_base, const VbSharedPlan* plan, float sm_scale, int out_xt_tile,
                              void* stream) {
  if (int rc = check_shared("vb_shared_attn", plan)) return rc;
  VB_CHECK_ARG(d_out && d_q && d_kv, "vb_shared_attn: null pointer");
  VB_CHECK_ARG(slabs > 0 && slabs <= 0x7fffffff && slab_base >= 0 && slab_base < slabs, "vb_shared_attn: slab %lld of %lld", static_cast<long long>(slab_base),
               static_cast<long long>(slabs));
  VB_CHECK_ARG(reinterpret_cast<uintptr_t>(d_kv) % 16 == 0 && reinterpret_cast<uintptr_t>(d_q) % 16 == 0 && reinterpret_cast<uintptr_t>(d_out) % 16 == 0,
               "vb_shared_attn: unaligned tensors");
  const SharedLayout l = shared_layout(plan);
  const int D = plan->head_dim, H = plan->n_kv, P = plan->page_size;
  auto fn = encode_fn();
  VB_CHECK_ARG(fn, "vb_shared_attn: cuTensorMapEncodeTiled not available (no CUDA driver?)");
  SharedMaps maps;
  const cuuint64_t dims[5] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(P), static_cast<cuuint64_t>(H), 2, static_cast<cuuint64_t>(slabs)};
  const cuuint64_t row = 2ull * H * D;
  const cuuint64_t strides[4] = {row, 2ull * D, row * P, 2 * row * P};
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  for (int i = 0; i < SA_TILE_PIECES; ++i) {
    if ((i + 1) * SA_PIECE > P) {                        // (no run of so many)
      maps.rows[i] = maps.rows[0];
      continue;
    }
    const cuuint32_t box[5] = {64, static_cast<cuuint32_t>((i + 1) * SA_PIECE), 1, 1, 1};
    const CUresult r = fn(&maps.rows[i], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void*>(d_kv), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    VB_CHECK_ARG(r == CUDA_SUCCESS, "vb_shared_attn: cuTensorMapEncodeTiled failed: CUresult %d", static_cast<int>(r));
  }
  uint8_t* at = static_cast<uint8_t*>(plan->d_buffer);
  SharedAttnParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(d_q), p.out = static_cast<__nv_bfloat16*>(d_out), p.kv = static_cast<const __nv_bfloat16*>(d_kv);
  p.entries = reinterpret_cast<const int4*>(at), p.parts = reinterpret_cast<const int4*>(at + l.parts);
  p.counts = reinterpret_cast<const int32_t*>(at + l.ints);
  p.whole = p.counts + l.groups, p.len = p.whole + 2 * l.groups + 1;
  p.blocks_of = reinterpret_cast<const int2*>(at + l.blocks_of);
  p.acc = reinterpret_cast<float*>(at + l.acc), p.stat = reinterpret_cast<float2*>(at + l.stat);
  p.slab_base = slab_base, p.slabs = slabs;
  VB_CHECK_ARG((p.wait_flag = wait_flag(WK_PREFILL_ATTN)) && (p.plan_flag = wait_flag(WK_PLAN)), "vb_shared_attn: no mapped host memory");
  p.expect = plan->d_row_tokens;
  p.rows = plan->rows, p.width = plan->width, p.sub = l.sub, p.subs = l.subs, p.groups = l.groups, p.cap = l.cap, p.page_size = P;
  p.n_q = plan->n_q, p.heads = H, p.G = plan->n_q / H, p.mpad = l.mpad, p.xt_tile = out_xt_tile;
  p.scale_log2 = sm_scale * 1.44269504088896f;
  return D == 64 ? launch_shared<64>(maps, p, plan->grid, stream) : launch_shared<128>(maps, p, plan->grid, stream);
}
