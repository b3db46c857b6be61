// Attention of one new token a row over a paged cache in which rows share pages: beams of one search, continuations of one prompt.
//
//   out[r] = sum_t softmax_t(q[r] . k[t] / sqrt d) v[t]     over row r's own tokens t
//
// What bounds it is the cache that is read.  Rows stand in groups (the rows of a request); of every column of their page table each DIFFERENT page is read
// once, with the set of rows that hold it, instead of once for every row.  A group's rows times the query heads of a key head, up to 128, are the accumulator
// rows of the tcgen05 core (attn_tc.cuh): a tile of 64 keys meets all of them while it is on chip.
//
//   plan (once a step)   a cluster a group lists its different pages in pieces of 16 to 64 tokens {place in the cache, position, rows, tokens}: first the tiles
//                        that all living rows see whole, then the rest; a block cuts the tiles of every group and key head into segments, two an SM in all
//   attention            a block a segment: maximum, denominator and unnormalised output of its rows
//   join                 the segments of a group and head meet, in their order
//
// Tiles that are seen whole need no masks.  In the others a row's probability is 0 where it does not see, and 0 times what is not finite is not 0.  So a block
// whose results are not finite, and that had such tiles, walks its segment again: values that are not finite are taken out on the way, and the rows that see
// them get them back at the end.  Finite caches never go there; what stands behind a row's last token is cleared in any case.
// Probabilities enter the second product as two bf16 parts (2^-17).
#include "../../include/vb_api.h"
#define VB_PDL_FAMILY 1
#include "attn_tc.cuh"
#include "rowmma.cuh"

namespace vb {

constexpr int SA_MAX_ROWS = 128;                 // rows of a group times query heads of a key head
inline int sa_piece(int page_size) { return page_size % 64 == 0 ? 64 : page_size % 32 == 0 ? 32 : 16; }

// ---- the plan -------------------------------------------------------------------------------------------------------------------
struct SharedPlanParams {
  int4* entries;                 // [groups][cap]: {token's place in a layer's pages, its position, rows that hold it, tokens}
  int4* segments;                // [grid + units] {group, head, first tile, tiles}
  int32_t *counts, *whole, *len; // [groups] pieces and tiles that are seen whole, [rows]
  int32_t* seg0;                 // [units + 1] segments in front of a unit
  const int32_t *table, *tokens;
  int rows, width, sub, subs, groups, cap, columns, pages, page_size, piece, tile_pieces, heads, grid;
};

constexpr int SP_THREADS = 512, SP_WARPS = SP_THREADS / 32, SP_MAX_COLUMNS = 16384, SP_CLUSTER = 8;

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
  c.pieces = leads ? (most + p.piece - 1) / p.piece : 0;
  c.whole = leads && (c.same & alive) == alive ? min(least, p.page_size) / p.piece : 0;
  return c;
}

// A cluster a group, its columns dealt out to the blocks in turn stretches.  Counted first, then written behind what stands in front.
__global__ void __launch_bounds__(SP_THREADS) shared_list_kernel(const __grid_constant__ SharedPlanParams p) {
  extern __shared__ int2 sp_first[];                   // whole pieces and others in front of a column, within the block
  __shared__ int2 sums[SP_WARPS], carry;
  __shared__ float totals[2];                          // (ints, read by the other blocks)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = cluster_ctarank(), blocks = cluster_nctarank(), g = blockIdx.x / blocks;
  pdl_sync();
  int n;
  const int r0 = shared_first_row(p, g, n);
  int len = 0;
  if (lane < n) {
    len = p.tokens[r0 + lane];
    len = len < 0 ? 0 : min(len, p.columns * p.page_size);
    if (rank == 0 && warp == 0) p.len[r0 + lane] = len;
  }
  const int32_t* row = p.table + static_cast<long long>(r0 + (lane < n ? lane : 0)) * p.columns;
  const uint32_t alive = __ballot_sync(0xffffffffu, len > 0);
  const int longest = __reduce_max_sync(0xffffffffu, len), columns = (longest + p.page_size - 1) / p.page_size;
  const int each = (columns + blocks - 1) / blocks, c_lo = min(columns, rank * each), here = min(columns, c_lo + each) - c_lo;
  auto page_at = [&](int c) { return c * p.page_size < len ? row[c] : -1; };
  for (int c0 = warp * 4; c0 < here; c0 += SP_WARPS * 4) {
    int page[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) page[j] = c0 + j < here ? page_at(c_lo + c0 + j) : -1;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c0 + j < here) {
        const SharedColumn c = shared_column(p, page[j], len - (c_lo + c0 + j) * p.page_size, alive);
        const int all = __reduce_add_sync(0xffffffffu, c.pieces), whole = __reduce_add_sync(0xffffffffu, c.whole);
        if (lane == 0) sp_first[c0 + j] = make_int2(whole, all - whole);
      }
  }
  if (tid == 0) carry = make_int2(0, 0);
  __syncthreads();
  for (int c0 = 0; c0 < here; c0 += SP_THREADS) {       // exclusive prefix over the block's columns
    const int c = c0 + tid;
    const int2 mine = c < here ? sp_first[c] : make_int2(0, 0);
    int2 inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, inc.x, o), y = __shfl_up_sync(0xffffffffu, inc.y, o);
      if (lane >= o) inc.x += x, inc.y += y;
    }
    if (lane == 31) sums[warp] = inc;
    __syncthreads();
    int2 before = carry, all = carry;
#pragma unroll
    for (int w = 0; w < SP_WARPS; ++w) {
      if (w < warp) before.x += sums[w].x, before.y += sums[w].y;
      all.x += sums[w].x, all.y += sums[w].y;
    }
    if (c < here) sp_first[c] = make_int2(before.x + inc.x - mine.x, before.y + inc.y - mine.y);
    __syncthreads();
    if (tid == 0) carry = all;
    __syncthreads();
  }
  if (tid == 0) totals[0] = __int_as_float(carry.x), totals[1] = __int_as_float(carry.y);
  cluster_sync_all();
  int w0 = 0, o0 = 0, all_w = 0, all_o = 0;             // pieces of the blocks in front, of all
  for (int b = 0; b < blocks; ++b) {
    const int w = __float_as_int(ld_dsmem_f32(&totals[0], b)), o = __float_as_int(ld_dsmem_f32(&totals[1], b));
    if (b < rank) w0 += w, o0 += o;
    all_w += w, all_o += o;
  }
  const int tiles_w = all_w / p.tile_pieces;            // (what is left of the whole ones fills the first of the others)
  if (rank == 0 && tid == 0) p.counts[g] = all_w + all_o, p.whole[g] = tiles_w;
  int4* out = p.entries + static_cast<long long>(g) * p.cap;
  for (int c0 = warp * 4; c0 < here; c0 += SP_WARPS * 4) {
    int page[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) page[j] = c0 + j < here ? page_at(c_lo + c0 + j) : -1;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c0 + j < here) {
        const int col = c_lo + c0 + j;
        const SharedColumn c = shared_column(p, page[j], len - col * p.page_size, alive);
        int2 inc = make_int2(c.whole, c.pieces - c.whole);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, inc.x, o), y = __shfl_up_sync(0xffffffffu, inc.y, o);
          if (lane >= o) inc.x += x, inc.y += y;
        }
        const int2 first = sp_first[c0 + j];
        int at_w = w0 + first.x + inc.x - c.whole, at_o = all_w + o0 + first.y + inc.y - (c.pieces - c.whole);
        for (int i = 0; i < c.pieces; ++i) {
          const int off = i * p.piece;
          out[i < c.whole ? at_w++ : at_o++] = make_int4(c.page * p.page_size + off, col * p.page_size + off, static_cast<int>(c.same), min(p.piece, c.tokens - off));
        }
      }
  }
  cluster_sync_all();                                   // (totals have been read)
}

__global__ void __launch_bounds__(1024) shared_deal_kernel(const __grid_constant__ SharedPlanParams p) {
  __shared__ int sums[33];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_sync();
  auto tiles_of = [&](int g) { return (__ldcg(p.counts + g) + p.tile_pieces - 1) / p.tile_pieces; };
  // sum (op 0) or maximum over the block
  auto meet = [&](int v, bool maximum) {
    v = maximum ? __reduce_max_sync(0xffffffffu, v) : __reduce_add_sync(0xffffffffu, v);
    __syncthreads();
    if (lane == 0) sums[warp] = v;
    __syncthreads();
    v = sums[lane];
    return maximum ? __reduce_max_sync(0xffffffffu, v) : __reduce_add_sync(0xffffffffu, v);
  };
  int mine = 0, longest = 0;
  for (int g = tid; g < p.groups; g += 1024) {
    const int t = tiles_of(g);
    mine += t, longest = max(longest, t);
  }
  const int total = meet(mine, false) * p.heads, most = meet(longest, true);
  // tiles of a segment: the fewest with which all segments run at once, where that is possible
  int lo = max(1, (total + p.grid - 1) / p.grid), hi = max(lo, most);
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    mine = 0;
    for (int g = tid; g < p.groups; g += 1024) mine += (tiles_of(g) + mid - 1) / mid;
    if (meet(mine, false) * p.heads <= p.grid) hi = mid;
    else lo = mid + 1;
  }
  const int units = p.groups * p.heads;
  const int each = units <= p.grid ? lo : max(1, (total + p.grid - 1) / p.grid);
  int carry = 0;
  for (int u0 = 0; u0 < units; u0 += 1024) {
    const int u = u0 + tid, g = u / p.heads, h = u - g * p.heads;
    const int tiles = u < units ? tiles_of(g) : 0, n = (tiles + each - 1) / each;
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = inc;
    __syncthreads();
    int before = carry, all = carry;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) before += sums[w];
      all += sums[w];
    }
    const int at = before + inc - n;
    if (u < units) {
      p.seg0[u] = at;
      for (int i = 0; i < n; ++i) p.segments[at + i] = make_int4(g, h, i * each, min(each, tiles - i * each));
    }
    carry = all;
  }
  if (tid == 0) p.seg0[units] = carry;
  for (int i = carry + tid; i < p.grid + units; i += 1024) p.segments[i] = make_int4(0, 0, 0, 0);
}

// ---- attention -------------------------------------------------------------------------------------------------------------------
struct SharedAttnParams {
  const __nv_bfloat16 *q, *kv;
  __nv_bfloat16* out;
  const int4 *entries, *segments;
  const int32_t *counts, *whole, *len, *seg0;
  float* acc;                    // [segments][mpad][D]
  float2* stat;                  // [segments][mpad] maximum (base 2), denominator against it
  long long slab_base;
  unsigned char* wait_flag;
  int rows, width, sub, subs, groups, cap, page_size, piece, tile_pieces, n_q, heads, G, mpad, xt_tile;
  float scale_log2;
};

__device__ __forceinline__ int shared_group(const SharedAttnParams& p, int g, int& n) {
  const int in = g % p.subs * p.sub;
  n = min(p.sub, p.width - in);
  return g / p.subs * p.width + in;
}

// what this thread's row sees of a segment, and where its part goes
template <int D>
struct SharedRows {
  static constexpr bool HOLE = false, STAGED = false;
  static constexpr int hole0 = 0, hole1 = 0;
  const SharedAttnParams& p;
  uint8_t* smem;
  const int4 *entries, *meta;    // of the group; of the last four tiles with masks
  int count, whole, t0, n_tiles; // pieces; tiles that need no mask; the segment
  int row0, n_rows, head, group; // first row, rows, key head, query heads of it
  int len, bit;
  bool ok;
  float scale_log2;
  float2* stat;
  bool careful;                  // values that are not finite have been taken out
  mutable bool bad;              // a result that is not finite
  mutable uint64_t seen;
  __device__ __forceinline__ int tile(int it) const { return t0 + it; }
  __device__ __forceinline__ int4 piece(int i) const { return i < count ? entries[i] : make_int4(0, 0, 0, 0); }
  __device__ __forceinline__ uint64_t mask(const int4* pieces, int n_pieces) const {
    uint64_t m = 0ull;
    for (int i = 0; i < n_pieces; ++i) {
      const int4 e = pieces[i];
      const int n = (static_cast<uint32_t>(e.z) >> bit & 1u) ? min(len - e.y, e.w) : 0;
      if (n > 0) m |= (n < 64 ? (1ull << n) - 1ull : ~0ull) << (i * p.piece);
    }
    return m;
  }
  __device__ __forceinline__ bool full(int tok0) const {
    seen = ~0ull;
    const int t = tok0 / PTC_KT;
    if (t >= whole && ok) seen = mask(meta + (t - t0 & 3) * 4, p.tile_pieces);      // (a row that is none may have anything)
    return seen == ~0ull;
  }
  __device__ __forceinline__ bool visible(int kj) const { return seen >> (kj & (PTC_KT - 1)) & 1ull; }
  __device__ __forceinline__ const __nv_bfloat16* q_row(int t, int g) const {
    return t < n_rows ? p.q + (static_cast<size_t>(row0 + t) * p.n_q + head * group + g) * D : nullptr;
  }
  __device__ __forceinline__ uint4* out_at(int, int, int) const { return nullptr; }
  __device__ __forceinline__ float finish(float m_ref, float l) const {
    if (ok) *stat = make_float2(m_ref, l);
    return 1.f;
  }
  // a thread's row goes to the place of the keys and values (they have been multiplied): 16-byte chunk c of row r at chunk c ^ (r & 15) of its 16 or 32
  __device__ __forceinline__ float4* staged(int r, int c) const { return reinterpret_cast<float4*>(smem + PtcLayout<D>::K) + r * (D / 4) + ((c & ~15) | ((c ^ r) & 15)); }
  __device__ __forceinline__ void store(int c0, const uint32_t (&o)[32], float) const {
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(o[i]);
    if (careful && ok) give_back(c0, v);
#pragma unroll
    for (int i = 0; i < 32; ++i) bad |= !isfinite(v[i]);
#pragma unroll
    for (int c = 0; c < 8; ++c) *staged(threadIdx.x, (c0 >> 2) + c) = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
  }
  // what is not finite among the values that the row sees, in tiles where it was taken out
  __device__ __noinline__ void give_back(int c0, float (&v)[32]) const {
    for (int t = max(t0, whole); t < t0 + n_tiles; ++t) {
      const int first = t * p.tile_pieces;
      const uint64_t m = mask(entries + first, min(p.tile_pieces, count - first));
      for (int k = 0; k < PTC_KT; ++k) {
        if (!(m >> k & 1ull)) continue;
        const int4 e = piece(t * p.tile_pieces + k / p.piece);
        const int tok = e.x + k % p.piece, page = tok / p.page_size, slot = tok - page * p.page_size;
        const uint32_t* src = reinterpret_cast<const uint32_t*>(p.kv + ((((p.slab_base + page) * 2 + 1) * p.page_size + slot) * p.heads + head) * D + c0);
        for (int i = 0; i < 16; ++i) {
          const uint32_t w = src[i];
          if ((w & 0x7f80u) == 0x7f80u) v[2 * i] += bf16_lo(w);
          if ((w & 0x7f800000u) == 0x7f800000u) v[2 * i + 1] += bf16_hi(w);
        }
      }
    }
  }
};

// A lane a piece of the tile: its boxes, K or V
template <int D>
__device__ __forceinline__ void shared_fetch(const SharedAttnParams& p, const CUtensorMap* map, const int4& e, int part, int head, uint32_t dst, uint64_t* bar) {
  const int lane = threadIdx.x & 31;
  const bool has = e.w > 0;
  const int n = __popc(__ballot_sync(0xffffffffu, has));
  if (lane == 0) mbar_arrive_expect_tx(bar, n * p.piece * D * 2);
  __syncwarp();
  if (has) {
    const int page = e.x / p.page_size, slot = e.x - page * p.page_size;
#pragma unroll
    for (int kb = 0; kb < D / 64; ++kb)
      ptc_tma_5d(dst + kb * (PTC_KT * 128) + lane * p.piece * 128, map, smem_u32(bar), kb * 64, slot, head, part, static_cast<int>(p.slab_base + page));
  }
  __syncwarp();
}

template <int D>
__global__ void __launch_bounds__(PTC_THREADS, 2) shared_attn_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ SharedAttnParams p) {
  using L = PtcLayout<D>;
  extern __shared__ uint8_t sa_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(sa_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  static_assert(sizeof(PtcShared) <= 256, "two of them and four tiles' pieces behind the operands");
  PtcShared *sh = reinterpret_cast<PtcShared*>(smem + L::BAR), *sh2 = reinterpret_cast<PtcShared*>(smem + L::BAR + 256);
  int4* meta = reinterpret_cast<int4*>(smem + L::BAR + 512);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  BoundedWait bw{p.wait_flag};
  pdl_wait();
  const int4 seg = p.segments[blockIdx.x];
  pdl_trigger();
  if (seg.w == 0) return;
  if (tid == 0) {
    ptc_init(sh, 1);
    ptc_init(sh2, 1);
    prefetch_tmap(&map);
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

  const int g = seg.x, head = seg.y, n_tiles = seg.w;
  int n_rows;
  const int row0 = shared_group(p, g, n_rows), t = tid / p.G;
  const bool ok = warp < 4 && t < n_rows;
  SharedRows<D> rows{p, smem, p.entries + static_cast<long long>(g) * p.cap, meta, p.counts[g], p.whole[g], seg.z, n_tiles, row0, n_rows, head, p.G,
                     ok ? p.len[row0 + t] : 0, ok ? t : 0, ok, p.scale_log2, p.stat + static_cast<long long>(blockIdx.x) * p.mpad + tid, false, false, ~0ull};
#pragma unroll 1
  for (int pass = 0;; ++pass) {
    rows.careful = pass != 0;
    rows.bad = false;
    if (warp < 4) {
      ptc_softmax<D>(smem, sh, rows, bw);
      fence_proxy_async();                                    // (results stand where keys and values may come again)
    } else if (warp == 4) {
      ptc_issue<D>(smem, sh, n_tiles, bw);
    } else {
      const bool values = warp == 6;
      uint64_t *full = values ? sh->v_full : sh->k_full, *empty = values ? sh->v_empty : sh->k_empty;
      const uint32_t ring = smem_u32(smem + (values ? L::V : L::K));
      auto find = [&](int j) { return lane < p.tile_pieces && j < n_tiles ? rows.piece((seg.z + j) * p.tile_pieces + lane) : make_int4(0, 0, 0, 0); };
      int4 next = find(0);
      uint32_t turn = 0;                                      // bit s: parity of stage s's next tile that is changed
      for (int j = 0; j < n_tiles; ++j) {
        const int s = j & 1;
        const int4 e = next;
        next = find(j + 1);
        bw.wait(&empty[s], ((j >> 1) & 1) ^ 1);
        if (!__all_sync(0xffffffffu, !bw.dead)) {
          bw.dead = true;
          break;
        }
        const bool masked = seg.z + j >= rows.whole;
        // (tile j + 4's stands where tile j's was: its stage was empty, so tile j + 2's scores have been multiplied, and tile j's output with them)
        if (!values && masked && lane < p.tile_pieces) meta[(j & 3) * 4 + lane] = e;
        const uint32_t short_ = __ballot_sync(0xffffffffu, lane < p.tile_pieces && e.w < p.piece);
        const bool change = values && masked && (short_ || rows.careful);
        shared_fetch<D>(p, &map, e, values ? 1 : 0, head, ring + s * L::TILE, change ? &sh->v_part[s] : &full[s]);
        if (!change) continue;
        bw.wait(&sh->v_part[s], turn >> s & 1u);
        if (!__all_sync(0xffffffffu, !bw.dead)) {
          bw.dead = true;
          break;
        }
        turn ^= 1u << s;
        uint4* v_tile = reinterpret_cast<uint4*>(smem + L::V + s * L::TILE);
        for (uint32_t left = short_; left; left &= left - 1) {      // rows that are no tokens become zeros
          const int i = __ffs(left) - 1, tokens = __shfl_sync(0xffffffffu, e.w, i), from = (i * p.piece + tokens) * 8, n = (p.piece - tokens) * 8;
#pragma unroll
          for (int kb = 0; kb < D / 64; ++kb)
            for (int k = lane; k < n; k += 32) v_tile[kb * PTC_KT * 8 + from + k] = make_uint4(0u, 0u, 0u, 0u);
        }
        if (rows.careful) {
          __syncwarp();
          for (int i = lane; i < (D / 64) * PTC_KT * 8; i += 32) {
            uint4 v = v_tile[i];
            uint32_t* w = &v.x;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if ((w[k] & 0x7f80u) == 0x7f80u) w[k] &= 0xffff0000u;
              if ((w[k] & 0x7f800000u) == 0x7f800000u) w[k] &= 0xffffu;
            }
            v_tile[i] = v;
          }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[s]);
      }
      ptc_let_land(bw.dead);
      __syncwarp();
    }
    tc_fence_before();
    const bool again = __syncthreads_or(rows.bad && rows.len > 0 && seg.z + n_tiles > rows.whole && !bw.dead);
    tc_fence_after();
    if (!again || pass) break;
    sh = sh2;
  }
  if (warp < 4 && !bw.dead) {                                 // whole rows, 16 bytes a lane
    float4* acc = reinterpret_cast<float4*>(p.acc + static_cast<long long>(blockIdx.x) * p.mpad * D);
    const int n = n_rows * p.G * (D / 4);
    for (int i = tid; i < n; i += 128) acc[i] = *rows.staged(i / (D / 4), i % (D / 4));
  }
  if (warp == 4) tmem_dealloc(tmem_base, 256);
}

// The segments of a group and head meet: WPR warps a row, each every WPR-th segment, a lane D / 32 neighbouring dimensions.
constexpr int SJ_WARPS = 8;
template <int D, int WPR>
__global__ void __launch_bounds__(32 * SJ_WARPS) shared_join_kernel(const __grid_constant__ SharedAttnParams p) {
  constexpr int E = D / 32;
  __shared__ float part[SJ_WARPS][32][E + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, unit = blockIdx.x, g = unit / p.heads, h = unit - g * p.heads;
  const int m = blockIdx.y * (SJ_WARPS / WPR) + warp / WPR, sub = warp % WPR;
  pdl_sync();
  int n_rows;
  const int r0 = shared_group(p, g, n_rows);
  const bool on = m < n_rows * p.G;
  const int row = r0 + (on ? m / p.G : 0), k = (h * p.G + (on ? m % p.G : 0)) * D + lane * E;
  float acc[E], total = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  if (on && p.len[row] > 0) {
    const int s0 = p.seg0[unit], s1 = p.seg0[unit + 1];
    float top = -INFINITY;
    for (int s = s0 + lane; s < s1; s += 32) top = fmaxf(top, p.stat[static_cast<long long>(s) * p.mpad + m].x);
    top = warp_max(top);
    if (top == -INFINITY) top = 0.f;                            // (scores that are all NaN: the sums below say so)
#pragma unroll 8
    for (int s = s0 + sub; s < s1; s += WPR) {
      const long long at = static_cast<long long>(s) * p.mpad + m;
      const float2 st = p.stat[at];
      const float f = st.x == -INFINITY ? (st.y == 0.f ? 0.f : 1.f) : ptc_ex2(st.x - top);      // (nothing seen; scores that are NaN)
      float v[E];
      if (E == 4) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(p.acc + at * D + lane * E);
      else *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(p.acc + at * D + lane * E);
      total += st.y * f;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += v[e] * f;
    }
  }
  if (WPR > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) part[warp][lane][e] = acc[e];
    part[warp][lane][E] = total;
    __syncthreads();
    if (sub == 0) {
#pragma unroll
      for (int w = 1; w < WPR; ++w) {
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += part[warp + w][lane][e];
        total += part[warp + w][lane][E];
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
static int launch_shared(const CUtensorMap& map, const SharedAttnParams& p, int grid, void* stream) {
  const int units = p.groups * p.heads, m = p.sub * p.G;
  VB_CHECK_CUDA(rm_smem<shared_attn_kernel<D>>(PtcLayout<D>::TOTAL + 512));
  VB_LAUNCH_PDL(shared_attn_kernel<D>, grid + units, PTC_THREADS, PtcLayout<D>::TOTAL + 512, stream, map, p);
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
  const int64_t pieces = static_cast<int64_t>(s->rows) * s->columns * (s->page_size / sa_piece(s->page_size));
  VB_CHECK_ARG(pieces * s->n_kv <= 0x3fffffff, "%s: %d rows of %d pages on %d heads", who, s->rows, s->columns, s->n_kv);
  return 0;
}

struct SharedLayout {
  int sub, subs, groups, cap, mpad;
  size_t segments, acc, stat, ints, bytes;      // entries first
};
static SharedLayout shared_layout(const VbSharedPlan* s) {
  SharedLayout l;
  const int G = s->n_q / s->n_kv;
  l.sub = shared_sub(s->width, G);
  l.subs = (s->width + l.sub - 1) / l.sub;
  l.groups = s->rows / s->width * l.subs;
  l.cap = l.sub * s->columns * (s->page_size / sa_piece(s->page_size));
  l.mpad = (l.sub * G + 15) / 16 * 16;
  const size_t units = static_cast<size_t>(l.groups) * s->n_kv, segments = s->grid + units;
  l.segments = 16ull * l.groups * l.cap;
  l.acc = l.segments + 16ull * segments;
  l.stat = l.acc + 4ull * segments * l.mpad * s->head_dim;
  l.ints = l.stat + 8ull * segments * l.mpad;
  l.bytes = l.ints + 4ull * (2ull * l.groups + units + 1 + s->rows);
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
  p.segments = reinterpret_cast<int4*>(at + l.segments);
  p.counts = reinterpret_cast<int32_t*>(at + l.ints);
  p.whole = p.counts + l.groups, p.seg0 = p.whole + l.groups, p.len = p.seg0 + l.groups * plan->n_kv + 1;
  p.table = d_table, p.tokens = d_tokens;
  p.rows = plan->rows, p.width = plan->width, p.sub = l.sub, p.subs = l.subs, p.groups = l.groups, p.cap = l.cap;
  p.columns = plan->columns, p.pages = pages, p.page_size = plan->page_size, p.piece = sa_piece(plan->page_size);
  p.tile_pieces = PTC_KT / p.piece, p.heads = plan->n_kv, p.grid = plan->grid;
  const int cluster = plan->columns > 256 ? SP_CLUSTER : plan->columns > 64 ? 4 : plan->columns > 16 ? 2 : 1;
  VB_CHECK_CUDA(rm_smem<shared_list_kernel>(SP_MAX_COLUMNS * 8));
  VB_LAUNCH_PDL_CLUSTER(shared_list_kernel, l.groups * cluster, SP_THREADS, (plan->columns + cluster - 1) / cluster * 8, stream, cluster, p);
  VB_LAUNCH_PDL(shared_deal_kernel, 1, 1024, 0, stream, p);
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
  const int D = plan->head_dim, H = plan->n_kv, P = plan->page_size, piece = sa_piece(P);
  auto fn = encode_fn();
  VB_CHECK_ARG(fn, "vb_shared_attn: cuTensorMapEncodeTiled not available (no CUDA driver?)");
  CUtensorMap map;
  const cuuint64_t dims[5] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(P), static_cast<cuuint64_t>(H), 2, static_cast<cuuint64_t>(slabs)};
  const cuuint64_t row = 2ull * H * D;
  const cuuint64_t strides[4] = {row, 2ull * D, row * P, 2 * row * P};
  const cuuint32_t box[5] = {64, static_cast<cuuint32_t>(piece), 1, 1, 1}, estr[5] = {1, 1, 1, 1, 1};
  const CUresult r = fn(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void*>(d_kv), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  VB_CHECK_ARG(r == CUDA_SUCCESS, "vb_shared_attn: cuTensorMapEncodeTiled failed: CUresult %d", static_cast<int>(r));
  uint8_t* at = static_cast<uint8_t*>(plan->d_buffer);
  SharedAttnParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(d_q), p.out = static_cast<__nv_bfloat16*>(d_out), p.kv = static_cast<const __nv_bfloat16*>(d_kv);
  p.entries = reinterpret_cast<const int4*>(at), p.segments = reinterpret_cast<const int4*>(at + l.segments);
  p.counts = reinterpret_cast<const int32_t*>(at + l.ints);
  p.whole = p.counts + l.groups, p.seg0 = p.whole + l.groups, p.len = p.seg0 + l.groups * H + 1;
  p.acc = reinterpret_cast<float*>(at + l.acc), p.stat = reinterpret_cast<float2*>(at + l.stat);
  p.slab_base = slab_base;
  VB_CHECK_ARG(p.wait_flag = wait_flag(WK_PREFILL_ATTN), "vb_shared_attn: no mapped host memory");
  p.rows = plan->rows, p.width = plan->width, p.sub = l.sub, p.subs = l.subs, p.groups = l.groups, p.cap = l.cap, p.page_size = P, p.piece = piece;
  p.tile_pieces = PTC_KT / piece, p.n_q = plan->n_q, p.heads = H, p.G = plan->n_q / H, p.mpad = l.mpad, p.xt_tile = out_xt_tile;
  p.scale_log2 = sm_scale * 1.44269504088896f;
  return D == 64 ? launch_shared<64>(map, p, plan->grid, stream) : launch_shared<128>(map, p, plan->grid, stream);
}
