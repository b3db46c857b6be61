// Attention of one new token a row over a paged cache in which rows share pages: beams of one search, continuations of one prompt.
//
//   out[r] = sum_t softmax_t(q[r] . k[t] / sqrt d) v[t]     over row r's own tokens t
//
// What bounds it is the cache that is read.  Rows stand in groups (the rows of a request); of every column of their page table each DIFFERENT page is read
// once, with the set of rows that hold it, instead of once for every row.  A group's rows times the query heads of a key head, up to 64, are the rows of a
// matrix product: a tile of keys meets all of them while it is on chip.
//
//   plan (once a step)   a block a group lists its different pages in pieces of 16 to 64 tokens: {place in the cache, position, rows, tokens}; a block deals
//                        the tiles of all groups and key heads out to one block an SM in equal ranges
//   attention            a warp fetches the pieces of a tile by TMA into a ring; eight warps, each with 16 rows and a share of a tile's tokens, keep their own
//                        running maximum, sum and output in registers and meet at the end of a range only
//   join                 the ranges of a group and head meet
//
// Probabilities enter the second product as two bf16 parts (2^-17): what rounding them to one would add is as large as the rounding of the output.
#include <cudaTypedefs.h>

#include "../../include/vb_api.h"
#define VB_PDL_FAMILY 1
#include "rowmma.cuh"

namespace vb {

PFN_cuTensorMapEncodeTiled_v12000 encode_fn();

constexpr int SA_MAX_ROWS = 64;                  // rows of a group times query heads of a key head
constexpr int SA_WARPS = 8, SA_THREADS = 32 * (SA_WARPS + 1);
constexpr int SA_RING = 192 * 1024;
__host__ __device__ constexpr int sa_tile_tokens(int mt) { return mt == 1 ? 128 : 64; }
inline int sa_row_tiles(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }
inline int sa_piece(int page_size) { return page_size % 64 == 0 ? 64 : page_size % 32 == 0 ? 32 : 16; }

// ---- the plan -------------------------------------------------------------------------------------------------------------------
struct SharedPlanParams {
  int4* entries;                 // [groups][cap]: {token's place in a layer's pages, its position, rows that hold it, tokens | seen whole by all rows << 16}
  int32_t *counts, *tile0, *len; // [groups], [groups + 1], [rows]
  int4* parts;                   // [grid] {group, head, tile, tiles}
  int32_t* head;                 // {tiles of a block, tiles of all groups}
  const int32_t *table, *tokens;
  int rows, width, sub, subs, groups, cap, columns, pages, page_size, piece, tile_pieces, heads, grid;
};

constexpr int SP_THREADS = 512, SP_MAX_COLUMNS = 16384;

__device__ __forceinline__ int shared_first_row(const SharedPlanParams& p, int g, int& n) {
  const int in = g % p.subs * p.sub;
  n = min(p.sub, p.width - in);
  return g / p.subs * p.width + in;
}

// lane: row.  What its column c holds: the page (-1: none) and how many of the row's tokens stand there
__device__ __forceinline__ int shared_page(const SharedPlanParams& p, const int32_t* row, int len, int c, int& tokens) {
  tokens = min(p.page_size, len - c * p.page_size);
  if (tokens <= 0) return -1;
  const int g = row[c];
  return g >= 0 && g < p.pages ? g : -1;
}

__global__ void __launch_bounds__(SP_THREADS) shared_list_kernel(const __grid_constant__ SharedPlanParams p) {
  extern __shared__ int32_t sp_first[];                // [columns] pieces in front of a column
  __shared__ int sums[SP_THREADS / 32], carry;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = blockIdx.x;
  pdl_sync();
  int n;
  const int r0 = shared_first_row(p, g, n);
  int len = 0;
  if (lane < n) {
    len = p.tokens[r0 + lane];
    len = len < 0 ? 0 : min(len, p.columns * p.page_size);
    if (warp == 0) p.len[r0 + lane] = len;
  }
  const int32_t* row = p.table + static_cast<long long>(r0 + (lane < n ? lane : 0)) * p.columns;
  const uint32_t alive = __ballot_sync(0xffffffffu, len > 0);
  const int longest = __reduce_max_sync(0xffffffffu, len), columns = (longest + p.page_size - 1) / p.page_size;
  for (int c = warp; c < columns; c += SP_THREADS / 32) {
    int t;
    const int page = shared_page(p, row, len, c, t);
    const uint32_t same = __match_any_sync(0xffffffffu, page);
    int most = 0;
    for (uint32_t left = same; left; left &= left - 1) most = max(most, __shfl_sync(same, t, __ffs(left) - 1));
    const bool leads = page >= 0 && lane == __ffs(same) - 1;
    const int pieces = __reduce_add_sync(0xffffffffu, leads ? (most + p.piece - 1) / p.piece : 0);
    if (lane == 0) sp_first[c] = pieces;
  }
  if (tid == 0) carry = 0;
  __syncthreads();
  for (int c0 = 0; c0 < columns; c0 += SP_THREADS) {       // exclusive prefix over the columns
    const int c = c0 + tid, mine = c < columns ? sp_first[c] : 0;
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) sums[warp] = inc;
    __syncthreads();
    int before = carry, all = carry;
    for (int w = 0; w < SP_THREADS / 32; ++w) {
      if (w < warp) before += sums[w];
      all += sums[w];
    }
    if (c < columns) sp_first[c] = before + inc - mine;
    __syncthreads();
    if (tid == 0) carry = all;
    __syncthreads();
  }
  if (tid == 0) p.counts[g] = carry;
  int4* out = p.entries + static_cast<long long>(g) * p.cap;
  for (int c = warp; c < columns; c += SP_THREADS / 32) {
    int t;
    const int page = shared_page(p, row, len, c, t);
    const uint32_t same = __match_any_sync(0xffffffffu, page);
    int most = 0, least = p.page_size;
    for (uint32_t left = same; left; left &= left - 1) {
      const int v = __shfl_sync(same, t, __ffs(left) - 1);
      most = max(most, v), least = min(least, v);
    }
    const bool leads = page >= 0 && lane == __ffs(same) - 1;
    const int pieces = leads ? (most + p.piece - 1) / p.piece : 0;
    int inc = pieces;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    int at = sp_first[c] + inc - pieces;
    for (int i = 0; i < pieces; ++i) {
      const int off = i * p.piece, here = min(p.piece, most - off);
      const int whole = (same & alive) == alive && least >= off + p.piece;
      out[at++] = make_int4(page * p.page_size + off, c * p.page_size + off, static_cast<int>(same), here | whole << 16);
    }
  }
}

__global__ void __launch_bounds__(1024) shared_deal_kernel(const __grid_constant__ SharedPlanParams p) {
  __shared__ int sums[32], carry;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) carry = 0;
  pdl_sync();
  __syncthreads();
  for (int g0 = 0; g0 < p.groups; g0 += 1024) {
    const int g = g0 + tid, mine = g < p.groups ? (__ldcg(p.counts + g) + p.tile_pieces - 1) / p.tile_pieces : 0;
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) sums[warp] = inc;
    __syncthreads();
    int before = carry, all = carry;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) before += sums[w];
      all += sums[w];
    }
    if (g < p.groups) p.tile0[g] = before + inc - mine;
    __syncthreads();
    if (tid == 0) carry = all;
    __syncthreads();
  }
  const int total = carry, work = total * p.heads, each = max(1, (work + p.grid - 1) / p.grid);
  if (tid == 0) p.tile0[p.groups] = total, p.head[0] = each, p.head[1] = total;
  __syncthreads();
  for (int i = tid; i < p.grid; i += 1024) {
    const long long start = static_cast<long long>(i) * each;
    int4 part = make_int4(0, 0, 0, 0);
    if (start < work) {
      int lo = 0, hi = p.groups - 1;                    // the last group that begins at or before the start (later ones of the same start are empty)
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (static_cast<long long>(p.tile0[mid]) * p.heads <= start) lo = mid;
        else hi = mid - 1;
      }
      const int tiles = p.tile0[lo + 1] - p.tile0[lo], in = static_cast<int>(start - static_cast<long long>(p.tile0[lo]) * p.heads);
      part = make_int4(lo, in / tiles, in % tiles, min(each, static_cast<int>(work - start)));
    }
    p.parts[i] = part;
  }
}

// ---- attention -------------------------------------------------------------------------------------------------------------------
struct SharedAttnParams {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  const int4 *entries, *parts;
  const int32_t *counts, *tile0, *len, *head;
  float *acc, *stat;             // [slots][row tiles * 16][D], [slots][row tiles * 16][2]
  int64_t slab_base;
  unsigned char* wait_flag;
  int rows, width, sub, subs, groups, cap, page_size, piece, piece_log, n_q, heads, G, xt_tile;
  float scale_log2;
};

__device__ __forceinline__ int shared_group(const SharedAttnParams& p, int g, int& n) {
  const int in = g % p.subs * p.sub;
  n = min(p.sub, p.width - in);
  return g / p.subs * p.width + in;
}
__device__ __forceinline__ float sa_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <int D, int MT>
struct SaShape {
  static constexpr int TT = sa_tile_tokens(MT);                // tokens of a tile
  static constexpr int HALF = TT * 128;                        // bytes of 64 dimensions of its keys
  static constexpr int KV = HALF * (D / 64), STAGE = 2 * KV;
  static constexpr int STAGES = SA_RING / STAGE;
  static constexpr int WT = SA_WARPS / MT;                     // warps that share a tile's tokens
  static constexpr int TOK = TT / WT, BLOCKS = TOK / 16;       // tokens of a warp, 16 at a time
  static constexpr int MERGE = 4 * 16 * D * 4;                 // bytes: outputs of half the warps
  static constexpr int SMEM = 1024 + SA_RING + MERGE;
};

template <int D, int MT>
__global__ void __launch_bounds__(SA_THREADS, 1) shared_attn_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ SharedAttnParams p) {
  using L = SaShape<D, MT>;
  extern __shared__ uint8_t sa_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(sa_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float* merge = reinterpret_cast<float*>(ring + SA_RING);
  __shared__ uint64_t full[L::STAGES], empty[L::STAGES];
  __shared__ int4 meta[L::STAGES][8];
  __shared__ float merge_ml[4][16][2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  BoundedWait bw{p.wait_flag};
  if (tid == 0) {
#pragma unroll
    for (int s = 0; s < L::STAGES; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], SA_WARPS);
    fence_barrier_init();
    prefetch_tmap(&map);
  }
  __syncthreads();
  pdl_sync();
  int4 part = p.parts[blockIdx.x];
  if (part.w == 0) return;
  const int pieces = L::TT / p.piece;

  if (warp == SA_WARPS) {
    // ---- the warp that fetches: a lane a piece ----
    int g = part.x, h = part.y, tile = part.z, count = p.counts[g], tiles = p.tile0[g + 1] - p.tile0[g];
    auto entry = [&](int gg, int t, int n) {
      const int i = t * pieces + lane;
      return lane < pieces && i < n ? p.entries[static_cast<long long>(gg) * p.cap + i] : make_int4(0, 0, 0, 0);
    };
    int4 e = entry(g, tile, count);
    int stage = 0, asked = 0;
    uint32_t phase = 1;
    for (; asked < part.w; ++asked) {
      const int i = asked;
      const int4 now = e;
      const int head = h;
      if (i + 1 < part.w) {                                       // the next tile's pieces, while this one's place is still in use
        if (++tile == tiles) {
          tile = 0;
          if (++h == p.heads) {
            h = 0;
            do {
              ++g;
              tiles = p.tile0[g + 1] - p.tile0[g];
            } while (tiles == 0);
            count = p.counts[g];
          }
        }
        e = entry(g, tile, count);
      }
      bw.wait(&empty[stage], phase);
      if (__any_sync(0xffffffffu, bw.dead)) break;
      const bool has = (now.w & 0xffff) != 0;
      if (lane < pieces) meta[stage][lane] = now;
      const int n = __popc(__ballot_sync(0xffffffffu, has));
      __syncwarp();
      if (lane == 0) mbar_arrive_expect_tx(&full[stage], n * p.piece * D * 4);
      __syncwarp();
      if (has) {
        const int page = now.x / p.page_size, off = now.x - page * p.page_size, slab = static_cast<int>(p.slab_base + page);
        uint8_t* at = ring + stage * L::STAGE + lane * p.piece * 128;
#pragma unroll
        for (int d = 0; d < D / 64; ++d) {
          tma_load_5d(at + d * L::HALF, &map, &full[stage], d * 64, off, head, 0, slab);
          tma_load_5d(at + L::KV + d * L::HALF, &map, &full[stage], d * 64, off, head, 1, slab);
        }
      }
      if (++stage == L::STAGES) stage = 0, phase ^= 1;
    }
    // what has been asked for lands before the block leaves, whether or not the others waited for it
    BoundedWait last{p.wait_flag};
    for (int i = max(0, asked - L::STAGES); i < asked; ++i) last.wait(&full[i % L::STAGES], (i / L::STAGES) & 1);
    return;
  }

  // ---- the warps that multiply: 16 rows (row tile mt), tokens tg * TOK and further of every tile ----
  const int mt = warp % MT, tg = warp / MT;
  const int m0 = mt * 16 + (lane >> 2), m1 = m0 + 8;             // this thread's rows of the group's products
  int stage = 0;
  uint32_t phase = 0;
  int g = part.x, h = part.y, tile = part.z, left = part.w;
  const uint32_t ring_at = smem_u32(ring);
  while (left > 0) {
    const int tiles = p.tile0[g + 1] - p.tile0[g];
    if (tiles == 0) {
      ++g, h = 0;
      continue;
    }
    const int n_here = min(left, tiles - tile);
    left -= n_here;
    int n_rows;
    const int r0 = shared_group(p, g, n_rows), n_m = n_rows * p.G;
    const int i0 = m0 / p.G, i1 = m1 / p.G;                      // rows of the group
    const int len0 = m0 < n_m ? p.len[r0 + i0] : 0, len1 = m1 < n_m ? p.len[r0 + i1] : 0;
    const uint32_t bit0 = m0 < n_m ? 1u << i0 : 0u, bit1 = m1 < n_m ? 1u << i1 : 0u;
    uint32_t qf[D / 16][4];
    {
      const uint32_t* q0 = reinterpret_cast<const uint32_t*>(p.q + (static_cast<long long>(r0 + i0) * p.n_q + h * p.G + m0 - i0 * p.G) * D) + (lane & 3);
      const uint32_t* q1 = reinterpret_cast<const uint32_t*>(p.q + (static_cast<long long>(r0 + i1) * p.n_q + h * p.G + m1 - i1 * p.G) * D) + (lane & 3);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        qf[k][0] = m0 < n_m ? q0[k * 8] : 0u;
        qf[k][1] = m1 < n_m ? q1[k * 8] : 0u;
        qf[k][2] = m0 < n_m ? q0[k * 8 + 4] : 0u;
        qf[k][3] = m1 < n_m ? q1[k * 8 + 4] : 0u;
      }
    }
    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    float mx0 = -INFINITY, mx1 = -INFINITY, l0 = 0.f, l1 = 0.f;

    for (int it = 0; it < n_here; ++it) {
      bw.wait(&full[stage], phase);
      const uint32_t k_at = ring_at + stage * L::STAGE, v_at = k_at + L::KV;
      const int tok0 = tg * L::TOK;
#pragma unroll
      for (int blk = 0; blk < L::BLOCKS; ++blk) {
        const int tb = tok0 + blk * 16;                          // 16 tokens of one piece
        const int4 e = meta[stage][tb >> p.piece_log];
        const int off = tb & (p.piece - 1), here = (e.w & 0xffff) - off;      // tokens of the piece from here on
        if (here <= 0) continue;                                  // (uniform over the warp)
        const bool whole = e.w >> 16;
        float s[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
        {
          const int row = tb + ((lane >> 4) << 3) + (lane & 7), c = (lane >> 3) & 1;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            uint32_t b[4];
            const int chunk = (k & 3) * 2 + c;
            ldmatrix_x4(b, k_at + (k >> 2) * L::HALF + row * 128 + ((chunk ^ (row & 7)) << 4));
            mma_bf16_16816(s[0], qf[k], b[0], b[1]);
            mma_bf16_16816(s[1], qf[k], b[2], b[3]);
          }
        }
        const int t0 = (lane & 3) * 2;
        // what a row does not see: other rows' pages, tokens behind its last
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int pos = e.y + off + n * 8 + t0 + j;
            s[n][j] = whole || ((e.z & bit0) && pos < len0) ? s[n][j] * p.scale_log2 : -INFINITY;
            s[n][2 + j] = whole || ((e.z & bit1) && pos < len1) ? s[n][2 + j] * p.scale_log2 : -INFINITY;
          }
        float a = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1])), b = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
        a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1)), b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, 1));
        a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2)), b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, 2));
        const bool up = a > mx0 || b > mx1;
        if (__any_sync(0xffffffffu, up)) {
          const float n0 = fmaxf(mx0, a), n1 = fmaxf(mx1, b);
          const float c0 = n0 == -INFINITY ? 1.f : sa_ex2(mx0 - n0), c1 = n1 == -INFINITY ? 1.f : sa_ex2(mx1 - n1);
          mx0 = n0, mx1 = n1, l0 *= c0, l1 *= c1;
#pragma unroll
          for (int n = 0; n < D / 8; ++n) o[n][0] *= c0, o[n][1] *= c0, o[n][2] *= c1, o[n][3] *= c1;
        }
        const float z0 = mx0 == -INFINITY ? 0.f : mx0, z1 = mx1 == -INFINITY ? 0.f : mx1;
        bool seen[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            seen[n][j] = !(s[n][j] == -INFINITY);
            s[n][j] = sa_ex2(s[n][j] - (j < 2 ? z0 : z1));
          }
        l0 += (s[0][0] + s[0][1]) + (s[1][0] + s[1][1]);
        l1 += (s[0][2] + s[0][3]) + (s[1][2] + s[1][3]);
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = s[j >> 1][(j & 1) * 2], y = s[j >> 1][(j & 1) * 2 + 1];
          hi[j] = pack_bf16(x, y);
          lo[j] = pack_bf16(x - bf16_lo(hi[j]), y - bf16_hi(hi[j]));
        }
        const int vrow = tb + ((lane >> 3) & 1) * 8 + (lane & 7), vc = lane >> 4;
        uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;       // tokens that are none: the page holds anything there
        bool odd = false;
        if (!whole) {
          keep0 = (t0 < here ? 0xffffu : 0u) | (t0 + 1 < here ? 0xffff0000u : 0u);
          keep1 = (t0 + 8 < here ? 0xffffu : 0u) | (t0 + 9 < here ? 0xffff0000u : 0u);
          // a value that is not finite must not reach the rows that do not see it, through 0 times infinity
          uint32_t any = 0u;
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            uint32_t v[4];
            const int chunk = (d & 3) * 2 + vc;
            ldmatrix_x4_trans(v, v_at + (d >> 2) * L::HALF + vrow * 128 + ((chunk ^ (vrow & 7)) << 4));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t w = v[j] & ((j & 1) ? keep1 : keep0);
              any |= (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
            }
          }
          odd = __any_sync(0xffffffffu, any != 0u);
        }
        if (!odd) {
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            uint32_t v[4];
            const int chunk = (d & 3) * 2 + vc;
            ldmatrix_x4_trans(v, v_at + (d >> 2) * L::HALF + vrow * 128 + ((chunk ^ (vrow & 7)) << 4));
            v[0] &= keep0, v[1] &= keep1, v[2] &= keep0, v[3] &= keep1;
            mma_bf16_16816(o[2 * d], lo, v[0], v[1]);
            mma_bf16_16816(o[2 * d + 1], lo, v[2], v[3]);
            mma_bf16_16816(o[2 * d], hi, v[0], v[1]);
            mma_bf16_16816(o[2 * d + 1], hi, v[2], v[3]);
          }
        } else {
          // token by token, each row what it sees
          for (int t = 0; t < 16; ++t) {
            const int from = (lane & ~3) | ((t & 7) >> 1);
            float pr[2];
            bool sees[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const float even = t < 8 ? s[0][r * 2] : s[1][r * 2], other = t < 8 ? s[0][r * 2 + 1] : s[1][r * 2 + 1];
              const bool se = t < 8 ? seen[0][r * 2] : seen[1][r * 2], so = t < 8 ? seen[0][r * 2 + 1] : seen[1][r * 2 + 1];
              pr[r] = __shfl_sync(0xffffffffu, t & 1 ? other : even, from);
              sees[r] = __shfl_sync(0xffffffffu, static_cast<int>(t & 1 ? so : se), from) != 0;
            }
            const int vr = tb + t;
#pragma unroll
            for (int n = 0; n < D / 8; ++n) {
              uint32_t w;
              asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(v_at + (n >> 3) * L::HALF + vr * 128 + (((n & 7) ^ (vr & 7)) << 4) + t0 * 2) : "memory");
              if (sees[0]) o[n][0] += pr[0] * bf16_lo(w), o[n][1] += pr[0] * bf16_hi(w);
              if (sees[1]) o[n][2] += pr[1] * bf16_lo(w), o[n][3] += pr[1] * bf16_hi(w);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[stage]);
      if (++stage == L::STAGES) stage = 0, phase ^= 1;
    }

    // ---- the warps of a row tile meet: the upper half hands its part to the lower one, as often as it takes ----
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1), l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2), l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
#pragma unroll
    for (int half = SA_WARPS / 2; half >= MT; half >>= 1) {
      consumers_sync();                                          // (the last part has been read)
      if (warp >= half && warp < 2 * half) {
        float* at = merge + (warp - half) * 16 * D;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          *reinterpret_cast<float2*>(at + (n * 64 + lane) * 2) = make_float2(o[n][0], o[n][1]);
          *reinterpret_cast<float2*>(at + (n * 64 + 32 + lane) * 2) = make_float2(o[n][2], o[n][3]);
        }
        if ((lane & 3) == 0) {
          merge_ml[warp - half][lane >> 2][0] = mx0, merge_ml[warp - half][lane >> 2][1] = l0;
          merge_ml[warp - half][8 + (lane >> 2)][0] = mx1, merge_ml[warp - half][8 + (lane >> 2)][1] = l1;
        }
      }
      consumers_sync();
      if (warp < half) {
        const float* at = merge + warp * 16 * D;
        const float a = merge_ml[warp][lane >> 2][0], b = merge_ml[warp][8 + (lane >> 2)][0];
        const float n0 = fmaxf(mx0, a), n1 = fmaxf(mx1, b);
        const float c0 = n0 == -INFINITY ? 0.f : sa_ex2(mx0 - n0), c1 = n1 == -INFINITY ? 0.f : sa_ex2(mx1 - n1);
        const float d0 = n0 == -INFINITY ? 0.f : sa_ex2(a - n0), d1 = n1 == -INFINITY ? 0.f : sa_ex2(b - n1);
        l0 = l0 * c0 + merge_ml[warp][lane >> 2][1] * d0, l1 = l1 * c1 + merge_ml[warp][8 + (lane >> 2)][1] * d1;
        mx0 = n0, mx1 = n1;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          const float2 x = *reinterpret_cast<const float2*>(at + (n * 64 + lane) * 2), y = *reinterpret_cast<const float2*>(at + (n * 64 + 32 + lane) * 2);
          o[n][0] = o[n][0] * c0 + x.x * d0, o[n][1] = o[n][1] * c0 + x.y * d0;
          o[n][2] = o[n][2] * c1 + y.x * d1, o[n][3] = o[n][3] * c1 + y.y * d1;
        }
      }
    }
    if (warp < MT) {
      const long long slot = blockIdx.x + static_cast<long long>(g) * p.heads + h;
      float* acc = p.acc + slot * (MT * 16) * D;
      float* st = p.stat + slot * (MT * 16) * 2;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        if (m0 < n_m) *reinterpret_cast<float2*>(acc + m0 * D + n * 8 + (lane & 3) * 2) = make_float2(o[n][0], o[n][1]);
        if (m1 < n_m) *reinterpret_cast<float2*>(acc + m1 * D + n * 8 + (lane & 3) * 2) = make_float2(o[n][2], o[n][3]);
      }
      if ((lane & 3) == 0) {
        if (m0 < n_m) *reinterpret_cast<float2*>(st + m0 * 2) = make_float2(mx0, l0);
        if (m1 < n_m) *reinterpret_cast<float2*>(st + m1 * 2) = make_float2(mx1, l1);
      }
    }
    tile = 0;
    if (++h == p.heads) h = 0, ++g;
  }
}

// A warp a row of a group and head: the parts that blocks left of it, in their order.
constexpr int SJ_WARPS = 8;
template <int D>
__global__ void __launch_bounds__(32 * SJ_WARPS) shared_join_kernel(const __grid_constant__ SharedAttnParams p, int mpad) {
  const int lane = threadIdx.x & 31, unit = blockIdx.x, g = unit / p.heads, h = unit - g * p.heads;
  const int m = blockIdx.y * SJ_WARPS + (threadIdx.x >> 5);
  pdl_sync();
  int n_rows;
  const int r0 = shared_group(p, g, n_rows);
  if (m >= n_rows * p.G) return;
  const int row = r0 + m / p.G, head = h * p.G + m % p.G;
  const int each = p.head[0], tiles = p.tile0[g + 1] - p.tile0[g];
  float acc[D / 32];
#pragma unroll
  for (int d = 0; d < D / 32; ++d) acc[d] = 0.f;
  float total = 0.f;
  if (tiles > 0 && p.len[row] > 0) {
    const long long first = static_cast<long long>(p.tile0[g]) * p.heads + static_cast<long long>(h) * tiles;
    const int b0 = static_cast<int>(first / each), b1 = static_cast<int>((first + tiles - 1) / each);
    float top = -INFINITY;
    for (int b = b0 + lane; b <= b1; b += 32) top = fmaxf(top, p.stat[((static_cast<long long>(b) + unit) * mpad + m) * 2]);
    top = warp_max(top);
    if (top == -INFINITY) top = 0.f;                             // (scores that are all infinite or NaN: the sums below say so)
#pragma unroll 4
    for (int b = b0; b <= b1; ++b) {
      const long long at = (static_cast<long long>(b) + unit) * mpad + m;
      const float2 st = *reinterpret_cast<const float2*>(p.stat + at * 2);
      const float f = st.x == -INFINITY ? (st.y == 0.f ? 0.f : 1.f) : sa_ex2(st.x - top);      // (nothing seen; scores that are NaN)
      total += st.y * f;
#pragma unroll
      for (int d = 0; d < D / 64; ++d) {
        const float2 x = *reinterpret_cast<const float2*>(p.acc + at * D + d * 64 + lane * 2);
        if (f != 0.f) acc[2 * d] += x.x * f, acc[2 * d + 1] += x.y * f;
      }
    }
  }
  const float by = total != 0.f ? 1.f / total : 0.f;
#pragma unroll
  for (int d = 0; d < D / 64; ++d) {
    const int k = head * D + d * 64 + lane * 2;
    const size_t at = p.xt_tile ? xt_index(row, k, p.xt_tile, p.n_q * D / 64) : static_cast<size_t>(row) * p.n_q * D + k;
    *reinterpret_cast<uint32_t*>(p.out + at) = pack_bf16(acc[2 * d] * by, acc[2 * d + 1] * by);
  }
}

template <int D, int MT>
static int launch_shared(const CUtensorMap& map, const SharedAttnParams& p, int grid, void* stream) {
  VB_CHECK_CUDA((rm_smem<shared_attn_kernel<D, MT>>(SaShape<D, MT>::SMEM)));
  VB_LAUNCH_PDL((shared_attn_kernel<D, MT>), grid, SA_THREADS, (SaShape<D, MT>::SMEM), stream, map, p);
  VB_LAUNCH_PDL(shared_join_kernel<D>, dim3(p.groups * p.heads, (p.sub * p.G + SJ_WARPS - 1) / SJ_WARPS), 32 * SJ_WARPS, 0, stream, p, MT * 16);
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
  const int sub = shared_sub(s->width, s->n_q / s->n_kv);
  const int64_t pieces = static_cast<int64_t>(s->rows) * s->columns * (s->page_size / sa_piece(s->page_size));
  VB_CHECK_ARG(pieces * s->n_kv <= 0x3fffffff && sub > 0, "%s: %d rows of %d pages on %d heads", who, s->rows, s->columns, s->n_kv);
  return 0;
}

struct SharedLayout {
  int sub, subs, groups, cap, mpad;
  size_t entries, parts, ints, stat, acc, bytes;
};
static SharedLayout shared_layout(const VbSharedPlan* s) {
  SharedLayout l;
  const int G = s->n_q / s->n_kv;
  l.sub = shared_sub(s->width, G);
  l.subs = (s->width + l.sub - 1) / l.sub;
  l.groups = s->rows / s->width * l.subs;
  l.cap = l.sub * s->columns * (s->page_size / sa_piece(s->page_size));
  l.mpad = 16 * sa_row_tiles(l.sub * G);
  const size_t slots = static_cast<size_t>(s->grid) + static_cast<size_t>(l.groups) * s->n_kv;
  l.entries = 0;
  l.parts = l.entries + 16ull * l.groups * l.cap;
  l.acc = l.parts + 16ull * s->grid;
  l.stat = l.acc + 4ull * slots * l.mpad * s->head_dim;
  l.ints = l.stat + 8ull * slots * l.mpad;
  l.bytes = l.ints + 4ull * (2ull * l.groups + 1 + s->rows + 2);
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
  p.entries = reinterpret_cast<int4*>(at + l.entries);
  p.parts = reinterpret_cast<int4*>(at + l.parts);
  int32_t* ints = reinterpret_cast<int32_t*>(at + l.ints);
  p.head = ints, p.counts = ints + 2, p.tile0 = p.counts + l.groups, p.len = p.tile0 + l.groups + 1;
  p.table = d_table, p.tokens = d_tokens;
  p.rows = plan->rows, p.width = plan->width, p.sub = l.sub, p.subs = l.subs, p.groups = l.groups, p.cap = l.cap;
  p.columns = plan->columns, p.pages = pages, p.page_size = plan->page_size, p.piece = sa_piece(plan->page_size);
  p.tile_pieces = sa_tile_tokens(l.mpad / 16) / p.piece, p.heads = plan->n_kv, p.grid = plan->grid;
  VB_CHECK_CUDA(rm_smem<shared_list_kernel>(SP_MAX_COLUMNS * 4));
  VB_LAUNCH_PDL(shared_list_kernel, l.groups, SP_THREADS, plan->columns * 4, stream, p);
  VB_LAUNCH_PDL(shared_deal_kernel, 1, 1024, 0, stream, p);
  return 0;
}

extern "C" int vb_shared_attn(void* d_out, const void* d_q, const void* d_kv, int64_t slabs, int64_t slab_base, const VbSharedPlan* plan, float sm_scale, int out_xt_tile,
                              void* stream) {
  if (int rc = check_shared("vb_shared_attn", plan)) return rc;
  VB_CHECK_ARG(d_out && d_q && d_kv, "vb_shared_attn: null pointer");
  VB_CHECK_ARG(slabs > 0 && slabs <= 0x7fffffff && slab_base >= 0 && slab_base < slabs, "vb_shared_attn: slab %lld of %lld", static_cast<long long>(slab_base),
               static_cast<long long>(slabs));
  VB_CHECK_ARG(reinterpret_cast<uintptr_t>(d_kv) % 16 == 0 && reinterpret_cast<uintptr_t>(d_q) % 4 == 0 && reinterpret_cast<uintptr_t>(d_out) % 4 == 0,
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
  const int32_t* ints = reinterpret_cast<const int32_t*>(at + l.ints);
  SharedAttnParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(d_q), p.out = static_cast<__nv_bfloat16*>(d_out);
  p.entries = reinterpret_cast<const int4*>(at + l.entries), p.parts = reinterpret_cast<const int4*>(at + l.parts);
  p.head = ints, p.counts = ints + 2, p.tile0 = p.counts + l.groups, p.len = p.tile0 + l.groups + 1;
  p.acc = reinterpret_cast<float*>(at + l.acc), p.stat = reinterpret_cast<float*>(at + l.stat);
  p.slab_base = slab_base;
  VB_CHECK_ARG(p.wait_flag = wait_flag(WK_PREFILL_ATTN), "vb_shared_attn: no mapped host memory");
  p.rows = plan->rows, p.width = plan->width, p.sub = l.sub, p.subs = l.subs, p.groups = l.groups, p.cap = l.cap, p.page_size = P, p.piece = piece, p.piece_log = piece == 64 ? 6 : piece == 32 ? 5 : 4;
  p.n_q = plan->n_q, p.heads = H, p.G = plan->n_q / H, p.xt_tile = out_xt_tile;
  p.scale_log2 = sm_scale * 1.44269504088896f;
  const int mt = l.mpad / 16;
  if (D == 64) return mt == 1 ? launch_shared<64, 1>(map, p, plan->grid, stream) : mt == 2 ? launch_shared<64, 2>(map, p, plan->grid, stream) : launch_shared<64, 4>(map, p, plan->grid, stream);
  return mt == 1 ? launch_shared<128, 1>(map, p, plan->grid, stream) : mt == 2 ? launch_shared<128, 2>(map, p, plan->grid, stream) : launch_shared<128, 4>(map, p, plan->grid, stream);
}
