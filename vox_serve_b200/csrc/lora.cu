// Low-rank adapters of many requests beside a shared projection.
//
//   v[t, s r + j] = scale_a sum_k A_a[s, j, k] x[t, k]            (a: the adapter of row t; s: slice of the projection's columns, q | k | v)
//   out[t, n] = base[t, n] + sum_j B_a[n, j] v[t, s(n) r + j]
//
//   vb_lora_plan      rows of a step by adapter: a table of row tiles that every projection of every layer works through
//   vb_lora           out as fp32 (one more split-K plane of the projection: its consumer sums planes anyway) or as bf16 rows with a base
//   vb_lora_gate_up   silu(gate) * up from the projection's fp32 planes with both adapters' products added
//
// A tile is up to 16 rows (steps of at most 64) or 64 rows of one adapter.  Two launches a call: the first product over pieces of K, its partial
// sums left as planes; the second adds the planes and walks the columns.  The bank keeps A and B in the order in which lanes take them (one
// 16-byte load per lane and product step, 512 bytes in a row per warp), so both are streamed once per tile without a detour through shared memory.
//
// Sums are fp32.  v is not rounded on its way into the second product: it enters as three bf16 parts (exact, rowmma.cuh) where the result is fp32, as
// two (off by 2^-15 of v at most) where the result is rounded to bf16 anyway.
#include "../../include/vb_api.h"
#define VB_PDL_FAMILY 4
#include "rowmma.cuh"

namespace vb {

constexpr int LORA_MAX_SLOTS = 1023;       // (a thread of the planning block each, and one for rows without an adapter)
constexpr int LORA_MAX_RANK = 128;
constexpr int LORA_MAX_SLICES = 4;
constexpr int LORA_THREADS = 256;

// ---- rows by adapter ------------------------------------------------------------------------------------------------------------
// tiles[0].x = how many; tiles[1 + i] = {adapter or -1, first place in `order`, rows, 0}.  One block: a counting sort in shared memory.  The
// order of an adapter's rows among themselves may differ from run to run; a row's result does not depend on its place.
__global__ void __launch_bounds__(1024) lora_plan_kernel(int32_t* __restrict__ order, int4* __restrict__ tiles, const int32_t* __restrict__ ids, int T,
                                                         int slots, int tile_rows) {
  __shared__ int cnt[1024], first[1024];
  __shared__ int warp_rows[32], warp_tiles[32];
  pdl_sync();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cnt[tid] = 0;
  __syncthreads();
  for (int t = tid; t < T; t += 1024) {
    const int a = ids[t];
    atomicAdd(&cnt[a >= 0 && a < slots ? a : slots], 1);
  }
  __syncthreads();
  const int rows = tid <= slots ? cnt[tid] : 0, n = (rows + tile_rows - 1) / tile_rows;
  int r = rows, m = n;                      // inclusive sums over the threads
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int rr = __shfl_up_sync(0xffffffffu, r, o), mm = __shfl_up_sync(0xffffffffu, m, o);
    if (lane >= o) { r += rr; m += mm; }
  }
  if (lane == 31) { warp_rows[warp] = r; warp_tiles[warp] = m; }
  __syncthreads();
  if (warp == 0) {
    int a = warp_rows[lane], b = warp_tiles[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int aa = __shfl_up_sync(0xffffffffu, a, o), bb = __shfl_up_sync(0xffffffffu, b, o);
      if (lane >= o) { a += aa; b += bb; }
    }
    warp_rows[lane] = a;
    warp_tiles[lane] = b;
  }
  __syncthreads();
  if (warp > 0) { r += warp_rows[warp - 1]; m += warp_tiles[warp - 1]; }
  const int row0 = r - rows, tile0 = m - n;
  first[tid] = row0;
  for (int i = 0; i < n; ++i)
    tiles[1 + tile0 + i] = make_int4(tid < slots ? tid : -1, row0 + i * tile_rows, min(tile_rows, rows - i * tile_rows), 0);
  if (tid == 1023) tiles[0] = make_int4(m, T, tile_rows, 0);
  __syncthreads();
  cnt[tid] = 0;
  __syncthreads();
  for (int t = tid; t < T; t += 1024) {
    int a = ids[t];
    a = a >= 0 && a < slots ? a : slots;
    order[first[a] + atomicAdd(&cnt[a], 1)] = t;
  }
}

struct LoraParams {
  const int4* tiles;
  const int32_t* order;
  const __nv_bfloat16* x;
  long long ldx;
  const uint4 *a, *b;              // [slots][S][rank / 16][K / 32][2][32 lanes], [slots][column blocks of 32][rank / 16][2][32 lanes]
  long long a_slot, b_slot;        // 16-byte units
  const float* scale;
  float* v;                        // [k_split][T][VR]
  int T, K, kb32, rank_tiles, VR, k_split;      // VR = S * rank
  // second product
  int blocks;                      // column blocks of 32 over all slices
  int slices, block0[LORA_MAX_SLICES + 1], col0[LORA_MAX_SLICES + 1];
  void* out;
  const void* base;
  long long ldo, ld_base;
  // gate | up
  const float* planes;
  int splits, half, width, ff, xt_rows, xt_kb;
};

// ---- first product: v = scale A x -------------------------------------------------------------------------------------------------
// Block: a tile x a piece of K, the warps taking turns of 64 k; RT rank tiles (16 each) at a time over NT column tiles of 8 rows.  Where rows have
// more rank tiles than RT the block walks its piece again (x from L2 then).
template <int NT, int RT>
__global__ void __launch_bounds__(LORA_THREADS) lora_down_kernel(const LoraParams p) {
  extern __shared__ float red[];            // [8 warps][16][NT * 8 + 4]
  constexpr int LD = NT * 8 + 4;
  __shared__ int rows_s[NT * 8];
  pdl_sync();
  const int tile = blockIdx.x;
  if (tile >= p.tiles[0].x) return;
  const int4 tl = p.tiles[1 + tile];
  if (tl.x < 0) return;                     // no adapter: the second kernel does not look at v
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int n = tl.z;
  if (tid < NT * 8) rows_s[tid] = tid < n ? p.order[tl.y + tid] : -1;
  __syncthreads();
  const __nv_bfloat16* xr[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int row = rows_s[j * 8 + g];
    xr[j] = row >= 0 ? p.x + row * p.ldx + t4 * 8 : nullptr;
  }
  const uint4* a = p.a + tl.x * p.a_slot + lane;
  // pieces in units of 64 k
  const int units = (p.kb32 + 1) >> 1, u0 = static_cast<int>(static_cast<long long>(units) * blockIdx.y / p.k_split),
            u1 = static_cast<int>(static_cast<long long>(units) * (blockIdx.y + 1) / p.k_split);
  const float scale = p.scale[tl.x];
  const int rts = p.VR >> 4;
  for (int rt0 = 0; rt0 < rts; rt0 += RT) {
    float acc[RT][NT][4];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[i][j][c] = 0.f;
    for (int u = u0 + warp; u < u1; u += LORA_THREADS / 32) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int kb = 2 * u + h;
        if (kb >= p.kb32) break;
        const bool in = kb * 32 + t4 * 8 < p.K;
        uint4 xv[NT], av[RT][2];
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int s = 0; s < 2; ++s)
            av[i][s] = rt0 + i < rts ? __ldg(a + ((static_cast<long long>(rt0 + i) * p.kb32 + kb) * 2 + s) * 32) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int j = 0; j < NT; ++j)
          xv[j] = in && xr[j] ? *reinterpret_cast<const uint4*>(xr[j] + kb * 32) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          if (j > 0 && j * 8 >= n) break;
#pragma unroll
          for (int i = 0; i < RT; ++i) {
            mma_bf16(acc[i][j], av[i][0].x, av[i][0].y, av[i][0].z, av[i][0].w, xv[j].x, xv[j].y);
            mma_bf16(acc[i][j], av[i][1].x, av[i][1].y, av[i][1].z, av[i][1].w, xv[j].z, xv[j].w);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      if (rt0 + i >= rts) break;
      __syncthreads();
      float* w = red + warp * 16 * LD;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        *reinterpret_cast<float2*>(w + g * LD + j * 8 + t4 * 2) = make_float2(acc[i][j][0], acc[i][j][1]);
        *reinterpret_cast<float2*>(w + (g + 8) * LD + j * 8 + t4 * 2) = make_float2(acc[i][j][2], acc[i][j][3]);
      }
      __syncthreads();
      for (int e = tid; e < 16 * NT * 8; e += LORA_THREADS) {
        const int r = e & 15, c = e >> 4;
        if (c >= n) break;
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < LORA_THREADS / 32; ++q) s += red[(q * 16 + r) * LD + c];
        p.v[(static_cast<long long>(blockIdx.y) * p.T + tl.y + c) * p.VR + (rt0 + i) * 16 + r] = scale * s;
      }
    }
  }
}

// ---- second product ---------------------------------------------------------------------------------------------------------------
// The rows of a tile's m16 block as the A operand, all rank tiles of a slice: PARTS parts of v, read from shared memory (fp32, rows of LDV).
template <int KS, int PARTS>
__device__ __forceinline__ void lora_rows(uint32_t (&f)[PARTS][KS][4], const float* v, int ldv, int g, int t4) {
#pragma unroll
  for (int k = 0; k < KS; ++k)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float2 w = *reinterpret_cast<const float2*>(v + (g + (q & 1) * 8) * ldv + k * 16 + t4 * 2 + (q >> 1) * 8);
      float h0, m0, l0, h1, m1, l1;
      bf16_parts(w.x, h0, m0, l0);
      bf16_parts(w.y, h1, m1, l1);
      f[0][k][q] = pack_cut(h0, h1);
      if constexpr (PARTS > 1) f[1][k][q] = pack_cut(m0, m1);
      if constexpr (PARTS > 2) f[2][k][q] = pack_cut(l0, l1);
    }
}
template <int KS, int PARTS>
__device__ __forceinline__ void lora_block(float (&d)[4][4], const uint32_t (&f)[PARTS][KS][4], const uint4* __restrict__ b) {
  uint4 w[KS][2];
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    w[k][0] = __ldg(b + k * 64);
    w[k][1] = __ldg(b + k * 64 + 32);
  }
#pragma unroll
  for (int k = 0; k < KS; ++k)
#pragma unroll
    for (int q = 0; q < PARTS; ++q) {
      mma_bf16(d[0], f[q][k][0], f[q][k][1], f[q][k][2], f[q][k][3], w[k][0].x, w[k][0].y);
      mma_bf16(d[1], f[q][k][0], f[q][k][1], f[q][k][2], f[q][k][3], w[k][0].z, w[k][0].w);
      mma_bf16(d[2], f[q][k][0], f[q][k][1], f[q][k][2], f[q][k][3], w[k][1].x, w[k][1].y);
      mma_bf16(d[3], f[q][k][0], f[q][k][1], f[q][k][2], f[q][k][3], w[k][1].z, w[k][1].w);
    }
}

enum LoraOut { LORA_F32 = 0, LORA_BF16 = 1, LORA_GLU = 2 };

// sums of the planes of v of a tile into shared memory; rows behind the tile's last as zeros
__device__ __forceinline__ void lora_sum_v(float* vs, int ldv, const LoraParams& p, const int4& tl, int m_tiles) {
  const int quads = p.VR >> 2;
  for (int e = threadIdx.x; e < m_tiles * 16 * quads; e += LORA_THREADS) {
    const int r = e / quads, q = e - r * quads;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < tl.z) {
      const float* src = p.v + (static_cast<long long>(tl.y) + r) * p.VR + q * 4;
      for (int z = 0; z < p.k_split; ++z) {
        const float4 w = *reinterpret_cast<const float4*>(src + static_cast<long long>(z) * p.T * p.VR);
        s.x += w.x; s.y += w.y; s.z += w.z; s.w += w.w;
      }
    }
    *reinterpret_cast<float4*>(vs + r * ldv + q * 4) = s;
  }
}

// Block: a tile x a range of column blocks (32 columns each).  The warps stand ceil(rows / 16) deep along the rows and divide the columns.
template <int KS, int OUT>
__global__ void __launch_bounds__(LORA_THREADS) lora_up_kernel(const LoraParams p) {
  constexpr int PARTS = OUT == LORA_F32 ? 3 : 2;
  extern __shared__ float vs[];             // [rows][VR + 4]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  // (the plan is older than the first product, whose results are all that has to be waited for)
  const int tile = blockIdx.x;
  const bool mine = tile < p.tiles[0].x;
  int4 tl = make_int4(-1, 0, 0, 0);
  if (mine) tl = p.tiles[1 + tile];
  const int ldv = p.VR + 4;
  pdl_sync();
  if (!mine) return;
  const int need = (tl.z + 15) >> 4, m_tiles = need == 3 ? 4 : need;
  const bool has = tl.x >= 0;
  if (has) {
    lora_sum_v(vs, ldv, p, tl, need);
    __syncthreads();
  }
  const int mt = warp & (m_tiles - 1), lanes_n = 8 / m_tiles, wn = warp / m_tiles;
  if (mt >= need) return;
  const int ra = mt * 16 + g, rb = ra + 8;
  const long long row_a = ra < tl.z ? p.order[tl.y + ra] : -1, row_b = rb < tl.z ? p.order[tl.y + rb] : -1;
  const int c0 = static_cast<int>(static_cast<long long>(p.blocks) * blockIdx.y / gridDim.y),
            c1 = static_cast<int>(static_cast<long long>(p.blocks) * (blockIdx.y + 1) / gridDim.y);
  const uint4* b = p.b + (has ? tl.x : 0) * p.b_slot + lane;
  if constexpr (OUT == LORA_GLU) {
    // the up columns' blocks follow the gate's
    uint32_t fg[PARTS][KS][4], fu[PARTS][KS][4];
    if (has) {
      lora_rows<KS, PARTS>(fg, vs + mt * 16 * ldv, ldv, g, t4);
      lora_rows<KS, PARTS>(fu, vs + mt * 16 * ldv + KS * 16, ldv, g, t4);
    }
    for (int c = c0 + wn; c < c1; c += lanes_n) {
      const int col = c * 32 + t4 * 8;
      float dg[4][4] = {}, du[4][4] = {};
      if (has) {
        lora_block<KS, PARTS>(dg, fg, b + static_cast<long long>(c) * KS * 64);
        lora_block<KS, PARTS>(du, fu, b + static_cast<long long>(p.blocks + c) * KS * 64);
      }
      if (col >= p.ff) continue;
      const int it = col / p.half, j = col - it * p.half;
      const long long at = static_cast<long long>(it) * 2 * p.half + (j >> 4) * 32 + (j & 15);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const long long row = h ? row_b : row_a;
        if (row < 0) continue;
        float gv[8], uv[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          gv[i] = dg[i >> 1][h * 2 + (i & 1)];
          uv[i] = du[i >> 1][h * 2 + (i & 1)];
        }
        for (int z = 0; z < p.splits; ++z) {
          const float* pl = p.planes + (static_cast<long long>(z) * p.T + row) * p.width + at;
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const float4 a4 = *reinterpret_cast<const float4*>(pl + q * 4), b4 = *reinterpret_cast<const float4*>(pl + 16 + q * 4);
            gv[q * 4] += a4.x; gv[q * 4 + 1] += a4.y; gv[q * 4 + 2] += a4.z; gv[q * 4 + 3] += a4.w;
            uv[q * 4] += b4.x; uv[q * 4 + 1] += b4.y; uv[q * 4 + 2] += b4.z; uv[q * 4 + 3] += b4.w;
          }
        }
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = gv[i] / (1.f + expf(-gv[i])) * uv[i];
        const uint4 o = make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out);
        const long long to = p.xt_rows ? static_cast<long long>(xt_index(static_cast<int>(row), col, p.xt_rows, p.xt_kb)) : row * p.ldo + col;
        *reinterpret_cast<uint4*>(out + to) = o;
      }
    }
  } else {
    uint32_t f[PARTS][KS][4];
    int slice = -1;
    for (int c = c0 + wn; c < c1; c += lanes_n) {
      int s = slice < 0 ? 0 : slice;
      while (c >= p.block0[s + 1]) ++s;
      if (s != slice) {
        slice = s;
        if (has) lora_rows<KS, PARTS>(f, vs + mt * 16 * ldv + s * KS * 16, ldv, g, t4);
      }
      const int col = p.col0[s] + (c - p.block0[s]) * 32 + t4 * 8;
      float d[4][4] = {};
      if (has) lora_block<KS, PARTS>(d, f, b + static_cast<long long>(c) * KS * 64);
      if (col >= p.col0[s + 1]) continue;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const long long row = h ? row_b : row_a;
        if (row < 0) continue;
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = d[i >> 1][h * 2 + (i & 1)];
        if constexpr (OUT == LORA_F32) {
          if (p.base) {
            const float* s4 = static_cast<const float*>(p.base) + row * p.ld_base + col;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const float4 w = *reinterpret_cast<const float4*>(s4 + q * 4);
              y[q * 4] += w.x; y[q * 4 + 1] += w.y; y[q * 4 + 2] += w.z; y[q * 4 + 3] += w.w;
            }
          }
          float* o = static_cast<float*>(p.out) + row * p.ldo + col;
          *reinterpret_cast<float4*>(o) = make_float4(y[0], y[1], y[2], y[3]);
          *reinterpret_cast<float4*>(o + 4) = make_float4(y[4], y[5], y[6], y[7]);
        } else {
          if (p.base) {
            const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.base) + row * p.ld_base + col);
            y[0] += bf16_lo(w.x); y[1] += bf16_hi(w.x); y[2] += bf16_lo(w.y); y[3] += bf16_hi(w.y);
            y[4] += bf16_lo(w.z); y[5] += bf16_hi(w.z); y[6] += bf16_lo(w.w); y[7] += bf16_hi(w.w);
          }
          *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + row * p.ldo + col) =
              make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
        }
      }
    }
  }
}

// how many tiles a step can have at most, and about how many it has (adapters of prompts are few)
static int lora_tile_rows(int T) { return T <= 64 ? 16 : 64; }
static int lora_max_tiles(int T, int slots) {
  const int tr = lora_tile_rows(T);
  return T / tr + (T < slots + 1 ? T : slots + 1);
}
static int lora_k_split(int T, int K, int slots) {
  const int tr = lora_tile_rows(T), units = (K + 63) / 64;
  const int tiles = T <= 64 ? (T < slots + 1 ? T : slots + 1) : (T + tr - 1) / tr;
  int split = (2 * 148 + tiles - 1) / tiles;                 // two blocks an SM
  const int most = units / 8 > 1 ? units / 8 : 1;            // a turn for each of the eight warps
  if (split > most) split = most;
  return split > 16 ? 16 : split;
}

template <int OUT>
static int lora_up_launch(const LoraParams& p, dim3 grid, size_t smem, void* stream) {
  switch (p.rank_tiles) {
    case 1: VB_CHECK_CUDA(max_dyn_smem_once(lora_up_kernel<1, OUT>)); VB_LAUNCH_PDL((lora_up_kernel<1, OUT>), grid, LORA_THREADS, smem, stream, p); break;
    case 2: VB_CHECK_CUDA(max_dyn_smem_once(lora_up_kernel<2, OUT>)); VB_LAUNCH_PDL((lora_up_kernel<2, OUT>), grid, LORA_THREADS, smem, stream, p); break;
    case 4: VB_CHECK_CUDA(max_dyn_smem_once(lora_up_kernel<4, OUT>)); VB_LAUNCH_PDL((lora_up_kernel<4, OUT>), grid, LORA_THREADS, smem, stream, p); break;
    default: VB_CHECK_CUDA(max_dyn_smem_once(lora_up_kernel<8, OUT>)); VB_LAUNCH_PDL((lora_up_kernel<8, OUT>), grid, LORA_THREADS, smem, stream, p); break;
  }
  return 0;
}

static int lora_down_launch(const LoraParams& p, int tile_rows, dim3 grid, void* stream) {
  if (tile_rows == 16) {
    const size_t smem = 8 * 16 * (2 * 8 + 4) * sizeof(float);
    VB_LAUNCH_PDL((lora_down_kernel<2, 2>), grid, LORA_THREADS, smem, stream, p);
  } else {
    const size_t smem = 8 * 16 * (8 * 8 + 4) * sizeof(float);
    VB_LAUNCH_PDL((lora_down_kernel<8, 2>), grid, LORA_THREADS, smem, stream, p);
  }
  return 0;
}

// checks and fills what both entry points share
static int lora_setup(const char* who, LoraParams& p, const void* d_x, long long ldx, const void* d_a, const void* d_b, const float* d_scale, int slots,
                      int rank, const int32_t* widths, int slices, const int32_t* d_order, const void* d_tiles, int T, int K, void* d_ws, size_t ws_bytes) {
  VB_CHECK_ARG(d_x && d_a && d_b && d_scale && d_order && d_tiles && widths && d_ws, "%s: null pointer", who);
  VB_CHECK_ARG(slots >= 1 && slots <= LORA_MAX_SLOTS, "%s: %d adapters; 1 to %d", who, slots, LORA_MAX_SLOTS);
  VB_CHECK_ARG(rank == 16 || rank == 32 || rank == 64 || rank == 128, "%s: padded rank %d must be 16, 32, 64 or 128", who, rank);
  VB_CHECK_ARG(slices >= 1 && slices <= LORA_MAX_SLICES, "%s: %d slices; 1 to %d", who, slices, LORA_MAX_SLICES);
  VB_CHECK_ARG(K >= 8 && K % 8 == 0 && ldx % 8 == 0 && ldx >= K && reinterpret_cast<uintptr_t>(d_x) % 16 == 0,
               "%s: rows of x must be multiples of 8 elements, 16-byte aligned (K %d, row stride %lld)", who, K, ldx);
  p.slices = slices;
  p.block0[0] = p.col0[0] = 0;
  for (int s = 0; s < slices; ++s) {
    VB_CHECK_ARG(widths[s] >= 8 && widths[s] % 8 == 0 && widths[s] <= (1 << 24), "%s: slice of %d columns; a multiple of 8", who, widths[s]);
    p.block0[s + 1] = p.block0[s] + (widths[s] + 31) / 32;
    p.col0[s + 1] = p.col0[s] + widths[s];
  }
  p.tiles = static_cast<const int4*>(d_tiles);
  p.order = d_order;
  p.x = static_cast<const __nv_bfloat16*>(d_x);
  p.ldx = ldx;
  p.a = static_cast<const uint4*>(d_a);
  p.b = static_cast<const uint4*>(d_b);
  p.scale = d_scale;
  p.T = T;
  p.K = K;
  p.kb32 = (K + 31) / 32;
  p.rank_tiles = rank / 16;
  p.VR = slices * rank;
  p.a_slot = static_cast<long long>(p.VR / 16) * p.kb32 * 64;
  p.b_slot = static_cast<long long>(p.block0[slices]) * p.rank_tiles * 64;
  p.blocks = p.block0[slices];
  p.k_split = lora_k_split(T, K, slots);
  p.v = static_cast<float*>(d_ws);
  const size_t need = static_cast<size_t>(p.k_split) * T * p.VR * sizeof(float);
  VB_CHECK_ARG(ws_bytes >= need && reinterpret_cast<uintptr_t>(d_ws) % 16 == 0, "%s: workspace of %zu bytes, 16-byte aligned, is needed (%zu given)", who, need,
               ws_bytes);
  return 0;
}

static dim3 lora_up_grid(const LoraParams& p, int slots) {
  const int tr = lora_tile_rows(p.T), tiles = p.T <= 64 ? (p.T < slots + 1 ? p.T : slots + 1) : (p.T + tr - 1) / tr;
  int split = (4 * 148 + tiles - 1) / tiles;                // four blocks an SM, at least a column block for every warp
  const int most = (p.blocks + 7) / 8;
  if (split > most) split = most;
  return dim3(lora_max_tiles(p.T, slots), split < 1 ? 1 : split);
}

}  // namespace vb

using namespace vb;

extern "C" {

int vb_lora_max_tiles(int T, int slots) { return T < 1 || slots < 1 ? 0 : lora_max_tiles(T, slots); }

int vb_lora_plan(int32_t* d_order, void* d_tiles, const int32_t* d_ids, int T, int slots, void* stream) {
  VB_CHECK_ARG(d_order && d_tiles && d_ids, "vb_lora_plan: null pointer");
  VB_CHECK_ARG(slots >= 1 && slots <= LORA_MAX_SLOTS, "vb_lora_plan: %d adapters; 1 to %d", slots, LORA_MAX_SLOTS);
  VB_CHECK_ARG(T >= 1, "vb_lora_plan: no rows");
  VB_LAUNCH_PDL(lora_plan_kernel, 1, 1024, 0, stream, d_order, static_cast<int4*>(d_tiles), d_ids, T, slots, lora_tile_rows(T));
  return 0;
}

size_t vb_lora_workspace_bytes(int T, int K, int slots, int rank, int slices) {
  if (T < 1 || K < 1 || slots < 1) return 0;
  return static_cast<size_t>(lora_k_split(T, K, slots)) * T * slices * rank * sizeof(float);
}

int vb_lora(void* d_out, long long ld_out, const void* d_base, long long ld_base, int out_f32, const void* d_x, long long ldx, const void* d_a, const void* d_b,
            const float* d_scale, int slots, int rank, const int32_t* widths, int slices, const int32_t* d_order, const void* d_tiles, int T, int K, void* d_ws,
            size_t ws_bytes, void* stream) {
  VB_CHECK_ARG(d_out, "vb_lora: null pointer");
  if (T <= 0) return 0;
  LoraParams p = {};
  const int rc = lora_setup("vb_lora", p, d_x, ldx, d_a, d_b, d_scale, slots, rank, widths, slices, d_order, d_tiles, T, K, d_ws, ws_bytes);
  if (rc) return rc;
  const int unit = out_f32 ? 4 : 8;
  VB_CHECK_ARG(ld_out % unit == 0 && ld_out >= p.col0[slices] && reinterpret_cast<uintptr_t>(d_out) % 16 == 0 &&
                   (!d_base || (ld_base % unit == 0 && ld_base >= p.col0[slices] && reinterpret_cast<uintptr_t>(d_base) % 16 == 0)),
               "vb_lora: rows of out and base must be 16-byte aligned and at least %d columns apart", p.col0[slices]);
  p.out = d_out;
  p.ldo = ld_out;
  p.base = d_base;
  p.ld_base = ld_base;
  const int tr = lora_tile_rows(T);
  const int rc1 = lora_down_launch(p, tr, dim3(lora_max_tiles(T, slots), p.k_split), stream);
  if (rc1) return rc1;
  const size_t smem = static_cast<size_t>(tr) * (p.VR + 4) * sizeof(float);
  return out_f32 ? lora_up_launch<LORA_F32>(p, lora_up_grid(p, slots), smem, stream) : lora_up_launch<LORA_BF16>(p, lora_up_grid(p, slots), smem, stream);
}

int vb_lora_gate_up(void* d_act, long long ld_act, int xt_rows, const float* d_planes, int splits, int half, int ff, const void* d_x, long long ldx,
                    const void* d_a, const void* d_b, const float* d_scale, int slots, int rank, const int32_t* d_order, const void* d_tiles, int T, int K,
                    void* d_ws, size_t ws_bytes, void* stream) {
  VB_CHECK_ARG(d_act && d_planes, "vb_lora_gate_up: null pointer");
  VB_CHECK_ARG(splits >= 1 && half >= 16 && half % 16 == 0 && half <= 64, "vb_lora_gate_up: %d planes, tiles of %d gate rows (16, 32, 48 or 64)", splits, half);
  if (T <= 0) return 0;
  LoraParams p = {};
  const int32_t widths[2] = {ff, ff};
  const int rc = lora_setup("vb_lora_gate_up", p, d_x, ldx, d_a, d_b, d_scale, slots, rank, widths, 2, d_order, d_tiles, T, K, d_ws, ws_bytes);
  if (rc) return rc;
  VB_CHECK_ARG(xt_rows >= 0 && reinterpret_cast<uintptr_t>(d_act) % 16 == 0 && reinterpret_cast<uintptr_t>(d_planes) % 16 == 0 &&
                   (xt_rows > 0 || (ld_act % 8 == 0 && ld_act >= ff)),
               "vb_lora_gate_up: rows of act must be 16-byte aligned and at least %d columns apart", ff);
  p.out = d_act;
  p.ldo = ld_act;
  p.planes = d_planes;
  p.splits = splits;
  p.half = half;
  p.ff = ff;
  p.width = (ff + half - 1) / half * 2 * half;
  p.xt_rows = xt_rows;
  p.xt_kb = (ff + 63) / 64;
  const int tr = lora_tile_rows(T);
  const int rc1 = lora_down_launch(p, tr, dim3(lora_max_tiles(T, slots), p.k_split), stream);
  if (rc1) return rc1;
  p.blocks = p.block0[1];              // column blocks of one of the two
  const size_t smem = static_cast<size_t>(tr) * (p.VR + 4) * sizeof(float);
  return lora_up_launch<LORA_GLU>(p, lora_up_grid(p, slots), smem, stream);
}

}  // extern "C"
