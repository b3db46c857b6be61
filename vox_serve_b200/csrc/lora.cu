// Low-rank adapters of many requests beside a shared projection.
//
//   v[t, s r + j] = scale_a sum_k A_a[s, j, k] x[t, k]            (a: the adapter of row t; s: slice of the projection's columns, q | k | v)
//   out[t, n] = base[t, n] + sum_j B_a[n, j] v[t, s(n) r + j]
//
//   vb_lora_plan      rows of a step by adapter: a table of row tiles, and of groups of them, that every projection of every layer works through
//   vb_lora           out as fp32 (one more split-K plane of the projection: its consumer sums planes anyway) or as bf16 rows with a base
//   vb_lora_gate_up   silu(gate) * up from the projection's fp32 planes with both adapters' products added
//
// A tile is up to 16 rows (steps of at most 64) or 64 rows of one adapter, a group up to 128.  The bank keeps A as swizzled tiles of 16 ranks x 64 k, which the
// tensor cores take as they are and lanes of mma.sync by 16-byte pieces, and B in the order in which lanes take it (512 bytes in a row per warp).  Three kernels:
//
//   few   steps of at most 64 rows whose adapters are small: one launch.  A cluster of eight blocks per tile divides K, adds up v through distributed
//         shared memory and divides the columns
//   down  v of any step: a group x a piece of K a block (tcgen05), the blocks of a group a cluster that adds up its parts
//   up    a tile x some columns a block (mma.sync: as many products as loads), all that it reads but v on its way before v is there
//
// Sums are fp32.  v is not rounded on its way into the second product: it enters as three bf16 parts (exact, rowmma.cuh).  But for large steps whose result is
// rounded to bf16 anyway, by up to 2^-8 of itself: two parts there (rounded to nearest, off by 2^-17 of v at most).  A third of the second product's reads and
// products less: 4096 rows of 2048 columns at rank 64 32.0 us a call instead of 36.2, gate | up of 1000 rows of 8192 at rank 32 25.5 instead of 28.7; in
// steps of at most 64 rows the third part costs nothing that can be measured (17 rows of gate | up 5.5 us with it and without).
#include "../../include/vb_api.h"
#define VB_PDL_FAMILY 4
#include "rowmma.cuh"

namespace vb {

constexpr int LORA_MAX_SLOTS = 1023;       // (a thread of the planning block each, and one for rows without an adapter)
constexpr int LORA_MAX_SLICES = 4;
constexpr int LORA_MAX_ROWS = 1 << 21;     // (tiles are a launch's second dimension)
constexpr int LORA_THREADS = 256;
constexpr int LORA_DOWN_ROWS = 128;        // rows of a block of the first product
constexpr int LORA_PLAN_HEAD = 4;          // words in front of the tiles
constexpr int LORA_PLAN_SMEM = 32 * (LORA_MAX_SLOTS + 1) * 4;

// ---- rows by adapter ------------------------------------------------------------------------------------------------------------
// Four words, rows and slots of the step in the first two (a call of another step does not read on), then a record per tile: adapter or -1, first place among the sorted rows, rows (0: no tile), 0, then the rows.  Behind them a record per group, the up to 128 rows of an
// adapter (neighbouring tiles) that a block of the first product takes: first tile (-1: no group), adapter, rows, the first row if they follow one another in x,
// else -1.  One block: a counting sort in shared memory
// that keeps an adapter's rows in their order (rows that follow one another in x are then fetched as boxes): a warp a piece of the rows, its counts per adapter [32 warps]
// [slots + 1], which become the first places of the warps' rows.  Two passes over the ids; then a thread writes an adapter's records.  Once a step, in a chain of
// captured calls: 3.5 us for 32 rows, 5.9 for 4096 of six adapters, 9.3 for 4096 of one, 29 for 16384 and 155 for 65536 of one (its thread's records: 2 us per 1024 rows).
__global__ void __launch_bounds__(1024) lora_plan_kernel(int32_t* __restrict__ tiles, const int32_t* __restrict__ ids, int T, int slots, int tile_rows, int max_tiles,
                                                         int max_groups) {
  extern __shared__ __align__(128) int cnt[];
  __shared__ int first_tile[1024];
  __shared__ int warp_rows[32], warp_tiles[32], warp_groups[32];
  pdl_sync();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, stride = 4 + tile_rows, counts = slots + 1;
  for (int i = tid; i < 32 * counts; i += 1024) cnt[i] = 0;
  if (tid == 0) *reinterpret_cast<int4*>(tiles - LORA_PLAN_HEAD) = make_int4(T, slots, 0, 0);
  __syncthreads();
  const int per = (T + 1023) / 1024 * 32, end = min(T, (warp + 1) * per);
  int* mine = cnt + warp * counts;
  for (int t0 = warp * per; t0 < end; t0 += 32) {
    const int t = t0 + lane;
    int a = t < end ? ids[t] : -1;
    a = a >= 0 && a < slots ? a : slots;
    const uint32_t same = __match_any_sync(0xffffffffu, t < end ? a : -1 - lane);
    if (t < end && (same & ((1u << lane) - 1u)) == 0u) mine[a] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  int rows = 0;
  if (tid <= slots)
    for (int w = 0; w < 32; ++w) {
      const int c = cnt[w * counts + tid];
      cnt[w * counts + tid] = rows;
      rows += c;
    }
  const int n = (rows + tile_rows - 1) / tile_rows;
  const int groups = tid < slots ? (rows + LORA_DOWN_ROWS - 1) / LORA_DOWN_ROWS : 0;
  int r = rows, m = n, q = groups;          // inclusive sums over the threads
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int rr = __shfl_up_sync(0xffffffffu, r, o), mm = __shfl_up_sync(0xffffffffu, m, o), qq = __shfl_up_sync(0xffffffffu, q, o);
    if (lane >= o) { r += rr; m += mm; q += qq; }
  }
  if (lane == 31) { warp_rows[warp] = r; warp_tiles[warp] = m; warp_groups[warp] = q; }
  __syncthreads();
  if (warp == 0) {
    int a = warp_rows[lane], b = warp_tiles[lane], c = warp_groups[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int aa = __shfl_up_sync(0xffffffffu, a, o), bb = __shfl_up_sync(0xffffffffu, b, o), cc = __shfl_up_sync(0xffffffffu, c, o);
      if (lane >= o) { a += aa; b += bb; c += cc; }
    }
    warp_rows[lane] = a;
    warp_tiles[lane] = b;
    warp_groups[lane] = c;
  }
  __syncthreads();
  if (warp > 0) { r += warp_rows[warp - 1]; m += warp_tiles[warp - 1]; q += warp_groups[warp - 1]; }
  const int row0 = r - rows, tile0 = m - n, all = warp_tiles[31], all_groups = warp_groups[31];
  int4* group = reinterpret_cast<int4*>(tiles + static_cast<long long>(max_tiles) * stride);
  first_tile[tid] = tile0;
  for (int i = 0; i < n; ++i)
    *reinterpret_cast<int4*>(tiles + static_cast<long long>(tile0 + i) * stride) = make_int4(tid < slots ? tid : -1, row0 + i * tile_rows, min(tile_rows, rows - i * tile_rows), 0);
  for (int i = all + tid; i < max_tiles; i += 1024) *reinterpret_cast<int4*>(tiles + static_cast<long long>(i) * stride) = make_int4(-1, 0, 0, 0);
  for (int i = all_groups + tid; i < max_groups; i += 1024) group[i] = make_int4(-1, 0, 0, 0);
  __syncthreads();
  for (int t0 = warp * per; t0 < end; t0 += 32) {
    const int t = t0 + lane;
    int a = t < end ? ids[t] : -1;
    a = a >= 0 && a < slots ? a : slots;
    const uint32_t same = __match_any_sync(0xffffffffu, t < end ? a : -1 - lane), below = same & ((1u << lane) - 1u);
    if (t < end) {
      const int at = mine[a] + __popc(below), i = at / tile_rows;
      tiles[static_cast<long long>(first_tile[a] + i) * stride + 4 + at - i * tile_rows] = t;
    }
    __syncwarp();
    if (t < end && below == 0u) mine[a] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  for (int i = 0; i < groups; ++i) {
    const int first = i * LORA_DOWN_ROWS, last = min(rows, first + LORA_DOWN_ROWS) - 1;
    auto row = [&](int k) { return tiles[static_cast<long long>(tile0 + k / tile_rows) * stride + 4 + k % tile_rows]; };
    const int a = row(first);
    group[q - groups + i] = make_int4(tile0 + first / tile_rows, tid, last - first + 1, row(last) - a == last - first ? a : -1);
  }
}

struct LoraParams {
  const int32_t* tiles;            // records of 4 + tile_rows words; in front of them (LORA_PLAN_HEAD) the step's rows and slots
  unsigned char* plan_flag;
  int slots;
  const int4* groups;
  int tile_rows;
  const __nv_bfloat16* x;
  long long ldx;
  const uint4 *a, *b;              // [slots][K / 64][S][rank / 16][16 ranks][128 B, swizzled], [slots][column blocks of 32][rank / 16][2][32 lanes]
  long long a_slot, b_slot;        // 16-byte units
  const float* scale;
  uint32_t* v;                     // [tiles][tile_rows / 16][S][parts][rank / 16][32 lanes][4]: v as the second product takes it
  int T, K, rank_tiles, VR, k_split, parts;      // VR = S * rank
  bool f32;                        // the result is fp32
  unsigned char* wait_flag;
  // second product
  int blocks;                      // column blocks of 32 over all slices (of gate | up: of one)
  int ahead;                       // 1: a step's copies go out a step ahead
  int slices, block0[LORA_MAX_SLICES + 1], col0[LORA_MAX_SLICES + 1];
  int part0[LORA_MAX_SLICES + 1];  // the blocks of a tile by slice
  void* out;
  const void* base;
  long long ldo, ld_base;
  // gate | up
  const float* planes;
  int splits, width, ff, xt_rows, xt_kb;
};

// What a plan was made for.  A captured call may meet one of another step, whose records it would take for rows and adapters: it raises a flag that the host reads and
// writes nothing.
__device__ __forceinline__ int2 lora_plan_of(const LoraParams& p) { return *reinterpret_cast<const int2*>(p.tiles - LORA_PLAN_HEAD); }
__device__ __forceinline__ bool lora_other_plan(const LoraParams& p, const int2& made) {
  if (made.x == p.T && made.y == p.slots) return false;
  if (threadIdx.x == 0) {
    *reinterpret_cast<volatile unsigned char*>(p.plan_flag) = 1;
    __threadfence_system();
  }
  return true;
}

// ---- v as the second product's A operand ------------------------------------------------------------------------------------------
// In the order of the lanes: [m16 block][slice][part][rank tile][32 lanes][4 registers].
__device__ __forceinline__ void lora_put(uint32_t* frags, int slices, int parts, int log_ks, int r, int k, float a, float b) {      // row r, v[k] and v[k + 1]
  const int tile = k >> 4, s = tile >> log_ks, ks = 1 << log_ks, t = tile & (ks - 1);
  uint32_t* at = frags + ((((r >> 4) * slices + s) * parts * ks + t) * 32 + (r & 7) * 4 + (k & 7) / 2) * 4 + (r & 15) / 8 + (k & 15) / 8 * 2;
  if (parts > 2) {
    float h0, m0, l0, h1, m1, l1;
    bf16_parts(a, h0, m0, l0);
    bf16_parts(b, h1, m1, l1);
    at[0] = pack_cut(h0, h1);
    at[ks * 128] = pack_cut(m0, m1);
    at[2 * ks * 128] = pack_cut(l0, l1);
  } else {
    float h0, m0, h1, m1;
    bf16_near(a, h0, m0);
    bf16_near(b, h1, m1);
    at[0] = pack_cut(h0, h1);
    at[ks * 128] = pack_bf16(m0, m1);
  }
}

// 16 bytes past the registers and L1; zeros where `bytes` is 0 instead of 16 (nothing is read then)
__device__ __forceinline__ void cp_async16(uint32_t to, const void* from, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// ---- first product: v = scale A x -------------------------------------------------------------------------------------------------
// Block: a group of up to 128 rows of an adapter x a piece of K, in stages of 64 k on the tensor cores (tcgen05): D[row][rank] += x[row][k] A[rank][k].  A lies in the
// bank as the tensor cores read it, one bulk copy a stage; rows that follow one another in x come as boxes of a tensor map, others by 16-byte copies of four
// warps (some 16 clocks an instruction of 512 bytes: that rate bounded a form with copies alone, at 38 us for 4096 rows of 8192 at rank 64 and the second
// product; mma.sync from such copies was bound by its shared-memory reads: 36 us, 69 at rank 128; this form takes 34 and 48).  A fifth warp multiplies.  Rows behind
// the last are whatever stands there, in lanes that nobody reads.  Stages go to ACCS sums in turn: the tensor cores cut a sum off at every step, and chains of a
// quarter lose a quarter (lora_long: when they are more than four or two).  More than RT rank tiles: further blocks with x again.  The pieces of K are a cluster, which adds them
// up and leaves v in parts.
constexpr int LORA_STAGE_K = 64, LORA_X_BYTES = LORA_DOWN_ROWS * 128, LORA_DOWN_THREADS = 160, LORA_LOADERS = 128, LORA_BOX_ROWS = 64;
template <int RT>
struct LoraDown {
  static constexpr int N = RT * 16, ACCS = RT == 8 ? 2 : 4, MOST_ACCS = 256 / N, STAGES = RT == 8 ? 3 : RT == 4 ? 4 : 5;      // (256 columns of tensor memory a block: two run on an SM)
  static constexpr int STAGE_BYTES = LORA_X_BYTES + RT * 2048, LD = N + 4;
  static constexpr size_t SMEM = 1024 + static_cast<size_t>(STAGES) * STAGE_BYTES + 256;       // (1 KB to align; barriers)
  static_assert(LORA_DOWN_ROWS * LD * 4 <= STAGES * STAGE_BYTES, "the sums stand where the stages stood");
};
template <int RT, int ACCS>
__global__ void __launch_bounds__(LORA_DOWN_THREADS, 2) lora_down_kernel(const LoraParams p, const __grid_constant__ CUtensorMap x_map) {
  extern __shared__ __align__(128) uint8_t smem8[];
  using D = LoraDown<RT>;
  constexpr int STAGES = D::STAGES, LD = D::LD, AHEAD = STAGES > 3 ? STAGES - 2 : 2;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* base = smem8 + ((1024u - (smem_u32(smem8) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(base + STAGES * D::STAGE_BYTES);
  uint64_t *empty = full + STAGES, *done = empty + STAGES;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(done + 1);
  pdl_sync();
  const int2 made = lora_plan_of(p);
  const int4 gr = p.groups[blockIdx.y];
  if (lora_other_plan(p, made) || gr.x < 0) return;        // (all blocks of the cluster)
  const int n = gr.z, rts = p.VR >> 4;
  const bool boxes = gr.w >= 0;
  if (warp == 4) {
    tmem_alloc(tmem_at, ACCS * D::N);
    tmem_relinquish();
  }
  // (the blocks of a group take stages in turn, so that at any time they read neighbouring pieces of the rows)
  const int s1 = (p.K + LORA_STAGE_K - 1) / LORA_STAGE_K, s0 = blockIdx.x, hop = p.k_split, turns = (s1 - s0 + hop - 1) / hop;
  const float scale = p.scale[gr.y];
  // a thread's copies: 16 bytes of eight rows.  k behind K is filled with zeros; rows behind the last hold anything.
  const int chunk = tid & 7, row0 = (tid >> 3) & 15, n_boxes = (n + LORA_BOX_ROWS - 1) / LORA_BOX_ROWS;
  int xr[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {             // (all tiles of a group but the last are full)
    const int r = row0 + i * 16;
    xr[i] = !boxes && r < n ? p.tiles[static_cast<long long>(gr.x + r / p.tile_rows) * (4 + p.tile_rows) + 4 + r % p.tile_rows] : -1;
  }
  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(full + i, boxes ? 1 : 1 + LORA_LOADERS / 32);
      mbar_init(empty + i, 1);
    }
    mbar_init(done, 1);
    fence_barrier_init();
  }
  const __nv_bfloat16* xs = p.x + chunk * 8;
  const uint32_t ring = smem_u32(base), x_to = ring + row0 * 128 + ((chunk ^ (row0 & 7)) << 4);
  BoundedWait bw{p.wait_flag};
  __syncthreads();                          // (barriers and TMEM are there)
  tc_fence_after();
  const uint32_t tmem = *tmem_at;
  int slot = 0;
  uint32_t parity = 0u;
  auto next = [&]() {
    slot = slot + 1 == STAGES ? 0 : slot + 1;
    parity ^= slot == 0 ? 1u : 0u;
  };
  const int rt0 = blockIdx.z * RT, here = min(RT, rts - rt0);
  // (one lane) A of a stage, all its rank tiles in a row, and how many bytes the stage waits for
  auto ask = [&](int s, uint32_t x_bytes) {
    mbar_arrive_expect_tx(full + slot, here * 2048 + x_bytes);
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(ring + slot * D::STAGE_BYTES + LORA_X_BYTES),
                 "l"(p.a + gr.y * p.a_slot + (static_cast<long long>(s) * rts + rt0) * 128), "r"(here * 2048), "r"(smem_u32(full + slot))
                 : "memory");
  };
  if (boxes && warp == 0) {
    for (int i = 0; i < turns; ++i) {
      bw.wait(empty + slot, parity ^ 1u);
      if (!__all_sync(0xffffffffu, !bw.dead)) bw.dead = true;
      if (bw.dead) break;
      const int s = s0 + i * hop;
      if (lane == 0) {
        ask(s, n_boxes * LORA_BOX_ROWS * 128);
        for (int b = 0; b < n_boxes; ++b)
          tma_load_2d(base + slot * D::STAGE_BYTES + b * LORA_BOX_ROWS * 128, &x_map, full + slot, s * LORA_STAGE_K, gr.w + b * LORA_BOX_ROWS);
      }
      __syncwarp();
      next();
    }
  } else if (!boxes && warp < 4) {
    int told = slot;                      // the oldest stage that the multiplying warp has not been told of
    for (int i = 0; i < turns + AHEAD; ++i) {
      if (i < turns && !bw.dead) {
        const int s = s0 + i * hop;
        bw.wait(empty + slot, parity ^ 1u);
        if (!__all_sync(0xffffffffu, !bw.dead)) bw.dead = true;
        if (!bw.dead) {
          if (tid == 0) ask(s, 0u);
          const uint32_t to = slot * D::STAGE_BYTES;
          const bool in = s * LORA_STAGE_K + chunk * 8 < p.K;
          const __nv_bfloat16* x = xs + (in ? static_cast<long long>(s) * LORA_STAGE_K : 0);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (xr[j] >= 0) cp_async16(x_to + to + j * 2048, x + xr[j] * p.ldx, in ? 16 : 0);
        }
        next();
      }
      cp_async_commit();
      if (i >= AHEAD) {
        cp_async_wait<AHEAD>();
        fence_proxy_async();              // (what the copies wrote, for the tensor cores' reads)
        __syncwarp();
        if (lane == 0 && !bw.dead) mbar_arrive(full + told);
        told = told + 1 == STAGES ? 0 : told + 1;
      }
    }
  } else if (warp == 4) {
    const uint32_t idesc = umma_idesc(128, here * 16, 1u);
    for (int i = 0; i < turns; ++i) {
      bw.wait(full + slot, parity);
      if (!__all_sync(0xffffffffu, !bw.dead)) bw.dead = true;
      if (bw.dead) break;
      tc_fence_after();
      const uint64_t x_desc = umma_desc_sw128_kmajor(ring + slot * D::STAGE_BYTES), a_desc = umma_desc_sw128_kmajor(ring + slot * D::STAGE_BYTES + LORA_X_BYTES);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_bf16(tmem + i % ACCS * D::N, x_desc + 2 * k, a_desc + 2 * k, idesc, i >= ACCS || k > 0);
        umma_commit(empty + slot);
        if (i + 1 == turns) umma_commit(done);
      }
      __syncwarp();
      next();
    }
  }
  // the products are through: rows of sums where the stages stood
  float* mine = reinterpret_cast<float*>(base);                  // [128 rows][LD]
  bw.wait(done, 0);
  tc_fence_after();
  if (warp * 32 < n && warp < 4) {
#pragma unroll 1
    for (int c0 = 0; c0 < here * 16; c0 += 16) {
      float s[16];
#pragma unroll
      for (int q = 0; q < ACCS; ++q) {
        if (q > 0 && q >= turns) break;
        uint32_t v[16];
        tmem_ld_32x16(tmem + (static_cast<uint32_t>(warp * 32) << 16) + q * D::N + c0, v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = q == 0 ? __uint_as_float(v[j]) : s[j] + __uint_as_float(v[j]);
      }
      float4* to = reinterpret_cast<float4*>(mine + (warp * 32 + lane) * LD + c0);
#pragma unroll
      for (int j = 0; j < 4; ++j) to[j] = make_float4(scale * s[4 * j], scale * s[4 * j + 1], scale * s[4 * j + 2], scale * s[4 * j + 3]);
    }
  }
  // Tensor memory goes back before the block waits for another: a block of another stream's cluster may wait for it on this SM while its neighbour holds what this cluster's
  // other blocks wait for.
  tc_fence_before();
  if (bw.dead) {                            // (copies and products in flight land first)
    const unsigned long long t0 = gtimer();
    while (gtimer() - t0 < 2000000ull) __nanosleep(1000);
  }
  __syncwarp();
  if (warp < 4) {
    asm volatile("barrier.cta.arrive 1, %0;" ::"n"(LORA_DOWN_THREADS) : "memory");
  } else {
    asm volatile("barrier.cta.sync 1, %0;" ::"n"(LORA_DOWN_THREADS) : "memory");
    tc_fence_after();
  }
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");       // (a cluster of one block meets itself)
  if (warp == 4) tmem_dealloc(tmem, ACCS * D::N);
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  const int log_ks = 31 - __clz(p.rank_tiles);
  uint32_t* v = p.v + static_cast<long long>(gr.x) * (p.tile_rows >> 4) * rts * p.parts * 128;
  for (int e = blockIdx.x * LORA_DOWN_THREADS + tid; e < n * RT * 4; e += p.k_split * LORA_DOWN_THREADS) {
    const int c = e / (RT * 4), k = e % (RT * 4) * 4;
    if (rt0 * 16 + k >= p.VR) continue;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (p.k_split > 1) {
#pragma unroll 4
      for (int z = 0; z < p.k_split; ++z) {
        const float4 w = ld_dsmem_f32x4(mine + c * LD + k, z);
        s.x += w.x; s.y += w.y; s.z += w.z; s.w += w.w;
      }
    } else {
      s = *reinterpret_cast<const float4*>(mine + c * LD + k);
    }
    lora_put(v, p.slices, p.parts, log_ks, c, rt0 * 16 + k, s.x, s.y);
    lora_put(v, p.slices, p.parts, log_ks, c, rt0 * 16 + k + 2, s.z, s.w);
  }
  if (p.k_split > 1) cluster_sync_all();                         // (others' parts have been read: the block may leave)
}

// ---- second product ---------------------------------------------------------------------------------------------------------------
template <int KS, int PARTS>
__device__ __forceinline__ void lora_block(float (&d)[4][4], const uint4* frags, const uint4 (&w)[KS][2]) {
#pragma unroll
  for (int q = PARTS - 1; q >= 0; --q)               // (the smallest parts first)
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const uint4 f = frags[(q * KS + k) * 32];
      mma_bf16(d[0], f.x, f.y, f.z, f.w, w[k][0].x, w[k][0].y);
      mma_bf16(d[1], f.x, f.y, f.z, f.w, w[k][0].z, w[k][0].w);
      mma_bf16(d[2], f.x, f.y, f.z, f.w, w[k][1].x, w[k][1].y);
      mma_bf16(d[3], f.x, f.y, f.z, f.w, w[k][1].z, w[k][1].w);
    }
}
// a column block's part of B from the bank
template <int KS>
__device__ __forceinline__ void lora_take(uint4 (&w)[KS][2], const uint4* b) {
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    w[k][0] = __ldg(b + k * 64);
    w[k][1] = __ldg(b + k * 64 + 32);
  }
}
// ... both operands from shared memory, NB neighbouring column blocks
template <int KS, int PARTS, int NB>
__device__ __forceinline__ void lora_product(float (*d)[4][4], uint32_t frags, uint32_t b) {
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    uint4 w[NB][2];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      w[i][0] = lds16(b + (i * KS + k) * 1024);
      w[i][1] = lds16(b + (i * KS + k) * 1024 + 512);
    }
#pragma unroll
    for (int q = PARTS - 1; q >= 0; --q) {
      const uint4 f = lds16(frags + (q * KS + k) * 512);
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        mma_bf16(d[i][0], f.x, f.y, f.z, f.w, w[i][0].x, w[i][0].y);
        mma_bf16(d[i][1], f.x, f.y, f.z, f.w, w[i][0].z, w[i][0].w);
        mma_bf16(d[i][2], f.x, f.y, f.z, f.w, w[i][1].x, w[i][1].y);
        mma_bf16(d[i][3], f.x, f.y, f.z, f.w, w[i][1].z, w[i][1].w);
      }
    }
  }
}

enum LoraOut { LORA_F32 = 0, LORA_BF16 = 1, LORA_GLU = 2 };
__device__ __forceinline__ void lora_add4(float* y, const float4& w) { y[0] += w.x; y[1] += w.y; y[2] += w.z; y[3] += w.w; }
__device__ __forceinline__ void lora_add8(float* y, const uint4& w) {
  y[0] += bf16_lo(w.x); y[1] += bf16_hi(w.x); y[2] += bf16_lo(w.y); y[3] += bf16_hi(w.y);
  y[4] += bf16_lo(w.z); y[5] += bf16_hi(w.z); y[6] += bf16_lo(w.w); y[7] += bf16_hi(w.w);
}
__device__ __forceinline__ uint4 lora_round(const float* y) {
  return make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
}

// Results of a lane: eight neighbouring columns.  y: the products; base: what is added (nullptr: nothing).
template <int OUT>
__device__ __forceinline__ void lora_result(void* out, float (&y)[8], const void* base) {
  if constexpr (OUT == LORA_F32) {
    if (base) {
      lora_add4(y, static_cast<const float4*>(base)[0]);
      lora_add4(y + 4, static_cast<const float4*>(base)[1]);
    }
    if ((reinterpret_cast<uintptr_t>(out) & 31) == 0) {
      asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(out), "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7])
                   : "memory");
    } else {
      static_cast<float4*>(out)[0] = make_float4(y[0], y[1], y[2], y[3]);
      static_cast<float4*>(out)[1] = make_float4(y[4], y[5], y[6], y[7]);
    }
  } else {
    if (base) lora_add8(y, *static_cast<const uint4*>(base));
    *static_cast<uint4*>(out) = lora_round(y);
  }
}
// g / (1 + exp(-g)) by the special function unit without its ranges below 2^-126 (1000 rows of gate | up: 26.3 us with the ranges, 25.8 without).  The power of
// two is off by 2^-22, its argument's rounding by 1.2 |g| units of 2^-24, the reciprocal by 2^-23: far below half a step of bf16, 2^-8.  Below g = -87 the reciprocal is 0 (the
// value 1e-36 at most).
__device__ __forceinline__ float lora_silu(float g) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return g * r;
}
// ... of gate | up: g0, g1, u0, u1 are the first plane's eight gate and eight up columns
__device__ __forceinline__ void lora_gated(const LoraParams& p, void* out, long long row, int col, float (&gv)[8], float (&uv)[8], const float4& g0, const float4& g1,
                                           const float4& u0, const float4& u1) {
  lora_add4(gv, g0);
  lora_add4(gv + 4, g1);
  lora_add4(uv, u0);
  lora_add4(uv + 4, u1);
  if (p.splits > 1)
#pragma unroll 1
    for (int z = 1; z < p.splits; ++z) {
      const float* more = p.planes + (static_cast<long long>(z) * p.T + row) * p.width + (col >> 4) * 32 + (col & 15);
      lora_add4(gv, *reinterpret_cast<const float4*>(more));
      lora_add4(gv + 4, *reinterpret_cast<const float4*>(more + 4));
      lora_add4(uv, *reinterpret_cast<const float4*>(more + 16));
      lora_add4(uv + 4, *reinterpret_cast<const float4*>(more + 20));
    }
#pragma unroll
  for (int i = 0; i < 8; ++i) gv[i] = lora_silu(gv[i]) * uv[i];
  *static_cast<uint4*>(out) = lora_round(gv);
}
// where column `col` of a row's results stands
template <int OUT>
__device__ __forceinline__ void* lora_place(const LoraParams& p, long long row, int col) {
  if constexpr (OUT == LORA_F32) return static_cast<float*>(p.out) + row * p.ldo + col;
  if (OUT == LORA_GLU && p.xt_rows) return static_cast<__nv_bfloat16*>(p.out) + xt_index(static_cast<int>(row), col, p.xt_rows, p.xt_kb);
  return static_cast<__nv_bfloat16*>(p.out) + row * p.ldo + col;
}
// bf16 parts of v; TALL: tiles of 64 rows
template <int OUT, bool TALL>
__host__ __device__ constexpr int lora_parts() { return OUT == LORA_F32 || !TALL ? 3 : 2; }

// Block: a tile x a range of column blocks, four warps, in steps: tiles of 64 rows, a warp per 16 rows, all warps the same one or two column blocks (so that of base and
// results 128 bytes of a row at least move together); tiles of 16 rows, a warp per column block.  What a step reads, its part of B and the rows' part of base or
// planes, is copied a step ahead; v is read once.  All but v is older than the first product, so the first steps' copies are on their way when that ends.  What bounds it are its
// own instructions' latencies (16 warps an SM, 40 % of the issue slots): 4096 rows of 2048 columns at rank 64 in bf16 10 us for 34 MB, gate | up of 1000 rows of 2 x 8192 columns
// 15 for 82 MB.  (Two steps ahead in half as many blocks: 38 us instead of 27 for the latter's whole call.)
constexpr int LORA_UP_THREADS = 128;
template <int OUT>
__host__ __device__ constexpr int lora_row_bytes() { return OUT == LORA_GLU ? 256 : OUT == LORA_F32 ? 128 : 64; }      // of a column block in base or planes
template <int OUT, bool TALL>
struct LoraUp {
  static constexpr int WIDE = TALL && OUT != LORA_GLU ? 2 : 1;           // column blocks of a warp
  static constexpr int BLOCKS = TALL ? WIDE : 4;                         // ... of a step
  // (rows of planes are not padded, so that four blocks fit; their 16-byte pieces change places instead: lora_swap)
  static constexpr int ROW = lora_row_bytes<OUT>() * WIDE, LD = OUT == LORA_GLU ? ROW : ROW + 16;
  static constexpr int ROWS_BYTES = (TALL ? 64 : 4 * 16) * LD;
};
// where piece q of row r of planes stands: the eight lanes of a 16-byte load have two neighbouring rows and pieces c, c + 2, c + 8, c + 10
__device__ __forceinline__ int lora_swap(int r, int q) { return q ^ (r & 1) ^ (q >> 3 << 2); }
template <int KS, int OUT, bool TALL>
__global__ void __launch_bounds__(LORA_UP_THREADS, 4) lora_up_kernel(const LoraParams p) {
  extern __shared__ __align__(128) uint8_t smem8[];
  using Up = LoraUp<OUT, TALL>;
  constexpr int PARTS = lora_parts<OUT, TALL>(), B_BYTES = KS * 1024, SEG = lora_row_bytes<OUT>(), LD = Up::LD, WIDE = Up::WIDE, STEP = Up::BLOCKS, BOTH = OUT == LORA_GLU ? 2 : 1;
  constexpr int TILE = TALL ? 64 : 16;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int32_t* rec = p.tiles + static_cast<long long>(blockIdx.y) * (4 + TILE);
  const int4 tl = *reinterpret_cast<const int4*>(rec);
  const int2 made = lora_plan_of(p);
  // (ranges of one slice, of gate | up of both, in whole steps)
  int s = 0;
  if (OUT != LORA_GLU)
    while (static_cast<int>(blockIdx.x) >= p.part0[s + 1]) ++s;
  const int n = tl.z, begin = OUT == LORA_GLU ? 0 : p.block0[s], blocks = OUT == LORA_GLU ? p.blocks : p.block0[s + 1] - begin, all = (blocks + STEP - 1) / STEP;
  const int parts = OUT == LORA_GLU ? gridDim.x : p.part0[s + 1] - p.part0[s], part = blockIdx.x - (OUT == LORA_GLU ? 0 : p.part0[s]);
  const int c0 = begin + static_cast<int>(static_cast<long long>(all) * part / parts) * STEP,
            c1 = begin + min(blocks, static_cast<int>(static_cast<long long>(all) * (part + 1) / parts) * STEP);
  const bool has = tl.x >= 0;
  if (lora_other_plan(p, made) || n == 0 || c0 >= c1) {
    pdl_sync();
    return;
  }
  // shared memory: v [m16 blocks][the block's slice, or both][PARTS][KS] of 512 bytes, then one or two steps: B of the column blocks (of gate, of up), rows of base or planes
  const bool adds = OUT == LORA_GLU || p.base != nullptr;
  constexpr bool PAIR = WIDE == 2 && (OUT == LORA_BF16 || KS >= 4);
  constexpr int V_BLOCK = BOTH * PARTS * KS * 512;          // of 16 rows
  const int step_bytes = STEP * BOTH * B_BYTES + (adds ? Up::ROWS_BYTES : 0);
  const uint32_t vs = smem_u32(smem8), steps = vs + (TILE / 16) * V_BLOCK;
  // a lane's copies of base or planes: 16 bytes (q) of every ROWS-th row of its 16
  constexpr int PER = Up::ROW / 16, ROWS = 32 / PER;
  const int q = lane % PER, mt = TALL ? warp : 0, r0 = mt * 16 + lane / PER;
  const uint8_t* src[16 / ROWS];
  bool there[16 / ROWS];
  if (adds) {
    const long long ld = (OUT == LORA_GLU ? p.width : p.ld_base) * (OUT == LORA_BF16 ? 2 : 4);
#pragma unroll
    for (int i = 0; i < 16 / ROWS; ++i) {
      there[i] = r0 + i * ROWS < n;
      src[i] = static_cast<const uint8_t*>(OUT == LORA_GLU ? p.planes : p.base) + (there[i] ? rec[4 + r0 + i * ROWS] : 0) * ld;
    }
  }
  const uint32_t rows_to = STEP * BOTH * B_BYTES + (TALL ? 0 : warp * 16 * LD);                // the warp's rows in a step (tall: all warps')
  const uint4* b = p.b + (has ? tl.x : 0) * p.b_slot;
  auto load = [&](int c, int turn) {
    if (c < c1) {
      const uint32_t to = steps + (turn & p.ahead) * step_bytes;
      if (has) {
        const int chunks = min(STEP, c1 - c) * KS * 64;
        for (int i = tid; i < chunks; i += LORA_UP_THREADS) {
          cp_async16(to + i * 16, b + static_cast<long long>(c) * KS * 64 + i, 16);
          if (OUT == LORA_GLU) cp_async16(to + STEP * B_BYTES + i * 16, b + static_cast<long long>(p.blocks + c) * KS * 64 + i, 16);      // (the up columns' blocks follow the gate's)
        }
      }
      const int block = c + (TALL ? q / (SEG / 16) : warp), in_block = q % (SEG / 16);
      if (adds && block < c1) {
        long long at;
        bool in;
        if constexpr (OUT == LORA_GLU) {
          at = block * 64 + in_block * 4;
          in = at < 2 * ((p.ff + 15) & ~15);
        } else {
          at = p.col0[s] + (block - p.block0[s]) * 32 + in_block * (OUT == LORA_F32 ? 4 : 8);
          in = at < p.col0[s + 1];
        }
        const uint32_t row_to = to + rows_to + r0 * LD + (OUT == LORA_GLU ? lora_swap(r0, q) : q) * 16;
        const long long bytes_at = (in ? at : 0) * (OUT == LORA_BF16 ? 2 : 4);
#pragma unroll
        for (int i = 0; i < 16 / ROWS; ++i)
          if (there[i]) cp_async16(row_to + i * ROWS * LD, src[i] + bytes_at, in ? 16 : 0);
      }
    }
    cp_async_commit();
  };
  const int ra = mt * 16 + g, rb = ra + 8;
  const long long row[2] = {ra < n ? rec[4 + ra] : -1, rb < n ? rec[4 + rb] : -1};
  load(c0, 0);
  pdl_sync();
  if (has) {
    const uint4* v = reinterpret_cast<const uint4*>(p.v) + (static_cast<long long>(blockIdx.y) * (TILE / 16) * p.slices + s) * PARTS * KS * 32;
    for (int m = 0; m < (n + 15) >> 4; ++m)
      for (int i = tid; i < V_BLOCK / 16; i += LORA_UP_THREADS) cp_async16(vs + m * V_BLOCK + i * 16, v + m * p.slices * PARTS * KS * 32 + i, 16);
  }
  cp_async_commit();
  const uint32_t frags = vs + mt * V_BLOCK + lane * 16;
  int turn = 0;
  for (int c = c0; c < c1; c += STEP, ++turn) {
    if (p.ahead) {
      load(c + STEP, turn + 1);
      cp_async_wait<1>();                                     // (all but the step ahead; v came before it)
    } else {
      cp_async_wait<0>();
    }
    __syncthreads();
    const uint32_t from = steps + (turn & p.ahead) * step_bytes;
    float ds[WIDE][4][4] = {}, u[4][4] = {};
    const int first = c + (TALL ? 0 : warp);
    // (two column blocks: v is read once for both.  4096 rows of bf16 at rank 64 34.0 -> 33.3 us, of q | k | v in fp32 82 -> 73; fp32 at rank 16 11.0 -> 11.7, too many
    // registers for what it saves)
    const bool pair = PAIR && first + 1 < c1;
    if (has && pair && mt * 16 < n) lora_product<KS, PARTS, PAIR ? 2 : 1>(ds, frags, from + lane * 16);
#pragma unroll
    for (int w = 0; w < WIDE; ++w) {
      const int mine = TALL ? w : warp, block = c + mine;
      if (mt * 16 >= n || block >= c1) break;
      float (&d)[4][4] = ds[w];
      if (has && !pair) {
        lora_product<KS, PARTS, 1>(&d, frags, from + mine * B_BYTES + lane * 16);
        if constexpr (OUT == LORA_GLU) lora_product<KS, PARTS, 1>(&u, frags + PARTS * KS * 512, from + (STEP + mine) * B_BYTES + lane * 16);
      }
      const int col = p.col0[s] + (block - p.block0[s]) * 32 + t4 * 8;
      if (col >= p.col0[s + 1]) continue;
      const uint8_t* add = smem8 + (from - vs) + rows_to + ra * LD + (OUT == LORA_GLU ? 0 : (TALL ? w * SEG : 0) + t4 * (SEG / 4));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (row[h] < 0) continue;
        float y[8], z[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          y[i] = d[i >> 1][h * 2 + (i & 1)];
          z[i] = u[i >> 1][h * 2 + (i & 1)];
        }
        void* out = lora_place<OUT>(p, row[h], col);
        if constexpr (OUT == LORA_GLU) {
          const float4* pl = reinterpret_cast<const float4*>(add + h * 8 * LD);
          const int c = lora_swap(g, (t4 >> 1) * 8 + (t4 & 1) * 2);               // (its neighbour, and the up columns', differ in one bit)
          lora_gated(p, out, row[h], col, y, z, pl[c], pl[c ^ 1], pl[c ^ 4], pl[c ^ 5]);
        }
        else lora_result<OUT>(out, y, p.base ? add + h * 8 * LD : nullptr);
      }
    }
    __syncthreads();                                          // (the step has been read: the one after the next, or the next, may come into its place)
    if (!p.ahead) load(c + STEP, 0);
  }
}

// ---- both, for few rows -------------------------------------------------------------------------------------------------------------
// A cluster of eight blocks per tile of up to 16 rows.  RT: rank tiles, all of them in one pass over the block's share of K.  One chain: the tile's record, a round or two of
// loads of x and A, the warps' and the cluster's meeting, the columns; each is latency.  32 rows with an adapter each, 2048 x 2048 at rank 16 (4.3 MB): 4.5 us a call in
// a chain; 64 rows with 12 adapters, 4096 to 4608 columns at rank 32 (14 MB): 8.1.  In two launches 8.3 and 11.7.
constexpr int LORA_CLUSTER = 8, LORA_FEW_RANKS = 128, LORA_FEW_LD = 20;
template <int KS, int OUT, int RT>
__global__ void __launch_bounds__(LORA_THREADS) lora_few_kernel(const LoraParams p) {
  extern __shared__ __align__(128) uint8_t smem8[];
  constexpr int LD = LORA_FEW_LD, VR = RT * 16, U = RT > 2 ? 1 : 2;
  float* red = reinterpret_cast<float*>(smem8);                         // [8 warps][VR][LD]
  float* mine = red + 8 * VR * LD;                                      // [16 rows][VR]: this block's part of v
  uint32_t* frags = reinterpret_cast<uint32_t*>(mine + 16 * VR);        // the sum, as parts
  constexpr int PARTS = lora_parts<OUT, false>();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int rank = blockIdx.x % LORA_CLUSTER;
  pdl_sync();
  const int2 made = lora_plan_of(p);
  const int32_t* rec = p.tiles + (blockIdx.x / LORA_CLUSTER) * (4 + 16);
  const int4 tl = *reinterpret_cast<const int4*>(rec);
  const int row_a = rec[4 + g], row_b = rec[12 + g]; // (places behind the tile's last hold anything)
  const int n = tl.z;
  if (lora_other_plan(p, made) || n == 0) return;    // (all blocks of the cluster)
  const bool has = tl.x >= 0;
  const int c1 = static_cast<int>(static_cast<long long>(p.blocks) * (rank + 1) / LORA_CLUSTER), first = static_cast<int>(static_cast<long long>(p.blocks) * rank / LORA_CLUSTER) + warp;
  const uint4* b = p.b + (has ? tl.x : 0) * p.b_slot + lane;
  const long long rows[2] = {g < n ? row_a : -1, g + 8 < n ? row_b : -1};
  uint4 w[KS][2];
  if (has) {
    const uint4* a = p.a + tl.x * p.a_slot + g * 8;
    const int even = t4 ^ g, odd = (4 + t4) ^ g;       // where this lane's eight k of 64 stand, of an even block of 32 and an odd one
    const float scale = p.scale[tl.x];
    const int rts = p.VR >> 4, kb32 = (p.K + 31) / 32, k0 = kb32 * rank / LORA_CLUSTER, k1 = kb32 * (rank + 1) / LORA_CLUSTER;
    const __nv_bfloat16 *xa = p.x + (g < n ? row_a : 0) * p.ldx + t4 * 8, *xb = p.x + (g + 8 < n ? row_b : 0) * p.ldx + t4 * 8;
    float acc[RT][2][4] = {};
    for (int kb = k0 + warp; kb < k1; kb += 8 * U) {
      uint4 av[U][RT][2], xv[U][2];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = kb + u * 8;
        const bool in = k < k1 && k * 32 + t4 * 8 < p.K;
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            av[u][i][h] = i < rts && k < k1 ? ldg_stream(a + (static_cast<long long>(k >> 1) * rts + i) * 128 + h * 64 + (k & 1 ? odd : even)) : make_uint4(0u, 0u, 0u, 0u);
        xv[u][0] = in ? *reinterpret_cast<const uint4*>(xa + k * 32) : make_uint4(0u, 0u, 0u, 0u);
        xv[u][1] = in && n > 8 ? *reinterpret_cast<const uint4*>(xb + k * 32) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (j > 0 && n <= 8) break;
#pragma unroll
          for (int i = 0; i < RT; ++i) mma_bf16(acc[i][j], av[u][i][0].x, av[u][i][1].x, av[u][i][0].y, av[u][i][1].y, xv[u][j].x, xv[u][j].y);
#pragma unroll
          for (int i = 0; i < RT; ++i) mma_bf16(acc[i][j], av[u][i][0].z, av[u][i][1].z, av[u][i][0].w, av[u][i][1].w, xv[u][j].z, xv[u][j].w);
        }
    }
    if (first < c1) lora_take<KS>(w, b + static_cast<long long>(first) * KS * 64);         // (on its way while the warps and the cluster meet)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (j > 0 && n <= 8) break;
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        float* to = red + (warp * VR + i * 16 + g) * LD + j * 8 + t4 * 2;
        *reinterpret_cast<float2*>(to) = make_float2(acc[i][j][0], acc[i][j][1]);
        *reinterpret_cast<float2*>(to + 8 * LD) = make_float2(acc[i][j][2], acc[i][j][3]);
      }
    }
    __syncthreads();
    for (int e = tid; e < n * VR; e += LORA_THREADS) {
      const int c = e / VR, r = e % VR;
      float s = 0.f;
#pragma unroll
      for (int q = 0; q < 8; ++q) s += red[(q * VR + r) * LD + c];
      mine[e] = scale * s;
    }
    cluster_sync_all();
    constexpr int LOG = KS == 1 ? 0 : KS == 2 ? 1 : 2;
    for (int e = tid; e < n * (VR / 4); e += LORA_THREADS) {             // (rows behind the last: a product's rows do not touch one another)
      const int c = e / (VR / 4), k = e % (VR / 4) * 4;
      if (k >= p.VR) continue;
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int z = 0; z < LORA_CLUSTER; ++z) {
        const float4 q = ld_dsmem_f32x4(mine + e * 4, z);
        s.x += q.x; s.y += q.y; s.z += q.z; s.w += q.w;
      }
      lora_put(frags, p.slices, PARTS, LOG, c, k, s.x, s.y);
      lora_put(frags, p.slices, PARTS, LOG, c, k + 2, s.z, s.w);
    }
    __syncthreads();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  }
  const uint4* fr = reinterpret_cast<const uint4*>(frags) + lane;
  for (int c = first, s = 0; c < c1; c += 8) {
    while (OUT != LORA_GLU && c >= p.block0[s + 1]) ++s;
    const int col = p.col0[s] + (c - p.block0[s]) * 32 + t4 * 8;
    const bool in = col < p.col0[s + 1];
    // base or planes first: they come from farther away than B
    float4 add[2][OUT == LORA_GLU ? 6 : 2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (in && rows[h] >= 0) {
        if constexpr (OUT == LORA_GLU) {
          const float4* pl = reinterpret_cast<const float4*>(p.planes + rows[h] * p.width + (col >> 4) * 32 + (col & 15));
          add[h][0] = pl[0];
          add[h][1] = pl[1];
          add[h][4] = pl[4];
          add[h][5] = pl[5];
        } else if (p.base) {
          const float4* from = reinterpret_cast<const float4*>(static_cast<const uint8_t*>(p.base) + (rows[h] * p.ld_base + col) * (OUT == LORA_F32 ? 4 : 2));
          add[h][0] = from[0];
          if (OUT == LORA_F32) add[h][1] = from[1];
        }
      }
    float d[4][4] = {}, u[4][4] = {};
    if (has) {
      lora_block<KS, PARTS>(d, fr + s * PARTS * KS * 32, w);
      if constexpr (OUT == LORA_GLU) {
        lora_take<KS>(w, b + static_cast<long long>(p.blocks + c) * KS * 64);
        lora_block<KS, PARTS>(u, fr + PARTS * KS * 32, w);
      }
      if (c + 8 < c1) lora_take<KS>(w, b + static_cast<long long>(c + 8) * KS * 64);
    }
    if (!in) continue;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (rows[h] < 0) continue;
      float y[8], z[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y[i] = d[i >> 1][h * 2 + (i & 1)];
        z[i] = u[i >> 1][h * 2 + (i & 1)];
      }
      void* out = lora_place<OUT>(p, rows[h], col);
      if constexpr (OUT == LORA_GLU) lora_gated(p, out, rows[h], col, y, z, add[h][0], add[h][1], add[h][4], add[h][5]);
      else lora_result<OUT>(out, y, p.base ? static_cast<const void*>(&add[h][0]) : nullptr);
    }
  }
  __syncwarp();
  if (has) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");       // (nobody leaves while others read its part)
}

// ---- host -------------------------------------------------------------------------------------------------------------------------
static int lora_tile_rows(int T) { return T <= 64 ? 16 : 64; }
// the most tiles a step can have
static int lora_max_tiles(int T, int slots) { return T / lora_tile_rows(T) + (T < slots + 1 ? T : slots + 1); }
// ... groups
static int lora_max_groups(int T, int slots) { return T / LORA_DOWN_ROWS + (T < slots ? T : slots); }
// ... and about how many tiles it has (half of the adapters)
static int lora_tiles(int T, int slots) {
  const int adapters = T < slots + 1 ? T : slots + 1;
  return T <= 64 ? adapters : (T + 63) / 64 + adapters / 2;
}
// Results in fp32: a sum takes at most eight stages, since the tensor cores cut it off at every step.  A cluster of eight with 256 columns of sums a block reaches
// rank tiles of a block x K = 65536, to which lora_launch brings the rank tiles; beyond K = 65536 the chains grow.  (Products of one sign at rank 128, off by, of the
// result: K = 14336 3.1e-6 with the usual sums, 2.1e-6 so; K = 65536 1.6e-5 and 2.2e-6.)
constexpr int LORA_CHAIN = 8, LORA_CHAIN_K = LORA_STAGE_K * LORA_CHAIN * 8 * 16;
template <int RT>
static bool lora_long(const LoraParams& p) { return p.f32 && (p.K + LORA_STAGE_K - 1) / LORA_STAGE_K > 8 * LORA_CHAIN * LoraDown<RT>::ACCS; }
template <int RT>
static int lora_k_split(const LoraParams& p, int slots) {
  const int stages = (p.K + LORA_STAGE_K - 1) / LORA_STAGE_K, adapters = p.T < slots + 1 ? p.T : slots + 1;
  const int groups = p.T <= 64 ? adapters : (p.T + LORA_DOWN_ROWS - 1) / LORA_DOWN_ROWS + adapters / 4, passes = (p.VR / 16 + RT - 1) / RT;
  // All clusters at once (4096 rows of 8192, some 35 clusters: of four 36.6 us, of seven, of which 37 fit, 34.1, of eight, of which 33 do, 39.7)
  // (Of a kernel with tensor memory the runtime counts one block an SM; these take half of it at most, so another kernel stands in with their shared memory.)
  constexpr auto like = lora_up_kernel<1, LORA_BF16, true>;
  int split = rm_smem<like>() == cudaSuccess ? 8 : 1;
  while (split > 1 && groups * passes > rm_clusters<like>(split, LORA_UP_THREADS, LoraDown<RT>::SMEM)) --split;
  const int most = stages > 4 ? stages / 4 : 1;          // four stages a block
  if (split > most) split = most;
  const int longest = LORA_CHAIN * (lora_long<RT>(p) ? LoraDown<RT>::MOST_ACCS : LoraDown<RT>::ACCS), least = (stages + longest - 1) / longest;
  if (p.f32 && split < least) split = least < 8 ? least : 8;
  return split;
}
// (its warps' chains: 32 steps of the matrix units, as many as eight stages have)
constexpr int LORA_FEW_K = 32768;
// One launch for a step of at most 64 rows, where an adapter is what eight SMs take in good time.  How many adapters the step's rows have the host does not know (the ids are on
// the device), so the rule sees an adapter's bytes alone; 3 MB is where both forms take the same for one row and for a dozen adapters.  K = N at rank 64, us in
// one launch / two:  1 row        1 MB 5.6 / 7.6   2 MB 8.6 / 9.6     3 MB 11.7 / 11.8   4 MB 14.5 / 14.0   6 MB 20.2 / 18.5
//                    64, of 1     1 MB 7.9 / 8.4   2 MB 11.4 / 10.8   3 MB 14.6 / 13.3   4 MB 17.8 / 15.8
//                    64, of 12    1 MB 8.0 / 10.8  2 MB 14.5 / 15.7   3 MB 18.2 / 19.7   4 MB 23.9 / 23.7   6 MB 30.7 / 32.2
//                    64, of 32    1 MB 10.5 / 14.9 2 MB 16.6 / 21.3   3 MB 21.9 / 27.6   4 MB 27.8 / 34.1
// (2 MB and more of one adapter for all rows lose 5 to 10 % by it, more than 3 MB of many up to 18 %; rank 16 to 1.5 MB: one launch takes half to 0.9 of two.)
static bool lora_few(const LoraParams& p) { return p.T <= 64 && p.VR <= LORA_FEW_RANKS && p.rank_tiles <= 4 && (p.a_slot + p.b_slot) * 16 <= 3 << 20 && p.K <= LORA_FEW_K; }

template <int KS, int OUT, bool TALL>
static int lora_up_tiles(LoraParams& p, int max_tiles, int tiles, void* stream) {
  using Up = LoraUp<OUT, TALL>;
  VB_CHECK_CUDA((rm_smem<lora_up_kernel<KS, OUT, TALL>>()));
  const size_t v_bytes = static_cast<size_t>(p.tile_rows >> 4) * (OUT == LORA_GLU ? 2 : 1) * lora_parts<OUT, TALL>() * KS * 512,
               step = static_cast<size_t>(Up::BLOCKS) * KS * 1024 * (OUT == LORA_GLU ? 2 : 1) + (OUT == LORA_GLU || p.base ? Up::ROWS_BYTES : 0);
  p.ahead = v_bytes + 2 * step <= VB_MAX_DYN_SMEM;
  const size_t smem = v_bytes + (p.ahead + 1) * step;
  // one wave of up to four blocks an SM (a wave and a few blocks take as long as two), a step each at least
  const int fit = smem <= 56 * 1024 ? 4 : smem <= 75 * 1024 ? 3 : smem <= 113 * 1024 ? 2 : 1;       // (227 KB and 1 KB of the system's a block make 228)
  int split = fit * sm_count() / tiles;
  const int most = (p.blocks + Up::BLOCKS - 1) / Up::BLOCKS;
  if (split > most) split = most;
  if (split < 1) split = 1;
  if (OUT != LORA_GLU) {                               // each slice its share of them
    for (int s = 0; s < p.slices; ++s) {
      const int blocks = p.block0[s + 1] - p.block0[s], steps = (blocks + Up::BLOCKS - 1) / Up::BLOCKS;
      const int share = static_cast<int>(static_cast<long long>(split) * blocks / p.blocks);
      p.part0[s + 1] = p.part0[s] + (share < 1 ? 1 : share > steps ? steps : share);
    }
    split = p.part0[p.slices];
  }
  VB_LAUNCH_PDL((lora_up_kernel<KS, OUT, TALL>), dim3(split, max_tiles), LORA_UP_THREADS, smem, stream, p);
  return 0;
}
template <int KS, int OUT>
static int lora_up_launch(LoraParams& p, int max_tiles, int tiles, void* stream) {
  return p.tile_rows == 16 ? lora_up_tiles<KS, OUT, false>(p, max_tiles, tiles, stream) : lora_up_tiles<KS, OUT, true>(p, max_tiles, tiles, stream);
}
template <int RT, int ACCS>
static int lora_down_sums(LoraParams& p, int slots, void* stream) {
  VB_CHECK_CUDA((rm_smem<lora_down_kernel<RT, ACCS>>()));
  p.k_split = lora_k_split<RT>(p, slots);
  CUtensorMap x_map;
  const int rc = vb_tensor_map_2d_bf16(&x_map, p.x, p.T, p.K, p.ldx, LORA_BOX_ROWS);
  if (rc) return rc;
  VB_CHECK_CUDA(launch_kernel_cluster3(lora_down_kernel<RT, ACCS>, dim3(p.k_split, lora_max_groups(p.T, slots), (p.VR / 16 + RT - 1) / RT), dim3(LORA_DOWN_THREADS), LoraDown<RT>::SMEM,
                                       static_cast<cudaStream_t>(stream), true, dim3(p.k_split, 1, 1), p, x_map));
  return 0;
}
template <int RT>
static int lora_down_launch(LoraParams& p, int slots, void* stream) {
  if constexpr (LoraDown<RT>::MOST_ACCS > LoraDown<RT>::ACCS)
    if (lora_long<RT>(p)) return lora_down_sums<RT, LoraDown<RT>::MOST_ACCS>(p, slots, stream);
  return lora_down_sums<RT, LoraDown<RT>::ACCS>(p, slots, stream);
}
template <int KS, int OUT, int RT>
static int lora_few_tiles(const LoraParams& p, int tiles, void* stream) {
  VB_CHECK_CUDA((rm_smem<lora_few_kernel<KS, OUT, RT>>()));
  const size_t smem = (8 * RT * 16 * LORA_FEW_LD + 16 * RT * 16) * sizeof(float) + static_cast<size_t>(p.VR >> 4) * lora_parts<OUT, false>() * 512;
  VB_LAUNCH_PDL_CLUSTER((lora_few_kernel<KS, OUT, RT>), tiles * LORA_CLUSTER, LORA_THREADS, smem, stream, LORA_CLUSTER, p);
  return 0;
}
template <int KS, int OUT>
static int lora_few_launch(const LoraParams& p, int tiles, void* stream) {
  const int rts = p.VR >> 4;
  if constexpr (KS == 1 && OUT != LORA_GLU)
    if (rts == 1) return lora_few_tiles<KS, OUT, 1>(p, tiles, stream);
  if constexpr (KS <= 2)
    if (rts <= 2) return lora_few_tiles<KS, OUT, 2>(p, tiles, stream);
  if (rts <= 4) return lora_few_tiles<KS, OUT, 4>(p, tiles, stream);
  return lora_few_tiles<KS, OUT, 8>(p, tiles, stream);
}
template <int OUT>
static int lora_launch(LoraParams& p, int slots, void* stream) {
  const int max_tiles = lora_max_tiles(p.T, slots);
  p.parts = p.tile_rows == 16 ? lora_parts<OUT, false>() : lora_parts<OUT, true>();
  p.f32 = OUT == LORA_F32;
  if (OUT == LORA_GLU) p.blocks = p.block0[1];         // column blocks of one of the two
  if (lora_few(p)) {
    if (p.rank_tiles == 1) return lora_few_launch<1, OUT>(p, max_tiles, stream);
    if (p.rank_tiles == 2) return lora_few_launch<2, OUT>(p, max_tiles, stream);
    return lora_few_launch<4, OUT>(p, max_tiles, stream);
  }
  VB_CHECK_ARG(p.wait_flag = wait_flag(WK_LORA), "vb_lora: no mapped host memory");
  int rt = p.VR <= 16 ? 1 : p.VR <= 32 ? 2 : p.VR <= 64 ? 4 : 8;
  while (p.f32 && rt > 1 && static_cast<long long>(p.K) * rt > LORA_CHAIN_K) rt /= 2;
  const int rc = rt == 1   ? lora_down_launch<1>(p, slots, stream)
                 : rt == 2 ? lora_down_launch<2>(p, slots, stream)
                 : rt == 4 ? lora_down_launch<4>(p, slots, stream)
                           : lora_down_launch<8>(p, slots, stream);
  if (rc) return rc;
  switch (p.rank_tiles) {
    case 1: return lora_up_launch<1, OUT>(p, max_tiles, lora_tiles(p.T, slots), stream);
    case 2: return lora_up_launch<2, OUT>(p, max_tiles, lora_tiles(p.T, slots), stream);
    case 4: return lora_up_launch<4, OUT>(p, max_tiles, lora_tiles(p.T, slots), stream);
    default: return lora_up_launch<8, OUT>(p, max_tiles, lora_tiles(p.T, slots), stream);
  }
}
// checks and fills what both entry points share
static int lora_bank(const char* who, LoraParams& p, const VbLoraBank* bank, int T) {
  VB_CHECK_ARG(bank && bank->d_a && bank->d_b && bank->d_scale, "%s: null pointer", who);
  VB_CHECK_ARG(reinterpret_cast<uintptr_t>(bank->d_a) % 16 == 0 && reinterpret_cast<uintptr_t>(bank->d_b) % 16 == 0 && reinterpret_cast<uintptr_t>(bank->d_scale) % 4 == 0,
               "%s: the bank must be 16-byte aligned", who);
  VB_CHECK_ARG(bank->slots >= 1 && bank->slots <= LORA_MAX_SLOTS, "%s: %d adapters; 1 to %d", who, bank->slots, LORA_MAX_SLOTS);
  VB_CHECK_ARG(bank->rank == 16 || bank->rank == 32 || bank->rank == 64 || bank->rank == 128, "%s: padded rank %d must be 16, 32, 64 or 128", who, bank->rank);
  VB_CHECK_ARG(bank->slices >= 1 && bank->slices <= LORA_MAX_SLICES, "%s: %d slices; 1 to %d", who, bank->slices, LORA_MAX_SLICES);
  VB_CHECK_ARG(bank->K >= 8 && bank->K % 8 == 0 && bank->K <= (1 << 24), "%s: inputs of %d; a multiple of 8", who, bank->K);
  p.slices = bank->slices;
  p.block0[0] = p.col0[0] = 0;
  for (int s = 0; s < p.slices; ++s) {
    const int w = bank->widths[s];
    VB_CHECK_ARG(w >= 8 && w % 8 == 0 && w <= (1 << 24), "%s: slice of %d columns; a multiple of 8", who, w);
    p.block0[s + 1] = p.block0[s] + (w + 31) / 32;
    p.col0[s + 1] = p.col0[s] + w;
  }
  p.tile_rows = lora_tile_rows(T);
  p.a = static_cast<const uint4*>(bank->d_a);
  p.b = static_cast<const uint4*>(bank->d_b);
  p.scale = bank->d_scale;
  p.T = T;
  p.K = bank->K;
  p.rank_tiles = bank->rank / 16;
  p.VR = p.slices * bank->rank;
  p.a_slot = static_cast<long long>(p.VR / 16) * ((p.K + 63) / 64) * 128;
  p.b_slot = static_cast<long long>(p.block0[p.slices]) * p.rank_tiles * 64;
  p.blocks = p.block0[p.slices];
  return 0;
}
// v of every tile in three parts; none where one launch does both products
static size_t lora_ws_bytes(const LoraParams& p, int slots) {
  return lora_few(p) ? 0 : static_cast<size_t>(lora_max_tiles(p.T, slots)) * (p.tile_rows / 16) * (p.VR / 16) * 3 * 512;
}
static int lora_setup(const char* who, LoraParams& p, const void* d_x, long long ldx, const VbLoraBank* bank, const void* d_tiles, int T, void* d_ws, size_t ws_bytes) {
  const int rc = lora_bank(who, p, bank, T);
  if (rc) return rc;
  VB_CHECK_ARG(d_x && d_tiles, "%s: null pointer", who);
  VB_CHECK_ARG(reinterpret_cast<uintptr_t>(d_tiles) % 16 == 0, "%s: the plan must be 16-byte aligned", who);
  VB_CHECK_ARG(T <= LORA_MAX_ROWS, "%s: %d rows; at most %d", who, T, LORA_MAX_ROWS);
  VB_CHECK_ARG(ldx % 8 == 0 && ldx >= p.K && reinterpret_cast<uintptr_t>(d_x) % 16 == 0, "%s: rows of x must be 16-byte aligned (K %d, row stride %lld)", who, p.K, ldx);
  VB_CHECK_ARG(p.plan_flag = wait_flag(WK_PLAN), "%s: no mapped host memory", who);
  p.slots = bank->slots;
  p.tiles = static_cast<const int32_t*>(d_tiles) + LORA_PLAN_HEAD;
  p.groups = reinterpret_cast<const int4*>(p.tiles + static_cast<long long>(lora_max_tiles(T, bank->slots)) * (4 + p.tile_rows));
  p.x = static_cast<const __nv_bfloat16*>(d_x);
  p.ldx = ldx;
  p.v = static_cast<uint32_t*>(d_ws);
  const size_t need = lora_ws_bytes(p, bank->slots);
  VB_CHECK_ARG(need == 0 || (d_ws && ws_bytes >= need && reinterpret_cast<uintptr_t>(d_ws) % 16 == 0), "%s: workspace of %zu bytes, 16-byte aligned, is needed (%zu given)",
               who, need, ws_bytes);
  return 0;
}

}  // namespace vb

using namespace vb;

extern "C" {

size_t vb_lora_plan_bytes(int T, int slots) {
  return T < 1 || slots < 1 ? 0 : LORA_PLAN_HEAD * 4 + static_cast<size_t>(lora_max_tiles(T, slots)) * (4 + lora_tile_rows(T)) * 4 + static_cast<size_t>(lora_max_groups(T, slots)) * 16;
}

int vb_lora_plan(void* d_tiles, const int32_t* d_ids, int T, int slots, void* stream) {
  VB_CHECK_ARG(d_tiles && d_ids, "vb_lora_plan: null pointer");
  VB_CHECK_ARG(reinterpret_cast<uintptr_t>(d_tiles) % 16 == 0 && reinterpret_cast<uintptr_t>(d_ids) % 4 == 0, "vb_lora_plan: the plan must be 16-byte aligned, ids 4-byte");
  VB_CHECK_ARG(slots >= 1 && slots <= LORA_MAX_SLOTS, "vb_lora_plan: %d adapters; 1 to %d", slots, LORA_MAX_SLOTS);
  VB_CHECK_ARG(T >= 1 && T <= LORA_MAX_ROWS, "vb_lora_plan: %d rows; 1 to %d", T, LORA_MAX_ROWS);
  VB_CHECK_CUDA((rm_smem<lora_plan_kernel>(LORA_PLAN_SMEM)));
  VB_LAUNCH_PDL(lora_plan_kernel, 1, 1024, 32 * (slots + 1) * 4, stream, static_cast<int32_t*>(d_tiles) + LORA_PLAN_HEAD, d_ids, T, slots, lora_tile_rows(T), lora_max_tiles(T, slots), lora_max_groups(T, slots));
  return 0;
}

size_t vb_lora_workspace_bytes(const VbLoraBank* bank, int T) {
  LoraParams p = {};
  return T < 1 || lora_bank("vb_lora_workspace_bytes", p, bank, T) ? 0 : lora_ws_bytes(p, bank->slots);
}

int vb_lora(void* d_out, long long ld_out, const void* d_base, long long ld_base, int out_f32, const void* d_x, long long ldx, const VbLoraBank* bank,
            const void* d_tiles, int T, void* d_ws, size_t ws_bytes, void* stream) {
  VB_CHECK_ARG(d_out, "vb_lora: null pointer");
  if (T <= 0) return 0;
  LoraParams p = {};
  const int rc = lora_setup("vb_lora", p, d_x, ldx, bank, d_tiles, T, d_ws, ws_bytes);
  if (rc) return rc;
  const int unit = out_f32 ? 4 : 8, N = p.col0[p.slices];
  VB_CHECK_ARG(ld_out % unit == 0 && ld_out >= N && reinterpret_cast<uintptr_t>(d_out) % 16 == 0 &&
                   (!d_base || (ld_base % unit == 0 && ld_base >= N && reinterpret_cast<uintptr_t>(d_base) % 16 == 0)),
               "vb_lora: rows of out and base must be 16-byte aligned and at least %d columns apart", N);
  p.out = d_out;
  p.ldo = ld_out;
  p.base = d_base;
  p.ld_base = ld_base;
  return out_f32 ? lora_launch<LORA_F32>(p, bank->slots, stream) : lora_launch<LORA_BF16>(p, bank->slots, stream);
}

int vb_lora_gate_up(void* d_act, long long ld_act, int xt_rows, const float* d_planes, int splits, int half, const void* d_x, long long ldx, const VbLoraBank* bank,
                    const void* d_tiles, int T, void* d_ws, size_t ws_bytes, void* stream) {
  VB_CHECK_ARG(d_act && d_planes, "vb_lora_gate_up: null pointer");
  VB_CHECK_ARG(splits >= 1 && half >= 16 && half % 16 == 0 && half <= 64, "vb_lora_gate_up: %d planes, tiles of %d gate rows (16, 32, 48 or 64)", splits, half);
  if (T <= 0) return 0;
  LoraParams p = {};
  const int rc = lora_setup("vb_lora_gate_up", p, d_x, ldx, bank, d_tiles, T, d_ws, ws_bytes);
  if (rc) return rc;
  const int ff = p.col0[1];
  VB_CHECK_ARG(p.slices == 2 && p.col0[2] == 2 * ff, "vb_lora_gate_up: a bank of two slices of equal width is needed");
  VB_CHECK_ARG(xt_rows >= 0 && reinterpret_cast<uintptr_t>(d_act) % 16 == 0 && reinterpret_cast<uintptr_t>(d_planes) % 16 == 0 &&
                   (xt_rows > 0 || (ld_act % 8 == 0 && ld_act >= ff)),
               "vb_lora_gate_up: rows of act must be 16-byte aligned and at least %d columns apart", ff);
  p.out = d_act;
  p.ldo = ld_act;
  p.planes = d_planes;
  p.splits = splits;
  p.ff = ff;
  p.width = (ff + half - 1) / half * 2 * half;
  p.xt_rows = xt_rows;
  p.xt_kb = (ff + 63) / 64;
  return lora_launch<LORA_GLU>(p, bank->slots, stream);
}

}  // extern "C"
