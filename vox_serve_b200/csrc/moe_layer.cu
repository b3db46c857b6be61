// The experts of a mixture for the rows of a decode step (at most 64), reading the matrices of the chosen experts only:
//
//   y[t] = sum_c w[t, c] down_e(act(gate_e h_t, up_e h_t)) + sg[t] down_s(act(gate_s h_t, up_s h_t)),   e = idx[t, c]
//
// Two launches behind the router's.  A stream of weights: 3 x ff x W values for every expert that any row chose, a few
// rows each, so the kernels are built around loads that never pause.  Weights go from the packed tiles (vb_pack_weight_tiles; the same buffers that the
// projections of larger steps multiply) straight into the registers of the warp that multiplies them, 16 bytes a lane; a lane takes whole 16-byte chunks
// of 8 k, and since a product's k may stand in any order as long as both operands agree, the rows of h are taken by the same chunks.
//
//   route eight blocks of a cluster share the experts' logits of eight rows (the router's fp32 matrix is read once per eight rows), then a block each picks
//         one row's experts from all of them
//   up    block = (expert, 32 rows of its gate | up matrix: 16 gated or 32 plain columns), the eight warps divide k; sums meet in shared memory, the
//         activation times the routing weight leaves as three bf16 parts (exact, rowmma.cuh), so nothing is rounded between the two products
//   down  block = 32 columns of the result x a share of the (expert, piece of ff) units of the chosen experts, every warp adding its products to rows
//         of its own in shared memory; up to eight blocks of a cluster share the units and add up through distributed shared memory.  No atomics:
//         units, warps and blocks are added in a fixed order
//
// A table that names an expert twice for a row counts it once with both weights; an index that is no expert counts as none.
#include "../../include/vb_api.h"
#define VB_PDL_FAMILY 4
#include "rowmma.cuh"

namespace vb {

constexpr int ML_MAX_ROWS = 64, ML_MAX_EXPERTS = 1024, ML_MAX_TOP = 32, ML_THREADS = 256, ML_WARPS = 8;
enum MlAct { ML_SILU_GLU = 0, ML_CLAMPED_GLU = 1, ML_RELU2 = 2, ML_GELU = 3, ML_GELU_TANH = 4 };

struct MoeLayerParams {
  const __nv_bfloat16* h;
  long long ldh;
  const uint8_t *up, *down;             // packed: [expert][tile][k block][rows][128 B], [tile of 128][k block of all experts][128][128 B]
  const int32_t* idx;                   // [T][top]
  const float *wts, *sgate;
  __nv_bfloat16* act;                   // [3 parts][T top + T][ld_act]
  float* y;
  long long ldy, expert_bytes, part_stride;
  int T, W, E, top, ff, sff, ld_act, kb, up_rows, down_kb, act_kind, up_units, shared_units, cluster;
  float limit, slope;
};

// ---- router -----------------------------------------------------------------------------------------------------------------------
enum MlRouter { ML_SOFTMAX = 0, ML_SIGMOID = 1, ML_SOFTMAX_ALL = 2, ML_TABLE = 3 };
constexpr int ML_ROUTE_CLUSTER = 8;      // blocks, and rows, of a cluster
struct MoeRouteParams {
  int32_t* idx;
  float *wts, *sgate;
  const __nv_bfloat16* h;
  long long ldh;
  const float *w, *bias, *wsg;           // [E][W], [E], [W]
  const int32_t *ids, *table;
  int T, W, E, top, kind, groups, keep, vocab, parts;
};
// floats as integers of the same order; NaN above all (so a row that holds one still picks experts that exist), 0 below all: not to be picked
__device__ __forceinline__ uint32_t ml_key(float v) {
  const uint32_t u = __float_as_uint(v);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// the largest key of keys[0 .. n) and its place (ties: the lowest), in every lane
__device__ __forceinline__ int ml_argmax(const uint32_t* keys, int n, int lane) {
  uint32_t best = 0u;
  int at = 0x7fffffff;
  for (int e = lane; e < n; e += 32)
    if (at == 0x7fffffff || keys[e] > best) { best = keys[e]; at = e; }
  const uint32_t top = __reduce_max_sync(0xffffffffu, best);
  return __reduce_min_sync(0xffffffffu, best == top ? at : 0x7fffffff);
}
__global__ void __launch_bounds__(ML_THREADS) moe_layer_route_kernel(const MoeRouteParams p) {
  extern __shared__ __align__(16) int smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x % ML_ROUTE_CLUSTER, t0 = blockIdx.x / ML_ROUTE_CLUSTER * ML_ROUTE_CLUSTER, rows = min(ML_ROUTE_CLUSTER, p.T - t0);
  // the matrix's rows: the experts, then the shared expert's gate
  const int E = p.kind == ML_TABLE ? 0 : p.E, all = E + (p.wsg ? 1 : 0), per = (all + ML_ROUTE_CLUSTER - 1) / ML_ROUTE_CLUSTER;
  float* part = reinterpret_cast<float*>(smem);                   // [per][parts][8 rows]
  float* mine = part + per * p.parts * ML_ROUTE_CLUSTER;          // [per][8]: this block's logits
  float* z = mine + per * ML_ROUTE_CLUSTER;                       // [E] the row's logits, then its scores
  uint32_t* keys = reinterpret_cast<uint32_t*>(z + p.E);          // [E]
  uint32_t* gkeys = keys + p.E;                                   // [groups]
  pdl_sync();
  // a row of the matrix per warp, or `parts` warps share it
  const int slots = ML_WARPS / p.parts, q = warp % p.parts;
  for (int i = warp / p.parts; i < per; i += slots) {
    const int e = i * ML_ROUTE_CLUSTER + rank;
    if (e >= all) break;
    const float* w = e < E ? p.w + static_cast<long long>(e) * p.W : p.wsg;
    float s[ML_ROUTE_CLUSTER] = {};
    for (int k = (q * 32 + lane) * 8; k < p.W; k += p.parts * 256) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(w + k)), b = __ldg(reinterpret_cast<const float4*>(w + k + 4));
#pragma unroll
      for (int t = 0; t < ML_ROUTE_CLUSTER; ++t) {
        if (t >= rows) break;
        const uint4 x = *reinterpret_cast<const uint4*>(p.h + (t0 + t) * p.ldh + k);
        float v = s[t];
        v = fmaf(bf16_lo(x.x), a.x, v); v = fmaf(bf16_hi(x.x), a.y, v); v = fmaf(bf16_lo(x.y), a.z, v); v = fmaf(bf16_hi(x.y), a.w, v);
        v = fmaf(bf16_lo(x.z), b.x, v); v = fmaf(bf16_hi(x.z), b.y, v); v = fmaf(bf16_lo(x.w), b.z, v); v = fmaf(bf16_hi(x.w), b.w, v);
        s[t] = v;
      }
    }
#pragma unroll
    for (int t = 0; t < ML_ROUTE_CLUSTER; ++t) {
      if (t >= rows) break;
      const float v = warp_sum(s[t]);
      if (lane == 0) part[(i * p.parts + q) * ML_ROUTE_CLUSTER + t] = v;
    }
  }
  __syncthreads();
  for (int i = tid; i < per * ML_ROUTE_CLUSTER; i += ML_THREADS) {
    float v = 0.f;
    for (int k = 0; k < p.parts; ++k) v += part[(i / ML_ROUTE_CLUSTER * p.parts + k) * ML_ROUTE_CLUSTER + i % ML_ROUTE_CLUSTER];
    mine[i] = v;                                     // (rows behind the last and experts that are none hold anything; nobody asks for them)
  }
  cluster_sync_all();
  const bool has = rank < rows;
  if (has) {
    for (int e = tid; e < E; e += ML_THREADS) {
      const float v = ld_dsmem_f32(mine + e / ML_ROUTE_CLUSTER * ML_ROUTE_CLUSTER + rank, e % ML_ROUTE_CLUSTER);
      z[e] = p.kind == ML_SOFTMAX && p.bias ? v + p.bias[e] : v;
    }
    if (p.wsg && tid == 0) {
      const float v = ld_dsmem_f32(mine + E / ML_ROUTE_CLUSTER * ML_ROUTE_CLUSTER + rank, E % ML_ROUTE_CLUSTER);
      p.sgate[t0 + rank] = 1.f / (1.f + expf(-v));
    }
  }
  cluster_sync_all();                                // (others' logits have been read; nobody leaves before)
  if (!has || warp != 0) return;
  const int t = t0 + rank;
  int32_t* idx = p.idx + t * p.top;
  float* wts = p.wts + t * p.top;
  if (p.kind == ML_TABLE) {
    const int32_t* row = p.table + static_cast<long long>(min(max(p.ids[t], 0), p.vocab - 1)) * p.top;
    if (lane < p.top) {
      idx[lane] = row[lane];
      wts[lane] = 1.f / p.top;
    }
    return;
  }
  float mx = -INFINITY, sum = 0.f;
  if (p.kind == ML_SOFTMAX_ALL) {
    for (int e = lane; e < E; e += 32) mx = fmaxf(mx, z[e]);
    mx = warp_max(mx);
    for (int e = lane; e < E; e += 32) sum += expf(z[e] - mx);
    sum = warp_sum(sum);
  }
  for (int e = lane; e < E; e += 32) {
    float v = z[e];
    if (p.kind == ML_SIGMOID) {
      z[e] = 1.f / (1.f + expf(-v));
      v = z[e] + (p.bias ? p.bias[e] : 0.f);
    }
    keys[e] = ml_key(v);                             // (softmax scores rank as their logits do)
  }
  __syncwarp();
  if (p.groups > 1 && p.keep < p.groups) {
    const int size = E / p.groups;
    for (int g = lane; g < p.groups; g += 32) {
      uint32_t a = 0u, b = 0u;                       // the two largest of the group
      int ia = g * size, ib = g * size;
      for (int e = g * size; e < (g + 1) * size; ++e) {
        const uint32_t k = keys[e];
        if (k > a) { b = a; ib = ia; a = k; ia = e; }
        else if (k > b) { b = k; ib = e; }
      }
      if (p.kind == ML_SIGMOID && size > 1) a = ml_key(z[ia] + (p.bias ? p.bias[ia] : 0.f) + (z[ib] + (p.bias ? p.bias[ib] : 0.f)));
      gkeys[g] = a;
    }
    __syncwarp();
    for (int c = 0; c < p.keep; ++c) {
      const int g = ml_argmax(gkeys, p.groups, lane);
      __syncwarp();
      if (lane == 0) gkeys[g] = 0u;                  // 0: kept (no score's key is 0)
      __syncwarp();
    }
    for (int e = lane; e < E; e += 32)
      if (gkeys[e / size] != 0u) keys[e] = 0u;
    __syncwarp();
  }
  float first = 0.f, denom = 0.f, my = 0.f;
  for (int c = 0; c < p.top; ++c) {
    const int e = ml_argmax(keys, E, lane);
    const float v = z[e];
    __syncwarp();
    if (lane == 0) {
      keys[e] = 0u;
      idx[c] = e;
    }
    if (c == 0) first = v;
    const float s = p.kind == ML_SOFTMAX ? expf(v - first) : p.kind == ML_SOFTMAX_ALL ? expf(v - mx) : v;
    denom += s;
    if (lane == c) my = s;                           // (top <= 32)
    __syncwarp();
  }
  if (lane < p.top) wts[lane] = my / (p.kind == ML_SOFTMAX_ALL ? sum : p.kind == ML_SIGMOID ? denom + 1e-20f : denom);
}

// The step's rows by expert, built by every block for itself (at most 64 x 32 pairs): `active` lists the experts that have rows, the shared one (number E) last.
// Shared memory: counts and sums of the warps [20], idx[P], weight[P], row[P + T] (place of a pair's activations), off[E + 2], active[E + 2], cur[E].
constexpr int ML_PLAN_HEAD = 20;
__host__ __device__ inline int ml_plan_words(int T, int E, int top) { return ML_PLAN_HEAD + 3 * T * top + T + 3 * E + 4; }
struct MoePlanView {
  int *n_active, *scan, *idx, *off, *active, *row, *cur;
  float* w;
};
__device__ __forceinline__ MoePlanView ml_view(int* s, int T, int E, int top) {
  MoePlanView v;
  const int P = T * top;
  v.n_active = s;
  v.scan = s + 4;
  s += ML_PLAN_HEAD;
  v.idx = s;
  v.w = reinterpret_cast<float*>(s + P);
  v.row = s + 2 * P;
  v.off = v.row + P + T;
  v.active = v.off + E + 2;
  v.cur = v.active + E + 2;
  return v;
}

__device__ __forceinline__ void ml_build(const MoePlanView& v, const MoeLayerParams& p) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, P = p.T * p.top;
  for (int e = tid; e < p.E; e += ML_THREADS) v.cur[e] = 0;
  for (int i = tid; i < P; i += ML_THREADS) {
    const int e = p.idx[i];
    v.idx[i] = e >= 0 && e < p.E ? e : -1;
    v.w[i] = p.wts[i];
  }
  __syncthreads();
  // an expert named twice for a row: the first place takes both weights.  (Found first, written behind a barrier: others still compare.)
  int keep[(ML_MAX_ROWS * ML_MAX_TOP) / ML_THREADS];
  float weight[(ML_MAX_ROWS * ML_MAX_TOP) / ML_THREADS];
#pragma unroll
  for (int k = 0; k < (ML_MAX_ROWS * ML_MAX_TOP) / ML_THREADS; ++k) {
    const int i = tid + k * ML_THREADS;
    keep[k] = -1;
    if (i >= P) continue;
    const int t = i / p.top, c = i - t * p.top, e = v.idx[i];
    bool first = e >= 0;
    float w = v.w[i];
    for (int j = 0; j < p.top; ++j)
      if (j != c && v.idx[t * p.top + j] == e) {
        if (j < c) first = false;
        else w += v.w[t * p.top + j];
      }
    if (first) {
      keep[k] = e;
      weight[k] = w;
      atomicAdd(&v.cur[e], 1);
    }
  }
  __syncthreads();
  // places of the experts' rows, and the list of those that have any: four neighbouring experts a thread
  int n[4], rows = 0, some = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int e = tid * 4 + k;
    n[k] = e < p.E ? v.cur[e] : 0;
    rows += n[k];
    some += n[k] > 0;
  }
  int r = rows, m = some;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int rr = __shfl_up_sync(0xffffffffu, r, o), mm = __shfl_up_sync(0xffffffffu, m, o);
    if (lane >= o) { r += rr; m += mm; }
  }
  if (lane == 31) { v.scan[warp] = r; v.scan[ML_WARPS + warp] = m; }
  __syncthreads();
  int r0 = r - rows, m0 = m - some, r_all = 0, m_all = 0;
#pragma unroll
  for (int q = 0; q < ML_WARPS; ++q) {
    if (q < warp) { r0 += v.scan[q]; m0 += v.scan[ML_WARPS + q]; }
    r_all += v.scan[q];
    m_all += v.scan[ML_WARPS + q];
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int e = tid * 4 + k;
    if (e < p.E) {
      v.off[e] = r0;
      v.cur[e] = r0;
      if (n[k] > 0) v.active[m0++] = e;
      r0 += n[k];
    }
  }
  if (tid == 0) {
    v.off[p.E] = r_all;
    v.off[p.E + 1] = r_all + (p.sff > 0 ? p.T : 0);
    if (p.sff > 0) v.active[m_all] = p.E;
    *v.n_active = m_all + (p.sff > 0 ? 1 : 0);
  }
  if (p.sff > 0 && tid < p.T) v.row[r_all + tid] = P + tid;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < (ML_MAX_ROWS * ML_MAX_TOP) / ML_THREADS; ++k)
    if (keep[k] >= 0) {
      const int i = tid + k * ML_THREADS;
      v.row[atomicAdd(&v.cur[keep[k]], 1)] = i;
      v.w[i] = weight[k];
    }
  __syncthreads();
}

__device__ __forceinline__ float ml_gelu_tanh(float x) { return 0.5f * x * (1.f + tanhf(0.7978845608028654f * (x + 0.044715f * x * x * x))); }
__device__ __forceinline__ float ml_act(int kind, float g, float u, float limit, float slope) {
  switch (kind) {
    case ML_SILU_GLU: return g / (1.f + expf(-g)) * u;
    case ML_CLAMPED_GLU: {
      g = g > limit ? limit : g;             // (comparisons, so that NaN stays NaN)
      u = u > limit ? limit : u < -limit ? -limit : u;
      return g / (1.f + expf(-slope * g)) * (u + 1.f);
    }
    case ML_RELU2: {
      const float v = u < 0.f ? 0.f : u;
      return v * v;
    }
    case ML_GELU: return 0.5f * u * (1.f + erff(u * 0.70710678118654752f));
    default: return ml_gelu_tanh(u);
  }
}

// ---- gate | up ------------------------------------------------------------------------------------------------------------------
// NT column tiles of 8 rows a pass over the weights (an expert with more rows takes further passes, its weights from L2 then).
template <int NT, bool GATED>
__global__ void __launch_bounds__(ML_THREADS) moe_up_kernel(const MoeLayerParams p) {
  extern __shared__ __align__(16) int smem[];
  constexpr int LD = NT * 8 + (NT > 1 ? 8 : 0);
  float* red = reinterpret_cast<float*>(smem);           // [8 warps][32][LD]
  const MoePlanView v = ml_view(smem + ML_WARPS * 32 * LD, p.T, p.E, p.top);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  pdl_sync();
  ml_build(v, p);
  const int P = p.T * p.top, n_active = *v.n_active;
  const int routed = p.sff > 0 ? n_active - 1 : n_active;
  const int items = routed * p.up_units + p.shared_units;
  // the four rows of weights that a lane takes of every k block: gate g, up g, gate g + 8, up g + 8 of 16 | 16 rows, or four of 32 plain ones
  for (int it = blockIdx.x; it < items; it += gridDim.x) {
    const int a = it < routed * p.up_units ? it / p.up_units : routed, unit = it - a * p.up_units, e = v.active[a];
    const int row0 = unit * 32, tile = row0 / p.up_rows, r0 = row0 - tile * p.up_rows;
    const uint8_t* wb = p.up + e * p.expert_bytes + (static_cast<long long>(tile) * p.kb * p.up_rows + r0) * 128;
    const int first = v.off[e], n = v.off[e + 1] - first;
    for (int n0 = 0; n0 < n; n0 += NT * 8) {
      const __nv_bfloat16* hr[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int c = n0 + j * 8 + g;
        hr[j] = nullptr;
        if (c < n) {
          const int pr = v.row[first + c], t = pr < P ? pr / p.top : pr - P;
          hr[j] = p.h + t * p.ldh;
        }
      }
      float acc[2][NT][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[i][j][c] = 0.f;
#pragma unroll 2
      for (int kb = warp; kb < p.kb; kb += ML_WARPS) {
        const uint8_t* wk = wb + static_cast<long long>(kb) * p.up_rows * 128;
        uint4 w[4][2];
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int s = 0; s < 2; ++s) w[q][s] = ldg_stream(wk + (q * 8 + g) * 128 + (((s * 4 + t4) ^ g) << 4));
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          if (j > 0 && n0 + j * 8 >= n) break;
          uint4 x[2];
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const int k = kb * 64 + (s * 4 + t4) * 8;
            x[s] = hr[j] && k < p.W ? *reinterpret_cast<const uint4*>(hr[j] + k) : make_uint4(0u, 0u, 0u, 0u);
          }
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              // gated: rows 0-7 gate, 8-15 of the tile their up rows; the packed order has 16 gate rows, then their 16 up rows
              const uint4 lo = w[GATED ? i : 2 * i][s], hi = w[GATED ? i + 2 : 2 * i + 1][s];
              mma_bf16(acc[i][j], lo.x, hi.x, lo.y, hi.y, x[s].x, x[s].y);
              mma_bf16(acc[i][j], lo.z, hi.z, lo.w, hi.w, x[s].z, x[s].w);
            }
        }
      }
      __syncthreads();                   // (the sums of the item before have been read)
      float* mine = red + warp * 32 * LD;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          *reinterpret_cast<float2*>(mine + (i * 16 + g) * LD + j * 8 + t4 * 2) = make_float2(acc[i][j][0], acc[i][j][1]);
          *reinterpret_cast<float2*>(mine + (i * 16 + g + 8) * LD + j * 8 + t4 * 2) = make_float2(acc[i][j][2], acc[i][j][3]);
        }
      __syncthreads();
      constexpr int COLS = GATED ? 16 : 32;
      const int cols = min(NT * 8, n - n0);
      for (int i = tid; i < COLS * cols; i += ML_THREADS) {
        const int col = i % COLS, c = i / COLS;
        const int r1 = GATED ? (col >> 3) * 16 + (col & 7) : col;
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int q = 0; q < ML_WARPS; ++q) {
          s1 += red[(q * 32 + r1) * LD + c];
          if (GATED) s2 += red[(q * 32 + r1 + 8) * LD + c];
        }
        const int pr = v.row[first + n0 + c];
        const float scale = pr < P ? v.w[pr] : (p.sgate ? p.sgate[pr - P] : 1.f);
        const float y = ml_act(p.act_kind, s1, GATED ? s2 : s1, p.limit, p.slope) * scale;
        float hi, mid, lo;
        bf16_parts(y, hi, mid, lo);
        __nv_bfloat16* o = p.act + static_cast<long long>(pr) * p.ld_act + unit * COLS + col;
        o[0] = __float2bfloat16_rn(hi);
        o[p.part_stride] = __float2bfloat16_rn(mid);
        o[2 * p.part_stride] = __float2bfloat16_rn(lo);
      }
    }
  }
}

// ---- down -------------------------------------------------------------------------------------------------------------------------
constexpr int ML_UNIT_KB = 4;            // k blocks (64 each) of an expert that a warp takes at a time
template <int NT>
__global__ void __launch_bounds__(ML_THREADS) moe_down_kernel(const MoeLayerParams p) {
  extern __shared__ __align__(16) int smem[];
  constexpr int LD = 36;                 // floats between rows of sums (32 columns)
  float* sums = reinterpret_cast<float*>(smem);          // [8 warps][T][LD]
  const MoePlanView v = ml_view(smem + ML_WARPS * p.T * LD, p.T, p.E, p.top);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int rank = blockIdx.x % p.cluster, block = blockIdx.x / p.cluster;
  // (routing and weights are older than the up kernel, whose activations are all that has to be waited for)
  ml_build(v, p);
  float* mine = sums + warp * p.T * LD;
  for (int i = lane; i < p.T * LD; i += 32) mine[i] = 0.f;
  __syncwarp();
  pdl_sync();
  const int P = p.T * p.top, n_active = *v.n_active;
  const int col0 = block * 32, tile = col0 >> 7;
  const uint8_t* wt = p.down + static_cast<long long>(tile) * p.down_kb * 16384 + (col0 & 127) * 128;
  const int per = (p.ff / 64 + ML_UNIT_KB - 1) / ML_UNIT_KB, per_shared = (p.sff / 64 + ML_UNIT_KB - 1) / ML_UNIT_KB;
  const int routed = p.sff > 0 ? n_active - 1 : n_active, units = routed * per + per_shared;
  for (int u = rank * ML_WARPS + warp; u < units; u += p.cluster * ML_WARPS) {
    const int a = u < routed * per ? u / per : routed, piece = u - a * per, e = v.active[a];
    const int kbs = (e < p.E ? p.ff : p.sff) / 64, k0 = piece * ML_UNIT_KB, k1 = min(kbs, k0 + ML_UNIT_KB);
    const uint8_t* wb = wt + static_cast<long long>(e) * (p.ff / 64) * 16384;
    const int first = v.off[e], n = v.off[e + 1] - first;
    for (int n0 = 0; n0 < n; n0 += NT * 8) {
      const __nv_bfloat16* ar[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int c = n0 + j * 8 + g;
        ar[j] = c < n ? p.act + static_cast<long long>(v.row[first + c]) * p.ld_act + t4 * 8 : nullptr;
      }
      float acc[2][NT][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[i][j][c] = 0.f;
#pragma unroll 2
      for (int kb = k0; kb < k1; ++kb) {
        const uint8_t* wk = wb + static_cast<long long>(kb) * 16384;
        uint4 w[4][2];
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int s = 0; s < 2; ++s) w[q][s] = ldg_stream(wk + (q * 8 + g) * 128 + (((s * 4 + t4) ^ g) << 4));
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          if (j > 0 && n0 + j * 8 >= n) break;
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int part = 0; part < 3; ++part) {
              const uint4 x = ar[j] ? *reinterpret_cast<const uint4*>(ar[j] + part * p.part_stride + kb * 64 + s * 32) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const uint4 lo = w[2 * i][s], hi = w[2 * i + 1][s];
                mma_bf16(acc[i][j], lo.x, hi.x, lo.y, hi.y, x.x, x.y);
                mma_bf16(acc[i][j], lo.z, hi.z, lo.w, hi.w, x.z, x.w);
              }
            }
        }
      }
      // (a row occurs once among an expert's, so no two lanes add to the same place)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int c = n0 + j * 8 + t4 * 2 + h;
          if (c < n) {
            const int pr = v.row[first + c], t = pr < P ? pr / p.top : pr - P;
            float* s = mine + t * LD + g;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              s[i * 16] += acc[i][j][h];
              s[i * 16 + 8] += acc[i][j][2 + h];
            }
          }
        }
      __syncwarp();
    }
  }
  __syncthreads();
  // the warps' sums, then the cluster's: each block adds up its share of the rows
  for (int i = tid; i < p.T * 32; i += ML_THREADS) {
    const int t = i >> 5, c = i & 31;
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < ML_WARPS; ++q) s += sums[(q * p.T + t) * LD + c];
    if (p.cluster > 1) sums[t * LD + c] = s;             // (warp 0's place; read before by this thread alone)
    else if (col0 + c < p.W) p.y[t * p.ldy + col0 + c] = s;
  }
  if (p.cluster > 1) {
    cluster_sync_all();
    for (int i = rank * ML_THREADS + tid; i < p.T * 32; i += p.cluster * ML_THREADS) {
      const int t = i >> 5, c = i & 31;
      float s = 0.f;
      for (int q = 0; q < p.cluster; ++q) s += ld_dsmem_f32(sums + t * LD + c, q);
      if (col0 + c < p.W) p.y[t * p.ldy + col0 + c] = s;
    }
    cluster_sync_all();                  // (nobody leaves while others read its sums)
  }
}

static size_t ml_act_elems(int T, int top, int ff, int sff) { return static_cast<size_t>(T) * (top + 1) * (ff > sff ? ff : sff); }

}  // namespace vb

using namespace vb;

extern "C" {

int vb_moe_layer_max_rows(void) { return ML_MAX_ROWS; }

size_t vb_moe_layer_workspace_bytes(int T, int top, int ff, int sff) {
  if (T < 1 || top < 1 || ff < 1 || sff < 0) return 0;
  return 3 * ml_act_elems(T, top, ff, sff) * sizeof(__nv_bfloat16);
}

int vb_moe_layer_route(int32_t* d_idx, float* d_wts, float* d_shared_gate, int kind, const void* d_h, long long ldh, const float* d_router_w, const float* d_bias,
                       const float* d_shared_gate_w, const int32_t* d_ids, const int32_t* d_table, int T, int W, int experts, int top, int groups, int keep,
                       int vocab, void* stream) {
  VB_CHECK_ARG(kind >= 0 && kind <= 3, "vb_moe_layer_route: kind %d", kind);
  VB_CHECK_ARG(d_idx && d_wts && d_h && (kind == ML_TABLE ? d_ids && d_table && vocab > 0 : d_router_w != nullptr), "vb_moe_layer_route: null pointer");
  VB_CHECK_ARG(experts >= 1 && experts <= ML_MAX_EXPERTS && top >= 1 && top <= ML_MAX_TOP && top <= experts, "vb_moe_layer_route: %d experts (1 to %d), top %d (1 to %d)",
               experts, ML_MAX_EXPERTS, top, ML_MAX_TOP);
  VB_CHECK_ARG(W >= 8 && W % 8 == 0 && ldh % 8 == 0 && ldh >= W && reinterpret_cast<uintptr_t>(d_h) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(d_router_w) % 16 == 0 && reinterpret_cast<uintptr_t>(d_shared_gate_w) % 16 == 0,
               "vb_moe_layer_route: rows must be multiples of 8 elements, 16-byte aligned (width %d)", W);
  VB_CHECK_ARG(groups <= 1 || ((kind == ML_SIGMOID || kind == ML_SOFTMAX_ALL) && experts % groups == 0 && keep >= 1 && keep <= groups && keep * (experts / groups) >= top),
               "vb_moe_layer_route: %d groups (keep %d) do not fit %d experts, top %d", groups, keep, experts, top);
  VB_CHECK_ARG(!d_shared_gate_w || d_shared_gate, "vb_moe_layer_route: the shared gate needs an output");
  VB_CHECK_ARG(T <= ML_MAX_ROWS, "vb_moe_layer_route: %d rows; at most %d", T, ML_MAX_ROWS);
  if (T <= 0) return 0;
  MoeRouteParams p = {};
  p.idx = d_idx;
  p.wts = d_wts;
  p.sgate = d_shared_gate;
  p.h = static_cast<const __nv_bfloat16*>(d_h);
  p.ldh = ldh;
  p.w = d_router_w;
  p.bias = d_bias;
  p.wsg = d_shared_gate_w;
  p.ids = d_ids;
  p.table = d_table;
  p.T = T;
  p.W = W;
  p.E = experts;
  p.top = top;
  p.kind = kind;
  p.groups = groups;
  p.keep = keep;
  p.vocab = vocab;
  const int all = (kind == ML_TABLE ? 0 : experts) + (d_shared_gate_w ? 1 : 0), per = (all + ML_ROUTE_CLUSTER - 1) / ML_ROUTE_CLUSTER;
  p.parts = per <= 1 ? 8 : per <= 2 ? 4 : per <= 4 ? 2 : 1;
  const size_t smem = (static_cast<size_t>(per) * (p.parts + 1) * ML_ROUTE_CLUSTER + 2 * static_cast<size_t>(experts) + (groups > 1 ? groups : 0)) * 4;
  VB_LAUNCH_PDL_CLUSTER(moe_layer_route_kernel, (T + ML_ROUTE_CLUSTER - 1) / ML_ROUTE_CLUSTER * ML_ROUTE_CLUSTER, ML_THREADS, smem, stream, ML_ROUTE_CLUSTER, p);
  return 0;
}

int vb_moe_layer_experts(float* d_y, long long ldy, const void* d_h, long long ldh, const void* d_up, const void* d_down, const int32_t* d_idx, const float* d_wts,
                         const float* d_shared_gate, int T, int W, int experts, int top, int ff, int shared_ff, int up_rows, int act, float limit, float slope,
                         void* d_ws, size_t ws_bytes, void* stream) {
  VB_CHECK_ARG(d_y && d_h && d_up && d_down && d_idx && d_wts && d_ws, "vb_moe_layer_experts: null pointer");
  VB_CHECK_ARG(T <= ML_MAX_ROWS, "vb_moe_layer_experts: %d rows; at most %d", T, ML_MAX_ROWS);
  VB_CHECK_ARG(experts >= 1 && experts <= ML_MAX_EXPERTS && top >= 1 && top <= ML_MAX_TOP, "vb_moe_layer_experts: %d experts (1 to %d), top %d (1 to %d)", experts,
               ML_MAX_EXPERTS, top, ML_MAX_TOP);
  VB_CHECK_ARG(W >= 8 && W % 8 == 0 && ldh % 8 == 0 && ldh >= W && ldy >= W && reinterpret_cast<uintptr_t>(d_h) % 16 == 0,
               "vb_moe_layer_experts: rows of h must be multiples of 8 elements, 16-byte aligned (width %d)", W);
  VB_CHECK_ARG(ff >= 64 && ff % 64 == 0 && shared_ff >= 0 && shared_ff % 64 == 0, "vb_moe_layer_experts: expert widths %d and %d must be multiples of 64", ff,
               shared_ff);
  VB_CHECK_ARG(act >= 0 && act <= 4 && (act != ML_CLAMPED_GLU || limit > 0.f), "vb_moe_layer_experts: activation %d, limit %f", act, limit);
  const bool gated = act <= ML_CLAMPED_GLU;
  VB_CHECK_ARG(up_rows >= 32 && up_rows <= 128 && up_rows % 32 == 0 && (gated ? 2 * ff : ff) % up_rows == 0 && (gated ? 2 * shared_ff : shared_ff) % up_rows == 0,
               "vb_moe_layer_experts: tiles of %d rows do not divide the experts", up_rows);
  VB_CHECK_ARG(!d_shared_gate || shared_ff > 0, "vb_moe_layer_experts: a gate without a shared expert");
  VB_CHECK_ARG(ws_bytes >= vb_moe_layer_workspace_bytes(T < 1 ? 1 : T, top, ff, shared_ff) && reinterpret_cast<uintptr_t>(d_ws) % 16 == 0,
               "vb_moe_layer_experts: workspace of %zu bytes is too small or not aligned", ws_bytes);
  if (T <= 0) return 0;
  MoeLayerParams p = {};
  p.h = static_cast<const __nv_bfloat16*>(d_h);
  p.ldh = ldh;
  p.up = static_cast<const uint8_t*>(d_up);
  p.down = static_cast<const uint8_t*>(d_down);
  p.idx = d_idx;
  p.wts = d_wts;
  p.sgate = d_shared_gate;
  p.act = static_cast<__nv_bfloat16*>(d_ws);
  p.y = d_y;
  p.ldy = ldy;
  p.T = T;
  p.W = W;
  p.E = experts;
  p.top = top;
  p.ff = ff;
  p.sff = shared_ff;
  p.ld_act = ff > shared_ff ? ff : shared_ff;
  p.part_stride = static_cast<long long>(ml_act_elems(T, top, ff, shared_ff));
  p.kb = (W + 63) / 64;
  p.up_rows = up_rows;
  p.expert_bytes = static_cast<long long>(gated ? 2 * ff : ff) * p.kb * 128;
  p.down_kb = (experts * ff + shared_ff) / 64;
  p.act_kind = act;
  p.limit = limit;
  p.slope = slope;
  p.up_units = (gated ? 2 * ff : ff) / 32;
  p.shared_units = (gated ? 2 * shared_ff : shared_ff) / 32;
  const int sms = sm_count(), nt = T <= 8 ? 1 : T <= 16 ? 2 : 4;
  const long long most = static_cast<long long>(experts < T * top ? experts : T * top) * p.up_units + p.shared_units;
  const int grid_up = static_cast<int>(most < 2 * sms ? most : 2 * sms);
  const size_t plan_bytes = static_cast<size_t>(ml_plan_words(T, experts, top)) * 4;
  const size_t smem_up = static_cast<size_t>(ML_WARPS) * 32 * (nt * 8 + (nt > 1 ? 8 : 0)) * 4 + plan_bytes;
#define ML_UP(NT, G)                                                              \
  do {                                                                            \
    VB_CHECK_CUDA(max_dyn_smem_once(moe_up_kernel<NT, G>));                       \
    VB_LAUNCH_PDL((moe_up_kernel<NT, G>), grid_up, ML_THREADS, smem_up, stream, p); \
  } while (0)
  if (gated) {
    if (nt == 1) ML_UP(1, true);
    else if (nt == 2) ML_UP(2, true);
    else ML_UP(4, true);
  } else {
    if (nt == 1) ML_UP(1, false);
    else if (nt == 2) ML_UP(2, false);
    else ML_UP(4, false);
  }
#undef ML_UP
  const int blocks = (W + 31) / 32;
  int cluster = 1;
  while (cluster < 8 && blocks * cluster < 2 * sms) cluster *= 2;
  p.cluster = cluster;
  const size_t smem_down = static_cast<size_t>(ML_WARPS) * T * 36 * 4 + plan_bytes;
#define ML_DOWN(NT)                                                                                                 \
  do {                                                                                                              \
    VB_CHECK_CUDA(max_dyn_smem_once(moe_down_kernel<NT>));                                                          \
    VB_LAUNCH_PDL_CLUSTER(moe_down_kernel<NT>, blocks * cluster, ML_THREADS, smem_down, stream, cluster, p);        \
  } while (0)
  if (nt == 1) ML_DOWN(1);
  else if (nt == 2) ML_DOWN(2);
  else ML_DOWN(4);
#undef ML_DOWN
  return 0;
}

}  // extern "C"
