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
//   down  block = 32 columns of the result x an equal share of the chosen experts' k blocks, every warp adding its products to rows of its own in
//         shared memory; up to eight blocks of a cluster divide the k blocks and add up through distributed shared memory.  No atomics: products,
//         warps and blocks are added in a fixed order
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
constexpr int ML_ROUTE_THREADS = 512;
struct MoeRouteParams {
  int32_t* idx;
  float *wts, *sgate;
  const __nv_bfloat16* h;
  long long ldh;
  const float *w, *bias, *wsg;           // [E][W], [E], [W]
  const int32_t *ids, *table;
  int T, W, E, top, kind, groups, keep, vocab;
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
// A block's rows of the matrix (its share of the experts, 16 at a time) by the cluster's rows of h: the fp32 values as three bf16 parts (exact), the k
// blocks of 32 divided by the warps.  What a warp needs first is asked for before the rows of h are there (the matrix is older than the kernel in front).
__global__ void __launch_bounds__(ML_ROUTE_THREADS) moe_layer_route_kernel(const MoeRouteParams p) {
  extern __shared__ __align__(16) int smem[];
  constexpr int WARPS = ML_ROUTE_THREADS / 32, AHEAD = 2;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int rank = blockIdx.x % ML_ROUTE_CLUSTER, t0 = blockIdx.x / ML_ROUTE_CLUSTER * ML_ROUTE_CLUSTER, rows = min(ML_ROUTE_CLUSTER, p.T - t0);
  // the matrix's rows: the experts, then the shared expert's gate; a block has every eighth
  const int E = p.kind == ML_TABLE ? 0 : p.E, all = E + (p.wsg ? 1 : 0), per = (all + ML_ROUTE_CLUSTER - 1) / ML_ROUTE_CLUSTER;
  float* part = reinterpret_cast<float*>(smem);                   // [16 warps][16 of the block's][8 rows]
  float* mine = part + WARPS * 16 * ML_ROUTE_CLUSTER;             // [per][8]: this block's logits
  float* z = mine + per * ML_ROUTE_CLUSTER;                       // [E] the row's logits, then its scores
  uint32_t* keys = reinterpret_cast<uint32_t*>(z + p.E);          // [E]
  uint32_t* gkeys = keys + p.E;                                   // [groups]
  const int kbs = (p.W + 31) / 32;
  float4 w[AHEAD][2][2];                                          // two rows, eight values each
  auto take = [&](int u, int i0, int kb) {
    const int k = kb * 32 + t4 * 8;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int e = (i0 + g + h * 8) * ML_ROUTE_CLUSTER + rank;
      const bool in = e < all && i0 + g + h * 8 < per && k < p.W;
      const float* r = (e < E ? p.w + static_cast<long long>(e) * p.W : p.wsg) + k;
      w[u][h][0] = in ? __ldg(reinterpret_cast<const float4*>(r)) : make_float4(0.f, 0.f, 0.f, 0.f);
      w[u][h][1] = in ? __ldg(reinterpret_cast<const float4*>(r + 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  if (per > 0)
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) take(u, 0, warp + u * WARPS);
  pdl_sync();
  const __nv_bfloat16* hr = p.h + (t0 + min(g, rows - 1)) * p.ldh;
  for (int i0 = 0; i0 < per; i0 += 16) {
    float acc[4] = {};
    for (int kb0 = warp; kb0 < kbs; kb0 += AHEAD * WARPS) {
      uint4 x[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int kb = kb0 + u * WARPS, k = kb * 32 + t4 * 8;
        if (i0 > 0 || kb0 != warp) take(u, i0, kb);
        x[u] = k < p.W ? *reinterpret_cast<const uint4*>(hr + k) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          float v[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) { v[h][0] = w[u][h][s].x; v[h][1] = w[u][h][s].y; v[h][2] = w[u][h][s].z; v[h][3] = w[u][h][s].w; }
          uint32_t f[3][4];              // part, {row g, row g + 8} x {first pair, second pair}
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float h0, m0, l0, h1, m1, l1;
            bf16_parts(v[q & 1][(q >> 1) * 2], h0, m0, l0);
            bf16_parts(v[q & 1][(q >> 1) * 2 + 1], h1, m1, l1);
            f[0][q] = pack_cut(h0, h1);
            f[1][q] = pack_cut(m0, m1);
            f[2][q] = pack_cut(l0, l1);
          }
#pragma unroll
          for (int q = 0; q < 3; ++q) mma_bf16(acc, f[q][0], f[q][1], f[q][2], f[q][3], s ? x[u].z : x[u].x, s ? x[u].w : x[u].y);
        }
    }
    float* o = part + warp * 16 * ML_ROUTE_CLUSTER;
    *reinterpret_cast<float2*>(o + g * ML_ROUTE_CLUSTER + t4 * 2) = make_float2(acc[0], acc[1]);
    *reinterpret_cast<float2*>(o + (g + 8) * ML_ROUTE_CLUSTER + t4 * 2) = make_float2(acc[2], acc[3]);
    __syncthreads();
    if (tid < 16 * ML_ROUTE_CLUSTER && i0 + tid / ML_ROUTE_CLUSTER < per) {
      float v = 0.f;
#pragma unroll
      for (int q = 0; q < WARPS; ++q) v += part[q * 16 * ML_ROUTE_CLUSTER + tid];
      mine[i0 * ML_ROUTE_CLUSTER + tid] = v;                      // (rows behind the last repeat it; nobody asks for them)
    }
    __syncthreads();
  }
  cluster_sync_all();
  const bool has = rank < rows;
  if (has) {
    for (int e = tid; e < E; e += ML_ROUTE_THREADS) {
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

// ROUNDS: pairs a thread looks after (a step of 8 rows has at most one a thread)
template <int ROUNDS>
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
  int keep[ROUNDS];
  float weight[ROUNDS];
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
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
  for (int k = 0; k < ROUNDS; ++k)
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
// All loads of a k block come before its first product.  A column tile's unused columns repeat the first row (a product's columns do not touch one another).
template <int NT>
__device__ __forceinline__ void ml_up_product(float (&acc)[2][NT][4], const uint8_t* wb, const __nv_bfloat16* const (&hr)[NT], int k0, int step,
                                              const MoeLayerParams& p, int g, int t4) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[i][j][c] = 0.f;
#pragma unroll 1
  for (int kb = k0; kb < p.kb; kb += step) {
    const uint8_t* wk = wb + static_cast<long long>(kb) * p.up_rows * 128;
    uint4 w[4][2], x[NT][2];
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int s = 0; s < 2; ++s) w[q][s] = ldg_stream(wk + (q * 8 + g) * 128 + (((s * 4 + t4) ^ g) << 4));
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int k = kb * 64 + (s * 4 + t4) * 8;
        x[j][s] = k < p.W ? *reinterpret_cast<const uint4*>(hr[j] + k) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 lo = w[i][s], hi = w[i + 2][s];
          mma_bf16(acc[i][j], lo.x, hi.x, lo.y, hi.y, x[j][s].x, x[j][s].y);
          mma_bf16(acc[i][j], lo.z, hi.z, lo.w, hi.w, x[j][s].z, x[j][s].w);
        }
  }
}
// one activation, times its row's routing weight, as parts
__device__ __forceinline__ void ml_store(const MoeLayerParams& p, const MoePlanView& v, int place, int col, float g, float u) {
  const int P = p.T * p.top, pr = v.row[place];
  const float scale = pr < P ? v.w[pr] : (p.sgate ? p.sgate[pr - P] : 1.f);
  float hi, mid, lo;
  bf16_parts(ml_act(p.act_kind, g, u, p.limit, p.slope) * scale, hi, mid, lo);
  __nv_bfloat16* o = p.act + static_cast<long long>(pr) * p.ld_act + col;
  o[0] = __float2bfloat16_rn(hi);
  o[p.part_stride] = __float2bfloat16_rn(mid);
  o[2 * p.part_stride] = __float2bfloat16_rn(lo);
}
template <int NT>
__device__ __forceinline__ void ml_rows(const __nv_bfloat16* (&r)[NT], const __nv_bfloat16* base, long long ld, const MoePlanView& v, int first, int cols, int g, int P,
                                        int top, bool by_row) {
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int c = j * 8 + g, pr = v.row[first + (c < cols ? c : 0)];
    r[j] = base + (by_row ? (pr < P ? pr / top : pr - P) : pr) * ld;
  }
}
// sums of one pass over an item: complete in the lanes (share 1), or parts of them that `share` warps leave in shared memory
template <int NT, int LD, bool GATED>
__device__ __forceinline__ void ml_up_pass(const MoeLayerParams& p, const MoePlanView& v, const uint8_t* wb, float* mine, int first, int cols, int unit, int part,
                                           int share, int g, int t4) {
  float acc[2][NT][4];
  const __nv_bfloat16* hr[NT];
  ml_rows<NT>(hr, p.h, p.ldh, v, first, cols, g, p.T * p.top, p.top, true);
  ml_up_product<NT>(acc, wb, hr, part, share, p, g, t4);
  if (share > 1) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        *reinterpret_cast<float2*>(mine + (i * 8 + g) * LD + j * 8 + t4 * 2) = make_float2(acc[i][j][0], acc[i][j][1]);
        *reinterpret_cast<float2*>(mine + (16 + i * 8 + g) * LD + j * 8 + t4 * 2) = make_float2(acc[i][j][2], acc[i][j][3]);
      }
    return;
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = j * 8 + t4 * 2 + h;
      if (c < cols)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (GATED) ml_store(p, v, first + c, unit * 16 + i * 8 + g, acc[i][j][h], acc[i][j][2 + h]);
          else {
            ml_store(p, v, first + c, unit * 32 + i * 8 + g, 0.f, acc[i][j][h]);
            ml_store(p, v, first + c, unit * 32 + 16 + i * 8 + g, 0.f, acc[i][j][2 + h]);
          }
        }
    }
}
// An item is 32 rows of an expert's matrix.  Where the step has items for all warps a warp takes one by itself, its sums complete in its registers (a gate
// row and its up row in the same lane); where it has few, 2, 4 or 8 warps divide an item's k and meet in shared memory.
template <int NT, bool GATED>
__global__ void __launch_bounds__(ML_THREADS, NT == 1 ? 3 : 2) moe_up_kernel(const MoeLayerParams p) {
  extern __shared__ __align__(16) int smem[];
  constexpr int LD = NT * 8 + (NT > 1 ? 8 : 0);
  float* red = reinterpret_cast<float*>(smem);           // two times [8 warps][32][LD]: a round's sums are read while the next round's are made
  const MoePlanView v = ml_view(smem + 2 * ML_WARPS * 32 * LD, p.T, p.E, p.top);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  pdl_sync();
  ml_build<NT == 1 ? 8 * ML_MAX_TOP / ML_THREADS : ML_MAX_ROWS * ML_MAX_TOP / ML_THREADS>(v, p);
  const int n_active = *v.n_active, routed = p.sff > 0 ? n_active - 1 : n_active;
  const int items = routed * p.up_units + p.shared_units;
  int share = 1;                                         // warps of an item
  while (share < ML_WARPS && items * share * 2 <= static_cast<int>(gridDim.x) * ML_WARPS) share *= 2;
  const int groups = ML_WARPS / share, group = warp / share, part = warp % share;
  const int rounds = (items + groups * gridDim.x - 1) / (groups * gridDim.x);
  int turn = 0;
  for (int round = 0; round < rounds; ++round) {
    const int it = (round * groups + group) * gridDim.x + blockIdx.x;
    const bool on = it < items;
    const int a = it < routed * p.up_units ? it / p.up_units : routed, unit = it - a * p.up_units, e = on ? v.active[a] : 0;
    const int row0 = unit * 32, tile = row0 / p.up_rows, r0 = row0 - tile * p.up_rows;
    const uint8_t* wb = p.up + e * p.expert_bytes + (static_cast<long long>(tile) * p.kb * p.up_rows + r0) * 128;
    const int first = on ? v.off[e] : 0, n = on ? v.off[e + 1] - first : 0;
    int passes = (n + NT * 8 - 1) / (NT * 8);
    if (share > 1 && p.T > NT * 8) passes = __syncthreads_or(passes > 1) ? (ML_MAX_ROWS + NT * 8 - 1) / (NT * 8) : 1;      // (all groups meet in every pass)
    else if (share > 1) passes = 1;
    for (int pass = 0; pass < passes; ++pass) {
      const int n0 = pass * NT * 8, cols = n - n0;
      float* sums = red + (turn++ & 1) * ML_WARPS * 32 * LD;
      if (NT > 1 && cols > 0 && cols <= 8) ml_up_pass<1, LD, GATED>(p, v, wb, sums + warp * 32 * LD, first + n0, cols, unit, part, share, g, t4);
      else if (cols > 0) ml_up_pass<NT, LD, GATED>(p, v, wb, sums + warp * 32 * LD, first + n0, cols, unit, part, share, g, t4);
      if (share == 1) continue;
      __syncthreads();
      constexpr int COLS = GATED ? 16 : 32;
      for (int i = part * 32 + lane; i < COLS * min(NT * 8, cols); i += share * 32) {
        const int col = i % COLS, c = i / COLS;
        float s1 = 0.f, s2 = 0.f;
        for (int q = 0; q < share; ++q) {
          s1 += sums[((group * share + q) * 32 + col) * LD + c];
          if (GATED) s2 += sums[((group * share + q) * 32 + 16 + col) * LD + c];
        }
        ml_store(p, v, first + n0 + c, unit * COLS + col, s1, GATED ? s2 : s1);
      }
    }
  }
}

// ---- down -------------------------------------------------------------------------------------------------------------------------
// Products of one expert's k blocks k0 .. k1 - 1 with NT column tiles, added to the warp's rows of sums.  All loads of a k block come before its first product.
constexpr int ML_LD = 36;                // floats between rows of sums (32 columns)
template <int NT>
__device__ __forceinline__ void ml_down_pass(const MoeLayerParams& p, const MoePlanView& v, const uint8_t* wb, float* mine, int first, int cols, int k0, int k1, int g,
                                             int t4) {
  const int P = p.T * p.top;
  const __nv_bfloat16* ar[NT];
  ml_rows<NT>(ar, p.act + t4 * 8, p.ld_act, v, first, cols, g, P, p.top, false);
  float acc[2][NT][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[i][j][c] = 0.f;
#pragma unroll 1
  for (int kb = k0; kb < k1; ++kb) {
    const uint8_t* wk = wb + static_cast<long long>(kb) * 16384;
    uint4 w[4][2];
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int s = 0; s < 2; ++s) w[q][s] = ldg_stream(wk + (q * 8 + g) * 128 + (((s * 4 + t4) ^ g) << 4));
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      uint4 x[3][2];
#pragma unroll
      for (int part = 0; part < 3; ++part)
#pragma unroll
        for (int s = 0; s < 2; ++s) x[part][s] = *reinterpret_cast<const uint4*>(ar[j] + part * p.part_stride + kb * 64 + s * 32);
#pragma unroll
      for (int part = 0; part < 3; ++part)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint4 lo = w[2 * i][s], hi = w[2 * i + 1][s];
            mma_bf16(acc[i][j], lo.x, hi.x, lo.y, hi.y, x[part][s].x, x[part][s].y);
            mma_bf16(acc[i][j], lo.z, hi.z, lo.w, hi.w, x[part][s].z, x[part][s].w);
          }
    }
  }
  // (a row occurs once among an expert's, so no two lanes add to the same place)
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = j * 8 + t4 * 2 + h;
      if (c < cols) {
        const int pr = v.row[first + c], t = pr < P ? pr / p.top : pr - P;
        float* s = mine + t * ML_LD + g;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          s[i * 16] += acc[i][j][h];
          s[i * 16 + 8] += acc[i][j][2 + h];
        }
      }
    }
  __syncwarp();
}
// The k blocks of all chosen experts stand in one line, of which every warp of the cluster takes an equal part.
template <int NT>
__global__ void __launch_bounds__(ML_THREADS, NT == 1 ? 3 : 2) moe_down_kernel(const MoeLayerParams p) {
  extern __shared__ __align__(16) int smem[];
  constexpr int LD = ML_LD;
  float* sums = reinterpret_cast<float*>(smem);          // [8 warps][T][LD]
  const MoePlanView v = ml_view(smem + ML_WARPS * p.T * LD, p.T, p.E, p.top);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int rank = blockIdx.x % p.cluster, block = blockIdx.x / p.cluster;
  // (routing and weights are older than the up kernel, whose activations are all that has to be waited for)
  ml_build<NT == 1 ? 8 * ML_MAX_TOP / ML_THREADS : ML_MAX_ROWS * ML_MAX_TOP / ML_THREADS>(v, p);
  float* mine = sums + warp * p.T * LD;
  for (int i = lane; i < p.T * LD; i += 32) mine[i] = 0.f;
  __syncwarp();
  pdl_sync();
  const int n_active = *v.n_active;
  const int col0 = block * 32, tile = col0 >> 7;
  const uint8_t* wt = p.down + static_cast<long long>(tile) * p.down_kb * 16384 + (col0 & 127) * 128;
  const int fkb = p.ff / 64, routed = p.sff > 0 ? n_active - 1 : n_active, line = routed * fkb + p.sff / 64;
  const int share = rank * ML_WARPS + warp, shares = p.cluster * ML_WARPS;
  const int end = static_cast<int>(static_cast<long long>(line) * (share + 1) / shares);
  for (int at = static_cast<int>(static_cast<long long>(line) * share / shares); at < end;) {
    const int a = at < routed * fkb ? at / fkb : routed, e = v.active[a], k0 = at - a * fkb, k1 = min(e < p.E ? fkb : p.sff / 64, k0 + end - at);
    const uint8_t* wb = wt + static_cast<long long>(e) * fkb * 16384;
    const int first = v.off[e], n = v.off[e + 1] - first;
    for (int n0 = 0; n0 < n; n0 += NT * 8) {
      if (NT > 1 && n - n0 <= 8) ml_down_pass<1>(p, v, wb, mine, first + n0, n - n0, k0, k1, g, t4);
      else ml_down_pass<NT>(p, v, wb, mine, first + n0, n - n0, k0, k1, g, t4);
    }
    at += k1 - k0;
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
  const size_t smem = (static_cast<size_t>(ML_ROUTE_THREADS / 32 * 16 + per) * ML_ROUTE_CLUSTER + 2 * static_cast<size_t>(experts) + (groups > 1 ? groups : 0)) * 4;
  VB_LAUNCH_PDL_CLUSTER(moe_layer_route_kernel, (T + ML_ROUTE_CLUSTER - 1) / ML_ROUTE_CLUSTER * ML_ROUTE_CLUSTER, ML_ROUTE_THREADS, smem, stream, ML_ROUTE_CLUSTER, p);
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
  // column tiles a pass: by the rows an expert has on average, so that most experts are read once
  const int sms = sm_count(), nt = T <= 8 ? 1 : T <= 16 || T * top <= 8 * experts ? 2 : 4;
  const long long most = static_cast<long long>(experts < T * top ? experts : T * top) * p.up_units + p.shared_units;
  const int fit = (nt == 1 ? 3 : 2) * sms, grid_up = static_cast<int>(most < fit ? most : fit);
  const size_t plan_bytes = static_cast<size_t>(ml_plan_words(T, experts, top)) * 4;
  const size_t smem_up = static_cast<size_t>(2 * ML_WARPS) * 32 * (nt * 8 + (nt > 1 ? 8 : 0)) * 4 + plan_bytes;
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
  int cluster = 1;                       // one wave
  while (cluster < 8 && blocks * cluster * 2 <= fit) cluster *= 2;
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
