// The experts of a mixture for the rows of a decode step (at most 64), reading the matrices of the chosen experts only:
//
//   y[t] = sum_c w[t, c] down_e(act(gate_e h_t, up_e h_t)) + sg[t] down_s(act(gate_s h_t, up_s h_t)),   e = idx[t, c]
//
// Two launches behind the router's.  A stream of weights: 3 x ff x W values for every expert that any row chose, a few
// rows each, so the kernels are built around loads that never pause.  Weights go from the packed tiles (vb_pack_weight_tiles; the same buffers that the
// projections of larger steps multiply) by bulk copies into a ring of each warp's own in shared memory, and from there, 16 bytes a lane, into the registers
// that it multiplies; a lane takes whole 16-byte chunks of 8 k, and since a product's k may stand in any order as long as both operands agree, the rows of h are
// taken by the same chunks.
//
// Units of work (32 rows of an expert's gate | up matrix, 64 k of its down matrix) stand in one line, the active experts one behind the other, each as long as its
// columns make it; blocks and warps take equal parts of the line.  Which experts the step chose therefore decides where a row's sums are cut: its last bits depend on
// the step's other rows (the same step gives the same bits).
//
//   route eight blocks of a cluster share the experts' logits of eight rows (the router's fp32 matrix is read once per eight rows), then a block each picks
//         one row's experts from all of them
//   up    a block takes a part of the line; the eight warps divide the k of a unit (16 gated or 32 plain columns), their sums meet in shared memory, the
//         activation times the routing weight leaves as three bf16 parts (exact, rowmma.cuh), so nothing is rounded between the two products
//         (the matrix units cut a sum off instead of rounding it: they add up a k block of 64, ordinary additions the k blocks)
//   down  block = 32 columns of the result; the warps of up to eight blocks of a cluster take a part of the line each, every warp adding its products to rows of
//         its own in shared memory, and the blocks add up through distributed shared memory.  No atomics: products, warps and blocks are added in a fixed order
//
// What bounds it: HBM at 64 rows (8 of 128 experts of 2048 x 768: 1.2 GB in 191 us, 6.3 TB/s), below that starts (three of 2 to 3 us) and blocks that end in whole units (8 rows, 6 of
// 64 experts of 2048 x 1024: 86 us for 440 MB; gate and up 5.6 TB/s, down 4.1; one row, 2 of 8 experts and the shared one of 1024 x 1024: 16 us for 19 MB).
//
// A table that names an expert twice for a row counts it once with both weights; an index that is no expert counts as none.
#include "../../include/vb_api.h"
#define VB_PDL_FAMILY 4
#include "rowmma.cuh"

#include <type_traits>

namespace vb {

constexpr int ML_MAX_ROWS = 64, ML_MAX_EXPERTS = 1024, ML_MAX_TOP = 32, ML_THREADS = 256, ML_WARPS = 8;
enum MlAct { ML_SILU_GLU = 0, ML_CLAMPED_GLU = 1, ML_RELU2 = 2, ML_GELU = 3, ML_GELU_TANH = 4 };

struct MoeLayerParams {
  const __nv_bfloat16* h;
  long long ldh;
  const uint8_t *up, *down;             // packed: [expert][tile][k block][rows][128 B], [tile of 128][k block of all experts][128][128 B]
  const int32_t* idx;                   // [T][top]
  const float *wts, *sgate;
  const int32_t *ids, *table;           // of a step without a router's launch (else nullptr): token ids, [vocab][top]
  const float* wsg;                     // ... and its shared expert's gate row
  int vocab;
  __nv_bfloat16* act;                   // [3 parts][T top + T][ld_act]
  float* y;
  long long ldy, expert_bytes, part_stride;
  int T, W, E, top, ff, sff, ld_act, kb, up_rows, down_kb, act_kind, up_units, shared_units, cluster;
  float limit, slope;
  unsigned char* wait_flag;
  uint32_t top_inverse;                  // 2^32 / top, rounded up
  int tile_inverse;                      // 2^16 / (units of a tile of up_rows), rounded up: exact below 2^15 units
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
__device__ __forceinline__ void st_dsmem_f32(const float* local_ptr, uint32_t cta_rank, float v) {
  uint32_t raddr;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(raddr) : "r"(smem_u32(local_ptr)), "r"(cta_rank));
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(raddr), "f"(v) : "memory");
}
// eight values of a row times eight fp32 ones
__device__ __forceinline__ float ml_dot8(const uint4& x, const float* w) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(w)), b = __ldg(reinterpret_cast<const float4*>(w + 4));
  float s = bf16_lo(x.x) * a.x;
  s = fmaf(bf16_hi(x.x), a.y, s); s = fmaf(bf16_lo(x.y), a.z, s); s = fmaf(bf16_hi(x.y), a.w, s);
  s = fmaf(bf16_lo(x.z), b.x, s); s = fmaf(bf16_hi(x.z), b.y, s); s = fmaf(bf16_lo(x.w), b.z, s);
  return fmaf(bf16_hi(x.w), b.w, s);
}
// First the logits of the cluster's eight rows: a block's share of the experts, 16 at a time, by the rows of h on the matrix units, the fp32 matrix as three
// bf16 parts (exact), the k blocks of 32 divided by the warps.  What a warp needs of the matrix first is on its way to L2 before the rows of h are there.  Every logit goes into the shared memory of the block that its row belongs to.  Then each block picks one row's experts: an
// expert's place is the number of those in front of it, which all threads count at once.
__global__ void __launch_bounds__(ML_ROUTE_THREADS) moe_layer_route_kernel(const MoeRouteParams p) {
  extern __shared__ __align__(128) int smem[];
  constexpr int THREADS = ML_ROUTE_THREADS, WARPS = THREADS / 32, AHEAD = 4;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int rank = blockIdx.x % ML_ROUTE_CLUSTER, t0 = blockIdx.x / ML_ROUTE_CLUSTER * ML_ROUTE_CLUSTER, rows = min(ML_ROUTE_CLUSTER, p.T - t0);
  const int E = p.kind == ML_TABLE ? 0 : p.E, per = (E + ML_ROUTE_CLUSTER - 1) / ML_ROUTE_CLUSTER, t = t0 + rank;
  const bool has = rank < rows;
  float* part = reinterpret_cast<float*>(smem);                   // [16 warps][16 of the block's experts][8 rows]
  float* z = part + WARPS * 16 * ML_ROUTE_CLUSTER;                // [E] the row's logits, then its scores
  uint32_t* keys = reinterpret_cast<uint32_t*>(z + p.E);          // [E]
  uint32_t* gkeys = keys + p.E;                                   // [groups]
  float* chosen = reinterpret_cast<float*>(gkeys + p.groups);     // [32]
  float* gate = chosen + 32;                                      // [16]
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");      // (every block has begun before another writes into it)
  const int kbs = (p.W + 31) / 32;
  float4 w[AHEAD][2][2];                                          // two rows, eight values each
  auto take = [&](int u, int i0, int kb) {
    const int k = kb * 32 + t4 * 8;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int e = (i0 + g + h * 8) * ML_ROUTE_CLUSTER + rank;
      const bool in = e < E && k < p.W;
      const float* r = p.w + static_cast<long long>(e) * p.W + k;
      w[u][h][0] = in ? __ldg(reinterpret_cast<const float4*>(r)) : make_float4(0.f, 0.f, 0.f, 0.f);
      w[u][h][1] = in ? __ldg(reinterpret_cast<const float4*>(r + 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  // (into L2, not into registers: the kernel in front may be the one that writes the matrix)
#pragma unroll
  for (int u = 0; u < AHEAD; ++u) {
    const int k = (warp + u * WARPS) * 32 + t4 * 8;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int e = (g + h * 8) * ML_ROUTE_CLUSTER + rank;
      if (e < E && k < p.W) asm volatile("prefetch.global.L2 [%0];" ::"l"(p.w + static_cast<long long>(e) * p.W + k));
    }
  }
  pdl_sync();
  const float my_bias = p.bias && tid < E ? __ldg(p.bias + tid) : 0.f;
  const __nv_bfloat16* hr = p.h + (t0 + min(g, rows - 1)) * p.ldh;
  if (p.wsg && has) {                                             // the shared expert's gate
    const __nv_bfloat16* hs = p.h + t * p.ldh;
    float s = 0.f;
    for (int k = tid * 8; k < p.W; k += THREADS * 8) {
      s += ml_dot8(*reinterpret_cast<const uint4*>(hs + k), p.wsg + k);
    }
    s = warp_sum(s);
    if (lane == 0) gate[warp] = s;
  }
  bool begun = false;
  for (int i0 = 0; i0 < per; i0 += 16) {
    const bool upper = per - i0 > 8;                              // (up to 64 experts: the lower half of a product's rows is not used)
    float acc[4] = {};
    for (int kb0 = warp; kb0 < kbs; kb0 += AHEAD * WARPS) {
      uint4 x[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int kb = kb0 + u * WARPS, k = kb * 32 + t4 * 8;
        take(u, i0, kb);
        x[u] = k < p.W ? *reinterpret_cast<const uint4*>(hr + k) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (kb0 + u * WARPS >= kbs) break;
        float sum[4] = {};
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          float v[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) { v[h][0] = w[u][h][s].x; v[h][1] = w[u][h][s].y; v[h][2] = w[u][h][s].z; v[h][3] = w[u][h][s].w; }
          uint32_t f[3][4];              // part, {row g, row g + 8} x {first pair, second pair}
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            f[0][q] = f[1][q] = f[2][q] = 0u;
            if ((q & 1) && !upper) continue;
            const float a = v[q & 1][(q >> 1) * 2], b = v[q & 1][(q >> 1) * 2 + 1];
            const float ra = a - bf16_cut(a), rb = b - bf16_cut(b), sa = ra - bf16_cut(ra), sb = rb - bf16_cut(rb);
            f[0][q] = pack_cut(a, b);
            f[1][q] = pack_cut(ra, rb);
            f[2][q] = pack_cut(sa, sb);
          }
#pragma unroll
          for (int q = 2; q >= 0; --q) mma_bf16(sum, f[q][0], f[q][1], f[q][2], f[q][3], s ? x[u].z : x[u].x, s ? x[u].w : x[u].y);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[c] += sum[c];
      }
    }
    if (i0 > 0) __syncthreads();                                  // (the sums before have been read)
    float* o = part + warp * 16 * ML_ROUTE_CLUSTER;
    *reinterpret_cast<float2*>(o + g * ML_ROUTE_CLUSTER + t4 * 2) = make_float2(acc[0], acc[1]);
    *reinterpret_cast<float2*>(o + (g + 8) * ML_ROUTE_CLUSTER + t4 * 2) = make_float2(acc[2], acc[3]);
    __syncthreads();
    if (!begun) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    begun = true;
    const int e = (i0 + tid / ML_ROUTE_CLUSTER) * ML_ROUTE_CLUSTER + rank, row = tid % ML_ROUTE_CLUSTER;
    if (tid < 16 * ML_ROUTE_CLUSTER && e < E && row < rows) {
      float v = 0.f;
#pragma unroll
      for (int q = 0; q < WARPS; ++q) v += part[q * 16 * ML_ROUTE_CLUSTER + tid];
      st_dsmem_f32(z + e, row, v);
    }
  }
  if (!begun) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  cluster_sync_all();
  if (!has) return;
  int32_t* idx = p.idx + t * p.top;
  float* wts = p.wts + t * p.top;
  if (p.wsg && tid == 0) {
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < WARPS; ++q) s += gate[q];
    p.sgate[t] = 1.f / (1.f + expf(-s));
  }
  if (p.kind == ML_TABLE) {
    const int32_t* row = p.table + static_cast<long long>(min(max(p.ids[t], 0), p.vocab - 1)) * p.top;
    if (tid < p.top) {
      idx[tid] = row[tid];
      wts[tid] = 1.f / p.top;
    }
    return;
  }
  if (E <= 32 && !(p.groups > 1 && p.keep < p.groups)) {
    // an expert a lane of one warp, which counts by looking at the others in turn
    if (warp != 0) return;
    const bool in = lane < E;
    const float l = in ? z[lane] : -INFINITY;
    const float logit = p.kind == ML_SOFTMAX ? l + my_bias : l, score = p.kind == ML_SIGMOID ? 1.f / (1.f + expf(-l)) : logit;
    const uint32_t key = in ? ml_key(p.kind == ML_SIGMOID ? score + my_bias : logit) : 0u;
    int before = 0;
#pragma unroll 8
    for (int o = 0; o < 32; ++o) {
      const uint32_t other = __shfl_sync(0xffffffffu, key, o);
      before += other > key || (other == key && o < lane);
    }
    const bool taken = in && before < p.top;
    float s = score;
    if (p.kind != ML_SIGMOID) {
      // (relative to the chosen ones' largest logit, or to all: the same one, unless NaN, which then reaches every weight)
      const float mx = __shfl_sync(0xffffffffu, logit, __ffs(__ballot_sync(0xffffffffu, in && before == 0)) - 1);
      s = expf(logit - mx);
    }
    const float sum = warp_sum((p.kind == ML_SOFTMAX_ALL ? in : taken) ? s : 0.f);
    if (taken) {
      idx[before] = lane;
      wts[before] = s / (p.kind == ML_SIGMOID ? sum + 1e-20f : sum);
    }
    return;
  }
  float mx = -INFINITY, sum = 0.f;
  if (p.kind == ML_SOFTMAX_ALL && warp == 0) {
    for (int e = lane; e < E; e += 32) mx = fmaxf(mx, z[e]);
    mx = warp_max(mx);
    for (int e = lane; e < E; e += 32) sum += expf(z[e] - mx);
    sum = warp_sum(sum);
  }
  for (int e = tid; e < E; e += THREADS) {
    const float bias = e == tid ? my_bias : p.bias ? p.bias[e] : 0.f;
    float v = z[e];
    if (p.kind == ML_SOFTMAX) {
      v += bias;
      z[e] = v;
    } else if (p.kind == ML_SIGMOID) {
      const float s = 1.f / (1.f + expf(-v));
      z[e] = s;
      v = s + bias;
    }
    keys[e] = ml_key(v);                             // (softmax scores rank as their logits do)
  }
  __syncthreads();
  if (p.groups > 1 && p.keep < p.groups) {
    const int size = E / p.groups;
    for (int gr = tid; gr < p.groups; gr += THREADS) {
      uint32_t a = 0u, b = 0u;                       // the two largest of the group
      int ia = gr * size, ib = gr * size;
      for (int e = gr * size; e < (gr + 1) * size; ++e) {
        const uint32_t k = keys[e];
        if (k > a) { b = a; ib = ia; a = k; ia = e; }
        else if (k > b) { b = k; ib = e; }
      }
      if (p.kind == ML_SIGMOID && size > 1) a = ml_key(z[ia] + (p.bias ? p.bias[ia] : 0.f) + (z[ib] + (p.bias ? p.bias[ib] : 0.f)));
      gkeys[gr] = a;
    }
    __syncthreads();
    for (int e = tid; e < E; e += THREADS) {
      const int mine = e / size;
      const uint32_t k = gkeys[mine];
      int before = 0;
      for (int o = 0; o < p.groups; ++o) before += gkeys[o] > k || (gkeys[o] == k && o < mine);
      if (before >= p.keep) keys[e] = 0u;            // (no score's key is 0)
    }
    __syncthreads();
  }
  // up to 32 neighbouring threads count for an expert
  int share = 1;
  while (share < 32 && 2 * share * E <= THREADS) share *= 2;
  for (int e0 = 0; e0 < E; e0 += THREADS / share) {
    const int e = e0 + tid / share, q = tid % share;
    const uint32_t k = e < E ? keys[e] : 0u;
    int before = 0;
    if (k != 0u)
      for (int o = q; o < E; o += share) {
        const uint32_t other = keys[o];
        before += other > k || (other == k && o < e);
      }
    for (int o = share >> 1; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    if (k != 0u && q == 0 && before < p.top) {
      idx[before] = e;
      chosen[before] = z[e];
    }
  }
  __syncthreads();
  if (warp != 0) return;
  float s = 0.f;
  if (lane < p.top) {                                // (top <= 32)
    s = chosen[lane];
    if (p.kind == ML_SOFTMAX) s = expf(s - chosen[0]);
    else if (p.kind == ML_SOFTMAX_ALL) s = expf(s - mx);
  }
  const float denom = warp_sum(s);
  if (lane < p.top) wts[lane] = s / (p.kind == ML_SOFTMAX_ALL ? sum : p.kind == ML_SIGMOID ? denom + 1e-20f : denom);
}

// row of a pair (no division: the step has at most 2^11 pairs)
__device__ __forceinline__ int ml_row_of(const MoeLayerParams& p, int pair) { return p.top == 1 ? pair : static_cast<int>(__umulhi(static_cast<uint32_t>(pair), p.top_inverse)); }

// The step's rows by expert, built by every block for itself (at most 64 x 32 pairs): `active` lists the experts that have rows, the shared one (number E) last.
// Shared memory: counts and sums of the warps [32], idx[P], weight[P], row[P + T] (place of a pair's activations), first[E + 2] (an active
// expert's rows among them), active[E + 2], line[E + 2], an expert's first row [E], its
// rows as bits [2 E], gates [8].
// `line`: where an active expert's work starts when all of it stands in one line (the blocks take equal parts of it); a unit of work, 32 rows of weights or a
// block of 64 k, costs what its columns take.
constexpr int ML_PLAN_HEAD = 32;
__host__ __device__ inline int ml_plan_words(int T, int E, int top) { return ML_PLAN_HEAD + 3 * T * top + T + 6 * E + 16; }
struct MoePlanView {
  int *n_active, *n_named, *scan, *idx, *first, *active, *row, *line, *place;
  uint32_t* bits;
  float *w, *gates;
};
__device__ __forceinline__ MoePlanView ml_view(int* s, int T, int E, int top) {
  MoePlanView v;
  const int P = T * top;
  v.n_active = s;
  v.n_named = s + 1;
  v.scan = s + 4;
  s += ML_PLAN_HEAD;
  v.idx = s;
  v.w = reinterpret_cast<float*>(s + P);
  v.row = s + 2 * P;
  v.first = v.row + P + T;
  v.active = v.first + E + 2;
  v.line = v.active + E + 2;
  v.place = v.line + E + 2;
  v.bits = reinterpret_cast<uint32_t*>(v.place + E);
  v.gates = reinterpret_cast<float*>(v.bits + 2 * E);
  return v;
}

// Cost of a unit with n columns, in eighths of one with up to 8 (whose weights take longer to come than to multiply); measured as the times at which blocks of
// such units end.
__device__ __forceinline__ int ml_cost(int n, bool down) { return n <= 8 ? 8 : n <= 16 ? (down ? 12 : 10) : n <= 32 ? (down ? 24 : 18) : (down ? 56 : 38); }
// what the router (or, in steps without one, the table) says of a pair: its expert (-1: none) and its weight
__device__ __forceinline__ void ml_pair(const MoeLayerParams& p, int i, int& e, float& w) {
  if (p.table) {
    const int t = ml_row_of(p, i);
    e = p.table[static_cast<long long>(min(max(p.ids[t], 0), p.vocab - 1)) * p.top + i - t * p.top];
    w = 1.f / p.top;
  } else {
    e = p.idx[i];
    w = p.wts[i];
  }
  if (e < 0 || e >= p.E) e = -1;
}
// The same for steps of at most 32 pairs, by each warp for itself: pairs of an expert find one another by their values.  (The list stands in the order of the
// pairs; 0.6 us where the other way takes 1.8.)
__device__ __forceinline__ void ml_build_few(const MoePlanView& v, const MoeLayerParams& p, int units, int shared_units, bool down) {
  const int tid = threadIdx.x, lane = tid & 31, P = p.T * p.top;
  int e = -1;
  float w = 0.f;
  if (lane < P) ml_pair(p, lane, e, w);
  const int t = ml_row_of(p, lane);
  const uint32_t all = 0xffffffffu, below = (1u << lane) - 1u;
  const uint32_t twins = __match_any_sync(all, e >= 0 ? e * 64 + t : -1 - lane);        // pairs of one row that name one expert: the first takes all weights
  if (__any_sync(all, __popc(twins) > 1)) {
    float sum = w;
    for (int j = 0; j < 32; ++j) {
      const float other = __shfl_sync(all, w, j);
      if (j != lane && (twins >> j & 1u)) sum += other;
    }
    w = sum;
  }
  const bool kept = e >= 0 && (twins & below) == 0u;
  const uint32_t group = __match_any_sync(all, kept ? e : -1 - lane);
  const bool leader = kept && (group & below) == 0u;
  const uint32_t leaders = __ballot_sync(all, leader);
  const int n = __popc(group), first = __ffs(group) - 1;
  int r = leader ? n : 0, l = leader ? ml_cost(n, down) * units : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int rr = __shfl_up_sync(all, r, o), ll = __shfl_up_sync(all, l, o);
    if (lane >= o) { r += rr; l += ll; }
  }
  const int r_all = __shfl_sync(all, r, 31), l_all = __shfl_sync(all, l, 31), m_all = __popc(leaders);
  const int r0 = __shfl_sync(all, r - n, first);                 // (a leader's own: the rows of those in front)
  if (tid < 32) {
    if (leader) {
      const int a = __popc(leaders & below);
      v.active[a] = e;
      v.first[a] = r - n;
      v.line[a] = l - ml_cost(n, down) * units;
    }
    if (kept) {
      v.row[r0 + __popc(group & below)] = lane;
      v.w[lane] = w;
    }
    if (lane == 0) {
      v.first[m_all] = r_all;
      v.line[m_all] = l_all;
      if (p.sff > 0) {
        v.first[m_all + 1] = r_all + p.T;
        v.active[m_all] = p.E;
        v.line[m_all + 1] = l_all + ml_cost(p.T, down) * shared_units;
      }
      *v.n_active = m_all + (p.sff > 0 ? 1 : 0);
    }
  }
  if (p.sff > 0 && tid < p.T) v.row[r_all + tid] = P + tid;
  __syncthreads();
}

// ROUNDS: pairs a thread looks after (a step of 8 rows has at most one a thread).  An expert's rows are collected as bits, which sorts them and counts a
// row once however often it names the expert.
template <int ROUNDS>
__device__ __forceinline__ void ml_build(const MoePlanView& v, const MoeLayerParams& p, int units, int shared_units, bool down) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, P = p.T * p.top, rounds = (P + ML_THREADS - 1) / ML_THREADS;
  if (P <= 32) {
    ml_build_few(v, p, units, shared_units, down);
    return;
  }
  int mine[ROUNDS] = {};
  float weight[ROUNDS] = {};
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    if (k >= rounds) break;
    const int i = tid + k * ML_THREADS;
    mine[k] = -1;
    weight[k] = 0.f;
    if (i < P) ml_pair(p, i, mine[k], weight[k]);
  }
  for (int e = tid; e < 2 * p.E; e += ML_THREADS) v.bits[e] = 0u;
  if (tid == 0) *v.n_named = 0;
  int named = 0;
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    if (k >= rounds) break;
    const int i = tid + k * ML_THREADS;
    if (i < P) {
      v.idx[i] = mine[k];
      v.w[i] = weight[k];
      named += mine[k] >= 0;
    }
  }
  named = __reduce_add_sync(0xffffffffu, named);
  __syncthreads();
  if (lane == 0 && named) atomicAdd(v.n_named, named);
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    if (k >= rounds) break;
    const int t = ml_row_of(p, tid + k * ML_THREADS);
    if (mine[k] >= 0) atomicOr(v.bits + 2 * mine[k] + (t >> 5), 1u << (t & 31));
  }
  __syncthreads();
  // places of the experts' rows, and the list of those that have any: four neighbouring experts a thread
  int n[4], rows = 0, some = 0, cost = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int e = tid * 4 + k;
    n[k] = e < p.E ? __popc(v.bits[2 * e]) + __popc(v.bits[2 * e + 1]) : 0;
    rows += n[k];
    some += n[k] > 0;
    cost += n[k] > 0 ? ml_cost(n[k], down) * units : 0;
  }
  int r = rows, m = some, l = cost;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int rr = __shfl_up_sync(0xffffffffu, r, o), mm = __shfl_up_sync(0xffffffffu, m, o), ll = __shfl_up_sync(0xffffffffu, l, o);
    if (lane >= o) { r += rr; m += mm; l += ll; }
  }
  if (lane == 31) { v.scan[warp] = r; v.scan[ML_WARPS + warp] = m; v.scan[2 * ML_WARPS + warp] = l; }
  __syncthreads();
  int r0 = r - rows, m0 = m - some, l0 = l - cost, r_all = 0, m_all = 0, l_all = 0;
#pragma unroll
  for (int q = 0; q < ML_WARPS; ++q) {
    if (q < warp) { r0 += v.scan[q]; m0 += v.scan[ML_WARPS + q]; l0 += v.scan[2 * ML_WARPS + q]; }
    r_all += v.scan[q];
    m_all += v.scan[ML_WARPS + q];
    l_all += v.scan[2 * ML_WARPS + q];
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int e = tid * 4 + k;
    if (e < p.E) {
      v.place[e] = r0;
      if (n[k] > 0) {
        v.first[m0] = r0;
        v.line[m0] = l0;
        v.active[m0++] = e;
        l0 += ml_cost(n[k], down) * units;
      }
      r0 += n[k];
    }
  }
  if (tid == 0) {
    v.first[m_all] = r_all;
    v.line[m_all] = l_all;
    if (p.sff > 0) {
      v.first[m_all + 1] = r_all + p.T;
      v.active[m_all] = p.E;
      v.line[m_all + 1] = l_all + ml_cost(p.T, down) * shared_units;
    }
    *v.n_active = m_all + (p.sff > 0 ? 1 : 0);
  }
  if (p.sff > 0 && tid < p.T) v.row[r_all + tid] = P + tid;
  const bool twice = *v.n_named != r_all;                // (the same in all threads) a row names an expert twice: the first place takes both weights
  if (twice) {
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k) {
      if (k >= rounds) break;
      const int i = tid + k * ML_THREADS, t = ml_row_of(p, i), c = i - t * p.top;
      if (mine[k] < 0) continue;
      const int e = mine[k];
      for (int j = 0; j < p.top; ++j)
        if (j != c && v.idx[t * p.top + j] == e) {
          if (j < c) mine[k] = -1;
          else weight[k] += v.w[t * p.top + j];
        }
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    if (k >= rounds) break;
    if (mine[k] >= 0) {
      const int i = tid + k * ML_THREADS, t = ml_row_of(p, i);
      const uint32_t b0 = v.bits[2 * mine[k]], b1 = v.bits[2 * mine[k] + 1], below = (1u << (t & 31)) - 1u;
      v.row[v.place[mine[k]] + (t < 32 ? __popc(b0 & below) : __popc(b0) + __popc(b1 & below))] = i;
      v.w[i] = weight[k];
    }
  }
  __syncthreads();
}

// A part of the line: units from (a, unit) on that start before `end`.
struct MlWalk {
  int a, unit, at, step, units;          // the active expert, its unit, where that starts, its cost, how many the expert has
  bool down;
};
__device__ __forceinline__ void ml_expert(MlWalk& w, const MoePlanView& v, int E, int units, int shared_units) {
  const int e = v.active[w.a];
  w.units = e < E ? units : shared_units;
  w.step = ml_cost(v.first[w.a + 1] - v.first[w.a], w.down);
}
__device__ __forceinline__ MlWalk ml_walk(const MoePlanView& v, int begin, int E, int units, int shared_units, bool down) {
  MlWalk w;
  w.down = down;
  int lo = 0, hi = *v.n_active;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (v.line[mid] <= begin) lo = mid;
    else hi = mid;
  }
  w.a = lo;
  ml_expert(w, v, E, units, shared_units);
  w.unit = (begin - v.line[lo] + w.step - 1) / w.step;
  w.at = v.line[lo] + w.unit * w.step;
  if (w.unit >= w.units && lo + 1 < *v.n_active) {       // (begins inside the expert's last unit)
    ++w.a;
    w.unit = 0;
    ml_expert(w, v, E, units, shared_units);
  }
  return w;
}
__device__ __forceinline__ void ml_next(MlWalk& w, const MoePlanView& v, int E, int units, int shared_units) {
  w.at += w.step;
  if (++w.unit < w.units) return;
  w.unit = 0;
  if (++w.a < *v.n_active) ml_expert(w, v, E, units, shared_units);
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

// ---- weights on their way ---------------------------------------------------------------------------------------------------------
// Every warp has a ring of its own in shared memory: places of 4 KB, a block of 64 k of 32 rows each (one run of the packed tiles), filled by bulk copies that
// its first lane asks for as soon as the warp has read a place.  What is on its way neither holds registers nor stops at the end of an item, and no
// warp waits for another's data: 96 KB an SM are always on their way (2.2 us at an SM's share of the memory's rate).
constexpr int ML_SLOT_BYTES = 4096;
__host__ __device__ constexpr int ml_ring_bytes(int slots) { return ML_WARPS * slots * (ML_SLOT_BYTES + 8); }
template <int SLOTS>
struct MlRing {
  uint8_t* slots;
  uint64_t* bars;
  int put = 0, got = 0;
  uint32_t parity = 0u;
  __device__ __forceinline__ void ask(const uint8_t* src) {              // (one lane)
    mbar_arrive_expect_tx(bars + put, ML_SLOT_BYTES);
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(slots + put * ML_SLOT_BYTES)), "l"(src),
                 "r"(ML_SLOT_BYTES), "r"(smem_u32(bars + put))
                 : "memory");
  }
  __device__ __forceinline__ void asked() { put = put + 1 == SLOTS ? 0 : put + 1; }
  __device__ __forceinline__ const uint8_t* wait(BoundedWait& bw) {
    bw.wait(bars + got, parity);
    return slots + got * ML_SLOT_BYTES;
  }
  __device__ __forceinline__ void read() {
    got = got + 1 == SLOTS ? 0 : got + 1;
    parity ^= got == 0 ? 1u : 0u;
  }
};
// a warp that gave up: the copies on their way land before the block may leave
__device__ __noinline__ void ml_land() {
  const unsigned long long t0 = gtimer();
  while (gtimer() - t0 < 2000000ull) __nanosleep(1000);
}
// shared memory of both kernels: the rings, their barriers, then the kernel's own
template <int SLOTS>
__device__ __forceinline__ MlRing<SLOTS> ml_ring(int* smem, int warp) {
  MlRing<SLOTS> r;
  r.slots = reinterpret_cast<uint8_t*>(smem) + warp * SLOTS * ML_SLOT_BYTES;
  r.bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(smem) + ML_WARPS * SLOTS * ML_SLOT_BYTES) + warp * SLOTS;
  if ((threadIdx.x & 31) == 0) {
    for (int i = 0; i < SLOTS; ++i) mbar_init(r.bars + i, 1);
    fence_barrier_init();
    fence_proxy_async();
  }
  __syncwarp();
  return r;
}
// The lane's place among 8 rows.  Lanes 0 to 7 of a 16-byte load read two rows of 128 swizzled bytes; rows four apart lie in different banks.
__device__ __forceinline__ int ml_row(int g) { return (g >> 1) | ((g & 1) << 2); }
__device__ __forceinline__ void ml_weights(uint4 (&w)[4][2], const uint8_t* slot, int r, int t4) {
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int s = 0; s < 2; ++s) w[q][s] = *reinterpret_cast<const uint4*>(slot + (q * 8 + r) * 128 + (((s * 4 + t4) ^ r) << 4));
}
// row of the step that a place of activations belongs to (the shared expert's follow the pairs')
__device__ __forceinline__ int ml_token(const MoeLayerParams& p, int place) {
  const int P = p.T * p.top;
  return place < P ? ml_row_of(p, place) : place - P;
}
// rows of a column tile: a tile's unused columns repeat the first row (a product's columns do not touch one another)
template <int NT>
__device__ __forceinline__ void ml_rows(const __nv_bfloat16* (&r)[NT], const __nv_bfloat16* base, long long ld, const MoePlanView& v, int first, int cols, int g,
                                        const MoeLayerParams& p, bool by_row) {
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int c = j * 8 + g, pr = v.row[first + (c < cols ? c : 0)];
    r[j] = base + (by_row ? ml_token(p, pr) : pr) * ld;
  }
}
// calls f with 1, 2 or 4 column tiles, as `cols` columns need and the kernel has
template <int NT, typename F>
__device__ __forceinline__ void ml_by_columns(int cols, F&& f) {
  if constexpr (NT == 1) {
    f(std::integral_constant<int, 1>());
  } else {
    if (cols <= 8) f(std::integral_constant<int, 1>());
    else if (NT == 2 || cols <= 16) f(std::integral_constant<int, 2>());
    else if constexpr (NT == 4) f(std::integral_constant<int, 4>());
  }
}

// ---- gate | up ------------------------------------------------------------------------------------------------------------------
// A unit is 32 rows of an expert's matrix (NT * 8 of the expert's rows a pass; further passes take the weights from L2), k blocks w, w + 8, .. to warp w.
struct MlUpUnit {
  const uint8_t* w;
  int first, n, passes;
};
template <int NT>
__device__ __forceinline__ MlUpUnit ml_up_unit(const MoeLayerParams& p, const MoePlanView& v, const MlWalk& at) {
  MlUpUnit m;
  const int e = v.active[at.a], tile = at.unit * p.tile_inverse >> 16, r0 = at.unit * 32 - tile * p.up_rows;
  m.w = p.up + e * p.expert_bytes + (static_cast<long long>(tile) * p.kb * p.up_rows + r0) * 128;
  m.first = v.first[at.a];
  m.n = v.first[at.a + 1] - m.first;
  m.passes = (m.n + NT * 8 - 1) / (NT * 8);
  return m;
}
// one activation, times its row's routing weight, as parts
__device__ __forceinline__ void ml_store(const MoeLayerParams& p, const MoePlanView& v, int place, int col, float g, float u) {
  const int P = p.T * p.top, pr = v.row[place];
  const float scale = pr < P ? v.w[pr] : p.wsg ? v.gates[pr - P] : p.sgate ? p.sgate[pr - P] : 1.f;
  float hi, mid, lo;
  bf16_parts(ml_act(p.act_kind, g, u, p.limit, p.slope) * scale, hi, mid, lo);
  __nv_bfloat16* o = p.act + static_cast<long long>(pr) * p.ld_act + col;
  o[0] = __float2bfloat16_rn(hi);
  o[p.part_stride] = __float2bfloat16_rn(mid);
  o[2 * p.part_stride] = __float2bfloat16_rn(lo);
}
template <int NT, bool GATED, int SLOTS>
__global__ void __launch_bounds__(ML_THREADS, NT == 1 ? 2 : 1) moe_up_kernel(const MoeLayerParams p) {
  extern __shared__ __align__(128) int smem[];
  constexpr int LD_MAX = NT * 8 + (NT > 1 ? 8 : 0);
  // two times [8 warps][32][LD_MAX]: a pass's sums are read while the next one's are made
  float* red = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(smem) + ml_ring_bytes(SLOTS));
  const MoePlanView v = ml_view(reinterpret_cast<int*>(red + 2 * ML_WARPS * 32 * LD_MAX), p.T, p.E, p.top);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3, r = ml_row(g);
  MlRing<SLOTS> ring = ml_ring<SLOTS>(smem, warp);
  BoundedWait bw{p.wait_flag};
  pdl_sync();
  ml_build<NT == 1 ? 8 * ML_MAX_TOP / ML_THREADS : ML_MAX_ROWS * ML_MAX_TOP / ML_THREADS>(v, p, p.up_units, p.shared_units, false);
  const int n_active = *v.n_active;
  if (n_active == 0) return;
  const int total = v.line[n_active], warps = min(ML_WARPS, p.kb);      // (a warp takes every eighth k block)
  const int begin = static_cast<int>(static_cast<long long>(total) * blockIdx.x / gridDim.x),
            end = static_cast<int>(static_cast<long long>(total) * (blockIdx.x + 1) / gridDim.x);
  const MlWalk start = ml_walk(v, begin, p.E, p.up_units, p.shared_units, false);
  // what is asked for next
  MlWalk ask_at = start;
  int ask_pass = 0, ask_kb = warp;
  MlUpUnit ask_m = {};
  if (warp >= warps) ask_at.at = end;
  if (ask_at.at < end) ask_m = ml_up_unit<NT>(p, v, ask_at);
  auto ask = [&]() {
    if (ask_at.at >= end) return;
    if (lane == 0 && !bw.dead) ring.ask(ask_m.w + static_cast<long long>(ask_kb) * p.up_rows * 128);
    ring.asked();
    ask_kb += ML_WARPS;
    if (ask_kb < p.kb) return;
    ask_kb = warp;
    if (++ask_pass < ask_m.passes) return;
    ask_pass = 0;
    ml_next(ask_at, v, p.E, p.up_units, p.shared_units);
    if (ask_at.at < end) ask_m = ml_up_unit<NT>(p, v, ask_at);
  };
#pragma unroll 1                         // (once a launch: its instructions have to come first)
  for (int i = 0; i < SLOTS; ++i) ask();
  if (NT == 1 && p.wsg && warp < p.T && end > v.line[n_active - 1]) {       // (the block has units of the shared expert: its rows' gates, a row a warp)
    const __nv_bfloat16* hs = p.h + warp * p.ldh;
    float s = 0.f;
#pragma unroll 8
    for (int k = lane * 8; k < p.W; k += 256) s += ml_dot8(*reinterpret_cast<const uint4*>(hs + k), p.wsg + k);
    s = warp_sum(s);
    if (lane == 0) v.gates[warp] = 1.f / (1.f + expf(-s));                   // (read behind the next barrier)
  }
  int turn = 0;
  for (MlWalk at = start; at.at < end; ml_next(at, v, p.E, p.up_units, p.shared_units)) {
    const MlUpUnit m = ml_up_unit<NT>(p, v, at);
    for (int pass = 0; pass < m.passes; ++pass, ++turn) {
      const int n0 = pass * NT * 8, cols = m.n - n0;
      float* sums = red + (turn & 1) * ML_WARPS * 32 * LD_MAX;
      ml_by_columns<NT>(cols, [&](auto tiles) {
        constexpr int N = decltype(tiles)::value, LD = N * 8 + (N > 1 ? 8 : 0);
        float acc[2][N][4] = {};
        const __nv_bfloat16* hr[N];
        ml_rows<N>(hr, p.h + t4 * 8, p.ldh, v, m.first + n0, cols, g, p, true);
        uint4 next[N][2];
        auto take = [&](int kb) {
#pragma unroll
          for (int j = 0; j < N; ++j)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              const int k = kb * 64 + s * 32;
              next[j][s] = k + t4 * 8 < p.W ? *reinterpret_cast<const uint4*>(hr[j] + k) : make_uint4(0u, 0u, 0u, 0u);
            }
        };
        take(warp);
        for (int kb = warp; kb < p.kb; kb += ML_WARPS) {
          uint4 x[N][2], w[4][2];
#pragma unroll
          for (int j = 0; j < N; ++j) { x[j][0] = next[j][0]; x[j][1] = next[j][1]; }
          take(kb + ML_WARPS);
          ml_weights(w, ring.wait(bw), r, t4);
#pragma unroll
          for (int j = 0; j < N; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float sum[4] = {};
#pragma unroll
              for (int s = 0; s < 2; ++s) {
                // gated: 16 gate rows, then their up rows; a product's upper half takes the one, its lower half the other
                const uint4 lo = w[i][s], hi = w[i + 2][s];
                mma_bf16(sum, lo.x, hi.x, lo.y, hi.y, x[j][s].x, x[j][s].y);
                mma_bf16(sum, lo.z, hi.z, lo.w, hi.w, x[j][s].z, x[j][s].w);
              }
#pragma unroll
              for (int c = 0; c < 4; ++c) acc[i][j][c] += sum[c];
            }
          __syncwarp();
          ring.read();
          ask();
        }
        if (warp < warps) {
          float* mine = sums + warp * 32 * LD;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j) {
              *reinterpret_cast<float2*>(mine + (i * 8 + r) * LD + j * 8 + t4 * 2) = make_float2(acc[i][j][0], acc[i][j][1]);
              *reinterpret_cast<float2*>(mine + (16 + i * 8 + r) * LD + j * 8 + t4 * 2) = make_float2(acc[i][j][2], acc[i][j][3]);
            }
        }
        __syncthreads();
        // (another warp begins each time: a unit of few columns is one warp's work, and the others go on)
        constexpr int COLS = GATED ? 16 : 32;
        for (int i = (tid + 32 * turn) & (ML_THREADS - 1); i < COLS * min(N * 8, cols); i += ML_THREADS) {
          const int col = i % COLS, c = i / COLS;
          float s1 = 0.f, s2 = 0.f;
          for (int q = 0; q < warps; ++q) {
            s1 += sums[(q * 32 + col) * LD + c];
            if (GATED) s2 += sums[(q * 32 + 16 + col) * LD + c];
          }
          ml_store(p, v, m.first + n0 + c, at.unit * COLS + col, s1, GATED ? s2 : s1);
        }
      });
    }
  }
  if (bw.dead) ml_land();
}

// ---- down -------------------------------------------------------------------------------------------------------------------------
// A unit is a block of 64 k of an expert; every warp of the cluster takes an equal part of the line, and what a part has of one expert is a piece.
constexpr int ML_LD = 36;                // floats between rows of sums (32 columns)
struct MlDownPiece {
  const uint8_t* w;
  int first, n, passes, k0, k1;
};
template <int NT>
__device__ __forceinline__ MlDownPiece ml_down_piece(const MoeLayerParams& p, const MoePlanView& v, const uint8_t* wt, const MlWalk& at, int end) {
  MlDownPiece m;
  const int e = v.active[at.a];
  m.k0 = at.unit;
  m.k1 = min(at.units, at.unit + (end - at.at + at.step - 1) / at.step);
  m.w = wt + static_cast<long long>(e) * (p.ff / 64) * 16384;
  m.first = v.first[at.a];
  m.n = v.first[at.a + 1] - m.first;
  m.passes = (m.n + NT * 8 - 1) / (NT * 8);
  return m;
}
// four neighbours of a row of the result (its rows may start anywhere)
__device__ __forceinline__ void ml_result(const MoeLayerParams& p, int t, int col, const float4& s) {
  float* y = p.y + t * p.ldy + col;
  if (col + 4 <= p.W && (reinterpret_cast<uintptr_t>(y) & 15) == 0) {
    *reinterpret_cast<float4*>(y) = s;
    return;
  }
  if (col < p.W) y[0] = s.x;
  if (col + 1 < p.W) y[1] = s.y;
  if (col + 2 < p.W) y[2] = s.z;
  if (col + 3 < p.W) y[3] = s.w;
}
template <int NT, int SLOTS>
__global__ void __launch_bounds__(ML_THREADS, NT <= 2 ? 2 : 1) moe_down_kernel(const MoeLayerParams p) {
  extern __shared__ __align__(128) int smem[];
  constexpr int LD = ML_LD;
  float* sums = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(smem) + ml_ring_bytes(SLOTS));          // [8 warps][T][LD]
  const MoePlanView v = ml_view(reinterpret_cast<int*>(sums + ML_WARPS * p.T * LD), p.T, p.E, p.top);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3, r = ml_row(g);
  const int rank = blockIdx.x % p.cluster, block = blockIdx.x / p.cluster;
  MlRing<SLOTS> ring = ml_ring<SLOTS>(smem, warp);
  BoundedWait bw{p.wait_flag};
  // (routing and weights are older than the up kernel, whose activations are all that has to be waited for)
  const int units = p.ff / 64, shared_units = p.sff / 64;
  ml_build<NT == 1 ? 8 * ML_MAX_TOP / ML_THREADS : ML_MAX_ROWS * ML_MAX_TOP / ML_THREADS>(v, p, units, shared_units, true);
  const int n_active = *v.n_active, total = n_active ? v.line[n_active] : 0;
  const int col0 = block * 32, tile = col0 >> 7;
  const uint8_t* wt = p.down + static_cast<long long>(tile) * p.down_kb * 16384 + (col0 & 127) * 128;
  const int share = rank * ML_WARPS + warp, shares = p.cluster * ML_WARPS;
  const int begin = static_cast<int>(static_cast<long long>(total) * share / shares), end = static_cast<int>(static_cast<long long>(total) * (share + 1) / shares);
  MlWalk start = {};
  start.at = end;
  if (begin < end) start = ml_walk(v, begin, p.E, units, shared_units, true);
  // past a piece: the walk stands at the next expert, or at the end of the part
  auto past = [&](MlWalk& w, const MlDownPiece& m) {
    w.at += (m.k1 - m.k0) * w.step;
    w.unit = m.k1;
    if (w.unit < w.units) return;
    w.unit = 0;
    if (++w.a < n_active) ml_expert(w, v, p.E, units, shared_units);
  };
  MlWalk ask_at = start;
  int ask_pass = 0, ask_kb = 0;
  MlDownPiece ask_m = {};
  if (ask_at.at < end) {
    ask_m = ml_down_piece<NT>(p, v, wt, ask_at, end);
    ask_kb = ask_m.k0;
  }
  auto ask = [&]() {
    if (ask_at.at >= end) return;
    if (lane == 0 && !bw.dead) ring.ask(ask_m.w + static_cast<long long>(ask_kb) * 16384);
    ring.asked();
    if (++ask_kb < ask_m.k1) return;
    ask_kb = ask_m.k0;
    if (++ask_pass < ask_m.passes) return;
    ask_pass = 0;
    past(ask_at, ask_m);
    if (ask_at.at < end) {
      ask_m = ml_down_piece<NT>(p, v, wt, ask_at, end);
      ask_kb = ask_m.k0;
    }
  };
#pragma unroll 1                         // (once a launch: its instructions have to come first)
  for (int i = 0; i < SLOTS; ++i) ask();
  float* mine = sums + warp * p.T * LD;
  for (int i = lane; i < p.T * (LD / 4); i += 32) reinterpret_cast<float4*>(mine)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  __syncwarp();
  pdl_sync();
  for (MlWalk at = start; at.at < end;) {
    const MlDownPiece m = ml_down_piece<NT>(p, v, wt, at, end);
    for (int pass = 0; pass < m.passes; ++pass) {
      const int n0 = pass * NT * 8, cols = m.n - n0;
      ml_by_columns<NT>(cols, [&](auto tiles) {
        constexpr int N = decltype(tiles)::value, HALF = NT == 2 ? 1 : N > 2 ? 2 : N;      // (registers: activations of one or two column tiles at a time)
        float acc[2][N][4] = {};
        const __nv_bfloat16* ar[N];
        ml_rows<N>(ar, p.act + t4 * 8, p.ld_act, v, m.first + n0, cols, g, p, false);
        uint4 next[HALF][3][2];
        auto take = [&](int j0, int kb) {
#pragma unroll
          for (int j = 0; j < HALF; ++j)
#pragma unroll
            for (int part = 0; part < 3; ++part)
#pragma unroll
              for (int s = 0; s < 2; ++s) next[j][part][s] = *reinterpret_cast<const uint4*>(ar[j0 + j] + part * p.part_stride + kb * 64 + s * 32);
        };
        take(0, m.k0);
        for (int kb = m.k0; kb < m.k1; ++kb) {
          uint4 w[4][2];
#pragma unroll
          for (int j0 = 0; j0 < N; j0 += HALF) {
            uint4 x[HALF][3][2];
#pragma unroll
            for (int j = 0; j < HALF; ++j)
#pragma unroll
              for (int part = 0; part < 3; ++part) { x[j][part][0] = next[j][part][0]; x[j][part][1] = next[j][part][1]; }
            if (j0 + HALF < N) take(j0 + HALF, kb);
            else take(0, min(kb + 1, m.k1 - 1));
            if (j0 == 0) ml_weights(w, ring.wait(bw), r, t4);
#pragma unroll
            for (int j = 0; j < HALF; ++j)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                float sum[4] = {};
#pragma unroll
                for (int part = 2; part >= 0; --part)            // (the smallest first)
#pragma unroll
                  for (int s = 0; s < 2; ++s) {
                    const uint4 lo = w[2 * i][s], hi = w[2 * i + 1][s];
                    mma_bf16(sum, lo.x, hi.x, lo.y, hi.y, x[j][part][s].x, x[j][part][s].y);
                    mma_bf16(sum, lo.z, hi.z, lo.w, hi.w, x[j][part][s].z, x[j][part][s].w);
                  }
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[i][j0 + j][c] += sum[c];
              }
          }
          __syncwarp();
          ring.read();
          ask();
        }
        // (a row occurs once among an expert's, so no two lanes add to the same place)
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int c = j * 8 + t4 * 2 + h;
            if (c < cols) {
              const int t = ml_token(p, v.row[m.first + n0 + c]);
              float* s = mine + t * LD + r;
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                s[i * 16] += acc[i][j][h];
                s[i * 16 + 8] += acc[i][j][2 + h];
              }
            }
          }
        __syncwarp();
      });
    }
    past(at, m);
  }
  if (bw.dead) ml_land();
  __syncthreads();
  // the warps' sums, then the cluster's: each block adds up its share of the rows
  for (int i = tid; i < p.T * 8; i += ML_THREADS) {
    const int t = i >> 3, c = (i & 7) * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int q = 0; q < ML_WARPS; ++q) {
      const float4 a = *reinterpret_cast<const float4*>(sums + (q * p.T + t) * LD + c);
      s.x += a.x; s.y += a.y; s.z += a.z; s.w += a.w;
    }
    if (p.cluster > 1) *reinterpret_cast<float4*>(sums + t * LD + c) = s;             // (warp 0's place; read before by this thread alone)
    else ml_result(p, t, col0 + c, s);
  }
  if (p.cluster > 1) {
    cluster_sync_all();
    for (int i = rank * ML_THREADS + tid; i < p.T * 8; i += p.cluster * ML_THREADS) {
      const int t = i >> 3, c = (i & 7) * 4;
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int q = 0; q < p.cluster; ++q) {
        const float4 a = ld_dsmem_f32x4(sums + t * LD + c, q);
        s.x += a.x; s.y += a.y; s.z += a.z; s.w += a.w;
      }
      ml_result(p, t, col0 + c, s);
    }
    cluster_sync_all();                  // (nobody leaves while others read its sums)
  }
}

static size_t ml_act_elems(int T, int top, int ff, int sff) { return static_cast<size_t>(T) * (top + 1) * (ff > sff ? ff : sff); }

}  // namespace vb

using namespace vb;

extern "C" {

int vb_moe_layer_max_rows(void) { return ML_MAX_ROWS; }

// idx, weights and the shared expert's gates of every row, then the activations
static size_t ml_head_bytes(int T, int top) { return (static_cast<size_t>(T) * (2 * top + 1) * 4 + 15) / 16 * 16; }
size_t vb_moe_layer_workspace_bytes(const VbMoeWeights* weights, const VbMoeRouter* router, int T) {
  if (!weights || !router || T < 1 || router->top < 1 || weights->ff < 1 || weights->shared_ff < 0) return 0;
  return ml_head_bytes(T, router->top) + 3 * ml_act_elems(T, router->top, weights->ff, weights->shared_ff) * sizeof(__nv_bfloat16);
}

int vb_moe_layer(float* d_y, long long ldy, const void* d_h, long long ldh, const VbMoeWeights* weights, const VbMoeRouter* router, const int32_t* d_ids, int T,
                 void* d_ws, size_t ws_bytes, void* stream) {
  VB_CHECK_ARG(d_y && d_h && weights && router && weights->d_up && weights->d_down && d_ws, "vb_moe_layer: null pointer");
  const int W = weights->width, experts = weights->experts, ff = weights->ff, shared_ff = weights->shared_ff, up_rows = weights->up_rows, act = weights->act;
  const int kind = router->kind, top = router->top, groups = router->groups > 0 ? router->groups : 0, keep = router->keep;
  VB_CHECK_ARG(T <= ML_MAX_ROWS, "vb_moe_layer: %d rows; at most %d", T, ML_MAX_ROWS);
  VB_CHECK_ARG(experts >= 1 && experts <= ML_MAX_EXPERTS && top >= 1 && top <= ML_MAX_TOP && top <= experts, "vb_moe_layer: %d experts (1 to %d), top %d (1 to %d)", experts,
               ML_MAX_EXPERTS, top, ML_MAX_TOP);
  VB_CHECK_ARG(kind >= 0 && kind <= 3, "vb_moe_layer: router %d", kind);
  VB_CHECK_ARG(kind == ML_TABLE ? d_ids && router->d_table && router->vocab > 0 : router->d_weight != nullptr, "vb_moe_layer: the router lacks its matrix, or its table and ids");
  const auto off = [](const void* ptr, int align) { return reinterpret_cast<uintptr_t>(ptr) % align != 0; };
  VB_CHECK_ARG(!off(weights->d_up, 16) && !off(weights->d_down, 16) && !off(d_y, 4) && !off(d_ids, 4) && !off(router->d_bias, 4) && !off(router->d_table, 4),
               "vb_moe_layer: the experts' matrices must be 16-byte aligned, y, ids, bias and table 4-byte");
  VB_CHECK_ARG(W >= 8 && W <= (1 << 24) && W % 8 == 0 && ldh % 8 == 0 && ldh >= W && ldy >= W && reinterpret_cast<uintptr_t>(d_h) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(router->d_weight) % 16 == 0 && reinterpret_cast<uintptr_t>(router->d_shared_gate) % 16 == 0,
               "vb_moe_layer: rows must be multiples of 8 elements, 16-byte aligned (width %d)", W);
  VB_CHECK_ARG(groups <= 1 || ((kind == ML_SIGMOID || kind == ML_SOFTMAX_ALL) && experts % groups == 0 && keep >= 1 && keep <= groups && keep * (experts / groups) >= top),
               "vb_moe_layer: %d groups (keep %d) do not fit %d experts, top %d", groups, keep, experts, top);
  VB_CHECK_ARG(ff >= 64 && ff % 64 == 0 && shared_ff >= 0 && shared_ff % 64 == 0, "vb_moe_layer: expert widths %d and %d must be multiples of 64", ff, shared_ff);
  VB_CHECK_ARG(ff <= (1 << 17) && shared_ff <= (1 << 17), "vb_moe_layer: expert widths %d and %d; at most %d", ff, shared_ff, 1 << 17);
  VB_CHECK_ARG(act >= 0 && act <= 4 && (act != ML_CLAMPED_GLU || weights->limit > 0.f), "vb_moe_layer: activation %d, limit %f", act, weights->limit);
  const bool gated = act <= ML_CLAMPED_GLU;
  VB_CHECK_ARG(up_rows >= 32 && up_rows <= 128 && up_rows % 32 == 0 && (gated ? 2 * ff : ff) % up_rows == 0 && (gated ? 2 * shared_ff : shared_ff) % up_rows == 0,
               "vb_moe_layer: tiles of %d rows do not divide the experts", up_rows);
  VB_CHECK_ARG(!router->d_shared_gate || shared_ff > 0, "vb_moe_layer: a gate without a shared expert");
  if (T <= 0) return 0;
  VB_CHECK_ARG(ws_bytes >= vb_moe_layer_workspace_bytes(weights, router, T) && reinterpret_cast<uintptr_t>(d_ws) % 16 == 0,
               "vb_moe_layer: workspace of %zu bytes is too small or not aligned", ws_bytes);
  MoeLayerParams p = {};
  int32_t* d_idx = static_cast<int32_t*>(d_ws);
  float *d_wts = reinterpret_cast<float*>(d_idx + T * top), *d_gate = router->d_shared_gate ? d_wts + T * top : nullptr;
  MoeRouteParams r = {};
  r.idx = d_idx;
  r.wts = d_wts;
  r.sgate = d_gate;
  r.h = static_cast<const __nv_bfloat16*>(d_h);
  r.ldh = ldh;
  r.w = router->d_weight;
  r.bias = kind == ML_SOFTMAX || kind == ML_SIGMOID ? router->d_bias : nullptr;
  r.wsg = router->d_shared_gate;
  r.ids = d_ids;
  r.table = router->d_table;
  r.T = T;
  r.W = W;
  r.E = experts;
  r.top = top;
  r.kind = kind;
  r.groups = groups;
  r.keep = keep;
  r.vocab = router->vocab;
  p.h = r.h;
  p.ldh = ldh;
  p.up = static_cast<const uint8_t*>(weights->d_up);
  p.down = static_cast<const uint8_t*>(weights->d_down);
  p.idx = d_idx;
  p.wts = d_wts;
  p.sgate = d_gate;
  p.act = reinterpret_cast<__nv_bfloat16*>(static_cast<uint8_t*>(d_ws) + ml_head_bytes(T, top));
  p.y = d_y;
  p.ldy = ldy;
  p.T = T;
  p.W = W;
  p.E = experts;
  p.top = top;
  p.top_inverse = static_cast<uint32_t>(((1ull << 32) + top - 1) / top);
  p.ff = ff;
  p.sff = shared_ff;
  p.ld_act = ff > shared_ff ? ff : shared_ff;
  p.part_stride = static_cast<long long>(ml_act_elems(T, top, ff, shared_ff));
  p.kb = (W + 63) / 64;
  p.up_rows = up_rows;
  p.tile_inverse = (65536 + up_rows / 32 - 1) / (up_rows / 32);
  p.expert_bytes = static_cast<long long>(gated ? 2 * ff : ff) * p.kb * 128;
  p.down_kb = (experts * ff + shared_ff) / 64;
  p.act_kind = act;
  p.limit = weights->limit;
  p.slope = weights->slope;
  p.up_units = (gated ? 2 * ff : ff) / 32;
  p.shared_units = (gated ? 2 * shared_ff : shared_ff) / 32;
  VB_CHECK_ARG(p.wait_flag = wait_flag(WK_MOE_LAYER), "vb_moe_layer: no mapped host memory");
  if (kind == ML_TABLE && T <= 8) {
    // (every block looks the experts up by itself, and those of the shared expert form its gates: a launch less)
    p.table = router->d_table;
    p.ids = d_ids;
    p.vocab = router->vocab;
    p.wsg = router->d_shared_gate;
  } else {
    const size_t smem_route = (static_cast<size_t>(ML_ROUTE_THREADS / 32 * 16) * ML_ROUTE_CLUSTER + 2 * static_cast<size_t>(experts) + groups + 48) * 4;
    VB_LAUNCH_PDL_CLUSTER(moe_layer_route_kernel, (T + ML_ROUTE_CLUSTER - 1) / ML_ROUTE_CLUSTER * ML_ROUTE_CLUSTER, ML_ROUTE_THREADS, smem_route, stream, ML_ROUTE_CLUSTER, r);
  }
  const int sms = sm_count();
  const long long most = static_cast<long long>(experts < T * top ? experts : T * top) * p.up_units + p.shared_units;
  const int grid_up = static_cast<int>(most < sms ? most : sms), nt = T <= 8 ? 1 : T <= 16 ? 2 : 4;
  const size_t plan_bytes = static_cast<size_t>(ml_plan_words(T, experts, top)) * 4;
  // Ring places a warp: three where one block an SM runs, and where a block of the next kernel stands beside (steps of up to 8 rows: it has its first weights before
  // this one ends); two in the down kernel of up to 16 rows, of which an SM then holds two.
  constexpr int PLACES = 3;
  const size_t smem_up = ml_ring_bytes(PLACES) + static_cast<size_t>(2 * ML_WARPS) * 32 * (nt == 1 ? 8 : nt * 8 + 8) * 4 + plan_bytes;
#define ML_UP(NT, G)                                                                      \
  do {                                                                                    \
    VB_CHECK_CUDA((rm_smem<moe_up_kernel<NT, G, PLACES>>()));                             \
    VB_LAUNCH_PDL((moe_up_kernel<NT, G, PLACES>), grid_up, ML_THREADS, smem_up, stream, p); \
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
  const size_t smem_down = ml_ring_bytes(nt == 2 ? 2 : PLACES) + static_cast<size_t>(ML_WARPS) * T * ML_LD * 4 + plan_bytes;
  const int blocks = (W + 31) / 32;
  // one wave of clusters (16 rows of 1536, 48 blocks of columns: of four 57.7 us, of five, of which 56 fit, 56.7, of six, of which 45 do, 70.9; 64 rows of 1280: of two 156, of three 138)
#define ML_DOWN(NT, S)                                                                                                  \
  do {                                                                                                                  \
    VB_CHECK_CUDA((rm_smem<moe_down_kernel<NT, S>>()));                                                                 \
    p.cluster = 8;                                                                                                      \
    while (p.cluster > 1 && blocks > rm_clusters<moe_down_kernel<NT, S>>(p.cluster, ML_THREADS, smem_down)) --p.cluster; \
    VB_LAUNCH_PDL_CLUSTER((moe_down_kernel<NT, S>), blocks * p.cluster, ML_THREADS, smem_down, stream, p.cluster, p);   \
  } while (0)
  if (nt == 1) ML_DOWN(1, PLACES);
  else if (nt == 2) ML_DOWN(2, 2);
  else ML_DOWN(4, PLACES);
#undef ML_DOWN
  return 0;
}

}  // extern "C"
