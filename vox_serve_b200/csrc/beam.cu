// One step of a beam search: the n best continuations of a request's beams, and the recurrent states that follow them.
//
//   total[w][v] = score[w] + x[w][v] - log sum_v exp x[w][v]       (over the v whose logit is finite: the others are masked)
//   the n candidates of largest weight[w] * total[w][v]; equal ones in the order of (w, v)
//   a beam that has ended has one candidate, its end token at its own score
//
// Two launches.  The first reads the logits once: a block takes 8192 of a row, keeps them in registers, and leaves their maximum, their sum of exponentials
// and their n largest in order.  The second, a block a request, adds the sums up, ranks the n largest of every slice by their totals and writes the n best.
// What orders candidates is computed in 64 bits from the slices' sums, so that it hangs on those alone; a sum's terms carry 2^-22 each and no common error.
#include "../../include/vb_api.h"
#define VB_PDL_FAMILY 16
#include "common.cuh"

namespace vb {

constexpr int BS_THREADS = 256;
constexpr int BS_SLICE = 8192;            // logits of a block: 32 a thread
constexpr int BS_CAP = 512;               // candidates that a block ranks
constexpr int BS_MAX_N = 64, BS_MAX_W = 32;

struct BeamStats {
  float m, s;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float LOG2E = 1.44269502f, LOG2E_REST = 1.92596303e-8f;
// e^d, d <= 0: log2 e in two parts, so that the product's rounding (2^-24 of the exponent) is the only error and has no common sign
__device__ __forceinline__ float exp_down(float d) { return ex2(fmaf(d, LOG2E, d * LOG2E_REST)); }

// finite values in their order as unsigned numbers > 0 (-0 as 0); 0: not finite
__device__ __forceinline__ uint32_t order_f32(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  const uint32_t k = u ^ (static_cast<int32_t>(u) < 0 ? 0xffffffffu : 0x80000000u);
  return (u & 0x7f800000u) == 0x7f800000u ? 0u : k;
}
__device__ __forceinline__ float unorder_f32(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ uint64_t order_f64(double x) {
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(x + 0.0));
  const uint64_t k = u ^ (static_cast<int64_t>(u) < 0 ? ~0ull : 0x8000000000000000ull);
  return (u & 0x7ff0000000000000ull) == 0x7ff0000000000000ull ? 0ull : k;
}

// sum over the block of what its threads counted; `box`: three words, zero at first, used in turn
__device__ __forceinline__ int block_count(int mine, uint32_t* box, int& turn) {
  const int w = __reduce_add_sync(0xffffffffu, mine);
  if ((threadIdx.x & 31) == 0 && w) atomicAdd(&box[turn], static_cast<uint32_t>(w));
  __syncthreads();
  const int n = static_cast<int>(box[turn]);
  turn = turn == 2 ? 0 : turn + 1;
  if (threadIdx.x == 0) box[turn == 2 ? 0 : turn + 1] = 0u;      // the one before this: read before the barrier above, written behind the next one
  return n;
}

// Is the row's beam one whose logits are read?  (A dead beam's score is not finite, an ended one has a candidate without them.)
__device__ __forceinline__ bool beam_reads(const float* score, const float* weight, const uint8_t* ended, int row) {
  if (ended && ended[row]) return false;
  const float s = score[row], by = weight ? weight[row] : 1.f;
  return isfinite(s) && isfinite(by) && by > 0.f;
}

// 16 bytes from byte `by` of the 32 that two neighbouring vectors hold (by < 16, even)
__device__ __forceinline__ uint4 realign(uint4 p, uint4 q, int by) {
  uint32_t w[7] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z};
  uint32_t last = q.w;
  if (by & 8) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 2];
    w[5] = last;
  }
  if (by & 4) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  }
  if (by & 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The logits that a thread holds: 32, as they came
template <typename T>
struct Held;
template <>
struct Held<float> {
  uint32_t w[32];
  __device__ __forceinline__ float at(int k) const { return __uint_as_float(w[k]); }
  __device__ __forceinline__ void mask(int k) { w[k] = 0xff800000u; }
};
template <>
struct Held<__nv_bfloat16> {
  uint32_t w[16];
  __device__ __forceinline__ float at(int k) const { return (k & 1) ? bf16_hi(w[k >> 1]) : bf16_lo(w[k >> 1]); }
  __device__ __forceinline__ void mask(int k) { w[k >> 1] = (k & 1) ? (w[k >> 1] & 0xffffu) | 0xff800000u : (w[k >> 1] & 0xffff0000u) | 0xff80u; }
};

// One slice of one row.  T: bf16 or fp32 logits.  Rows may start at any element: a thread's vector is put together from the two aligned ones it lies in, so
// that which thread adds what does not hang on the address, and equal rows have equal sums.  (A vector that holds a byte of the row lies in the same 16 bytes.)
template <typename T>
__global__ void __launch_bounds__(BS_THREADS, 4) beam_slice_kernel(BeamStats* __restrict__ stats, uint64_t* __restrict__ best, const T* __restrict__ logits,
                                                                   long long stride, int V, int slices, const float* score, const float* weight,
                                                                   const uint8_t* ended, int n) {
  constexpr int EV = 16 / sizeof(T), NV = 32 / EV;
  __shared__ uint64_t list[BS_CAP];
  __shared__ uint32_t box[3], count;
  __shared__ float groups[64], cut_s, part_m[8], part_s[8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / slices, slice = blockIdx.x - row * slices;
  if (tid == 0) box[0] = box[1] = box[2] = count = 0u;
  pdl_sync();
  if (!beam_reads(score, weight, ended, row)) return;       // (the second kernel does not look at this row either)
  const uintptr_t at = reinterpret_cast<uintptr_t>(logits + static_cast<long long>(row) * stride);
  const int by = static_cast<int>(at & 15);
  const uint4* src = reinterpret_cast<const uint4*>(at - by);
  const int vecs = (V + EV - 1) / EV, held = (V * static_cast<int>(sizeof(T)) + by + 15) / 16, v0 = slice * (BS_SLICE / EV);

  Held<T> x;
  {
    uint4 q[NV];
    const uint4 none = sizeof(T) == 4 ? make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u) : make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int vi = v0 + i * BS_THREADS + tid;
      q[i] = vi < vecs ? __ldg(src + vi) : none;
    }
    if (by) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int vi = v0 + i * BS_THREADS + tid;
        if (vi < vecs) q[i] = realign(q[i], vi + 1 < held ? __ldg(src + vi + 1) : none, by);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) x.w[4 * i] = q[i].x, x.w[4 * i + 1] = q[i].y, x.w[4 * i + 2] = q[i].z, x.w[4 * i + 3] = q[i].w;
  }
  // the token of x.at(k)
  auto token = [&](int k) { return static_cast<uint32_t>((v0 + (k / EV) * BS_THREADS + tid) * EV + (k % EV)); };
  if (V % EV && v0 + BS_SLICE / EV >= vecs) {               // behind the row's last token
#pragma unroll
    for (int k = 0; k < 32; ++k)
      if (token(k) >= static_cast<uint32_t>(V)) x.mask(k);
  }

  // Maximum and sum of exponentials, each thread's own first.  One product and sum an element: 2^(x log2 e - c) with c the rounded m log2 e, and what the
  // rounding took is put back into the sum.  What is not finite shows up in the maximum or the sum and is masked then; huge values take the longer way.
  auto maximum = [&]() {
    float m = x.at(0);
#pragma unroll
    for (int k = 1; k < 32; ++k) m = fmaxf(m, x.at(k));
    return m;
  };
  float m = maximum(), s = 0.f;
  if (m != -INFINITY) {
    const float c = m * LOG2E;
    float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 32; ++k) t[k & 3] += ex2(fmaf(x.at(k), LOG2E, -c));
    s = (t[0] + t[1]) + (t[2] + t[3]);
    s *= ex2(fmaf(-m, LOG2E, c));
  }
  bool odd = !(s < INFINITY) || !(fabsf(m) < 1e37f);
  if (m == -INFINITY) {                                     // (masked all, or NaN)
    odd = false;
#pragma unroll
    for (int k = 0; k < 32; ++k) odd |= x.at(k) != x.at(k);
  }
  if (odd) {
#pragma unroll
    for (int k = 0; k < 32; ++k)
      if (!isfinite(x.at(k))) x.mask(k);
    m = maximum();
    s = 0.f;
    if (m != -INFINITY) {
#pragma unroll
      for (int k = 0; k < 32; ++k) s += exp_down(x.at(k) - m);
    }
  }
  const float wm = warp_max(m);
  const float ws = warp_sum(m != -INFINITY ? s * exp_down(m - wm) : 0.f);
  if (lane == 0) part_m[warp] = wm, part_s[warp] = ws;
  // A first cut: of at least n groups of threads each has an element that is not below the smallest of the groups' maxima.  Groups of 256 / G
  // neighbours, whose elements are spread over the whole slice.
  const int G = n <= 8 ? 8 : n <= 16 ? 16 : n <= 32 ? 32 : 64;
  float gm = m;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
    if (o < BS_THREADS / G) gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, o));
  if ((tid & (BS_THREADS / G - 1)) == 0) groups[tid / (BS_THREADS / G)] = gm;
  __syncthreads();
  if (warp == 0) {
    float low = lane < G ? groups[lane] : INFINITY;
    if (G == 64) low = fminf(low, groups[lane + 32]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    if (lane == 0) cut_s = fmaxf(low, -3.4028235e38f);
  }
  if (warp == 1) {
    const float pm = lane < 8 ? part_m[lane] : -INFINITY;
    const float top = warp_max(pm);
    const float sum = warp_sum(pm != -INFINITY ? part_s[lane & 7] * exp_down(pm - top) : 0.f);
    if (lane == 0) stats[blockIdx.x] = {top, top == -INFINITY ? 0.f : sum};
  }
  __syncthreads();
  // an element as one number: its value, then the lower token first
  auto keyed = [&](int k) {
    const uint32_t o = order_f32(x.at(k));
    return o ? (static_cast<uint64_t>(o) << 32 | (0xffffffffu - token(k))) : 0ull;
  };
  const float cut_f = cut_s;
  if (m >= cut_f) {
#pragma unroll
    for (int k = 0; k < 32; ++k)
      if (x.at(k) >= cut_f) {
        const uint32_t i = atomicAdd(&count, 1u);
        if (i < BS_CAP) list[i] = keyed(k);
      }
  }
  __syncthreads();
  int found = static_cast<int>(count);
  if (found > BS_CAP) {      // many equal or nearly equal values, or a group without any: halve the range until the list holds them
    uint64_t lo = static_cast<uint64_t>(order_f32(cut_f)) << 32, hi = ~0ull;
    int turn = 0;
    while (found > BS_CAP) {                                  // at least n are >= lo, fewer than n are >= hi
      const uint64_t mid = lo + ((hi - lo) >> 1);
      int mine = 0;
#pragma unroll
      for (int k = 0; k < 32; ++k) mine += keyed(k) >= mid ? 1 : 0;
      const int c = block_count(mine, box, turn);
      if (c >= n) lo = mid, found = c;
      else hi = mid;
    }
    if (tid == 0) count = 0u;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      const uint64_t key = keyed(k);
      if (key >= lo) list[atomicAdd(&count, 1u)] = key;
    }
    __syncthreads();
  }
  // every key's place in the order is the number of larger ones (they differ)
  uint64_t* out = best + static_cast<long long>(blockIdx.x) * n;
  for (int i = tid; i < found; i += BS_THREADS) {
    const uint64_t key = list[i];
    int rank = 0;
    for (int j = 0; j < found; ++j) rank += list[j] > key ? 1 : 0;
    if (rank < n) out[rank] = key;
  }
  for (int i = found + tid; i < n; i += BS_THREADS) out[i] = 0ull;
}

constexpr int BJ_THREADS = 512, BJ_CAP = 512;

// The n best of one request.  Candidate c of its W * slices * n: row, slice, place.
__global__ void __launch_bounds__(BJ_THREADS) beam_join_kernel(float* __restrict__ out_score, int32_t* __restrict__ out_parent, int64_t* __restrict__ out_token,
                                                               uint8_t* __restrict__ out_ended, const BeamStats* __restrict__ stats,
                                                               const uint64_t* __restrict__ best, const float* score, const float* weight,
                                                               const uint8_t* ended, int W, int slices, int n, long long end_token) {
  __shared__ double base[BS_MAX_W], tops[BS_MAX_W], by[BS_MAX_W];      // total = (x - top) + base: a row may hold nothing but lowest values; base of an ended beam: its score
  __shared__ uint8_t kind[BS_MAX_W];                   // 0: no candidates, 1: logits, 2: ended
  __shared__ uint64_t list_key[BJ_CAP], list_at[BJ_CAP];      // rank, (beam, token)
  __shared__ double list_total[BJ_CAP];
  __shared__ uint32_t box[3], count;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.x;
  if (tid == 0) box[0] = box[1] = box[2] = count = 0u;
  pdl_sync();
  for (int w = warp; w < W; w += BJ_THREADS / 32) {
    const int row = b * W + w;
    const float s = score[row], f = weight ? weight[row] : 1.f;
    const bool over = ended && ended[row];
    int k = over ? 2 : 1;
    if (!isfinite(s) || !isfinite(f) || !(f > 0.f)) k = 0;
    double log_sum = 0.0, peak = 0.0;
    if (k == 1) {
      float top = -INFINITY;
      for (int i = lane; i < slices; i += 32) top = fmaxf(top, stats[row * slices + i].m);
      top = warp_max(top);
      double sum = 0.0;
      for (int i = lane; i < slices; i += 32) {
        const BeamStats t = stats[row * slices + i];
        if (t.m != -INFINITY) sum += static_cast<double>(t.s) * exp(static_cast<double>(t.m) - static_cast<double>(top));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (top == -INFINITY) k = 0;                       // everything masked: nothing to go on with
      else peak = top, log_sum = log(sum);
    }
    if (lane == 0) base[w] = static_cast<double>(s) - log_sum, tops[w] = peak, by[w] = f, kind[w] = k;
  }
  __syncthreads();

  const int per_row = slices * n, all = W * per_row;
  auto key_of = [&](int c, uint64_t& at, double& total) -> uint64_t {
    const int w = c / per_row;
    if (kind[w] != 1) {
      if (kind[w] == 0 || c != w * per_row) return 0ull;
      at = static_cast<uint64_t>(w) << 32 | static_cast<uint64_t>(end_token);
      total = base[w];
    } else {
      const uint64_t e = best[static_cast<long long>(b) * all + c];
      if (!e) return 0ull;
      at = static_cast<uint64_t>(w) << 32 | (0xffffffffu - static_cast<uint32_t>(e));
      total = (static_cast<double>(unorder_f32(static_cast<uint32_t>(e >> 32))) - tops[w]) + base[w];
    }
    return order_f64(total * by[w]);
  };
  // All candidates if the list holds them, else those above a cut that leaves at least n: found by halving the range, first of ranks, then (equal ranks)
  // of places.
  int turn = 0;
  auto count_from = [&](uint64_t cut, uint64_t tie) {
    int mine = 0;
    for (int c = tid; c < all; c += BJ_THREADS) {
      uint64_t at;
      double total;
      const uint64_t key = key_of(c, at, total);
      mine += key > cut || (key == cut && key && at <= tie) ? 1 : 0;
    }
    return block_count(mine, box, turn);
  };
  uint64_t cut = 1ull, tie = ~0ull;
  int found = count_from(cut, tie);
  if (found > BJ_CAP) {
    uint64_t lo = 1ull, hi = ~0ull;
    while (found > BJ_CAP && hi - lo > 1ull) {
      const uint64_t mid = lo + ((hi - lo) >> 1);
      const int c = count_from(mid, tie);
      if (c >= n) lo = mid, found = c;
      else hi = mid;
    }
    cut = lo;
    uint64_t below = 0ull;                                  // (places of equal ranks: the fewest of the first ones that are enough)
    while (found > BJ_CAP) {
      const uint64_t mid = below + ((tie - below) >> 1);
      const int c = count_from(cut, mid);
      if (c >= n) tie = mid, found = c;
      else below = mid + 1ull;
    }
  }
  for (int c = tid; c < all; c += BJ_THREADS) {
    uint64_t at;
    double total;
    const uint64_t key = key_of(c, at, total);
    if (key > cut || (key == cut && at <= tie)) {
      const uint32_t i = atomicAdd(&count, 1u);
      list_key[i] = key, list_at[i] = at, list_total[i] = total;
    }
  }
  __syncthreads();
  for (int i = tid; i < found; i += BJ_THREADS) {
    const uint64_t key = list_key[i], at = list_at[i];
    int rank = 0;
    for (int j = 0; j < found; ++j) rank += list_key[j] > key || (list_key[j] == key && list_at[j] < at) ? 1 : 0;
    if (rank < n) {
      const int w = static_cast<int>(at >> 32), o = b * n + rank;
      const uint32_t v = static_cast<uint32_t>(at);
      out_score[o] = static_cast<float>(list_total[i]);
      out_parent[o] = w;
      out_token[o] = v;
      if (out_ended) out_ended[o] = kind[w] == 2 || static_cast<long long>(v) == end_token;
    }
  }
  for (int i = found + tid; i < n; i += BJ_THREADS) {
    out_score[b * n + i] = -INFINITY;
    out_parent[b * n + i] = -1;
    out_token[b * n + i] = -1;
    if (out_ended) out_ended[b * n + i] = 1;
  }
}

// ---- states that follow their beams ----------------------------------------------------------------------------------------------
// state[slot[b][i]] = what state[slot[b][parent[b][i]]] was.  A thread owns a vector's place in all W rows of a request: it reads what moves there, then
// writes, so that rows may change places without a second copy of the state.
constexpr int BR_TENSORS = 64, BR_THREADS = 256;
struct ReorderTensors {
  void* at[BR_TENSORS];
  uint32_t vecs[BR_TENSORS];        // vectors of a row
  uint32_t first[BR_TENSORS + 1];   // blocks in front
  uint8_t log_vec[BR_TENSORS];      // bytes of a vector, as a power of two
  int n, slots;
};

template <typename V, int MAXW>
__device__ __forceinline__ void reorder_column(V* at, long long vecs, uint32_t col, const int* src, const int* dst, int W) {
  V v[MAXW];
#pragma unroll
  for (int i = 0; i < MAXW; ++i)
    if (i < W && dst[i] >= 0) v[i] = at[src[i] * vecs + col];
#pragma unroll
  for (int i = 0; i < MAXW; ++i)
    if (i < W && dst[i] >= 0) at[dst[i] * vecs + col] = v[i];
}

template <int MAXW>
__global__ void __launch_bounds__(BR_THREADS) beam_reorder_kernel(const __grid_constant__ ReorderTensors t, const int32_t* parent, const int32_t* slots, int W) {
  __shared__ int src[MAXW], dst[MAXW], moves;
  const int tid = threadIdx.x, b = blockIdx.y;
  int lo = 0, hi = t.n - 1;                   // the tensor that this block is of
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= blockIdx.x) lo = mid;
    else hi = mid - 1;
  }
  if (tid == 0) moves = 0;
  pdl_sync();
  __syncthreads();
  if (tid < W) {
    const int p = parent[b * W + tid];
    int from = -1, to = -1;
    if (p >= 0 && p < W && p != tid) {
      from = slots ? slots[b * W + p] : b * W + p;
      to = slots ? slots[b * W + tid] : b * W + tid;
      if (from < 0 || from >= t.slots || to < 0 || to >= t.slots || from == to) to = -1;
    }
    src[tid] = from, dst[tid] = to;
    if (to >= 0) moves = 1;
  }
  __syncthreads();
  if (!moves) return;
  const uint32_t col = (blockIdx.x - t.first[lo]) * BR_THREADS + tid;
  const long long vecs = t.vecs[lo];
  if (col >= vecs) return;
  switch (t.log_vec[lo]) {
    case 4: reorder_column<uint4, MAXW>(static_cast<uint4*>(t.at[lo]), vecs, col, src, dst, W); break;
    case 3: reorder_column<uint2, MAXW>(static_cast<uint2*>(t.at[lo]), vecs, col, src, dst, W); break;
    case 2: reorder_column<uint32_t, MAXW>(static_cast<uint32_t*>(t.at[lo]), vecs, col, src, dst, W); break;
    case 1: reorder_column<uint16_t, MAXW>(static_cast<uint16_t*>(t.at[lo]), vecs, col, src, dst, W); break;
    default: reorder_column<uint8_t, MAXW>(static_cast<uint8_t*>(t.at[lo]), vecs, col, src, dst, W); break;
  }
}

inline long long beam_slices(long long vocab) { return (vocab + BS_SLICE - 1) / BS_SLICE; }

}  // namespace vb

using namespace vb;

extern "C" size_t vb_beam_select_workspace_bytes(int requests, int width, int vocab, int n) {
  if (requests <= 0 || width <= 0 || vocab <= 0 || n <= 0) return 0;
  return static_cast<size_t>(requests) * width * beam_slices(vocab) * (sizeof(BeamStats) + 8ull * n);
}

extern "C" int vb_beam_select(float* d_score, int32_t* d_parent, int64_t* d_token, uint8_t* d_out_ended, const void* d_logits, int64_t row_stride, int logits_f32,
                              const float* d_beam_score, const float* d_weight, const uint8_t* d_ended, int requests, int width, int vocab, int n, int64_t end_token,
                              void* d_workspace, size_t workspace_bytes, void* stream) {
  VB_CHECK_ARG(d_score && d_parent && d_token && d_logits && d_beam_score && d_workspace, "vb_beam_select: null pointer");
  VB_CHECK_ARG(requests > 0 && width > 0 && width <= BS_MAX_W && n > 0 && n <= BS_MAX_N, "vb_beam_select: %d requests of %d beams (1 to %d), the best %d (1 to %d)", requests,
               width, BS_MAX_W, n, BS_MAX_N);
  VB_CHECK_ARG(vocab > 0 && vocab <= (1 << 24), "vb_beam_select: vocabulary of %d (1 to 2^24)", vocab);
  VB_CHECK_ARG(reinterpret_cast<uintptr_t>(d_logits) % (logits_f32 ? 4 : 2) == 0, "vb_beam_select: logits that are not aligned to their type");
  VB_CHECK_ARG(row_stride >= 0, "vb_beam_select: row stride %lld", static_cast<long long>(row_stride));
  VB_CHECK_ARG(!(d_ended || d_out_ended) || (end_token >= 0 && end_token < vocab), "vb_beam_select: end token %lld outside the vocabulary of %d",
               static_cast<long long>(end_token), vocab);
  const long long slices = beam_slices(vocab), blocks = static_cast<long long>(requests) * width * slices;
  VB_CHECK_ARG(blocks <= 0x7fffffffll && blocks * n / requests <= 0x7fffffffll, "vb_beam_select: %lld slices of rows", blocks);
  VB_CHECK_ARG(workspace_bytes >= vb_beam_select_workspace_bytes(requests, width, vocab, n) && reinterpret_cast<uintptr_t>(d_workspace) % 8 == 0,
               "vb_beam_select: workspace of %zu bytes", workspace_bytes);
  uint64_t* best = static_cast<uint64_t*>(d_workspace);
  BeamStats* stats = reinterpret_cast<BeamStats*>(best + blocks * n);
  if (logits_f32)
    VB_LAUNCH_PDL(beam_slice_kernel<float>, static_cast<unsigned>(blocks), BS_THREADS, 0, stream, stats, best, static_cast<const float*>(d_logits),
                  static_cast<long long>(row_stride), vocab, static_cast<int>(slices), d_beam_score, d_weight, d_ended, n);
  else
    VB_LAUNCH_PDL(beam_slice_kernel<__nv_bfloat16>, static_cast<unsigned>(blocks), BS_THREADS, 0, stream, stats, best, static_cast<const __nv_bfloat16*>(d_logits),
                  static_cast<long long>(row_stride), vocab, static_cast<int>(slices), d_beam_score, d_weight, d_ended, n);
  VB_LAUNCH_PDL(beam_join_kernel, static_cast<unsigned>(requests), BJ_THREADS, 0, stream, d_score, d_parent, d_token, d_out_ended, stats, best, d_beam_score, d_weight,
                d_ended, width, static_cast<int>(slices), n, static_cast<long long>(end_token));
  return 0;
}

extern "C" int vb_beam_reorder(void* const* states, const int64_t* row_bytes, int n_states, int n_slots, const int32_t* d_parent, const int32_t* d_slots, int requests,
                               int width, void* stream) {
  VB_CHECK_ARG(states && row_bytes && d_parent, "vb_beam_reorder: null pointer");
  VB_CHECK_ARG(n_states > 0 && n_slots > 0, "vb_beam_reorder: %d states of %d slots", n_states, n_slots);
  VB_CHECK_ARG(requests > 0 && requests <= 65535 && width > 0 && width <= BS_MAX_W, "vb_beam_reorder: %d requests of %d beams (1 to %d)", requests, width, BS_MAX_W);
  VB_CHECK_ARG(d_slots || static_cast<int64_t>(requests) * width <= n_slots, "vb_beam_reorder: %d requests of %d beams in %d rows", requests, width, n_slots);
  for (int i = 0; i < n_states; ++i)
    VB_CHECK_ARG(states[i] && row_bytes[i] > 0 && row_bytes[i] < (1ll << 32), "vb_beam_reorder: state %d of %lld bytes a row", i,
                 static_cast<long long>(row_bytes[i]));
  for (int i0 = 0; i0 < n_states; i0 += BR_TENSORS) {
    ReorderTensors t = {};
    t.n = n_states - i0 < BR_TENSORS ? n_states - i0 : BR_TENSORS;
    t.slots = n_slots;
    long long blocks = 0;
    for (int i = 0; i < t.n; ++i) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(states[i0 + i]);
      const int64_t bytes = row_bytes[i0 + i];
      int log_vec = 4;
      while ((at | static_cast<uintptr_t>(bytes)) & ((1u << log_vec) - 1)) --log_vec;
      t.at[i] = states[i0 + i];
      t.log_vec[i] = static_cast<uint8_t>(log_vec);
      t.vecs[i] = static_cast<uint32_t>(bytes >> log_vec);
      t.first[i] = static_cast<uint32_t>(blocks);
      blocks += (t.vecs[i] + static_cast<long long>(BR_THREADS) - 1) / BR_THREADS;
    }
    t.first[t.n] = static_cast<uint32_t>(blocks);
    VB_CHECK_ARG(blocks <= 0x7fffffffll, "vb_beam_reorder: %lld blocks", blocks);
    const dim3 grid(static_cast<unsigned>(blocks), requests);
    if (width <= 4) VB_LAUNCH_PDL(beam_reorder_kernel<4>, grid, BR_THREADS, 0, stream, t, d_parent, d_slots, width);
    else if (width <= 8) VB_LAUNCH_PDL(beam_reorder_kernel<8>, grid, BR_THREADS, 0, stream, t, d_parent, d_slots, width);
    else if (width <= 16) VB_LAUNCH_PDL(beam_reorder_kernel<16>, grid, BR_THREADS, 0, stream, t, d_parent, d_slots, width);
    else VB_LAUNCH_PDL(beam_reorder_kernel<32>, grid, BR_THREADS, 0, stream, t, d_parent, d_slots, width);
  }
  return 0;
}
