// One step of a beam search: the n best continuations of a request's beams, and the recurrent states that follow them.
//
//   total[w][v] = score[w] + x[w][v] - log sum_v exp x[w][v]       (over the v whose logit is finite: the others are masked)
//   the n candidates of largest weight[w] * total[w][v]; equal ones in the order of (w, v)
//   a beam that has ended has one candidate, its end token at its own score
//
// Two kernels.  The first reads the logits once: a block takes a part of a row in chunks, by asynchronous copies into shared memory with the next one on its way,
// and leaves the part's maximum, its sum of exponentials and its n largest in order.  The second, a block a request, adds the sums up, ranks the n largest of every
// part by their totals and writes the n best.  Where a request has at most eight parts and all requests run at once both are one launch, a cluster a request.
//
// What orders candidates is computed in 64 bits from the parts' sums.  A sum's terms carry the special function unit's 2^-22 and, from one fp32 constant for log2 e,
// 1.3e-8 of the distance from the maximum: below 2^-20 of a term that counts (distance up to 40).  Sums of parts meet through log2 e in two constants.
//
// Measured (a captured chain of calls): 16 requests of 16 beams over 156940 bf16 tokens, n 32, four fifths of them masked, 32 us, all of them open 41; the 80 MB are 12.4 us
// of HBM.  What is above that: 512 blocks on 148 SMs, three or four each; 2.2 us a chunk of four blocks of an SM (its 64 KB are 1.3 of HBM, its exponentials 0.9 of the
// special function unit; the rest are instructions and a meeting of the block), 8 to 13 of cuts, orders, launches and the join.  16 of 5 over 32003 fp32 tokens, n 10: 12.1 us.
// One of two over 2051: 5.7, most of it the launch.
// The bf16 form is held at 64 registers for four blocks an SM and spills 148 bytes a thread in its stream.  Four blocks an SM with two chunks in shared memory: 31.2 us;
// three with three 33.3, with four 32.6; four with three 34.4 (a list of 512); five with two 31.6.  Parts so that all blocks run at once: more of them pay the first cut and
// the last order again, fewer leave SMs idle.  Lists are cut back once they hold twice what is wanted: open rows 45.7 us, three times 46.6, four 47.2, at 256 53.7 (masked
// ones 32.6, 32.2, 32.1, 32.0).
#include "../../include/vb_api.h"
#define VB_PDL_FAMILY 16
#include "rowmma.cuh"

namespace vb {

constexpr int BS_THREADS = 256, BS_VECS = 4, BS_STAGES = 2;     // a chunk: four vectors of 16 bytes a thread; chunks in shared memory
constexpr int BS_CAP = 1024;                                   // candidates that a block keeps
constexpr int BS_BLOCKS = 4;                                    // blocks an SM holds
constexpr int BS_MAX_N = 64, BS_MAX_W = 32;
constexpr int BS_CLUSTER = 8;                                   // blocks of a request that join in the same launch
static_assert(BS_CLUSTER * BS_MAX_N * 16 <= 16384, "the join's candidates stand where the ring stood");
constexpr int BJ_BINS = 1024;                                   // 16 to a doubling, from 2^-23 to 2^41
constexpr int BJ_FEW = 512, BJ_ALL = 8192;                  // candidates of a request: 128 KB of ranks and values

struct BeamStats {
  float m, s;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two fp32 at a time
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
constexpr float BS_SHORT = 1073741824.f;                        // maxima up to which a thread's sum takes the short way
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

__device__ __forceinline__ double unorder_f64(uint64_t k) {
  return __longlong_as_double(static_cast<long long>(k & 0x8000000000000000ull ? k ^ 0x8000000000000000ull : ~k));
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

__device__ __forceinline__ void copy16_async(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// Four words of shared memory at an address that is a multiple of ALIGN (two: the words that hold them are read)
template <int ALIGN>
__device__ __forceinline__ void read_words(uint32_t* w, uint32_t at) {
  if (ALIGN == 16) {
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
  } else if (ALIGN == 8) {
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[2]), "=r"(w[3]) : "r"(at + 8u) : "memory");
  } else {
    uint32_t v[5];
#pragma unroll
    for (int j = 0; j < (ALIGN == 4 ? 4 : 5); ++j) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[j]) : "r"(at - (ALIGN == 2 ? 2u : 0u) + 4u * j) : "memory");
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = ALIGN == 4 ? v[j] : __funnelshift_r(v[j], v[j + 1], 16);
  }
}

// The logits of a chunk that a thread holds, as they came
template <typename T>
struct Held {
  static constexpr int EV = 16 / sizeof(T), N = BS_VECS * EV;
  uint32_t w[4 * BS_VECS];
  __device__ __forceinline__ float at(int k) const {
    if (sizeof(T) == 4) return __uint_as_float(w[k]);
    return (k & 1) ? bf16_hi(w[k >> 1]) : bf16_lo(w[k >> 1]);
  }
  __device__ __forceinline__ void mask(int k) {
    if (sizeof(T) == 4) w[k] = 0xff800000u;
    else w[k >> 1] = (k & 1) ? (w[k >> 1] & 0xffffu) | 0xff800000u : (w[k >> 1] & 0xffff0000u) | 0xff80u;
  }
  // a bit for every value above `cut`, and whose bit it is (bf16 two at a time: the cut as the next bf16 value that is not above it)
  static __device__ __forceinline__ int place(int bit) { return sizeof(T) == 4 ? bit : (bit & 15) * 2 + (bit >> 4); }
  __device__ __forceinline__ uint32_t over(float cut) const {
    static_assert(sizeof(T) == 4 || N == 32, "sixteen words of two");
    uint32_t hits = 0u;
    if (sizeof(T) == 4) {
#pragma unroll
      for (int k = 0; k < N; ++k) hits |= at(k) > cut ? 1u << k : 0u;
    } else {
      const __nv_bfloat162 c = __bfloat162bfloat162(__float2bfloat16_rd(cut));
#pragma unroll
      for (int j = 0; j < 4 * BS_VECS; ++j) hits |= __hgt2_mask(*reinterpret_cast<const __nv_bfloat162*>(&w[j]), c) & (0x10001u << j);
    }
    return hits;
  }
  __device__ __forceinline__ float max() const {            // (NaN only where there is nothing else)
    if (sizeof(T) == 4) {
      float m = at(0);
#pragma unroll
      for (int k = 1; k < N; ++k) m = fmaxf(m, at(k));
      return m;
    }
    __nv_bfloat162 m = *reinterpret_cast<const __nv_bfloat162*>(&w[0]);
#pragma unroll
    for (int j = 1; j < 4 * BS_VECS; ++j) m = __hmax2(m, *reinterpret_cast<const __nv_bfloat162*>(&w[j]));
    return fmaxf(__low2float(m), __high2float(m));
  }
};

// The n largest keys of the list's first c, in order, to its front.  (They differ: a key's place is the number of larger ones, which four neighbours count.)
__device__ __forceinline__ void keep_largest(uint64_t* list, uint64_t* sorted, int c, int n) {
  const uint32_t quad = 0xfu << (threadIdx.x & 28);
  for (int i = threadIdx.x >> 2; i < c; i += BS_THREADS / 4) {
    const uint64_t key = list[i];
    int r = 0;
#pragma unroll 4
    for (int j = threadIdx.x & 3; j < c; j += 4) r += list[j] > key ? 1 : 0;
    r += __shfl_xor_sync(quad, r, 1);
    r += __shfl_xor_sync(quad, r, 2);
    if ((threadIdx.x & 3) == 0 && r < n) sorted[r] = key;
  }
  __syncthreads();
  if (threadIdx.x < min(c, n)) list[threadIdx.x] = sorted[threadIdx.x];
  __syncthreads();
}

constexpr int BS_SPAN = 32 * BS_VECS, BS_SLOT = (BS_SPAN + 1) * 16;      // vectors of a chunk that a warp reads, and bytes of the aligned ones that hold them
struct PartShared {
  uint8_t ring[BS_STAGES][BS_THREADS / 32][BS_SLOT];
  uint64_t list[BS_CAP], sorted[BS_MAX_N];
  uint32_t box[3], count, tops[8];
  float part_m[8], part_s[8];
};

// One part of one row: every parts-th chunk, so that a masked stretch of the vocabulary is shared out.  T: bf16 or fp32 logits.  Rows may start at any
// element: aligned vectors go to shared memory (each holds a byte of the row, and a vector lies within a page), the width of the reads there goes by the
// row's address (ALIGN).  Which thread adds what does not, and equal rows have equal sums.  A warp's span is its own: no block waits for another warp's.
template <typename T, int ALIGN>
__device__ __forceinline__ void beam_part(PartShared& sh, BeamStats* stats, uint64_t* best, const uint8_t* at, int V, int part, int parts, int n) {
  constexpr int EV = Held<T>::EV, N = Held<T>::N, CHUNK = BS_THREADS * BS_VECS;      // (vectors)
  uint64_t* list = sh.list;
  uint32_t *box = sh.box, &count = sh.count;
  float *part_m = sh.part_m, *part_s = sh.part_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int by = ALIGN == 16 ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(at) & 15);
  const int vecs = (V + EV - 1) / EV, held = (V * static_cast<int>(sizeof(T)) + by + 15) / 16;
  const int step = parts * CHUNK, first = part * CHUNK + warp * BS_SPAN;      // (this warp's vectors)
  const uint8_t* src = at - by;
  const uint32_t ring = smem_u32(sh.ring) + warp * BS_SLOT;
  constexpr uint32_t STAGE = (BS_THREADS / 32) * BS_SLOT;
  auto fetch = [&](int v0, int slot) {
#pragma unroll
    for (int j = 0; j < BS_VECS; ++j) {
      const int vi = v0 + j * 32 + lane;
      if (vi < held) copy16_async(ring + slot * STAGE + (j * 32 + lane) * 16, src + 16ll * vi);
    }
    if (ALIGN != 16 && lane == 0 && v0 + BS_SPAN < held) copy16_async(ring + slot * STAGE + BS_SPAN * 16, src + 16ll * (v0 + BS_SPAN));
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < BS_STAGES - 1; ++i) fetch(min(first + i * step, held), i);      // (held: nothing)
  int slot = 0;
  float m = -INFINITY, s = 0.f;
  // Candidates are above this.  Once the list holds n that is the last one's value: of equal ones the lower tokens came first.
  float above = -INFINITY;
  bool low_cut = true;
  const uint32_t enough = max(2 * n, 32);
  for (int v0 = first; v0 - warp * BS_SPAN < vecs; v0 += step) {      // (as often in every warp: they meet)
    asm volatile("cp.async.wait_group %0;" ::"n"(BS_STAGES - 2) : "memory");
    __syncwarp();
    Held<T> x;
    const uint32_t mine_at = ring + slot * STAGE + lane * 16 + by;
#pragma unroll
    for (int j = 0; j < BS_VECS; ++j) read_words<ALIGN>(x.w + 4 * j, mine_at + j * 512);
    // (the last chunk's slot: this warp is through with it)
    fetch(min(v0 + (BS_STAGES - 1) * step, held), slot == 0 ? BS_STAGES - 1 : slot - 1);
    slot = slot + 1 == BS_STAGES ? 0 : slot + 1;
    const bool more = v0 - warp * BS_SPAN + step < vecs;
    // the token of x.at(k)
    auto token = [&](int k) { return static_cast<uint32_t>((v0 + (k / EV) * 32 + lane) * EV + (k % EV)); };
    if (v0 + BS_SPAN > V / EV) {                     // behind the row's last token
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (token(k) >= static_cast<uint32_t>(V)) x.mask(k);
    }
    // Maximum and sum of exponentials of what the thread holds.  One product and sum an element: 2^(x log2 e - c) with c the rounded m log2 e, and what the
    // rounding took is put back into the sum.  That is at most half a step of c, 64 below |m| = 2^30 (c < 2^31): neither factor is flushed there.  From 2^30 on (fp32 logits
    // lost their whole sum from 1.49e9 on) the longer way.  What is not finite shows up in the maximum or the sum and is masked on that way.
    float cm = x.max(), cs = 0.f;
    if (!(cm >= -INFINITY)) cm = -INFINITY;                  // (NaN alone)
    if (cm != -INFINITY) {
      const float c = cm * LOG2E;
      float2 t[2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
      for (int k = 0; k < N; k += 2) {
        const float2 y = fma2(make_float2(x.at(k), x.at(k + 1)), make_float2(LOG2E, LOG2E), make_float2(-c, -c));
        t[(k >> 1) & 1] = add2(t[(k >> 1) & 1], make_float2(ex2(y.x), ex2(y.y)));
      }
      cs = ((t[0].x + t[0].y) + (t[1].x + t[1].y)) * ex2(fmaf(-cm, LOG2E, c));
      if (!(cs < INFINITY) || !(fabsf(cm) < BS_SHORT)) {
#pragma unroll
        for (int k = 0; k < N; ++k)
          if (!isfinite(x.at(k))) x.mask(k);
        cm = x.max();
        cs = 0.f;
        if (cm != -INFINITY) {
#pragma unroll
          for (int k = 0; k < N; ++k) cs += exp_down(x.at(k) - cm);
        }
      }
      if (cm > m) {
        s = (m != -INFINITY ? s * exp_down(m - cm) : 0.f) + cs;
        m = cm;
      } else if (cm != -INFINITY) {
        s += cs * exp_down(cm - m);
      }
    }
    if (low_cut) {
      if (!__syncthreads_or(cm != -INFINITY)) continue;      // (a masked stretch)
      // A cut of the chunk's own while the list is short of n: at least n threads' maxima are not below it, found from the largest one down by steps that
      // double, then by halving.  Little more than n elements are above it.
      const uint32_t key = order_f32(cm);
      const uint32_t wtop = __reduce_max_sync(0xffffffffu, key);
      if (lane == 0) sh.tops[warp] = wtop;
      __syncthreads();
      uint32_t lo = __reduce_max_sync(0xffffffffu, sh.tops[lane & 7]), hi = lo + 1u, step = 1u << 20;
      int got;
      for (;;) {
        lo = lo > step ? lo - step : 1u;
        step <<= 1;
        got = __syncthreads_count(key >= lo);
        if (got >= n || lo == 1u) break;
        hi = lo;
      }
      while (got > n + n / 4 + 2 && hi - lo > 1u) {
        const uint32_t mid = lo + ((hi - lo) >> 1);
        const int c = __syncthreads_count(key >= mid);
        if (c >= n) lo = mid, got = c;
        else hi = mid;
      }
      const uint32_t under = lo - 1u;                       // (the next value below; 0x7fffffff would be -0, which is none)
      above = lo <= 0x00800000u ? -INFINITY : unorder_f32(under - (under == 0x7fffffffu ? 1u : 0u));
    }
    // What few threads do they do one element after the other, from shared memory: unrolled it took registers from the stream.  An element as one number: its
    // value, then the lower token first.
    auto keyed = [&](int k) {
      const uint32_t from = mine_at + (k / EV) * 512 + (k % EV) * sizeof(T);
      uint32_t w;
      if (sizeof(T) == 4) {
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(from) : "memory");
      } else {
        uint16_t h;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(from) : "memory");
        w = static_cast<uint32_t>(h) << 16;
      }
      const uint32_t o = order_f32(__uint_as_float(w));
      return o && token(k) < static_cast<uint32_t>(V) ? (static_cast<uint64_t>(o) << 32 | (0xffffffffu - token(k))) : 0ull;
    };
    bool full = low_cut && more;
    if (cm > above) {
      uint32_t hits = x.over(above);
      uint32_t i = atomicAdd(&count, static_cast<uint32_t>(__popc(hits)));
      for (; hits; hits &= hits - 1u, ++i) {
        if (i < BS_CAP) list[i] = keyed(Held<T>::place(__ffs(hits) - 1));
        full |= i >= (more ? enough : BS_CAP);
      }
    }
    if (!__syncthreads_or(full)) continue;
    int c = static_cast<int>(count);
    if (c > BS_CAP) {      // many equal or rising values: of the list and this chunk together those above a cut that leaves at least n, found by halving
      const uint32_t start = 0xffffffffu - static_cast<uint32_t>(v0 - warp * BS_SPAN) * EV;
      auto earlier = [&](int e) {                            // (of earlier chunks: this one's are looked at where they came from)
        const uint64_t key = list[tid + e * BS_THREADS];
        return static_cast<uint32_t>(key) > start ? key : 0ull;
      };
      int turn = 0, found = c;
      // (values first, then tokens; at least n are >= cut, fewer than n are >= end)
      uint64_t cut = static_cast<uint64_t>(above == -INFINITY ? 1u : order_f32(above) + 1u) << 32, end = ~0ull;
#pragma unroll 1
      while (found > BS_CAP / 4) {
        const uint64_t mid = cut + ((end - cut) >> 1);
        int mine = 0;
#pragma unroll 1
        for (int k = 0; k < N; ++k) mine += keyed(k) >= mid ? 1 : 0;
#pragma unroll 1
        for (int e = 0; e < BS_CAP / BS_THREADS; ++e) mine += earlier(e) >= mid ? 1 : 0;
        const int got = block_count(mine, box, turn);
        if (got >= n) cut = mid, found = got;
        else end = mid;
      }
      uint64_t kept[BS_CAP / BS_THREADS];
#pragma unroll
      for (int e = 0; e < BS_CAP / BS_THREADS; ++e) kept[e] = earlier(e);
      __syncthreads();
      if (tid == 0) count = 0u;
      __syncthreads();
#pragma unroll 1
      for (int k = 0; k < N; ++k) {
        const uint64_t key = keyed(k);
        if (key >= cut) list[atomicAdd(&count, 1u)] = key;
      }
#pragma unroll
      for (int e = 0; e < BS_CAP / BS_THREADS; ++e)
        if (kept[e] >= cut) list[atomicAdd(&count, 1u)] = kept[e];
      if (tid < 3) box[tid] = 0u;
      __syncthreads();
      c = static_cast<int>(count);
    }
    keep_largest(list, sh.sorted, c, n);
    if (tid == 0) count = min(c, n);
    if (c >= n) above = unorder_f32(static_cast<uint32_t>(list[n - 1] >> 32)), low_cut = false;
    __syncthreads();
  }

  asm volatile("cp.async.wait_all;" ::: "memory");          // (empty groups: nothing is on its way)
  const float wm = warp_max(m);
  const float ws = warp_sum(m != -INFINITY ? s * exp_down(m - wm) : 0.f);
  if (lane == 0) part_m[warp] = wm, part_s[warp] = ws;
  __syncthreads();
  if (warp == 0) {
    const float pm = lane < 8 ? part_m[lane] : -INFINITY;
    const float top = warp_max(pm);
    const float sum = warp_sum(pm != -INFINITY ? part_s[lane & 7] * exp_down(pm - top) : 0.f);
    if (lane == 0) *stats = {top, top == -INFINITY ? 0.f : sum};
  }
  const int c = static_cast<int>(count);
  keep_largest(list, sh.sorted, c, n);
  if (tid < n) best[tid] = tid < c ? list[tid] : 0ull;
}

// the same place in the shared memory of the cluster's first block, as an ordinary address
template <typename T>
__device__ __forceinline__ T* in_first_block(T* at) {
  T* r;
  asm("mapa.u64 %0, %1, 0;" : "=l"(r) : "l"(at));
  return r;
}

struct BeamCall {
  BeamStats* stats;              // [rows * parts]
  uint64_t* best;                // [rows * parts][n]
  const void* logits;
  long long stride;
  const float *score, *weight;
  const uint8_t* ended;
  float* out_score;
  int32_t* out_parent;
  int64_t* out_token;
  uint8_t* out_ended;
  int V, parts, W, n;
  long long end_token;
};

template <typename T>
__device__ __forceinline__ void beam_one_part(PartShared& sh, const BeamCall& p, BeamStats* st, uint64_t* out) {      // (where its statistics and its best go)
  const int row = blockIdx.x / p.parts, part = blockIdx.x - row * p.parts;
  if (threadIdx.x == 0) sh.box[0] = sh.box[1] = sh.box[2] = sh.count = 0u;
  pdl_sync();
  if (!beam_reads(p.score, p.weight, p.ended, row)) return;       // (the join does not look at this row either)
  __syncthreads();
  const uint8_t* at = static_cast<const uint8_t*>(p.logits) + static_cast<long long>(row) * p.stride * static_cast<long long>(sizeof(T));
  const int by = static_cast<int>(reinterpret_cast<uintptr_t>(at) & 15);
  if (by == 0) beam_part<T, 16>(sh, st, out, at, p.V, part, p.parts, p.n);
  else if (by == 8) beam_part<T, 8>(sh, st, out, at, p.V, part, p.parts, p.n);
  else if (sizeof(T) == 4 || by % 4 == 0) beam_part<T, 4>(sh, st, out, at, p.V, part, p.parts, p.n);
  else beam_part<T, sizeof(T)>(sh, st, out, at, p.V, part, p.parts, p.n);
}

template <typename T>
__global__ void __launch_bounds__(BS_THREADS, BS_BLOCKS) beam_part_kernel(const __grid_constant__ BeamCall p) {
  extern __shared__ __align__(16) uint8_t bs_raw[];
  beam_one_part<T>(*reinterpret_cast<PartShared*>(bs_raw), p, p.stats + blockIdx.x, p.best + static_cast<long long>(blockIdx.x) * p.n);
}

// The n best of one request.  Candidate c of its W * parts * n: beam, part, place; its rank stands in shared memory (in registers, unrolled, the code took longer
// to arrive than to run).
template <int THREADS>
struct JoinShared {
  static constexpr int CAP = BS_MAX_N + 32;
  // total = (x - top) + base: a row may hold nothing but lowest values; base of an ended beam: its score
  double base[BS_MAX_W], tops[BS_MAX_W];
  float factor[BS_MAX_W];
  uint64_t list_key[CAP], list_at[CAP], warp_most[THREADS / 32];      // rank, (beam, token)
  double list_total[CAP];
  uint32_t box[3], count;
  int bins[BJ_BINS], warp_sum_s[THREADS / 32], box_bin, box_upto;
  uint8_t kind[BS_MAX_W];                              // 0: no candidates, 1: logits, 2: ended
};
template <int THREADS>
__device__ __forceinline__ void beam_join(JoinShared<THREADS>& sh, uint64_t* bj_key, const BeamCall& p, int b, const BeamStats* stats, const uint64_t* mine_of) {      // (of the request)
  double *base = sh.base, *tops = sh.tops, *list_total = sh.list_total;
  uint64_t *list_key = sh.list_key, *list_at = sh.list_at, *warp_most = sh.warp_most;
  uint32_t *box = sh.box, &count = sh.count;
  int *bins = sh.bins, *warp_sum_s = sh.warp_sum_s, &box_bin = sh.box_bin, &box_upto = sh.box_upto;
  uint8_t* kind = sh.kind;
  const float *score = p.score, *weight = p.weight;
  const uint8_t* ended = p.ended;
  const int W = p.W, parts = p.parts, n = p.n;
  const long long end_token = p.end_token;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per_row = parts * n, all = W * per_row;
  uint64_t* bj_e = bj_key + all;
  auto total_of = [&](int w, uint64_t e) { return kind[w] == 2 ? base[w] : (static_cast<double>(unorder_f32(static_cast<uint32_t>(e >> 32))) - tops[w]) + base[w]; };
  auto place_of = [&](int w, uint64_t e) {
    return static_cast<uint64_t>(w) << 32 | (kind[w] == 2 ? static_cast<uint32_t>(end_token) : 0xffffffffu - static_cast<uint32_t>(e));
  };
  uint64_t e[4];                                       // (the first of a thread's candidates, on their way while the sums are added up)
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = tid + i * THREADS < all ? mine_of[tid + i * THREADS] : 0ull;
  for (int w = warp; w < W; w += THREADS / 32) {       // a warp a beam
    const int row = b * W + w;
    const float s = score[row], f = weight ? weight[row] : 1.f;
    const bool over = ended && ended[row];
    const BeamStats t0 = lane < parts ? stats[w * parts + lane] : BeamStats{-INFINITY, 0.f};      // (of a row that was not read: anything)
    int k = !isfinite(s) || !isfinite(f) || !(f > 0.f) ? 0 : over ? 2 : 1;
    double log_sum = 0.0, peak = 0.0;
    if (k == 1) {
      float top = t0.m;
      for (int i = lane + 32; i < parts; i += 32) top = fmaxf(top, stats[w * parts + i].m);
      top = warp_max(top);
      double sum = t0.m == -INFINITY ? 0.0 : static_cast<double>(t0.s) * exp(static_cast<double>(t0.m) - static_cast<double>(top));
      for (int i = lane + 32; i < parts; i += 32) {
        const BeamStats t = stats[w * parts + i];
        if (t.m != -INFINITY) sum += static_cast<double>(t.s) * exp(static_cast<double>(t.m) - static_cast<double>(top));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (top == -INFINITY) k = 0;                       // everything masked: nothing to go on with
      else peak = top, log_sum = log(sum);
    }
    if (lane == 0) base[w] = static_cast<double>(s) - log_sum, tops[w] = peak, sh.factor[w] = f, kind[w] = k;
  }
  __syncthreads();
  uint64_t most = 0ull;
  int mine = 0;
#pragma unroll 1
  for (int c = tid, i = 0; c < all; c += THREADS, ++i) {
    const int w = c / per_row, k = kind[w];
    const uint64_t x = k != 1 ? 0ull : i == 0 ? e[0] : i == 1 ? e[1] : i == 2 ? e[2] : i == 3 ? e[3] : mine_of[c];
    // (an ended beam's one candidate stands in its first place; what the memory holds there is not looked at)
    const uint64_t key = (k == 2 ? c == w * per_row : x != 0ull) ? order_f64(total_of(w, x) * static_cast<double>(sh.factor[w])) : 0ull;
    bj_key[c] = key, bj_e[c] = x;
    mine += key != 0ull;
    most = max(most, key);
  }
  // All candidates if the list holds them, else those above a cut that leaves at least n.  Candidates are counted by their distance from the largest, 16 bins
  // to every doubling of it; what a bin holds too much of (equal or nearly equal ranks) is found by halving, first of ranks, then of places.
  int turn = 0, found = block_count(mine, box, turn);    // (its barrier: keys and totals are there)
  uint64_t cut = 1ull, tie = ~0ull;
  const int room = n + 32;
  if (found > room) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (lane == 0) warp_most[warp] = most;
    for (int i = tid; i < BJ_BINS; i += THREADS) bins[i] = 0;
    __syncthreads();
    uint64_t top = 0ull;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) top = max(top, warp_most[i]);
    const double best_rank = unorder_f64(top);
    auto bin_of = [&](uint64_t key) {                       // (monotone: the same subtraction and conversion for all)
      const int i = static_cast<int>(__float_as_uint(static_cast<float>(best_rank - unorder_f64(key))) >> 19) - (104 << 4);
      return i < 0 ? 0 : i < BJ_BINS ? i : BJ_BINS - 1;
    };
#pragma unroll 2
    for (int c = tid; c < all; c += THREADS)
      if (bj_key[c]) atomicAdd(&bins[bin_of(bj_key[c])], 1);
    __syncthreads();
    // the bin in which the n-th is
    constexpr int OWN = BJ_BINS / THREADS;
    int upto = 0;
#pragma unroll
    for (int i = 0; i < OWN; ++i) upto += bins[OWN * tid + i];
    const int own = upto;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) warp_sum_s[warp] = upto;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i)
      if (i < warp) upto += warp_sum_s[i];
    if (upto >= n && upto - own < n) {                      // (one thread)
      int bin = OWN * tid, sum = upto - own + bins[bin];
      while (sum < n) sum += bins[++bin];
      box_bin = bin, box_upto = sum;
    }
    __syncthreads();
    const int last = box_bin;
    found = box_upto;
    if (found <= room) {
      // the lowest rank of the bins that count: what is below stays out
      uint64_t least = ~0ull;
#pragma unroll 2
      for (int c = tid; c < all; c += THREADS)
        if (bj_key[c] && bin_of(bj_key[c]) <= last) least = min(least, bj_key[c]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
      if (lane == 0) warp_most[warp] = least;
      __syncthreads();
      cut = ~0ull;
#pragma unroll
      for (int i = 0; i < THREADS / 32; ++i) cut = min(cut, warp_most[i]);
    }
    auto count_from = [&](uint64_t from) {
      int m = 0;
#pragma unroll 4
      for (int c = tid; c < all; c += THREADS) m += bj_key[c] >= from;
      return block_count(m, box, turn);
    };
    uint64_t lo = cut, hi = top + 1ull;
    while (found > room && hi - lo > 1ull) {
      const uint64_t mid = lo + ((hi - lo) >> 1);
      const int c = count_from(mid);
      if (c >= n) lo = mid, found = c;
      else hi = mid;
    }
    cut = lo;
    uint64_t below = 0ull;                                  // (places of equal ranks: the fewest of the first ones that are enough)
    while (found > room) {
      const uint64_t mid = below + ((tie - below) >> 1);
      mine = 0;
#pragma unroll 1
      for (int c = tid; c < all; c += THREADS) mine += bj_key[c] > cut || (bj_key[c] == cut && place_of(c / per_row, bj_e[c]) <= mid);
      const int c = block_count(mine, box, turn);
      if (c >= n) tie = mid, found = c;
      else below = mid + 1ull;
    }
  }
#pragma unroll 1
  for (int c = tid; c < all; c += THREADS) {
    const uint64_t key = bj_key[c];
    if (key < cut) continue;
    const int w = c / per_row;
    const uint64_t e = bj_e[c], at = place_of(w, e);
    if (key == cut && at > tie) continue;
    const uint32_t o = atomicAdd(&count, 1u);
    list_key[o] = key, list_at[o] = at, list_total[o] = total_of(w, e);
  }
  __syncthreads();
  const uint32_t quad = 0xfu << (lane & 28);
  for (int i = tid >> 2; i < found; i += THREADS / 4) {
    const uint64_t k = list_key[i], at = list_at[i];
    int rank = 0;
#pragma unroll 4
    for (int j = tid & 3; j < found; j += 4) {
      const uint64_t kj = list_key[j], aj = list_at[j];
      rank += (kj > k) | ((kj == k) & (aj < at));
    }
    rank += __shfl_xor_sync(quad, rank, 1);
    rank += __shfl_xor_sync(quad, rank, 2);
    if ((tid & 3) == 0 && rank < n) {
      const int w = static_cast<int>(at >> 32), o = b * n + rank;
      const uint32_t v = static_cast<uint32_t>(at);
      p.out_score[o] = static_cast<float>(list_total[i]);
      p.out_parent[o] = w;
      p.out_token[o] = v;
      if (p.out_ended) p.out_ended[o] = kind[w] == 2 || static_cast<long long>(v) == end_token;
    }
  }
  for (int i = found + tid; i < n; i += THREADS) {
    p.out_score[b * n + i] = -INFINITY;
    p.out_parent[b * n + i] = -1;
    p.out_token[b * n + i] = -1;
    if (p.out_ended) p.out_ended[b * n + i] = 1;
  }
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) beam_join_kernel(const __grid_constant__ BeamCall p) {
  extern __shared__ uint64_t bj_key[];                 // [W * parts * n] ranks as ordered numbers, 0: none; behind them the candidates
  __shared__ JoinShared<THREADS> sh;
  if (threadIdx.x == 0) sh.box[0] = sh.box[1] = sh.box[2] = sh.count = 0u;
  pdl_sync();
  const long long first = static_cast<long long>(blockIdx.x) * p.W * p.parts;
  beam_join<THREADS>(sh, bj_key, p, blockIdx.x, p.stats + first, p.best + first * p.n);
}

// Both in one launch where a request's parts are few and all requests run at once (beam_one_launch): a cluster a request, whose blocks leave what they found in the
// first one's shared memory.  (One beam of two over 2051 tokens: 6.45 -> 5.9 us in a graph, the call 16.1 -> 13.6.)
template <typename T>
__global__ void __launch_bounds__(BS_THREADS) beam_small_kernel(const __grid_constant__ BeamCall p) {
  extern __shared__ __align__(16) uint8_t bs_raw[];
  __shared__ JoinShared<BS_THREADS> sh;
  __shared__ BeamStats stats[BS_CLUSTER];
  __shared__ uint64_t best[BS_CLUSTER * BS_MAX_N];
  if (threadIdx.x == 0) sh.box[0] = sh.box[1] = sh.box[2] = sh.count = 0u;
  cluster_sync_all();                                  // (the first block runs)
  const int rank = cluster_ctarank();
  beam_one_part<T>(*reinterpret_cast<PartShared*>(bs_raw), p, in_first_block(stats + rank), in_first_block(best + rank * p.n));
  cluster_sync_all();
  if (rank == 0) beam_join<BS_THREADS>(sh, reinterpret_cast<uint64_t*>(bs_raw), p, blockIdx.x / (p.W * p.parts), stats, best);
}

// ---- states that follow their beams ----------------------------------------------------------------------------------------------
// state[slot[b][i]] = what state[slot[b][parent[b][i]]] was.  A thread owns a vector's place in all W rows of a request: it reads what moves there, then
// writes, so that rows may change places without a second copy of the state.  All states in one launch (64 a launch).  Bound by HBM: 8 requests of 8 beams,
// 413 MB read and 413 written, 131 us, 98 % of a copy's rate; one small request 2.0 us, the launch.
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

// Parts of a row: as many blocks as run at a time, of equally many chunks, and no more candidates of a request than the second kernel holds.
static int beam_parts(int requests, int width, int vocab, int n, int elem) {
  const int chunk = BS_THREADS * BS_VECS * 16 / elem, chunks = (vocab + chunk - 1) / chunk;
  const long long rows = static_cast<long long>(requests) * width, blocks = static_cast<long long>(sm_count()) * BS_BLOCKS / rows;
  int parts = static_cast<int>(blocks < 1 ? 1 : blocks < chunks ? blocks : chunks);
  const int most = BJ_ALL / (width * n);
  if (parts > most) parts = most;
  const int each = (chunks + parts - 1) / parts;
  return (chunks + each - 1) / each;
}

// One launch where a request's parts are a cluster's work and all clusters run at once, by the device's own count: its blocks take more registers (bf16: three an SM, not
// four) and stay until their request has been joined, so a second wave of them costs more than a second launch.  One / two launches, bf16, where all run at once: 1 x 2 rows of
// 2051 6.2 / 6.7 us, 100 x 1 of 32003 7.7 / 9.5, 64 x 4 of 8192 7.5 / 7.7, 111 x 3 of 156940 39.8 / 46.1; where they do not: 64 x 4 of 32003 18.3 / 14.8, of 156940 42.0 / 33.0, 74 x 8 of
// 2051 14.7 / 12.8, 300 x 8 of 8192 42.6 / 26.5.  fp32: 128 x 2 of 32003 14.4 / 15.7, 296 x 2 of 8192 9.7 / 10.2; 74 x 4 of 8192 12.8 / 9.3, 74 x 8 of 156940 97 / 69.  (fp32
// clusters of eight all run at once but unevenly over the SMs: 40 x 8 of 156940 61.3 / 52.4, 64 x 4 of 8192 10.7 / 9.2 stay one.)
template <auto Kernel>
static bool beam_fits(int requests, int cluster) {
  if (rm_smem<Kernel>(sizeof(PartShared)) != cudaSuccess) {      // (no device: sizes are asked for, nothing runs)
    cudaGetLastError();
    return true;
  }
  return requests <= rm_clusters<Kernel>(cluster, BS_THREADS, sizeof(PartShared));
}
static bool beam_one_launch(int requests, int width, int parts, bool f32) {
  if (width * parts > BS_CLUSTER) return false;
  return f32 ? beam_fits<beam_small_kernel<float>>(requests, width * parts) : beam_fits<beam_small_kernel<__nv_bfloat16>>(requests, width * parts);
}

}  // namespace vb

using namespace vb;

extern "C" size_t vb_beam_select_workspace_bytes(int requests, int width, int vocab, int n, int logits_f32) {
  if (requests <= 0 || width <= 0 || width > BS_MAX_W || vocab <= 0 || n <= 0 || n > BS_MAX_N) return 0;
  const int parts = beam_parts(requests, width, vocab, n, logits_f32 ? 4 : 2);
  return beam_one_launch(requests, width, parts, logits_f32) ? 0 : static_cast<size_t>(requests) * width * parts * (sizeof(BeamStats) + 8ull * n);
}

extern "C" int vb_beam_select(float* d_score, int32_t* d_parent, int64_t* d_token, uint8_t* d_out_ended, const void* d_logits, int64_t row_stride, int logits_f32,
                              const float* d_beam_score, const float* d_weight, const uint8_t* d_ended, int requests, int width, int vocab, int n, int64_t end_token,
                              void* d_workspace, size_t workspace_bytes, void* stream) {
  VB_CHECK_ARG(d_score && d_parent && d_token && d_logits && d_beam_score, "vb_beam_select: null pointer");
  VB_CHECK_ARG(requests > 0 && width > 0 && width <= BS_MAX_W && n > 0 && n <= BS_MAX_N, "vb_beam_select: %d requests of %d beams (1 to %d), the best %d (1 to %d)", requests,
               width, BS_MAX_W, n, BS_MAX_N);
  VB_CHECK_ARG(vocab > 0 && vocab <= (1 << 24), "vb_beam_select: vocabulary of %d (1 to 2^24)", vocab);
  VB_CHECK_ARG(reinterpret_cast<uintptr_t>(d_logits) % (logits_f32 ? 4 : 2) == 0, "vb_beam_select: logits that are not aligned to their type");
  VB_CHECK_ARG(row_stride >= 0, "vb_beam_select: row stride %lld", static_cast<long long>(row_stride));
  VB_CHECK_ARG(!(d_ended || d_out_ended) || (end_token >= 0 && end_token < vocab), "vb_beam_select: end token %lld outside the vocabulary of %d",
               static_cast<long long>(end_token), vocab);
  const int parts = beam_parts(requests, width, vocab, n, logits_f32 ? 4 : 2);
  const long long blocks = static_cast<long long>(requests) * width * parts;
  VB_CHECK_ARG(blocks <= 0x7fffffffll && static_cast<long long>(requests) * n <= 0x7fffffffll, "vb_beam_select: %lld parts of rows", blocks);
  const size_t need = vb_beam_select_workspace_bytes(requests, width, vocab, n, logits_f32);
  VB_CHECK_ARG(need == 0 || (d_workspace && workspace_bytes >= need && reinterpret_cast<uintptr_t>(d_workspace) % 8 == 0), "vb_beam_select: workspace of %zu bytes, not %zu",
               workspace_bytes, need);
  uint64_t* best = static_cast<uint64_t*>(d_workspace);
  BeamStats* stats = need ? reinterpret_cast<BeamStats*>(best + blocks * n) : nullptr;
  BeamCall p = {stats, best, d_logits, static_cast<long long>(row_stride), d_beam_score, d_weight, d_ended, d_score, d_parent, d_token, d_out_ended,
                vocab, parts, width, n, static_cast<long long>(end_token)};
  if (need == 0) {                                     // (beam_fits has asked for their shared memory)
    if (logits_f32) VB_LAUNCH_PDL_CLUSTER(beam_small_kernel<float>, static_cast<unsigned>(blocks), BS_THREADS, sizeof(PartShared), stream, width * parts, p);
    else VB_LAUNCH_PDL_CLUSTER(beam_small_kernel<__nv_bfloat16>, static_cast<unsigned>(blocks), BS_THREADS, sizeof(PartShared), stream, width * parts, p);
    return 0;
  }
  VB_CHECK_CUDA(logits_f32 ? rm_smem<beam_part_kernel<float>>(sizeof(PartShared)) : rm_smem<beam_part_kernel<__nv_bfloat16>>(sizeof(PartShared)));
  if (logits_f32) VB_LAUNCH_PDL(beam_part_kernel<float>, static_cast<unsigned>(blocks), BS_THREADS, sizeof(PartShared), stream, p);
  else VB_LAUNCH_PDL(beam_part_kernel<__nv_bfloat16>, static_cast<unsigned>(blocks), BS_THREADS, sizeof(PartShared), stream, p);
  const size_t all = static_cast<size_t>(width) * parts * n;
  // Fewer threads meet sooner, more get through longer lists.  256 / 512 threads: 80 to 320 candidates a request 8.2 / 8.9 and 12.1 / 12.8 us, 1024 42.2 / 41.1, 2560 14.7 /
  // 12.8, 8192 30.1 / 22.5 (1024 threads: 14.3 for 2560, 22.3 for 8192).
  if (all <= BJ_FEW) {
    VB_LAUNCH_PDL(beam_join_kernel<256>, static_cast<unsigned>(requests), 256, all * 16, stream, p);
  } else {
    VB_CHECK_CUDA(rm_smem<beam_join_kernel<512>>(BJ_ALL * 16));
    VB_LAUNCH_PDL(beam_join_kernel<512>, static_cast<unsigned>(requests), 512, all * 16, stream, p);
  }
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
    // (a thread's registers hold its vector of every row: 8 requests of 8 rows 131 us, with room for 32 rows 503.  2 of 32 rows of 1 MB, 16 bytes a row at a time: 133;
    // 8 bytes 166, 4 bytes 162.)
    if (width <= 4) VB_LAUNCH_PDL(beam_reorder_kernel<4>, grid, BR_THREADS, 0, stream, t, d_parent, d_slots, width);
    else if (width <= 8) VB_LAUNCH_PDL(beam_reorder_kernel<8>, grid, BR_THREADS, 0, stream, t, d_parent, d_slots, width);
    else if (width <= 16) VB_LAUNCH_PDL(beam_reorder_kernel<16>, grid, BR_THREADS, 0, stream, t, d_parent, d_slots, width);
    else VB_LAUNCH_PDL(beam_reorder_kernel<32>, grid, BR_THREADS, 0, stream, t, d_parent, d_slots, width);
  }
  return 0;
}
