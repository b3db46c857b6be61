// What the operators share whose weights a row brings with it (lora.cu, moe_layer.cu): weights as the streamed operand of mma.sync (straight into registers in
// adapters' steps of few rows, else through shared memory), a few rows of activations as the other operand.  Few rows make these products a stream of weights,
// which mma.sync keeps up with (an m16n8k16 product takes 2 clocks of an SM for 512 bytes of weights that arrive in 22).
#pragma once
#include "common.cuh"

namespace vb {

// 16 bytes that are read once: past L1
__device__ __forceinline__ uint4 ldg_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// An fp32 value as three bf16 parts whose sum it is: the upper 8 bits of the significand, the next 8, the last 8 (cut off, not rounded, so that a part
// never overflows and nothing is lost).  What is not finite stays whole in the first part (inf - inf would make it NaN).
__device__ __forceinline__ float bf16_cut(float v) { return __uint_as_float(__float_as_uint(v) & 0xffff0000u); }
__device__ __forceinline__ void bf16_parts(float v, float& hi, float& mid, float& lo) {
  hi = bf16_cut(v);
  if ((__float_as_uint(v) & 0x7f800000u) == 0x7f800000u) {
    hi = __uint_as_float((__float_as_uint(v) & 0x7fffffffu) > 0x7f800000u ? 0x7fc00000u : __float_as_uint(v));
    mid = lo = 0.f;
    return;
  }
  const float r = v - hi;
  mid = bf16_cut(r);
  lo = r - mid;
}
// ... as two: the nearest bf16 value (cut off instead where that is infinite), and what is left, which is exact in fp32 and rounded by whoever packs it: together
// off by at most half a step of what 16 bits hold, 2^-17 of the value.
__device__ __forceinline__ void bf16_near(float v, float& hi, float& rest) {
  const bool finite = (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u;
  hi = __bfloat162float(__float2bfloat16_rn(v));
  if (finite && isinf(hi)) hi = bf16_cut(v);
  rest = finite ? v - hi : 0.f;
}
// two neighbours' upper halves as one register (both hold bf16 values)
__device__ __forceinline__ uint32_t pack_cut(float first, float second) {
  return __byte_perm(__float_as_uint(first), __float_as_uint(second), 0x7632);
}

// (distributed shared memory: the same place in another block of the cluster)
__device__ __forceinline__ float4 ld_dsmem_f32x4(const float* local_ptr, uint32_t cta_rank) {
  uint32_t raddr;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(raddr) : "r"(smem_u32(local_ptr)), "r"(cta_rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(raddr) : "memory");
  return v;
}

// The opt-in shared memory of a kernel, once per device.  (A flag of its own for every kernel: max_dyn_smem_once keeps one per type, and these share theirs.)
template <auto Kernel>
inline cudaError_t rm_smem(int bytes = VB_MAX_DYN_SMEM) {
  static std::atomic<unsigned long long> done{0ull};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 64 && (done.load(std::memory_order_acquire) >> dev & 1ull)) return cudaSuccess;
  e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_release);
  return e;
}

// How many clusters of `size` blocks run at a time (they live on one part of the chip each, so this is less than the blocks that fit divided by the size): asked for
// once per device, size and number of blocks an SM holds.  rm_smem first.
template <auto Kernel>
inline int rm_clusters(int size, int threads, size_t smem) {
  static std::atomic<int> known[16][5][9] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 1;
  const size_t per_sm = 228 * 1024 / (smem + 1024);
  std::atomic<int>& n = known[dev & 15][per_sm > 4 ? 4 : per_sm][size];
  int clusters = dev < 16 ? n.load(std::memory_order_relaxed) : 0;
  if (clusters > 0) return clusters;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(size);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&clusters, Kernel, &cfg) != cudaSuccess || clusters < 1) {
    cudaGetLastError();
    return 1;
  }
  if (dev < 16) n.store(clusters, std::memory_order_relaxed);
  return clusters;
}

}  // namespace vb
