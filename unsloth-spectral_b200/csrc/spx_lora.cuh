// What the two files of the adapter kernels share (spx_lora.cu, spx_lora_tc.cu).
#pragma once
#include <math.h>

#include <atomic>

#include "spx_common.cuh"

namespace spx {
namespace lora {

struct Params {
  const void *x, *y, *a, *b;
  void* out;
  int64_t xs, ys, os;
  const int32_t* ranks;
  const float* scales;
  const int4* tiles;
  const int32_t* order;
  float* t;      // [rows][SR] inner products, then one word: set when a wait expired
  int K, parts, R, SR, OUT, rows, slots;
  int width[SPX_LORA_MAX_PARTS];
};

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1);
template <>
__device__ __forceinline__ void mma<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                   uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack2(__half lo, __half hi) {
  return (uint32_t)__half_as_ushort(lo) | ((uint32_t)__half_as_ushort(hi) << 16);
}
__device__ __forceinline__ uint32_t pack2(__nv_bfloat16 lo, __nv_bfloat16 hi) {
  return (uint32_t)__bfloat16_as_ushort(lo) | ((uint32_t)__bfloat16_as_ushort(hi) << 16);
}

// Lets a kernel have `bytes` of dynamic shared memory (asked for once for a device and size: the
// call takes about 1 us of a launch).  `have`: what each device allows so far, one array a kernel.
template <typename F>
inline cudaError_t allow_smem(F kernel, int bytes, std::atomic<int> (&have)[64]) {
  int dev = 0;
  const cudaError_t d = cudaGetDevice(&dev);
  if (d != cudaSuccess) return d;
  if (dev >= 0 && dev < 64 && have[dev].load(std::memory_order_relaxed) >= bytes) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev >= 0 && dev < 64) have[dev].store(bytes, std::memory_order_relaxed);
  return e;
}

// Cluster helpers: partial sums are pushed into the shared memory of the CTA that adds them up
// (its start announced by cluster_started, their arrival by cluster_pushed), in a fixed order.
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_started() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_pushed() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t in_cta(const void* p, uint32_t rank) {   // address of p's counterpart
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return r;
}

// t of 16 rows (row r at t + r * ld; rows past `rows` and columns past the rank are zeros) as
// MMA fragments: f[ks][0] the high halves, f[ks][1] the low ones, each the four registers of
// step ks (row g k-pair 0, row g + 8 k-pair 0, row g k-pair 1, row g + 8 k-pair 1), where the
// k of lane c are ks * 16 + 4c..4c+3.  Two values of T hold t within (eps / 2)^2.
// sc: what rows g and g + 8 of the product are to be multiplied by.
template <typename T, int KS>
__device__ __forceinline__ void split_t(const float* t, int ld, int rows, int rank, int g, int c, uint4 (&f)[KS][2],
                                        float (&sc)[2]) {
  float4 tv[KS][2];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      tv[ks][h] = h * 8 + g < rows && ks * 16 < rank
                      ? *reinterpret_cast<const float4*>(t + (int64_t)(h * 8 + g) * ld + ks * 16 + 4 * c)
                      : make_float4(0.f, 0.f, 0.f, 0.f);
  sc[0] = sc[1] = 1.f;
  if (!__is_same(T, __nv_bfloat16)) {
    // f16: the row is scaled by a power of two so that its largest value is near 2^8 (no
    // overflow of the high parts, no underflow of the low parts)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float mx = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        mx = fmaxf(fmaxf(fmaxf(fabsf(tv[ks][h].x), fabsf(tv[ks][h].y)), fmaxf(fabsf(tv[ks][h].z), fabsf(tv[ks][h].w))), mx);
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      int ex = (int)((__float_as_uint(mx) >> 23) & 0xff) - 127 - 8;
      ex = max(-118, min(118, ex));
      const float dn = __uint_as_float((uint32_t)(127 - ex) << 23);
      sc[h] = __uint_as_float((uint32_t)(127 + ex) << 23);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) tv[ks][h].x *= dn, tv[ks][h].y *= dn, tv[ks][h].z *= dn, tv[ks][h].w *= dn;
    }
  }
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float4 v = tv[ks][e & 1];
      const float f0 = e < 2 ? v.x : v.z, f1 = e < 2 ? v.y : v.w;
      const T h0 = from_f<T>(f0), h1 = from_f<T>(f1);
      // an infinity has no low part
      const float l0 = fabsf(to_f(h0)) < INFINITY ? f0 - to_f(h0) : 0.f;
      const float l1 = fabsf(to_f(h1)) < INFINITY ? f1 - to_f(h1) : 0.f;
      hi[e] = pack2(h0, h1);
      lo[e] = pack2(from_f<T>(l0), from_f<T>(l1));
    }
    f[ks][0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    f[ks][1] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
}

// t = A x of tiles of up to 128 adjacent rows, on tcgen05 (spx_lora_tc.cu).
int shrink_block_launch(const Params& p, int dtype, int tiles, cudaStream_t st);
// out = y + scale * B t of the same tiles.
int expand_block_launch(const Params& p, int dtype, int tiles, cudaStream_t st);

}  // namespace lora
}  // namespace spx
