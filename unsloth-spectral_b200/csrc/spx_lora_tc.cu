// Adapters of prompts: t = A x of tiles of up to 128 adjacent rows of one slot (the first of
// the two kernels of spx_lora.cu, for tokens that lie together).  A stream of x with few
// columns beside it: TMA brings tiles of 128 rows x 64 values of x and of the slot's A
// (128-byte swizzle) through a ring of stages, one thread issues tcgen05.mma (M = 128 rows,
// N = parts * rank columns, f32 in tensor memory), and x is read once, whatever the rank.
// Bound by memory: 2 * N flops a byte of x at most.  Two CTAs an SM keep about 128 KB of x in
// flight, where the mma.sync kernel (fragments loaded by the warps that use them) had 8 warps
// an SM.  Few tiles: the CTAs of a cluster split k and add their sums over distributed shared
// memory in a fixed order.  Rows of the next sequence that a tile's box covers are computed
// and not stored.  Every wait is bounded; an expired one leaves NaN in t.
#include <cooperative_groups.h>
#include <cuda.h>

#include "spx_lora.cuh"
#include "spx_sm100.cuh"

namespace spx {
namespace lora {

using namespace sm100;
namespace cg = cooperative_groups;

constexpr int M = 128, KB = 64;            // rows of a tile, values of k in a stage
constexpr int XBYTES = M * KB * 2;

struct Cfg {
  int nb, groups, stages, cs;              // columns of a group, groups, stages of the ring, CTAs of a cluster
  size_t smem;
};

__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// K-major operand tiles of 128-byte rows, 128-byte swizzle: groups of eight rows 1024 bytes apart.
__device__ __forceinline__ uint64_t desc128(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | (1ull << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void umma(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void tld16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int u = 0; u < 16; ++u) v[u] = __uint_as_float(r[u]);
}

// 128 threads: thread 0 copies, thread 32 issues the MMAs, all four warps read the sums.
__global__ void __launch_bounds__(128) shrink_block_kernel(const __grid_constant__ CUtensorMap mx,
                                                           const __grid_constant__ CUtensorMap ma, const Params p,
                                                           const int nb, const int stages, const uint32_t idesc) {
  extern __shared__ uint8_t raw_smem[];
  __shared__ __align__(8) uint64_t bars[2 * 8 + 1];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  cg::cluster_group cl = cg::this_cluster();
  const int cs = (int)cl.num_blocks(), cr = (int)cl.block_rank();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int4 tile = p.tiles[blockIdx.x / cs];
  if (tile.x < 0) return;   // rows without an adapter: the whole cluster leaves
  const int tid = threadIdx.x, warp = tid >> 5;
  const int col0 = blockIdx.y * nb, row0 = p.order[tile.y];
  const uint32_t base = (smem_u32(raw_smem) + 1023u) & ~1023u;
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * 8, done = full0 + 16 * 8;
  const int sbytes = XBYTES + nb * KB * 2;
  uint32_t ncols = 32;
  while ((int)ncols < nb) ncols *= 2;
  if (warp == 0) {
    tmem_alloc(smem_u32(&s_tmem), ncols);
    tmem_relinquish();
  }
  if (tid == 0) {
    s_abort = 0;
    for (int s = 0; s < stages; ++s) mbar_init(full0 + 8 * s, 1), mbar_init(empty0 + 8 * s, 1);
    mbar_init(done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const Abort ab{&s_abort, reinterpret_cast<int*>(p.t + (int64_t)p.rows * p.SR)};
  const int steps = (p.K + KB - 1) / KB;   // CTA cr of the cluster takes steps cr, cr + cs, ...
  const int mine = steps > cr ? (steps - cr + cs - 1) / cs : 0;
  if (tid == 0) {
    int i = 0;
    for (; i < mine; ++i) {
      const int s = i % stages;
      if (i >= stages && !wait1(empty0 + 8 * s, (uint32_t)((i / stages - 1) & 1), ab)) break;
      const uint32_t dst = base + s * sbytes;
      const int k = (cr + i * cs) * KB;
      mbar_expect_tx(full0 + 8 * s, (uint32_t)sbytes);
      tma_2d(dst, &mx, k, row0, full0 + 8 * s);
      tma_2d(dst + XBYTES, &ma, k, tile.x * p.SR + col0, full0 + 8 * s);
    }
    if (i < mine) {   // given up: the copies in flight land before the shared memory goes
      for (int q = i > stages ? i - stages : 0; q < i; ++q) {
        const uint64_t t0 = gtimer();
        while (!mbar_try_wait_sleep(full0 + 8 * (q % stages), (uint32_t)((q / stages) & 1)) && gtimer() - t0 < kWaitNs) {
        }
      }
    }
  } else if (tid == 32) {
    for (int i = 0; i < mine; ++i) {
      const int s = i % stages;
      if (!wait1(full0 + 8 * s, (uint32_t)((i / stages) & 1), ab)) break;
      tc_fence_after();
      const uint32_t xa = base + s * sbytes, aa = xa + XBYTES;
#pragma unroll
      for (int ks = 0; ks < KB / 16; ++ks)
        umma(tmem, desc128(xa + 32 * ks), desc128(aa + 32 * ks), idesc, (i > 0 || ks > 0) ? 1u : 0u);
      umma_commit(empty0 + 8 * s);
    }
    if (mine > 0) umma_commit(done);
  }
  __syncwarp();
  bool ok = true;
  if (mine > 0) ok = waitw(done, 0, ab);
  ok = __syncthreads_and(ok && !*ab.flag);
  tc_fence_after();
  // thread = row (tensor memory lane); the sums of a part past its slot's rank are exact zeros
  const uint32_t lane_base = tmem + ((uint32_t)(warp * 32) << 16);
  const float nanv = __int_as_float(0x7fc00000);
  float* part = reinterpret_cast<float*>(raw_smem + (base - smem_u32(raw_smem)));   // [128][nb + 4]
  const int ld = nb + 4;
  for (int c = 0; c < nb; c += 16) {
    float v[16];
    if (mine > 0) {
      tld16(lane_base + c, v);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = 0.f;
    }
    const int col = col0 + c;
    const int rank = col < p.SR ? p.ranks[tile.x * p.parts + col / p.R] - col % p.R : 0;   // in use of these 16
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = !ok ? nanv : e < rank ? v[e] : 0.f;
    if (cs > 1) {
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<float4*>(part + tid * ld + c + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
    } else if (tid < tile.z && col < p.SR) {
      float4* o = reinterpret_cast<float4*>(p.t + (int64_t)(tile.y + tid) * p.SR + col);
#pragma unroll
      for (int e = 0; e < 16; e += 4) o[e / 4] = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
    }
  }
  if (cs > 1) {
    cl.sync();
    const int quads = M * nb / 4;
    for (int q = cr * 128 + tid; q < quads; q += cs * 128) {
      const int r = q / (nb / 4), c = q % (nb / 4) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k = 0; k < cs; ++k) {
        const float4 w = *reinterpret_cast<const float4*>(cl.map_shared_rank(part, k) + r * ld + c);
        v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
      }
      if (r < tile.z && col0 + c < p.SR)
        *reinterpret_cast<float4*>(p.t + (int64_t)(tile.y + r) * p.SR + col0 + c) = v;
    }
    cl.sync();   // no CTA leaves while its shared memory may be read
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, ncols);
}

// ------------------------------------------------------------------------- expand ----
// out = y + scale * B t as a stream of chunks of 128 rows x 64 columns: a fifth warp copies y
// and the chunk's rows of B through a ring of stages with TMA; four warps take 32 rows each,
// add the product (mma.sync: 2 * rank flops for 4 bytes of y and out, so the tensor cores
// idle either way) in the stage itself and store from there with TMA.  The chunks of all
// tiles are dealt out evenly to a grid that is resident at once.  The stream through registers
// (16 warps an SM, 2 KB in flight each) reached 4.6 TB/s.
constexpr int EC = 64, EROWS = 32, YBYTES = M * EC * 2;

struct Chunks {
  int per_tile, total;                          // chunks of a tile, of all tiles
  int first[SPX_LORA_MAX_PARTS + 1];            // first chunk of each part
};

template <typename T, int KS>
__global__ void __launch_bounds__(160) expand_block_kernel(const __grid_constant__ CUtensorMap my,
                                                           const __grid_constant__ CUtensorMap mb,
                                                           const __grid_constant__ CUtensorMap mo, const Params p,
                                                           const Chunks ch, const int stages) {
  extern __shared__ uint8_t raw_smem[];
  __shared__ __align__(8) uint64_t bars[2 * 8];
  __shared__ int s_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = (smem_u32(raw_smem) + 1023u) & ~1023u;
  uint8_t* const sm = raw_smem + (base - smem_u32(raw_smem));
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * 8;
  const int bbytes = EC * p.R * 2, sbytes = YBYTES + (bbytes + 1023) / 1024 * 1024;
  if (tid == 0) {
    s_abort = 0;
    for (int s = 0; s < stages; ++s) mbar_init(full0 + 8 * s, 1), mbar_init(empty0 + 8 * s, 4);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async;" ::: "memory");
  }
  __syncthreads();
  const Abort ab{&s_abort, reinterpret_cast<int*>(p.t + (int64_t)p.rows * p.SR)};
  const int c0 = (int)((int64_t)ch.total * blockIdx.x / gridDim.x), c1 = (int)((int64_t)ch.total * (blockIdx.x + 1) / gridDim.x);
  // chunk q: its tile, part, first column within the part's range of y
  const auto where = [&](int q, int& tile, int& part, int& col) {
    tile = q / ch.per_tile;
    const int k = q - tile * ch.per_tile;
    part = 0;
    int off = 0;
    while (k >= ch.first[part + 1]) off += p.width[part++];
    col = off + (k - ch.first[part]) * EC;
  };
  if (warp == 4) {
    if (lane == 0) {
      int i = 0;
      for (; c0 + i < c1; ++i) {
        const int s = i % stages;
        if (i >= stages && !wait1(empty0 + 8 * s, (uint32_t)((i / stages - 1) & 1), ab)) break;
        int tl, part, col;
        where(c0 + i, tl, part, col);
        const int4 tile = p.tiles[tl];
        const uint32_t dst = base + s * sbytes, bar = full0 + 8 * s;
        mbar_expect_tx(bar, (uint32_t)(YBYTES + (tile.x >= 0 ? bbytes : 0)));
        tma_2d(dst, &my, col, p.order[tile.y], bar);
        if (tile.x >= 0) tma_2d(dst + YBYTES, &mb, 0, tile.x * p.OUT + col, bar);
      }
      if (c0 + i < c1) {   // given up: the copies in flight land before the shared memory goes
        for (int q = i > stages ? i - stages : 0; q < i; ++q) {
          const uint64_t t0 = gtimer();
          while (!mbar_try_wait_sleep(full0 + 8 * (q % stages), (uint32_t)((q / stages) & 1)) && gtimer() - t0 < kWaitNs) {
          }
        }
      }
    }
    return;
  }
  // t of the shrink kernel; also before the first store, so that this grid never ends before
  // the one that still reads x and writes the workspace
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int g = lane >> 2, c = lane & 3;
  int held = -1, held_part = -1, rank = 0, row0 = 0;
  float scale = 0.f, sc[2][2];
  uint4 f[2][KS][2];
  int4 tile = make_int4(0, 0, 0, 0);
  for (int i = 0; c0 + i < c1; ++i) {
    const int s = i % stages;
    int tl, part, col;
    where(c0 + i, tl, part, col);
    if (tl != held || part != held_part) {   // t of another tile or part
      held = tl, held_part = part;
      tile = p.tiles[tl];
      row0 = p.order[tile.y];
      rank = tile.x < 0 ? 0 : p.ranks[tile.x * p.parts + part];
      scale = tile.x < 0 ? 0.f : p.scales[tile.x * p.parts + part];
      if (rank > 0) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
          split_t<T, KS>(p.t + (int64_t)(tile.y + warp * EROWS + m * 16) * p.SR + part * p.R, p.SR,
                         tile.z - warp * EROWS - m * 16, rank, g, c, f[m], sc[m]);
      }
    }
    int left = -col;   // columns of the part from here on
    for (int q = 0; q <= part; ++q) left += p.width[q];
    if (!waitw(full0 + 8 * s, (uint32_t)((i / stages) & 1), ab)) break;
    uint8_t* const ys = sm + s * sbytes;
    const uint8_t* const bs = ys + YBYTES;
    const int rows = min(tile.z - warp * EROWS, EROWS);
    const bool tma_out = rows == EROWS && left >= EC;
    if (rows > 0) {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        float acc[8][4];
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
        if (rank > 0) {
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            if (ks * 16 >= rank) break;
#pragma unroll
            for (int n = 0; n < 8; ++n) {
              const int bc = (n / 4) * 32 + 8 * (g >> 1) + 2 * (n % 4) + (g & 1);
              const uint2 b = *reinterpret_cast<const uint2*>(bs + bc * p.R * 2 + ks * 32 + 8 * c);
              mma<T>(acc[n], f[m][ks][1].x, f[m][ks][1].y, f[m][ks][1].z, f[m][ks][1].w, b.x, b.y);
              mma<T>(acc[n], f[m][ks][0].x, f[m][ks][0].y, f[m][ks][0].z, f[m][ks][0].w, b.x, b.y);
            }
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = warp * EROWS + m * 16 + h * 8 + g;   // row of the tile
          const float s1 = scale * (rank > 0 ? sc[m][h] : 0.f);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            uint4* at = reinterpret_cast<uint4*>(ys + r * 128 + (((q * 4 + c) ^ (r & 7)) << 4));
            uint4 o = *at;
            if (rank > 0) {
              T* oe = reinterpret_cast<T*>(&o);
#pragma unroll
              for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  oe[2 * j + e] = from_f<T>(fmaf(s1, acc[4 * q + j][2 * h + e], to_f(oe[2 * j + e])));
            }
            if (tma_out) {
              if (rank > 0) *at = o;
            } else if (r < tile.z && q * 32 + 8 * c < left) {   // neither rows of the next sequence nor columns of the next part
              *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (int64_t)(row0 + r) * p.os + col + q * 32 + 8 * c) = o;
            }
          }
        }
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) {
      if (tma_out) {
        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(&mo),
                     "r"(col), "r"(row0 + warp * EROWS), "r"(base + s * sbytes + warp * EROWS * 128)
                     : "memory");
      }
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      // the chunk before this one is read out: its stage is free
      asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
      if (i > 0) mbar_arrive(empty0 + 8 * ((i - 1) % stages));
    }
    __syncwarp();
  }
  if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Looked up through the runtime: the library does not link the driver.
static EncodeTiledFn encode_tiled() {
  static EncodeTiledFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiledFn>(f);
  }();
  return fn;
}

// Rows of `cols` 16-bit values, `stride` apart, in boxes of box_cols x box_rows.
static int rows_map(CUtensorMap* m, const void* ptr, int dtype, int64_t rows, int64_t stride, int64_t cols, int box_cols,
                    int box_rows, bool swizzle) {
  const EncodeTiledFn enc = encode_tiled();
  if (!enc) {
    set_error("cuTensorMapEncodeTiled is not available from the driver");
    return SPX_ERR_CUDA;
  }
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)stride * 2};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows}, estr[2] = {1, 1};
  const CUresult r = enc(m, dtype == SPX_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                         const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled(adapter rows): error %d", (int)r);
    return SPX_ERR_CUDA;
  }
  return SPX_OK;
}

int shrink_block_launch(const Params& p, int dtype, int tiles, cudaStream_t st) {
  Cfg c;
  c.groups = (p.SR + 127) / 128;
  c.nb = ((p.SR + c.groups - 1) / c.groups + 15) / 16 * 16;
  const int sbytes = XBYTES + c.nb * KB * 2;
  c.stages = 110 * 1024 / sbytes;          // two CTAs an SM
  if (c.stages > 8) c.stages = 8;
  // the cluster's CTAs split k until the grid fills the SMs, with at least four steps each
  c.cs = 1;
  while (c.cs < 8 && (int64_t)tiles * c.groups * c.cs * 2 <= 2 * 148 && p.K >= 4 * KB * 2 * c.cs) c.cs *= 2;
  const size_t sums = c.cs > 1 ? (size_t)M * (c.nb + 4) * 4 : 0;
  c.smem = (size_t)c.stages * sbytes;
  c.smem = (c.smem > sums ? c.smem : sums) + 1024;
  CUtensorMap mx, ma;
  int rc = rows_map(&mx, p.x, dtype, p.rows, p.xs, p.K, KB, M, true);
  if (rc == SPX_OK) rc = rows_map(&ma, p.a, dtype, (int64_t)p.slots * p.SR, p.K, p.K, KB, c.nb, true);
  if (rc != SPX_OK) return rc;
  const uint32_t fmt = dtype == SPX_F16 ? 0u : 1u;
  const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(c.nb >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
  cudaError_t e = cudaFuncSetAttribute(shrink_block_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)c.smem);
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(tiles * c.cs), (unsigned)c.groups);
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = c.smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)c.cs, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, shrink_block_kernel, mx, ma, p, c.nb, c.stages, idesc);
  }
  if (e != cudaSuccess) {
    set_error("lora shrink_block_kernel: %s", cudaGetErrorString(e));
    return SPX_ERR_CUDA;
  }
  return launch_status("lora shrink_block_kernel");
}

template <typename T, int KS>
static int launch_expand_block(const Params& p, int dtype, int tiles, cudaStream_t st) {
  Chunks ch{};
  for (int s = 0; s < p.parts; ++s) ch.first[s + 1] = ch.first[s] + (p.width[s] + EC - 1) / EC;
  ch.per_tile = ch.first[p.parts];
  SPX_REQUIRE((int64_t)tiles * ch.per_tile <= 0x3fffffff, SPX_ERR_SHAPE, "spx_lora_add: too many rows");
  ch.total = tiles * ch.per_tile;
  const int sbytes = YBYTES + (EC * p.R * 2 + 1023) / 1024 * 1024;
  int stages = 108 * 1024 / sbytes;          // two CTAs an SM
  if (stages > 8) stages = 8;
  const size_t smem = (size_t)stages * sbytes + 1024;
  CUtensorMap my, mb, mo;
  int rc = rows_map(&my, p.y, dtype, p.rows, p.ys, p.OUT, EC, M, true);
  if (rc == SPX_OK) rc = rows_map(&mb, p.b, dtype, (int64_t)p.slots * p.OUT, p.R, p.R, p.R, EC, false);
  if (rc == SPX_OK) rc = rows_map(&mo, p.out, dtype, p.rows, p.os, p.OUT, EC, EROWS, true);
  if (rc != SPX_OK) return rc;
  const int most = 2 * num_sms();
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(ch.total < most ? ch.total : most));
  cfg.blockDim = dim3(160);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaError_t e = cudaFuncSetAttribute(expand_block_kernel<T, KS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, expand_block_kernel<T, KS>, my, mb, mo, p, ch, stages);
  if (e != cudaSuccess) {
    set_error("lora expand_block_kernel: %s", cudaGetErrorString(e));
    return SPX_ERR_CUDA;
  }
  return launch_status("lora expand_block_kernel");
}

template <typename T>
static int expand_block_as(const Params& p, int dtype, int tiles, cudaStream_t st) {
  switch (p.R / 16) {
    case 1: return launch_expand_block<T, 1>(p, dtype, tiles, st);
    case 2: return launch_expand_block<T, 2>(p, dtype, tiles, st);
    case 3:
    case 4: return launch_expand_block<T, 4>(p, dtype, tiles, st);
    default: return launch_expand_block<T, 8>(p, dtype, tiles, st);
  }
}

int expand_block_launch(const Params& p, int dtype, int tiles, cudaStream_t st) {
  return dtype == SPX_F16 ? expand_block_as<__half>(p, dtype, tiles, st) : expand_block_as<__nv_bfloat16>(p, dtype, tiles, st);
}

}  // namespace lora
}  // namespace spx
