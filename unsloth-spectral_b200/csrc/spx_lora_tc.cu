// Adapters of prompts: t = A x of tiles of up to 128 adjacent rows of one slot (the first of
// the two kernels of spx_lora.cu, for tokens that lie together).  A stream of x with few
// columns beside it: TMA brings tiles of 128 rows x 64 values of x and of the slot's A
// (128-byte swizzle) through a ring of stages, one thread issues tcgen05.mma (M = 128 rows,
// N = parts * rank columns, f32 in tensor memory), and x is read once, whatever the rank.
// Bound by memory: 2 * N flops a byte of x at most.  Two CTAs an SM keep about 128 KB of x in
// flight: 268 MB of x (8 x 4096 rows of 4096 bf16) take 55 to 61 us, as long as a plain sum
// over them; the mma.sync kernel (fragments loaded by the warps that use them, 8 warps an SM)
// took 214.  More stages, or boxes twice as wide, measured level.  Few tiles: the CTAs of a
// cluster split k and push their sums into one another's shared memory, added in a fixed
// order.  Rows of the next sequence that a tile's box covers are computed and not stored.
// Every wait is bounded; an expired one leaves NaN in t.
#include <cuda.h>

#include "spx_lora.cuh"
#include "spx_sm100.cuh"

namespace spx {
namespace lora {

using namespace sm100;

constexpr int M = 128, KB = 64;            // rows of a tile, values of k in a stage
constexpr int MAXSTAGES = 8;               // barriers of a ring
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
                                                           const int nb, const int groups, const int stages, const uint32_t idesc) {
  extern __shared__ uint8_t raw_smem[];
  __shared__ __align__(8) uint64_t bars[2 * MAXSTAGES + 1];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_rank[16];   // ranks in use of each 16 columns
  cluster_arrive_relaxed();
  const int cs = (int)cluster_size(), cr = (int)cluster_rank();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // the groups of columns of a tile after one another: x comes from memory once
  const int unit = blockIdx.x / cs, group = unit % groups;
  const int4 tile = p.tiles[unit / groups];
  if (tile.x < 0) return;   // rows without an adapter: the whole cluster leaves
  const int tid = threadIdx.x, warp = tid >> 5;
  const int col0 = group * nb, row0 = tile.w;
  const uint32_t base = (smem_u32(raw_smem) + 1023u) & ~1023u;
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * MAXSTAGES, done = empty0 + 8 * MAXSTAGES;
  const int sbytes = XBYTES + nb * KB * 2;
  uint32_t ncols = 32;
  while ((int)ncols < nb) ncols *= 2;
  if (warp == 0) {
    tmem_alloc(smem_u32(&s_tmem), ncols);
    tmem_relinquish();
  }
  if (tid >= 64 && tid < 64 + nb / 16) {
    const int col = col0 + (tid - 64) * 16;
    s_rank[tid - 64] = col < p.SR ? p.ranks[tile.x * p.parts + col / p.R] - col % p.R : 0;
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
  // [cs][128 / cs][nb + 4], behind the ring: the cluster's sums of this CTA's share of the rows
  float* const got = reinterpret_cast<float*>(raw_smem + (base - smem_u32(raw_smem)) + stages * sbytes);
  const int ld = nb + 4, share = M / cs;
  uint32_t to = 0;
  if (cs > 1) {
    cluster_started();
    to = in_cta(got + (cr * share + tid % share) * ld, tid / share);
  }
  for (int c = 0; c < nb; c += 16) {
    float v[16];
    if (mine > 0) {
      tld16(lane_base + c, v);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = 0.f;
    }
    const int col = col0 + c, rank = s_rank[c / 16];
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = !ok ? nanv : e < rank ? v[e] : 0.f;
    if (cs > 1) {
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to + 4 * (c + e)), "f"(v[e]), "f"(v[e + 1]),
                     "f"(v[e + 2]), "f"(v[e + 3])
                     : "memory");
    } else if (tid < tile.z && col < p.SR) {
      float4* o = reinterpret_cast<float4*>(p.t + (int64_t)(tile.y + tid) * p.SR + col);
#pragma unroll
      for (int e = 0; e < 16; e += 4) o[e / 4] = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
    }
  }
  if (cs > 1) {
    cluster_pushed();
    for (int q = tid; q < share * nb / 4; q += 128) {
      const int r = q / (nb / 4), c = q % (nb / 4) * 4;
      float4 v = *reinterpret_cast<const float4*>(got + r * ld + c);
      for (int k = 1; k < cs; ++k) {
        const float4 w = *reinterpret_cast<const float4*>(got + (k * share + r) * ld + c);
        v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
      }
      if (cr * share + r < tile.z && col0 + c < p.SR)
        *reinterpret_cast<float4*>(p.t + (int64_t)(tile.y + cr * share + r) * p.SR + col0 + c) = v;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, ncols);
}

// ------------------------------------------------------------------------- expand ----
// out = y + scale * B t as a stream of chunks of 128 rows x 128 columns, one CTA an SM.  One
// warp copies y and the chunk's rows of B through a ring of stages with TMA; four warps make
// the A operand of a tile and part (t, its high and low halves in two values of the row type
// each), one ahead of its use; one thread issues the MMAs (f32 in tensor memory, two buffers);
// two groups of eight warps take the chunks in turn, add the product to y in the stage itself
// (thread = row, half of the columns) and store from there with TMA.
// Bound by memory: 8 x 4096 rows of 6144 bf16 take 135 to 140 us, at rank 16 as at rank 0 (the
// ring alone), where a copy of y takes 125.  What it took: y through registers (16 warps an SM)
// 174; this ring with mma.sync 165 (500 at rank 64); tcgen05 with one group of eight warps 147
// (a chunk's waits, 1.7 us, were longer than its share of the stream, 1.4); the chunks dealt
// out so that the CTAs move along whole rows, four chunks (1 KB) each at a time, instead of
// each its own rows (128 pages open a CTA): 6 us less; eight chunks 4 us more, two 8.
constexpr int EC = 128, EROWS = 32, YBOX = M * 64 * 2, YBYTES = 2 * YBOX, EGROUP = 8, EWARPS = 2 * EGROUP, BWARPS = 4;
constexpr int ETHREADS = (EWARPS + 2 + BWARPS) * 32;

// What the warps need to know of a tile and part: a version of the A operand.
struct Version {
  int rank, row0, rows;
  float scale;
};

struct Chunks {
  int per_tile, unit, units_per_tile, units;    // chunks of a tile, of a unit, units of a tile, of all tiles
  int first[SPX_LORA_MAX_PARTS + 1];            // first chunk of each part
  int kw;                                       // ranks of a box of B: 16, 32 or 64
};

// K-major operand tiles of rows of 2 * kw bytes, swizzled over that width.
__device__ __forceinline__ uint64_t desc_kw(uint32_t saddr, int kw) {
  const uint64_t type = kw == 64 ? 2ull : kw == 32 ? 4ull : 6ull;
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | (1ull << 16) | ((uint64_t)(uint32_t)kw << 32) | (1ull << 46) | (type << 61);
}
__device__ __forceinline__ void tld32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int u = 0; u < 32; ++u) v[u] = __uint_as_float(r[u]);
}

// A row of t on its way to the A operand: its first 16 values in registers, the others into L2.
struct TRow {
  static constexpr int HELD = 4;
  const float* t;
  float4 v[HELD];
  __device__ __forceinline__ float4 at(int q) const { return reinterpret_cast<const float4*>(t)[q]; }
  __device__ __forceinline__ void load(const float* row, bool in, int R) {
    t = row;
#pragma unroll
    for (int q = 0; q < HELD; ++q) v[q] = in && 4 * q < R ? at(q) : make_float4(0.f, 0.f, 0.f, 0.f);
    for (int q = HELD; in && 4 * q < R; q += 8) asm volatile("prefetch.global.L2 [%0];" ::"l"(t + 4 * q));
  }
};

// Row r of a tile's t as the high and low parts of the A operand: element (row, k) at
// (k / 8) * 2048 + row * 16 + (k % 8) * 2, the low parts 256 R bytes on.  Returns what the row
// of the product is to be multiplied by.
template <typename T>
__device__ __forceinline__ float stage_t(const TRow& row, bool in, int R, int r, uint8_t* a) {
  float dn = 1.f, up = 1.f;
  if (!__is_same(T, __nv_bfloat16)) {
    // f16: scaled by a power of two so that the row's largest value is near 2^8 (no overflow
    // of the high parts, no underflow of the low parts)
    float mx = 0.f;
    const auto see = [&](const float4& v) {
      mx = fmaxf(fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))), mx);
    };
#pragma unroll
    for (int q = 0; q < TRow::HELD; ++q) see(row.v[q]);
#pragma unroll 4
    for (int q = TRow::HELD; q < R / 4; ++q)
      if (in) see(row.at(q));
    int ex = (int)((__float_as_uint(mx) >> 23) & 0xff) - 127 - 8;
    ex = max(-118, min(118, ex));
    dn = __uint_as_float((uint32_t)(127 - ex) << 23);
    up = __uint_as_float((uint32_t)(127 + ex) << 23);
  }
  const auto put = [&](int k8, const float4& u, const float4& w) {
    uint4 hi, lo;
    const float f[8] = {u.x * dn, u.y * dn, u.z * dn, u.w * dn, w.x * dn, w.y * dn, w.z * dn, w.w * dn};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const T h = from_f<T>(f[e]);
      reinterpret_cast<T*>(&hi)[e] = h;
      // an infinity has no low part
      reinterpret_cast<T*>(&lo)[e] = from_f<T>(fabsf(to_f(h)) < INFINITY ? f[e] - to_f(h) : 0.f);
    }
    *reinterpret_cast<uint4*>(a + k8 * 2048 + r * 16) = hi;
    *reinterpret_cast<uint4*>(a + 256 * R + k8 * 2048 + r * 16) = lo;
  };
#pragma unroll
  for (int k8 = 0; k8 < TRow::HELD / 2; ++k8)
    if (8 * k8 < R) put(k8, row.v[2 * k8], row.v[2 * k8 + 1]);
  const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int k8 = TRow::HELD / 2; k8 < R / 8; ++k8) put(k8, in ? row.at(2 * k8) : zero, in ? row.at(2 * k8 + 1) : zero);
  return up;
}

template <typename T>
__global__ void __launch_bounds__(ETHREADS) expand_block_kernel(const __grid_constant__ CUtensorMap my,
                                                                         const __grid_constant__ CUtensorMap mb,
                                                                         const __grid_constant__ CUtensorMap mo,
                                                                         const Params p, const Chunks ch,
                                                                         const int stages, const int abufs, const uint32_t idesc) {
  extern __shared__ uint8_t raw_smem[];
  __shared__ __align__(8) uint64_t bars[2 * MAXSTAGES + 8];
  __shared__ Version versions[2];
  __shared__ float row_scale[2][M];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = (smem_u32(raw_smem) + 1023u) & ~1023u;
  uint8_t* const sm = raw_smem + (base - smem_u32(raw_smem));
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * MAXSTAGES, acc_full0 = empty0 + 8 * MAXSTAGES,
                 acc_empty0 = acc_full0 + 16, t_ready0 = acc_empty0 + 16, t_free0 = t_ready0 + 16;
  const int bbytes = EC * p.R * 2, sbytes = YBYTES + bbytes;
  uint8_t* const a_op = sm + stages * sbytes;   // abufs buffers of 512 R bytes
  if (warp == EWARPS + 1) {
    tmem_alloc(smem_u32(&s_tmem), 2 * EC);
    tmem_relinquish();
  }
  if (tid == 0) {
    s_abort = 0;
    for (int s = 0; s < stages; ++s) mbar_init(full0 + 8 * s, 1), mbar_init(empty0 + 8 * s, EGROUP);
    for (int s = 0; s < 2; ++s) {
      mbar_init(acc_full0 + 8 * s, 1), mbar_init(acc_empty0 + 8 * s, EGROUP);
      mbar_init(t_ready0 + 8 * s, BWARPS), mbar_init(t_free0 + 8 * s, EWARPS + 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const Abort ab{&s_abort, reinterpret_cast<int*>(p.t + (int64_t)p.rows * p.SR)};

  // The walk over the CTA's chunks, the same in every role: every gridDim-th unit of `unit`
  // chunks that follow one another in a tile, so that the CTAs together move along whole rows.
  struct Walk {
    int u, tl, part, k, end, col, left;   // unit, tile, part, chunk, end of the unit; first column, columns of the part from there
    bool fresh;                           // another unit or part than the chunk before: a new version
    __device__ __forceinline__ Walk(const Params& p, const Chunks& ch) : u(blockIdx.x) { start(p, ch); }
    __device__ __forceinline__ bool valid(const Chunks& ch) const { return u < ch.units; }
    __device__ __forceinline__ void start(const Params& p, const Chunks& ch) {
      tl = u / ch.units_per_tile;
      k = (u - tl * ch.units_per_tile) * ch.unit;
      end = min(k + ch.unit, ch.per_tile);
      part = 0, col = 0;
      while (k >= ch.first[part + 1]) col += p.width[part++];
      left = p.width[part] - (k - ch.first[part]) * EC;
      col += (k - ch.first[part]) * EC;
      fresh = true;
    }
    __device__ __forceinline__ void next(const Params& p, const Chunks& ch) {
      if (++k == end) {
        u += gridDim.x;
        if (u < ch.units) start(p, ch);
        return;
      }
      fresh = k == ch.first[part + 1];
      if (fresh) {
        col += left;
        left = p.width[++part];
      } else {
        col += EC, left -= EC;
      }
    }
  };

  if (warp == EWARPS) {
    if (lane == 0) {
      // the tile of the unit after this one is looked up ahead: the ring never waits for it
      const auto tile_of = [&](int u) { return p.tiles[min(u, ch.units - 1) / ch.units_per_tile]; };
      int i = 0, unit = -1;
      int4 tile, ahead = tile_of(blockIdx.x);
      Walk w(p, ch);
      for (; w.valid(ch); ++i, w.next(p, ch)) {
        if (w.u != unit) unit = w.u, tile = ahead, ahead = tile_of(w.u + gridDim.x);
        const int s = i % stages;
        if (i >= stages && !wait1(empty0 + 8 * s, (uint32_t)((i / stages - 1) & 1), ab)) break;
        const uint32_t dst = base + s * sbytes, bar = full0 + 8 * s;
        // a box that begins past the part is not wanted (and past the last one lies outside)
        const bool two = w.left > 64;
        mbar_expect_tx(bar, (uint32_t)((two ? YBYTES : YBOX) + (tile.x >= 0 ? bbytes : 0)));
        tma_2d(dst, &my, w.col, tile.w, bar);
        if (two) tma_2d(dst + YBOX, &my, w.col + 64, tile.w, bar);
        if (tile.x >= 0)
          for (int b = 0; b < p.R / ch.kw; ++b)
            tma_2d(dst + YBYTES + b * EC * ch.kw * 2, &mb, b * ch.kw, tile.x * p.OUT + w.col, bar);
      }
      if (w.valid(ch)) {   // given up: the copies in flight land before the shared memory goes
        for (int q = i > stages ? i - stages : 0; q < i; ++q) {
          const uint64_t t0 = gtimer();
          while (!mbar_try_wait_sleep(full0 + 8 * (q % stages), (uint32_t)((q / stages) & 1)) && gtimer() - t0 < kWaitNs) {
          }
        }
      }
    }
  } else if (warp == EWARPS + 1) {
    if (lane == 0) {
      // Every chunk takes its turn at the accumulators, also one without an adapter (its barriers
      // are then arrived at without an MMA): so a group of warps always has the same buffer, and
      // the sums of chunk i being there means that the copies of every chunk up to i are.
      int i = 0, v = -1, rank = 0, buf = 0;   // chunk, version of the A operand
      for (Walk w(p, ch); w.valid(ch); ++i, w.next(p, ch)) {
        if (w.fresh) {
          if (v >= 0) umma_commit(t_free0 + 8 * buf);   // once the MMAs that read it are done
          ++v;
          buf = v % abufs;
          if (!wait1(t_ready0 + 8 * buf, (uint32_t)((v / abufs) & 1), ab)) break;
          rank = versions[buf].rank;
        }
        const int s = i % stages, a = i & 1;
        if (!wait1(full0 + 8 * s, (uint32_t)((i / stages) & 1), ab)) break;
        if (i >= 2 && !wait1(acc_empty0 + 8 * a, (uint32_t)((i / 2 - 1) & 1), ab)) break;
        if (rank <= 0) {
          mbar_arrive(acc_full0 + 8 * a);
          continue;
        }
        tc_fence_after();
        const uint32_t bo = base + s * sbytes + YBYTES, ao = smem_u32(a_op) + buf * 512 * p.R;
        for (int ks = 0; ks * 16 < rank; ++ks) {
          const uint64_t bd = desc_kw(bo + (ks * 16 / ch.kw) * EC * ch.kw * 2 + ks * 16 % ch.kw * 2, ch.kw);
          umma(tmem + a * EC, umma_desc(ao + 256 * p.R + ks * 4096, 2048, 128), bd, idesc, ks > 0 ? 1u : 0u);
          umma(tmem + a * EC, umma_desc(ao + ks * 4096, 2048, 128), bd, idesc, 1u);
        }
        umma_commit(acc_full0 + 8 * a);
      }
      if (i > 0) {   // the last MMAs are done before their tensor memory goes
        const uint64_t t0 = gtimer();
        while (!mbar_try_wait_sleep(acc_full0 + 8 * ((i - 1) & 1), (uint32_t)(((i - 1) / 2) & 1)) && gtimer() - t0 < kWaitNs) {
        }
      }
    }
  } else if (warp > EWARPS + 1) {
    asm volatile("griddepcontrol.wait;" ::: "memory");   // t of the shrink kernel
    // Under the stream a load takes microseconds: what a version needs is fetched while the one
    // before it is staged, its tile while the one before that is.
    struct Next {
      bool ok;
      int part;
      int4 tile;
    };
    const int r = tid - (EWARPS + 2) * 32;
    Walk w(p, ch);
    const auto take = [&]() {
      Next n{w.valid(ch), w.part, make_int4(-1, 0, 0, 0)};
      if (n.ok) {
        n.tile = p.tiles[w.tl];
        do w.next(p, ch);
        while (w.valid(ch) && !w.fresh);
      }
      return n;
    };
    const auto fetch = [&](const Next& n, Version& ver, TRow& t) {
      const bool slot = n.ok && n.tile.x >= 0;
      ver.rank = slot ? p.ranks[n.tile.x * p.parts + n.part] : 0;
      ver.scale = slot ? p.scales[n.tile.x * p.parts + n.part] : 0.f;
      ver.row0 = n.tile.w;
      ver.rows = n.tile.z;
      t.load(p.t + (int64_t)(n.tile.y + r) * p.SR + n.part * p.R, slot && r < n.tile.z, p.R);
    };
    Next now = take(), next = take();
    Version ver, ver_next;
    TRow t, t_next;
    fetch(now, ver, t);
    for (int v = 0; now.ok; ++v) {
      fetch(next, ver_next, t_next);
      const Next after = take();
      const int buf = v % abufs;
      if (v >= abufs && !waitw(t_free0 + 8 * buf, (uint32_t)((v / abufs - 1) & 1), ab)) break;
      if (ver.rank > 0)
        row_scale[buf][r] = ver.scale * stage_t<T>(t, r < ver.rows, p.R, r, a_op + buf * 512 * p.R);
      if (r == 0) versions[buf] = ver;
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(t_ready0 + 8 * buf);
      now = next, next = after, ver = ver_next, t = t_next;
    }
  } else {
    // before the first store, so that this grid never ends before the one that still reads x
    // and writes the workspace
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // two groups of eight warps take the chunks in turn, so that the waits of one chunk (its sums,
    // its store) pass while the other is worked on
    const int quad = warp & 3, half = (warp >> 2) & 1, group = warp / EGROUP, r = quad * 32 + lane;
    int i = 0, v = -1;
    Version ver{};
    float s1 = 0.f;
    Walk w(p, ch);
    for (; w.valid(ch); ++i, w.next(p, ch)) {
      const int s = i % stages;
      if (w.fresh) {
        ++v;
        const int buf = v % abufs;
        if (!waitw(t_ready0 + 8 * buf, (uint32_t)((v / abufs) & 1), ab)) break;
        ver = versions[buf];
        s1 = row_scale[buf][r];
        __syncwarp();
        if (lane == 0) mbar_arrive(t_free0 + 8 * buf);
      }
      const bool act = ver.rank > 0;
      if ((i & 1) != group) continue;
      if (!waitw(full0 + 8 * s, (uint32_t)((i / stages) & 1), ab)) break;
      uint8_t* const yrow = sm + s * sbytes + half * YBOX + r * 128;
      const int left = w.left - half * 64;   // columns of this half
      const bool tma_out = ver.rows >= quad * EROWS + EROWS && left >= 64;
      if (!waitw(acc_full0 + 8 * group, (uint32_t)((i / 2) & 1), ab)) break;
      tc_fence_after();
#pragma unroll
      for (int hc = 0; hc < 2; ++hc) {
        float x[32];
        if (act) tld32(tmem + ((uint32_t)(quad * 32) << 16) + group * EC + half * 64 + hc * 32, x);
        if (hc == 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(acc_empty0 + 8 * group);
        }
        if (!act && tma_out) continue;   // stored as it came
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint4* at = reinterpret_cast<uint4*>(yrow + (((hc * 4 + q) ^ (r & 7)) << 4));
          uint4 o = *at;
          if (act) {
            T* oe = reinterpret_cast<T*>(&o);
#pragma unroll
            for (int e = 0; e < 8; ++e) oe[e] = from_f<T>(fmaf(s1, x[q * 8 + e], to_f(oe[e])));
          }
          if (tma_out) {
            *at = o;
          } else if (r < ver.rows && hc * 32 + q * 8 < left) {   // neither rows of the next sequence nor columns of the next part
            *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (int64_t)(ver.row0 + r) * p.os + w.col + half * 64 + hc * 32 +
                                      q * 8) = o;
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        if (tma_out) {
          asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(&mo),
                       "r"(w.col + half * 64), "r"(ver.row0 + r),
                       "r"(base + s * sbytes + half * YBOX + quad * EROWS * 128)
                       : "memory");
        }
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");   // read out: the stage is free
        mbar_arrive(empty0 + 8 * s);
      }
      __syncwarp();
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    for (; w.valid(ch); ++i, w.next(p, ch)) {   // a wait expired: what is left is NaN, not what lay there
      if ((i & 1) != group) continue;
      const int4 tile = p.tiles[w.tl];
      T* o = static_cast<T*>(p.out) + (int64_t)(tile.w + r) * p.os + w.col + half * 64;
      for (int e = 0; r < tile.z && e < 64 && half * 64 + e < w.left; ++e) o[e] = from_f<T>(__int_as_float(0x7fc00000));
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == EWARPS + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 2 * EC);
  }
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
                    int box_rows, CUtensorMapSwizzle swizzle) {
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
                         swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled(adapter rows): error %d", (int)r);
    return SPX_ERR_CUDA;
  }
  return SPX_OK;
}

// Clusters of 16 CTAs (more than the portable 8) of the kernel that the device holds at once, one or
// two CTAs an SM; asked for once.
static int wide_clusters(int an_sm) {
  static std::atomic<int> known[64][2];   // the number + 1
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return 0;
  std::atomic<int>& k = known[dev][an_sm - 1];
  if (k.load(std::memory_order_relaxed) == 0) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(16), cfg.blockDim = dim3(128), cfg.dynamicSmemBytes = (an_sm == 2 ? 111 : 221) * 1024;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 16, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    cfg.attrs = at, cfg.numAttrs = 1;
    if (cudaFuncSetAttribute(shrink_block_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 221 * 1024) != cudaSuccess ||
        cudaFuncSetAttribute(shrink_block_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, shrink_block_kernel, &cfg) != cudaSuccess) {
      cudaGetLastError();   // not an error of this call: smaller clusters
      n = 0;
    }
    k.store(n + 1, std::memory_order_relaxed);
  }
  return k.load(std::memory_order_relaxed) - 1;
}

int shrink_block_launch(const Params& p, int dtype, int tiles, cudaStream_t st) {
  // Two CTAs an SM, and all columns in one group up to 256: x is read once (rank 64 in three parts:
  // 77 us against 109 in two groups).  Few tiles: the CTAs of a cluster split k until they fill the
  // SMs (clusters of eight do not fill every GPC: two thirds of the places), with at least four steps
  // each: 77 tiles at K = 12560 95 us with one CTA a tile, 65 with two; four tiles at K = 14336 25.3
  // us a call with eight, 21.3 with sixteen.  More columns than 128 are two groups then, or one where
  // two do not fit (38 tiles of 192 columns 61 us with one CTA each, 50).  Where the CTAs leave an SM
  // to each, or the cluster's sums take the room, a ring has all of its shared memory.
  Cfg c;
  int sbytes = 0, got = 0;
  const auto shape = [&](int cs, int widest, bool alone) {   // CTAs an SM
    c.cs = cs;
    c.groups = (p.SR + widest - 1) / widest;
    c.nb = ((p.SR + c.groups - 1) / c.groups + 15) / 16 * 16;
    sbytes = XBYTES + c.nb * KB * 2, got = cs > 1 ? M * (c.nb + 4) * 4 : 0;
    const bool two = !alone && (cs == 1 || (110 * 1024 - got) / sbytes >= 3);
    c.stages = ((two ? 110 : 220) * 1024 - got) / sbytes;   // 2 (256 columns) to 8
    if (c.stages > MAXSTAGES) c.stages = MAXSTAGES;
    return two ? 2 : 1;
  };
  const auto fits = [&](int cs, int widest) {
    const int an_sm = shape(cs, widest, false);
    const int64_t places = cs < 8 ? an_sm * num_sms() : cs == 8 ? an_sm * 96 : 16 * wide_clusters(an_sm);
    return (int64_t)tiles * c.groups * cs <= places;
  };
  int cs = 1, widest = 256;
  for (; cs < 16 && p.K >= 4 * KB * 2 * cs; cs *= 2) {
    if (fits(2 * cs, 128)) {
      widest = 128;
    } else if (p.SR > 128 && p.SR <= 192 && fits(2 * cs, 192)) {
      widest = 192;
    } else {
      break;
    }
  }
  shape(cs, widest, false);
  if ((int64_t)tiles * c.groups * cs <= (cs < 8 ? num_sms() : cs == 8 ? 96 : 16 * wide_clusters(1))) shape(cs, widest, true);
  c.smem = (size_t)c.stages * sbytes + got + 1024;
  CUtensorMap mx, ma;
  int rc = rows_map(&mx, p.x, dtype, p.rows, p.xs, p.K, KB, M, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc == SPX_OK) rc = rows_map(&ma, p.a, dtype, (int64_t)p.slots * p.SR, p.K, p.K, KB, c.nb, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != SPX_OK) return rc;
  const uint32_t fmt = dtype == SPX_F16 ? 0u : 1u;
  const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(c.nb >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
  static std::atomic<int> have[64];
  cudaError_t e = allow_smem(shrink_block_kernel, (int)c.smem, have);
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(tiles * c.groups * c.cs));
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = c.smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)c.cs, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, shrink_block_kernel, mx, ma, p, c.nb, c.groups, c.stages, idesc);
  }
  if (e != cudaSuccess) {
    set_error("lora shrink_block_kernel: %s", cudaGetErrorString(e));
    return SPX_ERR_CUDA;
  }
  return launch_status("lora shrink_block_kernel");
}

template <typename T>
static int launch_expand_block(const Params& p, int dtype, int tiles, cudaStream_t st) {
  Chunks ch{};
  for (int s = 0; s < p.parts; ++s) ch.first[s + 1] = ch.first[s] + (p.width[s] + EC - 1) / EC;
  ch.per_tile = ch.first[p.parts];
  ch.kw = p.R % 64 == 0 ? 64 : p.R % 32 == 0 ? 32 : 16;
  SPX_REQUIRE((int64_t)tiles * ch.per_tile <= 0x3fffffff, SPX_ERR_SHAPE, "spx_lora_add: too many rows");
  // Four chunks (1 KB of a row) to a unit; with few units an SM the size whose slowest CTA is
  // done first, a change of unit (another A operand) counted as three quarters of a chunk:
  // 8 x 512 rows of 4096 columns at rank 64 45 us with one chunk, 36 with eight.
  const int most = num_sms();
  ch.unit = 4;
  if ((int64_t)tiles * ch.per_tile < (int64_t)64 * most) {
    int best = 0x7fffffff;
    for (int u = 1; u <= 16; u *= 2) {
      const int units = tiles * ((ch.per_tile + u - 1) / u), cost = (units + most - 1) / most * (4 * (u < ch.per_tile ? u : ch.per_tile) + 3);
      if (cost < best) best = cost, ch.unit = u;
    }
  }
  ch.units_per_tile = (ch.per_tile + ch.unit - 1) / ch.unit;
  ch.units = tiles * ch.units_per_tile;
  const int abufs = p.R <= 64 ? 2 : 1, sbytes = YBYTES + EC * p.R * 2, abytes = abufs * 2 * M * p.R * 2;
  int stages = (220 * 1024 - abytes) / sbytes;   // 2 (rank 128) to 5 (rank 16)
  if (stages > MAXSTAGES) stages = MAXSTAGES;
  const size_t smem = (size_t)stages * sbytes + abytes + 1024;
  CUtensorMap my, mb, mo;
  int rc = rows_map(&my, p.y, dtype, p.rows, p.ys, p.OUT, 64, M, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc == SPX_OK)
    rc = rows_map(&mb, p.b, dtype, (int64_t)p.slots * p.OUT, p.R, p.R, ch.kw, EC,
                  ch.kw == 64   ? CU_TENSOR_MAP_SWIZZLE_128B
                  : ch.kw == 32 ? CU_TENSOR_MAP_SWIZZLE_64B
                                : CU_TENSOR_MAP_SWIZZLE_32B);
  if (rc == SPX_OK) rc = rows_map(&mo, p.out, dtype, p.rows, p.os, p.OUT, 64, EROWS, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != SPX_OK) return rc;
  const uint32_t fmt = dtype == SPX_F16 ? 0u : 1u;
  const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(EC >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(ch.units < most ? ch.units : most));
  cfg.blockDim = dim3(ETHREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  static std::atomic<int> have[64];
  cudaError_t e = allow_smem(expand_block_kernel<T>, (int)smem, have);
  if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, expand_block_kernel<T>, my, mb, mo, p, ch, stages, abufs, idesc);
  if (e != cudaSuccess) {
    set_error("lora expand_block_kernel: %s", cudaGetErrorString(e));
    return SPX_ERR_CUDA;
  }
  return launch_status("lora expand_block_kernel");
}

int expand_block_launch(const Params& p, int dtype, int tiles, cudaStream_t st) {
  return dtype == SPX_F16 ? launch_expand_block<__half>(p, dtype, tiles, st)
                          : launch_expand_block<__nv_bfloat16>(p, dtype, tiles, st);
}

}  // namespace lora
}  // namespace spx
