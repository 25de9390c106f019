// Low-rank adapters of many requests beside one shared projection (spx_lora_add,
// include/spx.h):  out[r] = y[r] + scale * B[a] (A[a] x[r]),  a = the slot of row r.
// Two kernels over tiles of rows of one slot:
//   shrink  t = A x      (K = in_features is long, the result has `rank` columns: the warps
//                         and the CTAs of a cluster split K, the partial sums meet in
//                         shared and distributed shared memory in a fixed order)
//   expand  out = y + scale * B t   (each warp owns 64 output columns, or 32 at ranks above 64 and
//                         where there are few columns, and keeps their B fragments in
//                         registers over the tile's rows)
// Both are streams with little arithmetic (2 * rank flops a value of x and of y), so each lane
// fetches the values of its own mma fragments: of x and A through a ring of its own, of y and
// B into registers.  The sum over k may take its
// terms in any order, so lane c of a quad takes k = 8c..8c+7 of 32 as the k of two
// m16n8k16 steps (16-byte loads, whole sectors); the same choice over the output columns
// gives 16-byte accesses of y and out.
// These are the kernels for few rows of a slot; prompts take spx_lora_tc.cu's.  Bound by latency
// and by the weights: one request on q|k|v at rank 16 takes 4.6 us (two launches, the second
// one waiting for the first inside the GPU), 64 requests with 24 adapters of rank 64 and 32 at
// K = 14336 18.0 us, of which 50 MB of weights need 7.6.
// t is kept in float32; for the second product it is split into a high and a low value of
// the row type (two MMAs), which keeps about 16 (bf16) or 22 (f16) bits of it.
#include "spx_lora.cuh"

namespace spx {
namespace lora {

constexpr int SW = 8;    // warps of a shrink CTA
constexpr int EW = 4;    // warps of an expand CTA

// ------------------------------------------------------------------------- shrink ----
// Tile of 16 * MT rows x 8 * NT of the parts * max_rank columns; the CTAs of a cluster and
// their warps take the 32-wide steps of k in turn.  Each lane copies the 16-byte vectors that
// it will use itself into a ring of its own (cp.async, no barrier), so that a warp has several
// steps in flight without registers: loaded into registers, 64 rows of 24 slots at K = 14336,
// rank 64 took 19 us, with 10 warps an SM waiting for memory.
template <int MT, int NT>
struct Ring {
  static constexpr int VECS = 2 * MT + NT;                                   // 16 bytes a lane each
  static constexpr int FIT = 73 * 1024 / (SW * VECS * 512), STAGES = FIT > 6 ? 6 : FIT < 2 ? 2 : FIT;   // three CTAs an SM
  static constexpr int SUMS = SW * MT * 16 * NT * 8, COPIES = SW * STAGES * VECS * 128;   // floats
  static constexpr int FLOATS = SUMS > COPIES ? SUMS : COPIES;
  static constexpr size_t BYTES = 4 * ((size_t)FLOATS + MT * 16 * NT * 8);
};

__device__ __forceinline__ void copy16(uint4* dst, const void* src, bool in) {   // zeros unless `in`
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src),
               "r"(in ? 16 : 0)
               : "memory");
}

template <typename T, int MT, int NT>
__global__ void __launch_bounds__(SW * 32, MT * NT > 8 ? 2 : 3) shrink_kernel(const Params p) {
  using Ri = Ring<MT, NT>;
  extern __shared__ uint4 ring[];
  __shared__ int s_left[NT];   // of each group of eight columns: how many hold a rank in use
  constexpr int N = NT * 8, E = MT * 16 * N;
  float* const sums = reinterpret_cast<float*>(ring);   // [SW][MT * 16][N], after the stream
  float* const got = reinterpret_cast<float*>(ring) + Ri::FLOATS;   // [cs][E / cs]: the cluster's sums of this CTA's share
  cluster_arrive_relaxed();
  const int cs = (int)cluster_size(), cr = (int)cluster_rank();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int4 tile = p.tiles[blockIdx.x / cs];
  if (tile.x < 0) return;   // rows without an adapter: the whole cluster leaves
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int col0 = blockIdx.y * (NT * 8);
  const T* xr[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = m * 16 + h * 8 + g;
      xr[m][h] = r < tile.z ? static_cast<const T*>(p.x) + (int64_t)p.order[tile.y + r] * p.xs + 8 * c : nullptr;
    }
  int in_use = 0;   // lane n: group n of eight columns
  if (lane < NT && col0 + lane * 8 < p.SR) {
    const int col = col0 + lane * 8, part = col / p.R;
    in_use = p.ranks[tile.x * p.parts + part] - (col - part * p.R);
  }
  const uint32_t act = __ballot_sync(0xffffffffu, in_use > 0);   // groups that hold a rank in use
  if (warp == 0 && lane < NT) s_left[lane] = in_use;
  const T* ar = static_cast<const T*>(p.a) + ((int64_t)tile.x * p.SR + col0 + g) * p.K + 8 * c;
  float acc[MT][NT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[m][n][e] = 0.f;
  const int steps = (p.K + 31) / 32, first = cr * SW + warp, stride = cs * SW;
  const int mine = act && first < steps ? (steps - first + stride - 1) / stride : 0;
  uint4* const own = ring + (size_t)warp * Ri::STAGES * Ri::VECS * 32 + lane;
  const auto fetch = [&](int i) {
    if (i < mine) {
      const int s = first + i * stride;
      const bool in = s * 32 + 8 * c < p.K;
      uint4* d = own + (i % Ri::STAGES) * Ri::VECS * 32;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          copy16(d + (2 * m + h) * 32, in && xr[m][h] ? (const void*)(xr[m][h] + s * 32) : p.x, in && xr[m][h]);
#pragma unroll
      for (int n = 0; n < NT; ++n)
        if ((act >> n) & 1u)
          copy16(d + (2 * MT + n) * 32, in ? (const void*)(ar + (int64_t)n * 8 * p.K + s * 32) : p.a, in);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < Ri::STAGES - 1; ++i) fetch(i);
  for (int i = 0; i < mine; ++i) {
    fetch(i + Ri::STAGES - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(Ri::STAGES - 1) : "memory");
    const uint4* d = own + (i % Ri::STAGES) * Ri::VECS * 32;
    uint4 xa[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) xa[m][h] = d[(2 * m + h) * 32];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (!((act >> n) & 1u)) continue;
      const uint4 bw = d[(2 * MT + n) * 32];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        mma<T>(acc[m][n], xa[m][0].x, xa[m][1].x, xa[m][0].y, xa[m][1].y, bw.x, bw.y);
        mma<T>(acc[m][n], xa[m][0].z, xa[m][1].z, xa[m][0].w, xa[m][1].w, bw.z, bw.w);
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();   // the ring becomes the sums
  float* part = sums + warp * E;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      *reinterpret_cast<float2*>(part + (m * 16 + g) * N + n * 8 + 2 * c) = make_float2(acc[m][n][0], acc[m][n][1]);
      *reinterpret_cast<float2*>(part + (m * 16 + g + 8) * N + n * 8 + 2 * c) = make_float2(acc[m][n][2], acc[m][n][3]);
    }
  __syncthreads();
  cluster_started();
  const int share = E / cs;   // cs is a power of two up to 16, E a multiple of 256
  const int used = tile.z * N;
#pragma unroll 4
  for (int e = threadIdx.x; e < E; e += SW * 32) {
    if (e >= used) break;
    float v = sums[e];
#pragma unroll
    for (int w = 1; w < SW; ++w) v += sums[w * E + e];
    const int owner = e * cs / E;   // e / share
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(in_cta(got + cr * share + e - owner * share, owner)), "f"(v) : "memory");
  }
  cluster_pushed();
  for (int i = threadIdx.x; i < share; i += SW * 32) {
    const int e = cr * share + i, r = e / N, col = col0 + e % N;
    if (r >= tile.z || col >= p.SR) continue;
    float v = got[i];
    for (int k = 1; k < cs; ++k) v += got[k * share + i];
    // past the rank: exact zeros, also where x holds an infinity
    p.t[(int64_t)(tile.y + r) * p.SR + col] = e % 8 < s_left[e % N / 8] ? v : 0.f;
  }
}

// ------------------------------------------------------------------------- expand ----
// KS = max_rank / 16 steps of k; a warp owns NC * 8 columns, a CTA EW such groups of one
// part.  The tile's t is split into its high and low halves once for the CTA, into shared
// memory in the order of the MMA's fragments (split by every warp for itself and fetched from
// L2 in the loop it cost 1 to 4 us a call).
template <typename T, int KS, int NC>
__global__ void __launch_bounds__(EW * 32) expand_kernel(const Params p, const int cblocks) {
  extern __shared__ uint4 frag[];   // [steps of 16 rows][KS][hi, lo][32 lanes], then the row scales (f16)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  // column blocks of a tile after one another, so that whole rows of y and out are in flight
  const int blk = blockIdx.x / cblocks;
  int cb = blockIdx.x - blk * cblocks, part = 0, first = 0;
  for (;; ++part) {   // the part that this block of columns lies in
    const int n = (p.width[part] + EW * NC * 8 - 1) / (EW * NC * 8);
    if (cb < n) break;
    cb -= n;
    first += p.width[part];
  }
  const int col0 = (cb * EW + warp) * NC * 8, left = p.width[part] - col0;   // columns of this part from col0 on
  const int4 tile = p.tiles[blk];
  const int rank = tile.x < 0 ? 0 : p.ranks[tile.x * p.parts + part], msteps = (tile.z + 15) / 16;
  const float scale = tile.x < 0 ? 0.f : p.scales[tile.x * p.parts + part];
  float* row_scale = reinterpret_cast<float*>(frag + msteps * KS * 64);
  // rows g and g + 8 of a 16-row step
  int64_t row[2];
  uint4 yv[NC / 4][2];
  const auto load = [&](int m, int64_t (&rw)[2], uint4 (&v)[NC / 4][2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = m * 16 + h * 8 + g;
      rw[h] = r < tile.z ? p.order[tile.y + r] : -1;
#pragma unroll
      for (int q = 0; q < NC / 4; ++q)
        if (rw[h] >= 0 && q * 32 + 8 * c < left)
          v[q][h] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.y) + rw[h] * p.ys + first + col0 + q * 32 +
                                                    8 * c);
    }
  };
  load(0, row, yv);
  // B fragments: k of the lane in step ks is ks * 16 + 4c..4c+3; column of n-tile 4q + j,
  // n = g, is 32q + 8 (g / 2) + 2j + g % 2, so that a lane's results are 8 adjacent columns
  uint2 bw[NC][KS];
  if (rank > 0) {
    const T* bb = static_cast<const T*>(p.b) + ((int64_t)tile.x * p.OUT + first + col0) * p.R + 4 * c;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int col = (n / 4) * 32 + 8 * (g >> 1) + 2 * (n % 4) + (g & 1);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        bw[n][ks] = col < left && ks * 16 < rank ? *reinterpret_cast<const uint2*>(bb + (int64_t)col * p.R + ks * 16)
                                                 : make_uint2(0u, 0u);
    }
  }
  // t of the shrink kernel; also before the first store, so that this grid never ends
  // before the one that still reads x and writes the workspace
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (rank > 0) {
    for (int m = warp; m < msteps; m += EW) {
      float sc[2];
      uint4 f[KS][2];
      split_t<T, KS>(p.t + (int64_t)(tile.y + m * 16) * p.SR + part * p.R, p.SR, tile.z - m * 16, rank, g, c, f, sc);
      if (!__is_same(T, __nv_bfloat16) && c == 0) row_scale[m * 16 + g] = sc[0], row_scale[m * 16 + 8 + g] = sc[1];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        frag[(m * KS + ks) * 64 + lane] = f[ks][0];
        frag[(m * KS + ks) * 64 + 32 + lane] = f[ks][1];
      }
    }
    __syncthreads();   // rank is the same for the whole CTA
  }
  if (left <= 0) return;
  for (int m = 0; m < msteps; ++m) {
    int64_t next_row[2] = {-1, -1};
    uint4 next[NC / 4][2];
    if (m + 1 < msteps) load(m + 1, next_row, next);
    float acc[NC][4];
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
    float sc[2] = {scale, scale};
    if (rank > 0) {
      if (!__is_same(T, __nv_bfloat16)) {
        sc[0] *= row_scale[m * 16 + g];
        sc[1] *= row_scale[m * 16 + 8 + g];
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if (ks * 16 >= rank) break;
        const uint4 hi = frag[(m * KS + ks) * 64 + lane], lo = frag[(m * KS + ks) * 64 + 32 + lane];
#pragma unroll
        for (int n = 0; n < NC; ++n) {
          mma<T>(acc[n], lo.x, lo.y, lo.z, lo.w, bw[n][ks].x, bw[n][ks].y);
          mma<T>(acc[n], hi.x, hi.y, hi.z, hi.w, bw[n][ks].x, bw[n][ks].y);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int q = 0; q < NC / 4; ++q) {
        if (row[h] < 0 || q * 32 + 8 * c >= left) continue;
        uint4 o = yv[q][h];
        if (rank > 0) {
          T* oe = reinterpret_cast<T*>(&o);
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              oe[2 * j + e] = from_f<T>(fmaf(sc[h], acc[4 * q + j][2 * h + e], to_f(oe[2 * j + e])));
        }
        *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + row[h] * p.os + first + col0 + q * 32 + 8 * c) = o;
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      row[h] = next_row[h];
#pragma unroll
      for (int q = 0; q < NC / 4; ++q) yv[q][h] = next[q][h];
    }
  }
}

template <typename T, int MT, int NT>
int launch_shrink(const Params& p, int tiles, int groups, cudaStream_t st) {
  const size_t smem = Ring<MT, NT>::BYTES;
  static std::atomic<int> have[64], places[64][5];   // places: clusters of 1 .. 16 CTAs that a device holds (-1: none)
  cudaError_t e = allow_smem(shrink_kernel<T, MT, NT>, (int)smem, have);
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(SW * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const auto cluster = [&](int cs) {
    cfg.gridDim = dim3((unsigned)(tiles * cs), (unsigned)groups);
    at[0].val.clusterDim.x = (unsigned)cs, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  };
  // CTAs that share a tile's k: as many as the device holds at once, with at least two steps of 32
  // for each warp, 16 at most (more than the portable 8, so it has to be asked for).
  int dev = 0, l = 0;
  if (e == cudaSuccess) e = cudaGetDevice(&dev);
  for (; e == cudaSuccess && l < 4 && p.K >= 32 * SW * 2 << l; ++l) {
    cluster(2 << l);
    int n = dev < 64 ? places[dev][l + 1].load(std::memory_order_relaxed) : 0;
    if (n == 0) {
      cudaError_t q = l < 3 ? cudaSuccess : cudaFuncSetAttribute(shrink_kernel<T, MT, NT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (q == cudaSuccess) q = cudaOccupancyMaxActiveClusters(&n, shrink_kernel<T, MT, NT>, &cfg);
      if (q != cudaSuccess) cudaGetLastError();   // not an error of this call: a smaller cluster
      if (q != cudaSuccess || n == 0) n = -1;
      if (dev < 64) places[dev][l + 1].store(n, std::memory_order_relaxed);
    }
    if ((int64_t)tiles * groups > n + n / 16) break;   // a few more than fit, or tiles without an adapter, cost less than half the CTAs
  }
  cluster(1 << l);
  if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, shrink_kernel<T, MT, NT>, p);
  if (e != cudaSuccess) {
    set_error("lora shrink_kernel: %s", cudaGetErrorString(e));
    return SPX_ERR_CUDA;
  }
  return launch_status("lora shrink_kernel");
}

template <typename T, int KS, int NC>
int launch_expand(const Params& p, int tiles, int tile_rows, cudaStream_t st) {
  int cblocks = 0;
  for (int s = 0; s < p.parts; ++s) cblocks += (p.width[s] + EW * NC * 8 - 1) / (EW * NC * 8);
  SPX_REQUIRE((int64_t)tiles * cblocks <= 0x7fffffff, SPX_ERR_SHAPE, "spx_lora_add: too many rows");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(tiles * cblocks));
  cfg.blockDim = dim3(EW * 32);
  cfg.dynamicSmemBytes = (size_t)tile_rows / 16 * KS * 1024 + tile_rows * sizeof(float);   // up to 16.1 KB
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, expand_kernel<T, KS, NC>, p, cblocks);
  if (e != cudaSuccess) {
    set_error("lora expand_kernel: %s", cudaGetErrorString(e));
    return SPX_ERR_CUDA;
  }
  return launch_status("lora expand_kernel");
}

template <typename T>
int launch_shrink_rows(const Params& p, int tiles, int tile_rows, cudaStream_t st) {
  // Columns of a CTA: 16 while two CTAs an SM hold the whole grid (one request on q|k|v 5.6 us
  // against 6.8 with 48), else as many as leave the rows enough warps: each group reads x again.
  const int cols = (int64_t)tiles * (p.SR / 16) * 8 <= 2 * 148 ? 16 : tile_rows == 16 ? 32 : 64;
  const int groups = (p.SR + cols - 1) / cols;
  const int nt = ((p.SR / 8 + groups - 1) / groups + 1) / 2 * 2;  // 2, 4, 6 or 8; 2 or 4 of up to 32 columns
  if (tile_rows == 16) return nt == 2 ? launch_shrink<T, 1, 2>(p, tiles, groups, st) : launch_shrink<T, 1, 4>(p, tiles, groups, st);
  return nt == 2   ? launch_shrink<T, 2, 2>(p, tiles, groups, st)
         : nt == 4 ? launch_shrink<T, 2, 4>(p, tiles, groups, st)
         : nt == 6 ? launch_shrink<T, 2, 6>(p, tiles, groups, st)
                   : launch_shrink<T, 2, 8>(p, tiles, groups, st);
}

template <typename T>
int launch(const Params& p, int dtype, int tiles, int tile_rows, cudaStream_t st) {
  if (tile_rows == 128) {
    const int rc = shrink_block_launch(p, dtype, tiles, st);
    return rc == SPX_OK ? expand_block_launch(p, dtype, tiles, st) : rc;
  }
  const int rc = launch_shrink_rows<T>(p, tiles, tile_rows, st);
  if (rc != SPX_OK) return rc;
  switch (p.R / 16) {
    case 1:
      // few columns in all: half as many a warp, so that each is done sooner (one row on 6144 columns
      // 4.66 us a call against 4.76, 12 x 7 rows on 6568 7.05 against 7.33; at rank 64, 6 rows on
      // 2936 columns, 6.4 against 5.7)
      if ((int64_t)tiles * p.OUT <= 4 * 148 * 128) return launch_expand<T, 1, 4>(p, tiles, tile_rows, st);
      return launch_expand<T, 1, 8>(p, tiles, tile_rows, st);
    case 2: return launch_expand<T, 2, 8>(p, tiles, tile_rows, st);
    case 3: return launch_expand<T, 3, 8>(p, tiles, tile_rows, st);
    case 4: return launch_expand<T, 4, 8>(p, tiles, tile_rows, st);
    case 5:
    case 6: return launch_expand<T, 6, 4>(p, tiles, tile_rows, st);
    default: return launch_expand<T, 8, 4>(p, tiles, tile_rows, st);
  }
}

// the inner products and the word that says a wait expired
static size_t workspace_bytes(const spx_lora_args* a) {
  return ((size_t)a->num_rows * a->parts * a->max_rank + 4) * sizeof(float);
}

static int validate(const spx_lora_args* a) {
  SPX_REQUIRE(a, SPX_ERR_NULL, "spx_lora_add: args are required");
  SPX_REQUIRE(a->dtype == SPX_F16 || a->dtype == SPX_BF16, SPX_ERR_UNSUPPORTED,
              "spx_lora_add: dtype must be F16 or BF16");
  SPX_REQUIRE(a->num_tiles >= 0 && a->num_rows >= 0 && (a->tile_rows == 16 || a->tile_rows == 32 || a->tile_rows == 128) &&
                  a->num_tiles <= (1 << 27),
              SPX_ERR_SHAPE, "spx_lora_add: bad tiling: %d tiles of %d rows", a->num_tiles, a->tile_rows);
  SPX_REQUIRE(a->in_features >= 8 && a->in_features % 8 == 0 && a->in_features <= (1 << 24), SPX_ERR_SHAPE,
              "spx_lora_add: in_features %d must be a multiple of 8", a->in_features);
  SPX_REQUIRE(a->parts >= 1 && a->parts <= SPX_LORA_MAX_PARTS && a->slots >= 1 && a->max_rank >= 16 &&
                  a->max_rank % 16 == 0 && a->max_rank <= SPX_LORA_MAX_RANK,
              SPX_ERR_SHAPE, "spx_lora_add: bad pool: %d parts, %d slots, max_rank %d", a->parts, a->slots, a->max_rank);
  int64_t out = 0;
  for (int s = 0; s < a->parts; ++s) {
    SPX_REQUIRE(a->part_width[s] >= 8 && a->part_width[s] % 8 == 0 && a->part_width[s] <= (1 << 22), SPX_ERR_SHAPE,
                "spx_lora_add: width %d of part %d must be a multiple of 8", a->part_width[s], s);
    out += a->part_width[s];
  }
  // the rows of A and B are counted in 32 bits (the coordinates of a copy's box)
  SPX_REQUIRE(a->slots * (out > a->parts * a->max_rank ? out : (int64_t)a->parts * a->max_rank) <= 0x7fffffff, SPX_ERR_SHAPE,
              "spx_lora_add: %d slots of %lld columns are too many", a->slots, (long long)out);
  if (a->num_tiles == 0) return SPX_OK;
  SPX_REQUIRE(a->x && a->y && a->out && a->a && a->b && a->ranks && a->scales && a->tiles && a->order, SPX_ERR_NULL,
              "spx_lora_add: every pointer is required");
  SPX_REQUIRE(a->x_stride >= a->in_features && a->y_stride >= out && a->out_stride >= out, SPX_ERR_SHAPE,
              "spx_lora_add: a row stride is shorter than a row");
  SPX_REQUIRE(aligned16(a->x) && aligned16(a->y) && aligned16(a->out) && aligned16(a->a) && aligned16(a->b) &&
                  aligned16(a->tiles) && aligned16(a->workspace) &&
                  (a->x_stride | a->y_stride | a->out_stride) % 8 == 0,
              SPX_ERR_ALIGN, "spx_lora_add: rows of x, y and out, A, B, tiles and workspace must start on 16 bytes");
  return SPX_OK;
}

}  // namespace lora
}  // namespace spx

using namespace spx;

size_t spx_lora_workspace_size(const spx_lora_args* a) {
  if (!a || lora::validate(a) != SPX_OK) return 0;
  return lora::workspace_bytes(a);
}

int spx_lora_add(const spx_lora_args* a, void* stream) {
  const int rc = lora::validate(a);
  if (rc != SPX_OK || a->num_tiles == 0) return rc;
  const size_t need = lora::workspace_bytes(a);
  SPX_REQUIRE(a->workspace && a->workspace_bytes >= need, SPX_ERR_WORKSPACE,
              "spx_lora_add: workspace of %zu bytes needed, %zu given", need, a->workspace ? a->workspace_bytes : 0);
  lora::Params p{};
  p.x = a->x, p.y = a->y, p.a = a->a, p.b = a->b, p.out = a->out;
  p.xs = a->x_stride, p.ys = a->y_stride, p.os = a->out_stride;
  p.ranks = a->ranks, p.scales = a->scales;
  p.tiles = static_cast<const int4*>(static_cast<const void*>(a->tiles));
  p.order = a->order, p.t = a->workspace;
  p.rows = a->num_rows, p.slots = a->slots;
  p.K = a->in_features, p.parts = a->parts, p.R = a->max_rank, p.SR = a->parts * a->max_rank;
  for (int s = 0; s < a->parts; ++s) p.width[s] = a->part_width[s], p.OUT += a->part_width[s];
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return a->dtype == SPX_BF16 ? lora::launch<__nv_bfloat16>(p, a->dtype, a->num_tiles, a->tile_rows, st)
                              : lora::launch<__half>(p, a->dtype, a->num_tiles, a->tile_rows, st);
}
