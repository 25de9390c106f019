// Rules on a decode step's logits and the greedy choice under them (spx_logits_rules,
// include/spx.h): repetition, frequency and presence penalties, sparse biases, a grammar's
// bit mask, argmax.  One pass over the row.  Bound by memory: the logits once in, once out
// when they are wanted, and two bitmaps of 1/16 of the bytes of 16-bit logits each (tokens
// that a rule touches, allowed tokens).  The touched tokens - seen before or biased, a few
// per cent - are only noted in the streaming pass, in a list in shared memory; then the
// threads take them one each, with the loads that they need (count, bias) side by side.
// Handled where they were met, they held up every warp that had one.
// Device time of 128 rows of 131072 float32 logits, every rule on: 71 us with the rules in
// the stream, 54 with the list worked off every two units of a lane, 31 to 32 with four units
// in flight a lane and the list at the end (floor 21.7 us; 25 without touched tokens; a plain
// copy of the logits 22).  What is left is the list: its loads come after the stream's.
// A row is shared by a cluster of CTAs; their best tokens meet over distributed shared
// memory, so that one launch gives the token and no workspace is shared by calls.  Each
// operation is rounded in float32 (no contraction), as the float32 expression is.

#include <atomic>

#include "spx_common.cuh"

namespace spx {
namespace lgt {

constexpr int NT = 256, WARPS = NT / 32;
constexpr int BATCH = 3;     // listed tokens that a thread takes together
constexpr int SEG = 16384;   // tokens of a CTA between two runs through its list (16 bits an entry, 32 KB)

__device__ __forceinline__ uint32_t cluster_dim() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

struct Params {
  const void* x;
  void* out;
  int64_t xs, os;
  int64_t* token;
  const float *rep, *freq, *pres;
  const uint32_t *allow, *bbits;
  uint32_t *seen, *touched;
  int32_t* counts;
  const int32_t* bfirst;
  const float* bvals;
  int64_t as;
  int V, W, record;
};

__device__ __forceinline__ float max_nan(float a, float b) {   // a NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Larger for the better token: value first (NaN on top, -0 as 0), then the lower index.
__device__ __forceinline__ unsigned long long key(float v, int t) {
  v += 0.f;
  const uint32_t u = __float_as_uint(v);
  const uint32_t k = v != v ? 0xffffffffu : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)k << 32) | (uint32_t)~t;
}

// A warp takes tiles of U x 32 units, a unit being the N tokens of one 16-byte boundary of
// memory, wherever the row starts: a row that starts `off` values past a boundary begins
// with a part of a unit.  All loads of a tile are issued together (U x 16 bytes a lane).
// Lane l holds the tile's l-th 32 bits of each bitmap, moved by `off`, and the units get
// theirs by shuffles.  The CTAs of a cluster take turns at tiles, so that a dense stretch of
// touched tokens (low ids are common ones) is shared.
template <typename T, int U_>
struct Tile {
  static constexpr int N = 16 / (int)sizeof(T), U = U_, TOKENS = 32 * N * U, WORDS = TOKENS / 32;
};

// Word `lane` of the tile's bits: token 32 * lane of the tile is token w * 32 - off of the row.
__device__ __forceinline__ uint32_t tile_bits(const uint32_t* row, int w, int words, int off, int W, int lane) {
  const uint32_t mine = lane < words && w < W ? row[w] : 0u;
  if (!off) return mine;
  uint32_t before = __shfl_up_sync(0xffffffffu, mine, 1);
  if (lane == 0) before = w > 0 ? row[w - 1] : 0u;
  return __funnelshift_l(before, mine, off);
}

__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

template <typename T, int U_>
__global__ void __launch_bounds__(NT, 4) rules_kernel(const Params p) {
  using Ti = Tile<T, U_>;
  __shared__ unsigned long long red[WARPS];
  __shared__ unsigned long long tops[16];   // of the cluster's CTAs, in the first one's shared memory
  __shared__ int listed[2];
  extern __shared__ uint16_t list[];
  constexpr int N = Ti::N, U = Ti::U, TOK = Ti::TOKENS, WORDS = Ti::WORDS;
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // "my shared memory exists"
  const int cs = (int)cluster_dim(), cr = (int)cluster_rank();
  const int64_t b = blockIdx.x / cs;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = p.V, W = p.W;
  const T* x = static_cast<const T*>(p.x) + b * p.xs;
  T* out = p.out ? static_cast<T*>(p.out) + b * p.os : nullptr;
  const int off = (int)((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % N);
  const bool vout = out && (int)((reinterpret_cast<uintptr_t>(out) / sizeof(T)) % N) == off;
  const uint32_t* tb = p.touched ? p.touched + b * W : nullptr;
  const uint32_t* ab = p.allow ? p.allow + b * p.as : nullptr;
  const int32_t* cnt = p.counts + b * (int64_t)V;
  const float rep = p.rep ? p.rep[b] : 1.f, freq = p.freq ? p.freq[b] : 0.f, pres = p.pres ? p.pres[b] : 0.f;
  if (tid < 2) listed[tid] = 0;
  __syncthreads();
  // the best unit of the tokens without a rule: its largest value, first token, logits and the
  // tokens that count; a thread's units ascend
  float best = -INFINITY;
  int best_t = 0;
  uint4 best_raw = make_uint4(0u, 0u, 0u, 0u);
  uint32_t best_ok = 0u;
  unsigned long long k = 0ull;
  const int tiles = (V + off + TOK - 1) / TOK, step = WARPS * cs;
  constexpr int ROUNDS = SEG / (WARPS * TOK);
  for (int r0 = 0, it = 0; r0 * step < tiles; r0 += ROUNDS, it ^= 1) {
    for (int r = 0; r < ROUNDS; ++r) {
      const int tile = (r0 + r) * step + warp * cs + cr;
      if (tile >= tiles) break;
      const int base = tile * TOK - off;   // first token
      const bool whole = base >= 0 && base + TOK <= V;
      uint4 raw[U];
      if (whole) {
#pragma unroll
        for (int j = 0; j < U; ++j) raw[j] = *reinterpret_cast<const uint4*>(x + base + (j * 32 + lane) * N);
      } else {
#pragma unroll
        for (int j = 0; j < U; ++j)
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const int t = base + (j * 32 + lane) * N + e;
            reinterpret_cast<T*>(&raw[j])[e] = t >= 0 && t < V ? x[t] : from_f<T>(0.f);
          }
      }
      const int w = tile * WORDS + lane;
      uint32_t okw = ab ? tile_bits(ab, w, WORDS, off, W, lane) : 0xffffffffu;   // allowed, and of the row
      uint32_t tw = tb ? tile_bits(tb, w, WORDS, off, W, lane) : 0u;             // touched
      if (!whole) {
        const int t = base + 32 * lane;
        if (t < 0) okw &= 0xffffffffu << off;
        if (t + 32 > V) okw &= t >= V ? 0u : 0xffffffffu >> (t + 32 - V);
      }
      tw = WORDS < 32 && lane >= WORDS ? 0u : tw & okw;
      const bool masks = ab || !whole, any_touch = tb && __any_sync(0xffffffffu, tw != 0u);
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int t0 = base + (j * 32 + lane) * N, src = (j * 32 + lane) * N / 32, sh = lane * N % 32;
        float v[N];
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = to_f(reinterpret_cast<const T*>(&raw[j])[e]);
        uint32_t ok = (1u << N) - 1u;
        if (masks) {
          ok &= __shfl_sync(0xffffffffu, okw, src) >> sh;
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (!((ok >> e) & 1u)) v[e] = -INFINITY;
        }
        if (out) {   // a touched token's place holds its logit as it came in until the list is worked off
          if (vout && whole) {
            uint4 o = raw[j];
            if (masks) {
#pragma unroll
              for (int e = 0; e < N; ++e) reinterpret_cast<T*>(&o)[e] = from_f<T>(v[e]);
            }
            *reinterpret_cast<uint4*>(out + t0) = o;
          } else {
#pragma unroll
            for (int e = 0; e < N; ++e)
              if (t0 + e >= 0 && t0 + e < V) out[t0 + e] = from_f<T>(v[e]);
          }
        }
        if (any_touch) {
          const uint32_t touch = __shfl_sync(0xffffffffu, tw, src) >> sh;
          ok &= ~touch;
#pragma unroll
          for (int e = 0; e < N; ++e)
            if ((touch >> e) & 1u) v[e] = -INFINITY;
        }
        float m = max_nan(max_nan(v[0], v[1]), max_nan(v[2], v[3]));
        if (N == 8) m = max_nan(m, max_nan(max_nan(v[N - 4], v[N - 3]), max_nan(v[N - 2], v[N - 1])));
        if (!(m <= best) && best == best) best = m, best_t = t0, best_raw = raw[j], best_ok = ok;   // or the first NaN
      }
      if (any_touch) {
        constexpr int PART = TOK / 32;   // a lane's part of the tile: 8, 16 or 32 tokens, or 4
        uint32_t mine = __shfl_sync(0xffffffffu, tw, lane * PART / 32) >> (lane * PART % 32);
        if (PART < 32) mine &= (1u << (PART & 31)) - 1u;
        const int n = __popc(mine);
        int at = n;   // place in the list: the warp's lanes after one another
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int other = __shfl_up_sync(0xffffffffu, at, o);
          if (lane >= o) at += other;
        }
        int first = 0;
        if (lane == 31) first = atomicAdd(&listed[it], at);
        first = __shfl_sync(0xffffffffu, first, 31) + at - n;
        while (mine) {
          const int e = __ffs(mine) - 1;
          mine &= mine - 1;
          list[first++] = (uint16_t)((r * WARPS + warp) * TOK + lane * PART + e);
        }
      }
    }
    if (!tb) continue;
    __syncthreads();
    const int n = listed[it];
    if (tid == 0) listed[it ^ 1] = 0;
    for (int i = tid; i < n; i += NT * BATCH) {   // the loads of a batch first: they have the latency
      int t[BATCH], c[BATCH], bf[BATCH];
      uint32_t sw[BATCH], bw[BATCH];
      float v[BATCH];
#pragma unroll
      for (int q = 0; q < BATCH; ++q) {
        t[q] = -1, c[q] = 0, bf[q] = 0, sw[q] = 0xffffffffu, bw[q] = 0u, v[q] = 0.f;
        if (i + q * NT < n) {
          const int l = list[i + q * NT], rw = l / TOK;   // round and warp that noted it
          t[q] = ((r0 + rw / WARPS) * step + rw % WARPS * cs + cr) * TOK - off + l % TOK;
          v[q] = to_f(x[t[q]]);
          if (p.freq || p.pres) c[q] = cnt[t[q]];
          if (p.bbits) {   // else every touched token is a seen one
            const int64_t wb = b * W + (t[q] >> 5);
            sw[q] = p.seen ? p.seen[wb] : 0u, bw[q] = p.bbits[wb], bf[q] = p.bfirst[wb];
          }
        }
      }
#pragma unroll
      for (int q = 0; q < BATCH; ++q) {
        if (t[q] < 0) break;
        const int sh = t[q] & 31;
        float f = v[q];
        if (p.rep && ((sw[q] >> sh) & 1u)) f = f > 0.f ? __fdiv_rn(f, rep) : __fmul_rn(f, rep);
        if (c[q] > 0) f = __fsub_rn(__fsub_rn(f, __fmul_rn(freq, (float)c[q])), pres);
        // the biases lie by row and token: the first one of this word, then by the bits before this one
        if ((bw[q] >> sh) & 1u) f = __fadd_rn(f, p.bvals[bf[q] + __popc(bw[q] & ((1u << sh) - 1u))]);
        if (out) out[t[q]] = from_f<T>(f);
        const unsigned long long other = f == -INFINITY ? 0ull : key(f, t[q]);   // -inf: as if not there
        k = other > k ? other : k;
      }
    }
    __syncthreads();
  }
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  if (!p.token && !p.record) return;   // uniform over the grid
  if (best_ok) {   // something above -inf (or a NaN): the first of its unit
#pragma unroll
    for (int e = N - 1; e >= 0; --e) {
      const float v = to_f(reinterpret_cast<const T*>(&best_raw)[e]);
      if (((best_ok >> e) & 1u) && (v == best || (v != v && best != best))) {
        const unsigned long long other = key(v, best_t + e);
        k = other > k ? other : k;
      }
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, k, o);
    k = other > k ? other : k;
  }
  if (lane == 0) red[warp] = k;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < WARPS; ++w) k = red[w] > k ? red[w] : k;
    const uint32_t at = mapa((uint32_t)__cvta_generic_to_shared(&tops[cr]), 0);
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(k) : "memory");
  }
  __syncwarp();
  // every CTA's best lies with the first one, and every read of the history is done
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (cr == 0 && tid == 0) {
    for (int c = 0; c < cs; ++c) k = tops[c] > k ? tops[c] : k;
    const int t = k ? (int)~(uint32_t)k : 0;
    if (p.token) p.token[b] = t;
    if (p.record) {
      p.seen[b * W + (t >> 5)] |= 1u << (t & 31);
      if (p.touched != p.seen) p.touched[b * W + (t >> 5)] |= 1u << (t & 31);
      p.counts[b * (int64_t)V + t] += 1;
    }
  }
}

__global__ void observe_kernel(const int64_t* tokens, int64_t stride, int count, int V, int W, uint32_t* seen,
                               uint32_t* touched, int32_t* counts) {
  const int64_t b = blockIdx.y;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < count; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t t = tokens[b * stride + i];
    if (t < 0 || t >= V) continue;
    // whole numbers: any order gives the same
    atomicOr(seen + b * W + (t >> 5), 1u << (t & 31));
    if (touched != seen) atomicOr(touched + b * W + (t >> 5), 1u << (t & 31));
    if (counts) atomicAdd(counts + b * V + t, 1);
  }
}

// Whether the device takes clusters of 16 CTAs of a kernel (more than the portable 8), which has to
// be asked for once.
template <typename F>
bool wide_clusters(F kernel, std::atomic<int> (&known)[64]) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return false;
  int k = known[dev].load(std::memory_order_relaxed);
  if (k == 0) {
    int n = 0;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(16), cfg.blockDim = dim3(NT), cfg.dynamicSmemBytes = 2 * SEG;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 16, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    cfg.attrs = at, cfg.numAttrs = 1;
    const bool ok = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                    cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) == cudaSuccess && n > 0;
    if (!ok) cudaGetLastError();   // not an error of this call
    known[dev].store(k = ok ? 2 : 1, std::memory_order_relaxed);
  }
  return k == 2;
}

// CTAs of a row: as many as are resident at once (four an SM), at most the portable 8; or 16 where
// those leave a third of the places free, which clusters of that size need (one row of 131072 bf16
// 6.4 us with 16, 7.8 with 8; eight rows 6.9 and 8.4; 30 rows of 50000 7.8 and 6.5).
inline int row_ctas(int batch) {
  const int fit = 4 * 148 / batch;
  return fit >= 24 ? 16 : fit > 8 ? 8 : fit < 1 ? 1 : fit;
}

template <typename T, int U>
int launch_tiles(const Params& p, int batch, cudaStream_t st) {
  // CTAs of a row: at most one for a round of tiles of its warps.
  static std::atomic<int> known[64];
  constexpr int ROUND = WARPS * Tile<T, U>::TOKENS;
  const int most = (p.V + Tile<T, U>::N + ROUND - 1) / ROUND;
  int cs = row_ctas(batch);
  cs = cs > most ? most : cs;
  if (cs > 8 && !wide_clusters(rules_kernel<T, U>, known)) cs = 8;
  const int64_t mine = (int64_t)((most + cs - 1) / cs) * ROUND;
  const size_t smem = p.touched ? 2 * (size_t)(mine < SEG ? mine : SEG) : 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(batch * cs));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)cs, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, rules_kernel<T, U>, p);
  if (e != cudaSuccess) {
    set_error("logits rules_kernel: %s", cudaGetErrorString(e));
    return SPX_ERR_CUDA;
  }
  return launch_status("logits rules_kernel");
}

template <typename T>
int launch(const Params& p, int batch, cudaStream_t st) {
  // Loads that a lane has in flight: as many as its CTAs need for the row at once, at most four
  // (128 x 131072 f32: 51 us with one, 31 with four).
  const int row = row_ctas(batch) * NT * Tile<T, 1>::N;
  if (p.V <= row) return launch_tiles<T, 1>(p, batch, st);
  if (p.V <= 2 * row) return launch_tiles<T, 2>(p, batch, st);
  return launch_tiles<T, 4>(p, batch, st);
}

}  // namespace lgt
}  // namespace spx

using namespace spx;

int spx_logits_rules(const spx_logits_args* a, void* stream) {
  SPX_REQUIRE(a, SPX_ERR_NULL, "spx_logits_rules: args are required");
  SPX_REQUIRE(dtype_ok(a->dtype), SPX_ERR_UNSUPPORTED, "spx_logits_rules: bad dtype %d", a->dtype);
  SPX_REQUIRE(a->batch >= 0 && a->batch <= (1 << 24) && a->vocab >= 1 && a->vocab <= (1 << 30), SPX_ERR_SHAPE,
              "spx_logits_rules: bad shape batch %d vocab %d", a->batch, a->vocab);
  SPX_REQUIRE(a->logits && (a->out || a->token || a->record), SPX_ERR_NULL,
              "spx_logits_rules: logits and at least one of out, token and record are required");
  SPX_REQUIRE(!(a->repetition || a->frequency || a->presence || a->record) || (a->seen_bits && a->counts),
              SPX_ERR_NULL, "spx_logits_rules: penalties and record need seen_bits and counts");
  SPX_REQUIRE(!(a->repetition || a->frequency || a->presence || a->record || a->bias_bits) || a->touched_bits,
              SPX_ERR_NULL, "spx_logits_rules: penalties, biases and record need touched_bits");
  SPX_REQUIRE(!a->bias_bits || (a->bias_first && a->bias_values), SPX_ERR_NULL,
              "spx_logits_rules: biases need bias_first and bias_values");
  const int W = (a->vocab + 31) / 32;
  SPX_REQUIRE((a->batch <= 1 || a->logits_stride >= a->vocab) && (!a->out || a->batch <= 1 || a->out_stride >= a->vocab) &&
                  (!a->allow || a->allow_stride == 0 || a->allow_stride >= W),
              SPX_ERR_SHAPE, "spx_logits_rules: a row stride is shorter than a row");
  if (a->batch == 0) return SPX_OK;
  lgt::Params p{};
  p.x = a->logits, p.out = a->out, p.xs = a->logits_stride, p.os = a->out_stride, p.token = a->token;
  p.rep = a->repetition, p.freq = a->frequency, p.pres = a->presence;
  p.seen = a->seen_bits, p.touched = a->touched_bits, p.counts = a->counts;
  p.bbits = a->bias_bits, p.bfirst = a->bias_first, p.bvals = a->bias_values;
  p.allow = a->allow, p.as = a->allow_stride;
  p.V = a->vocab, p.W = W, p.record = a->record;
  return SPX_DISPATCH_DTYPE(a->dtype, T,
                            [&] { return lgt::launch<T>(p, a->batch, reinterpret_cast<cudaStream_t>(stream)); });
}

int spx_logits_observe(const int64_t* tokens, int64_t stride, int batch, int count, int vocab, uint32_t* seen_bits,
                       uint32_t* touched_bits, int32_t* counts, void* stream) {
  SPX_REQUIRE(batch >= 0 && batch <= 65535 && count >= 0 && vocab >= 1 && vocab <= (1 << 30) && stride >= 0,
              SPX_ERR_SHAPE, "spx_logits_observe: bad shape batch %d count %d vocab %d", batch, count, vocab);
  SPX_REQUIRE(seen_bits && touched_bits && (tokens || count == 0), SPX_ERR_NULL,
              "spx_logits_observe: tokens, seen_bits and touched_bits are required");
  if (batch == 0 || count == 0) return SPX_OK;
  const unsigned gx = (unsigned)(count < 256 * 64 ? (count + 255) / 256 : 64);
  lgt::observe_kernel<<<dim3(gx, (unsigned)batch), 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      tokens, stride, count, vocab, (vocab + 31) / 32, seen_bits, touched_bits, counts);
  return launch_status("logits observe_kernel");
}
