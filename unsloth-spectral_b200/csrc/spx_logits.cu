// Rules on a decode step's logits and the greedy choice under them (spx_logits_rules,
// include/spx.h): repetition, frequency and presence penalties, sparse biases, a grammar's
// bit mask, argmax.  One pass over the row.  Bound by memory (the logits once in, once out
// when they are wanted): the history is kept as bitmaps, 1/16 of the bytes of 16-bit
// logits each, and the int32 counts and bias values are read only at tokens whose bit is
// set.  A row is shared by a cluster of CTAs; their best tokens meet over distributed
// shared memory, so that one launch gives the token and no workspace is shared by calls.
// Each operation is rounded in float32 (no contraction), as the float32 expression is.
#include <cooperative_groups.h>

#include "spx_common.cuh"

namespace spx {
namespace lgt {

constexpr int NT = 512;

struct Params {
  const void* x;
  void* out;
  int64_t xs, os;
  int64_t* token;
  const float *rep, *freq, *pres;
  const uint32_t *pbits, *allow, *bbits;
  uint32_t* obits;
  int32_t* counts;
  const int32_t *brows, *btoks;
  const float* bvals;
  int64_t as;
  int V, W, record;
};

// What one row's rules are.
struct Row {
  const uint32_t *pb, *ob, *bb, *al;
  const int32_t* cnt;
  const int32_t* btok;
  const float* bval;
  int nb;
  float rep, freq, pres;
};

__device__ __forceinline__ float bias_of(const Row& r, int t) {
  int lo = 0, hi = r.nb;
  while (lo < hi) {
    const int m = (lo + hi) >> 1;
    if (r.btok[m] < t) lo = m + 1;
    else hi = m;
  }
  return lo < r.nb && r.btok[lo] == t ? r.bval[lo] : 0.f;
}

// A token that one of the bits names.
__device__ __forceinline__ float touched(const Row& r, float x, int t, bool out, bool seen, bool bias) {
  if (seen) x = x > 0.f ? __fdiv_rn(x, r.rep) : __fmul_rn(x, r.rep);
  if (out) {
    if (r.freq != 0.f) x = __fsub_rn(x, __fmul_rn(r.freq, (float)r.cnt[t]));
    x = __fsub_rn(x, r.pres);
  }
  if (bias) x = __fadd_rn(x, bias_of(r, t));
  return x;
}

struct Best {
  float v;
  int i;
  __device__ __forceinline__ void see(float x, int t) {   // tokens in ascending order
    if (x > v || (x != x && v == v)) v = x, i = t;
  }
};

// Larger for the better token: value first (NaN on top, -0 as 0), then the lower index.
__device__ __forceinline__ unsigned long long key(const Best& b) {
  if (b.i == 0x7fffffff) return 0ull;   // nothing above -inf
  const float v = b.v + 0.f;
  const uint32_t u = __float_as_uint(v);
  const uint32_t k = v != v ? 0xffffffffu : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)k << 32) | (uint32_t)~b.i;
}

// 8 tokens a thread with 16-byte loads (VEC), or a warp over 32 tokens (one bitmap word)
// at a time for rows that do not start on 16 bytes.
template <typename T, bool VEC>
__global__ void __launch_bounds__(NT) rules_kernel(const Params p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cl = cg::this_cluster();
  __shared__ unsigned long long red[NT / 32];
  __shared__ unsigned long long top;
  const int cs = (int)cl.num_blocks(), cr = (int)cl.block_rank();
  const int64_t b = blockIdx.x / cs;
  const int tid = threadIdx.x, lane = tid & 31, V = p.V;
  const T* x = static_cast<const T*>(p.x) + b * p.xs;
  T* out = p.out ? static_cast<T*>(p.out) + b * p.os : nullptr;
  Row r;
  const bool hist = p.rep || p.freq || p.pres;
  r.pb = p.rep ? p.pbits + b * p.W : nullptr;
  r.ob = hist ? p.obits + b * p.W : nullptr;
  r.bb = p.bbits ? p.bbits + b * p.W : nullptr;
  r.al = p.allow ? p.allow + b * p.as : nullptr;
  r.cnt = p.counts + b * (int64_t)V;
  r.rep = p.rep ? p.rep[b] : 1.f;
  r.freq = p.freq ? p.freq[b] : 0.f;
  r.pres = p.pres ? p.pres[b] : 0.f;
  r.btok = nullptr, r.bval = nullptr, r.nb = 0;
  if (r.bb) {
    const int at = p.brows[b];
    r.btok = p.btoks + at, r.bval = p.bvals + at, r.nb = p.brows[b + 1] - at;
  }
  Best best{-INFINITY, 0x7fffffff};
  if (VEC) {
    const int units = (V + 7) / 8;
    for (int u = cr * NT + tid; u < units; u += cs * NT) {
      const int t0 = 8 * u, sh = t0 & 31, w = t0 >> 5, n = min(8, V - t0);
      uint32_t seen = 0, outb = 0, bias = 0, allow = 0xffu;
      if (r.ob) outb = (r.ob[w] >> sh) & 0xffu;
      if (r.pb) seen = (r.pb[w] >> sh) & 0xffu;
      if (r.bb) bias = (r.bb[w] >> sh) & 0xffu;
      if (r.al) allow = (r.al[w] >> sh) & 0xffu;
      seen |= outb;
      float v[8];
      if (n == 8) {
        uint4 raw[sizeof(T) / 2];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = reinterpret_cast<const uint4*>(x + t0)[i];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = to_f(reinterpret_cast<const T*>(raw)[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < n ? to_f(x[t0 + e]) : -INFINITY;
      }
      const uint32_t any = seen | bias;
      if (any) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (((any >> e) & 1u) && e < n)
            v[e] = touched(r, v[e], t0 + e, (outb >> e) & 1u, (seen >> e) & 1u, (bias >> e) & 1u);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (!((allow >> e) & 1u)) v[e] = -INFINITY;
        if (e < n) best.see(v[e], t0 + e);
      }
      if (out) {
        if (n == 8) {
          uint4 raw[sizeof(T) / 2];
#pragma unroll
          for (int e = 0; e < 8; ++e) reinterpret_cast<T*>(raw)[e] = from_f<T>(v[e]);
#pragma unroll
          for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(out + t0)[i] = raw[i];
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e < n) out[t0 + e] = from_f<T>(v[e]);
        }
      }
    }
  } else {
    constexpr int U = 4;
    const int words = p.W, warp = cr * (NT / 32) + (tid >> 5), nw = cs * (NT / 32);
    for (int w0 = warp; w0 < words; w0 += U * nw) {
      float v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = (w0 + u * nw) * 32 + lane;
        v[u] = w0 + u * nw < words && t < V ? to_f(x[t]) : -INFINITY;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int w = w0 + u * nw, t = w * 32 + lane;
        if (w >= words || t >= V) break;
        const bool outb = r.ob && ((r.ob[w] >> lane) & 1u);
        const bool seen = outb || (r.pb && ((r.pb[w] >> lane) & 1u));
        const bool bias = r.bb && ((r.bb[w] >> lane) & 1u);
        if (seen || bias) v[u] = touched(r, v[u], t, outb, seen, bias);
        if (r.al && !((r.al[w] >> lane) & 1u)) v[u] = -INFINITY;
        best.see(v[u], t);
        if (out) out[t] = from_f<T>(v[u]);
      }
    }
  }
  if (!p.token && !p.record) return;   // uniform over the grid
  unsigned long long k = key(best);
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, k, o);
    k = other > k ? other : k;
  }
  if (lane == 0) red[tid >> 5] = k;
  __syncthreads();
  if (tid < 32) {
    k = tid < NT / 32 ? red[tid] : 0ull;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, k, o);
      k = other > k ? other : k;
    }
    if (tid == 0) top = k;
  }
  cl.sync();   // every CTA's best is written, and every read of the history is done
  if (cr == 0 && tid == 0) {
    for (int c = 1; c < cs; ++c) {
      const unsigned long long other = *cl.map_shared_rank(&top, c);
      k = other > k ? other : k;
    }
    const int t = k ? (int)~(uint32_t)k : 0;
    if (p.token) p.token[b] = t;
    if (p.record) {
      p.obits[b * p.W + (t >> 5)] |= 1u << (t & 31);
      p.counts[b * (int64_t)V + t] += 1;
    }
  }
  cl.sync();   // no CTA leaves while its shared memory may be read
}

__global__ void observe_kernel(const int64_t* tokens, int64_t stride, int count, int V, int W, uint32_t* bits,
                               int32_t* counts) {
  const int64_t b = blockIdx.y;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < count; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t t = tokens[b * stride + i];
    if (t < 0 || t >= V) continue;
    atomicOr(bits + b * W + (t >> 5), 1u << (t & 31));   // whole numbers: any order gives the same
    if (counts) atomicAdd(counts + b * V + t, 1);
  }
}

template <typename T>
int launch(const Params& p, int batch, bool vec, cudaStream_t st) {
  // CTAs a row: enough that the grid fills the SMs (two CTAs each), at least 2048 tokens for
  // one of them, 8 at most (the portable cluster size).
  int cs = 1;
  while (cs < 8 && (int64_t)batch * cs < 2 * 148 && p.V >= 4096 * cs) cs *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(batch * cs));
  cfg.blockDim = dim3(NT);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)cs, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = vec ? cudaLaunchKernelEx(&cfg, rules_kernel<T, true>, p)
                            : cudaLaunchKernelEx(&cfg, rules_kernel<T, false>, p);
  if (e != cudaSuccess) {
    set_error("logits rules_kernel: %s", cudaGetErrorString(e));
    return SPX_ERR_CUDA;
  }
  return launch_status("logits rules_kernel");
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
  SPX_REQUIRE(!a->repetition || a->prompt_bits, SPX_ERR_NULL,
              "spx_logits_rules: a repetition penalty needs prompt_bits");
  SPX_REQUIRE(!(a->repetition || a->frequency || a->presence || a->record) || (a->output_bits && a->counts),
              SPX_ERR_NULL, "spx_logits_rules: penalties and record need output_bits and counts");
  SPX_REQUIRE(!a->bias_bits || (a->bias_rows && a->bias_tokens && a->bias_values), SPX_ERR_NULL,
              "spx_logits_rules: biases need bias_rows, bias_tokens and bias_values");
  const int W = (a->vocab + 31) / 32;
  SPX_REQUIRE((a->batch <= 1 || a->logits_stride >= a->vocab) && (!a->out || a->batch <= 1 || a->out_stride >= a->vocab) &&
                  (!a->allow || a->allow_stride == 0 || a->allow_stride >= W),
              SPX_ERR_SHAPE, "spx_logits_rules: a row stride is shorter than a row");
  if (a->batch == 0) return SPX_OK;
  lgt::Params p{};
  p.x = a->logits, p.out = a->out, p.xs = a->logits_stride, p.os = a->out_stride, p.token = a->token;
  p.rep = a->repetition, p.freq = a->frequency, p.pres = a->presence;
  p.pbits = a->prompt_bits, p.obits = a->output_bits, p.counts = a->counts;
  p.bbits = a->bias_bits, p.brows = a->bias_rows, p.btoks = a->bias_tokens, p.bvals = a->bias_values;
  p.allow = a->allow, p.as = a->allow_stride;
  p.V = a->vocab, p.W = W, p.record = a->record;
  const int64_t per = 16 / dtype_size(a->dtype);
  const bool vec = aligned16(a->logits) && (a->batch == 1 || a->logits_stride % per == 0) &&
                   (!a->out || (aligned16(a->out) && (a->batch == 1 || a->out_stride % per == 0)));
  return SPX_DISPATCH_DTYPE(a->dtype, T,
                            [&] { return lgt::launch<T>(p, a->batch, vec, reinterpret_cast<cudaStream_t>(stream)); });
}

int spx_logits_observe(const int64_t* tokens, int64_t stride, int batch, int count, int vocab, uint32_t* bits,
                       int32_t* counts, void* stream) {
  SPX_REQUIRE(batch >= 0 && batch <= 65535 && count >= 0 && vocab >= 1 && vocab <= (1 << 30) && stride >= 0,
              SPX_ERR_SHAPE, "spx_logits_observe: bad shape batch %d count %d vocab %d", batch, count, vocab);
  SPX_REQUIRE(bits && (tokens || count == 0), SPX_ERR_NULL, "spx_logits_observe: tokens and bits are required");
  if (batch == 0 || count == 0) return SPX_OK;
  const unsigned gx = (unsigned)(count < 256 * 64 ? (count + 255) / 256 : 64);
  lgt::observe_kernel<<<dim3(gx, (unsigned)batch), 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      tokens, stride, count, vocab, (vocab + 31) / 32, bits, counts);
  return launch_status("logits observe_kernel");
}
