// Per-head RMS norms of queries and keys with the position rotation in the same pass
// (spx_qk_norm_rope, include/spx.h).  For a head vector x of D values, h = D / 2:
//   y = x * rsqrt(sum(x^2) / D + eps) * w,   out = (y1 c - y2 s, y2 c + y1 s)
// Everything between the load and the store is float32 (one rounding, at the store: the
// norm's output never exists in the row type, so nothing is lost between it and the
// rotation).  Bound by memory: each value is read once and written once; the tables' rows
// come from L2 and are held in registers over the heads of a token.
// What it takes is warps: 8 x 4096 tokens of 32/8 heads of 128 bf16 take 115 us (floor 103)
// with 32 warps an SM and the next vector fetched ahead, at 64 registers a thread, of which most
// variants spill a few (8 to 60 bytes; eight lanes of bf16 28); 155 with four vectors at once and
// 16 warps, 126 without fetching ahead; narrower lanes (four values of a half) 150; more warps
// still 150 to 230.
#include <type_traits>

#include "spx_common.cuh"

namespace spx {
namespace qkn {

// Warps of a CTA.  Small ones: where the grid is about one wave, what counts is the SM that got the
// most (8 x 2048 rows of 12 heads of 128: bf16 21.4 us with eight warps, 20.0 with four; float32
// 42.9 with eight, 42.1 with four, 41.3 with two).
template <typename T>
constexpr int kWarps = sizeof(T) == 4 ? 2 : 4;
constexpr int ANY_WARPS = 8;

struct Params {
  const void *q, *k, *qw, *kw;
  void *qo, *ko;
  const float *cosT, *sinT;
  const int64_t* pos;
  int64_t qsb, qst, ksb, kst, psb, pst, pos0, kob, koh;
  int64_t rows;
  int T, Hq, H, D, len, rotk;
  float eps;
  int slots;   // groups of lanes that share the heads of one token row
};

__device__ __forceinline__ int64_t position(const Params& p, int64_t b, int64_t t) {
  const int64_t v = p.pos ? p.pos[b * p.psb + t * p.pst] : p.pos0 + t;
  return v < 0 ? 0 : (v >= p.len ? p.len - 1 : v);
}

// N consecutive values of a type, moved in words of up to 16 bytes.
template <typename T, int N>
struct Raw {
  static constexpr int BYTES = N * (int)sizeof(T), WORD = BYTES < 16 ? BYTES : 16;
  using W = typename std::conditional<WORD == 16, uint4, uint2>::type;
  W v[BYTES / WORD];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < BYTES / WORD; ++i) v[i] = reinterpret_cast<const W*>(p)[i];
  }
  __device__ __forceinline__ float get(int e) const { return to_f(reinterpret_cast<const T*>(v)[e]); }
  __device__ __forceinline__ void set(int e, float f) { reinterpret_cast<T*>(v)[e] = from_f<T>(f); }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < BYTES / WORD; ++i) reinterpret_cast<W*>(p)[i] = v[i];
  }
};

// The sum of ss over the G lanes of a group, the same in all of them.
template <int G>
__device__ __forceinline__ float group_sum(float ss, unsigned mask) {
  if ((G & (G - 1)) == 0) {
#pragma unroll
    for (int o = G / 2; o; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
    return ss;
  }
  constexpr int P = G <= 2 ? 2 : G <= 4 ? 4 : G <= 8 ? 8 : G <= 16 ? 16 : 32;
  const int lane = threadIdx.x & 31, l = lane % G, base = lane - l;
#pragma unroll
  for (int o = P / 2; o; o >>= 1) {   // complete in the first lane; the missing lanes are zeros
    const bool there = (l ^ o) < G;
    const float v = __shfl_sync(mask, ss, there ? base + (l ^ o) : lane);
    ss += there ? v : 0.f;
  }
  return __shfl_sync(mask, ss, base);
}

// G lanes hold one head vector: lane l its values Nl..Nl+N-1 of both halves, so that the two
// values of a rotation meet in one lane and only the sum of squares crosses lanes.  The
// table row is held in registers over the heads of a token; the weights are read from shared
// memory for each, which leaves registers for more warps.
template <typename T, int N, int G>
__device__ __forceinline__ void heads(const T* src, T* dst, int64_t dst_h, const T* w, const float (&c)[N],
                                      const float (&s)[N], bool turn, int j, int n, int step, bool on, int h, float eps,
                                      Raw<T, N>& a, Raw<T, N>& b, bool loaded) {
  if (j >= n) return;   // uniform over the G lanes; the shuffles below name them alone
  const unsigned mask = G == 32 ? 0xffffffffu : ((1u << (G & 31)) - 1u) << ((threadIdx.x & 31) / G * G);
  src += (int64_t)j * (2 * h);
  dst += j * dst_h;
  Raw<T, N> na, nb;
  if (on && !loaded) a.load(src), b.load(src + h);
  const float inv_d = 1.f / (float)(2 * h);
  while (true) {
    const bool more = j + step < n;
    src += step * 2 * h;
    if (on && more) na.load(src), nb.load(src + h);
    float ss = 0.f;
    if (on) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float x1 = a.get(e), x2 = b.get(e);
        ss = fmaf(x1, x1, ss);
        ss = fmaf(x2, x2, ss);
      }
    }
    ss = group_sum<G>(ss, mask);
    const float inv = rsqrtf(fmaf(ss, inv_d, eps));
    if (on) {
      Raw<T, N> wa, wb;
      wa.load(w), wb.load(w + h);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float y1 = a.get(e) * inv * wa.get(e), y2 = b.get(e) * inv * wb.get(e);
        a.set(e, turn ? y1 * c[e] - y2 * s[e] : y1);
        b.set(e, turn ? y2 * c[e] + y1 * s[e] : y2);
      }
      a.store(dst), b.store(dst + h);
    }
    if (!more) break;
    j += step, dst += step * dst_h;
    a = na, b = nb;
  }
}

template <typename T, int N, int G>
__global__ void __launch_bounds__(kWarps<T> * 32, (sizeof(T) == 4 ? 24 : 32) / kWarps<T>) vec_kernel(const Params p) {
  constexpr int WARPS = kWarps<T>;
  constexpr int NG = 32 / G;
  __shared__ __align__(16) T weights[2][2 * N * G];
  const int lane = threadIdx.x & 31, l = lane % G, h = p.D / 2;
  const uint32_t gi = (blockIdx.x * WARPS + (threadIdx.x >> 5)) * NG + lane / G;
  const bool live = lane < NG * G && gi < (uint32_t)p.rows * p.slots;
  const uint32_t row = live ? gi / (uint32_t)p.slots : 0u;
  const int64_t b = row / (uint32_t)p.T, t = row - (uint32_t)b * (uint32_t)p.T;
  const int g = (int)(gi - row * (uint32_t)p.slots), step = p.slots;
  const bool on = live && N * l < h;
  const T* q = static_cast<const T*>(p.q) + b * p.qsb + t * p.qst + N * l;
  const T* k = static_cast<const T*>(p.k) + b * p.ksb + t * p.kst + N * l;
  // the group's first vector is on its way before its position and table row are looked up
  Raw<T, N> xa, xb;
  if (on) {
    const T* x = g < p.Hq ? q + (int64_t)g * p.D : k + (int64_t)(g - p.Hq) * p.D;
    xa.load(x), xb.load(x + h);
  }
  const int64_t at = position(p, b, t) * p.D + N * l, plane = (int64_t)p.T * p.D;
  for (int i = threadIdx.x; i < p.D; i += WARPS * 32) {
    weights[0][i] = static_cast<const T*>(p.qw)[i];
    if (p.H) weights[1][i] = static_cast<const T*>(p.kw)[i];
  }
  float c[N], s[N];
  {
    Raw<float, N> cr, sr;
    if (on) cr.load(p.cosT + at), sr.load(p.sinT + at);
#pragma unroll
    for (int e = 0; e < N; ++e) c[e] = on ? cr.get(e) : 1.f, s[e] = on ? sr.get(e) : 0.f;
  }
  __syncthreads();
  if (!live) return;
  heads<T, N, G>(q, static_cast<T*>(p.qo) + b * p.Hq * plane + t * p.D + N * l, plane, weights[0] + N * l, c, s, true,
                        g, p.Hq, step, on, h, p.eps, xa, xb, true);
  // the group after the last one of the queries takes the first key head
  const int first = (g - p.Hq % step + step) % step;
  heads<T, N, G>(k, static_cast<T*>(p.ko) + b * p.kob + t * p.D + N * l, p.koh, weights[1] + N * l, c, s,
                        p.rotk != 0, first, p.H, step, on, h, p.eps, xa, xb, g >= p.Hq);
}

// Any even head dim, any alignment: one warp per head vector, value by value, read twice (the
// second time from L1).  bf16, 64 rows of 40 heads of 128 off 16 bytes 3.4 us on the device (as
// the vector kernel on aligned ones), 8 x 4096 rows 530 us (120 aligned); heads of 72: 3 x 1037 rows
// of 12 heads 17 us, 8 x 4096 of 40 heads 539 (58 us of bytes).
template <typename T>
__global__ void __launch_bounds__(ANY_WARPS * 32) any_kernel(const Params p) {
  const int lane = threadIdx.x & 31, h = p.D / 2, n = p.Hq + p.H;
  const int64_t wid = (int64_t)blockIdx.x * ANY_WARPS + (threadIdx.x >> 5);
  const int64_t row = wid / n;
  if (row >= p.rows) return;
  const int64_t b = row / p.T, t = row - b * p.T;
  const int j = (int)(wid - row * n);
  const bool isq = j < p.Hq;
  const T* x = isq ? static_cast<const T*>(p.q) + b * p.qsb + t * p.qst + (int64_t)j * p.D
                   : static_cast<const T*>(p.k) + b * p.ksb + t * p.kst + (int64_t)(j - p.Hq) * p.D;
  T* o = isq ? static_cast<T*>(p.qo) + ((b * p.Hq + j) * p.T + t) * p.D
             : static_cast<T*>(p.ko) + b * p.kob + (j - p.Hq) * p.koh + t * p.D;
  const T* w = static_cast<const T*>(isq ? p.qw : p.kw);
  float ss = 0.f;
  for (int i = lane; i < p.D; i += 32) {
    const float v = to_f(x[i]);
    ss = fmaf(v, v, ss);
  }
  ss = warp_sum(ss);
  const float inv = rsqrtf(ss / (float)p.D + p.eps);
  const int64_t at = position(p, b, t) * p.D;
  const bool turn = isq || p.rotk;
  for (int i = lane; i < h; i += 32) {
    const float y1 = to_f(x[i]) * inv * to_f(w[i]), y2 = to_f(x[i + h]) * inv * to_f(w[i + h]);
    const float c = turn ? p.cosT[at + i] : 1.f, s = turn ? p.sinT[at + i] : 0.f;
    o[i] = from_f<T>(y1 * c - y2 * s);
    o[i + h] = from_f<T>(y2 * c + y1 * s);
  }
}

template <typename T>
int launch(const Params& p, bool vec, cudaStream_t st) {
  const int h = p.D / 2;
  int64_t warps;
  if (!vec) {
    warps = p.rows * (p.Hq + p.H);
    const int64_t grid = (warps + ANY_WARPS - 1) / ANY_WARPS;
    SPX_REQUIRE(grid <= 0x7fffffff, SPX_ERR_SHAPE, "spx_qk_norm_rope: too many rows");
    any_kernel<T><<<(unsigned)grid, ANY_WARPS * 32, 0, st>>>(p);
    return launch_status("qk_norm any_kernel");
  }
  constexpr int VP = 8, WARPS = kWarps<T>;
  // Lanes of a head: a power of two, or as many as it has vectors where a warp then holds more heads
  // and the rows fill the SMs (the sum takes a step more).  bf16, 12 heads of 80: 8 x 2048 rows 15.0
  // us with five lanes, 17.8 with eight; 3 x 1037 rows 6.5 and 6.0; of 160: 3 x 1037 rows 8.7 us
  // with ten, 10.3 with sixteen, 8 x 2048 32.6 and 34.4.
  int G = 1;
  const int vectors = (h + VP - 1) / VP;
  while (G < vectors) G *= 2;
  if (32 / vectors > 32 / G && (vectors > 8 || (vectors > 4 && p.rows * G > (int64_t)148 * 16 * 32))) G = vectors;
  Params q = p;
  // The heads of a row are spread over several groups of lanes.  Few rows: up to 16 warps an SM or
  // one head a group (3 x 1037 rows of 12 heads of 80: 8.8 us with one group a row, 5.9 with three,
  // 7.3 with four, 7.6 with six: each group looks up its position and table row); from four on a
  // power of two, so that a warp's groups are of one row (1024 rows of 40 heads of 128: 6.6 us with
  // eight, 6.8 with nine, 7.4 with ten).  Three where the SMs hold three but not four: over 80 shapes
  // of 1315 to 6110 rows, heads of 64 to 256, against two groups, bf16 rows of 12 heads 5.7 and 6.8
  // us, of 26 heads 9.2 and 10.2, of 20 and 40 heads level, of 8 heads 5.6 and 5.1 (float32: 12 heads
  // 7 to 11 % less, 26 heads up to 8 % less, 8 heads 1 to 7 % more).  Many rows: at most 14 heads a
  // group (8 x 1024 rows of 40 heads 41.2 us with one group a row, 33.6 with two, 32.5 with four, 33.8
  // with eight; of 12 heads 11.5 with one, 11.7 with two).
  const int ng = 32 / G, most = p.Hq + p.H;
  const int64_t fit = (int64_t)148 * 16 * ng / p.rows;
  int slots = 1;
  while (slots * 14 < most || (slots * 2 <= fit && slots * 2 <= most)) slots *= 2;
  if (fit == 3 && slots < 3) slots = 3;
  q.slots = fit >= most || slots > most ? most : slots;
  warps = (p.rows * q.slots + ng - 1) / ng;
  SPX_REQUIRE(warps * 32 <= 0x7fffffff, SPX_ERR_SHAPE, "spx_qk_norm_rope: too many rows");   // 32-bit indexes
  const unsigned grid = (unsigned)((warps + WARPS - 1) / WARPS);
  switch (G) {
    case 1: vec_kernel<T, VP, 1><<<grid, WARPS * 32, 0, st>>>(q); break;
    case 2: vec_kernel<T, VP, 2><<<grid, WARPS * 32, 0, st>>>(q); break;
    case 4: vec_kernel<T, VP, 4><<<grid, WARPS * 32, 0, st>>>(q); break;
    case 5: vec_kernel<T, VP, 5><<<grid, WARPS * 32, 0, st>>>(q); break;
    case 6: vec_kernel<T, VP, 6><<<grid, WARPS * 32, 0, st>>>(q); break;
    case 8: vec_kernel<T, VP, 8><<<grid, WARPS * 32, 0, st>>>(q); break;
    case 9: vec_kernel<T, VP, 9><<<grid, WARPS * 32, 0, st>>>(q); break;
    case 10: vec_kernel<T, VP, 10><<<grid, WARPS * 32, 0, st>>>(q); break;
    case 16: vec_kernel<T, VP, 16><<<grid, WARPS * 32, 0, st>>>(q); break;
    default: vec_kernel<T, VP, 32><<<grid, WARPS * 32, 0, st>>>(q); break;
  }
  return launch_status("qk_norm vec_kernel");
}

}  // namespace qkn
}  // namespace spx

using namespace spx;

int spx_qk_norm_rope(const spx_qk_norm_args* a, void* stream) {
  SPX_REQUIRE(a, SPX_ERR_NULL, "spx_qk_norm_rope: args are required");
  SPX_REQUIRE(dtype_ok(a->dtype), SPX_ERR_UNSUPPORTED, "spx_qk_norm_rope: bad dtype %d", a->dtype);
  SPX_REQUIRE(a->batch >= 0 && a->tokens >= 0 && a->num_q_heads >= 1 && a->num_q_heads <= 65535 &&
                  a->num_kv_heads >= 0 && a->num_kv_heads <= 65535 && a->head_dim >= 2 && a->head_dim % 2 == 0 &&
                  a->head_dim <= 1024 && a->rope_len >= 1 && a->eps >= 0.f,
              SPX_ERR_SHAPE, "spx_qk_norm_rope: bad shape batch %d tokens %d heads %d/%d head_dim %d rope_len %d",
              a->batch, a->tokens, a->num_q_heads, a->num_kv_heads, a->head_dim, a->rope_len);
  const bool keys = a->num_kv_heads > 0;
  SPX_REQUIRE(a->q && a->q_weight && a->cos_table && a->sin_table && a->q_out, SPX_ERR_NULL,
              "spx_qk_norm_rope: q, q_weight, tables and q_out are required");
  SPX_REQUIRE(!keys || (a->k && a->k_weight && a->k_out), SPX_ERR_NULL,
              "spx_qk_norm_rope: k, k_weight and k_out are required with key heads");
  SPX_REQUIRE(a->q_stride_b >= 0 && a->q_stride_t >= 0 && a->k_stride_b >= 0 && a->k_stride_t >= 0 &&
                  a->k_out_stride_b >= 0 && a->k_out_stride_h >= 0,
              SPX_ERR_SHAPE, "spx_qk_norm_rope: negative stride");
  if (a->batch == 0 || a->tokens == 0) return SPX_OK;
  qkn::Params p{};
  p.q = a->q, p.k = a->k, p.qw = a->q_weight, p.kw = a->k_weight, p.qo = a->q_out, p.ko = a->k_out;
  p.cosT = a->cos_table, p.sinT = a->sin_table, p.pos = a->pos;
  p.qsb = a->q_stride_b, p.qst = a->q_stride_t, p.ksb = a->k_stride_b, p.kst = a->k_stride_t;
  p.psb = a->pos_stride_b, p.pst = a->pos_stride_t, p.pos0 = a->pos_start;
  p.kob = a->k_out_stride_b, p.koh = a->k_out_stride_h;
  p.rows = (int64_t)a->batch * a->tokens;
  p.T = a->tokens, p.Hq = a->num_q_heads, p.H = a->num_kv_heads, p.D = a->head_dim, p.len = a->rope_len;
  p.rotk = a->rotate_keys, p.eps = a->eps;
  // 16-byte loads: both halves of a head start on 16 bytes and hold whole groups of eight
  const int per = 16 / dtype_size(a->dtype);
  const int64_t strides = a->q_stride_b | a->q_stride_t | (keys ? a->k_stride_b | a->k_stride_t | a->k_out_stride_b |
                                                                      a->k_out_stride_h : 0);
  const bool vec = a->head_dim % 16 == 0 && a->head_dim <= 512 && strides % per == 0 && aligned16(a->q) &&
                   aligned16(a->q_weight) && aligned16(a->q_out) && aligned16(a->cos_table) && aligned16(a->sin_table) &&
                   (!keys || (aligned16(a->k) && aligned16(a->k_weight) && aligned16(a->k_out)));
  return SPX_DISPATCH_DTYPE(a->dtype, T, [&] { return qkn::launch<T>(p, vec, reinterpret_cast<cudaStream_t>(stream)); });
}
