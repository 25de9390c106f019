// The tensor side of the entry points that a decode step calls for every layer
// (spx_qk_norm_rope, spx_lora_add, spx_logits_rules): checks of the tensors, outputs, the
// current stream and device, then the C call.  In Python, on ctypes, the same took 11 to 14 us
// a call, of which the GPU needs 3 to 6; here it takes 4 to 7.5.  No CUDA code: the kernels are
// libspx.so's, called through include/spx.h.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAEvent.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <map>
#include <numeric>
#include <optional>
#include <vector>

#include "spx.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return SPX_F32;
    case at::kHalf: return SPX_F16;
    case at::kBFloat16: return SPX_BF16;
    default: TORCH_CHECK_TYPE(false, "unsupported dtype ", t, "; expected float32, float16 or bfloat16");
  }
}

// A failed call: the package's exception for it (or for a device that the library is not for).
void raise_status(int rc, const char* what) {
  py::module_ n = py::module_::import("unsloth_spectral._native");
  n.attr("check")(n.attr("load")(), rc, what);
}
void require_device(const at::Device& d) {
  static bool ok[64] = {};
  if (d.is_cuda() && d.index() >= 0 && d.index() < 64 && ok[d.index()]) return;
  py::module_::import("unsloth_spectral._native").attr("lib_for")(py::cast(d));   // raises unless sm_100
  if (d.is_cuda() && d.index() >= 0 && d.index() < 64) ok[d.index()] = true;
}

template <typename F, typename A>
void launch(F fn, const A& args, const at::Device& d, const char* what) {
  c10::cuda::CUDAGuard guard(d);   // a launch goes to the current device
  const int rc = fn(&args, at::cuda::getCurrentCUDAStream(d.index()).stream());
  if (rc != SPX_OK) raise_status(rc, what);
}

// A new tensor on the GPU, without the dispatcher (at::empty takes 0.4 us more).
Tensor fresh(at::IntArrayRef sizes, at::ScalarType t, const at::Device& d) {
  return at::detail::empty_cuda(sizes, t, d, std::nullopt);
}

// Rows of `width` values, `os` and `ys` apart: out may be y itself or lie beside it (also between
// y's rows), but a row of it must not fall on another place of y, which is still to be read.
void no_partial_overlap(const Tensor& out, int64_t os, const Tensor& y, int64_t ys, int64_t rows, int64_t width) {
  const int64_t size = y.element_size(), d = (static_cast<const char*>(out.const_data_ptr()) -
                                              static_cast<const char*>(y.const_data_ptr())) / size;
  if (d >= (rows - 1) * ys + width || -d >= (rows - 1) * os + width) return;
  bool fine = d == 0 && (rows == 1 || os == ys);
  if (!fine && rows > 1 && os == ys && os > 0) {
    const int64_t m = (d % os + os) % os;
    fine = m >= width && os - m >= width;
  }
  TORCH_CHECK(fine, "out overlaps the input without being the same rows");
}

// A contiguous float32 [len, D] table on the device.
Tensor table(const Tensor& t, const at::Device& d) {
  Tensor x = t.dim() == 3 && t.size(0) == 1 ? t[0] : t;
  TORCH_CHECK_VALUE(x.dim() == 2, "cos/sin must be [max_len, head_dim] tables, got shape ", t.sizes());
  if (x.scalar_type() == at::kFloat && x.device() == d && x.is_contiguous()) return x;
  return x.to(d, at::kFloat).contiguous();
}

std::pair<Tensor, OptTensor> qk_norm_rope(Tensor q, OptTensor k, Tensor qw, const OptTensor& kw_, const Tensor& cos_,
                                          const Tensor& sin_, const OptTensor& pos, int64_t start, double eps,
                                          bool rotate_keys) {
  const auto dt = q.scalar_type();
  spx_qk_norm_args a{};
  a.dtype = dtype_code(dt);
  TORCH_CHECK_VALUE(q.dim() == 3 && qw.dim() == 1, "q must be [B, T, H * D] and q_weight [D], got ", q.sizes(), " and ",
                    qw.sizes());
  const int64_t B = q.size(0), T = q.size(1), n = q.size(2), D = qw.size(0);
  TORCH_CHECK_VALUE(D > 0 && D % 2 == 0 && n > 0 && n % D == 0, n, " query columns are no whole heads of ", D,
                    " (an even number)");
  TORCH_CHECK_VALUE(eps >= 0, "eps must not be negative, got ", eps);
  const at::Device dev = q.device();
  bool fits = qw.scalar_type() == dt && qw.device() == dev;
  int64_t H = 0;
  Tensor kw;
  if (k) {
    TORCH_CHECK_VALUE(kw_, "k needs k_weight");
    kw = *kw_;
    TORCH_CHECK_VALUE(k->dim() == 3 && k->size(0) == B && k->size(1) == T && kw.sizes() == qw.sizes() && k->size(2) % D == 0,
                      "k ", k->sizes(), " / k_weight ", kw.sizes(), " do not fit q ", q.sizes(), " with heads of ", D);
    H = k->size(2) / D;
    fits = fits && k->scalar_type() == dt && kw.scalar_type() == dt && k->device() == dev && kw.device() == dev;
  }
  TORCH_CHECK_VALUE(fits, "q, k and their weights must share dtype and device: q has ", dt, " on ", dev);
  TORCH_CHECK_VALUE(B <= INT32_MAX && T <= INT32_MAX && n / D <= INT32_MAX && D <= INT32_MAX, "q ", q.sizes(), " is too large");
  require_device(dev);
  const Tensor cos = table(cos_, dev), sin = table(sin_, dev);
  TORCH_CHECK_VALUE(cos.sizes() == sin.sizes() && cos.size(1) == D && cos.size(0) > 0 && cos.size(0) <= INT32_MAX,
                    "cos/sin must be [len, ", D, "] tables, got ", cos.sizes(), " and ", sin.sizes());
  if (pos) {
    const int64_t d = pos->dim(), rows = d == 2 ? pos->size(0) : 1;
    TORCH_CHECK_VALUE((d == 1 || d == 2) && pos->size(-1) == T && (rows == 1 || rows == B) &&
                          pos->scalar_type() == at::kLong && pos->device() == dev,
                      "position_ids must be int64 [", T, "], [1, ", T, "] or [", B, ", ", T, "] on ", dev, ", got ",
                      pos->scalar_type(), " ", pos->sizes(), " on ", pos->device());
    a.pos = pos->const_data_ptr<int64_t>();
    a.pos_stride_b = rows > 1 ? pos->stride(0) : 0;
    a.pos_stride_t = pos->stride(-1);
  }
  a.pos_start = start;
  if (q.stride(2) != 1) q = q.contiguous();
  qw = qw.contiguous();
  Tensor qo = fresh({B, n / D, T, D}, dt, dev);
  OptTensor ko;
  a.batch = (int32_t)B, a.tokens = (int32_t)T, a.num_q_heads = (int32_t)(n / D), a.num_kv_heads = (int32_t)H;
  a.head_dim = (int32_t)D, a.rope_len = (int32_t)cos.size(0), a.rotate_keys = rotate_keys, a.eps = (float)eps;
  a.q = q.const_data_ptr(), a.q_weight = qw.const_data_ptr(), a.q_out = qo.mutable_data_ptr();
  a.q_stride_b = q.stride(0), a.q_stride_t = q.stride(1);
  a.cos_table = cos.const_data_ptr<float>(), a.sin_table = sin.const_data_ptr<float>();
  if (k) {
    if (k->stride(2) != 1) k = k->contiguous();
    kw = kw.contiguous();
    ko = fresh({B, H, T, D}, dt, dev);
    a.k = k->const_data_ptr(), a.k_weight = kw.const_data_ptr(), a.k_out = ko->mutable_data_ptr();
    a.k_stride_b = k->stride(0), a.k_stride_t = k->stride(1);
    a.k_out_stride_b = H * T * D, a.k_out_stride_h = T * D;
  }
  if (B && T) launch(spx_qk_norm_rope, a, dev, "spx_qk_norm_rope");
  return {qo, ko};
}

// ---------------------------------------------------------------------- adapters ----
constexpr int64_t kBlockTokens = 64;   // tokens of a sequence from which on its rows may be taken as blocks

bool capturing() {   // the current stream, into a graph
  return c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None;
}

// Rows grouped by slot, cut into tiles of one slot: int32 tiles [n][4], then the order of rows.
// Tiles of 16 rows of any sequences, or 32 where a slot has more, which reads the adapter's weights
// half as often; or blocks of up to 128 tokens of one sequence, which name their first row
// themselves (no order).
struct Grouping {
  int tile_rows = 16, tiles = 0;
  std::vector<int32_t> held;
};

Grouping group_rows(const std::vector<int32_t>& slots, int64_t tokens, bool blocks) {
  const int n = (int)slots.size(), T = (int)tokens;
  std::vector<int32_t> seqs(n);
  std::iota(seqs.begin(), seqs.end(), 0);
  std::stable_sort(seqs.begin(), seqs.end(), [&](int a, int b) { return slots[a] < slots[b]; });
  Grouping g;
  const auto put = [&](int slot, int first, int rows, int row0) {
    g.held.insert(g.held.end(), {slot, first, rows, row0});
    ++g.tiles;
  };
  if (blocks) {
    g.tile_rows = 128;
    for (int i = 0; i < n; ++i)
      for (int t = 0; t < T; t += 128) put(slots[seqs[i]], i * T + t, std::min(128, T - t), seqs[i] * T + t);
    return g;
  }
  std::vector<std::pair<int, int>> runs;   // sequences of one slot: from, to
  for (int i = 0; i < n; ++i) {
    if (!i || slots[seqs[i]] != slots[seqs[i - 1]]) runs.emplace_back(i, i);
    ++runs.back().second;
  }
  for (const auto& r : runs)
    if ((r.second - r.first) * (int64_t)T > 16) g.tile_rows = 32;
  for (const auto& r : runs)
    for (int at = r.first * T; at < r.second * T; at += g.tile_rows)
      put(slots[seqs[r.first]], at, std::min(g.tile_rows, r.second * T - at), 0);
  for (int i = 0; i < n; ++i)
    for (int t = 0; t < T; ++t) g.held.push_back(seqs[i] * T + t);
  return g;
}

// Which rows use which slot: the groupings of a LoraBatch, by tokens per sequence.
struct Batch {
  struct Plan {
    int tile_rows, tiles, rows;
    Tensor held;
    c10::Stream made;
    at::cuda::CUDAEvent copied;
    bool there = false;   // the copy to the device is known to be done

    // Before a launch.  The copy was queued without waiting for it (a new batch does not hold up
    // the host): work on the stream that it was queued on follows it anyway; other streams, and
    // graphs, whose replays follow nothing, wait for it here, once.  On another stream the memory is
    // also kept until that stream's work is done (callers cannot record it, they never see it).
    void use(const at::cuda::CUDAStream& now) {
      const bool other = now.unwrap() != made;
      if (other) held.record_stream(now);
      if (there) return;
      const bool wait = other || capturing();
      const c10::cuda::CUDAStreamCaptureModeGuard allowed(cudaStreamCaptureModeRelaxed);
      if (wait) copied.synchronize();
      there = wait || copied.query();
    }
  };
  std::vector<int32_t> slots;
  int64_t sequences, highest;
  at::Device device;
  std::map<std::pair<int64_t, bool>, Plan> plans;

  Batch(std::vector<int32_t> s, const at::Device& d) : slots(std::move(s)), sequences((int64_t)slots.size()), highest(-1), device(d) {
    for (const int32_t v : slots) highest = std::max<int64_t>(highest, v);
  }

  Plan& plan(int64_t tokens, bool blocks) {
    const auto found = plans.find({tokens, blocks});
    if (found != plans.end()) return found->second;
    TORCH_CHECK_VALUE(tokens >= 0 && tokens <= 1 << 30 && sequences * tokens <= 1 << 30, sequences, " x ", tokens, " rows in one call");
    require_device(device);
    const c10::cuda::CUDAGuard guard(device);
    const auto now = at::cuda::getCurrentCUDAStream(device.index());
    TORCH_CHECK(!capturing(), "call LoraBatch.prepare(", tokens, ") before capturing a graph that uses the batch");
    const Grouping g = group_rows(slots, tokens, blocks);
    const int64_t n = (int64_t)g.held.size();
    Plan p{g.tile_rows, g.tiles, (int)(sequences * tokens), fresh({n}, at::kInt, device), now.unwrap()};
    if (n) {
      const Tensor host = at::empty({n}, at::TensorOptions().dtype(at::kInt).pinned_memory(true));
      std::copy(g.held.begin(), g.held.end(), host.mutable_data_ptr<int32_t>());
      p.held.copy_(host, true);
    }
    p.copied.record(now);
    return plans.emplace(std::make_pair(tokens, blocks), std::move(p)).first->second;
  }
  void prepare(int64_t tokens) {
    for (const bool blocks : {false, true})
      if (!blocks || tokens >= kBlockTokens) {
        Plan& p = plan(tokens, blocks);
        if (p.there) continue;
        const c10::cuda::CUDAStreamCaptureModeGuard allowed(cudaStreamCaptureModeRelaxed);   // of an earlier, uncaptured copy
        p.copied.synchronize();
        p.there = true;
      }
  }
};

// The distance between the rows of t [.., n], which must be even (one row: any, so its length).
int64_t row_stride(const Tensor& t) {
  TORCH_CHECK_VALUE(t.stride(-1) == 1, "the last dimension must be contiguous, got strides ", t.strides());
  if (t.numel() == t.size(-1)) return t.size(-1);
  if (t.dim() == 2 || t.size(1) == 1) return t.stride(0);
  TORCH_CHECK_VALUE(t.size(0) == 1 || t.stride(0) == t.size(1) * t.stride(1), "rows must be evenly spaced, got strides ",
                    t.strides(), " of ", t.sizes());
  return t.stride(1);
}

struct Pool {
  spx_lora_args args{};
  Tensor a, b, ranks, scales;
  int64_t in, out;

  Pool(Tensor a_, Tensor b_, Tensor ranks_, Tensor scales_, const std::vector<int>& widths)
      : a(std::move(a_)), b(std::move(b_)), ranks(std::move(ranks_)), scales(std::move(scales_)) {
    in = a.size(3), out = b.size(1);
    args.in_features = (int32_t)in, args.parts = (int32_t)widths.size();
    for (size_t i = 0; i < widths.size(); ++i) args.part_width[i] = widths[i];
    args.max_rank = (int32_t)a.size(2), args.slots = (int32_t)a.size(0), args.dtype = dtype_code(a.scalar_type());
    args.a = a.const_data_ptr(), args.b = b.const_data_ptr();
    args.ranks = ranks.const_data_ptr<int32_t>(), args.scales = scales.const_data_ptr<float>();
  }

  Tensor add(const Tensor& y, const Tensor& x, Batch& batch, const OptTensor& out_) const {
    const int64_t d = x.dim();
    TORCH_CHECK_VALUE((d == 2 || d == 3) && y.dim() == d && x.size(-1) == in && y.size(-1) == out && x.size(0) == y.size(0) &&
                          (d == 2 || x.size(1) == y.size(1)) && x.size(0) == batch.sequences,
                      "x [B, T, ", in, "] and y [B, T, ", out, "] of ", batch.sequences, " sequences expected, got ",
                      x.sizes(), " and ", y.sizes());
    TORCH_CHECK_INDEX(batch.highest < args.slots, "the batch names slot ", batch.highest, ", the pool has ", args.slots);
    TORCH_CHECK_VALUE(!out_ || out_->sizes() == y.sizes(), "out ", out_ ? out_->sizes() : y.sizes(),
                      " must have the shape of y ", y.sizes());
    const auto fits = [&](const Tensor& t) { return t.scalar_type() == a.scalar_type() && t.device() == a.device(); };
    TORCH_CHECK_VALUE(fits(x) && fits(y) && (!out_ || fits(*out_)), "x, y and out must be ", a.scalar_type(), " on ",
                      a.device());
    TORCH_CHECK_VALUE(batch.device == a.device(), "the batch is on ", batch.device, ", the pool on ", a.device());
    const int64_t tokens = d == 3 ? x.size(1) : 1, rows = batch.sequences * tokens;
    TORCH_CHECK_VALUE(rows <= 1 << 30, rows, " rows in one call");
    spx_lora_args v = args;
    if (rows) {
      v.x_stride = row_stride(x), v.y_stride = row_stride(y);
      if (out_) no_partial_overlap(*out_, v.out_stride = row_stride(*out_), y, v.y_stride, rows, out);
    }
    require_device(a.device());
    if (rows == 0) return out_ ? *out_ : at::empty_like(y);
    // Prompts take the kernels for blocks of adjacent rows, whose start takes longer, whose time does
    // not grow with the rank, and whose blocks of 128 rows end with a sequence.  Over 110 calls (300
    // to 95000 rows, 24 to 3900 tokens a sequence, rank 16 to 64) this rule takes the faster side
    // but for 0.7 %; rank 64, 9982 rows of 322 tokens 112 us by rows, 55 by blocks; rank 16, 3267 rows
    // of 363 tokens 21.8 and 22.2; 5548 rows of 76 tokens 16.5 and 28.0.
    const double fill = (double)tokens / ((tokens + 127) / 128 * 128);
    const bool blocks = tokens >= kBlockTokens &&
                        fill * fill * fill * rows * ((double)in * args.parts + out) * args.max_rank >= 1.5e8;
    const c10::cuda::CUDAGuard guard(a.device());
    Batch::Plan& p = batch.plan(tokens, blocks);
    p.use(at::cuda::getCurrentCUDAStream(a.device().index()));
    Tensor o = out_ ? *out_ : fresh(y.sizes(), y.scalar_type(), a.device());
    if (!out_) v.out_stride = out;
    v.num_tiles = p.tiles, v.tile_rows = p.tile_rows, v.num_rows = p.rows;
    v.tiles = p.held.const_data_ptr<int32_t>(), v.order = v.tiles + 4 * (int64_t)p.tiles;
    // the inner products, a buffer of each call's own: two streams or two captured graphs never
    // share one (the caching allocator hands it out in stream order)
    v.workspace_bytes = ((size_t)p.rows * args.parts * args.max_rank + 4) * sizeof(float);
    const at::DataPtr ws = c10::cuda::CUDACachingAllocator::get()->allocate(v.workspace_bytes);
    v.workspace = static_cast<float*>(ws.get());
    v.x = x.const_data_ptr(), v.y = y.const_data_ptr(), v.out = o.mutable_data_ptr();
    launch(spx_lora_add, v, a.device(), "spx_lora_add");
    return o;
  }
};

// ------------------------------------------------------------------------ logits ----
struct Rules {
  spx_logits_args args{};
  std::vector<Tensor> held;
  at::Device device;

  Rules(int batch, int vocab, const OptTensor& rep, const OptTensor& freq, const OptTensor& pres, const Tensor& seen,
        const Tensor& touched, const Tensor& counts, const OptTensor& bias_bits, const OptTensor& bias_first,
        const OptTensor& bias_values)
      : device(counts.device()) {
    const auto ptr = [&](const OptTensor& t) -> void* {
      if (!t) return nullptr;
      held.push_back(*t);
      return t->data_ptr();
    };
    args.batch = batch, args.vocab = vocab;
    args.repetition = static_cast<const float*>(ptr(rep)), args.frequency = static_cast<const float*>(ptr(freq));
    args.presence = static_cast<const float*>(ptr(pres)), args.seen_bits = static_cast<uint32_t*>(ptr(seen));
    args.touched_bits = static_cast<uint32_t*>(ptr(touched)), args.counts = static_cast<int32_t*>(ptr(counts));
    args.bias_bits = static_cast<const uint32_t*>(ptr(bias_bits));
    args.bias_first = static_cast<const int32_t*>(ptr(bias_first));
    args.bias_values = static_cast<const float*>(ptr(bias_values));
  }

  void rows_of(const Tensor& t, const char* name, at::ScalarType dt) const {
    TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == args.batch && t.size(1) == args.vocab && t.device() == device &&
                          t.scalar_type() == dt && (t.stride(1) == 1 || args.vocab == 1),
                      name, " must be [", args.batch, ", ", args.vocab, "] ", dt, " rows on ", device, ", got ",
                      t.scalar_type(), " ", t.sizes(), " (strides ", t.strides(), ") on ", t.device());
  }

  Tensor run(const Tensor& logits, const OptTensor& allow, OptTensor out, bool record) const {
    return call(logits, allow, out, record, false);
  }

  Tensor call(const Tensor& logits, const OptTensor& allow, OptTensor& out, bool record, bool make_out) const {
    spx_logits_args v = args;
    v.dtype = dtype_code(logits.scalar_type());
    rows_of(logits, "logits", logits.scalar_type());
    if (out) rows_of(*out, "out", logits.scalar_type());
    if (allow) {
      const int64_t d = allow->dim(), words = (args.vocab + 31) / 32, rows = d == 2 ? allow->size(0) : 1;
      TORCH_CHECK_VALUE((d == 1 || d == 2) && (rows == 1 || rows == args.batch) && allow->size(-1) >= words &&
                            allow->stride(-1) == 1 && allow->scalar_type() == at::kInt && allow->device() == device,
                        "allow must be int32 [", args.batch, " or 1, ", words, "] on ", device, ", got ",
                        allow->scalar_type(), " ", allow->sizes(), " on ", allow->device());
      v.allow = reinterpret_cast<const uint32_t*>(allow->const_data_ptr<int32_t>());
      v.allow_stride = rows > 1 ? allow->stride(0) : 0;
    }
    if (out) no_partial_overlap(*out, out->stride(0), logits, logits.stride(0), args.batch, args.vocab);
    require_device(device);
    if (!out && make_out) out = fresh({args.batch, args.vocab}, logits.scalar_type(), device);
    Tensor token = fresh({args.batch}, at::kLong, device);
    v.record = record, v.logits = logits.const_data_ptr(), v.logits_stride = logits.stride(0);
    if (out) v.out = out->mutable_data_ptr(), v.out_stride = out->stride(0);
    v.token = token.mutable_data_ptr<int64_t>();
    launch(spx_logits_rules, v, device, "spx_logits_rules");
    return token;
  }

  std::pair<Tensor, Tensor> apply(const Tensor& logits, const OptTensor& allow, OptTensor out) const {
    Tensor token = call(logits, allow, out, false, true);
    return {*out, token};
  }
};

}  // namespace

PYBIND11_MODULE(_spx_front, m) {
  m.def("qk_norm_rope", &qk_norm_rope);
  py::class_<Batch>(m, "Batch")
      .def(py::init<std::vector<int32_t>, const at::Device&>())
      .def_readonly("highest", &Batch::highest)
      .def("prepare", &Batch::prepare);
  m.def("group_rows", [](const std::vector<int32_t>& slots, int64_t tokens, bool blocks) {
    const Grouping g = group_rows(slots, tokens, blocks);
    return std::make_tuple(g.tile_rows, g.tiles, g.held);
  });
  py::class_<Pool>(m, "Pool")
      .def(py::init<Tensor, Tensor, Tensor, Tensor, const std::vector<int>&>())
      .def("add", &Pool::add);
  py::class_<Rules>(m, "Rules")
      .def(py::init<int, int, const OptTensor&, const OptTensor&, const OptTensor&, const Tensor&, const Tensor&,
                    const Tensor&, const OptTensor&, const OptTensor&, const OptTensor&>())
      .def("run", &Rules::run)
      .def("apply", &Rules::apply);
}
