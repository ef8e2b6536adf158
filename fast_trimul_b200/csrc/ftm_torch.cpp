// Host side of layer norm and attention for torch tensors: allocation, the C problem, the
// launch and autograd in C++. A call of these operators on small inputs takes the GPU some
// microseconds, and the same steps in Python (ctypes, autograd.Function) took 20 to 40 for a
// forward and 150 and more for a training step.
//
// Every entry point here returns None where a call is not plain -- another type, shape, device
// or layout than the kernels read in place, or an error to report -- and the Python function
// around it then checks, copies, runs elsewhere or raises, and may call again. The library's
// functions come as addresses from the ctypes binding, so there is one loaded library.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <array>
#include <atomic>
#include <cmath>

#include "../../include/fast_trimul_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Library {
  decltype(&ftm_layer_norm_fwd) ln_fwd = nullptr;
  decltype(&ftm_layer_norm_bwd) ln_bwd = nullptr;
  decltype(&ftm_layer_norm_bwd_workspace_bytes) ln_bytes = nullptr;
  decltype(&ftm_attention_fwd) at_fwd = nullptr;
  decltype(&ftm_attention_bwd) at_bwd = nullptr;
  decltype(&ftm_attention_workspace_bytes) at_bytes = nullptr;
  decltype(&ftm_attention_bwd_workspace_bytes) at_bwd_bytes = nullptr;
  decltype(&ftm_last_launch_count) launches = nullptr;
  decltype(&ftm_status_string) status = nullptr;
  decltype(&ftm_pad_rows) pad_rows = nullptr;
} lib;

// error words of each GPU: the device word and the pinned host word (see ops/attention.py)
constexpr int kMaxGpus = 64;
struct Words {
  int* dev = nullptr;
  volatile int* host = nullptr;
};
std::array<Words, kMaxGpus> words;

// Failures of each GPU that were cleared, and for each thread how many it knows of (plus one; 0: it
// has made no call yet, and missed none).
std::array<std::atomic<unsigned>, kMaxGpus> failures{};
thread_local std::array<unsigned, kMaxGpus> known{};

bool knows_all(int d) {
  const unsigned now = failures[d].load() + 1;
  if (!known[d]) known[d] = now;
  return known[d] == now;
}

std::atomic<long> n_calls{0}, n_launches{0};

void count(bool call) {
  n_launches += lib.launches();
  if (call) ++n_calls;
}

void check(int st, const char* what) {
  TORCH_CHECK(st == FTM_OK, what, ": ", lib.status(st), " (status ", st, ")");
}

int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return FTM_F32;
    case at::kHalf: return FTM_F16;
    case at::kBFloat16: return FTM_BF16;
    default: return -1;
  }
}
bool is16(const Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }

ftm_stream_t stream_of(const Tensor& t) {
  return reinterpret_cast<ftm_stream_t>(at::cuda::getCurrentCUDAStream(t.get_device()).stream());
}
void* ptr(const OptTensor& t) { return t.has_value() && t->defined() ? t->data_ptr() : nullptr; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
bool has(const OptTensor& t) { return t.has_value() && t->defined(); }

// ---------------------------------------------------------------------------- autograd
// The gradients of a backward. With create_graph they hang on a node that raises when it is
// differentiated in turn, `from` (what they were formed of) behind it: these operators have
// first derivatives only, and a second one must not come out as zero.
variable_list once(variable_list grads, const variable_list& from) {
  const size_t n = grads.size();
  for (Tensor& t : grads)
    if (t.defined()) t = t.detach().set_requires_grad(true);
  grads.insert(grads.end(), from.begin(), from.end());
  const auto stop = std::make_shared<torch::autograd::DelayedError>(
      "layer norm and attention of fast_trimul_b200 are differentiable once", static_cast<int64_t>(grads.size()));
  variable_list out = (*stop)(std::move(grads));
  out.resize(n);
  return out;
}

// A tensor without elements at `t`'s place in the graph: what a backward keeps of an input whose
// values it does not need, so that `once` can name it.
Tensor place_of(const OptTensor& t) {
  if (!t.has_value() || !t->defined() || !t->requires_grad()) return Tensor();
  Tensor place = at::empty({0}, t->options());
  torch::autograd::impl::set_gradient_edge(place, torch::autograd::impl::gradient_edge(*t));
  return place;
}

// Forward-mode derivatives are not formed. Below autograd a dual tensor's tangent would be lost, and
// a result without one is read as a derivative of zero.
void no_tangent(std::initializer_list<const Tensor*> inputs) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : inputs)
    TORCH_CHECK(!t || !t->defined() || !t->_fw_grad(0).defined(),
                "layer norm and attention of fast_trimul_b200 have no forward-mode derivatives on a GPU");
}

bool capturing() { return c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None; }

// A leaf whose gradients an eager graph that still lives collects on the default stream. A
// backward pass in a captured graph would wait on that stream, which cannot take part in a
// capture: such a backward is refused (`not_held`) while the error can still be raised.
bool held(std::initializer_list<const Tensor*> leaves) {
  if (!capturing()) return false;
  for (const Tensor* t : leaves) {
    if (!t || !t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    const auto stream = node ? node->stream() : std::nullopt;
    if (stream && stream->device_type() == at::kCUDA && !c10::cuda::CUDAStream(*stream).stream()) return true;
  }
  return false;
}
void not_held(bool held) {
  TORCH_CHECK(!held || !capturing(),
              "a backward pass cannot be captured while a graph made on the default stream holds the same leaves: "
              "drop its outputs first, or run it on another stream");
}
const Tensor* given(const OptTensor& t) { return has(t) ? &*t : nullptr; }

// -------------------------------------------------------------------------- layer norm
// rows of `width` contiguous elements one stride apart; false: some other layout
bool rows_of(const Tensor& t, int64_t& rows, int64_t& stride) {
  const int64_t d = t.dim(), width = t.size(d - 1);
  if (width > 1 && t.stride(d - 1) != 1) return false;
  rows = 1;
  stride = width;
  int64_t next = -1;      // stride the next dimension outwards must have
  for (int64_t i = d - 2; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (next < 0) stride = t.stride(i);
    else if (t.stride(i) != next) return false;
    rows *= t.size(i);
    next = t.stride(i) * t.size(i);
  }
  return true;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor run(const Tensor& x, const Tensor& w, const Tensor& b, double eps, Tensor* stats) {
    int64_t rows, stride;
    rows_of(x, rows, stride);
    const c10::cuda::OptionalCUDAGuard guard(x.device());
    Tensor out = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
    if (stats) *stats = at::empty({rows, 2}, x.options().dtype(at::kFloat));
    check(lib.ln_fwd(x.data_ptr(), dtype_of(x), stride, ptr(w), w.defined() ? dtype_of(w) : 0, ptr(b),
                     b.defined() ? dtype_of(b) : 0, static_cast<float>(eps), out.data_ptr(),
                     stats ? stats->data_ptr<float>() : nullptr, rows, static_cast<int>(x.size(-1)), stream_of(x)),
          "ftm_layer_norm_fwd");
    count(true);
    return out;
  }

  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w, const OptTensor& b, double eps) {
    Tensor stats;
    Tensor out = run(x, w.value_or(Tensor()), b.value_or(Tensor()), eps, &stats);
    ctx->save_for_backward({x, w.value_or(Tensor()), stats});
    ctx->saved_data["bias"] = has(b) ? static_cast<int64_t>(b->scalar_type()) : int64_t(-1);
    ctx->saved_data["held"] = held({&x, given(w), given(b)});
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    not_held(ctx->saved_data["held"].toBool());
    no_tangent({&grads[0]});
    variable_list res = gradients(ctx, grads);
    if (!at::GradMode::is_enabled()) return res;
    const auto saved = ctx->get_saved_variables();
    return once(std::move(res), {grads[0], saved[0], saved[1]});
  }

  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    const at::AutoDispatchBelowAutograd below;
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &stats = saved[2];
    const int64_t bias = ctx->saved_data["bias"].toInt();
    Tensor g = grads[0];
    if (!g.defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    if (g.scalar_type() != x.scalar_type()) g = g.to(x.scalar_type());
    int64_t rows, xs, gs;
    rows_of(x, rows, xs);
    if (!rows_of(g, rows, gs)) {
      g = g.contiguous();
      rows_of(g, rows, gs);
    }
    const c10::cuda::OptionalCUDAGuard guard(x.device());
    const int width = static_cast<int>(x.size(-1));
    const auto o = x.options().memory_format(at::MemoryFormat::Contiguous);
    Tensor dx, dw, db, ws;
    if (ctx->needs_input_grad(0)) dx = at::empty(x.sizes(), o);
    if (w.defined() && ctx->needs_input_grad(1)) dw = at::empty({width}, w.options());
    // absent tensors have no edge: the bias' is the second without a weight
    if (bias >= 0 && ctx->needs_input_grad(w.defined() ? 2 : 1)) db = at::empty({width}, o.dtype(static_cast<at::ScalarType>(bias)));
    if (!dx.defined() && !dw.defined() && !db.defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    size_t bytes = 0;
    if (dw.defined() || db.defined()) {
      bytes = lib.ln_bytes(rows, width);
      ws = at::empty({static_cast<int64_t>(bytes)}, o.dtype(at::kByte));
    }
    check(lib.ln_bwd(x.data_ptr(), dtype_of(x), xs, g.data_ptr(), gs, ptr(w), w.defined() ? dtype_of(w) : 0,
                     stats.data_ptr<float>(), ptr(dx), ptr(dw), ptr(db), db.defined() ? dtype_of(db) : 0, ptr(ws),
                     bytes, rows, width, stream_of(x)),
          "ftm_layer_norm_bwd");
    count(false);
    return {dx, dw, db, Tensor()};
  }
};

py::object layer_norm(const Tensor& x, const OptTensor& w, const OptTensor& b, double eps) {
  int64_t rows, stride;
  if (x.is_cuda()) no_tangent({&x, given(w), given(b)});
  if (!x.is_cuda() || x.dim() < 1 || x.numel() == 0 || dtype_of(x) < 0 || !(eps >= 0) || !rows_of(x, rows, stride) ||
      x.size(-1) > INT_MAX)
    return py::none();
  for (const auto* p : {&w, &b})
    if (has(*p) && (dtype_of(**p) < 0 || (*p)->device() != x.device() || (*p)->dim() != 1 ||
                    (*p)->size(0) != x.size(-1) || !(*p)->is_contiguous()))
      return py::none();
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || (has(w) && w->requires_grad()) || (has(b) && b->requires_grad())))
    return py::cast(LayerNorm::apply(x, w, b, eps));
  const at::AutoDispatchBelowAutograd below;
  return py::cast(LayerNorm::run(x, w.value_or(Tensor()), b.value_or(Tensor()), eps, nullptr));
}

// --------------------------------------------------------------------------- attention
// What a call is beside its tensors.
struct Call {
  int seqs = 0, q_len = 0, kv_len = 0, bias_seqs = 0;
  bool causal = false, held = false;
  double scale = 0;
  Tensor cu_q, cu_k, lengths, mask, ready_bias;
};

// read in place by the kernels: dense last dimension, the others whole 16-byte vectors apart
bool ready(const Tensor& t) {
  const int64_t d = t.dim();
  if (t.stride(d - 1) != 1 || (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15)) return false;
  for (int64_t i = 0; i < d - 1; ++i)
    if (t.size(i) > 1 && (t.stride(i) <= 0 || t.stride(i) % 8)) return false;
  return true;
}
Tensor made_ready(const Tensor& t) {
  if (ready(t)) return t;
  return t.is_contiguous() ? t.clone() : t.contiguous();
}

ftm_attention problem(const Call& c, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& bias,
                      const Tensor& out, const Tensor& stats, const Tensor& low) {
  const bool batched = k.dim() == 4;
  const int64_t kr = k.dim() - 3;
  ftm_attention p{};
  p.dtype = dtype_of(q);
  p.heads = static_cast<int>(q.size(1));
  p.kv_heads = static_cast<int>(k.size(kr + 1));
  p.head_dim = static_cast<int>(q.size(2));
  p.causal = c.causal;
  p.scale = static_cast<float>(c.scale);
  p.sequences = c.seqs;
  p.q_len = c.q_len;
  p.kv_len = c.kv_len;
  p.q_rows = q.size(0);
  p.kv_rows = k.size(kr);
  p.cu_q = static_cast<const int32_t*>(ptr(c.cu_q));
  p.cu_k = static_cast<const int32_t*>(ptr(c.cu_k));
  p.kv_lengths = static_cast<const int32_t*>(ptr(c.lengths));
  p.q = q.data_ptr();
  p.q_row_stride = q.stride(0);
  p.q_head_stride = q.stride(1);
  p.k = k.data_ptr();
  p.k_row_stride = k.stride(kr);
  p.k_head_stride = k.stride(kr + 1);
  p.k_batch_stride = batched ? k.stride(0) : 0;
  p.v = v.data_ptr();
  p.v_row_stride = v.stride(kr);
  p.v_head_stride = v.stride(kr + 1);
  p.v_batch_stride = batched ? v.stride(0) : 0;
  p.key_mask = static_cast<const uint8_t*>(ptr(c.mask));
  p.bias = ptr(bias);
  p.bias_seqs = c.bias_seqs;
  if (bias.defined()) {
    p.bias_row_stride = bias.stride(2);
    p.bias_head_stride = bias.stride(1);
    p.bias_batch_stride = bias.stride(0);
  }
  p.out = out.data_ptr();
  p.stats = stats.defined() ? stats.data_ptr<float>() : nullptr;
  p.out_low = ptr(low);
  return p;
}

Tensor bytes_on(const Tensor& like, size_t n) {
  return n ? at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte)) : Tensor();
}

// what a backward needs of the forward beside its output
struct Kept {
  Tensor stats, low, lists;
};

Tensor attend(const Call& c, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& bias, Kept* kept) {
  const c10::cuda::OptionalCUDAGuard guard(q.device());
  const int train = kept != nullptr;
  Kept none;
  Kept& t = train ? *kept : none;
  Tensor out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  if (train) {
    t.stats = at::empty({q.size(0), q.size(1), 2}, q.options().dtype(at::kFloat));
    t.low = at::empty_like(out);
  }
  const ftm_attention p = problem(c, q, k, v, bias, out, t.stats, t.low);
  const size_t n = lib.at_bytes(&p, train);
  t.lists = bytes_on(q, n);
  const Words& w = words[q.get_device()];
  check(lib.at_fwd(&p, train, ptr(t.lists), n, w.dev, const_cast<int*>(w.host), stream_of(q)), "ftm_attention_fwd");
  count(true);
  return out;
}

struct Attention : torch::autograd::Function<Attention> {
  // `ready_bias` (what the kernels read) rides in the call: only `bias` itself has a gradient
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& bias,
                        const Call& c) {
    Kept t;
    Tensor out = attend(c, q, k, v, c.ready_bias, &t);
    ctx->save_for_backward({q, k, v, c.ready_bias, out, t.stats, t.lists, c.cu_q, c.cu_k, c.mask, t.low,
                            place_of(bias)});
    ctx->saved_data["n"] = std::vector<int64_t>{c.seqs, c.q_len, c.kv_len, c.bias_seqs, c.causal};
    ctx->saved_data["scale"] = c.scale;
    ctx->saved_data["held"] = c.held;
    if (has(bias)) ctx->saved_data["bias"] = bias->sizes().vec();
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    not_held(ctx->saved_data["held"].toBool());
    no_tangent({&grads[0]});
    variable_list res = gradients(ctx, grads);
    if (!at::GradMode::is_enabled()) return res;
    const auto saved = ctx->get_saved_variables();
    variable_list from{grads[0], saved[0], saved[1], saved[2]};
    if (saved[11].defined()) from.push_back(saved[11]);
    return once(std::move(res), from);
  }

  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    const at::AutoDispatchBelowAutograd below;
    const auto s = ctx->get_saved_variables();
    const Tensor &q = s[0], &k = s[1], &v = s[2], &bias = s[3], &out = s[4], &stats = s[5], &lists = s[6];
    const auto n = ctx->saved_data["n"].toIntVector();
    Call c;
    c.seqs = static_cast<int>(n[0]);
    c.q_len = static_cast<int>(n[1]);
    c.kv_len = static_cast<int>(n[2]);
    c.bias_seqs = static_cast<int>(n[3]);
    c.causal = n[4] != 0;
    c.scale = ctx->saved_data["scale"].toDouble();
    c.cu_q = s[7];
    c.cu_k = s[8];
    c.mask = s[9];
    Tensor g = grads[0];
    variable_list res(5);
    if (!g.defined()) return res;
    if (g.scalar_type() != q.scalar_type()) g = g.to(q.scalar_type());
    g = made_ready(g);
    const c10::cuda::OptionalCUDAGuard guard(q.device());
    const auto fresh = [](const Tensor& t) {
      return at::empty(t.sizes(), t.options().memory_format(at::MemoryFormat::Contiguous));
    };
    const bool nk = ctx->needs_input_grad(1), nv = ctx->needs_input_grad(2);
    Tensor dq, dk, dv, db;
    if (ctx->needs_input_grad(0)) dq = fresh(q);
    if (nk || nv) {
      dk = fresh(k);
      dv = fresh(v);
    }
    if (bias.defined() && ctx->needs_input_grad(3))
      db = at::empty(ctx->saved_data["bias"].toIntVector(), q.options().memory_format(at::MemoryFormat::Contiguous));
    if (!dq.defined() && !dk.defined() && !db.defined()) return res;
    const ftm_attention p = problem(c, q, k, v, bias, out, stats, s[10]);
    const size_t bytes = lib.at_bwd_bytes(&p, db.defined());
    Tensor ws = bytes_on(q, bytes);
    const Words& w = words[q.get_device()];
    check(lib.at_bwd(&p, g.data_ptr(), g.stride(0), g.stride(1), ptr(lists), lists.defined() ? lists.numel() : 0,
                     ptr(ws), bytes, ptr(dq), ptr(dk), ptr(dv), ptr(db), w.dev, const_cast<int*>(w.host),
                     stream_of(q)),
          "ftm_attention_bwd");
    count(false);
    res[0] = dq;
    if (nk) res[1] = dk;
    if (nv) res[2] = dv;
    res[3] = db;
    return res;
  }
};

Tensor run(const Call& c, const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& bias) {
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() ||
                                     (has(bias) && bias->requires_grad())))
    return Attention::apply(q, k, v, bias, c);
  const at::AutoDispatchBelowAutograd below;
  return attend(c, q, k, v, c.ready_bias, nullptr);
}

// q, k, v of one 16-bit type on one GPU whose error words are known and clear, heads that
// share, a head dimension of the kernels, everything readable in place
bool plain(const Tensor& q, const Tensor& k, const Tensor& v, double scale, int64_t heads, int64_t kv_heads,
           int64_t dim) {
  if (!q.is_cuda() || !is16(q) || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() ||
      k.device() != q.device() || v.device() != q.device() || k.sizes() != v.sizes() || q.numel() == 0 ||
      k.numel() == 0 || !(scale >= 0) || !std::isfinite(scale))
    return false;
  const int d = q.get_device();
  if (d >= kMaxGpus || !words[d].dev || *words[d].host || !knows_all(d)) return false;
  return heads <= INT_MAX && heads % kv_heads == 0 && heads / kv_heads <= 128 && dim % 8 == 0 && dim <= 128 &&
         ready(q) && ready(k) && ready(v);
}
bool index_ok(const Tensor& t, const Tensor& q) {
  return t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous() && t.device() == q.device();
}
// an absent mask is fine; a present one is bool, contiguous and of `shape`
bool mask_ok(const OptTensor& m, const Tensor& q, at::IntArrayRef shape) {
  return !has(m) || (m->scalar_type() == at::kBool && m->is_contiguous() && m->device() == q.device() &&
                     m->sizes() == shape);
}

py::object packed(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_q, const Tensor& cu_k,
                  bool causal, std::optional<double> scale, const OptTensor& mask) {
  no_tangent({&q, &k, &v});
  if (q.dim() != 3 || k.dim() != 3 || v.dim() != 3 || q.size(2) != k.size(2)) return py::none();
  const double s = scale ? *scale : 1.0 / std::sqrt(static_cast<double>(q.size(2)));
  if (k.size(1) < 1 || !plain(q, k, v, s, q.size(1), k.size(1), q.size(2)) || !index_ok(cu_q, q) ||
      !index_ok(cu_k, q) || cu_q.size(0) != cu_k.size(0) || cu_q.size(0) < 2 || cu_q.size(0) > INT_MAX ||
      !mask_ok(mask, q, {k.size(0)}))
    return py::none();
  Call c;
  c.seqs = static_cast<int>(cu_q.size(0) - 1);
  c.causal = causal;
  c.scale = s;
  c.cu_q = cu_q;
  c.cu_k = cu_k;
  if (has(mask)) c.mask = *mask;
  c.held = held({&q, &k, &v});
  return py::cast(run(c, q, k, v, std::nullopt));
}

py::object cached(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lengths,
                  std::optional<double> scale) {
  no_tangent({&q, &k, &v});
  if (q.dim() != 3 || k.dim() != 4 || v.dim() != 4 || q.size(0) != k.size(0) || q.size(2) != k.size(3))
    return py::none();
  const double s = scale ? *scale : 1.0 / std::sqrt(static_cast<double>(q.size(2)));
  if (k.size(2) < 1 || !plain(q, k, v, s, q.size(1), k.size(2), q.size(2)) || !index_ok(lengths, q) ||
      lengths.size(0) != q.size(0) || q.size(0) > INT_MAX)
    return py::none();
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad())) return py::none();
  Call c;
  c.seqs = static_cast<int>(q.size(0));
  c.q_len = 1;
  c.scale = s;
  c.lengths = lengths;
  const at::AutoDispatchBelowAutograd below;
  return py::cast(attend(c, q, k, v, Tensor(), nullptr));
}

py::object pair(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& bias, const OptTensor& mask,
                std::optional<double> scale) {
  no_tangent({&q, &k, &v, given(bias)});
  if (q.dim() != 5 || k.sizes() != q.sizes() || v.sizes() != q.sizes()) return py::none();
  const int64_t B = q.size(0), R = q.size(1), N = q.size(2), H = q.size(3), D = q.size(4);
  const double s = scale ? *scale : 1.0 / std::sqrt(static_cast<double>(D));
  if (H < 1 || !plain(q, k, v, s, H, H, D) || !mask_ok(mask, q, {B, R, N})) return py::none();
  Tensor b;
  if (has(bias)) {
    b = *bias;
    if (b.dim() != 4 || (b.size(0) != B && b.size(0) != 1) || b.size(1) != H || b.size(2) != N || b.size(3) != N ||
        b.scalar_type() != q.scalar_type() || b.device() != q.device())
      return py::none();
  }
  // copies that the kernels need of the bias: rows of whole vectors
  Tensor rb;
  if (b.defined()) {
    const at::NoGradGuard no_grad;
    rb = b.detach();
    if (!ready(b)) {
      const int64_t wide = (N + 7) / 8 * 8;
      rb = at::empty({b.size(0), H, N, wide}, q.options().memory_format(at::MemoryFormat::Contiguous)).slice(3, 0, N);
      if (b.is_contiguous()) {
        const c10::cuda::OptionalCUDAGuard guard(q.device());
        check(lib.pad_rows(b.data_ptr(), N, rb.data_ptr(), wide, b.size(0) * H * N, static_cast<int>(N), stream_of(q)),
              "ftm_pad_rows");
        count(false);
      } else {
        rb.copy_(b.detach());
      }
    }
  }
  if (B * R * N > INT_MAX) return py::none();
  Call c;
  c.seqs = static_cast<int>(B * R);
  c.q_len = c.kv_len = static_cast<int>(N);
  c.scale = s;
  if (b.defined()) c.bias_seqs = static_cast<int>(B * R / b.size(0));
  if (has(mask)) c.mask = *mask;
  c.ready_bias = rb;
  c.held = held({&q, &k, &v, given(bias)});
  const auto rows = [&](const Tensor& t) { return t.reshape({B * R * N, H, D}); };
  Tensor qf = rows(q), kf = rows(k), vf = rows(v);
  if (!ready(qf) || !ready(kf) || !ready(vf)) return py::none();
  return py::cast(run(c, qf, kf, vf, has(bias) ? OptTensor(b) : OptTensor()).view({B, R, N, H, D}));
}

void bind_library(const std::vector<uintptr_t>& f) {
  TORCH_CHECK(f.size() == 10, "ten functions");
  int i = 0;
  const auto set = [&](auto& p) { p = reinterpret_cast<std::decay_t<decltype(p)>>(f[i++]); };
  set(lib.ln_fwd);
  set(lib.ln_bwd);
  set(lib.ln_bytes);
  set(lib.at_fwd);
  set(lib.at_bwd);
  set(lib.at_bytes);
  set(lib.at_bwd_bytes);
  set(lib.launches);
  set(lib.status);
  set(lib.pad_rows);
}

void known_gpu(int device) { TORCH_CHECK(device >= 0 && device < kMaxGpus, "device ", device); }

void count_failure(int device) {
  known_gpu(device);
  ++failures[device];
}

// whether a failure was cleared since this thread last asked (or called)
bool missed_failure(int device) {
  known_gpu(device);
  const bool missed = !knows_all(device);
  known[device] = failures[device].load() + 1;
  return missed;
}

void set_words(int device, uintptr_t dev, uintptr_t host) {
  known_gpu(device);
  words[device].dev = reinterpret_cast<int*>(dev);
  words[device].host = reinterpret_cast<volatile int*>(host);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind_library", &bind_library);
  m.def("set_words", &set_words);
  m.def("count_failure", &count_failure);
  m.def("missed_failure", &missed_failure);
  m.def("layer_norm", &layer_norm);
  m.def("packed", &packed);
  m.def("cached", &cached);
  m.def("pair", &pair);
  m.def("calls", [] { return n_calls.load(); });
  m.def("launches", [] { return n_launches.load(); });
}
