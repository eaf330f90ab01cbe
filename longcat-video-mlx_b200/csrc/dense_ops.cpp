// Python binding of the C ABI's dense side: q/k norm with rotary positions, attention over key intervals, and the
// 8-bit key/value cache.  Checks of tensors, allocation of outputs and scratch, and the call on the tensors' device
// and its current stream, and the autograd nodes, in C++: at a few tokens these calls are shorter than the same steps in
// Python (host time of norm and rope of 390 tokens 7 us, there 20; of a lookup 5, there 16; a tiny torch addition takes 4).
//
// The entries are looked up in the engine's library, which Python has loaded; errors of the C ABI come back as
// ValueError (arguments) or BSAError, with its message.
#include <dlfcn.h>
#include <algorithm>
#include <array>
#include <cmath>
#include <optional>
#include <string>
#include <torch/extension.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include "../../include/bsa_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
namespace py = pybind11;

struct Api {
#define ENTRY(name) decltype(&::name) name = nullptr
  ENTRY(bsa_last_error);
  ENTRY(bsa_norm_rope);
  ENTRY(bsa_norm_rope_backward_scratch_bytes);
  ENTRY(bsa_norm_rope_backward);
  ENTRY(bsa_attention_ranges);
  ENTRY(bsa_masked_attention_scratch_bytes);
  ENTRY(bsa_masked_attention);
  ENTRY(bsa_masked_attention_backward_scratch_bytes);
  ENTRY(bsa_masked_attention_backward);
  ENTRY(bsa_kv8_append);
  ENTRY(bsa_kv8_unpack);
  ENTRY(bsa_kv8_attention_scratch_bytes);
  ENTRY(bsa_kv8_attention);
#undef ENTRY
} api;

PyObject* cuda_error = nullptr;  // BSAError, kept for the life of the process

void load(const std::string& path, const py::object& error) {
  cuda_error = py::object(error).release().ptr();
  void* lib = dlopen(path.c_str(), RTLD_NOW);
  if (!lib) throw std::runtime_error("cannot load " + path + ": " + dlerror());
#define ENTRY(name)                                                                        \
  api.name = reinterpret_cast<decltype(api.name)>(dlsym(lib, #name));                       \
  if (!api.name) throw std::runtime_error(std::string("missing entry ") + #name)
  ENTRY(bsa_last_error);
  ENTRY(bsa_norm_rope);
  ENTRY(bsa_norm_rope_backward_scratch_bytes);
  ENTRY(bsa_norm_rope_backward);
  ENTRY(bsa_attention_ranges);
  ENTRY(bsa_masked_attention_scratch_bytes);
  ENTRY(bsa_masked_attention);
  ENTRY(bsa_masked_attention_backward_scratch_bytes);
  ENTRY(bsa_masked_attention_backward);
  ENTRY(bsa_kv8_append);
  ENTRY(bsa_kv8_unpack);
  ENTRY(bsa_kv8_attention_scratch_bytes);
  ENTRY(bsa_kv8_attention);
#undef ENTRY
}

[[noreturn]] void refuse(const std::string& what) { throw py::value_error(what); }

// A CUDA-side failure; becomes BSAError where it reaches Python (autograd's own threads, which hold
// no interpreter lock, turn what a backward pass throws into RuntimeError).
struct CudaFailure : std::runtime_error {
  using std::runtime_error::runtime_error;
};

void check(int rc, const char* what) {
  if (rc == BSA_OK) return;
  char buf[512] = {0};
  api.bsa_last_error(buf, sizeof(buf));
  const std::string msg = buf[0] ? buf : std::string(what) + " failed";
  if (rc == BSA_ERR_SHAPE || rc == BSA_ERR_DTYPE || rc == BSA_ERR_ALIGN || rc == BSA_ERR_ARG) refuse(msg);
  throw CudaFailure(std::string(what) + " failed (code " + std::to_string(rc) + "): " + msg);
}

// The C ABI's sizes are 32-bit.
void small(const Tensor& t) {
  for (const int64_t n : t.sizes())
    if (n > INT32_MAX) refuse("a size of " + std::to_string(n) + " does not fit 32 bits");
}

int dtype_code(at::ScalarType t) {
  if (t == at::kBFloat16) return BSA_DTYPE_BF16;
  if (t == at::kHalf) return BSA_DTYPE_F16;
  if (t == at::kFloat) return BSA_DTYPE_F32;
  refuse(std::string("unsupported dtype ") + c10::toString(t));
}

void on_cuda(const Tensor& t) {
  if (!t.is_cuda()) refuse("BSA engine inputs must be CUDA tensors (there is no CPU path)");
}
void same_place(const Tensor& a, const Tensor& t) {
  on_cuda(t);
  if (t.device() != a.device()) refuse("all tensors must be on one device");
}
void same_place(const Tensor& a, const OptTensor& t) {
  if (t) same_place(a, *t);
}

void* ptr(const Tensor& t) { return t.data_ptr(); }
void* ptr(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

std::string shape_text(at::IntArrayRef s) {
  std::string r = "[";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + "]";
}

bool readable(const Tensor& t) {
  const int64_t unit = 16 / t.element_size();
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) return false;
  if (t.stride(3) != 1 && t.size(3) > 1) return false;
  for (int i = 0; i < 3; ++i)
    if (t.size(i) > 1 && (t.stride(i) % unit || t.stride(i) <= 0)) return false;
  return true;
}

// A [B, H, S, D] tensor that the kernels read in place, else a contiguous copy.  In place: d contiguous, base and strides
// in multiples of 16 bytes, nothing broadcast; any order and gaps of batch, heads and tokens otherwise.
struct View {
  Tensor t;
  int64_t strides[3];
  explicit View(const Tensor& given) : t(readable(given) ? given : given.clone(at::MemoryFormat::Contiguous)) {
    for (int i = 0; i < 3; ++i) strides[i] = t.stride(i);
  }
  void* p() const { return t.data_ptr(); }
};

Tensor like(const Tensor& t) { return at::empty(t.sizes(), t.options()); }
Tensor bytes(const Tensor& t, int64_t n) { return at::empty({n}, t.options().dtype(at::kByte)); }

// ------------------------------------------------------------------------------- q/k norm + rotary positions
struct Rope {
  OptTensor tables;
  int dt, dh, dw, T, H, W, start;
  const float* p() const { return tables ? static_cast<const float*>(tables->data_ptr()) : nullptr; }
  void check(const Tensor& x) const {
    if (!tables) return;
    same_place(x, tables);
    if (tables->scalar_type() != at::kFloat || !tables->is_contiguous()) refuse("rope tables must be contiguous fp32");
    if (tables->numel() != int64_t(T) * dt + int64_t(H) * dh + int64_t(W) * dw)
      refuse("rope tables of " + std::to_string(tables->numel()) + " values do not match their grid and dims");
  }
};

void check_pair(const Tensor& q, const OptTensor& k) {
  on_cuda(q);
  dtype_code(q.scalar_type());
  if (q.dim() != 4) refuse("expected tensors of shape [B, H, S, D]");
  small(q);
  if (k) {
    same_place(q, *k);
    if (k->scalar_type() != q.scalar_type() || k->dim() != 4 || k->size(0) != q.size(0) || k->size(2) != q.size(2) ||
        k->size(3) != q.size(3))
      refuse("q and k must share dtype, batch, length and head_dim");
    small(*k);
  }
}

// Contiguous weights of one type: fp32 or the input's are read as they are, others as fp32.
int weights(const Tensor& q, OptTensor& wq, OptTensor& wk) {
  at::ScalarType kind = at::kFloat;
  bool one = true, any = false;
  for (OptTensor* w : {&wq, &wk})
    if (*w) {
      same_place(q, **w);
      if ((*w)->dim() != 1 || (*w)->size(0) != q.size(3)) refuse("norm weight must be [" + std::to_string(q.size(3)) + "]");
      const at::ScalarType t = (*w)->scalar_type();
      one = one && (t == at::kFloat || t == q.scalar_type()) && (!any || t == kind) && (*w)->is_contiguous();
      kind = t;
      any = true;
    }
  if (!one) {
    for (OptTensor* w : {&wq, &wk})
      if (*w) *w = (*w)->to(at::kFloat).contiguous();
    kind = at::kFloat;
  }
  return dtype_code(kind);
}

std::pair<Tensor, OptTensor> norm_rope_forward(const Tensor& q, const OptTensor& k, OptTensor wq, OptTensor wk, double eps,
                                               const Rope& rope) {
  const int wcode = weights(q, wq, wk);
  const c10::cuda::CUDAGuard guard(q.device());
  Tensor y0 = like(q);
  OptTensor y1;
  if (k) y1 = like(*k);
  // the sides that hold values: one or both, or none
  const bool has_q = q.numel() > 0, has_k = k && k->numel() > 0;
  if (has_q || has_k) {
    const Tensor& first = has_q ? q : *k;
    const bool both = has_q && has_k;
    const View x0(first);
    std::optional<View> x1;
    if (both) x1.emplace(*k);
    check(api.bsa_norm_rope(x0.p(), x0.strides, first.size(1), ptr(has_q ? wq : wk), ptr(has_q ? OptTensor(y0) : y1),
                            both ? x1->p() : nullptr, both ? x1->strides : nullptr, both ? k->size(1) : 0,
                            both ? ptr(wk) : nullptr, both ? ptr(y1) : nullptr, dtype_code(q.scalar_type()), wcode, q.size(0),
                            q.size(2), q.size(3), static_cast<float>(eps), rope.p(), rope.dt, rope.dh, rope.dw, rope.T, rope.H,
                            rope.W, rope.start, stream_of(q)),
          "bsa_norm_rope");
  }
  return {y0, y1};
}

// One or two sides that hold values (x, gradient, weight, whether its weight's gradient is wanted): [dx0, dw0, dx1, dw1]
std::array<Tensor, 4> norm_rope_backward(const Tensor& x0, const Tensor& g0, OptTensor w0, bool want0, const OptTensor& x1,
                                         const OptTensor& g1, OptTensor w1, bool want1, double eps, const Rope& rope) {
  const int wcode = weights(x0, w0, w1);
  const c10::cuda::CUDAGuard guard(x0.device());
  const int64_t D = x0.size(3);
  Tensor dx0 = like(x0);
  OptTensor dx1, dw0, dw1, scratch;
  if (x1) dx1 = like(*x1);
  auto grad = [&] { return at::empty({D}, x0.options().dtype(at::kFloat)); };
  if (want0) dw0 = grad();
  if (want1) dw1 = grad();
  if (want0 || want1) scratch = bytes(x0, api.bsa_norm_rope_backward_scratch_bytes(x0.size(1), x1 ? x1->size(1) : 0, D));
  const View a(x0), ga(g0);
  std::optional<View> b, gb;
  if (x1) {
    b.emplace(*x1);
    gb.emplace(*g1);
  }
  check(api.bsa_norm_rope_backward(
            a.p(), a.strides, ga.p(), ga.strides, x0.size(1), ptr(w0), ptr(dx0), static_cast<float*>(ptr(dw0)),
            b ? b->p() : nullptr, b ? b->strides : nullptr, gb ? gb->p() : nullptr, gb ? gb->strides : nullptr,
            x1 ? x1->size(1) : 0, ptr(w1), ptr(dx1), static_cast<float*>(ptr(dw1)), dtype_code(x0.scalar_type()), wcode,
            x0.size(0), x0.size(2), D, static_cast<float>(eps), rope.p(), rope.dt, rope.dh, rope.dw, rope.T, rope.H, rope.W,
            rope.start, ptr(scratch), stream_of(x0)),
        "bsa_norm_rope_backward");
  const Tensor none;
  return {dx0, dw0.value_or(none), dx1.value_or(none), dw1.value_or(none)};
}

// Refused: inputs with a tangent (forward-mode derivatives), which these operators would drop
void no_tangent(std::initializer_list<const OptTensor*> ts) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const OptTensor* t : ts)
    if (*t && (*t)->_fw_grad(/*level=*/0).defined()) refuse("no forward-mode derivatives: an input has a tangent");
}

// Whether a graph has to be recorded.  Refused in a capture: a leaf whose gradient node an eager graph still holds.  Its
// gradient is added up on that graph's stream, which the capture cannot reach; autograd then ends the process.
bool any_grad(std::initializer_list<const OptTensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  bool any = false;
  for (const OptTensor* t : ts) any = any || (*t && (*t)->requires_grad());
  if (!any || c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return any;
  for (const OptTensor* t : ts)
    if (*t && (*t)->requires_grad() && (*t)->is_leaf())
      if (const auto node = torch::autograd::impl::try_get_grad_accumulator(**t))
        if (const auto s = node->stream(); s && *s != c10::cuda::getCurrentCUDAStream(s->device_index()).unwrap())
          refuse("an eager graph of this leaf is alive on another stream: drop its outputs before the capture");
  return any;
}

// Called in a backward pass: autograd records it only for create_graph.
void first_order() {
  if (at::GradMode::is_enabled()) throw std::runtime_error("these gradients cannot be differentiated again (create_graph=True)");
}

OptTensor some(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

class NormRope : public torch::autograd::Function<NormRope> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k, const OptTensor& wq,
                               const OptTensor& wk, const OptTensor& tables, double eps, std::array<int, 7> r) {
    const Rope rope{tables, r[0], r[1], r[2], r[3], r[4], r[5], r[6]};
    const auto y = norm_rope_forward(q, k, wq, wk, eps, rope);
    const Tensor none;
    ctx->save_for_backward({q, k.value_or(none), wq.value_or(none), wk.value_or(none), tables.value_or(none)});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["rope"] = std::vector<int64_t>(r.begin(), r.end());
    ctx->set_materialize_grads(false);
    return y.second ? variable_list{y.first, *y.second} : variable_list{y.first};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order();
    const variable_list saved = ctx->get_saved_variables();
    const auto r = ctx->saved_data["rope"].toIntVector();
    const Rope rope{some(saved[4]),          static_cast<int>(r[0]), static_cast<int>(r[1]), static_cast<int>(r[2]),
                    static_cast<int>(r[3]), static_cast<int>(r[4]), static_cast<int>(r[5]), static_cast<int>(r[6])};
    // the edges count the tensors that were given: q, k, wq, wk, tables
    bool need[4];
    for (int i = 0, edge = 0; i < 4; ++i) need[i] = saved[i].defined() && ctx->needs_input_grad(edge++);
    int sides[2], n = 0;
    variable_list res(7);
    for (int i = 0; i < 2; ++i)
      if (saved[i].defined() && grads[i].defined() && (need[i] || need[2 + i])) {
        if (saved[i].numel()) {
          sides[n++] = i;
        } else {  // no tokens or no heads
          if (need[i]) res[i] = at::empty(saved[i].sizes(), saved[i].options());
          if (need[2 + i]) res[2 + i] = at::zeros(saved[2 + i].sizes(), saved[2 + i].options());
        }
      }
    if (n) {
      auto grad = [&](int i) { return grads[i].to(saved[i].scalar_type()); };
      const int a = sides[0], b = sides[n - 1];
      const auto got = norm_rope_backward(saved[a], grad(a), some(saved[2 + a]), need[2 + a], n > 1 ? some(saved[b]) : std::nullopt,
                                          n > 1 ? OptTensor(grad(b)) : std::nullopt,
                                          n > 1 ? some(saved[2 + b]) : std::nullopt, n > 1 && need[2 + b],
                                          ctx->saved_data["eps"].toDouble(), rope);
      for (int s = 0; s < n; ++s) {
        const int i = sides[s];
        if (need[i]) res[i] = got[2 * s];
        if (need[2 + i]) res[2 + i] = got[2 * s + 1].to(saved[2 + i].scalar_type());
      }
    }
    return res;
  }
};

py::object norm_rope(const Tensor& q, const OptTensor& k, const OptTensor& wq, const OptTensor& wk, double eps,
                     const OptTensor& tables, int dt, int dh, int dw, int T, int H, int W, int start) {
  check_pair(q, k);
  const Rope rope{tables, dt, dh, dw, T, H, W, start};
  rope.check(q);
  const OptTensor q0(q);
  no_tangent({&q0, &k, &wq, &wk});
  if (any_grad({&q0, &k, &wq, &wk})) {
    const variable_list y = NormRope::apply(q, k, wq, wk, tables, eps, std::array<int, 7>{dt, dh, dw, T, H, W, start});
    return k ? py::object(py::make_tuple(y[0], y[1])) : py::cast(y[0]);
  }
  const auto y = norm_rope_forward(q, k, wq, wk, eps, rope);
  return k ? py::object(py::make_tuple(y.first, *y.second)) : py::cast(y.first);
}

// ------------------------------------------------------------------------------------------- key intervals
const int32_t* i32(const Tensor& place, OptTensor& t, const char* name, int64_t n) {
  if (!t) return nullptr;
  same_place(place, *t);
  if (t->scalar_type() != at::kInt) refuse(std::string(name) + " must be int32");
  if (n >= 0 && t->numel() != n) refuse(std::string(name) + " must have " + std::to_string(n) + " values");
  t = t->contiguous();
  return static_cast<const int32_t*>(t->data_ptr());
}

// (buffer, batch entries, places of the table in the buffer): the intervals and, on 16 bytes, their tile table
py::tuple attention_ranges(const py::object& device, int64_t Sq, int64_t Sk, int64_t batch, OptTensor given, bool causal,
                           int64_t prefix, OptTensor prefixes, OptTensor q_offsets, OptTensor k_offsets,
                           OptTensor q_lengths, OptTensor k_lengths, int64_t k_add) {
  if (Sq < 0 || Sk < 0 || Sq > INT32_MAX || Sk > INT32_MAX) refuse("lengths must be >= 0 and fit 32 bits");
  if (prefix < 0) refuse("prefix must be >= 0");
  prefix = std::min<int64_t>(prefix, INT32_MAX);
  if (q_offsets.has_value() != k_offsets.has_value()) refuse("q_offsets and k_offsets come together");
  if (q_offsets && (q_lengths || k_lengths)) refuse("give documents or lengths, not both");
  int64_t n = -1;
  if (q_offsets) {
    if (q_offsets->dim() != 1 || k_offsets->dim() != 1 || q_offsets->numel() != k_offsets->numel() || q_offsets->numel() < 2)
      refuse("q_offsets and k_offsets must be [documents + 1]");
    n = q_offsets->numel() - 1;
  }
  for (const OptTensor* t : {&q_lengths, &k_lengths})
    if (*t) {
      if ((*t)->dim() != 1 || (n >= 0 && (*t)->numel() != n)) refuse("lengths must be [B]");
      batch = n = (*t)->numel();
    }
  if (prefixes && n < 0) batch = n = prefixes->numel();
  if (prefixes && prefixes->dim() != 1) refuse("prefix must be one number or one for each document or entry");
  c10::Device dev(c10::kCUDA, -1);
  for (const OptTensor* t : {&given, &prefixes, &q_offsets, &q_lengths, &k_lengths})
    if (*t) small(**t);
  for (const OptTensor* t : {&given, &prefixes, &q_offsets, &q_lengths, &k_lengths})
    if (*t && device.is_none()) {
      on_cuda(**t);
      dev = (*t)->device();
    }
  if (!device.is_none()) dev = py::cast<c10::Device>(device);
  if (!dev.is_cuda()) refuse("BSA engine inputs must be CUDA tensors (there is no CPU path)");
  if (!dev.has_index()) dev.set_index(c10::cuda::current_device());
  const c10::cuda::CUDAGuard guard(dev);
  const int64_t at0 = (batch * Sq * 2 + 3) & ~int64_t(3);
  const Tensor buf = at::empty({at0 + batch * ((Sq + 127) / 128) * 4}, at::TensorOptions().device(dev).dtype(at::kInt));
  const int32_t* g = i32(buf, given, "ranges", -1);
  if (g && reinterpret_cast<uintptr_t>(g) & 7) {
    given = given->clone();
    g = static_cast<const int32_t*>(given->data_ptr());
  }
  const int32_t* pre = i32(buf, prefixes, "prefix", n);
  const int32_t* qo = i32(buf, q_offsets, "q_offsets", -1);
  const int32_t* ko = i32(buf, k_offsets, "k_offsets", -1);
  const int32_t* ql = i32(buf, q_lengths, "q_lengths", -1);
  const int32_t* kl = i32(buf, k_lengths, "k_lengths", -1);
  if (batch * Sq) {
    int32_t* r = static_cast<int32_t*>(buf.data_ptr());
    check(api.bsa_attention_ranges(r, r + at0, batch, Sq, Sk, g, causal, prefix, pre, qo, ko, qo ? n : 0, ql, kl, k_add,
                                   stream_of(buf)),
          "bsa_attention_ranges");
  }
  return py::make_tuple(buf, batch, at0);
}

struct Mask {
  const int32_t *ranges = nullptr, *table = nullptr;
  int64_t batch = 1;
  Mask(const Tensor& q, const OptTensor& buf, int64_t batch_, int64_t at0) {
    if (!buf) return;
    same_place(q, *buf);
    if (batch_ != 1 && batch_ != q.size(0))
      refuse("the mask has " + std::to_string(batch_) + " batch entries, q has " + std::to_string(q.size(0)));
    ranges = static_cast<const int32_t*>(buf->data_ptr());
    table = ranges + at0;
    batch = batch_;
  }
};

// ------------------------------------------------------------------------------------------ dense attention
void check_qkv(const Tensor& q, const Tensor& k, const Tensor& v) {
  on_cuda(q);
  same_place(q, k);
  same_place(q, v);
  if (q.dim() != 4 || k.dim() != 4) refuse("q, k and v must be [B, H, S, D]");
  if (k.sizes() != v.sizes()) refuse("k and v must have the same shape");
  small(q);
  small(k);
  const at::ScalarType t = q.scalar_type();
  if (k.scalar_type() != t || v.scalar_type() != t) refuse("q, k, v must share one dtype");
  if (t != at::kBFloat16 && t != at::kHalf) refuse(std::string("unsupported dtype ") + c10::toString(t) + " (bf16 or fp16)");
  const int64_t D = q.size(3);
  if (q.size(0) != k.size(0) || k.size(3) != D) refuse("q and k must share batch and head_dim");
  if (D % 8 || D <= 0 || D > 128) refuse("head_dim D=" + std::to_string(D) + " must be a multiple of 8 and <= 128");
  if (k.size(1) == 0 || q.size(1) % k.size(1))
    refuse(std::to_string(q.size(1)) + " query heads are no multiple of " + std::to_string(k.size(1)) + " key heads");
}

void check_scale(double sm_scale, double softcap) {
  if (!(sm_scale > 0) || std::isinf(sm_scale)) refuse("sm_scale must be positive and finite");
  if (!(softcap >= 0) || std::isinf(softcap)) refuse("softcap must be finite and >= 0");
  if (softcap > 0 && static_cast<float>(softcap) == 0.f) refuse("softcap is out of fp32's range");
}

// Whether views share bytes.  A place of a view is its base and a sum of strides times indexes, so two views meet where
// sum step_i x_i = distance has a solution with lo_i <= x_i <= hi_i.  Steps are tried from the largest down; what the smaller
// ones can still reach leaves two or three x_i each for views of one layout.
enum class Meet { kNo, kYes, kUnknown };

class Steps {
 public:
  void add(int64_t step, int64_t lo, int64_t hi) {
    if (lo == hi) return;
    for (int i = 0; i < n_; ++i)
      if (axis_[i].step == step) {
        axis_[i].lo += lo;
        axis_[i].hi += hi;
        return;
      }
    axis_[n_++] = {step, lo, hi};
  }
  // whether there are `want` solutions
  Meet reach(int64_t distance, int want) {
    std::sort(axis_, axis_ + n_, [](const Axis& a, const Axis& b) { return a.step > b.step; });
    lo_[n_] = hi_[n_] = 0;
    for (int i = n_ - 1; i >= 0; --i) {
      lo_[i] = lo_[i + 1] + axis_[i].step * axis_[i].lo;
      hi_[i] = hi_[i + 1] + axis_[i].step * axis_[i].hi;
    }
    left_ = 1 << 16;
    missing_ = want;
    search(0, distance);
    return missing_ <= 0 ? Meet::kYes : left_ < 0 ? Meet::kUnknown : Meet::kNo;
  }

 private:
  struct Axis {
    int64_t step, lo, hi;
  };
  void search(int i, int64_t distance) {
    if (distance < lo_[i] || distance > hi_[i] || missing_ <= 0 || --left_ < 0) return;
    if (i == n_) {
      --missing_;
      return;
    }
    const Axis& a = axis_[i];
    auto floor_div = [](int64_t x, int64_t d) { return x >= 0 ? x / d : -((-x + d - 1) / d); };
    const int64_t first = std::max(a.lo, -floor_div(hi_[i + 1] - distance, a.step));
    const int64_t last = std::min(a.hi, floor_div(distance - lo_[i + 1], a.step));
    for (int64_t x = first; x <= last && missing_ > 0 && left_ >= 0; ++x) search(i + 1, distance - x * a.step);
  }
  Axis axis_[12];
  int n_ = 0, missing_ = 0, left_ = 0;
  int64_t lo_[13], hi_[13];
};

bool same_view(const Tensor& a, const Tensor& b) {
  return a.data_ptr() == b.data_ptr() && a.sizes() == b.sizes() && a.strides() == b.strides();
}

Meet meet(const Tensor& a, const Tensor& b) {
  if (!a.numel() || !b.numel()) return Meet::kNo;
  const int64_t size[2] = {a.element_size(), b.element_size()};
  const int64_t distance = static_cast<const char*>(b.data_ptr()) - static_cast<const char*>(a.data_ptr());
  Steps s;
  for (int i = 0; i < 4; ++i) {
    if (a.stride(i)) s.add(a.stride(i) * size[0], 0, a.size(i) - 1);
    if (b.stride(i)) s.add(b.stride(i) * size[1], 1 - b.size(i), 0);
  }
  s.add(1, 1 - size[1], size[0] - 1);
  return s.reach(distance, 1);
}

Meet meets_itself(const Tensor& t) {
  if (!t.numel()) return Meet::kNo;
  Steps s;
  for (int i = 0; i < 4; ++i) {
    if (t.size(i) > 1 && !t.stride(i)) return Meet::kYes;
    s.add(t.stride(i), 1 - t.size(i), t.size(i) - 1);
  }
  // axes of one step meet, and are one axis to the search below, which looks for a way to 0 beside zeros alone
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < i; ++j)
      if (t.size(i) > 1 && t.size(j) > 1 && t.stride(i) == t.stride(j)) return Meet::kYes;
  return s.reach(0, 2);
}

// The output may be q itself: a row of it is written by who has read that row of q.  It overlaps no input otherwise, nor
// itself.  True: views too entangled to tell, whose result is computed aside.
bool check_out(const Tensor& q, const OptTensor& out, std::initializer_list<const OptTensor*> others) {
  if (!out) return false;
  same_place(q, *out);
  if (out->sizes() != q.sizes() || out->scalar_type() != q.scalar_type()) refuse("out must have q's shape and dtype");
  if (at::GradMode::is_enabled() && out->requires_grad()) refuse("out= is for calls without gradients");
  Meet m = meets_itself(*out);
  if (m == Meet::kYes) refuse("out overlaps itself");
  bool aside = m == Meet::kUnknown;
  auto against = [&](const Tensor& t) {
    m = meet(*out, t);
    if (m == Meet::kYes) refuse("out overlaps an input");
    aside = aside || m == Meet::kUnknown;
  };
  if (!same_view(*out, q)) against(q);
  for (const OptTensor* t : others)
    if (*t) against(**t);
  return aside;
}

// The caller's output where the kernels can write it, else a new tensor that is copied there at the end.
struct Output {
  Tensor t;
  bool copy;
  int64_t strides[3];
  Output(const Tensor& q, const OptTensor& out, bool aside) : copy(out && (aside || !readable(*out))) {
    t = out && !copy ? *out : like(q);
    for (int i = 0; i < 3; ++i) strides[i] = t.stride(i);
  }
  Tensor done(const OptTensor& out) {
    if (copy)
      out->copy_(t);
    else if (out && !out->is_inference())
      out->unsafeGetTensorImpl()->bump_version();  // what autograd saved of it is stale, as after any in-place write
    return out ? *out : t;
  }
};

struct Attended {
  Tensor out;
  OptTensor lse, rest;
};

Attended attention_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Mask& m, double sm_scale, double softcap,
                           const OptTensor& out, bool aside, bool want_lse, bool want_rest) {
  const int64_t B = q.size(0), H = q.size(1), Sq = q.size(2), D = q.size(3), Hk = k.size(1), Sk = k.size(2);
  const c10::cuda::CUDAGuard guard(q.device());
  Output o(q, out, aside);
  OptTensor lse, rest;
  if (want_lse) lse = at::empty({B, H, Sq}, q.options().dtype(at::kFloat));
  if (want_rest) rest = like(q);
  if (q.numel() && Sk) {
    const View a(q), b(k), c(v);
    OptTensor scratch;
    const int64_t n = api.bsa_masked_attention_scratch_bytes(B, H, Sq, Sk, D);
    if (n) scratch = bytes(q, n);
    check(api.bsa_masked_attention(a.p(), b.p(), c.p(), dtype_code(q.scalar_type()), B, H, Hk, Sq, Sk, D, a.strides,
                                   b.strides, c.strides, m.ranges, m.table, m.batch, static_cast<float>(sm_scale),
                                   static_cast<float>(softcap), ptr(o.t), o.strides, ptr(rest),
                                   static_cast<float*>(ptr(lse)), ptr(scratch), stream_of(q)),
          "bsa_masked_attention");
  } else {  // no rows, or no keys: zeros
    o.t.zero_();
    if (rest) rest->zero_();
    if (lse) lse->fill_(-INFINITY);
  }
  return {o.done(out), lse, rest};
}

std::array<Tensor, 3> attention_backward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out,
                                         const Tensor& rest, const Tensor& lse, const Tensor& grad, const Mask& m,
                                         double sm_scale, double softcap, bool want_q, bool want_kv) {
  const int64_t B = q.size(0), H = q.size(1), Sq = q.size(2), D = q.size(3), Hk = k.size(1), Sk = k.size(2);
  const c10::cuda::CUDAGuard guard(q.device());
  const bool empty = !q.numel() || !Sk;
  auto grad_of = [&](const Tensor& t) { return empty ? at::zeros(t.sizes(), t.options()) : like(t); };
  Tensor dq, dk, dv;
  auto to = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
  if (want_q) dq = grad_of(q);
  if (want_kv) {
    dk = grad_of(k);
    dv = grad_of(v);
  }
  if (!empty) {
    const View a(q), b(k), c(v), o(out), g(grad);
    const Tensor scratch = bytes(q, api.bsa_masked_attention_backward_scratch_bytes(B, H, Sq, m.ranges ? m.batch : 0));
    check(api.bsa_masked_attention_backward(
              a.p(), b.p(), c.p(), o.p(), ptr(rest), g.p(), static_cast<const float*>(ptr(lse)),
              dtype_code(q.scalar_type()), B, H, Hk, Sq, Sk, D, a.strides, b.strides, c.strides, o.strides, g.strides,
              m.ranges, m.table, m.batch, static_cast<float>(sm_scale), static_cast<float>(softcap), to(dq), to(dk), to(dv),
              ptr(scratch), stream_of(q)),
          "bsa_masked_attention_backward");
  }
  return {dq, dk, dv};
}

class MaskedAttention : public torch::autograd::Function<MaskedAttention> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                               const OptTensor& mask, int64_t mask_batch, int64_t mask_table, double sm_scale,
                               double softcap) {
    const Attended a = attention_forward(q, k, v, Mask(q, mask, mask_batch, mask_table), sm_scale, softcap, std::nullopt,
                                         false, true, true);
    ctx->save_for_backward({q, k, v, a.out, *a.rest, *a.lse, mask.value_or(Tensor())});
    ctx->saved_data["mask"] = std::vector<int64_t>{mask_batch, mask_table};
    ctx->saved_data["scale"] = std::vector<double>{sm_scale, softcap};
    ctx->mark_non_differentiable({*a.lse});
    ctx->set_materialize_grads(false);
    return {a.out, *a.lse};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order();
    variable_list res(8);
    if (!grads[0].defined()) return res;
    const variable_list s = ctx->get_saved_variables();
    const auto at = ctx->saved_data["mask"].toIntVector();
    const auto scale = ctx->saved_data["scale"].toDoubleVector();
    const bool need[3] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2)};
    const auto d = attention_backward(s[0], s[1], s[2], s[3], s[4], s[5], grads[0].to(s[0].scalar_type()),
                                      Mask(s[0], some(s[6]), at[0], at[1]), scale[0], scale[1], need[0],
                                      need[1] || need[2]);
    for (int i = 0; i < 3; ++i)
      if (need[i]) res[i] = d[i];
    return res;
  }
};

// (out, lse or None)
py::tuple masked_attention(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& mask, int64_t mask_batch,
                           int64_t mask_table, int64_t mask_q, int64_t mask_k, double sm_scale, double softcap,
                           const OptTensor& out, bool want_lse) {
  check_qkv(q, k, v);
  check_scale(sm_scale, softcap);
  if (mask && (mask_q != q.size(2) || mask_k != k.size(2)))
    refuse("the mask is for " + std::to_string(mask_q) + " queries and " + std::to_string(mask_k) + " keys, got " +
           std::to_string(q.size(2)) + " and " + std::to_string(k.size(2)));
  const Mask m(q, mask, mask_batch, mask_table);
  const OptTensor q0(q), k0(k), v0(v);
  no_tangent({&q0, &k0, &v0, &out});
  const bool aside = check_out(q, out, {&k0, &v0});
  if (any_grad({&q0, &k0, &v0})) {
    if (out) refuse("out= is for calls without gradients");
    const variable_list r = MaskedAttention::apply(q, k, v, mask, mask_batch, mask_table, sm_scale, softcap);
    return py::make_tuple(r[0], r[1]);
  }
  const Attended a = attention_forward(q, k, v, m, sm_scale, softcap, out, aside, want_lse, false);
  return py::make_tuple(a.out, a.lse);
}

// ---------------------------------------------------------------------------------------------- 8-bit cache
struct Cache {
  Tensor kc, ks, vc, vs, len;
  int64_t B, Hk, cap, D;

  Cache(Tensor k_codes, Tensor k_scale, Tensor v_codes, Tensor v_scale, Tensor lengths)
      : kc(std::move(k_codes)), ks(std::move(k_scale)), vc(std::move(v_codes)), vs(std::move(v_scale)),
        len(std::move(lengths)) {
    on_cuda(kc);
    for (const Tensor* t : {&ks, &vc, &vs, &len}) same_place(kc, *t);
    if (kc.dim() != 4 || kc.sizes() != vc.sizes()) refuse("codes must be [B, Hk, capacity, D]");
    small(kc);
    B = kc.size(0), Hk = kc.size(1), cap = kc.size(2), D = kc.size(3);
    if (Hk == 0) refuse("a cache needs key heads");
    if (cap % 64 || cap == 0) refuse("capacity " + std::to_string(cap) + " must be a positive multiple of 64");
    if (D % 8 || D <= 0 || D > 128) refuse("head_dim D=" + std::to_string(D) + " must be a multiple of 8 and <= 128");
    for (const Tensor* t : {&kc, &vc})
      if (t->scalar_type() != at::kFloat8_e4m3fn || !t->is_contiguous() || reinterpret_cast<uintptr_t>(t->data_ptr()) & 15)
        refuse("codes must be contiguous, 16-byte aligned float8_e4m3fn");
    for (const Tensor* t : {&ks, &vs})
      if (t->scalar_type() != at::kFloat || !t->is_contiguous() || t->dim() != 3 || t->size(0) != B || t->size(1) != Hk ||
          t->size(2) != cap / 64)
        refuse("scales must be contiguous fp32 " + shape_text({B, Hk, cap / 64}));
    if (len.scalar_type() != at::kInt || !len.is_contiguous() || len.dim() != 1 || len.size(0) != B)
      refuse("lengths must be contiguous int32 " + shape_text({B}));
  }

  float* scale(const Tensor& t) const { return static_cast<float*>(t.data_ptr()); }
  int32_t* lengths() const { return static_cast<int32_t*>(len.data_ptr()); }

  void check_kv(const Tensor& k, const Tensor& v) const {
    same_place(kc, k);
    same_place(kc, v);
    if (k.dim() != 4 || k.sizes() != v.sizes() || k.size(0) != B || k.size(1) != Hk || k.size(3) != D)
      refuse("k and v must be [" + std::to_string(B) + ", " + std::to_string(Hk) + ", n, " + std::to_string(D) + "]");
    const at::ScalarType t = k.scalar_type();
    if (t != v.scalar_type() || (t != at::kBFloat16 && t != at::kHalf)) refuse("k and v must both be bf16 or fp16");
  }

  void append(const Tensor& k, const Tensor& v, OptTensor counts) {
    check_kv(k, v);
    if (k.size(2) > cap) refuse(std::to_string(k.size(2)) + " tokens for a capacity of " + std::to_string(cap));
    const int32_t* n = i32(kc, counts, "counts", B);
    if (!k.numel()) return;
    const c10::cuda::CUDAGuard guard(kc.device());
    const View a(k), b(v);
    check(api.bsa_kv8_append(ptr(kc), scale(ks), ptr(vc), scale(vs), lengths(), B, Hk, cap, D, a.p(), b.p(),
                             dtype_code(k.scalar_type()), k.size(2), a.strides, b.strides, n, stream_of(kc)),
          "bsa_kv8_append");
  }

  // (k, v) in 16 bits: the held tokens, the fresh ones and, where asked for, zeros up to capacity + fresh
  std::pair<Tensor, Tensor> unpack(at::ScalarType dtype, const OptTensor& k, const OptTensor& v, bool zeros) {
    if (dtype != at::kBFloat16 && dtype != at::kHalf) refuse("dequantize to bf16 or fp16");
    const c10::cuda::CUDAGuard guard(kc.device());
    const int64_t n = k ? k->size(2) : 0;
    const auto opt = kc.options().dtype(dtype);
    Tensor ko = at::empty({B, Hk, cap + n, D}, opt), vo = at::empty({B, Hk, cap + n, D}, opt);
    std::optional<View> a, b;
    if (n) {
      a.emplace(*k);
      b.emplace(*v);
    }
    check(api.bsa_kv8_unpack(ptr(kc), scale(ks), ptr(vc), scale(vs), lengths(), B, Hk, cap, D, a ? a->p() : nullptr,
                             b ? b->p() : nullptr, dtype_code(dtype), n, a ? a->strides : nullptr,
                             b ? b->strides : nullptr, ptr(ko), ptr(vo), cap + n, zeros, stream_of(kc)),
          "bsa_kv8_unpack");
    return {ko, vo};
  }

  Tensor attend(const Tensor& q, const OptTensor& k, const OptTensor& v, bool causal, std::optional<double> sm_scale,
                const OptTensor& out, int64_t few_rows) {
    same_place(kc, q);
    if (q.dim() != 4 || q.size(0) != B || q.size(3) != D)
      refuse("q must be [" + std::to_string(B) + ", H, Sq, " + std::to_string(D) + "]");
    const int64_t H = q.size(1), Sq = q.size(2);
    if (H % Hk) refuse(std::to_string(H) + " query heads are no multiple of " + std::to_string(Hk) + " key heads");
    const at::ScalarType t = q.scalar_type();
    if (t != at::kBFloat16 && t != at::kHalf) refuse(std::string("unsupported dtype ") + c10::toString(t) + " (bf16 or fp16)");
    if (k.has_value() != v.has_value()) refuse("k and v come together");
    if (k) {
      check_kv(*k, *v);
      if (k->scalar_type() != t) refuse("q, k, v must share one dtype");
    }
    if (at::GradMode::is_enabled() && (q.requires_grad() || (k && (k->requires_grad() || v->requires_grad()))))
      refuse("attention over a cache has no gradient");
    const OptTensor q0(q);
    no_tangent({&q0, &k, &v, &out});
    const double s = sm_scale ? *sm_scale : 1.0 / std::sqrt(static_cast<double>(D));
    check_scale(s, 0.0);
    const bool aside = check_out(q, out, {&k, &v});
    const c10::cuda::CUDAGuard guard(kc.device());
    if (!q.numel()) return out ? *out : like(q);
    const int64_t n = k ? k->size(2) : 0;
    if (n == 0 && H / Hk * Sq <= few_rows && B * Hk * ((H / Hk * Sq + 15) / 16) <= 65535) {  // (a grid's height)
      Output o(q, out, aside);
      const View a(q);
      OptTensor scratch;
      const int64_t need = api.bsa_kv8_attention_scratch_bytes(B, H, Hk, Sq, cap, D);
      if (need) scratch = bytes(q, need);
      check(api.bsa_kv8_attention(a.p(), dtype_code(t), B, H, Sq, a.strides, ptr(kc), scale(ks), ptr(vc), scale(vs),
                                  lengths(), Hk, cap, D, causal, static_cast<float>(s), ptr(o.t), o.strides, ptr(scratch),
                                  stream_of(q)),
            "bsa_kv8_attention");
      return o.done(out);
    }
    // what lies behind the last token is masked, whatever it holds
    const auto kv = n ? unpack(t, k, v, false) : unpack(t, std::nullopt, std::nullopt, false);
    const py::tuple m = attention_ranges(py::cast(kc.device()), Sq, cap + n, B, std::nullopt, causal, 0, std::nullopt,
                                         std::nullopt, std::nullopt, std::nullopt, len, n);
    const OptTensor buf = py::cast<Tensor>(m[0]);
    return attention_forward(q, kv.first, kv.second, Mask(q, buf, B, py::cast<int64_t>(m[2])), s, 0.0, out, aside, false, false)
        .out;
  }
};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const CudaFailure& e) {
      PyErr_SetString(cuda_error, e.what());
    }
  });
  m.def("load", &load, "The engine's library, and the exception of its CUDA errors");
  m.def("norm_rope", &norm_rope);
  m.def("attention_ranges", &attention_ranges);
  m.def("masked_attention", &masked_attention);
  py::class_<Cache>(m, "Cache")
      .def(py::init<Tensor, Tensor, Tensor, Tensor, Tensor>())
      .def("append", &Cache::append)
      .def("unpack", [](Cache& c, at::ScalarType dtype) { return c.unpack(dtype, std::nullopt, std::nullopt, true); })
      .def("attend", &Cache::attend);
}
