// Autograd of the token operators (ops.layer_norm, dropout, rotary, window_attention) in C++: the module indm_amd._token.
//
// On small tensors a training call of these is host time: a backward pass runs on autograd's own thread, where a Python function
// takes the interpreter's lock and starts with cold caches (layer norm forward and backward of 256 x 256: 108 us through Python
// functions, of which the kernels are 12).  Here a call is one crossing into C++: checks, allocations, the launch, and a backward node
// that never enters the interpreter.  The kernels stay behind the C ABI: bind() takes the addresses of the entry points from the one
// loaded library (indm_amd/hip.py), nothing is linked.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <c10/util/accumulate.h>
#include <c10/util/strides.h>
#include <atomic>
#include <map>
#include <mutex>
#include "indm_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

// ---------------------------------------------------------------------------------------------- the C ABI (include/indm_hip.h)
// the entry points' addresses, with the types that the header declares
#define ENTRIES(X)                                                                                                              \
  X(layernorm_fwd_f32) X(layernorm_fwd_bf16) X(layernorm_bwd_ws_floats) X(layernorm_bwd_f32) X(layernorm_bwd_bf16)             \
  X(dropout_f32) X(dropout_bf16) X(rotary_f32) X(rotary_bf16)                                                                  \
  X(wattn_fwd_f32) X(wattn_fwd_bf16) X(wattn_bwd_ws_floats) X(wattn_bwd_f32) X(wattn_bwd_bf16)
struct Abi {
#define X(name) decltype(&indm_##name) name;
  ENTRIES(X)
#undef X
} abi;

void bind(const std::map<std::string, uint64_t>& at) {
#define X(name) abi.name = reinterpret_cast<decltype(abi.name)>(at.at("indm_" #name));
  ENTRIES(X)
#undef X
}
// the float32 or the bfloat16 entry point; their tensors' pointers are the only arguments whose types differ
struct Elements {
  void* at;
  template <typename T>
  operator T*() const { return static_cast<T*>(at); }
};
template <typename F32, typename BF16, typename... A>
int either(int type, F32 f32, BF16 bf16, A... a) {
  return type == 0 ? f32(a...) : bf16(a...);
}
#define CALL(type, name, ...) either(type, abi.name##_f32, abi.name##_bf16, __VA_ARGS__)

// ---------------------------------------------------------------------------------------------- what all of them do
#define REFUSE(...) TORCH_CHECK(false, "indm_amd: ", __VA_ARGS__)

void ok(int status, const char* name) {
  const char* what = status == -1 ? "INDM_E_SHAPE" : status == -2 ? "INDM_E_DTYPE" : status == -3 ? "INDM_E_LAUNCH" : "INDM_E_ARG";
  TORCH_CHECK(status == 0, name, " failed: ", what);
}
bool given(const Maybe& t) { return t.has_value() && t->defined(); }
// The tensor with the values it stands for in memory: a view may be lazily negated (the imaginary part of a conjugate), and a tensor of
// zeros that autograd made may have no memory at all.  Differentiable.
Tensor whole(const Tensor& t) { return t.defined() && (t.is_neg() || t._is_zerotensor()) ? t.clone() : t; }
Tensor plain(const Maybe& t) { return given(t) ? whole(*t) : Tensor(); }
bool tracked(std::initializer_list<const Tensor*> ts) {
  if (!c10::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
// What these functions cannot carry through is refused, not dropped: the tangent of a forward-mode derivative (a dual tensor need not
// require grad; the gradient that a backward pass is given may have one), and the call itself under torch.jit.trace, which would record an
// allocation in its place.
void carries(const char* op, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t->defined() && t->_fw_grad(/*level=*/0).defined()) REFUSE(op, ": forward-mode derivatives are not computed");
  if (torch::jit::tracer::isTracing()) REFUSE(op, ": cannot be traced by torch.jit.trace");
}
// which entry point: 0 float32, 1 bfloat16
int type_of(const char* op, const Tensor& x) {
  if (x.scalar_type() == at::kFloat) return 0;
  if (x.scalar_type() != at::kBFloat16) REFUSE(op, ": expected float32 or bfloat16, got ", x.scalar_type());
  return 1;
}
void on_one_gpu(const char* op, std::initializer_list<const Tensor*> ts) {
  const Tensor& x = **ts.begin();
  for (const Tensor* t : ts) {
    if (!t->defined()) continue;
    TORCH_CHECK(t->is_cuda(), "indm_amd.hip: tensor is not on the GPU; the HIP path has no CPU fallback");
    if (t->device() != x.device()) REFUSE(op, ": tensors on ", x.device(), " and ", t->device());
  }
}
void* stream_of(const Tensor& x) { return c10::hip::getCurrentHIPStream(x.get_device()).stream(); }
// Every tensor that a kernel writes comes from here.  guard(bytes) pads them with bands of that many bytes of a pattern on both sides
// (a debugging mode, like POISON_WS: a store outside of a tensor that hits a free block would go unseen).  The padded tensors are kept until
// broken_guards() counts the bands that were written to and forgets them; each remembers its bands, whatever guard() says by then.
struct Guarded {
  Tensor raw;
  int64_t band;
};
struct Guards {
  std::atomic<int64_t> band{0};   // (calls on other threads read it while guard() sets it: once each)
  std::mutex lock;
  std::vector<Guarded> kept;
} guards;
constexpr uint8_t GUARD = 0xA5;
Tensor fresh(at::IntArrayRef sizes, const at::TensorOptions& opt) {
  const int64_t band = guards.band.load(std::memory_order_relaxed);
  if (band == 0) return at::empty(sizes, opt);
  const int64_t n = c10::multiply_integers(sizes), e = (int64_t)opt.dtype().itemsize();
  Tensor raw = at::empty({n * e + 2 * band}, opt.dtype(at::kByte));
  raw.fill_(GUARD);
  Tensor t = at::empty({0}, opt).set_(raw.storage(), band / e, sizes, c10::contiguous_strides(sizes));
  const std::lock_guard<std::mutex> hold(guards.lock);
  guards.kept.push_back({raw, band});
  return t;
}
void guard(int64_t bytes) {
  if (bytes < 0) REFUSE("guard: bands of 0 bytes or more, got ", bytes);
  guards.band = (bytes + 255) / 256 * 256;
}
int64_t broken_guards() {
  std::vector<Guarded> kept;
  {
    const std::lock_guard<std::mutex> hold(guards.lock);
    kept.swap(guards.kept);
  }
  int64_t broken = 0;
  for (const Guarded& g : kept)
    for (const int64_t at : {(int64_t)0, g.raw.size(0) - g.band}) broken += g.raw.narrow(0, at, g.band).ne(GUARD).any().item<bool>();
  return broken;
}
Tensor dense_like(const Tensor& x) { return fresh(x.sizes(), x.options()); }
Tensor floats(int64_t n, const Tensor& x) { return fresh({n}, x.options().dtype(at::kFloat)); }
template <typename P = float>
P* ptr(const Tensor& t) {
  return t.defined() ? static_cast<P*>(t.data_ptr()) : nullptr;
}
Elements elements(const Tensor& t) { return {ptr<void>(t)}; }
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }

// A backward pass that is itself recorded (create_graph): its results refuse to be differentiated again
variable_list once(variable_list grads) {
  if (!c10::GradMode::is_enabled()) return grads;
  variable_list leaves;
  for (const Tensor& g : grads)
    if (g.defined()) leaves.push_back(g.detach().set_requires_grad(true));
  auto refuse = std::make_shared<torch::autograd::DelayedError>("indm_amd: the token operators are differentiable once", static_cast<int64_t>(leaves.size()));
  variable_list out = (*refuse)(std::move(leaves));
  size_t k = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = out[k++];
  return grads;
}

// ---------------------------------------------------------------------------------------------- layer norm
constexpr int64_t LN_MAX_C = 16384;

// x [..., C] as R rows with one stride and dense columns; a copy only where its strides allow no such view
struct Rows {
  Tensor x;
  long n, ld;
};
Rows rows_of(const Tensor& x) {
  const int64_t C = x.size(-1), R = x.numel() / C;
  if (x.is_contiguous()) return {x, R, C};
  if (R > 0 && (x.stride(-1) == 1 || C == 1)) {
    int64_t ld = -1, run = 1;   // the rows' stride, and how many of them the dimensions seen so far make
    bool one = true;
    for (int64_t d = x.dim() - 2; d >= 0; --d) {
      if (x.size(d) == 1) continue;
      if (ld < 0) ld = x.stride(d);
      one = one && x.stride(d) == ld * run;
      run *= x.size(d);
    }
    if (one) return {x, R, ld < 0 ? C : ld};
  }
  return {x.contiguous(), R, C};
}

void layer_norm_check(const Tensor& x, const Tensor& gamma, const Tensor& beta, double eps) {
  type_of("layer_norm", x);
  if (x.dim() < 1 || x.size(-1) < 1) REFUSE("layer_norm: x needs a last dimension that is not empty, got ", x.sizes());
  const int64_t C = x.size(-1);
  if (C > LN_MAX_C) REFUSE("layer_norm: rows of up to ", LN_MAX_C, " elements, got ", C);
  for (const Tensor* p : {&gamma, &beta}) {
    if (!p->defined()) continue;
    const char* name = p == &gamma ? "gamma" : "beta";
    if (p->scalar_type() != at::kFloat) REFUSE("layer_norm: ", name, " is float32, got ", p->scalar_type());
    if (p->dim() != 1 || p->size(0) != C) REFUSE("layer_norm: ", name, " is [", C, "], got ", p->sizes());
  }
  if (!(eps >= 0.)) REFUSE("layer_norm: eps >= 0, got ", eps);
  on_one_gpu("layer_norm", {&x, &gamma, &beta});
}
// -> y, and with stats [2 R]: the rows' means, then their 1 / standard deviations
std::pair<Tensor, Tensor> layer_norm_run(const Tensor& x, const Tensor& gamma_, const Tensor& beta_, double eps, bool stats) {
  const c10::DeviceGuard guard(x.device());
  const Tensor gamma = dense(gamma_), beta = dense(beta_);
  const Rows r = rows_of(x);
  Tensor y = dense_like(x), st = stats ? floats(2 * r.n, x) : Tensor();
  ok(CALL(type_of("layer_norm", x), layernorm_fwd, elements(r.x), r.ld, ptr(gamma), ptr(beta), elements(y), ptr(st), stats ? ptr(st) + r.n : nullptr, r.n,
          (int)x.size(-1), (float)eps, stream_of(x)),
     "indm_layernorm_fwd");
  return {y, st};
}
struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& gamma_, const Maybe& beta_, double eps) {
    const Tensor gamma = plain(gamma_), beta = plain(beta_);
    auto [y, stats] = layer_norm_run(x, gamma, beta, eps, true);
    ctx->save_for_backward({x, gamma, stats});
    ctx->saved_data["want"] = (int64_t)((x.requires_grad() ? 1 : 0) | (gamma.defined() && gamma.requires_grad() ? 2 : 0) | (beta.defined() && beta.requires_grad() ? 4 : 0));
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &stats = saved[2];
    carries("layer_norm", {&grads[0]});
    const int64_t want = ctx->saved_data["want"].toInt(), C = x.size(-1);
    const c10::DeviceGuard guard(x.device());
    const Tensor gamma = dense(saved[1]), dy = whole(grads[0]).contiguous();
    const Rows r = rows_of(x);
    Tensor dx = want & 1 ? dense_like(x) : Tensor(), dgamma = want & 2 ? floats(C, x) : Tensor(), dbeta = want & 4 ? floats(C, x) : Tensor(), ws;
    // (the scratch is an allocation of its own: calls on other streams and in other captured graphs share nothing)
    if (want & 6) ws = floats(std::max(1L, abi.layernorm_bwd_ws_floats(r.n, (int)C, (int)x.element_size())), x);
    ok(CALL(type_of("layer_norm", x), layernorm_bwd, elements(dy), elements(r.x), r.ld, ptr(gamma), ptr(stats), ptr(stats) + r.n, elements(dx), ptr(dgamma),
            ptr(dbeta), ptr(ws), r.n, (int)C, stream_of(x)),
       "indm_layernorm_bwd");
    return once({dx, dgamma, dbeta, Tensor()});
  }
};
Tensor layer_norm(const Tensor& x_, const Maybe& gamma_, const Maybe& beta_, double eps) {
  const Tensor x = whole(x_), gamma = plain(gamma_), beta = plain(beta_);
  carries("layer_norm", {&x, &gamma, &beta});
  layer_norm_check(x, gamma, beta, eps);
  return tracked({&x, &gamma, &beta}) ? LayerNorm::apply(x, Maybe(gamma), Maybe(beta), eps) : layer_norm_run(x, gamma, beta, eps, false).first;
}

// ---------------------------------------------------------------------------------------------- dropout
Tensor dropout_run(const Tensor& x_, double p, uint64_t seed, const Tensor& res_, const Tensor& seed_dev) {
  const c10::DeviceGuard guard(x_.device());
  const Tensor x = dense(x_), res = dense(res_);
  Tensor y = dense_like(x);
  ok(CALL(type_of("dropout", x), dropout, elements(x), elements(res), elements(y), x.numel(), (float)p, seed, ptr<void>(seed_dev), stream_of(x)),
     "indm_dropout");
  return y;
}
struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& res_, double p, int64_t seed, const Maybe& seed_dev_) {
    const Tensor res = plain(res_), seed_dev = plain(seed_dev_);
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["want"] = (int64_t)((x.requires_grad() ? 1 : 0) | (res.defined() && res.requires_grad() ? 2 : 0));
    if (seed_dev.defined()) ctx->saved_data["seed_dev"] = seed_dev;   // (not a saved variable: a graph's owner advances it in place)
    return dropout_run(x, p, (uint64_t)seed, res, seed_dev);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const int64_t want = ctx->saved_data["want"].toInt();
    const auto at = ctx->saved_data.find("seed_dev");
    Tensor dx;
    if (want & 1) carries("dropout", {&grads[0]});
    if (want & 1)
      dx = dropout_run(whole(grads[0]), ctx->saved_data["p"].toDouble(), (uint64_t)ctx->saved_data["seed"].toInt(), Tensor(),
                       at == ctx->saved_data.end() ? Tensor() : at->second.toTensor());
    variable_list out = once({dx});
    return {out[0], want & 2 ? grads[0] : Tensor(), Tensor(), Tensor(), Tensor()};
  }
};
Tensor dropout(const Tensor& x_, double p, uint64_t seed, const Maybe& res_, const Maybe& seed_dev_) {
  const Tensor x = whole(x_), res = plain(res_), seed_dev = plain(seed_dev_);
  carries("dropout", {&x, &res});
  type_of("dropout", x);
  if (!(p >= 0. && p <= 1.)) REFUSE("dropout: 0 <= p <= 1, got ", p);
  if (res.defined() && (res.sizes() != x.sizes() || res.scalar_type() != x.scalar_type()))
    REFUSE("dropout: res is ", x.sizes(), " ", x.scalar_type(), ", got ", res.sizes(), " ", res.scalar_type());
  if (seed_dev.defined() && (seed_dev.scalar_type() != at::kLong || seed_dev.numel() != 1)) REFUSE("dropout: seed_dev is one int64 on the device");
  on_one_gpu("dropout", {&x, &res, &seed_dev});
  return tracked({&x, &res}) ? Dropout::apply(x, Maybe(res), p, (int64_t)seed, Maybe(seed_dev)) : dropout_run(x, p, seed, res, seed_dev);
}

// ---------------------------------------------------------------------------------------------- rotary positions
void rotary_check(const Tensor& q, const Tensor& k, const Tensor& pos, const Tensor& freqs, const std::vector<int64_t>& sections) {
  type_of("rotary", q);
  if (q.dim() != 4) REFUSE("rotary: q is [B, T, H, D], got ", q.sizes());
  const int64_t B = q.size(0), T = q.size(1), D = q.size(3), A = (int64_t)sections.size();
  if (D > 4096) REFUSE("rotary: heads of up to 4096 entries, got ", D);
  if (k.defined() && (k.scalar_type() != q.scalar_type() || k.dim() != 4 || k.size(0) != B || k.size(1) != T || k.size(3) != D))
    REFUSE("rotary: k is [", B, ", ", T, ", Hk, ", D, "] ", q.scalar_type(), ", got ", k.sizes(), " ", k.scalar_type());
  for (const Tensor* x : {&q, &k})
    if (x->defined() && (B > INT32_MAX || x->size(2) > INT32_MAX)) REFUSE("rotary: up to 2^31 - 1 samples and heads, got ", x->sizes());
  int64_t sum = 0;
  bool even = A >= 1 && A <= 8;
  for (int64_t n : sections) {
    even = even && n >= 2 && n % 2 == 0 && n <= D - sum;
    sum += even ? n : 0;
  }
  if (!even) REFUSE("rotary: sections are 1 to 8 even positive numbers that sum to ", D, " at most, got ", sections);
  const auto type = pos.scalar_type();
  if (type != at::kInt && type != at::kLong && type != at::kFloat) REFUSE("rotary: positions are int32, int64 or float32, got ", type);
  const int64_t lead = pos.dim() - 2;
  if (lead < 0 || lead > 1 || pos.size(lead) != T || pos.size(lead + 1) != A || (lead == 1 && pos.size(0) != B))
    REFUSE("rotary: pos is [", T, ", ", A, "] or [", B, ", ", T, ", ", A, "], got ", pos.sizes());
  if (freqs.scalar_type() != at::kDouble || freqs.dim() != 1 || freqs.size(0) != sum / 2)
    REFUSE("rotary: freqs is float64 [", sum / 2, "], got ", freqs.sizes(), " ", freqs.scalar_type());
  if (c10::GradMode::is_enabled() && (pos.requires_grad() || freqs.requires_grad())) REFUSE("rotary: positions and frequencies have no gradient; detach them");
  on_one_gpu("rotary", {&q, &k, &pos, &freqs});
}
Tensor unit_columns(const Tensor& x) { return !x.defined() || x.stride(3) == 1 || x.size(3) == 1 ? x : x.contiguous(); }
// q or k may be undefined, not both -> the rotated ones (dense)
std::pair<Tensor, Tensor> rotary_run(const Tensor& q_, const Tensor& k_, const Tensor& pos_, const Tensor& freqs_, at::IntArrayRef sections, bool interleaved,
                                     bool inverse) {
  const Tensor& any = q_.defined() ? q_ : k_;
  const c10::DeviceGuard guard(any.device());
  const Tensor q = unit_columns(q_), k = unit_columns(k_), pos = pos_.contiguous(), freqs = freqs_.contiguous();
  Tensor yq = q.defined() ? dense_like(q) : Tensor(), yk = k.defined() ? dense_like(k) : Tensor();
  long strides[6] = {};
  for (int i = 0; i < 3; ++i) {
    if (q.defined()) strides[i] = q.stride(i);
    if (k.defined()) strides[3 + i] = k.stride(i);
  }
  int s[8];
  for (size_t i = 0; i < sections.size(); ++i) s[i] = (int)sections[i];
  const int64_t B = any.size(0), T = any.size(1), A = (int64_t)sections.size();
  const auto type = pos.scalar_type();
  ok(CALL(type_of("rotary", any), rotary, elements(q), elements(k), elements(yq), elements(yk), strides, (int)B, T, q.defined() ? (int)q.size(2) : 0,
          k.defined() ? (int)k.size(2) : 0, (int)any.size(3), pos.data_ptr(), type == at::kInt ? 0 : type == at::kFloat ? 1 : 2, pos.dim() == 3 ? T * A : 0,
          ptr<double>(freqs), s, (int)A, interleaved, inverse, stream_of(any)),
     "indm_rotary");
  return {yq, yk};
}
struct Rotary : torch::autograd::Function<Rotary> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Maybe& k_, const Tensor& pos, const Tensor& freqs, at::IntArrayRef sections,
                               bool interleaved) {
    const Tensor k = plain(k_);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({pos, freqs});
    ctx->saved_data["sections"] = sections.vec();
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["want"] = (int64_t)((q.requires_grad() ? 1 : 0) | (k.defined() && k.requires_grad() ? 2 : 0));
    auto [yq, yk] = rotary_run(q, k, pos, freqs, sections, interleaved, false);
    return k.defined() ? variable_list{yq, yk} : variable_list{yq};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const int64_t want = ctx->saved_data["want"].toInt();
    const Tensor dq = want & 1 ? whole(grads[0]) : Tensor(), dk = want & 2 && grads.size() > 1 ? whole(grads[1]) : Tensor();
    std::pair<Tensor, Tensor> g;
    carries("rotary", {&dq, &dk});
    if (dq.defined() || dk.defined())
      g = rotary_run(dq, dk, saved[0], saved[1], ctx->saved_data["sections"].toIntVector(), ctx->saved_data["interleaved"].toBool(), true);
    return once({g.first, g.second, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};
std::pair<Tensor, Maybe> rotary(const Tensor& q_, const Maybe& k_, const Tensor& pos_, const Tensor& freqs_, const std::vector<int64_t>& sections,
                                bool interleaved) {
  const Tensor q = whole(q_), k = plain(k_), pos = whole(pos_), freqs = whole(freqs_);
  carries("rotary", {&q, &k, &pos, &freqs});
  rotary_check(q, k, pos, freqs, sections);
  Tensor yq, yk;
  if (tracked({&q, &k})) {
    const variable_list y = Rotary::apply(q, Maybe(k), pos, freqs, at::IntArrayRef(sections), interleaved);
    yq = y[0];
    if (y.size() > 1) yk = y[1];
  } else {
    std::tie(yq, yk) = rotary_run(q, k, pos, freqs, sections, interleaved, false);
  }
  return {yq, yk.defined() ? Maybe(yk) : std::nullopt};
}

// ---------------------------------------------------------------------------------------------- window attention
struct Window {
  int64_t left, right, sinks;
  bool causal;
  double scale;
};
void window_check(const Tensor& q, const Tensor& k, const Tensor& v, const Window& w, const Tensor& lengths) {
  type_of("window_attention", q);
  if (q.dim() != 4) REFUSE("window_attention: q is [B, T, H, D], got ", q.sizes());
  const int64_t B = q.size(0), T = q.size(1), H = q.size(2), D = q.size(3);
  for (const Tensor* x : {&k, &v})
    if (x->scalar_type() != q.scalar_type() || x->dim() != 4 || x->size(0) != B || x->size(1) != T || x->size(3) != D || x->sizes() != k.sizes())
      REFUSE("window_attention: ", x == &k ? "k" : "v", " is [", B, ", ", T, ", Hk, ", D, "] ", q.scalar_type(), ", got ", x->sizes(), " ", x->scalar_type());
  const int64_t Hk = k.size(2);
  if (H < 1 || Hk < 1 || H % Hk) REFUSE("window_attention: the ", H, " heads of q are a multiple of the ", Hk, " of k and v");
  if (D % 8 || D < 8 || D > 128) REFUSE("window_attention: heads of 8, 16, ... 128 entries, got ", D);
  if (T > (1 << 28) || B > INT32_MAX || H * D > (1 << 22)) REFUSE("window_attention: up to ", 1 << 28, " tokens of ", 1 << 22, " entries, got ", T, " of ", H * D);
  if (w.left < 0 || w.right < 0 || w.sinks < 0) REFUSE("window_attention: window and sinks >= 0, got (", w.left, ", ", w.right, "), ", w.sinks);
  if (!((float)w.scale > 0.f && w.scale < 2e38)) REFUSE("window_attention: scale > 0 and below 2e38, got ", w.scale);
  if (lengths.defined() && (lengths.scalar_type() != at::kInt || lengths.dim() != 1 || lengths.size(0) != B))
    REFUSE("window_attention: lengths is int32 [", B, "], got ", lengths.sizes(), " ", lengths.scalar_type());
  on_one_gpu("window_attention", {&q, &k, &v, &lengths});
}
// x with dense columns, every row on 16 bytes and tokens at most 2^22 elements apart; a copy where it is not so
Tensor aligned_rows(const Tensor& x) {
  const int64_t e = 16 / x.element_size();
  if (x.stride(3) == 1 && x.stride(0) % e == 0 && x.stride(1) % e == 0 && x.stride(2) % e == 0 && x.stride(1) <= (1 << 22) &&
      (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15) == 0)
    return x;
  return x.clone(at::MemoryFormat::Contiguous);
}
struct Heads {
  long strides[9];
  Heads(const Tensor& q, const Tensor& k, const Tensor& v) {
    const Tensor* t[3] = {&q, &k, &v};
    for (int i = 0; i < 9; ++i) strides[i] = t[i / 3]->stride(i % 3);
  }
};
struct WindowOut {
  Tensor o, rest, lse, q, k, v;   // rest: what rounding o to bfloat16 left; q, k, v as the kernels read them
};
WindowOut window_run(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Window& w, const Tensor& lengths_, bool stats) {
  const c10::DeviceGuard guard(q_.device());
  WindowOut r;
  r.q = aligned_rows(q_);
  r.k = aligned_rows(k_);
  r.v = aligned_rows(v_);
  const Tensor lengths = dense(lengths_);
  const int64_t B = r.q.size(0), T = r.q.size(1), H = r.q.size(2), D = r.q.size(3);
  r.o = dense_like(r.q);
  if (stats) {
    r.lse = floats(B * H * T, r.q);
    if (r.q.scalar_type() == at::kBFloat16) r.rest = dense_like(r.q);
  }
  const Heads heads(r.q, r.k, r.v);
  ok(CALL(type_of("window_attention", r.q), wattn_fwd, elements(r.q), elements(r.k), elements(r.v), heads.strides, elements(r.o), ptr<void>(r.rest), ptr(r.lse),
          ptr<int>(lengths), (int)B, (int)T, (int)H, (int)r.k.size(2), (int)D, (int)std::min(w.left, T), (int)std::min(w.right, T), (int)std::min(w.sinks, T),
          (int)w.causal, (float)w.scale, stream_of(r.q)),
     "indm_wattn_fwd");
  return r;
}
struct WindowAttention : torch::autograd::Function<WindowAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, int64_t left, int64_t right, int64_t sinks, bool causal,
                        const Maybe& lengths_, double scale) {
    const Tensor lengths = plain(lengths_);
    WindowOut r = window_run(q, k, v, {left, right, sinks, causal, scale}, lengths, true);
    ctx->save_for_backward({r.q, r.k, r.v, r.o, r.rest, r.lse, lengths});
    ctx->saved_data["window"] = std::vector<int64_t>{left, right, sinks, causal};
    ctx->saved_data["want"] = (int64_t)((q.requires_grad() ? 1 : 0) | (k.requires_grad() || v.requires_grad() ? 2 : 0));   // (dk and dv come together)
    ctx->saved_data["scale"] = scale;
    return r.o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &o = saved[3], &rest = saved[4], &lse = saved[5];
    const c10::DeviceGuard guard(q.device());
    const Tensor lengths = dense(saved[6]);
    carries("window_attention", {&grads[0]});
    Tensor dout = whole(grads[0]).contiguous();
    if (reinterpret_cast<uintptr_t>(dout.data_ptr()) & 15) dout = dout.clone();
    const std::vector<int64_t> w = ctx->saved_data["window"].toIntVector();
    const int64_t T = q.size(1);
    const int B = (int)q.size(0), H = (int)q.size(2), Hk = (int)k.size(2), D = (int)q.size(3);
    const int left = (int)std::min(w[0], T), right = (int)std::min(w[1], T), sinks = (int)std::min(w[2], T), causal = (int)w[3];
    const int64_t want = ctx->saved_data["want"].toInt();
    Tensor dq = want & 1 ? dense_like(q) : Tensor(), dk = want & 2 ? dense_like(k) : Tensor(), dv = want & 2 ? dense_like(v) : Tensor();
    // (the scratch is an allocation of its own: calls on other streams and in other captured graphs share nothing)
    Tensor ws = floats(std::max(1L, abi.wattn_bwd_ws_floats(B, (int)T, H, Hk, D, left, right, sinks, causal)), q);
    const Heads heads(q, k, v);
    ok(CALL(type_of("window_attention", q), wattn_bwd, elements(q), elements(k), elements(v), heads.strides, elements(o), ptr<void>(rest), elements(dout), ptr(lse),
            ptr<int>(lengths), elements(dq), elements(dk), elements(dv), ptr(ws), B, (int)T, H, Hk, D, left, right, sinks, causal,
            (float)ctx->saved_data["scale"].toDouble(), stream_of(q)),
       "indm_wattn_bwd");
    return once({dq, dk, dv, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};
Tensor window_attention(const Tensor& q_, const Tensor& k_, const Tensor& v_, int64_t left, int64_t right, int64_t sinks, bool causal, const Maybe& lengths_,
                        double scale) {
  const Tensor q = whole(q_), k = whole(k_), v = whole(v_), lengths = plain(lengths_);
  const Window w = {left, right, sinks, causal, scale};
  carries("window_attention", {&q, &k, &v});
  window_check(q, k, v, w, lengths);
  return tracked({&q, &k, &v}) ? WindowAttention::apply(q, k, v, left, right, sinks, causal, Maybe(lengths), scale) : window_run(q, k, v, w, lengths, false).o;
}

}  // namespace

PYBIND11_MODULE(_token, m) {
  namespace py = pybind11;
  m.def("bind", &bind);
  m.def("guard", &guard);
  m.def("broken_guards", &broken_guards);
  m.def("layer_norm", &layer_norm, py::call_guard<py::gil_scoped_release>());
  m.def("dropout", &dropout, py::call_guard<py::gil_scoped_release>());
  m.def("rotary", &rotary, py::call_guard<py::gil_scoped_release>());
  m.def("window_attention", &window_attention, py::call_guard<py::gil_scoped_release>());
}
