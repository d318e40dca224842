/* torch binding of the policy operators (include/ur3e_policy.h), loaded by ur3e_amd/rl/ops.py.
 *
 * An update of the policy is a few microseconds of kernels a call, so what a call costs on the host is what a small
 * minibatch waits for: the checks, the outputs, the workspace and the autograd node are C++ (a Python
 * autograd.Function with ctypes calls took 190 us forward and backward for 16 environments x 16 steps, whose
 * kernels run 21 us). */
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/extension.h>

#include <cmath>
#include <unordered_set>

#include "../../include/ur3e_batch.h"
#include "../../include/ur3e_policy.h"

namespace {

using at::Tensor;
using OptT = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int dtype_of(const Tensor& x) {
  switch (x.scalar_type()) {
    case at::kFloat: return UR3E_F32;
    case at::kBFloat16: return UR3E_BF16;
    case at::kHalf: return UR3E_F16;
    default: return -1;
  }
}

void chk(int rc) {
  TORCH_CHECK_VALUE(rc != UR3E_EINVAL, ur3e_last_error());
  TORCH_CHECK(rc == UR3E_OK, "ur3e library error ", rc, ": ", ur3e_last_error());
}

void* stream_of(const Tensor& x) {
  return (void*)at::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.device().index()).stream();
}

const void* ptr(const Tensor& x) { return x.defined() ? x.const_data_ptr() : nullptr; }

/* the tensor, with the channels of a token next to each other */
Tensor unit(const Tensor& x) { return x.stride(-1) == 1 || x.size(-1) == 1 ? x : x.contiguous(); }

/* Forward-mode derivatives: the kernels compute none, and their outputs would be taken for constants. */
bool has_tangent(const Tensor& x) {
  return x.defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode() && x._fw_grad(0).defined();
}
void check_tangents(const char* what, std::initializer_list<Tensor> xs) {
  for (const Tensor& x : xs)
    TORCH_CHECK_VALUE(!has_tangent(x), what, ": no forward-mode derivatives on the GPU; pass primals (forward_ad.unpack_dual)");
}

/* Gradients under capture: where a leaf in front of x is held by an eager graph that still lives, its gradient is
   accumulated on that graph's stream.  From a capture, torch's engine then makes the default stream wait for work that is
   only being recorded, and the process ends.  So the call is refused while its graph is built. */
void check_capture(const char* what, std::initializer_list<Tensor> xs) {
  using torch::autograd::Node;
  const hipStream_t stream = (hipStream_t)stream_of(*xs.begin());
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  /* (the default stream cannot be captured) */
  if (!stream || hipStreamIsCapturing(stream, &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;
  std::vector<std::shared_ptr<Node>> todo;
  std::unordered_set<const Node*> met;
  for (const Tensor& x : xs)
    if (x.defined() && x.requires_grad()) todo.push_back(torch::autograd::impl::gradient_edge(x).function);
  while (!todo.empty()) {
    const std::shared_ptr<Node> n = todo.back();
    todo.pop_back();
    if (!n || !met.insert(n.get()).second) continue;
    if (n->name() == "torch::autograd::AccumulateGrad") {
      const auto st = n->stream();
      TORCH_CHECK(!st || st->id() != 0, what, ": under capture, but an eager graph of the default stream still holds one "
                  "of the leaves, which a captured backward pass cannot reach; drop its outputs first (or capture the "
                  "forward pass alone under torch.no_grad())");
    }
    for (const auto& edge : n->next_edges()) todo.push_back(edge.function);
  }
}

/* ---- attention ---- */

/* dims: 4 for sequences [b, t, heads, d], 3 for one token [b, heads, d] */
void check_attention(const std::string& what, int64_t dims, const Tensor& q, const Tensor& k, const Tensor& v,
                     const Tensor& log_decay, const OptT& starts, double scale) {
  TORCH_CHECK_VALUE(dtype_of(q) >= 0, what, ": q must be float32, bfloat16 or float16, got ", q.scalar_type());
  TORCH_CHECK_VALUE(q.dim() == dims && k.dim() == dims && v.dim() == dims, what, ": q, k and v must have ", dims,
                    " dimensions, got ", q.sizes(), ", ", k.sizes(), ", ", v.sizes());
  const auto lead = q.sizes().slice(0, dims - 2);
  for (const auto& [n, x] : {std::pair<const char*, const Tensor&>("k", k), {"v", v}}) {
    TORCH_CHECK_VALUE(x.scalar_type() == q.scalar_type() && x.device() == q.device(), what, ": ", n, " is ",
                      x.scalar_type(), " on ", x.device(), ", q ", q.scalar_type(), " on ", q.device());
    TORCH_CHECK_VALUE(x.sizes().slice(0, dims - 2) == lead, what, ": ", n, " has leading sizes ",
                      x.sizes().slice(0, dims - 2), ", q ", lead);
  }
  const int64_t h = q.size(-2), hk = k.size(-2);
  TORCH_CHECK_VALUE(h >= 1 && hk >= 1 && h % hk == 0 && v.size(-2) == hk, what, ": ", h, " query heads over ", hk,
                    " key heads and ", v.size(-2),
                    " value heads: the key and value heads must be as many, and divide the query heads");
  TORCH_CHECK_VALUE(k.size(-1) == q.size(-1), what, ": q has ", q.size(-1), " channels, k ", k.size(-1));
  TORCH_CHECK_VALUE(q.size(-1) >= 1 && q.size(-1) <= UR3E_ATTN_MAX_DIM, what, ": q and k must have 1 to ",
                    UR3E_ATTN_MAX_DIM, " channels, got ", q.size(-1));
  TORCH_CHECK_VALUE(v.size(-1) >= 1 && v.size(-1) <= UR3E_ATTN_MAX_DIM, what, ": v must have 1 to ",
                    UR3E_ATTN_MAX_DIM, " channels, got ", v.size(-1));
  TORCH_CHECK_VALUE(log_decay.scalar_type() == at::kFloat && log_decay.device() == q.device() && log_decay.dim() == 1 &&
                        log_decay.size(0) == h,
                    what, ": log_decay must be a float32 tensor of shape (", h, ",) on ", q.device());
  TORCH_CHECK_VALUE(!(log_decay.requires_grad() && at::GradMode::is_enabled()), what,
                    ": log_decay is a constant of the heads and gets no gradient; detach it");
  TORCH_CHECK_VALUE(!has_tangent(log_decay), what, ": log_decay is a constant of the heads and has no forward-mode derivative; detach it");
  if (starts)
    TORCH_CHECK_VALUE((starts->scalar_type() == at::kBool || starts->scalar_type() == at::kByte) &&
                          starts->device() == q.device() && starts->sizes() == lead,
                      what, ": starts must be a bool or uint8 tensor of shape ", lead, " on ", q.device());
  TORCH_CHECK_VALUE(std::isfinite(scale), what, ": scale must be finite, got ", scale);
  for (int64_t i = 0; i < dims - 1; i++)
    TORCH_CHECK_VALUE(q.size(i) <= INT32_MAX, what, ": a size of ", q.size(i), " is past 32 bits");
}

void check_state(const std::string& what, const char* name, const Tensor& s, const Tensor& q, const Tensor& v) {
  TORCH_CHECK_VALUE(s.scalar_type() == at::kFloat && s.device() == q.device() && s.dim() == 4 &&
                        s.size(0) == q.size(0) && s.size(1) == q.size(-2) && s.size(2) == q.size(-1) &&
                        s.size(3) == v.size(-1),
                    what, ": ", name, " must be a float32 tensor of shape (", q.size(0), ", ", q.size(-2), ", ",
                    q.size(-1), ", ", v.size(-1), ") on ", q.device());
}

void check_sequences(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const OptT& s0,
                     const OptT& starts, const OptT& lengths, double scale) {
  const std::string what = "decay_attention";
  check_attention(what, 4, q, k, v, log_decay, starts, scale);
  if (s0) check_state(what, "initial_state", *s0, q, v);
  if (lengths)
    TORCH_CHECK_VALUE(lengths->scalar_type() == at::kInt && lengths->device() == q.device() && lengths->dim() == 1 &&
                          lengths->size(0) == q.size(0),
                      what, ": lengths must be an int32 tensor of shape (", q.size(0), ",) on ", q.device());
}

void check_step(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Tensor& state,
                const OptT& starts, double scale, const OptT& next, bool update) {
  const std::string what = "decay_attention_step";
  check_attention(what, 3, q, k, v, log_decay, starts, scale);
  check_state(what, "state", state, q, v);
  TORCH_CHECK_VALUE(state.is_contiguous(), what, ": state must be contiguous");
  TORCH_CHECK_VALUE(!at::GradMode::is_enabled() || !(q.requires_grad() || k.requires_grad() || v.requires_grad() || state.requires_grad()),
                    what, ": one token has no gradients; call it under torch.no_grad(), or decay_attention");
  if (next) {
    TORCH_CHECK_VALUE(update, what, ": next_state without an update");
    check_state(what, "next_state", *next, q, v);
    TORCH_CHECK_VALUE(next->is_contiguous(), what, ": next_state must be contiguous");
    const char *x = (const char*)state.const_data_ptr(), *y = (const char*)next->const_data_ptr();
    const int64_t n = state.numel() * 4;
    TORCH_CHECK_VALUE(x == y || (x > y ? x - y >= n : y - x >= n), what, ": next_state overlaps state");
  }
}

ur3e_tokens_t tok(const Tensor& x) { return {(void*)x.const_data_ptr(), x.stride(0), x.stride(1), x.stride(2)}; }

/* an empty [b, t, heads, d] in the memory order of `ref` (sequence- or time-major) */
Tensor tokens_like(const Tensor& ref, int64_t heads, int64_t d) {
  const int64_t b = ref.size(0), t = ref.size(1);
  if (t > 1 && b > 1 && ref.stride(1) > ref.stride(0)) return at::empty({t, b, heads, d}, ref.options()).transpose(0, 1);
  return at::empty({b, t, heads, d}, ref.options());
}

ur3e_attn_t args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Tensor& s0,
                 const Tensor& starts, const Tensor& lengths, double scale) {
  ur3e_attn_t a = {};
  a.b = (int)q.size(0); a.t = (int)q.size(1); a.heads = (int)q.size(2); a.kv_heads = (int)k.size(2);
  a.dk = (int)q.size(3); a.dv = (int)v.size(3);
  a.dtype = dtype_of(q);
  a.scale = (float)scale;
  a.q = tok(q); a.k = tok(k); a.v = tok(v);
  a.log_decay = (const float*)ptr(log_decay);
  a.s0 = (const float*)ptr(s0);
  a.starts = (const unsigned char*)ptr(starts);
  if (starts.defined()) { a.starts_sb = starts.stride(0); a.starts_st = starts.stride(1); }
  a.lengths = (const int*)ptr(lengths);
  return a;
}

Tensor workspace(const ur3e_attn_t& a, int backward, const Tensor& like) {
  size_t n = 0;
  chk(ur3e_attn_workspace(&a, backward, &n));
  return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : Tensor();
}

/* Input tensors of a call, as the kernels take them; unused ones are undefined. */
struct Inputs {
  Tensor q, k, v, s0, log_decay, starts, lengths;
  double scale;
};

std::pair<Tensor, Tensor> forward(const Inputs& x, bool return_state) {
  c10::DeviceGuard guard(x.q.device());
  Tensor out = tokens_like(x.q, x.q.size(2), x.v.size(3)), state;
  if (return_state) state = at::empty({x.q.size(0), x.q.size(2), x.q.size(3), x.v.size(3)}, x.q.options().dtype(at::kFloat));
  const ur3e_attn_t a = args(x.q, x.k, x.v, x.log_decay, x.s0, x.starts, x.lengths, x.scale);
  const Tensor ws = workspace(a, 0, x.q);
  const ur3e_tokens_t o = tok(out);
  chk(ur3e_attn_forward(&a, &o, (float*)ptr(state), (void*)ptr(ws), ws.defined() ? ws.numel() : 0, stream_of(x.q)));
  return {out, state};
}

struct DecayAttention : torch::autograd::Function<DecayAttention> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                               const OptT& s0, const Tensor& log_decay, const OptT& starts, const OptT& lengths,
                               double scale, bool return_state) {
    const Inputs x{q, k, v, s0.value_or(Tensor()), log_decay, starts.value_or(Tensor()), lengths.value_or(Tensor()), scale};
    const auto [out, state] = ::forward(x, return_state);
    ctx->save_for_backward({x.q, x.k, x.v, x.s0, x.log_decay, x.starts, x.lengths});
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    if (!return_state) return {out};
    return {out, state};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "decay_attention is differentiable once");
    const variable_list x = ctx->get_saved_variables();
    const Tensor &q = x[0], &k = x[1], &v = x[2], &s0 = x[3];
    c10::DeviceGuard guard(q.device());
    Tensor dout = grads[0], ds = grads.size() > 1 ? grads[1] : Tensor();
    check_tangents("decay_attention", {dout, ds});
    dout = dout.defined() ? unit(dout) : at::zeros({1, 1, 1, v.size(3)}, q.options()).expand({q.size(0), q.size(1), q.size(2), v.size(3)});
    if (ds.defined()) ds = ds.contiguous();
    const Tensor dq = tokens_like(q, q.size(2), q.size(3)), dk = tokens_like(k, k.size(2), k.size(3)),
                 dv = tokens_like(v, v.size(2), v.size(3));
    Tensor ds0;
    if (s0.defined() && ctx->needs_input_grad(3)) /* an absent state has no edge */
      ds0 = at::empty_like(s0);
    const ur3e_attn_t a = args(q, k, v, x[4], s0, x[5], x[6], ctx->saved_data["scale"].toDouble());
    const ur3e_tokens_t g = tok(dout), tq = tok(dq), tk = tok(dk), tv = tok(dv);
    const Tensor ws = workspace(a, 1, q);
    chk(ur3e_attn_backward(&a, &g, (const float*)ptr(ds), &tq, &tk, &tv, (float*)ptr(ds0), (void*)ptr(ws),
                           ws.defined() ? ws.numel() : 0, stream_of(q)));
    return {dq, dk, dv, ds0, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::pair<Tensor, OptT> decay_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay,
                                        const OptT& s0, const OptT& starts, const OptT& lengths, double scale,
                                        bool return_state) {
  check_sequences(q, k, v, log_decay, s0, starts, lengths, scale);
  check_tangents("decay_attention", {q, k, v, s0.value_or(Tensor())});
  Inputs x{unit(q), unit(k), unit(v), s0 ? s0->contiguous() : Tensor(), log_decay.detach().contiguous(),
           starts ? *starts : Tensor(), lengths ? lengths->contiguous() : Tensor(), scale};
  const bool grad = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() ||
                                                   (s0 && s0->requires_grad()));
  if (!grad) {
    const auto [out, state] = forward(x, return_state);
    return {out, return_state ? OptT(state) : OptT()};
  }
  check_capture("decay_attention", {x.q, x.k, x.v, x.s0});
  auto opt = [](const Tensor& t) { return t.defined() ? OptT(t) : OptT(); };
  const variable_list r = DecayAttention::apply(x.q, x.k, x.v, opt(x.s0), x.log_decay, opt(x.starts), opt(x.lengths), scale,
                                                return_state);
  return {r[0], return_state ? OptT(r[1]) : OptT()};
}

Tensor decay_attention_step(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, Tensor state,
                            const OptT& starts, double scale, const OptT& next, bool update) {
  check_step(q, k, v, log_decay, state, starts, scale, next, update);
  check_tangents("decay_attention_step", {q, k, v, state, next.value_or(Tensor())});
  at::NoGradGuard no_grad;
  c10::DeviceGuard guard(q.device());
  const Tensor q1 = unit(q), k1 = unit(k), v1 = unit(v), ld = log_decay.contiguous();
  Tensor out = at::empty({q.size(0), q.size(1), v.size(2)}, q.options());
  auto one = [](const Tensor& x) { return ur3e_tokens_t{(void*)x.const_data_ptr(), x.stride(0), 0, x.stride(1)}; };
  ur3e_attn_t a = {};
  a.b = (int)q.size(0); a.t = 1; a.heads = (int)q.size(1); a.kv_heads = (int)k.size(1);
  a.dk = (int)q.size(2); a.dv = (int)v.size(2);
  a.dtype = dtype_of(q);
  a.scale = (float)scale;
  a.q = one(q1); a.k = one(k1); a.v = one(v1);
  a.log_decay = ld.const_data_ptr<float>();
  if (starts) { a.starts = (const unsigned char*)starts->const_data_ptr(); a.starts_sb = starts->stride(0); }
  const Tensor to = !update ? Tensor() : next ? *next : state;
  const ur3e_tokens_t o = one(out);
  chk(ur3e_attn_step(&a, &o, (const float*)state.const_data_ptr(), (float*)ptr(to), stream_of(q)));
  if (to.defined() && !to.is_inference()) to.unsafeGetTensorImpl()->bump_version(); /* autograd notices the write */
  return out;
}

/* ---- keyed dropout ---- */

void check_dropout(const Tensor& x, const OptT& rows, const OptT& residual) {
  const char* what = "keyed_dropout";
  TORCH_CHECK_VALUE(dtype_of(x) >= 0 && x.dim() >= 1, what,
                    ": x must be a float32, bfloat16 or float16 tensor of at least one dimension");
  const int64_t n = c10::multiply_integers(x.sizes().slice(0, x.dim() - 1));
  if (rows)
    TORCH_CHECK_VALUE(rows->scalar_type() == at::kLong && rows->device() == x.device() && rows->numel() == n, what,
                      ": rows must be ", n, " int64 ids on ", x.device());
  if (residual)
    TORCH_CHECK_VALUE(residual->scalar_type() == x.scalar_type() && residual->device() == x.device() &&
                          residual->sizes() == x.sizes(),
                      what, ": residual must be like x: ", x.sizes(), " ", x.scalar_type(), " on ", x.device());
}

/* x as [rows, columns] with contiguous columns, without a copy where its strides allow it */
Tensor rows2d(const Tensor& x) { return unit(x.dim() == 2 ? x : x.reshape({-1, x.size(-1)})); }

struct Key {
  int64_t count, substream;
  uint64_t seed;
};

Tensor dropout(const Tensor& x, const Tensor& residual, const Tensor& rows, const Key& key) {
  c10::DeviceGuard guard(x.device());
  if (x.numel() == 0) return at::empty(x.sizes(), x.options());
  const Tensor x2 = rows2d(x), r2 = residual.defined() ? rows2d(residual) : Tensor();
  const Tensor y = at::empty(x.sizes(), x.options());
  TORCH_CHECK_VALUE(x2.size(1) <= INT32_MAX - 8, "keyed_dropout: too many columns");
  chk(ur3e_keyed_dropout(dtype_of(x), x2.size(0), (int)x2.size(1), ptr(x2), x2.stride(0), ptr(r2),
                         r2.defined() ? r2.stride(0) : 0, (void*)y.const_data_ptr(), x2.size(1),
                         (const long long*)ptr(rows), key.seed, (unsigned)key.substream, (int)key.count, stream_of(x)));
  return y;
}

struct KeyedDropout : torch::autograd::Function<KeyedDropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptT& residual, const OptT& rows,
                        int64_t count, int64_t seed, int64_t substream) {
    const Tensor ids = rows.value_or(Tensor());
    ctx->save_for_backward({ids});
    ctx->saved_data["key"] = std::vector<int64_t>{count, seed, substream, residual.has_value()};
    return dropout(x, residual.value_or(Tensor()), ids, {count, substream, (uint64_t)seed});
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "keyed_dropout is differentiable once");
    const auto key = ctx->saved_data["key"].toIntVector();
    const Tensor& dy = grads[0];
    check_tangents("keyed_dropout", {dy});
    Tensor dx;
    if (ctx->needs_input_grad(0))
      dx = dropout(dy, Tensor(), ctx->get_saved_variables()[0], {key[0], key[2], (uint64_t)key[1]});
    return {dx, key[3] && ctx->needs_input_grad(1) ? dy : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor keyed_dropout(const Tensor& x, int64_t count, uint64_t seed, const OptT& rows, int64_t substream,
                     const OptT& residual) {
  check_dropout(x, rows, residual);
  check_tangents("keyed_dropout", {x, residual.value_or(Tensor())});
  const OptT ids = rows ? OptT(rows->reshape(-1).contiguous()) : OptT();
  if (at::GradMode::is_enabled() && (x.requires_grad() || (residual && residual->requires_grad()))) {
    check_capture("keyed_dropout", {x, residual.value_or(Tensor())});
    return KeyedDropout::apply(x, residual, ids, count, (int64_t)seed, substream);
  }
  return dropout(x, residual.value_or(Tensor()), ids.value_or(Tensor()), {count, substream, seed});
}

}  // namespace

PYBIND11_MODULE(ur3e_policy_torch, m) {
  m.def("check_sequences", &check_sequences);
  m.def("check_step", &check_step);
  m.def("check_dropout", &check_dropout);
  m.def("decay_attention", &decay_attention);
  m.def("decay_attention_step", &decay_attention_step);
  m.def("keyed_dropout", &keyed_dropout);
}
