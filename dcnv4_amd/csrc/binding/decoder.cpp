// What stands between the sampling layers of a deformable decoder: attention among queries and the normalised sum.  Checks, dense
// rows where the kernels need them, allocation and autograd nodes.
#include <ATen/autocast_mode.h>

#include <cmath>
#include <tuple>

#include "../add_norm.hpp"
#include "../query_attention.hpp"
#include "layers.hpp"

namespace dcn::binding {
namespace {

constexpr int64_t kIntMax = 0x7fffffff;

// ---------------------------------------------------------------- attention among queries
struct AttnInputs {
  Tensor q, k, v, q_segments, k_segments, q_points, k_points, slopes;
  float scale, cap;
};

struct AttnShape {
  int code;
  int64_t batch, nq, nk, heads, kv_heads, width;
  int64_t padded() const { return (width + 7) / 8 * 8; }
};

std::string text(at::IntArrayRef sizes) {
  std::string r = "(";
  for (size_t i = 0; i < sizes.size(); ++i) r += (i ? ", " : "") + std::to_string(sizes[i]);
  return r + ")";
}

void check_beside(const Tensor &t, const char *name, const Tensor &q, at::ScalarType dtype, at::IntArrayRef sizes) {
  if (!t.is_cuda()) raise_runtime("%s must be a CUDA tensor (Not implemented on the CPU)", name);
  if (t.device() != q.device()) raise_runtime("%s is on another device than query", name);
  if (t.scalar_type() != dtype) raise_runtime("%s has dtype %s, expected %s", name, c10::toString(t.scalar_type()), c10::toString(dtype));
  if (t.sizes() != sizes) raise_runtime("%s has shape %s, expected %s", name, text(t.sizes()).c_str(), text(sizes).c_str());
  if (!in_memory(t)) raise_runtime("%s has no memory of its own", name);
}

AttnShape attn_check(const AttnInputs &a) {
  if (!a.q.is_cuda()) raise_runtime("query must be a CUDA tensor (Not implemented on the CPU)");
  if (a.q.dim() != 4 || a.k.dim() != 4 || a.v.dim() != 4) raise_runtime("query, key and value must be 4-d (N, L, M, D)");
  AttnShape s;
  s.code = dtype_code(a.q, "query");
  const auto q = a.q.sizes(), k = a.k.sizes();
  s.batch = q[0]; s.nq = q[1]; s.heads = q[2]; s.width = q[3]; s.nk = k[1]; s.kv_heads = k[2];
  check_beside(a.q, "query", a.q, a.q.scalar_type(), q);
  check_beside(a.k, "key", a.q, a.q.scalar_type(), {s.batch, s.nk, s.kv_heads, s.width});
  check_beside(a.v, "value", a.q, a.q.scalar_type(), k);
  if (s.heads < 1 || s.kv_heads < 1 || s.heads % s.kv_heads != 0)
    raise_runtime("%lld heads of the query do not share %lld heads of the key evenly", (long long)s.heads, (long long)s.kv_heads);
  if (s.width < 1 || s.width > kMaxAttnWidth) raise_runtime("heads of %lld channels are not supported (1 to %d)", (long long)s.width, kMaxAttnWidth);
  // rows are counted in 32 bits by the kernels
  if (s.nq > (1 << 30) || s.nk > (1 << 30)) raise_runtime("sequences of more than 2^30 tokens");
  if (s.batch * s.nq * s.heads > kIntMax || s.batch * s.nk * s.kv_heads > kIntMax) raise_runtime("more than 2^31 - 1 rows of queries or keys");
  // the kernels address the rows of a tile, up to 256, in 31 bits; dense tensors, among them the result, have all heads between rows
  const int64_t row_bytes = s.padded() * a.q.element_size();
  for (const auto &[tokens, heads, name] : {std::tuple{s.nq, s.heads, "query"}, std::tuple{s.nk, s.kv_heads, "key"}})
    if (tokens > 1 && std::min<int64_t>(tokens, 256) * heads * row_bytes > kIntMax)
      raise_runtime("%lld heads of the %s: %lld tokens in a row reach over more than 2^31 - 1 bytes", (long long)heads, name, (long long)std::min<int64_t>(tokens, 256));
  // a launch has fewer than 2^32 threads: workgroups of 256 for 128 tokens of a head, of the wider rows 64
  const int64_t piece = row_bytes > 128 ? 64 : 128;
  if (s.batch * s.heads * ((s.nq + piece - 1) / piece) >= 1 << 24 || s.batch * s.kv_heads * ((s.nk + piece - 1) / piece) >= 1 << 24)
    raise_runtime("more than 2^24 - 1 pieces of %lld queries or keys of a head", (long long)piece);
  // (the kernels multiply both by a number below three: what passes fp32 would be NaN where a product is zero)
  if (!(std::fabs(a.scale) <= 1e30f)) raise_runtime("scale must be between -1e30 and 1e30");
  if (a.cap != 0.f && !(a.cap >= 1e-30f && a.cap <= 1e30f)) raise_runtime("cap must be zero (none) or between 1e-30 and 1e30");
  if (a.cap != 0.f && std::fabs(a.scale) > 1.000001e30 * a.cap) raise_runtime("scale may be up to 1e30 times cap");
  if (a.q_segments.defined()) {
    check_beside(a.q_segments, "segments", a.q, at::kInt, {s.batch, s.nq});
    if (!a.k_segments.defined()) raise_runtime("segments without key_segments");
  }
  if (a.k_segments.defined()) check_beside(a.k_segments, "key_segments", a.q, at::kInt, {s.batch, s.nk});
  if (a.slopes.defined() != a.q_points.defined() || a.slopes.defined() != a.k_points.defined())
    raise_runtime("positions, key_positions and slopes go together");
  if (a.slopes.defined()) {
    check_beside(a.slopes, "slopes", a.q, at::kFloat, {s.heads});
    check_beside(a.q_points, "positions", a.q, at::kFloat, {s.batch, s.nq, 2});
    check_beside(a.k_points, "key_positions", a.q, at::kFloat, {s.batch, s.nk, 2});
  }
  return s;
}

// Rows as the kernels read them: a dense width of a multiple of 8 (zeros behind the tensor's own), every row on 16 bytes.
Tensor attn_rows(const Tensor &t, const AttnShape &s) {
  if (s.padded() != s.width) return at::constant_pad_nd(t, {0, s.padded() - s.width}).contiguous();
  const int64_t size = t.element_size();
  bool fits = (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0 && (t.stride(3) == 1 || t.size(3) == 1);
  // (the kernels address the up to 256 rows of a tile in 31 bits; a copy's do as far as attn_check lets pass)
  for (int d = 0; d < 3; ++d) fits = fits && (t.size(d) <= 1 || (t.stride(d) * size % 16 == 0 && (d != 1 || t.stride(d) * size < (1 << 23))));
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}
AttnRows row_view(const Tensor &t) {
  auto step = [&](int d) { return t.size(d) > 1 ? (long long)t.stride(d) : 0; };
  return {t.const_data_ptr(), step(0), step(1), step(2)};
}
Tensor narrowed(const Tensor &t, const AttnShape &s) { return s.padded() == s.width ? t : t.narrow(3, 0, s.width).contiguous(); }

// What a launch points to, alive while it is enqueued.
struct AttnCall {
  Tensor q, k, v, q_segments, k_segments, q_points, k_points, slopes;
  AttnLaunch l = {};

  AttnCall(const AttnInputs &a, const AttnShape &s) : q(attn_rows(a.q, s)), k(attn_rows(a.k, s)), v(attn_rows(a.v, s)) {
    auto dense = [](const Tensor &t) { return t.defined() ? t.contiguous() : t; };
    q_segments = dense(a.q_segments); k_segments = dense(a.k_segments);
    q_points = dense(a.q_points); k_points = dense(a.k_points); slopes = dense(a.slopes);
    l.q = row_view(q); l.k = row_view(k); l.v = row_view(v);
    l.batch = (int)s.batch; l.nq = (int)s.nq; l.nk = (int)s.nk; l.heads = (int)s.heads; l.kv_heads = (int)s.kv_heads; l.width = (int)s.padded();
    l.scale = a.scale; l.cap = a.cap;
    l.q_segments = static_cast<const int *>(ptr(q_segments)); l.k_segments = static_cast<const int *>(ptr(k_segments));
    l.q_points = static_cast<const float *>(ptr(q_points)); l.k_points = static_cast<const float *>(ptr(k_points));
    l.slopes = static_cast<const float *>(ptr(slopes));
  }
};

// What the backward needs of a forward: the result, what rounding took from it (16-bit types) and (batch, heads, queries) logarithms.
struct AttnOutputs {
  Tensor out, rest, lse;
};
AttnOutputs attn_forward(const AttnInputs &a, bool train) {
  const AttnShape s = attn_check(a);
  OnDevice guard(a.q);
  Tensor out = at::empty({s.batch, s.nq, s.heads, s.padded()}, a.q.options()), rest, lse;
  if (train) lse = at::empty({s.batch, s.heads, s.nq}, a.q.options().dtype(at::kFloat));
  if (train && s.code != DCNV4_DTYPE_F32) rest = at::empty(out.sizes(), out.options());
  if (out.numel() != 0) {
    AttnCall c(a, s);
    c.l.out = out.data_ptr();
    c.l.out_rest = ptr(rest);
    c.l.lse = static_cast<float *>(ptr(lse));
    const Tensor ws = workspace(attn_forward_workspace_bytes(s.code, c.l), a.q);
    c.l.workspace = ptr(ws);
    hip_check(launch_attn_forward(s.code, c.l, static_cast<hipStream_t>(stream_of(a.q))), "query_attention");
  }
  return {narrowed(out, s), rest.defined() ? narrowed(rest, s) : rest, lse};
}

// Gradients of query, key, value and slopes, those that are wanted.
std::array<Tensor, 4> attn_backward(const AttnInputs &a, const AttnOutputs &found, const Tensor &grad_out, std::array<bool, 4> want) {
  const AttnShape s = attn_check(a);
  check_beside(grad_out, "grad_output", a.q, a.q.scalar_type(), a.q.sizes());
  check_beside(found.out, "output", a.q, a.q.scalar_type(), a.q.sizes());
  if (found.rest.defined()) check_beside(found.rest, "rest", a.q, a.q.scalar_type(), a.q.sizes());
  check_beside(found.lse, "lse", a.q, at::kFloat, {s.batch, s.heads, s.nq});
  OnDevice guard(a.q);
  std::array<Tensor, 4> grads;
  const auto options = a.q.options();
  const bool empty = a.q.numel() == 0 || a.k.numel() == 0;
  auto make = [&](at::IntArrayRef sizes, const at::TensorOptions &o) { return empty ? at::zeros(sizes, o) : at::empty(sizes, o); };
  if (want[0]) grads[0] = make({s.batch, s.nq, s.heads, s.padded()}, options);
  for (int i : {1, 2})
    if (want[i]) grads[i] = make({s.batch, s.nk, s.kv_heads, s.padded()}, options);
  if (want[3] && a.slopes.defined()) grads[3] = make({s.heads}, a.slopes.options());
  if (!empty) {
    AttnCall c(a, s);
    const Tensor o = attn_rows(found.out, s).contiguous(), r = found.rest.defined() ? attn_rows(found.rest, s).contiguous() : found.rest;
    const Tensor g = attn_rows(grad_out, s), l = found.lse.contiguous();
    c.l.out = o.data_ptr();
    c.l.out_rest = ptr(r);
    c.l.lse = l.data_ptr<float>();
    c.l.grad_out = row_view(g);
    c.l.grad_q = ptr(grads[0]); c.l.grad_k = ptr(grads[1]); c.l.grad_v = ptr(grads[2]);
    c.l.grad_slopes = static_cast<float *>(ptr(grads[3]));
    const Tensor ws = workspace(attn_backward_workspace_bytes(s.code, c.l), a.q);
    c.l.workspace = ptr(ws);
    hip_check(launch_attn_backward(s.code, c.l, static_cast<hipStream_t>(stream_of(a.q))), "the gradient of query_attention");
  }
  for (int i = 0; i < 3; ++i)
    if (grads[i].defined()) grads[i] = narrowed(grads[i], s);
  return grads;
}

struct QueryAttentionBackward final : torch::autograd::Node {
  SavedVariable q, k, v, q_segments, k_segments, q_points, k_points, slopes, out, rest, lse;      // all that hooks for saved tensors may pack
  float scale, cap;

  explicit QueryAttentionBackward(const AttnInputs &a)
      : q(a.q, false), k(a.k, false), v(a.v, false), q_segments(a.q_segments, false), k_segments(a.k_segments, false),
        q_points(a.q_points, false), k_points(a.k_points, false), slopes(a.slopes, false), scale(a.scale), cap(a.cap) {}
  std::string name() const override { return "QueryAttentionFunctionBackward"; }
  void release_variables() override {
    for (SavedVariable *s : {&q, &k, &v, &q_segments, &k_segments, &q_points, &k_points, &slopes, &out, &rest, &lse}) s->reset_data();
  }
  variable_list apply(variable_list &&grads) override {
    if (!grads[0].defined()) return variable_list(4);
    std::array<Tensor, 4> got;
    {
      at::AutoGradMode no_grad(false);
      const AttnInputs a = {q.unpack(), k.unpack(), v.unpack(), q_segments.unpack(), k_segments.unpack(), q_points.unpack(), k_points.unpack(),
                            slopes.unpack(), scale, cap};
      const Tensor o = out.unpack(shared_from_this());
      Tensor g = grads[0]._is_zerotensor() ? at::zeros(grads[0].sizes(), grads[0].options()) : grads[0];
      got = attn_backward(a, {o, rest.unpack(), lse.unpack()}, g, {task_should_compute_output(0), task_should_compute_output(1), task_should_compute_output(2),
                                         task_should_compute_output(3)});
    }
    return once_differentiable({got[0], got[1], got[2], got[3]});
  }
};

AttnInputs attn_inputs(Args &a) {
  AttnInputs in;
  in.q = a.tensor();
  in.k = a.tensor();
  in.v = a.tensor();
  in.q_segments = a.optional_tensor();
  in.k_segments = a.optional_tensor();
  in.q_points = a.optional_tensor();
  in.k_points = a.optional_tensor();
  in.slopes = a.optional_tensor();
  in.scale = a.real();
  in.cap = a.real();
  return in;
}

// query_attention(query, key, value, segments, key_segments, positions, key_positions, slopes, scale, cap), or None where the
// Function's methods have to run
PyObject *py_query_attention(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a("query_attention", args, n, 10);
  const AttnInputs in = attn_inputs(a);
  if (observed() || !plain(in.q) || !plain(in.k) || !plain(in.v) || (in.slopes.defined() && !plain(in.slopes))) Py_RETURN_NONE;
  Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    const bool train = wants_grad({&in.q, &in.k, &in.v, &in.slopes});
    AttnOutputs found = attn_forward(in, train);
    out = found.out;
    if (train) {
      std::shared_ptr<QueryAttentionBackward> node(new QueryAttentionBackward(in), torch::autograd::deleteNode);
      node->set_next_edges(torch::autograd::collect_next_edges(in.q, in.k, in.v, in.slopes));
      record(node, out);
      node->out = SavedVariable(out, true);
      node->rest = SavedVariable(found.rest, false);
      node->lse = SavedVariable(found.lse, false);
    }
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyObject *wrapped(const Tensor &t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}

// The arguments above: [out, rest or None, lse]
PyObject *py_query_attention_forward(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a("query_attention_forward", args, n, 10);
  const AttnInputs in = attn_inputs(a);
  at::AutoGradMode no_grad(false);
  const AttnOutputs r = attn_forward(in, true);
  return Py_BuildValue("[NNN]", wrapped(r.out), wrapped(r.rest), wrapped(r.lse));
  END_HANDLE_TH_ERRORS
}

// The arguments above, out, rest or None, lse, grad_output: [grad_query, grad_key, grad_value, grad_slopes or None]
PyObject *py_query_attention_backward(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a("query_attention_backward", args, n, 14);
  const AttnInputs in = attn_inputs(a);
  AttnOutputs found;
  found.out = a.tensor();
  found.rest = a.optional_tensor();
  found.lse = a.tensor();
  const Tensor &grad = a.tensor();
  at::AutoGradMode no_grad(false);
  const auto g = attn_backward(in, found, grad, {true, true, true, true});
  return Py_BuildValue("[NNNN]", wrapped(g[0]), wrapped(g[1]), wrapped(g[2]), wrapped(g[3]));
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- the normalised sum
struct NormInputs {
  Tensor x, residual, weight, bias;
  float eps;
  bool wide;      // a result in fp32 whatever the inputs
  at::ScalarType sum_dtype() const { return residual.defined() ? c10::promoteTypes(x.scalar_type(), residual.scalar_type()) : x.scalar_type(); }
  at::ScalarType out_dtype() const { return wide ? at::kFloat : sum_dtype(); }
};

void norm_check(const NormInputs &a) {
  if (!a.x.is_cuda()) raise_runtime("input must be a CUDA tensor (Not implemented on the CPU)");
  dtype_code(a.x, "input");
  if (a.x.dim() < 1 || a.x.size(-1) < 1 || a.x.size(-1) > kMaxNormWidth) raise_runtime("rows of 1 to %d channels are normalised, input has shape %s", kMaxNormWidth, text(a.x.sizes()).c_str());
  const int64_t width = a.x.size(-1);
  if (!in_memory(a.x)) raise_runtime("input has no memory of its own");
  if (a.residual.defined()) {
    check_beside(a.residual, "residual", a.x, a.residual.scalar_type(), a.x.sizes());
    dtype_code(a.residual, "residual");
    if (a.x.scalar_type() != a.residual.scalar_type() && a.sum_dtype() != a.x.scalar_type() && a.sum_dtype() != a.residual.scalar_type())
      raise_runtime("input and residual are of different 16-bit types");
  }
  for (const Tensor *t : {&a.weight, &a.bias})
    if (t->defined()) {
      check_beside(*t, t == &a.weight ? "weight" : "bias", a.x, t->scalar_type(), {width});
      dtype_code(*t, "weight and bias");
    }
  if (a.weight.defined() && a.bias.defined() && a.weight.scalar_type() != a.bias.scalar_type()) raise_runtime("weight and bias are of different types");
}

Tensor rows_of(const Tensor &t) {
  Tensor r = t.reshape({-1, t.size(-1)});
  return r.size(1) == 1 || r.stride(1) == 1 ? r : r.contiguous();
}

struct NormCall {
  Tensor x, residual, weight, bias;
  AddNormLaunch l = {};
  bool turned = false;      // x and residual have changed places

  explicit NormCall(const NormInputs &a) : x(rows_of(a.x)) {
    if (a.residual.defined()) residual = rows_of(a.residual);
    // the kernel wants the fp32 one of two types second
    turned = residual.defined() && x.scalar_type() != residual.scalar_type() && x.scalar_type() == at::kFloat;
    if (turned) std::swap(x, residual);
    if (a.weight.defined()) weight = a.weight.contiguous();
    if (a.bias.defined()) bias = a.bias.contiguous();
    l.x = view(x);
    if (residual.defined()) l.residual = view(residual);
    l.weight = ptr(weight); l.bias = ptr(bias);
    if (weight.defined() || bias.defined()) l.param_dtype = dtype_code(weight.defined() ? weight : bias, "weight");
    l.rows = x.size(0);
    l.width = (int)x.size(1);
    l.eps = a.eps;
    l.wide = a.wide;
  }
  static int code(at::ScalarType t) { return t == at::kFloat ? DCNV4_DTYPE_F32 : t == at::kHalf ? DCNV4_DTYPE_F16 : DCNV4_DTYPE_BF16; }

 private:
  static NormRows view(const Tensor &t) { return {t.const_data_ptr(), code(t.scalar_type()), t.size(0) > 1 ? (long long)t.stride(0) : 0}; }
};

struct NormOutputs {
  Tensor out, sum, stats;
};
NormOutputs norm_forward(const NormInputs &a, bool want_sum, bool want_stats) {
  norm_check(a);
  OnDevice guard(a.x);
  NormOutputs o;
  o.out = at::empty(a.x.sizes(), a.x.options().dtype(a.out_dtype()));
  if (want_sum) o.sum = at::empty(a.x.sizes(), a.x.options().dtype(a.sum_dtype()));
  if (want_stats) o.stats = at::empty({a.x.numel() / a.x.size(-1), 2}, a.x.options().dtype(at::kFloat));
  if (a.x.numel() != 0) {
    NormCall c(a);
    c.l.out = o.out.data_ptr();
    c.l.sum = ptr(o.sum);
    c.l.stats = static_cast<float *>(ptr(o.stats));
    hip_check(launch_add_norm_forward(c.l, static_cast<hipStream_t>(stream_of(a.x))), "add_layer_norm");
  }
  return o;
}

// Gradients of the two summands (one tensor for both where they have one type), weight and bias.
std::array<Tensor, 4> norm_backward(const NormInputs &a, const Tensor &stats, const Tensor &grad_out, const Tensor &grad_sum, std::array<bool, 4> want) {
  norm_check(a);
  const at::ScalarType sum_dtype = a.sum_dtype(), x_dtype = a.x.scalar_type(), residual_dtype = a.residual.defined() ? a.residual.scalar_type() : x_dtype;
  const int64_t width = a.x.size(-1), rows = a.x.numel() / width;
  check_beside(grad_out, "grad_output", a.x, a.wide ? at::kFloat : sum_dtype, a.x.sizes());
  if (grad_sum.defined()) check_beside(grad_sum, "grad_sum", a.x, sum_dtype, a.x.sizes());
  check_beside(stats, "stats", a.x, at::kFloat, {rows, 2});
  OnDevice guard(a.x);
  std::array<Tensor, 4> grads;
  const bool empty = rows == 0;
  auto make = [&](at::IntArrayRef sizes, at::ScalarType t) { return empty ? at::zeros(sizes, a.x.options().dtype(t)) : at::empty(sizes, a.x.options().dtype(t)); };
  if (want[0]) grads[0] = make(a.x.sizes(), x_dtype);
  if (want[1]) grads[1] = want[0] && x_dtype == residual_dtype ? grads[0] : make(a.x.sizes(), residual_dtype);
  if (want[2] && a.weight.defined()) grads[2] = make({width}, a.weight.scalar_type());
  if (want[3] && a.bias.defined()) grads[3] = make({width}, a.bias.scalar_type());
  if (!empty && (grads[0].defined() || grads[1].defined() || grads[2].defined() || grads[3].defined())) {
    NormCall c(a);
    const Tensor g = grad_out.contiguous(), s = grad_sum.defined() ? grad_sum.contiguous() : grad_sum, kept = stats.contiguous();
    c.l.stats = kept.data_ptr<float>();
    c.l.grad_out = g.data_ptr();
    c.l.grad_sum = ptr(s);
    c.l.grad_x = ptr(grads[0]);
    c.l.grad_residual = grads[1].is_same(grads[0]) ? nullptr : ptr(grads[1]);
    if (c.turned) std::swap(c.l.grad_x, c.l.grad_residual);
    c.l.grad_weight = ptr(grads[2]); c.l.grad_bias = ptr(grads[3]);
    const Tensor ws = workspace(add_norm_backward_workspace_bytes(c.l), a.x);
    c.l.workspace = ptr(ws);
    hip_check(launch_add_norm_backward(c.l, static_cast<hipStream_t>(stream_of(a.x))), "the gradient of add_layer_norm");
  }
  return grads;
}

// The summands are kept, not the sum: rounded to 16 bits it would show in the gradient of weight.
struct AddLayerNormBackward final : torch::autograd::Node {
  SavedVariable x, residual, weight, bias, stats;
  float eps;
  bool wide, has_residual;
  at::ScalarType x_dtype, residual_dtype;

  explicit AddLayerNormBackward(const NormInputs &a)
      : x(a.x, false), residual(a.residual, false), weight(a.weight, false), bias(a.bias, false), eps(a.eps), wide(a.wide),
        has_residual(a.residual.defined()), x_dtype(a.x.scalar_type()), residual_dtype(has_residual ? a.residual.scalar_type() : x_dtype) {}
  std::string name() const override { return "AddLayerNormFunctionBackward"; }
  void release_variables() override {
    for (SavedVariable *s : {&x, &residual, &weight, &bias, &stats}) s->reset_data();
  }
  variable_list apply(variable_list &&grads) override {
    const Tensor around = grads.size() > 1 ? grads[1] : Tensor();
    if (!grads[0].defined() && !around.defined()) return variable_list(4);
    std::array<Tensor, 4> got;
    {
      at::AutoGradMode no_grad(false);
      auto dense = [](const Tensor &t) { return t.defined() && t._is_zerotensor() ? at::zeros(t.sizes(), t.options()) : t; };
      if (!grads[0].defined()) {
        got[0] = around.to(x_dtype);
        if (has_residual) got[1] = around.to(residual_dtype);
      } else {
        NormInputs a;
        a.x = x.unpack();
        a.residual = residual.unpack();
        a.weight = weight.unpack();
        a.bias = bias.unpack();
        a.eps = eps;
        a.wide = wide;
        got = norm_backward(a, stats.unpack(), dense(grads[0]), dense(around),
                            {task_should_compute_output(0), has_residual && task_should_compute_output(1), task_should_compute_output(2),
                             task_should_compute_output(3)});
      }
    }
    return once_differentiable({got[0], got[1], got[2], got[3]});
  }
};

NormInputs norm_inputs(Args &a) {
  NormInputs in;
  in.x = a.tensor();
  in.residual = a.optional_tensor();
  in.weight = a.optional_tensor();
  in.bias = a.optional_tensor();
  in.eps = a.real();
  in.wide = a.integer() != 0;
  return in;
}

// Whether the kernels take a call as it is: rows of a length and of types that they know, all on one GPU.
bool norm_takes(const NormInputs &a) {
  if (!a.x.is_cuda() || a.x.dim() < 1 || a.x.size(-1) < 1 || a.x.size(-1) > kMaxNormWidth) return false;
  at::ScalarType half = at::kFloat;
  for (const Tensor *t : {&a.x, &a.residual, &a.weight, &a.bias}) {
    if (!t->defined()) continue;
    const at::ScalarType type = t->scalar_type();
    if (t->device() != a.x.device() || (type != at::kFloat && type != at::kHalf && type != at::kBFloat16)) return false;
    if (type != at::kFloat && half != at::kFloat && type != half) return false;
    if (type != at::kFloat) half = type;
    if (!plain(*t)) return false;
  }
  if (a.residual.defined() && a.residual.sizes() != a.x.sizes()) return false;
  for (const Tensor *t : {&a.weight, &a.bias})
    if (t->defined() && (t->dim() != 1 || t->size(0) != a.x.size(-1))) return false;
  return !a.weight.defined() || !a.bias.defined() || a.weight.scalar_type() == a.bias.scalar_type();
}

// The result or (result, sum), with its node; None where it is not taken.
PyObject *norm_call(const NormInputs &in, bool want_sum) {
  if (observed() || !norm_takes(in)) Py_RETURN_NONE;
  NormOutputs o;
  {
    pybind11::gil_scoped_release no_gil;
    const bool train = wants_grad({&in.x, &in.residual, &in.weight, &in.bias});
    o = norm_forward(in, want_sum, train);
    if (train) {
      std::shared_ptr<AddLayerNormBackward> node(new AddLayerNormBackward(in), torch::autograd::deleteNode);
      node->set_next_edges(torch::autograd::collect_next_edges(in.x, in.residual, in.weight, in.bias));
      record(node, o.out);
      if (want_sum) record(node, o.sum);
      node->stats = SavedVariable(o.stats, false);
    }
  }
  if (!want_sum) return THPVariable_Wrap(std::move(o.out));
  return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(o.out)), THPVariable_Wrap(std::move(o.sum)));
}

// add_layer_norm(input, residual, weight, bias, eps, wide, want_sum)
PyObject *py_add_layer_norm(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a("add_layer_norm", args, n, 7);
  const NormInputs in = norm_inputs(a);
  return norm_call(in, a.integer() != 0);
  END_HANDLE_TH_ERRORS
}

// Whether a call of the module is torch's layer norm over the last axis with its parameters, and nothing else.
bool plain_norm(const Module &norm, int64_t width) {
  if (global_module_hooks() || !norm.called_as(kLayerNorm)) return false;
  PyObject *shape = norm.attribute("normalized_shape");
  return shape != nullptr && PyTuple_CheckExact(shape) && PyTuple_GET_SIZE(shape) == 1 && PyLong_Check(PyTuple_GET_ITEM(shape, 0)) &&
         PyLong_AsLongLong(PyTuple_GET_ITEM(shape, 0)) == width;
}

// add_layer_norm_of(norm, input, residual, want_sum): the same of a module, read and checked here (its parameters by attribute take as long as
// all the rest of a small call does on the host)
PyObject *py_add_layer_norm_of(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a("add_layer_norm_of", args + 1, n - 1, 3);
  const Module norm(args[0]);
  NormInputs in;
  in.x = a.tensor();
  in.residual = a.optional_tensor();
  const bool want_sum = a.integer() != 0;
  if (in.x.dim() < 1 || !plain_norm(norm, in.x.size(-1))) Py_RETURN_NONE;
  in.weight = norm.parameter("weight");
  in.bias = norm.parameter("bias");
  const double eps = norm.real("eps", NAN);
  if (std::isnan(eps)) Py_RETURN_NONE;      // a number of another class, which Python reads
  in.eps = (float)eps;
  in.wide = at::autocast::is_autocast_enabled(at::kCUDA);
  return norm_call(in, want_sum);
  END_HANDLE_TH_ERRORS
}

// plain_layer_norm(norm, width)
PyObject *py_plain_layer_norm(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a("plain_layer_norm", args + 1, n - 1, 1);
  const long long width = PyLong_AsLongLong(args[1]);
  if (width == -1 && PyErr_Occurred()) throw python_error();
  return PyBool_FromLong(plain_norm(Module(args[0]), width));
  END_HANDLE_TH_ERRORS
}

// add_layer_norm_forward(input, residual, weight, bias, eps, wide): [result, sum, stats]
PyObject *py_add_layer_norm_forward(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a("add_layer_norm_forward", args, n, 6);
  const NormInputs in = norm_inputs(a);
  at::AutoGradMode no_grad(false);
  const NormOutputs o = norm_forward(in, true, true);
  return Py_BuildValue("[NNN]", THPVariable_Wrap(o.out), THPVariable_Wrap(o.sum), THPVariable_Wrap(o.stats));
  END_HANDLE_TH_ERRORS
}

// add_layer_norm_backward(input, residual, weight, bias, eps, wide, stats, grad_output, grad_sum or None):
// [grad_input, grad_residual, grad_weight, grad_bias]
PyObject *py_add_layer_norm_backward(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a("add_layer_norm_backward", args, n, 9);
  const NormInputs in = norm_inputs(a);
  const Tensor &stats = a.tensor(), &grad = a.tensor();
  const Tensor around = a.optional_tensor();
  at::AutoGradMode no_grad(false);
  const bool residual = in.residual.defined();
  const auto g = norm_backward(in, stats, grad, around, {true, residual, true, true});
  return Py_BuildValue("[NNNN]", wrapped(g[0]), wrapped(g[1]), wrapped(g[2]), wrapped(g[3]));
  END_HANDLE_TH_ERRORS
}

#define FASTCALL(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(fn)), METH_FASTCALL, nullptr}

}  // namespace

PyMethodDef decoder_methods[] = {FASTCALL("query_attention", py_query_attention),
                                 FASTCALL("query_attention_forward", py_query_attention_forward),
                                 FASTCALL("query_attention_backward", py_query_attention_backward),
                                 FASTCALL("add_layer_norm", py_add_layer_norm),
                                 FASTCALL("add_layer_norm_of", py_add_layer_norm_of),
                                 FASTCALL("plain_layer_norm", py_plain_layer_norm),
                                 FASTCALL("add_layer_norm_forward", py_add_layer_norm_forward),
                                 FASTCALL("add_layer_norm_backward", py_add_layer_norm_backward),
                                 {nullptr, nullptr, 0, nullptr}};

}  // namespace dcn::binding
