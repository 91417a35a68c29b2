// torch.ops.bdh.* of the parts of a state-space layer (causal convolution, per-head norm + rotation, selective
// scan). Shapes that the kernels rely on are checked here once more, so that a direct call cannot make them read or
// write out of range. Unlike in bindings.cpp, results and scratch are allocated here, from torch's allocator on the
// current stream, and the derivatives of the sequence forms are autograd nodes of C++: a small call is as long as its
// way through Python, and every tensor and node made there adds to it.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/library.h>

#include <algorithm>
#include <initializer_list>
#include <memory>
#include <string>
#include <vector>

#include "bdh_kernels.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

void check_rc(int rc, const char* what) { TORCH_CHECK(rc == BDH_OK, "bdh kernel '", what, "' failed with code ", rc); }

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

int elem_type(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return BDH_F32;
    case at::kHalf: return BDH_F16;
    case at::kBFloat16: return BDH_BF16;
    default: TORCH_CHECK(false, name, ": expected fp32, fp16 or bf16");
  }
}

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

// `t` on the device of `on`, of type `type` and the given sizes, the last dimension adjacent
void check_rows(const Tensor& t, const Tensor& on, at::ScalarType type, at::IntArrayRef sizes, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == on.device(), name, ": expected a tensor on ", on.device());
  TORCH_CHECK(t.scalar_type() == type, name, ": expected ", type, ", got ", t.scalar_type());
  TORCH_CHECK(t.sizes() == sizes, name, ": expected sizes ", sizes, ", got ", t.sizes());
  TORCH_CHECK(t.dim() == 0 || t.size(-1) <= 1 || t.stride(-1) == 1, name, ": expected a last dimension of stride 1");
}

void check_dense(const Tensor& t, const Tensor& on, at::ScalarType type, at::IntArrayRef sizes, const char* name) {
  check_rows(t, on, type, sizes, name);
  TORCH_CHECK(t.is_contiguous(), name, ": expected a contiguous tensor");
}

void check_f32(const OptTensor& t, const Tensor& on, at::IntArrayRef sizes, const char* name) {
  if (given(t)) check_dense(*t, on, at::kFloat, sizes, name);
}

const float* f32_ptr(const OptTensor& t) { return given(t) ? t->const_data_ptr<float>() : nullptr; }

void set_lengths(const OptTensor& t, const Tensor& on, int64_t B, const void*& ptr, int& is64) {
  ptr = nullptr;
  is64 = 0;
  if (!given(t)) return;
  TORCH_CHECK(t->is_cuda() && t->device() == on.device() && t->dim() == 1 && t->size(0) == B && t->is_contiguous() &&
              (t->scalar_type() == at::kInt || t->scalar_type() == at::kLong), "lengths: expected int32 or int64 [", B, "] on ",
              on.device());
  ptr = t->const_data_ptr();
  is64 = t->scalar_type() == at::kLong;
}

const unsigned char* active_ptr(const OptTensor& t, const Tensor& on, int64_t B) {
  if (!given(t)) return nullptr;
  check_dense(*t, on, at::kBool, {B}, "active");
  return reinterpret_cast<const unsigned char*>(t->const_data_ptr());
}

// Bytes from the first element of a tensor's dimensions from `dim` on to behind their last
int64_t reach(const Tensor& t, int64_t dim) {
  int64_t n = 1;
  for (int64_t i = dim; i < t.dim(); ++i) n += (t.size(i) - 1) * t.stride(i);
  return n * static_cast<int64_t>(t.element_size());
}

// Do two tensors share memory? Where they repeat at the same distance (streams of one buffer, which may interleave) part by
// part, else by all that lies between their ends.
bool meet(const Tensor& a, const Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  const int64_t delta = static_cast<const char*>(b.const_data_ptr()) - static_cast<const char*>(a.const_data_ptr());
  const int64_t step = a.dim() > 1 && a.size(0) > 1 ? a.stride(0) * static_cast<int64_t>(a.element_size()) : 0;
  if (step > 0 && b.dim() > 1 && b.size(0) > 1 && b.stride(0) * static_cast<int64_t>(b.element_size()) == step) {
    const int64_t from = -reach(b, 1) - delta, below = from / step - (from % step < 0);
    const int64_t k = std::max(below + 1, 1 - a.size(0));      // the first part of b, counted from a's, that ends behind its start
    return k < b.size(0) && delta + k * step < reach(a, 1);
  }
  return delta < reach(a, 0) && -delta < reach(b, 0);
}

// A step writes its states while other threads still read their inputs.
void check_apart(const Tensor& out, std::initializer_list<const Tensor*> inputs, std::initializer_list<const OptTensor*> others) {
  for (const Tensor* t : inputs) TORCH_CHECK(!meet(out, *t), "out overlaps an input other than the state");
  for (const OptTensor* t : others) TORCH_CHECK(!given(*t) || !meet(out, **t), "out overlaps an input other than the state");
}

// What a kernel wrote through a pointer counts as a change of the tensor for autograd too: a backward pass that kept `out`
// as a sequence's state refuses it. (The alias mark of the schema alone does not count.)
void changed(const OptTensor& out) {
  if (given(out)) torch::autograd::impl::bump_version(*out);
}

Tensor new_f32(const Tensor& on, at::IntArrayRef sizes) { return at::empty(sizes, on.options().dtype(at::kFloat)); }
Tensor new_rows(const Tensor& like, at::IntArrayRef sizes) { return at::empty(sizes, like.options()); }

// ---- autograd ----------------------------------------------------------------------------------------
Tensor tensor_of(const OptTensor& t) { return given(t) ? *t : Tensor(); }
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : c10::nullopt; }
OptTensor dense(const Tensor& t) { return t.defined() ? OptTensor(t.contiguous()) : c10::nullopt; }
OptTensor adjacent(const Tensor& t) {
  if (!t.defined()) return c10::nullopt;
  return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }

// A call records a node only if one of these has a gradient.
bool records(std::initializer_list<const Tensor*> tensors, std::initializer_list<const OptTensor*> others) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (wants(*t)) return true;
  for (const OptTensor* t : others)
    if (given(*t) && wants(**t)) return true;
  return false;
}

// There is no forward mode: a tangent would be lost without a word, since the kernels see values only.
void no_tangents(std::initializer_list<const Tensor*> tensors, std::initializer_list<const OptTensor*> others, const char* name) {
  const auto check = [&](const Tensor& t) {
    TORCH_CHECK(!t._fw_grad(/*level=*/0).defined(), name, " has no forward-mode derivative, and an input carries a tangent");
  };
  for (const Tensor* t : tensors) check(*t);
  for (const OptTensor* t : others)
    if (given(*t)) check(**t);
}

// Gradients are not differentiable again: a second derivative that reaches them ends in an error. A backward pass under
// grad mode (create_graph) gives them this node, whose edges are those of everything they depend on - the incoming gradients
// and the inputs, constant as the seed may be - so that no way from a later loss to an input goes around it.
struct NoSecondDerivative : torch::autograd::Node {
  std::string operator_name;
  variable_list apply(variable_list&&) override { TORCH_CHECK(false, operator_name, " has no second derivative"); }
};

variable_list first_derivative(variable_list grads, variable_list incoming, AutogradContext* ctx, const char* name) {
  if (!at::GradMode::is_enabled()) return grads;
  const variable_list inputs = ctx->get_saved_variables();
  incoming.insert(incoming.end(), inputs.begin(), inputs.end());
  const std::shared_ptr<NoSecondDerivative> node(new NoSecondDerivative, torch::autograd::deleteNode);
  node->operator_name = name;
  node->set_next_edges(torch::autograd::collect_next_edges(incoming));
  for (Tensor& t : grads)
    if (t.defined()) {
      t = t.detach();
      torch::autograd::set_history(t, node);
    }
  return grads;
}

int to_int(int64_t v, const char* name) {
  TORCH_CHECK(v >= 0 && v <= 0x7fffffff - 4096, name, ": too large");
  return static_cast<int>(v);
}

// ---- causal convolution ------------------------------------------------------------------------------
// x: [B, T, C], or [B, C] for one row of each
BdhConvDesc conv_desc(const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& state, const OptTensor& lengths,
                      bool silu) {
  const bool one = x.dim() == 2;
  const int64_t B = x.size(0), T = one ? 1 : x.size(1), C = x.size(-1), k = w.size(1);
  BdhConvDesc d{};
  d.dtype = elem_type(x, "x");
  check_rows(x, x, x.scalar_type(), x.sizes(), "x");
  check_dense(w, x, at::kFloat, {C, k}, "w");
  check_f32(bias, x, {C}, "bias");
  d.x = x.const_data_ptr(); d.x_sb = x.stride(0); d.x_st = one ? 0 : x.stride(1);
  d.w = w.const_data_ptr<float>(); d.bias = f32_ptr(bias);
  if (given(state)) {
    check_rows(*state, x, x.scalar_type(), {B, k - 1, C}, "state");
    d.state = state->const_data_ptr(); d.state_sb = state->stride(0); d.state_sr = state->stride(1);
  }
  set_lengths(lengths, x, B, d.lengths, d.lengths64);
  d.B = to_int(B, "B"); d.T = to_int(T, "T"); d.C = to_int(C, "C"); d.k = to_int(k, "k");
  d.silu = silu;
  return d;
}

void set_state_out(BdhConvDesc& d, const Tensor& x, const Tensor& out) {
  check_rows(out, x, x.scalar_type(), {x.size(0), d.k - 1, x.size(-1)}, "state_out");
  d.state_out = out.data_ptr(); d.state_out_sb = out.stride(0); d.state_out_sr = out.stride(1);
}

std::vector<Tensor> causal_conv_fwd(const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& state,
                                    const OptTensor& lengths, bool silu) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 3 && w.dim() == 2, "x: [B, T, C] on a GPU, w: [C, k]");
  c10::cuda::CUDAGuard guard(x.device());
  BdhConvDesc d = conv_desc(x, w, bias, state, lengths, silu);
  Tensor y = new_rows(x, x.sizes()), end = new_rows(x, {d.B, d.k - 1, d.C});
  d.y = y.data_ptr();
  set_state_out(d, x, end);
  check_rc(bdh_causal_conv_fwd(&d, cur_stream()), "causal_conv_fwd");
  return {y, end};
}

// dx, then those of dw, db, dstate that are wanted
std::vector<Tensor> causal_conv_bwd(const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& state, const OptTensor& lengths,
                                    bool silu, const OptTensor& dy, const OptTensor& dstate_out, bool want_w, bool want_bias,
                                    bool want_state) {
  c10::cuda::CUDAGuard guard(x.device());
  TORCH_CHECK(x.dim() == 3 && w.dim() == 2, "x: [B, T, C], w: [C, k]");
  BdhConvDesc d = conv_desc(x, w, bias, state, lengths, silu);
  TORCH_CHECK(d.B > 0 && d.T > 0, "no rows");
  TORCH_CHECK(!want_state || given(state), "state: needed for its gradient");
  const Tensor g = given(dy) ? *dy : at::zeros(x.sizes(), x.options());
  check_rows(g, x, x.scalar_type(), x.sizes(), "dy");
  d.dy = g.const_data_ptr(); d.dy_sb = g.stride(0); d.dy_st = g.stride(1);
  if (given(dstate_out)) {
    check_dense(*dstate_out, x, x.scalar_type(), {d.B, d.k - 1, d.C}, "dstate_out");
    d.dstate_out = dstate_out->const_data_ptr();
  }
  std::vector<Tensor> out{new_rows(x, x.sizes())};
  d.dx = out[0].data_ptr();
  float *dw = nullptr, *db = nullptr;
  if (want_w) dw = out.emplace_back(new_f32(x, w.sizes())).data_ptr<float>();
  if (want_bias) db = out.emplace_back(new_f32(x, {d.C})).data_ptr<float>();
  if (want_state) d.dstate = out.emplace_back(new_rows(x, {d.B, d.k - 1, d.C})).data_ptr();
  Tensor partial;
  if (want_w || want_bias) partial = new_f32(x, {bdh_causal_conv_partials(&d)});
  check_rc(bdh_causal_conv_bwd(&d, dw, db, partial.defined() ? partial.data_ptr<float>() : nullptr, cur_stream()), "causal_conv_bwd");
  return out;
}

struct CausalConv : Function<CausalConv> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& state,
                               const OptTensor& lengths, bool silu) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, w, tensor_of(bias), tensor_of(state), tensor_of(lengths)});
    ctx->saved_data["silu"] = silu;
    ctx->saved_data["want"] = int64_t{wants(w)} | int64_t{wants(tensor_of(bias))} << 1 | int64_t{wants(tensor_of(state))} << 2;
    return causal_conv_fwd(x, w, bias, state, lengths, silu);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(6);                              // x, w, bias, state, lengths, silu
    if (!grads[0].defined() && !grads[1].defined()) return out;
    {
      at::AutoGradMode off(false);
      const variable_list in = ctx->get_saved_variables();
      const int64_t want = ctx->saved_data["want"].toInt();
      if (in[0].size(0) * in[0].size(1) == 0) {        // no rows: the state went through unchanged
        out[0] = at::empty_like(in[0]);
        for (int i = 1; i < 4; ++i)
          if (want >> (i - 1) & 1) out[i] = i == 3 && grads[1].defined() ? grads[1] : at::zeros_like(in[i]);
      } else {
        const std::vector<Tensor> made = causal_conv_bwd(in[0], in[1], opt(in[2]), opt(in[3]), opt(in[4]), ctx->saved_data["silu"].toBool(),
                                                         adjacent(grads[0]), dense(grads[1]), want & 1, want & 2, want & 4);
        size_t at = 0;
        out[0] = made[at++];
        for (int i = 1; i < 4; ++i)
          if (want >> (i - 1) & 1) out[i] = made[at++];
      }
    }
    return first_derivative(std::move(out), std::move(grads), ctx, "causal_conv");
  }
};

std::vector<Tensor> causal_conv(const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& state, const OptTensor& lengths,
                                bool silu) {
  no_tangents({&x, &w}, {&bias, &state}, "causal_conv");
  if (!records({&x, &w}, {&bias, &state})) return causal_conv_fwd(x, w, bias, state, lengths, silu);
  return CausalConv::apply(x, w, bias, state, lengths, silu);
}

// y, and the new state unless it goes to `out`
std::vector<Tensor> causal_conv_step(const Tensor& x, const Tensor& state, const Tensor& w, const OptTensor& bias, const OptTensor& active,
                                     bool silu, const OptTensor& out) {
  c10::cuda::CUDAGuard guard(x.device());
  TORCH_CHECK(x.dim() == 2 && w.dim() == 2, "x: [B, C], w: [C, k]");
  no_tangents({&x, &state, &w}, {&bias, &out}, "causal_conv_step");
  BdhConvDesc d = conv_desc(x, w, bias, state, c10::nullopt, silu);
  std::vector<Tensor> result{new_rows(x, x.sizes())};
  d.y = result[0].data_ptr();
  if (given(out)) check_apart(*out, {&x, &w}, {&bias, &active});
  set_state_out(d, x, given(out) ? *out : result.emplace_back(new_rows(x, state.sizes())));
  check_rc(bdh_causal_conv_step(&d, active_ptr(active, x, x.size(0)), cur_stream()), "causal_conv_step");
  changed(out);
  return result;
}

// ---- per-head norm + rotation ------------------------------------------------------------------------
BdhNormRotateDesc norm_desc(const Tensor& q, const OptTensor& k, const OptTensor& q_weight, const OptTensor& k_weight,
                            const OptTensor& q_bias, const OptTensor& k_bias, const OptTensor& angles, const OptTensor& freqs,
                            const OptTensor& positions, int64_t pos0, const OptTensor& lengths, double eps) {
  TORCH_CHECK(q.dim() == 4, "q: [B, T, heads, Dh]");
  const int64_t B = q.size(0), T = q.size(1), Hq = q.size(2), Dh = q.size(3);
  BdhNormRotateDesc d{};
  d.dtype = elem_type(q, "q");
  check_rows(q, q, q.scalar_type(), q.sizes(), "q");
  d.q = q.const_data_ptr(); d.q_sb = q.stride(0); d.q_st = q.stride(1); d.q_sh = q.stride(2);
  int64_t Hk = 0;
  if (given(k)) {
    TORCH_CHECK(k->dim() == 4, "k: [B, T, heads, Dh]");
    Hk = k->size(2);
    check_rows(*k, q, q.scalar_type(), {B, T, Hk, Dh}, "k");
    d.k = k->const_data_ptr(); d.k_sb = k->stride(0); d.k_st = k->stride(1); d.k_sh = k->stride(2);
  }
  for (const OptTensor* w : {&q_weight, &k_weight, &q_bias, &k_bias})
    if (given(*w) && (*w)->dim() == 2) d.per_head = 1;
  const auto check_param = [&](const OptTensor& t, int64_t heads, const char* name) {
    if (d.per_head) check_f32(t, q, {heads, Dh}, name);
    else check_f32(t, q, {Dh}, name);
    return f32_ptr(t);
  };
  d.q_weight = check_param(q_weight, Hq, "q_weight"); d.q_bias = check_param(q_bias, Hq, "q_bias");
  d.k_weight = check_param(k_weight, Hk, "k_weight"); d.k_bias = check_param(k_bias, Hk, "k_bias");
  int64_t P = 0;
  if (given(angles)) {
    TORCH_CHECK(angles->dim() == 3, "angles: [B, T, pairs]");
    P = angles->size(2);
    check_rows(*angles, q, at::kFloat, {B, T, P}, "angles");
    d.angles = angles->const_data_ptr<float>(); d.ang_sb = angles->stride(0); d.ang_st = angles->stride(1);
  } else if (given(freqs)) {
    TORCH_CHECK(freqs->dim() == 1 && freqs->size(0) % 2 == 0, "freqs: [2 * pairs]");
    check_dense(*freqs, q, at::kFloat, freqs->sizes(), "freqs");
    P = freqs->size(0) / 2;
    d.freqs = freqs->const_data_ptr<float>();
  }
  TORCH_CHECK(2 * P <= Dh, "more rotated channels than a head has");
  d.pos0 = pos0;
  if (given(positions)) {
    TORCH_CHECK(positions->is_cuda() && positions->device() == q.device() && positions->dim() == 2 && positions->size(0) == B &&
                positions->size(1) == T && (positions->scalar_type() == at::kInt || positions->scalar_type() == at::kLong),
                "positions: expected int32 or int64 [B, T] on ", q.device());
    d.positions = positions->const_data_ptr(); d.positions64 = positions->scalar_type() == at::kLong;
    d.pos_sb = positions->stride(0); d.pos_st = positions->stride(1);
  }
  set_lengths(lengths, q, B, d.lengths, d.lengths64);
  d.B = to_int(B, "B"); d.T = to_int(T, "T"); d.Hq = to_int(Hq, "heads"); d.Hk = to_int(Hk, "heads"); d.Dh = to_int(Dh, "Dh");
  d.P = static_cast<int>(P);
  d.eps = static_cast<float>(eps);
  return d;
}

std::vector<Tensor> norm_rotate_fwd(const Tensor& q, const OptTensor& k, const OptTensor& q_weight, const OptTensor& k_weight,
                                    const OptTensor& q_bias, const OptTensor& k_bias, const OptTensor& angles, const OptTensor& freqs,
                                    const OptTensor& positions, int64_t pos0, const OptTensor& lengths, double eps) {
  TORCH_CHECK(q.is_cuda(), "q: expected a tensor on a GPU");
  c10::cuda::CUDAGuard guard(q.device());
  BdhNormRotateDesc d = norm_desc(q, k, q_weight, k_weight, q_bias, k_bias, angles, freqs, positions, pos0, lengths, eps);
  std::vector<Tensor> out{new_rows(q, q.sizes())};
  d.q_out = out[0].data_ptr();
  if (given(k)) d.k_out = out.emplace_back(new_rows(q, k->sizes())).data_ptr();
  check_rc(bdh_norm_rotate_fwd(&d, cur_stream()), "norm_rotate_fwd");
  return out;
}

// dq, dk (with k), then those of q_weight, k_weight, q_bias, k_bias and angles that `want` has a bit for
std::vector<Tensor> norm_rotate_bwd(const Tensor& q, const OptTensor& k, const OptTensor& q_weight, const OptTensor& k_weight,
                                    const OptTensor& q_bias, const OptTensor& k_bias, const OptTensor& angles, const OptTensor& freqs,
                                    const OptTensor& positions, int64_t pos0, const OptTensor& lengths, double eps,
                                    const OptTensor& dq_out, const OptTensor& dk_out, int64_t want) {
  c10::cuda::CUDAGuard guard(q.device());
  BdhNormRotateDesc d = norm_desc(q, k, q_weight, k_weight, q_bias, k_bias, angles, freqs, positions, pos0, lengths, eps);
  TORCH_CHECK(d.B > 0 && d.T > 0, "no rows");
  const auto type = q.scalar_type();
  std::vector<Tensor> out{new_rows(q, q.sizes())};
  d.dq = out[0].data_ptr();
  const Tensor gq = given(dq_out) ? *dq_out : at::zeros(q.sizes(), q.options());
  check_dense(gq, q, type, q.sizes(), "dq_out");
  d.dq_out = gq.const_data_ptr();
  Tensor gk;
  if (given(k)) {
    gk = given(dk_out) ? *dk_out : at::zeros(k->sizes(), q.options());
    check_dense(gk, q, type, k->sizes(), "dk_out");
    d.dk_out = gk.const_data_ptr();
    d.dk = out.emplace_back(new_rows(q, k->sizes())).data_ptr();
  }
  const OptTensor* params[5] = {&q_weight, &k_weight, &q_bias, &k_bias, &angles};
  float* grads[5] = {};
  for (int i = 0; i < 5; ++i)
    if (want >> i & 1) {
      TORCH_CHECK(given(*params[i]), "a gradient is wanted of something that was not given");
      grads[i] = out.emplace_back(new_f32(q, (*params[i])->sizes())).data_ptr<float>();
    }
  const bool bias = grads[2] || grads[3];
  const long long need = bdh_norm_rotate_scratch(&d, bias || grads[0] || grads[1], bias, grads[4] != nullptr);
  Tensor scratch;
  if (need > 0) scratch = new_f32(q, {need});
  check_rc(bdh_norm_rotate_bwd(&d, grads[0], grads[1], grads[2], grads[3], grads[4], need > 0 ? scratch.data_ptr<float>() : nullptr,
                               cur_stream()), "norm_rotate_bwd");
  return out;
}

struct NormRotate : Function<NormRotate> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k, const OptTensor& q_weight, const OptTensor& k_weight,
                               const OptTensor& q_bias, const OptTensor& k_bias, const OptTensor& angles, const OptTensor& freqs,
                               const OptTensor& positions, int64_t pos0, const OptTensor& lengths, double eps) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({q, tensor_of(k), tensor_of(q_weight), tensor_of(k_weight), tensor_of(q_bias), tensor_of(k_bias), tensor_of(angles),
                            tensor_of(freqs), tensor_of(positions), tensor_of(lengths)});
    int64_t want = 0, i = 0;
    for (const OptTensor* t : {&q_weight, &k_weight, &q_bias, &k_bias, &angles}) want |= int64_t{wants(tensor_of(*t))} << i++;
    ctx->saved_data["want"] = want;
    ctx->saved_data["pos0"] = pos0;
    ctx->saved_data["eps"] = eps;
    return norm_rotate_fwd(q, k, q_weight, k_weight, q_bias, k_bias, angles, freqs, positions, pos0, lengths, eps);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(12);                             // in the order of the arguments
    const Tensor dq = grads[0], dk = grads.size() > 1 ? grads[1] : Tensor();
    if (!dq.defined() && !dk.defined()) return out;
    {
      at::AutoGradMode off(false);
      const variable_list in = ctx->get_saved_variables();
      const int64_t want = ctx->saved_data["want"].toInt();
      if (in[0].size(0) * in[0].size(1) == 0) {
        for (int i = 0; i < 7; ++i)
          if (in[i].defined() && (i < 2 || (want >> (i - 2) & 1))) out[i] = at::zeros_like(in[i]);
      } else {
        const std::vector<Tensor> made =
            norm_rotate_bwd(in[0], opt(in[1]), opt(in[2]), opt(in[3]), opt(in[4]), opt(in[5]), opt(in[6]), opt(in[7]), opt(in[8]),
                            ctx->saved_data["pos0"].toInt(), opt(in[9]), ctx->saved_data["eps"].toDouble(), dense(dq), dense(dk), want);
        size_t at = 0;
        for (int i = 0; i < 7; ++i)
          if (i == 0 || (i == 1 && in[1].defined()) || (i > 1 && (want >> (i - 2) & 1))) out[i] = made[at++];
      }
    }
    return first_derivative(std::move(out), std::move(grads), ctx, "norm_rotate");
  }
};

std::vector<Tensor> norm_rotate(const Tensor& q, const OptTensor& k, const OptTensor& q_weight, const OptTensor& k_weight,
                                const OptTensor& q_bias, const OptTensor& k_bias, const OptTensor& angles, const OptTensor& freqs,
                                const OptTensor& positions, int64_t pos0, const OptTensor& lengths, double eps) {
  no_tangents({&q}, {&k, &q_weight, &k_weight, &q_bias, &k_bias, &angles, &freqs}, "norm_rotate");
  if (!records({&q}, {&k, &q_weight, &k_weight, &q_bias, &k_bias, &angles}))
    return norm_rotate_fwd(q, k, q_weight, k_weight, q_bias, k_bias, angles, freqs, positions, pos0, lengths, eps);
  return NormRotate::apply(q, k, q_weight, k_weight, q_bias, k_bias, angles, freqs, positions, pos0, lengths, eps);
}

// ---- selective scan ----------------------------------------------------------------------------------
BdhScanDesc scan_desc(const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& Bm, const Tensor& Cm, const OptTensor& skip,
                      const OptTensor& dt_bias, bool softplus, const OptTensor& h0, const OptTensor& lengths) {
  TORCH_CHECK((u.dim() == 3 || u.dim() == 2) && A.dim() == 2, "u: [B, T, D] (or [B, D] for one row of each), A: [D, N]");
  const bool one = u.dim() == 2;
  const int64_t B = u.size(0), T = one ? 1 : u.size(1), D = u.size(-1), N = A.size(1);
  const auto type = u.scalar_type();
  BdhScanDesc d{};
  d.dtype = elem_type(u, "u");
  check_rows(u, u, type, u.sizes(), "u");
  check_rows(dt, u, type, u.sizes(), "dt");
  for (const Tensor* t : {&Bm, &Cm}) {
    if (one) check_rows(*t, u, type, {B, N}, "B, C");
    else check_rows(*t, u, type, {B, T, N}, "B, C");
  }
  check_dense(A, u, at::kFloat, {D, N}, "A");
  check_f32(skip, u, {D}, "D");
  check_f32(dt_bias, u, {D}, "dt_bias");
  check_f32(h0, u, {B, D, N}, "h0");
  d.u = u.const_data_ptr(); d.u_sb = u.stride(0); d.u_st = one ? 0 : u.stride(1);
  d.dt = dt.const_data_ptr(); d.dt_sb = dt.stride(0); d.dt_st = one ? 0 : dt.stride(1);
  d.B_ = Bm.const_data_ptr(); d.b_sb = Bm.stride(0); d.b_st = one ? 0 : Bm.stride(1);
  d.C_ = Cm.const_data_ptr(); d.c_sb = Cm.stride(0); d.c_st = one ? 0 : Cm.stride(1);
  d.A = A.const_data_ptr<float>(); d.skip = f32_ptr(skip); d.dt_bias = f32_ptr(dt_bias); d.h0 = f32_ptr(h0);
  set_lengths(lengths, u, B, d.lengths, d.lengths64);
  d.B = to_int(B, "B"); d.T = to_int(T, "T"); d.D = to_int(D, "D"); d.N = to_int(N, "N");
  d.softplus = softplus;
  return d;
}

// y, hT and, for a backward pass (train), the states at the tiles' starts
std::vector<Tensor> selective_scan_fwd(const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& Bm, const Tensor& Cm,
                                       const OptTensor& skip, const OptTensor& dt_bias, bool softplus, const OptTensor& h0,
                                       const OptTensor& lengths, bool train) {
  TORCH_CHECK(u.is_cuda() && u.dim() == 3, "u: [B, T, D] on a GPU");
  c10::cuda::CUDAGuard guard(u.device());
  BdhScanDesc d = scan_desc(u, dt, A, Bm, Cm, skip, dt_bias, softplus, h0, lengths);
  long long n_marks, n_fwd, n_bwd;
  bdh_selective_scan_sizes(&d, &n_marks, &n_fwd, &n_bwd);
  std::vector<Tensor> out{new_rows(u, u.sizes()), new_f32(u, {d.B, d.D, d.N})};
  d.y = out[0].data_ptr(); d.hT = out[1].data_ptr<float>();
  float* marks = train ? out.emplace_back(new_f32(u, {n_marks})).data_ptr<float>() : nullptr;
  Tensor scratch;
  if (n_fwd > 0) scratch = new_f32(u, {n_fwd});
  check_rc(bdh_selective_scan_fwd(&d, marks, n_fwd > 0 ? scratch.data_ptr<float>() : nullptr, cur_stream()), "selective_scan_fwd");
  return out;
}

// du, ddt, dA, dB, dC, then dD and ddt_bias where these were given and dh0 where it is wanted
std::vector<Tensor> selective_scan_bwd(const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& Bm, const Tensor& Cm,
                                       const OptTensor& skip, const OptTensor& dt_bias, bool softplus, const OptTensor& h0,
                                       const OptTensor& lengths, const Tensor& marks, const OptTensor& dy, const OptTensor& dhT,
                                       bool want_h0) {
  c10::cuda::CUDAGuard guard(u.device());
  TORCH_CHECK(u.dim() == 3, "u: [B, T, D]");
  BdhScanDesc d = scan_desc(u, dt, A, Bm, Cm, skip, dt_bias, softplus, h0, lengths);
  TORCH_CHECK(d.B > 0 && d.T > 0, "no rows");
  const auto type = u.scalar_type();
  const Tensor g = given(dy) ? *dy : at::zeros(u.sizes(), u.options());
  check_rows(g, u, type, u.sizes(), "dy");
  check_f32(dhT, u, {d.B, d.D, d.N}, "dhT");
  long long n_marks, n_fwd, n_bwd;
  bdh_selective_scan_sizes(&d, &n_marks, &n_fwd, &n_bwd);
  check_dense(marks, u, at::kFloat, {n_marks}, "marks");
  std::vector<Tensor> out{new_rows(u, u.sizes()), new_rows(u, u.sizes()), new_f32(u, A.sizes()), new_rows(u, Bm.sizes()), new_rows(u, Cm.sizes())};
  float* dD = given(skip) ? out.emplace_back(new_f32(u, {d.D})).data_ptr<float>() : nullptr;
  float* dbias = given(dt_bias) ? out.emplace_back(new_f32(u, {d.D})).data_ptr<float>() : nullptr;
  d.dh0 = want_h0 ? out.emplace_back(new_f32(u, {d.B, d.D, d.N})).data_ptr<float>() : nullptr;
  d.dy = g.const_data_ptr(); d.dy_sb = g.stride(0); d.dy_st = g.stride(1);
  d.du = out[0].data_ptr(); d.ddt = out[1].data_ptr(); d.dhT = f32_ptr(dhT);
  Tensor scratch = new_f32(u, {n_bwd});
  check_rc(bdh_selective_scan_bwd(&d, marks.const_data_ptr<float>(), scratch.data_ptr<float>(), out[2].data_ptr<float>(), dD, dbias,
                                  out[3].data_ptr(), out[4].data_ptr(), cur_stream()), "selective_scan_bwd");
  return out;
}

// Kept for the backward pass: the inputs and the states at every 16th step (fp32).
struct SelectiveScan : Function<SelectiveScan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& Bm, const Tensor& Cm,
                               const OptTensor& skip, const OptTensor& dt_bias, bool softplus, const OptTensor& h0, const OptTensor& lengths) {
    ctx->set_materialize_grads(false);
    std::vector<Tensor> made = selective_scan_fwd(u, dt, A, Bm, Cm, skip, dt_bias, softplus, h0, lengths, true);
    ctx->save_for_backward({u, dt, A, Bm, Cm, tensor_of(skip), tensor_of(dt_bias), tensor_of(h0), tensor_of(lengths), made[2]});
    ctx->saved_data["softplus"] = softplus;
    ctx->saved_data["want_h0"] = wants(tensor_of(h0));
    made.pop_back();
    return made;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(10);                             // in the order of the arguments
    if (!grads[0].defined() && !grads[1].defined()) return out;
    {
      at::AutoGradMode off(false);
      const variable_list in = ctx->get_saved_variables();
      const bool want_h0 = ctx->saved_data["want_h0"].toBool();
      const std::vector<Tensor> made =
          selective_scan_bwd(in[0], in[1], in[2], in[3], in[4], opt(in[5]), opt(in[6]), ctx->saved_data["softplus"].toBool(), opt(in[7]),
                             opt(in[8]), in[9], adjacent(grads[0]), dense(grads[1]), want_h0);
      size_t at = 0;
      for (int i = 0; i < 7; ++i)
        if (in[i].defined()) out[i] = made[at++];
      if (want_h0) out[8] = made[at];
    }
    return first_derivative(std::move(out), std::move(grads), ctx, "selective_scan");
  }
};

std::vector<Tensor> selective_scan(const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& Bm, const Tensor& Cm,
                                   const OptTensor& skip, const OptTensor& dt_bias, bool softplus, const OptTensor& h0,
                                   const OptTensor& lengths) {
  no_tangents({&u, &dt, &A, &Bm, &Cm}, {&skip, &dt_bias, &h0}, "selective_scan");
  if (!records({&u, &dt, &A, &Bm, &Cm}, {&skip, &dt_bias, &h0}))
    return selective_scan_fwd(u, dt, A, Bm, Cm, skip, dt_bias, softplus, h0, lengths, false);
  return SelectiveScan::apply(u, dt, A, Bm, Cm, skip, dt_bias, softplus, h0, lengths);
}

// y, and the new state unless it goes to `out`
std::vector<Tensor> selective_scan_step(const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& Bm, const Tensor& Cm, const Tensor& h,
                                        const OptTensor& skip, const OptTensor& dt_bias, bool softplus, const OptTensor& active,
                                        const OptTensor& out) {
  c10::cuda::CUDAGuard guard(u.device());
  TORCH_CHECK(u.dim() == 2 && dt.dim() == 2 && Bm.dim() == 2 && Cm.dim() == 2, "u, dt: [B, D], B, C: [B, N]");
  no_tangents({&u, &dt, &A, &Bm, &Cm, &h}, {&skip, &dt_bias, &out}, "selective_scan_step");
  BdhScanDesc d = scan_desc(u, dt, A, Bm, Cm, skip, dt_bias, softplus, c10::nullopt, c10::nullopt);
  std::vector<Tensor> result{new_rows(u, u.sizes())};
  d.y = result[0].data_ptr();
  if (given(out)) check_apart(*out, {&u, &dt, &A, &Bm, &Cm}, {&skip, &dt_bias, &active});
  const Tensor to = given(out) ? *out : result.emplace_back(new_f32(u, {d.B, d.D, d.N}));
  for (const Tensor* t : {&h, &to}) {
    check_rows(*t, u, at::kFloat, {d.B, d.D, d.N}, "h");
    TORCH_CHECK(d.D == 1 || t->stride(1) == d.N, "h: expected dense [D, N] states");
  }
  check_rc(bdh_selective_scan_step(&d, h.const_data_ptr<float>(), h.stride(0), to.data_ptr<float>(), to.stride(0),
                                   active_ptr(active, u, d.B), cur_stream()), "selective_scan_step");
  changed(out);
  return result;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(bdh, m) {
  m.def("causal_conv(Tensor x, Tensor w, Tensor? bias, Tensor? state, Tensor? lengths, bool silu) -> Tensor[]");
  m.def("causal_conv_step(Tensor x, Tensor state, Tensor w, Tensor? bias, Tensor? active, bool silu, Tensor(a!)? out) -> Tensor[]");
  m.def("norm_rotate(Tensor q, Tensor? k, Tensor? q_weight, Tensor? k_weight, Tensor? q_bias, Tensor? k_bias, Tensor? angles, "
        "Tensor? freqs, Tensor? positions, int pos0, Tensor? lengths, float eps) -> Tensor[]");
  m.def("selective_scan(Tensor u, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor? D, Tensor? dt_bias, bool softplus, Tensor? h0, "
        "Tensor? lengths) -> Tensor[]");
  m.def("selective_scan_step(Tensor u, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor h, Tensor? D, Tensor? dt_bias, bool softplus, "
        "Tensor? active, Tensor(a!)? out) -> Tensor[]");
}

TORCH_LIBRARY_IMPL(bdh, CUDA, m) {
  m.impl("causal_conv_step", &causal_conv_step);
  m.impl("selective_scan_step", &selective_scan_step);
}

// (these record their own nodes)
TORCH_LIBRARY_IMPL(bdh, CompositeImplicitAutograd, m) {
  m.impl("causal_conv", &causal_conv);
  m.impl("norm_rotate", &norm_rotate);
  m.impl("selective_scan", &selective_scan);
}
