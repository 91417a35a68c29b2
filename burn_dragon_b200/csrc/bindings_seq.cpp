// torch.ops.bdh.* of the parts of a state-space layer (causal convolution, per-head norm + rotation, selective
// scan). As in bindings.cpp the caller allocates every output and all scratch; shapes that the kernels rely on are
// checked here once more, so that a direct call cannot make them read or write out of range.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include "bdh_kernels.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

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
float* f32_out(const OptTensor& t) { return given(t) ? t->data_ptr<float>() : nullptr; }

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

void causal_conv_fwd(const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& state, const OptTensor& lengths,
                     bool silu, Tensor& y, Tensor& state_out) {
  c10::cuda::CUDAGuard guard(x.device());
  TORCH_CHECK(x.dim() == 3 && w.dim() == 2, "x: [B, T, C], w: [C, k]");
  BdhConvDesc d = conv_desc(x, w, bias, state, lengths, silu);
  check_dense(y, x, x.scalar_type(), x.sizes(), "y");
  d.y = y.data_ptr();
  set_state_out(d, x, state_out);
  check_rc(bdh_causal_conv_fwd(&d, cur_stream()), "causal_conv_fwd");
}

int64_t causal_conv_partials(int64_t B, int64_t T, int64_t C, int64_t k) {
  BdhConvDesc d{};
  d.B = to_int(B, "B"); d.T = to_int(T, "T"); d.C = to_int(C, "C"); d.k = to_int(k, "k");
  return bdh_causal_conv_partials(&d);
}

void causal_conv_bwd(const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& state, const OptTensor& lengths,
                     bool silu, const Tensor& dy, const OptTensor& dstate_out, Tensor& dx, const OptTensor& dstate,
                     const OptTensor& dw, const OptTensor& db, const OptTensor& partial) {
  c10::cuda::CUDAGuard guard(x.device());
  TORCH_CHECK(x.dim() == 3 && w.dim() == 2, "x: [B, T, C], w: [C, k]");
  BdhConvDesc d = conv_desc(x, w, bias, state, lengths, silu);
  const int64_t B = x.size(0), C = x.size(2);
  check_rows(dy, x, x.scalar_type(), x.sizes(), "dy");
  d.dy = dy.const_data_ptr(); d.dy_sb = dy.stride(0); d.dy_st = dy.stride(1);
  check_dense(dx, x, x.scalar_type(), x.sizes(), "dx");
  d.dx = dx.data_ptr();
  if (given(dstate_out)) {
    check_dense(*dstate_out, x, x.scalar_type(), {B, d.k - 1, C}, "dstate_out");
    d.dstate_out = dstate_out->const_data_ptr();
  }
  if (given(dstate)) {
    check_dense(*dstate, x, x.scalar_type(), {B, d.k - 1, C}, "dstate");
    d.dstate = dstate->data_ptr();
  }
  check_f32(dw, x, {C, d.k}, "dw");
  check_f32(db, x, {C}, "db");
  if (given(dw) || given(db)) {
    TORCH_CHECK(given(partial), "partial: needed for dw and db");
    check_f32(partial, x, {partial->size(0)}, "partial");
    TORCH_CHECK(partial->size(0) >= bdh_causal_conv_partials(&d), "partial: too small");
  }
  check_rc(bdh_causal_conv_bwd(&d, f32_out(dw), f32_out(db), f32_out(partial), cur_stream()), "causal_conv_bwd");
}

void causal_conv_step(const Tensor& x, const Tensor& state, const Tensor& w, const OptTensor& bias, const OptTensor& active, bool silu,
                      Tensor& y, Tensor& state_out) {
  c10::cuda::CUDAGuard guard(x.device());
  TORCH_CHECK(x.dim() == 2 && w.dim() == 2, "x: [B, C], w: [C, k]");
  BdhConvDesc d = conv_desc(x, w, bias, state, c10::nullopt, silu);
  check_dense(y, x, x.scalar_type(), x.sizes(), "y");
  d.y = y.data_ptr();
  set_state_out(d, x, state_out);
  check_rc(bdh_causal_conv_step(&d, active_ptr(active, x, x.size(0)), cur_stream()), "causal_conv_step");
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

void norm_rotate_fwd(const Tensor& q, const OptTensor& k, const OptTensor& q_weight, const OptTensor& k_weight, const OptTensor& q_bias,
                     const OptTensor& k_bias, const OptTensor& angles, const OptTensor& freqs, const OptTensor& positions,
                     int64_t pos0, const OptTensor& lengths, double eps, Tensor& q_out, const OptTensor& k_out) {
  c10::cuda::CUDAGuard guard(q.device());
  BdhNormRotateDesc d = norm_desc(q, k, q_weight, k_weight, q_bias, k_bias, angles, freqs, positions, pos0, lengths, eps);
  check_dense(q_out, q, q.scalar_type(), q.sizes(), "q_out");
  d.q_out = q_out.data_ptr();
  if (given(k)) {
    TORCH_CHECK(given(k_out), "k_out: needed");
    check_dense(*k_out, q, q.scalar_type(), k->sizes(), "k_out");
    d.k_out = k_out->data_ptr();
  }
  check_rc(bdh_norm_rotate_fwd(&d, cur_stream()), "norm_rotate_fwd");
}

int64_t norm_rotate_scratch(int64_t B, int64_t T, int64_t Hq, int64_t Hk, int64_t Dh, int64_t P, bool per_head, bool want_weight,
                            bool want_bias, bool want_angles) {
  BdhNormRotateDesc d{};
  d.B = to_int(B, "B"); d.T = to_int(T, "T"); d.Hq = to_int(Hq, "heads"); d.Hk = to_int(Hk, "heads"); d.Dh = to_int(Dh, "Dh");
  d.P = to_int(P, "pairs"); d.per_head = per_head;
  return bdh_norm_rotate_scratch(&d, want_weight, want_bias, want_angles);
}

void norm_rotate_bwd(const Tensor& q, const OptTensor& k, const OptTensor& q_weight, const OptTensor& k_weight, const OptTensor& q_bias,
                     const OptTensor& k_bias, const OptTensor& angles, const OptTensor& freqs, const OptTensor& positions,
                     int64_t pos0, const OptTensor& lengths, double eps, const Tensor& dq_out, const OptTensor& dk_out, Tensor& dq,
                     const OptTensor& dk, const OptTensor& dq_weight, const OptTensor& dk_weight, const OptTensor& dq_bias,
                     const OptTensor& dk_bias, const OptTensor& dangles, const OptTensor& scratch) {
  c10::cuda::CUDAGuard guard(q.device());
  BdhNormRotateDesc d = norm_desc(q, k, q_weight, k_weight, q_bias, k_bias, angles, freqs, positions, pos0, lengths, eps);
  const auto type = q.scalar_type();
  check_dense(dq_out, q, type, q.sizes(), "dq_out");
  check_dense(dq, q, type, q.sizes(), "dq");
  d.dq_out = dq_out.const_data_ptr(); d.dq = dq.data_ptr();
  if (given(k)) {
    TORCH_CHECK(given(dk_out) && given(dk), "dk_out, dk: needed");
    check_dense(*dk_out, q, type, k->sizes(), "dk_out");
    check_dense(*dk, q, type, k->sizes(), "dk");
    d.dk_out = dk_out->const_data_ptr(); d.dk = dk->data_ptr();
  }
  const auto check_grad = [&](const OptTensor& t, int64_t heads, const char* name) {
    if (d.per_head) check_f32(t, q, {heads, d.Dh}, name);
    else check_f32(t, q, {d.Dh}, name);
    return f32_out(t);
  };
  float* gqw = check_grad(dq_weight, d.Hq, "dq_weight");
  float* gkw = check_grad(dk_weight, d.Hk, "dk_weight");
  float* gqb = check_grad(dq_bias, d.Hq, "dq_bias");
  float* gkb = check_grad(dk_bias, d.Hk, "dk_bias");
  check_f32(dangles, q, {d.B, d.T, d.P}, "dangles");
  const long long need = bdh_norm_rotate_scratch(&d, gqw || gkw || gqb || gkb, gqb || gkb, given(dangles));
  if (need > 0) {
    TORCH_CHECK(given(scratch) && scratch->numel() >= need, "scratch: too small");
    check_f32(scratch, q, {scratch->numel()}, "scratch");
  }
  check_rc(bdh_norm_rotate_bwd(&d, gqw, gkw, gqb, gkb, f32_out(dangles), f32_out(scratch), cur_stream()), "norm_rotate_bwd");
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

std::tuple<int64_t, int64_t, int64_t> selective_scan_sizes(int64_t B, int64_t T, int64_t D, int64_t N) {
  BdhScanDesc d{};
  d.B = to_int(B, "B"); d.T = to_int(T, "T"); d.D = to_int(D, "D"); d.N = to_int(N, "N");
  long long marks, fwd, bwd;
  bdh_selective_scan_sizes(&d, &marks, &fwd, &bwd);
  return {marks, fwd, bwd};
}

float* scratch_of(const OptTensor& t, const Tensor& on, long long need, const char* name) {
  if (need <= 0) return nullptr;
  TORCH_CHECK(given(t) && t->numel() >= need, name, ": too small");
  check_f32(t, on, {t->numel()}, name);
  return t->data_ptr<float>();
}

void selective_scan_fwd(const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& Bm, const Tensor& Cm, const OptTensor& skip,
                        const OptTensor& dt_bias, bool softplus, const OptTensor& h0, const OptTensor& lengths, Tensor& y, Tensor& hT,
                        const OptTensor& marks, const OptTensor& scratch) {
  c10::cuda::CUDAGuard guard(u.device());
  TORCH_CHECK(u.dim() == 3, "u: [B, T, D]");
  BdhScanDesc d = scan_desc(u, dt, A, Bm, Cm, skip, dt_bias, softplus, h0, lengths);
  check_dense(y, u, u.scalar_type(), u.sizes(), "y");
  check_dense(hT, u, at::kFloat, {d.B, d.D, d.N}, "hT");
  d.y = y.data_ptr(); d.hT = hT.data_ptr<float>();
  long long n_marks, n_fwd, n_bwd;
  bdh_selective_scan_sizes(&d, &n_marks, &n_fwd, &n_bwd);
  float* m = given(marks) ? scratch_of(marks, u, n_marks, "marks") : nullptr;
  check_rc(bdh_selective_scan_fwd(&d, m, scratch_of(scratch, u, n_fwd, "scratch"), cur_stream()), "selective_scan_fwd");
}

void selective_scan_bwd(const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& Bm, const Tensor& Cm, const OptTensor& skip,
                        const OptTensor& dt_bias, bool softplus, const OptTensor& h0, const OptTensor& lengths, const Tensor& marks,
                        const Tensor& scratch, const Tensor& dy, const OptTensor& dhT, Tensor& du, Tensor& ddt, Tensor& dA, Tensor& dB,
                        Tensor& dC, const OptTensor& dskip, const OptTensor& ddt_bias, const OptTensor& dh0) {
  c10::cuda::CUDAGuard guard(u.device());
  TORCH_CHECK(u.dim() == 3, "u: [B, T, D]");
  BdhScanDesc d = scan_desc(u, dt, A, Bm, Cm, skip, dt_bias, softplus, h0, lengths);
  const auto type = u.scalar_type();
  check_rows(dy, u, type, u.sizes(), "dy");
  check_dense(du, u, type, u.sizes(), "du");
  check_dense(ddt, u, type, u.sizes(), "ddt");
  check_dense(dA, u, at::kFloat, A.sizes(), "dA");
  check_dense(dB, u, type, Bm.sizes(), "dB");
  check_dense(dC, u, type, Cm.sizes(), "dC");
  check_f32(dskip, u, {d.D}, "dD");
  check_f32(ddt_bias, u, {d.D}, "ddt_bias");
  check_f32(dhT, u, {d.B, d.D, d.N}, "dhT");
  check_f32(dh0, u, {d.B, d.D, d.N}, "dh0");
  d.dy = dy.const_data_ptr(); d.dy_sb = dy.stride(0); d.dy_st = dy.stride(1);
  d.du = du.data_ptr(); d.ddt = ddt.data_ptr(); d.dhT = f32_ptr(dhT); d.dh0 = f32_out(dh0);
  long long n_marks, n_fwd, n_bwd;
  bdh_selective_scan_sizes(&d, &n_marks, &n_fwd, &n_bwd);
  const float* m = scratch_of(marks, u, n_marks, "marks");
  check_rc(bdh_selective_scan_bwd(&d, m, scratch_of(scratch, u, n_bwd, "scratch"), dA.data_ptr<float>(), f32_out(dskip), f32_out(ddt_bias),
                                  dB.data_ptr(), dC.data_ptr(), cur_stream()), "selective_scan_bwd");
}

void selective_scan_step(const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& Bm, const Tensor& Cm, const Tensor& h,
                         const OptTensor& skip, const OptTensor& dt_bias, bool softplus, const OptTensor& active, Tensor& y, Tensor& out) {
  c10::cuda::CUDAGuard guard(u.device());
  TORCH_CHECK(u.dim() == 2 && dt.dim() == 2 && Bm.dim() == 2 && Cm.dim() == 2, "u, dt: [B, D], B, C: [B, N]");
  BdhScanDesc d = scan_desc(u, dt, A, Bm, Cm, skip, dt_bias, softplus, c10::nullopt, c10::nullopt);
  check_dense(y, u, u.scalar_type(), u.sizes(), "y");
  d.y = y.data_ptr();
  for (const Tensor* t : {&h, static_cast<const Tensor*>(&out)}) {
    check_rows(*t, u, at::kFloat, {d.B, d.D, d.N}, "h");
    TORCH_CHECK(d.D == 1 || t->stride(1) == d.N, "h: expected dense [D, N] states");
  }
  check_rc(bdh_selective_scan_step(&d, h.const_data_ptr<float>(), h.stride(0), out.data_ptr<float>(), out.stride(0),
                                   active_ptr(active, u, d.B), cur_stream()), "selective_scan_step");
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(bdh, m) {
  m.def("causal_conv_fwd(Tensor x, Tensor w, Tensor? bias, Tensor? state, Tensor? lengths, bool silu, Tensor(a!) y, "
        "Tensor(b!) state_out) -> ()");
  m.def("causal_conv_partials(int B, int T, int C, int k) -> int");
  m.def("causal_conv_bwd(Tensor x, Tensor w, Tensor? bias, Tensor? state, Tensor? lengths, bool silu, Tensor dy, "
        "Tensor? dstate_out, Tensor(a!) dx, Tensor(b!)? dstate, Tensor(c!)? dw, Tensor(d!)? db, Tensor(e!)? partial) -> ()");
  m.def("causal_conv_step(Tensor x, Tensor state, Tensor w, Tensor? bias, Tensor? active, bool silu, Tensor(a!) y, "
        "Tensor(b!) state_out) -> ()");
  m.def("norm_rotate_fwd(Tensor q, Tensor? k, Tensor? q_weight, Tensor? k_weight, Tensor? q_bias, Tensor? k_bias, Tensor? angles, "
        "Tensor? freqs, Tensor? positions, int pos0, Tensor? lengths, float eps, Tensor(a!) q_out, Tensor(b!)? k_out) -> ()");
  m.def("norm_rotate_scratch(int B, int T, int Hq, int Hk, int Dh, int P, bool per_head, bool want_weight, bool want_bias, "
        "bool want_angles) -> int");
  m.def("norm_rotate_bwd(Tensor q, Tensor? k, Tensor? q_weight, Tensor? k_weight, Tensor? q_bias, Tensor? k_bias, Tensor? angles, "
        "Tensor? freqs, Tensor? positions, int pos0, Tensor? lengths, float eps, Tensor dq_out, Tensor? dk_out, Tensor(a!) dq, "
        "Tensor(b!)? dk, Tensor(c!)? dq_weight, Tensor(d!)? dk_weight, Tensor(e!)? dq_bias, Tensor(f!)? dk_bias, "
        "Tensor(g!)? dangles, Tensor(h!)? scratch) -> ()");
  m.def("selective_scan_sizes(int B, int T, int D, int N) -> (int, int, int)");
  m.def("selective_scan_fwd(Tensor u, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor? D, Tensor? dt_bias, bool softplus, Tensor? h0, "
        "Tensor? lengths, Tensor(a!) y, Tensor(b!) hT, Tensor(c!)? marks, Tensor(d!)? scratch) -> ()");
  m.def("selective_scan_bwd(Tensor u, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor? D, Tensor? dt_bias, bool softplus, Tensor? h0, "
        "Tensor? lengths, Tensor marks, Tensor(a!) scratch, Tensor dy, Tensor? dhT, Tensor(b!) du, Tensor(c!) ddt, Tensor(d!) dA, "
        "Tensor(e!) dB, Tensor(f!) dC, Tensor(g!)? dD, Tensor(h!)? ddt_bias, Tensor(i!)? dh0) -> ()");
  m.def("selective_scan_step(Tensor u, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor h, Tensor? D, Tensor? dt_bias, bool softplus, "
        "Tensor? active, Tensor(a!) y, Tensor(b!) out) -> ()");
}

TORCH_LIBRARY_IMPL(bdh, CUDA, m) {
  m.impl("selective_scan_fwd", &selective_scan_fwd);
  m.impl("selective_scan_bwd", &selective_scan_bwd);
  m.impl("selective_scan_step", &selective_scan_step);
  m.impl("norm_rotate_fwd", &norm_rotate_fwd);
  m.impl("norm_rotate_bwd", &norm_rotate_bwd);
  m.impl("causal_conv_fwd", &causal_conv_fwd);
  m.impl("causal_conv_bwd", &causal_conv_bwd);
  m.impl("causal_conv_step", &causal_conv_step);
}
TORCH_LIBRARY_IMPL(bdh, CompositeExplicitAutograd, m) {
  m.impl("causal_conv_partials", &causal_conv_partials);
  m.impl("norm_rotate_scratch", &norm_rotate_scratch);
  m.impl("selective_scan_sizes", &selective_scan_sizes);
}
