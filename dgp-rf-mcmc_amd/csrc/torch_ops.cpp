// torch_ops.cpp — the hot-path entry points of libdgprf.so registered as PyTorch operators
// (TORCH_LIBRARY(dgprf, m)), so torch's dispatcher, its current HIP stream and torch.cuda.graph
// capture see the work.  Each op validates its tensors (device, dtype, contiguity, sizes against the
// plan), assembles the C-ABI structs of include/dgprf.h and calls the extern "C" entry point on the
// current HIP stream.  The plan travels as a CPU uint8 tensor holding a dgprf_plan_t filled by
// dgprf_plan_init (dgprf/_native.py make_plan), i.e. the model shape of DGP_RF.__init__
// (models/dgp.py:9-115).
//
//   dgprf::sghmc_step_     DGP_RF.sgmcmc_update            models/dgp.py:184-216
//   dgprf::potential_grad  U + tape.gradient               models/dgp.py:161-182, 194-204
//   dgprf::forward         BNN(X) + eval_log_likelihood(_and_se) + online LSE fold
//                          utils.py:10-44, models/regression_model.py:33-50,
//                          experiments/utils_training.py:63-65
//   dgprf::lse_finalize    experiments/utils_training.py:79-85
//   dgprf::linear, dropout the dense operators (include/dgprf.h), differentiable: every size, type and
//                          stride is checked here, before anything is enqueued
#include <cmath>
#include <cstring>
#include <string>
#include <unordered_set>
#include <vector>

#include <ATen/ops/add.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/library.h>

#include "../../include/dgprf.h"

namespace {

using at::Tensor;
using OptT = std::optional<Tensor>;

void check_rc(int rc, const char* fn) {
  if (rc == DGPRF_OK) return;
  if (rc == DGPRF_E_SHAPE) TORCH_CHECK_VALUE(false, fn, ": unsupported shape (", dgprf_error_string(rc), ")");
  TORCH_CHECK(false, fn, " failed: ", dgprf_error_string(rc), " (code ", rc, ")");
}

dgprf_plan_t plan_of(const Tensor& p) {
  TORCH_CHECK(p.device().is_cpu() && p.scalar_type() == at::kByte && p.is_contiguous() &&
                  p.numel() == (int64_t)sizeof(dgprf_plan_t),
              "dgprf: plan must be a CPU uint8 tensor of sizeof(dgprf_plan_t) bytes");
  dgprf_plan_t pl;
  std::memcpy(&pl, p.data_ptr(), sizeof(pl));
  TORCH_CHECK(pl.initialised == 1, "dgprf: plan not initialised (dgprf_plan_init)");
  return pl;
}

void* stream() { return c10::hip::getCurrentHIPStream().stream(); }

// device fp32 contiguous with at least `n` elements (n < 0: any size)
float* f32(const Tensor& t, const char* what, int64_t n = -1) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kFloat && t.is_contiguous(), "dgprf: ", what,
              " must be a contiguous float32 HIP tensor");
  TORCH_CHECK(n < 0 || t.numel() >= n, "dgprf: ", what, " has ", t.numel(), " elements, needs ", n);
  return t.data_ptr<float>();
}
float* f32o(const OptT& t, const char* what, int64_t n = -1) {
  return t.has_value() && t->defined() ? f32(*t, what, n) : nullptr;
}

dgprf_batch_t batch_of(const dgprf_plan_t& pl, const Tensor& X, const Tensor& Y, int64_t mode,
                       int64_t iters, int64_t perm_seed, const OptT& idx) {
  TORCH_CHECK(X.dim() == 2 && X.size(1) == pl.d_in, "dgprf: X must be [n, d_in]");
  TORCH_CHECK(Y.dim() == 2 && Y.size(0) == X.size(0), "dgprf: Y must be [n, y_cols]");
  dgprf_batch_t b;
  std::memset(&b, 0, sizeof(b));  // A1 = NULL: eager calls run the A_1 GEMM
  b.X = f32(X, "X");
  b.Y = f32(Y, "Y");
  b.n_data = X.size(0);
  b.y_cols = (int32_t)Y.size(1);
  b.mode = (int32_t)mode;
  b.iters_per_epoch = iters;
  b.perm_seed = (uint64_t)perm_seed;
  if (idx.has_value() && idx->defined()) {
    TORCH_CHECK(idx->is_cuda() && idx->scalar_type() == at::kInt && idx->is_contiguous() &&
                    idx->numel() >= (int64_t)pl.n_chains * pl.batch,
                "dgprf: idx must be int32 [C, B] on the device");
    b.idx = idx->data_ptr<int32_t>();
  }
  return b;
}

dgprf_chain_t chain_of(const dgprf_plan_t& pl, const Tensor& theta, const Tensor& mom,
                       const Tensor& omega, const Tensor& der, const Tensor& mass,
                       const Tensor& ws, const Tensor& step, int64_t seed, const OptT& z,
                       const OptT& hyp, const OptT& hmom, const OptT& hmass) {
  const int64_t C = pl.n_chains, ch = pl.hyp_per_chain ? C : 1;
  dgprf_chain_t c;
  std::memset(&c, 0, sizeof(c));
  c.theta = f32(theta, "theta", C * pl.w_total);
  c.mom = f32(mom, "mom", C * pl.w_total);
  c.omega = f32(omega, "omega", ch * pl.omega_total);
  c.der = f32(der, "der", ch * pl.der_total);
  c.mass = f32(mass, "mass", C * pl.n_layers);
  c.ws = f32(ws, "ws", pl.ws_total);
  TORCH_CHECK(step.is_cuda() && step.scalar_type() == at::kLong && step.numel() >= 1,
              "dgprf: step must be an int64 HIP tensor");
  c.step = step.data_ptr<int64_t>();
  c.seed = (uint64_t)seed;
  c.z = f32o(z, "z", pl.omega_total);
  c.hyp = f32o(hyp, "hyp", ch * pl.hyp_total);
  c.hmom = f32o(hmom, "hmom", C * pl.hyp_total);
  c.hmass = f32o(hmass, "hmass", C * DGPRF_HMASS);
  return c;
}

void sghmc_step_(const Tensor& plan, const Tensor& theta, const Tensor& mom, const Tensor& omega,
                 const Tensor& der, const Tensor& mass, const Tensor& ws, const Tensor& step,
                 int64_t seed, const Tensor& X, const Tensor& Y, int64_t mode, int64_t iters,
                 int64_t perm_seed, const OptT& idx, double lr, double momentum_decay,
                 double temperature, double data_size, bool resample, const OptT& xi,
                 const OptT& xi_resample, bool full_bayes, const OptT& z, const OptT& hyp,
                 const OptT& hmom, const OptT& hmass, const OptT& xi_hyp,
                 const OptT& xi_hyp_resample) {
  const dgprf_plan_t pl = plan_of(plan);
  const dgprf_chain_t c = chain_of(pl, theta, mom, omega, der, mass, ws, step, seed, z, hyp, hmom, hmass);
  const dgprf_batch_t b = batch_of(pl, X, Y, mode, iters, perm_seed, idx);
  dgprf_step_t st;
  std::memset(&st, 0, sizeof(st));
  st.lr = (float)lr;
  st.momentum_decay = (float)momentum_decay;
  st.temperature = (float)temperature;
  st.data_size = (float)data_size;
  st.resample_moments = resample ? 1 : 0;
  st.schedule = DGPRF_SCHED_CONST;
  st.cycle_length = 1;
  st.full_bayes = full_bayes ? 1 : 0;
  const int64_t nw = (int64_t)pl.n_chains * pl.w_total, nh = (int64_t)pl.n_chains * pl.hyp_total;
  st.xi = f32o(xi, "xi", nw);
  st.xi_resample = f32o(xi_resample, "xi_resample", nw);
  st.xi_hyp = f32o(xi_hyp, "xi_hyp", nh);
  st.xi_hyp_resample = f32o(xi_hyp_resample, "xi_hyp_resample", nh);
  check_rc(dgprf_sghmc_step(&pl, &c, &b, &st, stream()), "dgprf_sghmc_step");
}

Tensor potential_grad(const Tensor& plan, const Tensor& theta, const Tensor& omega,
                      const Tensor& der, const Tensor& mass, const Tensor& ws, const Tensor& step,
                      const Tensor& X, const Tensor& Y, int64_t mode, int64_t iters,
                      int64_t perm_seed, const OptT& idx, double data_size, bool full_bayes,
                      const OptT& z, const OptT& hyp, const OptT& hmom, const OptT& hmass) {
  const dgprf_plan_t pl = plan_of(plan);
  // the gradient pass reads but never writes theta / mom (mom only by the update)
  const dgprf_chain_t c = chain_of(pl, theta, theta, omega, der, mass, ws, step, 0, z, hyp, hmom, hmass);
  const dgprf_batch_t b = batch_of(pl, X, Y, mode, iters, perm_seed, idx);
  const int64_t n = pl.w_total + (full_bayes ? pl.hyp_total : 0);
  Tensor out = at::empty({(int64_t)pl.n_chains, n}, theta.options());
  check_rc(dgprf_potential_grad(&pl, &c, &b, (float)data_size, full_bayes ? 1 : 0,
                                out.data_ptr<float>(), stream()),
           "dgprf_potential_grad");
  return out;
}

std::tuple<std::vector<Tensor>, Tensor, Tensor> forward(
    const Tensor& plan, const Tensor& theta, const Tensor& omega, const Tensor& der,
    const Tensor& X, const OptT& Y, int64_t f_mask, bool logp, bool se, const OptT& lse_m,
    const OptT& lse_s, const OptT& se_sum, const OptT& scratch) {
  const dgprf_plan_t pl = plan_of(plan);
  const int64_t C = pl.n_chains, ch = pl.hyp_per_chain ? C : 1;
  TORCH_CHECK(X.dim() == 2 && X.size(1) == pl.d_in, "dgprf: X must be [n, d_in]");
  const int64_t n = X.size(0);
  float* Yp = nullptr;
  int32_t y_cols = 0;
  if (Y.has_value() && Y->defined()) {
    TORCH_CHECK(Y->dim() == 2 && Y->size(0) == n, "dgprf: Y must be [n, y_cols]");
    Yp = f32(*Y, "Y");
    y_cols = (int32_t)Y->size(1);
  }
  std::vector<Tensor> F;
  float* fptr[DGPRF_MAX_LAYERS] = {};
  for (int l = 0; l < pl.n_layers; ++l)
    if (f_mask & (1ll << l)) {
      F.push_back(at::empty({C, n, (int64_t)pl.n_gp[l]}, theta.options()));
      fptr[l] = F.back().data_ptr<float>();
    }
  Tensor lp = logp ? at::empty({C, n}, theta.options()) : at::empty({0}, theta.options());
  Tensor sq = se ? at::empty({C, n}, theta.options()) : at::empty({0}, theta.options());
  int64_t need = 0;
  check_rc(dgprf_forward_scratch(&pl, n, &need), "dgprf_forward_scratch");
  float* scr = f32o(scratch, "scratch", need);
  TORCH_CHECK(need == 0 || scr, "dgprf: forward needs ", need, " floats of scratch");
  check_rc(dgprf_forward(&pl, f32(theta, "theta", C * pl.w_total), f32(omega, "omega", ch * pl.omega_total),
                         f32(der, "der", ch * pl.der_total), f32(X, "X"), Yp, y_cols, n, fptr,
                         logp ? lp.data_ptr<float>() : nullptr, se ? sq.data_ptr<float>() : nullptr,
                         f32o(lse_m, "lse_m", C * n), f32o(lse_s, "lse_s", C * n),
                         f32o(se_sum, "se_sum", C * n), scr,
                         scr ? scratch->numel() : 0, stream()),
           "dgprf_forward");
  return {F, lp, sq};
}

// thetas [S][C][w_total]: every sample of every chain folded into the LSE accumulators [C][n]
void forward_samples(const Tensor& plan, const Tensor& thetas, const Tensor& omega,
                     const Tensor& der, const Tensor& X, const OptT& A1, const Tensor& Y,
                     const Tensor& lse_m, const Tensor& lse_s, const OptT& se_sum,
                     const OptT& scratch) {
  const dgprf_plan_t pl = plan_of(plan);
  const int64_t C = pl.n_chains, ch = pl.hyp_per_chain ? C : 1;
  TORCH_CHECK(X.dim() == 2 && X.size(1) == pl.d_in, "dgprf: X must be [n, d_in]");
  const int64_t n = X.size(0);
  TORCH_CHECK(Y.dim() == 2 && Y.size(0) == n, "dgprf: Y must be [n, y_cols]");
  TORCH_CHECK(thetas.dim() == 3 && thetas.size(1) == C && thetas.size(2) == pl.w_total,
              "dgprf: thetas must be [samples, n_chains, w_total]");
  const int64_t S = thetas.size(0);
  // A1 rows past n up to a multiple of 64 are read (whole 64-row tile-kernel workgroups)
  float* a1 = f32o(A1, "A1", (n + 63) / 64 * 64 * (int64_t)pl.n_rf[0]);
  int64_t need = 0;
  check_rc(dgprf_forward_scratch(&pl, n, &need), "dgprf_forward_scratch");
  // the A_1 chunks need `need` floats unless A1 is resident; more (dgprf_forward_samples_scratch)
  // lets every sample pair run in one launch
  float* scr = f32o(scratch, "scratch", a1 ? 0 : need);
  TORCH_CHECK(a1 || need == 0 || scr, "dgprf: forward needs ", need, " floats of scratch");
  check_rc(dgprf_forward_samples(&pl, f32(thetas, "thetas", S * C * pl.w_total), (int32_t)S,
                                 f32(omega, "omega", ch * pl.omega_total),
                                 f32(der, "der", ch * pl.der_total), f32(X, "X"), a1, f32(Y, "Y"),
                                 (int32_t)Y.size(1), n, f32(lse_m, "lse_m", C * n),
                                 f32(lse_s, "lse_s", C * n), f32o(se_sum, "se_sum", C * n), scr,
                                 scr ? scratch->numel() : 0, stream()),
           "dgprf_forward_samples");
}

std::tuple<Tensor, Tensor> lse_finalize(const Tensor& m, const Tensor& s, const OptT& e,
                                        double s_total, double y_std, bool lse_out) {
  TORCH_CHECK(m.dim() == 2 && s.sizes() == m.sizes(), "dgprf: accumulators must be [parts, n]");
  const int64_t parts = m.size(0), n = m.size(1);
  Tensor out = at::zeros({2}, m.options().dtype(at::kDouble));
  Tensor lo = lse_out ? at::empty({n}, m.options()) : at::empty({0}, m.options());
  check_rc(dgprf_lse_finalize(f32(m, "lse_m", parts * n), f32(s, "lse_s", parts * n),
                              f32o(e, "se_sum", parts * n), (int32_t)parts, n, s_total,
                              (float)std::log(y_std), (float)y_std,
                              lse_out ? lo.data_ptr<float>() : nullptr, out.data_ptr<double>(),
                              stream()),
           "dgprf_lse_finalize");
  return {out, lo};
}

// ---------------------------------------------------------------- dense operators
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int32_t dense_type(const Tensor& t, const char* what) {
  if (t.scalar_type() == at::kFloat) return DGPRF_F32;
  if (t.scalar_type() == at::kHalf) return DGPRF_F16;
  TORCH_CHECK_TYPE(t.scalar_type() == at::kBFloat16, "dgprf: ", what,
                   " must be float32, float16 or bfloat16, got ", t.scalar_type());
  return DGPRF_BF16;
}
// same element type and device as x
void dense_like(const Tensor& t, const Tensor& x, const char* what) {
  TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type(), "dgprf: ", what, " is ", t.scalar_type(), ", x is ",
                   x.scalar_type(), " (one type for a call)");
  TORCH_CHECK_VALUE(t.device() == x.device(), "dgprf: ", what, " is on ", t.device(), ", x is on ", x.device());
}
bool given(const OptT& t) { return t.has_value() && t->defined(); }
// A forward-mode tangent would be left out silently (a dual tensor need not ask for a gradient): an error.
void no_tangent(const Tensor& t, const char* what) {
  TORCH_CHECK(!t.defined() || !t._fw_grad(/*level=*/0).defined(), "dgprf: ", what,
              " has no forward-mode derivative; use torch.autograd.grad");
}
void no_tangent(const OptT& t, const char* what) {
  if (t.has_value()) no_tangent(*t, what);
}

// t with the values that its memory holds: the imaginary part of a conjugate is a view that is marked as negated
Tensor plain(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
// [..., n] as a matrix that the kernels can read: unit stride within a row, rows apart by 0 or by n and
// more.  A view where the strides allow one.
Tensor rows_of(const Tensor& t, int64_t n) {
  const Tensor m = plain(t.dim() == 2 ? t : t.reshape({-1, n}));
  const bool ok = (n <= 1 || m.stride(1) == 1) &&
                  (m.size(0) <= 1 || m.stride(0) == 0 || m.stride(0) >= n);
  return ok ? m : m.contiguous();
}
constexpr int64_t kMaxStride = 1 << 20;  // of the operands of a product
int64_t row_stride(const Tensor& t) { return t.size(0) <= 1 ? t.size(1) : t.stride(0); }
// the same where rows may not share memory
Tensor apart(const Tensor& t) { return t.size(0) > 1 && t.stride(0) < t.size(1) ? t.contiguous() : t; }

struct Drop {
  int64_t thr, seed, sub;
  Tensor step;  // undefined: none
  Drop(int64_t thr_, int64_t seed_, int64_t sub_, const OptT& step_, const Tensor& x)
      : thr(thr_), seed(seed_), sub(sub_) {
    TORCH_CHECK_VALUE(thr >= 0 && thr <= 65536, "dgprf: dropout threshold must be in [0, 65536], got ", thr);
    if (!given(step_)) return;
    TORCH_CHECK_VALUE(step_->device() == x.device() && step_->scalar_type() == at::kLong && step_->numel() >= 1,
                      "dgprf: step must be an int64 tensor on the device of x");
    if (thr) step = *step_;
  }
  const int64_t* ptr() const { return step.defined() ? step.data_ptr<int64_t>() : nullptr; }
};

Tensor scratch_of(int64_t bytes, const Tensor& x) {
  return bytes ? at::empty({bytes}, x.options().dtype(at::kByte)) : Tensor();
}

// y [m, n]; aux: if not null, receives what backward needs of z (nothing for no activation)
Tensor linear_call(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& res, int64_t act,
                   const Drop& drop, Tensor* aux) {
  dgprf_linear_t a;
  std::memset(&a, 0, sizeof(a));
  const c10::DeviceGuard guard(x.device());
  a.dtype = dense_type(x, "x");
  a.act = (int32_t)act;
  a.m = x.size(0);
  a.k = x.size(1);
  a.n = w.size(1);
  a.ldx = row_stride(x);
  a.ldw = row_stride(w);
  a.x = x.data_ptr();
  a.w = w.data_ptr();
  if (bias.defined()) a.bias = bias.data_ptr();
  if (res.defined()) {
    a.res = res.data_ptr();
    a.ldr = row_stride(res);
  }
  a.drop_thr = (int32_t)drop.thr;
  a.seed = (uint64_t)drop.seed;
  a.sub = (uint64_t)drop.sub;
  a.step = drop.ptr();
  int64_t need = 0;
  check_rc(dgprf_linear_scratch(&a, &need), "dgprf_linear_forward");
  Tensor y = at::empty({a.m, a.n}, x.options());
  a.y = y.data_ptr();
  if (aux && act != DGPRF_ACT_NONE) {
    *aux = at::empty({a.m, (a.n + 7) / 8 * 8}, x.options());
    a.aux = aux->data_ptr();
  }
  const Tensor scratch = scratch_of(need, x);
  check_rc(dgprf_linear_forward(&a, need ? scratch.data_ptr() : nullptr, need, stream()),
           "dgprf_linear_forward");
  return y;
}

Tensor dropout_call(const Tensor& x, const Tensor& res, const Drop& drop) {
  const c10::DeviceGuard guard(x.device());
  Tensor y = at::empty({x.size(0), x.size(1)}, x.options());
  check_rc(dgprf_dropout(dense_type(x, "x"), x.data_ptr(), x.size(0), x.size(1), row_stride(x),
                         res.defined() ? res.data_ptr() : nullptr, res.defined() ? row_stride(res) : 0,
                         (int32_t)drop.thr, (uint64_t)drop.seed, (uint64_t)drop.sub, drop.ptr(), y.data_ptr(),
                         stream()),
           "dgprf_dropout");
  return y;
}

// A gradient of these gradients would leave terms out silently: it is an error instead, on every path from
// them to what the backward pass is of (the current node's inputs) and to the gradient dy that it got.
void once(const Tensor& dy, const variable_list& grads, const char* what) {
  if (!at::GradMode::is_enabled()) return;
  torch::autograd::edge_list to;
  if (const auto node = torch::autograd::get_current_node())
    for (const auto& edge : node->next_edges())
      if (edge.is_valid()) to.push_back(edge);
  if (dy.requires_grad()) to.push_back(torch::autograd::impl::gradient_edge(dy));
  const auto error = std::make_shared<torch::autograd::Error>(
      std::string("dgprf: ") + what + " has no second derivative", std::move(to));
  for (const Tensor& g : grads)
    if (g.defined()) torch::autograd::set_history(g, error);
}

bool capturing(hipStream_t s) {  // (the null stream cannot be captured, and must not be asked while another is)
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  return s && hipStreamIsCapturing(s, &status) == hipSuccess && status == hipStreamCaptureStatusActive;
}
// A leaf that an earlier, living autograd graph uses has its accumulation on that graph's stream, and so has
// every node of that graph.  The engine makes that stream wait for the captured one: another stream joins the
// capture by that (torch.cuda.make_graphed_callables' warm-up leaves such a graph), but the null stream
// cannot, which ends the capture and then the process.  Called in a backward pass, before anything is
// enqueued.  Looks at all that this pass still has to run behind the current node: a leaf may stand behind
// views and copies of it.
void check_capture(const char* what) {
  if (!capturing(c10::hip::getCurrentHIPStream().stream())) return;
  const auto current = torch::autograd::get_current_node();
  if (!current) return;
  std::vector<torch::autograd::Node*> open{current.get()};
  std::unordered_set<torch::autograd::Node*> seen{current.get()};
  while (!open.empty()) {
    torch::autograd::Node* const node = open.back();
    open.pop_back();
    for (size_t i = 0; i < node->num_outputs(); ++i) {
      torch::autograd::Node* const next = node->next_edge(i).function.get();
      if (!next || !node->task_should_compute_output(i) || !seen.insert(next).second) continue;
      if (const auto s = next->stream()) {
        const c10::Stream h(c10::Stream::UNSAFE, c10::Device(c10::DeviceType::HIP, s->device_index()), s->id());
        TORCH_CHECK(c10::hip::HIPStream(c10::hip::HIPStream::UNCHECKED, h).stream(), "dgprf: ", what,
                    ": this backward pass is being captured while an autograd graph from before the capture, on the "
                    "default stream, holds one of its leaves; delete that graph's results first");
      }
      open.push_back(next);
    }
  }
}

struct LinearFunction : public torch::autograd::Function<LinearFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptT& bias,
                        const OptT& res, int64_t act, int64_t thr, int64_t seed, int64_t sub, const OptT& step) {
    const Drop drop(thr, seed, sub, step, x);
    const bool save = x.requires_grad() || w.requires_grad() || (given(bias) && bias->requires_grad());
    Tensor aux;
    Tensor y = linear_call(x, w, given(bias) ? *bias : Tensor(), given(res) ? *res : Tensor(), act, drop,
                           save ? &aux : nullptr);
    ctx->save_for_backward({x, w, aux, drop.step});
    ctx->saved_data["args"] = std::vector<int64_t>{act, thr, seed, sub, given(bias), given(res)};
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &aux = saved[2], &step = saved[3];
    const auto args = ctx->saved_data["args"].toIntVector();
    const bool bias = args[4], res = args[5];
    const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
    const bool want_b = bias && ctx->needs_input_grad(2), want_r = res && ctx->needs_input_grad(bias ? 3 : 2);
    const c10::DeviceGuard guard(x.device());
    no_tangent(grads[0], "linear's gradient");
    check_capture("linear");
    Tensor dx, dw, db;
    if (want_x || want_w || want_b) {
      const at::NoGradGuard no_grad;
      Tensor dy = rows_of(grads[0], w.size(1));
      if (row_stride(dy) > kMaxStride) dy = dy.contiguous();
      dgprf_linear_grad_t a;
      std::memset(&a, 0, sizeof(a));
      a.dtype = dense_type(x, "x");
      a.act = (int32_t)args[0];
      a.m = x.size(0);
      a.k = x.size(1);
      a.n = w.size(1);
      a.ldx = row_stride(x);
      a.ldw = row_stride(w);
      a.lddy = row_stride(dy);
      a.x = x.data_ptr();
      a.w = w.data_ptr();
      a.dy = dy.data_ptr();
      if (aux.defined()) a.aux = aux.data_ptr();
      a.drop_thr = (int32_t)args[1];
      a.seed = (uint64_t)args[2];
      a.sub = (uint64_t)args[3];
      if (step.defined()) a.step = step.data_ptr<int64_t>();
      if (want_x) a.dx = (dx = at::empty({a.m, a.k}, x.options())).data_ptr();
      if (want_w) a.dw = (dw = at::empty({a.k, a.n}, x.options())).data_ptr();
      if (want_b) a.db = (db = at::empty({a.n}, x.options())).data_ptr();
      int64_t need = 0;
      check_rc(dgprf_linear_grad_scratch(&a, &need), "dgprf_linear_backward");
      const Tensor scratch = scratch_of(need, x);
      check_rc(dgprf_linear_backward(&a, need ? scratch.data_ptr() : nullptr, need, stream()),
               "dgprf_linear_backward");
    }
    const Tensor none;
    once(grads[0], {dx, dw, db}, "linear");
    return {dx, dw, db, want_r ? grads[0] : none, none, none, none, none, none};
  }
};

struct DropoutFunction : public torch::autograd::Function<DropoutFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptT& res, int64_t thr, int64_t seed,
                        int64_t sub, const OptT& step) {
    const Drop drop(thr, seed, sub, step, x);
    ctx->save_for_backward({drop.step});
    ctx->saved_data["args"] = std::vector<int64_t>{thr, seed, sub, given(res)};
    return dropout_call(x, given(res) ? *res : Tensor(), drop);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor step = ctx->get_saved_variables()[0];
    const auto args = ctx->saved_data["args"].toIntVector();
    const c10::DeviceGuard guard(grads[0].device());
    no_tangent(grads[0], "dropout's gradient");
    check_capture("dropout");
    Tensor dx;
    if (ctx->needs_input_grad(0)) {
      const at::NoGradGuard no_grad;
      const Tensor dy = rows_of(grads[0], grads[0].size(1));
      dx = dropout_call(dy, Tensor(), Drop(args[0], args[1], args[2], step, dy));
    }
    const Tensor none;
    once(grads[0], {dx}, "dropout");
    return {dx, args[3] && ctx->needs_input_grad(1) ? grads[0] : none, none, none, none, none};
  }
};

bool tracks(const OptT& t) { return given(t) && t->requires_grad(); }
constexpr const char* kNoCpu = ": the dense operators need a HIP device (there is no CPU fallback)";

Tensor linear(const Tensor& x, const Tensor& weight, const OptT& bias, int64_t act, const OptT& residual,
              int64_t thr, int64_t seed, int64_t sub, const OptT& step) {
  dense_type(x, "x");
  no_tangent(x, "linear");
  no_tangent(weight, "linear");
  no_tangent(bias, "linear");
  no_tangent(residual, "linear");
  TORCH_CHECK(x.is_cuda(), "dgprf: x is on ", x.device(), kNoCpu);
  dense_like(weight, x, "weight");
  TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 2 && x.size(-1) == weight.size(0),
                    "dgprf: x [..., k] and weight [k, n] do not fit: ", x.sizes(), ", ", weight.sizes());
  const int64_t k = weight.size(0), n = weight.size(1);
  TORCH_CHECK_VALUE(k >= 1 && n >= 1, "dgprf: weight must not be empty, got ", weight.sizes());
  auto shape = x.sizes().vec();
  shape.back() = n;
  OptT b = bias, r = residual;
  if (given(b)) {
    dense_like(*b, x, "bias");
    TORCH_CHECK_VALUE(b->dim() == 1 && b->size(0) == n, "dgprf: bias must be [", n, "], got ", b->sizes());
    b = plain(b->contiguous());
  }
  if (given(r)) {
    dense_like(*r, x, "residual");
    TORCH_CHECK_VALUE(r->sizes() == at::IntArrayRef(shape), "dgprf: residual must have the result's shape ",
                      at::IntArrayRef(shape), ", got ", r->sizes());
    r = rows_of(*r, n);
  }
  const Tensor x2 = apart(rows_of(x, k)), w = apart(rows_of(weight, n));
  Tensor y;
  if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || tracks(bias) || tracks(residual)))
    y = LinearFunction::apply(x2, w, b, r, act, thr, seed, sub, step);
  else
    y = linear_call(x2, w, given(b) ? *b : Tensor(), given(r) ? *r : Tensor(), act,
                    Drop(thr, seed, sub, step, x), nullptr);
  return x.dim() == 2 ? y : y.view(shape);
}

Tensor dropout(const Tensor& x, const OptT& residual, int64_t thr, int64_t seed, int64_t sub, const OptT& step) {
  dense_type(x, "x");
  no_tangent(x, "dropout");
  no_tangent(residual, "dropout");
  TORCH_CHECK(x.is_cuda(), "dgprf: x is on ", x.device(), kNoCpu);
  TORCH_CHECK_VALUE(x.dim() >= 1, "dgprf: x must have at least one dimension");
  const int64_t n = x.size(-1);
  OptT r = residual;
  if (given(r)) {
    dense_like(*r, x, "residual");
    TORCH_CHECK_VALUE(r->sizes() == x.sizes(), "dgprf: residual must have x's shape ", x.sizes(), ", got ", r->sizes());
  }
  if (x.numel() == 0) return given(r) ? at::add(x, *r) : x.clone();
  if (given(r)) r = rows_of(*r, n);
  const Tensor x2 = rows_of(x, n);
  Tensor y;
  if (at::GradMode::is_enabled() && (x.requires_grad() || tracks(residual)))
    y = DropoutFunction::apply(x2, r, thr, seed, sub, step);
  else
    y = dropout_call(x2, given(r) ? *r : Tensor(), Drop(thr, seed, sub, step, x));
  return x.dim() == 2 ? y : y.view(x.sizes());
}

}  // namespace

TORCH_LIBRARY(dgprf, m) {
  m.def(
      "sghmc_step_(Tensor plan, Tensor(a!) theta, Tensor(b!) mom, Tensor(c!) omega, Tensor(d!) der, "
      "Tensor mass, Tensor(e!) ws, Tensor(f!) step, int seed, Tensor X, Tensor Y, int mode, "
      "int iters_per_epoch, int perm_seed, Tensor? idx, float lr, float momentum_decay, "
      "float temperature, float data_size, bool resample_moments, Tensor? xi, Tensor? xi_resample, "
      "bool full_bayes, Tensor? z, Tensor(g!)? hyp, Tensor(h!)? hmom, Tensor? hmass, "
      "Tensor? xi_hyp, Tensor? xi_hyp_resample) -> ()");
  m.def(
      "potential_grad(Tensor plan, Tensor theta, Tensor omega, Tensor der, Tensor mass, "
      "Tensor(a!) ws, Tensor step, Tensor X, Tensor Y, int mode, int iters_per_epoch, "
      "int perm_seed, Tensor? idx, float data_size, bool full_bayes, Tensor? z, Tensor? hyp, "
      "Tensor? hmom, Tensor? hmass) -> Tensor");
  m.def(
      "forward(Tensor plan, Tensor theta, Tensor omega, Tensor der, Tensor X, Tensor? Y, "
      "int f_mask, bool logp, bool se, Tensor(a!)? lse_m, Tensor(b!)? lse_s, Tensor(c!)? se_sum, "
      "Tensor(d!)? scratch) -> (Tensor[], Tensor, Tensor)");
  m.def(
      "forward_samples(Tensor plan, Tensor thetas, Tensor omega, Tensor der, Tensor X, Tensor? A1, "
      "Tensor Y, Tensor(a!) lse_m, Tensor(b!) lse_s, Tensor(c!)? se_sum, Tensor(d!)? scratch) "
      "-> ()");
  m.def("lse_finalize(Tensor m, Tensor s, Tensor? e, float s_total, float y_std, bool lse_out) "
        "-> (Tensor, Tensor)");
  m.def("linear(Tensor x, Tensor weight, Tensor? bias, int act, Tensor? residual, int drop_thr, int seed, "
        "int sub, Tensor? step) -> Tensor",
        &linear);
  m.def("dropout(Tensor x, Tensor? residual, int drop_thr, int seed, int sub, Tensor? step) -> Tensor",
        &dropout);
}

TORCH_LIBRARY_IMPL(dgprf, CUDA, m) {
  m.impl("sghmc_step_", &sghmc_step_);
  m.impl("potential_grad", &potential_grad);
  m.impl("forward", &forward);
  m.impl("forward_samples", &forward_samples);
  m.impl("lse_finalize", &lse_finalize);
}
