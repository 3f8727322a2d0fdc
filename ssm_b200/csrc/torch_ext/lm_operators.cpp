// The gated delta rule, token log probabilities and distillation: the operator surface of ssm_b200.ops over include/ssm_b200_lm.h.
#include "../../../include/ssm_b200_lm.h"

#include "call.h"

namespace ssm_ext {
namespace {

namespace py = pybind11;

// rows of the innermost axis as they lie, where that axis is contiguous
Tensor strided(const Tensor& t) {
  Tensor d = t.detach();
  return d.dim() == 0 || d.size(-1) <= 1 || d.stride(-1) == 1 ? d : d.contiguous();
}
// g and beta are read in their own type
Tensor coefficient(const Tensor& t, const char* what) {
  dtype_code(t, what);
  return t.detach();
}
Tensor lead(const Tensor& t, at::ScalarType type) { return strided(t.scalar_type() == type ? t.detach() : t.detach().to(type)); }

// ---------------------------------------------------------------------------------------------
// gated delta rule
// ---------------------------------------------------------------------------------------------
// An operand that the tensor-core kernels can copy: rows on 16-byte boundaries, no broadcast axis
Tensor copyable(const Tensor& t) {
  bool ok = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && (t.size(i) <= 1 || (t.stride(i) > 0 && t.stride(i) % 8 == 0));
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

struct DeltaCall final : Call {
  Tensor q, k, v, g, beta, init, cu, table, rest, states, kept;  // g, init, cu may be undefined
  int64_t nb, nl, nh, nk, kd, vd, seqs;
  at::ScalarType t_q, t_k, t_v, t_g{}, t_beta, t_init{};
  double scale;
  bool want_final, fp32_state, init_grad = false, chunked = false;

  DeltaCall(const Tensor& q_, const Tensor& k_, const Tensor& v_, const OptTensor& g_, const Tensor& beta_, const c10::optional<double>& scale_, const OptTensor& init_,
            bool want_final_, bool fp32_state_, const OptTensor& cu_)
      : t_q(q_.scalar_type()), t_k(k_.scalar_type()), t_v(v_.scalar_type()), t_beta(beta_.scalar_type()), want_final(want_final_), fp32_state(fp32_state_) {
    SSM_ARG(q_.dim() == 4 && k_.dim() == 4 && v_.dim() == 4, "q and k must have shape (B, L, Hk, K) and v (B, L, H, V).");
    nb = v_.size(0), nl = v_.size(1), nh = v_.size(2), vd = v_.size(3), nk = k_.size(2), kd = k_.size(3);
    SSM_ARG(k_.size(0) == nb && k_.size(1) == nl && q_.sizes() == k_.sizes(), "q and k must have shape (B, L, Hk, K) with v's B and L.");
    SSM_ARG(nk > 0 && nh > 0 && nh % nk == 0, "The key heads must divide the value heads.");
    SSM_ARG(kd > 0 && vd > 0, "K and V must be positive.");
    SSM_ARG(kd <= 256 && vd <= 65536 && nh <= 65535, "gated_delta_scan: K is at most 256, V at most 65536, the heads at most 65535.");
    auto per_head = [&](const Tensor& t) { return t.dim() == 3 && t.size(0) == nb && t.size(1) == nl && t.size(2) == nh; };
    SSM_ARG(per_head(beta_) && (!g_.has_value() || per_head(*g_)), "g and beta must have shape (B, L, H).");
    scale = scale_.has_value() ? *scale_ : 1.0 / std::sqrt((double)kd);
    SSM_ARG(std::isfinite(scale), "scale must be finite.");
    SSM_ARG(nl < ((int64_t)1 << 30) && nb < 65535, "gated_delta_scan: too many tokens or sequences.");
    seqs = nb;
    if (cu_.has_value()) {
      SSM_ARG(nb == 1, "cu_seqlens needs a batch of one (sequences packed along L).");
      SSM_ARG(cu_->dim() == 1 && cu_->numel() >= 2 && at::isIntegralType(cu_->scalar_type(), false), "cu_seqlens must hold S + 1 integers.");
      seqs = cu_->numel() - 1;
      SSM_ARG(seqs < 65535, "gated_delta_scan: too many sequences.");
    }
    if (init_.has_value())
      SSM_ARG(init_->dim() == 4 && init_->size(0) == seqs && init_->size(1) == nh && init_->size(2) == vd && init_->size(3) == kd,
              "initial_state must have shape (B, H, V, K), or (S, H, V, K) with cu_seqlens.");
    same_device(v_, {&q_, &k_, &beta_});
    need_cuda(v_, {&g_, &init_});
    dtype_code(v_, "gated_delta_scan"), dtype_code(q_, "gated_delta_scan"), dtype_code(k_, "gated_delta_scan");
    if (cu_.has_value()) {
      const Tensor c = cu_->detach();
      if (!c.is_cuda()) {
        const Tensor host = c.to(at::kLong).contiguous();
        const int64_t* p = host.data_ptr<int64_t>();
        bool ok = p[0] == 0 && p[seqs] <= nl;
        for (int64_t i = 0; i < seqs; ++i) ok = ok && p[i + 1] >= p[i];
        SSM_ARG(ok, "cu_seqlens must rise from 0 to at most L.");
        cu = host.to(v_.device());
      } else {
        SSM_ARG(c.device() == v_.device(), "all tensors must be on the same CUDA device");
        cu = (c.scalar_type() == at::kInt || c.scalar_type() == at::kLong ? c : c.to(at::kLong)).contiguous();
      }
    }
    for (const Tensor* t : {&q_, &k_, &v_}) input(*t);
    input(g_), input(beta_), input(init_);
    q = lead(q_, t_v), k = lead(k_, t_v), v = strided(v_), beta = coefficient(beta_, "gated_delta_scan beta");
    if (g_.has_value()) g = coefficient(*g_, "gated_delta_scan g"), t_g = g_->scalar_type();
    // A few tokens without gradients walk one by one: a chunk costs the same whatever its tokens.  Measured (K = V = 128, bf16, us, chunks | tokens):
    // 16 heads, 8 tokens 14.2 | 5.4, 16 tokens 14.3 | 7.6; 128 heads, 8 tokens 15.1 | 12.3, 16 tokens 15.2 | 18.2; 1024 heads, 4 tokens 56 | 54,
    // 8 tokens 56 | 74; 8192 heads, 4 tokens 416 | 414.  With gradients chunks win from one token on (16 heads 33 | 48, 1024 heads 185 | 439).
    const bool few = nl <= (nb * nh <= 128 ? 8 : 4) && !needs_grad();
    if (v.scalar_type() != at::kFloat && kd % 8 == 0 && kd <= 128 && vd % 8 == 0 && nl > 0 && nb > 0 && !few) {
      chunked = true;
      q = copyable(q), k = copyable(k), v = copyable(v);
    }
    if (init_.has_value()) init = f32c(*init_), t_init = init_->scalar_type(), init_grad = init_->requires_grad();
  }

  void fill(ssm_gated_delta_args& a) const {
    a.batch = (int)nb, a.len = (int)nl, a.heads = (int)nh, a.key_heads = (int)nk, a.kdim = (int)kd, a.vdim = (int)vd;
    a.io_dtype = dtype_code(v, "gated_delta_scan"), a.beta_dtype = dtype_code(beta, "gated_delta_scan beta"), a.scale = (float)scale;
    a.q = q.data_ptr(), a.q_sb = q.stride(0), a.q_st = q.stride(1), a.q_sh = q.stride(2);
    a.k = k.data_ptr(), a.k_sb = k.stride(0), a.k_st = k.stride(1), a.k_sh = k.stride(2);
    a.v = v.data_ptr(), a.v_sb = v.stride(0), a.v_st = v.stride(1), a.v_sh = v.stride(2);
    if (g.defined()) a.g = g.data_ptr(), a.g_dtype = dtype_code(g, "gated_delta_scan g"), a.g_sb = g.stride(0), a.g_st = g.stride(1), a.g_sh = g.stride(2);
    a.beta = beta.data_ptr(), a.beta_sb = beta.stride(0), a.beta_st = beta.stride(1), a.beta_sh = beta.stride(2);
    if (init.defined()) a.initial_state = init.data_ptr<float>();
    if (cu.defined()) a.num_seqs = (int)seqs, a.cu_seqlens = cu.data_ptr(), a.cu_is_64 = cu.scalar_type() == at::kLong, a.table = table.data_ptr<int32_t>();
    if (rest.defined()) a.rest = rest.data_ptr<float>(), a.states = states.data_ptr<float>();
  }
  at::TensorOptions f32() const { return v.options().dtype(at::kFloat).requires_grad(false); }

  variable_list forward(bool train) override {
    c10::cuda::CUDAGuard guard(v.device());
    Tensor o = at::empty({nb, nl, nh, vd}, v.options()), fin;
    if (cu.defined()) table = at::empty({ssm_gated_delta_table_ints((int)nb, (int)nl, (int)seqs)}, v.options().dtype(at::kInt));
    if (chunked && init.defined() && reinterpret_cast<uintptr_t>(init.data_ptr()) % 16 != 0) init = init.clone();
    if (train && !chunked) {
      rest = at::empty({nb, nl, nh, vd}, f32());
      states = at::empty({ssm_gated_delta_chunks((int)nb, (int)nl, (int)seqs * cu.defined()), nh, vd, kd}, f32());
    }
    ssm_gated_delta_args a{};
    fill(a);
    a.o = o.data_ptr();
    if (want_final) fin = at::empty({seqs, nh, vd, kd}, fp32_state ? f32() : v.options()), a.final_state = fin.data_ptr(), a.final_dtype = dtype_code(fin, "gated_delta_scan");
    if (chunked) {
      ssd_poll(v.get_device());  // a wait that ran out in an earlier launch surfaces here, without a synchronisation
      const auto bytes = v.options().dtype(at::kByte);
      Tensor scratch = at::empty({ssm_gated_delta_chunked_scratch_bytes((int)nb, (int)nl, a.num_seqs, (int)nh, (int)kd)}, bytes);
      kept = at::empty({ssm_gated_delta_chunked_kept_bytes((int)nb, (int)nl, a.num_seqs, (int)nh, (int)kd, (int)vd, train)}, bytes);
      run(ssm_gated_delta_chunked_fwd(&a, scratch.data_ptr(), kept.data_ptr(), train, ssd_status(v.get_device()).data_ptr<int32_t>(), stream_of(v)));
    } else {
      run(ssm_gated_delta_fwd(&a, stream_of(v)));
    }
    if (want_final) return {o, fin};
    return {o};
  }

  variable_list backward(const variable_list& grads) override {
    c10::cuda::CUDAGuard guard(v.device());
    Tensor go = grads[0].defined() ? like(grads[0], v) : at::zeros({nb, nl, nh, vd}, v.options()), gfin, dinit, dqk;
    if (grads.size() > 1 && grads[1].defined()) gfin = f32c(grads[1]);
    Tensor dq = at::empty({nb, nl, nk, kd}, v.options()), dk = at::empty_like(dq), dv = at::empty({nb, nl, nh, vd}, v.options());
    Tensor dg = at::empty({nb, nl, nh}, f32()), db = at::empty_like(dg), dv32, dstates;
    if (nh != nk) dqk = at::empty({2, nb, nl, nh, kd}, f32());
    if (init_grad) dinit = at::empty({seqs, nh, vd, kd}, f32());
    ssm_gated_delta_bwd_args a{};
    fill(a.fwd);
    auto aligned = [&](Tensor& t) {
      if (t.defined() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0) t = t.clone();
    };
    if (chunked) aligned(go), aligned(gfin);
    a.dout = go.data_ptr(), a.dfinal = gfin.defined() ? gfin.data_ptr<float>() : nullptr;
    a.dq = dq.data_ptr(), a.dk = dk.data_ptr(), a.dv = dv.data_ptr(), a.dg = dg.data_ptr<float>(), a.dbeta = db.data_ptr<float>();
    a.dinitial = dinit.defined() ? dinit.data_ptr<float>() : nullptr, a.dqk = dqk.defined() ? dqk.data_ptr<float>() : nullptr;
    if (chunked) {
      Tensor scratch = at::empty({ssm_gated_delta_chunked_bwd_scratch_bytes((int)nb, (int)nl, a.fwd.num_seqs, (int)nh, (int)kd, (int)vd)}, v.options().dtype(at::kByte));
      run(ssm_gated_delta_chunked_bwd(&a, kept.data_ptr(), scratch.data_ptr(), ssd_status(v.get_device()).data_ptr<int32_t>(), stream_of(v)));
    } else {
      dv32 = v.scalar_type() == at::kFloat ? dv : at::empty({nb, nl, nh, vd}, f32()), dstates = at::empty_like(states);
      a.dv32 = dv32.data_ptr<float>(), a.dstates = dstates.data_ptr<float>();
      run(ssm_gated_delta_bwd(&a, stream_of(v)));
    }
    variable_list res = {cast(dq, t_q), cast(dk, t_k), cast(dv, t_v)};
    if (g.defined()) res.push_back(cast(dg, t_g));
    res.push_back(cast(db, t_beta));
    if (init.defined()) res.push_back(init_grad ? cast(dinit, t_init) : Tensor());
    return res;
  }
};

py::object gated_delta_scan(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& g, const Tensor& beta, const c10::optional<double>& scale,
                            const OptTensor& init, bool want_final, bool fp32_state, const OptTensor& cu) {
  ValueErrors scope;
  variable_list r = invoke_call(c10::make_intrusive<DeltaCall>(q, k, v, g, beta, scale, init, want_final, fp32_state, cu));
  if (want_final) return py::make_tuple(r[0], r[1]);
  return py::cast(r[0]);
}

Tensor gated_delta_step(const Tensor& state, const Tensor& q_, const Tensor& k_, const Tensor& v_, const OptTensor& g_, const Tensor& beta_,
                        const c10::optional<double>& scale) {
  ValueErrors scope;
  SSM_ARG(state.dim() == 4, "state must have shape (B, H, V, K).");
  const int64_t nb = state.size(0), nh = state.size(1), vd = state.size(2), kd = state.size(3);
  SSM_ARG(q_.dim() == 3 && k_.dim() == 3 && q_.sizes() == k_.sizes() && k_.size(0) == nb && k_.size(2) == kd, "q and k must have shape (B, Hk, K).");
  SSM_ARG(v_.dim() == 3 && v_.size(0) == nb && v_.size(1) == nh && v_.size(2) == vd, "v must have shape (B, H, V).");
  const int64_t nk = k_.size(1);
  SSM_ARG(nk > 0 && nh > 0 && nh % nk == 0, "The key heads must divide the value heads.");
  SSM_ARG(kd > 0 && vd > 0, "K and V must be positive.");
  SSM_ARG(kd <= 256 && vd <= 65536 && nh <= 65535, "gated_delta_step: K is at most 256, V at most 65536, the heads at most 65535.");
  auto per_head = [&](const Tensor& t) { return t.dim() == 2 && t.size(0) == nb && t.size(1) == nh; };
  SSM_ARG(per_head(beta_) && (!g_.has_value() || per_head(*g_)), "g and beta must have shape (B, H).");
  same_device(state, {&q_, &k_, &v_, &beta_});
  need_cuda(state, {&g_});
  SSM_ARG(state.scalar_type() == at::kFloat, "state must be float32.");
  dtype_code(v_, "gated_delta_step"), dtype_code(q_, "gated_delta_step"), dtype_code(k_, "gated_delta_step");
  const double s = scale.has_value() ? *scale : 1.0 / std::sqrt((double)kd);
  SSM_ARG(std::isfinite(s), "scale must be finite.");
  SSM_ARG(nb < 65536, "gated_delta_step: too many sequences.");
  bool wanted = false;  // gradients
  for (const Tensor* t : {&state, &q_, &k_, &v_, &beta_, g_.has_value() ? &*g_ : &beta_}) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(0).defined(), "ssm_b200 operators have no forward-mode derivative");
    wanted = wanted || (at::GradMode::is_enabled() && t->requires_grad());
  }
  if (wanted) {
    const OptTensor g = g_.has_value() ? OptTensor(g_->unsqueeze(1)) : c10::nullopt;
    const variable_list r = invoke_call(c10::make_intrusive<DeltaCall>(q_.unsqueeze(1), k_.unsqueeze(1), v_.unsqueeze(1), g, beta_.unsqueeze(1), s, OptTensor(state.clone()), true, true, c10::nullopt));
    const Tensor o = r[0].select(1, 0);
    at::NoGradGuard values;
    state.copy_(r[1]);
    return o;
  }
  c10::cuda::CUDAGuard guard(state.device());
  const Tensor q = lead(q_, v_.scalar_type()), k = lead(k_, v_.scalar_type()), v = strided(v_), beta = coefficient(beta_, "gated_delta_step beta");
  const Tensor work = state.is_contiguous() ? state.detach() : state.detach().contiguous();
  Tensor o = at::empty({nb, nh, vd}, v.options());
  ssm_gated_delta_step_args a{};
  a.batch = (int)nb, a.heads = (int)nh, a.key_heads = (int)nk, a.kdim = (int)kd, a.vdim = (int)vd, a.io_dtype = dtype_code(v, "gated_delta_step");
  a.beta_dtype = dtype_code(beta, "gated_delta_step beta"), a.scale = (float)s, a.state = work.data_ptr<float>(), a.o = o.data_ptr();
  a.q = q.data_ptr(), a.q_sb = q.stride(0), a.q_sh = q.stride(1), a.k = k.data_ptr(), a.k_sb = k.stride(0), a.k_sh = k.stride(1);
  a.v = v.data_ptr(), a.v_sb = v.stride(0), a.v_sh = v.stride(1), a.beta = beta.data_ptr(), a.beta_sb = beta.stride(0), a.beta_sh = beta.stride(1);
  Tensor g;
  if (g_.has_value()) {
    g = coefficient(*g_, "gated_delta_step g");
    a.g = g.data_ptr(), a.g_dtype = dtype_code(g, "gated_delta_step g"), a.g_sb = g.stride(0), a.g_sh = g.stride(1);
  }
  run(ssm_gated_delta_step(&a, stream_of(state)));
  if (!state.is_contiguous()) state.detach().copy_(work);
  else if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();  // a graph that keeps this state for its backward pass notices
  return o;
}

// ---------------------------------------------------------------------------------------------
// log probabilities of given tokens
// ---------------------------------------------------------------------------------------------
// (..., V) as rows with a stride; copied where the axes before the last do not lie evenly
Tensor as_rows(const Tensor& t) {
  Tensor d = strided(t);
  int64_t rows = 1;
  for (int64_t i = 0; i + 1 < d.dim(); ++i) rows *= d.size(i);
  return strided(d.reshape({rows, d.size(-1)}));
}
std::vector<int64_t> without_last(const Tensor& t) {
  std::vector<int64_t> s = t.sizes().vec();
  s.pop_back();
  return s;
}
void logits_check(const Tensor& logits, double temperature, const char* what) {
  SSM_ARG(logits.dim() >= 1 && logits.size(-1) >= 1, "logits must have shape (..., V) with V of at least one.");
  SSM_ARG(logits.size(-1) <= (1 << 30), "logits: more than 2^30 columns.");
  SSM_ARG(temperature > 0 && std::isfinite(temperature), "temperature must be positive and finite.");
  TORCH_CHECK(logits.is_cuda(), "ssm_b200 operators run on CUDA tensors only; there is no CPU fallback");
  dtype_code(logits, what);
}

struct LogpCall final : Call {
  Tensor x, targets, stats, ids;
  std::vector<int64_t> shape, lead_shape;
  double temperature;
  int64_t top_k, ignore;
  bool want_entropy;

  LogpCall(const Tensor& logits, const Tensor& targets_, double temperature_, int64_t top_k_, bool want_entropy_, int64_t ignore_)
      : temperature(temperature_), top_k(top_k_), ignore(ignore_), want_entropy(want_entropy_) {
    logits_check(logits, temperature_, "token_log_probs");
    shape = logits.sizes().vec(), lead_shape = without_last(logits);
    SSM_ARG(targets_.sizes() == lead_shape, "targets must have the shape of logits without the last axis.");
    SSM_ARG(at::isIntegralType(targets_.scalar_type(), false), "targets must be integers.");
    SSM_ARG(top_k >= 0 && top_k <= std::min<int64_t>(logits.size(-1), 128), "top_k must lie between 0 and 128, and at most be V.");
    same_device(logits, {&targets_});
    input(logits), input(targets_);
    x = as_rows(logits), targets = targets_.detach().to(at::kLong).contiguous();
  }
  void fill(ssm_token_logp_args& a) const {
    a.rows = x.size(0), a.row_stride = x.stride(0), a.vocab = (int)x.size(1), a.io_dtype = dtype_code(x, "token_log_probs"), a.top_k = (int)top_k;
    a.ignore_index = ignore, a.temperature = (float)temperature, a.logits = x.data_ptr(), a.targets = targets.data_ptr<int64_t>();
    if (stats.defined()) a.stats = stats.data_ptr<float>();
  }
  variable_list forward(bool train) override {
    c10::cuda::CUDAGuard guard(x.device());
    const auto f32 = x.options().dtype(at::kFloat);
    Tensor logp = at::empty(lead_shape, f32), entropy, top;
    if (train) stats = at::empty({x.size(0), 4}, f32);
    ssm_token_logp_args a{};
    fill(a);
    a.logp = logp.data_ptr<float>();
    variable_list res = {logp};
    if (want_entropy) entropy = at::empty(lead_shape, f32), a.entropy = entropy.data_ptr<float>(), res.push_back(entropy);
    if (top_k) {
      std::vector<int64_t> s = lead_shape;
      s.push_back(top_k);
      top = at::empty(s, f32), ids = at::empty(s, x.options().dtype(at::kLong));
      a.top_logp = top.data_ptr<float>(), a.top_ids = ids.data_ptr<int64_t>();
      res.push_back(top), res.push_back(ids);
    }
    run(ssm_token_logp(&a, stream_of(x)));
    if (train && top_k) ids = ids.clone();  // the caller may edit what it was given
    return res;
  }
  variable_list backward(const variable_list& grads) override {
    c10::cuda::CUDAGuard guard(x.device());
    Tensor d = at::empty(shape, x.options()), gl, gh, gt;
    auto f = [](const Tensor& t) { return t.defined() ? f32c(t) : Tensor(); };
    gl = f(grads[0]);
    if (want_entropy) gh = f(grads[1]);
    if (top_k) gt = f(grads[want_entropy ? 2 : 1]);
    ssm_token_logp_bwd_args a{};
    fill(a.fwd);
    if (top_k) a.fwd.top_ids = ids.data_ptr<int64_t>();
    auto p = [](const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; };
    a.dlogp = p(gl), a.dentropy = p(gh), a.dtop_logp = p(gt), a.dlogits = d.data_ptr();
    run(ssm_token_logp_bwd(&a, stream_of(x)));
    return {d, Tensor()};
  }
};
py::object token_log_probs(const Tensor& logits, const Tensor& targets, double temperature, int64_t top_k, bool want_entropy, int64_t ignore) {
  ValueErrors scope;
  variable_list r = invoke_call(c10::make_intrusive<LogpCall>(logits, targets, temperature, top_k, want_entropy, ignore));
  if (r.size() == 1) return py::cast(r[0]);
  py::tuple t(r.size());
  for (size_t i = 0; i < r.size(); ++i) t[i] = py::cast(r[i]);
  return std::move(t);
}

// ---------------------------------------------------------------------------------------------
// distillation
// ---------------------------------------------------------------------------------------------
struct DistillCall final : Call {
  Tensor x, teacher, ids, stats;
  std::vector<int64_t> shape, lead_shape;
  double temperature;

  DistillCall(const Tensor& logits, const Tensor& teacher_, const Tensor& ids_, double temperature_) : temperature(temperature_) {
    logits_check(logits, temperature_, "topk_distill_loss");
    shape = logits.sizes().vec(), lead_shape = without_last(logits);
    SSM_ARG(teacher_.dim() == logits.dim() && without_last(teacher_) == lead_shape && teacher_.size(-1) >= 1 && teacher_.size(-1) <= 1024,
            "teacher_logits must have shape (..., k) with the axes of logits before the last and k from 1 to 1024.");
    SSM_ARG(ids_.sizes() == teacher_.sizes(), "teacher_ids must have the shape of teacher_logits.");
    SSM_ARG(at::isIntegralType(ids_.scalar_type(), false), "teacher_ids must be integers.");
    SSM_ARG(!(at::GradMode::is_enabled() && teacher_.requires_grad()), "teacher_logits: no gradient flows to the teacher; detach them.");
    same_device(logits, {&teacher_, &ids_});
    dtype_code(teacher_, "topk_distill_loss teacher");
    input(logits), input(teacher_), input(ids_);
    x = as_rows(logits), teacher = teacher_.detach().contiguous(), ids = ids_.detach().to(at::kLong).contiguous();
  }
  void fill(ssm_topk_distill_args& a) const {
    a.rows = x.size(0), a.row_stride = x.stride(0), a.vocab = (int)x.size(1), a.io_dtype = dtype_code(x, "topk_distill_loss"), a.top_k = (int)teacher.size(-1);
    a.teacher_dtype = dtype_code(teacher, "topk_distill_loss teacher"), a.temperature = (float)temperature;
    a.logits = x.data_ptr(), a.teacher = teacher.data_ptr(), a.ids = ids.data_ptr<int64_t>();
    if (stats.defined()) a.stats = stats.data_ptr<float>();
  }
  variable_list forward(bool train) override {
    c10::cuda::CUDAGuard guard(x.device());
    const auto f32 = x.options().dtype(at::kFloat);
    Tensor loss = at::empty(lead_shape, f32);
    if (train) stats = at::empty({x.size(0), 4}, f32);
    ssm_topk_distill_args a{};
    fill(a);
    a.loss = loss.data_ptr<float>();
    run(ssm_topk_distill(&a, stream_of(x)));
    return {loss};
  }
  variable_list backward(const variable_list& grads) override {
    c10::cuda::CUDAGuard guard(x.device());
    if (!grads[0].defined()) return {at::zeros(shape, x.options()), Tensor(), Tensor()};
    Tensor d = at::empty(shape, x.options()), gl = f32c(grads[0]);
    ssm_topk_distill_bwd_args a{};
    fill(a.fwd);
    a.dloss = gl.data_ptr<float>(), a.dlogits = d.data_ptr();
    run(ssm_topk_distill_bwd(&a, stream_of(x)));
    return {d, Tensor(), Tensor()};
  }
};
Tensor topk_distill_loss(const Tensor& logits, const Tensor& teacher, const Tensor& ids, double temperature) {
  ValueErrors scope;
  return invoke_call(c10::make_intrusive<DistillCall>(logits, teacher, ids, temperature))[0];
}

}  // namespace

void bind_lm_operators(py::module& m) {
  auto ops = m.attr("operators").cast<py::module>();
  ops.def("gated_delta_scan", &gated_delta_scan);
  ops.def("gated_delta_step", &gated_delta_step);
  ops.def("token_log_probs", &token_log_probs);
  ops.def("topk_distill_loss", &topk_distill_loss);
}

}  // namespace ssm_ext
