// The norms around a block, cross entropy from hidden states and the norm over many tensors with clipping: the operator surface of
// ssm_b200.ops over include/ssm_b200_lm.h.
#include "../../../include/ssm_b200_lm.h"

#include <algorithm>

#include <torch/csrc/autograd/python_variable.h>

#include "call.h"

namespace ssm_ext {
namespace {

namespace py = pybind11;

// the tensor itself where it hangs in no graph (a view takes longer than the look), dense
Tensor dense(const Tensor& t) {
  const Tensor d = torch::autograd::impl::get_autograd_meta(t) ? t.detach() : t;
  return d.is_contiguous() ? d : d.contiguous();
}
OptTensor dense(const OptTensor& t) { return t.has_value() ? OptTensor(dense(*t)) : OptTensor(); }

// ---------------------------------------------------------------------------------------------
// the norms after and before a block
// ---------------------------------------------------------------------------------------------
struct BlockNormCall final : Call {
  Tensor x, pw, w, stats;
  OptTensor res, pb, b, gate;
  at::ScalarType t_r{}, t_pw, t_w, t_pb{}, t_b{}, out_type;
  std::vector<int64_t> gate_shape;
  int64_t rows, len, dim;
  int gate_kind = 0;
  bool is_rms, has_pb, has_b;
  double scale, eps, post_eps;

  BlockNormCall(const Tensor& x_, const OptTensor& res_, const Tensor& pw_, const Tensor& w_, const OptTensor& pb_, const OptTensor& b_, const OptTensor& gate_, double scale_,
                bool is_rms_, double eps_, double post_eps_, bool in_fp32)
      : t_pw(pw_.scalar_type()), t_w(w_.scalar_type()), out_type(in_fp32 ? at::kFloat : x_.scalar_type()), is_rms(is_rms_), scale(scale_), eps(eps_), post_eps(post_eps_) {
    SSM_ARG(x_.dim() == 3, "x must have shape (B, L, D).");
    dim = x_.size(2), len = x_.size(1), rows = x_.size(0) * x_.size(1);
    SSM_ARG(dim >= 1 && dim <= 8192, "fused_block_norm: D lies between 1 and 8192.");
    SSM_ARG(rows < ((int64_t)1 << 30), "fused_block_norm: too many rows.");
    auto param = [&](const Tensor& t, const char* name) { SSM_ARG(t.dim() == 1 && t.size(0) == dim, name, " must have shape (D,)."); };
    param(pw_, "post_weight"), param(w_, "weight");
    if (pb_.has_value()) param(*pb_, "post_bias"), t_pb = pb_->scalar_type();
    if (b_.has_value()) param(*b_, "bias"), t_b = b_->scalar_type();
    if (res_.has_value()) {
      SSM_ARG(res_->sizes() == x_.sizes(), "residual must match the shape of x.");
      t_r = res_->scalar_type();
    }
    if (gate_.has_value()) {
      const Tensor& g = *gate_;
      if (g.dim() == 1 && g.size(0) == dim) gate_kind = 1;
      else if ((g.dim() == 2 && g.size(0) == x_.size(0) && g.size(1) == dim) || (g.dim() == 3 && g.size(0) == x_.size(0) && g.size(1) == 1 && g.size(2) == dim)) gate_kind = 2;
      else if (g.sizes() == x_.sizes()) gate_kind = 3;
      else reject("gate must have shape (D,), (B, D), (B, 1, D) or (B, L, D).");
      gate_shape = g.sizes().vec();
    }
    SSM_ARG(std::isfinite(scale) && std::abs(scale) < 3e38, "residual_scale must be finite, in fp32 too.");
    SSM_ARG(eps >= 0 && post_eps >= 0 && std::isfinite(eps) && std::isfinite(post_eps), "eps must be finite and not negative.");
    same_device(x_, {&pw_, &w_});
    need_cuda(x_, {&res_, &pb_, &b_, &gate_});
    dtype_code(x_, "fused_block_norm"), dtype_code(pw_, "fused_block_norm post_weight"), dtype_code(w_, "fused_block_norm weight");
    if (res_.has_value()) dtype_code(*res_, "fused_block_norm residual");
    if (pb_.has_value()) dtype_code(*pb_, "fused_block_norm post_bias");
    if (b_.has_value()) dtype_code(*b_, "fused_block_norm bias");
    if (gate_.has_value()) dtype_code(*gate_, "fused_block_norm gate");
    input(x_), input(res_), input(pw_), input(w_), input(pb_), input(b_), input(gate_);
    x = dense(x_), res = dense(res_), gate = dense(gate_);
    // the parameters go in as they are where they share a type
    if (t_pw == t_w && (!pb_.has_value() || t_pb == t_w) && (!b_.has_value() || t_b == t_w)) pw = dense(pw_), w = dense(w_), pb = dense(pb_), b = dense(b_);
    else pw = f32c(pw_), w = f32c(w_), pb = f32c(pb_), b = f32c(b_);
    has_pb = pb.has_value(), has_b = b.has_value();
    if (has_pb != has_b) (has_pb ? b : pb) = at::zeros(w.sizes(), w.options());  // the kernels take both or neither
  }
  void fill(ssm_block_norm_args& a) const {
    a.rows = rows, a.len = std::max<int64_t>(len, 1), a.dim = (int)dim, a.io_dtype = dtype_code(x, "fused_block_norm");
    a.res_dtype = res.has_value() ? dtype_code(*res, "fused_block_norm residual") : 0, a.resout_dtype = out_type == at::kFloat ? SSM_F32 : a.io_dtype;
    a.param_dtype = dtype_code(w, "fused_block_norm weight"), a.gate_dtype = gate.has_value() ? dtype_code(*gate, "fused_block_norm gate") : 0;
    a.gate_kind = gate_kind, a.is_rms = is_rms, a.eps = (float)eps, a.post_eps = (float)post_eps, a.scale = (float)scale;
    a.x = x.data_ptr(), a.residual = ptr(res), a.post_weight = pw.data_ptr(), a.weight = w.data_ptr(), a.post_bias = ptr(pb), a.bias = ptr(b), a.gate = ptr(gate);
    if (stats.defined()) a.stats = stats.data_ptr<float>();
  }
  variable_list forward(bool train) override {
    c10::cuda::CUDAGuard guard(x.device());
    Tensor y = at::empty(x.sizes(), x.options()), r = at::empty(x.sizes(), x.options().dtype(out_type));
    if (train) stats = at::empty({rows, 4}, x.options().dtype(at::kFloat));
    ssm_block_norm_args a{};
    fill(a);
    a.y = y.data_ptr(), a.residual_out = r.data_ptr();
    run(ssm_block_norm_fwd(&a, stream_of(x)));
    return {y, r};
  }
  variable_list backward(const variable_list& grads) override {
    c10::cuda::CUDAGuard guard(x.device());
    const auto like_empty = [&](const Tensor& t) { return rows ? at::empty(t.sizes(), t.options()) : at::zeros(t.sizes(), t.options()); };
    Tensor dy = grads[0].defined() ? like(grads[0], x) : at::zeros(x.sizes(), x.options()), dr;
    if (grads[1].defined()) dr = grads[1].detach().to(out_type).contiguous();
    Tensor dx = like_empty(x), dpw = like_empty(pw), dw = like_empty(w), dres, dpb, db, dgate;
    if (res.has_value()) dres = like_empty(*res);
    if (has_pb) dpb = like_empty(w);
    if (has_b) db = like_empty(w);
    if (gate.has_value()) dgate = like_empty(*gate);
    Tensor partial = at::empty({ssm_block_norm_bwd_scratch_floats(rows, (int)dim)}, x.options().dtype(at::kFloat));
    ssm_block_norm_bwd_args g{};
    fill(g.fwd);
    auto p = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
    g.dy = p(dy), g.dresidual_out = p(dr), g.dx = p(dx), g.dresidual = p(dres), g.dpost_weight = p(dpw), g.dweight = p(dw), g.dpost_bias = p(dpb), g.dbias = p(db), g.dgate = p(dgate);
    g.partial = partial.data_ptr<float>();
    run(ssm_block_norm_bwd(&g, stream_of(x)));
    variable_list out = {dx};
    if (res.has_value()) out.push_back(cast(dres, t_r));
    out.push_back(cast(dpw, t_pw)), out.push_back(cast(dw, t_w));
    if (has_pb) out.push_back(cast(dpb, t_pb));
    if (has_b) out.push_back(cast(db, t_b));
    if (gate.has_value()) out.push_back(dgate.view(gate_shape));
    return out;
  }
};
py::tuple fused_block_norm(const Tensor& x, const OptTensor& residual, const Tensor& post_weight, const Tensor& weight, const OptTensor& post_bias, const OptTensor& bias, const OptTensor& gate,
                           double scale, bool is_rms, double eps, double post_eps, bool in_fp32) {
  ValueErrors scope;
  const variable_list r = invoke_call(c10::make_intrusive<BlockNormCall>(x, residual, post_weight, weight, post_bias, bias, gate, scale, is_rms, eps, post_eps, in_fp32));
  return py::make_tuple(r[0], r[1]);
}

// ---------------------------------------------------------------------------------------------
// cross entropy from hidden states
// ---------------------------------------------------------------------------------------------
// (..., D) as rows with a stride; copied where the axes before the last do not lie evenly, or lie on one another
Tensor rows_of(const Tensor& t) {
  Tensor d = t.detach();
  int64_t rows = 1;
  for (int64_t i = 0; i + 1 < d.dim(); ++i) rows *= d.size(i);
  d = d.reshape({rows, d.size(-1)});
  return (d.size(1) <= 1 || d.stride(1) == 1) && (d.size(0) <= 1 || d.stride(0) >= d.size(1)) ? d : d.contiguous();
}
struct LinearCeCall final : Call {
  Tensor h, w, targets, stats, packs, dh32, dw32, kept;  // stats, packs: for a second pass; the others: of a pass that formed the gradients too
  std::vector<int64_t> shape, lead_shape;
  at::ScalarType t_w;
  int64_t ignore;
  int reduction;
  bool want_z, grad_h, grad_w;

  LinearCeCall(const Tensor& hidden, const Tensor& weight, const Tensor& targets_, int64_t ignore_, const std::string& reduction_, bool want_z_)
      : t_w(weight.scalar_type()), ignore(ignore_), want_z(want_z_), grad_h(hidden.requires_grad()), grad_w(weight.requires_grad()) {
    SSM_ARG(hidden.dim() >= 1 && weight.dim() == 2 && hidden.size(-1) == weight.size(1), "hidden must have shape (..., D) and weight (V, D).");
    SSM_ARG(weight.size(0) >= 1 && weight.size(1) >= 1, "weight must have at least one row and one column.");
    SSM_ARG(weight.size(0) <= (1 << 28) && weight.size(1) <= (1 << 20), "linear_cross_entropy: V is at most 2^28, D at most 2^20.");
    shape = hidden.sizes().vec(), lead_shape = shape;
    lead_shape.pop_back();
    SSM_ARG(targets_.sizes() == at::IntArrayRef(lead_shape), "targets must have the shape of hidden without the last axis.");
    SSM_ARG(at::isIntegralType(targets_.scalar_type(), false), "targets must be integers.");
    SSM_ARG(targets_.numel() <= (1 << 28), "linear_cross_entropy: more than 2^28 rows.");
    SSM_ARG(reduction_ == "none" || reduction_ == "sum" || reduction_ == "mean", "reduction must be 'none', 'sum' or 'mean'.");
    reduction = reduction_ == "none" ? 0 : reduction_ == "sum" ? 1 : 2;
    same_device(hidden, {&weight, &targets_});
    dtype_code(hidden, "linear_cross_entropy"), dtype_code(weight, "linear_cross_entropy weight");
    input(hidden), input(weight), input(targets_);
    h = rows_of(hidden), w = rows_of(weight.scalar_type() == hidden.scalar_type() ? weight : weight.detach().to(hidden.scalar_type()));
    targets = targets_.detach().to(at::kLong).contiguous();
  }
  int64_t rows() const { return targets.numel(); }
  // A sum or mean is multiplied by one number, which may come later: in bf16 loss and gradients are formed in one pass, 6 N D V operations instead of 8, and dW goes through memory in fp32.
  // Both sides, one pass and two, us: 8192 rows of 50280 x 2560 5334 and 6394, 1000 925 and 918, 300 668 and 517; 2000 rows of 50280 x 768 544 and 524, 400 258 and 214; 24 of 21417 x 1600 200 and
  // 159.  Below a thousand rows or two the other form is the faster one, and this one is taken all the same.
  bool one_pass() const { return reduction && !want_z && h.scalar_type() == at::kBFloat16 && rows() > 0 && (grad_h || grad_w); }
  bool reads(size_t i) const override { return i < 2 && !one_pass(); }  // the targets' part is packed in the first pass
  // fp32 gradients of the whole head, or the packed operands, go with the walk: the node lives as long as the loss does
  bool survives_its_walk() const override { return false; }
  at::TensorOptions f32() const { return h.options().dtype(at::kFloat).requires_grad(false); }
  void fill(ssm_linear_ce_args& a) const {
    a.rows = rows(), a.hidden_stride = rows() > 1 ? h.stride(0) : h.size(1), a.weight_stride = w.size(0) > 1 ? w.stride(0) : w.size(1), a.ignore_index = ignore;
    a.dim = (int)w.size(1), a.vocab = (int)w.size(0), a.io_dtype = dtype_code(h, "linear_cross_entropy"), a.reduction = reduction;
    a.hidden = h.data_ptr(), a.weight = w.data_ptr(), a.targets = targets.data_ptr<int64_t>();
    if (stats.defined()) a.stats = stats.data_ptr<float>();
    a.status = ssd_status(h.get_device()).data_ptr<int32_t>();
  }
  Tensor scratch(ssm_linear_ce_args& a, int pass) const {
    Tensor s = at::empty({std::max<int64_t>(ssm_linear_ce_scratch_bytes(&a, pass), 256)}, h.options().dtype(at::kByte));
    a.scratch = s.data_ptr();
    return s;
  }
  variable_list forward(bool train) override {
    c10::cuda::CUDAGuard guard(h.device());
    ssd_poll(h.get_device());  // a wait that ran out in an earlier launch surfaces here, without a synchronisation
    Tensor row_loss = at::empty(lead_shape, f32()), log_z = at::empty(lead_shape, f32()), loss;
    const bool both = train && one_pass();
    if (train && !both) stats = at::empty({std::max<int64_t>(rows(), 1), 4}, f32());
    ssm_linear_ce_args a{};
    fill(a);
    packs = at::empty({std::max<int64_t>(ssm_linear_ce_packs_bytes(&a), 256)}, h.options().dtype(at::kByte));
    a.packs = packs.data_ptr();
    const Tensor s = scratch(a, both ? 2 : 0);
    a.row_loss = row_loss.data_ptr<float>(), a.log_z = log_z.data_ptr<float>();
    if (reduction) loss = at::empty({}, f32()), a.loss = loss.data_ptr<float>();
    if (both) {
      kept = at::empty({4}, f32());
      if (grad_h) dh32 = at::empty(shape, f32());
      if (grad_w) dw32 = at::empty({w.size(0), (w.size(1) + 3) / 4 * 4}, f32());
      run(ssm_linear_ce_train(&a, grad_h ? dh32.data_ptr<float>() : nullptr, grad_w ? dw32.data_ptr<float>() : nullptr, kept.data_ptr<float>(), stream_of(h)));
    } else {
      run(ssm_linear_ce_fwd(&a, stream_of(h)));
    }
    if (both || !train) packs.reset();
    variable_list res = {reduction ? loss : row_loss};
    if (want_z) res.push_back(log_z);
    return res;
  }
  variable_list backward(const variable_list& grads) override {
    c10::cuda::CUDAGuard guard(h.device());
    ssd_poll(h.get_device());
    Tensor gl = grads[0].defined() ? f32c(grads[0]) : reduction ? at::zeros({}, f32()) : at::zeros(lead_shape, f32()), gz, dh, dw;
    if (want_z && grads[1].defined()) gz = f32c(grads[1]);
    if (grad_h) dh = at::empty(shape, h.options());
    if (grad_w) dw = at::empty(w.sizes(), w.options().dtype(t_w));
    if (kept.defined()) {
      const ssm_stream_t st = stream_of(h);
      if (grad_h) run(ssm_linear_ce_scale(dh32.data_ptr<float>(), w.size(1), rows(), (int)w.size(1), kept.data_ptr<float>(), gl.data_ptr<float>(), dh.data_ptr(), dtype_code(dh, "linear_cross_entropy"), st));
      if (grad_w)
        run(ssm_linear_ce_scale(dw32.data_ptr<float>(), dw32.size(1), w.size(0), (int)w.size(1), kept.data_ptr<float>(), gl.data_ptr<float>(), dw.data_ptr(), dtype_code(dw, "linear_cross_entropy weight"), st));
      return {dh, dw, Tensor()};
    }
    ssm_linear_ce_bwd_args b{};
    fill(b.fwd);
    b.fwd.packs = packs.data_ptr();
    const Tensor s = scratch(b.fwd, 1);
    b.dloss = gl.data_ptr<float>(), b.dlog_z = gz.defined() ? gz.data_ptr<float>() : nullptr;
    if (grad_h) b.dhidden = dh.data_ptr();
    if (grad_w) b.dweight = dw.data_ptr(), b.dweight_dtype = dtype_code(dw, "linear_cross_entropy weight");
    run(ssm_linear_ce_bwd(&b, stream_of(h)));
    return {dh, dw, Tensor()};
  }
};
py::object linear_cross_entropy(const Tensor& hidden, const Tensor& weight, const Tensor& targets, int64_t ignore, const std::string& reduction, bool want_z) {
  ValueErrors scope;
  const variable_list r = invoke_call(c10::make_intrusive<LinearCeCall>(hidden, weight, targets, ignore, reduction, want_z));
  if (want_z) return py::make_tuple(r[0], r[1]);
  return py::cast(r[0]);
}

// ---------------------------------------------------------------------------------------------
// the norm over many tensors, and clipping by it
// ---------------------------------------------------------------------------------------------
// Whether two tensors whose spans overlap share no byte all the same, as columns of one matrix do.  Modulo a stride S of either, axes whose strides are multiples of S move nothing, and the
// others cover a run of bytes: runs that do not meet on the circle of S are proof.
bool lie_apart(const Tensor& a, const Tensor& b) {
  const auto run = [](const Tensor& t, int64_t period) {
    int64_t bytes = t.element_size();
    for (int64_t i = 0; i < t.dim(); ++i) {
      const int64_t stride = t.stride(i) * t.element_size();
      if (stride % period != 0) bytes += (t.size(i) - 1) * stride;
    }
    return bytes;
  };
  for (const Tensor* t : {&a, &b}) {
    for (int64_t i = 0; i < t->dim(); ++i) {
      if (t->size(i) <= 1) continue;
      const int64_t period = t->stride(i) * t->element_size(), runs[2] = {run(a, period), run(b, period)};
      const int64_t at = (int64_t)(reinterpret_cast<uintptr_t>(a.data_ptr()) % period), to = (int64_t)(reinterpret_cast<uintptr_t>(b.data_ptr()) % period);
      const int64_t ahead = (to - at + period) % period;  // from a's run to b's
      if (ahead >= runs[0] && period - ahead >= runs[1]) return true;
    }
  }
  return false;
}

struct TensorList {
  struct Span {
    uintptr_t from, to;
    size_t index;
    bool operator<(const Span& o) const { return from < o.from; }
  };
  std::vector<ssm_tensor_ref> refs;
  std::vector<Tensor> held;                        // dense copies
  std::vector<std::pair<Tensor, Tensor>> strided;  // (given, copy) of those that do not fill their memory
  c10::Device device = c10::Device(c10::kCUDA, 0);

  // A step has a few hundred to a few thousand of them: what is looked at is what lies in the tensor itself (no views, no references; 410 tensors: 114 us with both)
  TensorList(const py::list& tensors, const char* what, bool in_place) {
    const size_t count = tensors.size();
    for (size_t i = 0; i < count; ++i)
      if (!THPVariable_Check(PyList_GET_ITEM(tensors.ptr(), i))) throw py::type_error(std::string(what) + " takes tensors");
    device = count == 0 ? c10::Device(c10::kCUDA, at::cuda::current_device()) : THPVariable_Unpack(PyList_GET_ITEM(tensors.ptr(), 0)).device();
    const bool recorded = at::GradMode::is_enabled();
    std::vector<Span> spans;
    refs.reserve(count);
    if (in_place) spans.reserve(count);
    for (size_t k = 0; k < count; ++k) {
      const Tensor& t = THPVariable_Unpack(PyList_GET_ITEM(tensors.ptr(), k));
      SSM_ARG(t.layout() == c10::kStrided, what, ": sparse tensors are not taken.");
      if (!t.is_cuda() || t.device() != device) same_device(THPVariable_Unpack(PyList_GET_ITEM(tensors.ptr(), 0)), {&t});
      const int type = dtype_code(t, what);
      if (torch::autograd::impl::get_autograd_meta(t)) {
        SSM_ARG(!(recorded && t.requires_grad()), what, ": no gradient flows through it; detach the tensors.");
        TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), "ssm_b200 operators have no forward-mode derivative");
      }
      const int64_t n = t.numel();
      if (n == 0) continue;
      const bool dense = t.is_non_overlapping_and_dense();
      const uintptr_t at = reinterpret_cast<uintptr_t>(t.data_ptr());
      if (in_place) {
        int64_t reach = n - 1;
        if (!dense) {
          reach = 0;
          for (int64_t i = 0; i < t.dim(); ++i) {
            SSM_ARG(t.size(i) <= 1 || t.stride(i) != 0, what, ": a broadcast tensor cannot be scaled in place.");
            reach += (t.size(i) - 1) * t.stride(i);
          }
        }
        spans.push_back(Span{at, at + (uintptr_t)(reach + 1) * t.element_size(), k});
      }
      if (dense) {
        refs.push_back(ssm_tensor_ref{reinterpret_cast<const void*>(at), n, type, 0});
      } else {
        c10::cuda::CUDAGuard guard(device);
        held.push_back(t.detach().contiguous());
        if (in_place) strided.emplace_back(t.detach(), held.back());
        refs.push_back(ssm_tensor_ref{held.back().data_ptr(), n, type, 0});
      }
    }
    if (!std::is_sorted(spans.begin(), spans.end())) std::sort(spans.begin(), spans.end());
    std::vector<Span> open;  // those that reach beyond where the next one begins
    for (const Span& s : spans) {
      open.erase(std::remove_if(open.begin(), open.end(), [&](const Span& o) { return o.to <= s.from; }), open.end());
      for (const Span& o : open)
        SSM_ARG(lie_apart(THPVariable_Unpack(PyList_GET_ITEM(tensors.ptr(), o.index)), THPVariable_Unpack(PyList_GET_ITEM(tensors.ptr(), s.index))), what,
                ": two of the tensors share memory (one given twice would be scaled twice), or lie between one another in a way that is not told from it.");
      open.push_back(s);
    }
  }
};
int max_of(double norm_type) {
  SSM_ARG(norm_type == 2.0 || norm_type == HUGE_VAL, "norm_type must be 2 or inf.");
  return norm_type != 2.0;
}
Tensor global_norm(const py::list& tensors, double norm_type) {
  ValueErrors scope;
  const int kind = max_of(norm_type);
  const TensorList list(tensors, "global_norm", false);
  c10::cuda::CUDAGuard guard(list.device);
  const auto bytes = at::TensorOptions().device(list.device).dtype(at::kByte);
  const int64_t n = (int64_t)list.refs.size();
  Tensor norm = at::empty({}, bytes.dtype(at::kFloat)), scratch = at::empty({ssm_global_norm_scratch_bytes(n)}, bytes);
  run(ssm_global_norm(list.refs.data(), n, kind, scratch.data_ptr(), norm.data_ptr<float>(), stream_of(norm)));
  return norm;
}
Tensor clip_global_norm_(const py::list& tensors, double max_norm, double norm_type) {
  ValueErrors scope;
  const int kind = max_of(norm_type);
  SSM_ARG(max_norm >= 0, "max_norm must not be negative.");
  TensorList list(tensors, "clip_global_norm_", true);
  c10::cuda::CUDAGuard guard(list.device);
  const auto bytes = at::TensorOptions().device(list.device).dtype(at::kByte);
  const int64_t n = (int64_t)list.refs.size();
  Tensor norm = at::empty({}, bytes.dtype(at::kFloat)), scratch = at::empty({ssm_global_norm_scratch_bytes(n)}, bytes);
  run(ssm_clip_global_norm(list.refs.data(), n, kind, (float)max_norm, scratch.data_ptr(), norm.data_ptr<float>(), stream_of(norm)));
  for (const auto& s : list.strided) s.first.copy_(s.second);
  for (size_t k = 0; k < tensors.size(); ++k) {
    const Tensor& t = THPVariable_Unpack(PyList_GET_ITEM(tensors.ptr(), k));
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();  // a graph that keeps one of them for its backward pass notices
  }
  return norm;
}

}  // namespace

void bind_training_operators(py::module& m) {
  auto ops = m.attr("operators").cast<py::module>();
  ops.def("fused_block_norm", &fused_block_norm);
  ops.def("linear_cross_entropy", &linear_cross_entropy);
  ops.def("global_norm", &global_norm);
  ops.def("clip_global_norm_", &clip_global_norm_);
}

}  // namespace ssm_ext
