// Host path of the operators of a gated linear recurrence block.  Part of native.cc.
#pragma once

#include <algorithm>

namespace gated {

using namespace state_space;

// ------------------------------------------------------------------ gated_scan
struct Scan {
  haste_b200_gated_scan a{};
  Tensor x, gate, inner, decay, state, lengths;
  Scan(const Tensor& x_, const Tensor& gate_, const OptTensor& decay_, const OptTensor& inner_, const OptTensor& state_,
       const OptTensor& lengths_, bool step = false) {
    dims(x_, "x", step ? 2 : 3);
    const int64_t T = step ? 1 : x_.size(0), N = x_.size(step ? 0 : 1), D = x_.size(-1);
    a.dtype = storage(x_);
    shape(gate_, "gate", {T, N, D}, step);
    type(gate_, "gate", x_.scalar_type());
    decay = given(decay_); inner = given(inner_); state = given(state_);
    if (decay.defined()) { shape(decay, "decay", {D}); type(decay, "decay", at::kFloat); }
    if (inner.defined()) { shape(inner, "input_gate", {T, N, D}, step); type(inner, "input_gate", x_.scalar_type()); }
    if (state.defined()) { shape(state, "state", {N, D}); type(state, "state", at::kFloat); }
    lengths = row_lengths(lengths_, N);
    devices(x_, {gate_, decay, inner, state, lengths});
    x = unit_strided(x_); gate = unit_strided(gate_); inner = unit_strided(inner);
    decay = contiguous(decay); state = contiguous(state);
    a.T = limited(T, "T"); a.N = limited(N, "N"); a.D = limited(D, "D");
    a.x = view(x, step); a.gate = view(gate, step); a.input_gate = view(inner, step);
    a.decay = data<float>(decay); a.state = data<float>(state);
    a.lengths = data<long long>(lengths);
  }
};

// `checkpoints`: whether a backward pass will follow.
std::tuple<Tensor, Tensor, OptTensor> gated_scan_forward(const Tensor& x, const Tensor& gate, const OptTensor& decay,
                                                         const OptTensor& inner, const OptTensor& state,
                                                         const OptTensor& lengths, bool checkpoints) {
  Scan c(x, gate, decay, inner, state, lengths);
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor y = output(c.x), last = at::empty({c.a.N, c.a.D}, x.options().dtype(at::kFloat)), saved, scratch;
  c.a.y = view(y);
  c.a.final_state = data<float>(last);
  if (checkpoints) {
    saved = floats(x, lib.gated_scan_checkpoints(&c.a));
    c.a.checkpoints = data<float>(saved);
  }
  if (const long long n = lib.gated_scan_scratch(&c.a, 0)) {
    scratch = floats(x, n);
    c.a.scratch = data<float>(scratch);
  }
  CALL(gated_scan_forward, &c.a, stream());
  return {y, last, maybe(saved)};
}

// One token: x, gate, input_gate [N,D].
std::tuple<Tensor, Tensor> gated_scan_step(const Tensor& x, const Tensor& gate, const Tensor& state, const OptTensor& decay,
                                           const OptTensor& inner, const OptTensor& out_state) {
  Scan c(x, gate, decay, inner, state, {}, true);
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor y = at::empty({c.a.N, c.a.D}, x.options());
  Tensor last = state_buffer(out_state, x, c.state, {c.x, c.gate, c.decay, c.inner}, {c.a.N, c.a.D}, at::kFloat);
  c.a.y = view(y, true);
  c.a.final_state = data<float>(last);
  CALL(gated_scan_forward, &c.a, stream());
  return {y, last};
}

// Gradients of x, gate, decay, input_gate, state (those of the optional ones where they are given).
std::vector<OptTensor> gated_scan_backward(const Tensor& x, const Tensor& gate, const OptTensor& decay, const OptTensor& inner,
                                           const OptTensor& state, const OptTensor& lengths, const Tensor& checkpoints,
                                           const Tensor& dy_, const OptTensor& dfinal_) {
  Scan c(x, gate, decay, inner, state, lengths);
  shape(dy_, "dy", {c.a.T, c.a.N, c.a.D});
  type(dy_, "dy", x.scalar_type());
  Tensor dfinal = given(dfinal_);
  if (dfinal.defined()) {
    shape(dfinal, "dfinal_state", {c.a.N, c.a.D});
    type(dfinal, "dfinal_state", at::kFloat);
  }
  type(checkpoints, "checkpoints", at::kFloat);
  shape(checkpoints, "checkpoints", {lib.gated_scan_checkpoints(&c.a)});
  devices(x, {dy_, dfinal, checkpoints});
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor saved = checkpoints.contiguous(), dy = unit_strided(dy_);
  dfinal = contiguous(dfinal);
  Tensor dx = output(c.x), dgate = output(c.gate), dinner, ddecay, ds;
  if (c.inner.defined()) dinner = output(c.inner);
  if (c.decay.defined()) ddecay = at::empty_like(c.decay);
  if (c.state.defined()) ds = at::empty_like(c.state);
  c.a.dy = view(dy); c.a.dx = view(dx); c.a.dgate = view(dgate); c.a.dinput_gate = view(dinner);
  c.a.checkpoints = data<float>(saved);
  c.a.dfinal_state = data<float>(dfinal);
  c.a.ddecay = data<float>(ddecay); c.a.dstate = data<float>(ds);
  Tensor scratch = floats(x, lib.gated_scan_scratch(&c.a, 1));
  c.a.scratch = data<float>(scratch);
  CALL(gated_scan_backward, &c.a, stream());
  return {dx, dgate, maybe(ddecay), maybe(dinner), maybe(ds)};
}

struct ScanNode : public torch::autograd::Function<ScanNode> {
  static variable_list forward(AutogradContext* ctx, OptTensor lengths, Tensor x, Tensor gate, OptTensor decay, OptTensor inner,
                               OptTensor state) {
    auto [y, last, saved] = gated_scan_forward(x, gate, decay, inner, state, lengths, true);
    ctx->save_for_backward({x, gate, given(decay), given(inner), given(state), given(lengths), given(saved)});
    ctx->set_materialize_grads(false);
    return {y, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    return guarded("gated_scan", [&]() -> variable_list {
      const variable_list v = ctx->get_saved_variables();
      const Tensor dy = grad[0].defined() ? grad[0] : at::zeros_like(v[0]);
      variable_list out(1);
      for (const OptTensor& t :
           gated_scan_backward(v[0], v[1], maybe(v[2]), maybe(v[3]), maybe(v[4]), maybe(v[5]), v[6], dy, maybe(grad[1])))
        out.push_back(given(t));
      return out;
    });
  }
};

std::tuple<Tensor, Tensor> gated_scan(const Tensor& x, const Tensor& gate, const OptTensor& decay, const OptTensor& inner,
                                      const OptTensor& state, const OptTensor& lengths) {
  if (!wants_grad({x, gate, decay, inner, state})) {
    auto [y, last, saved] = gated_scan_forward(x, gate, decay, inner, state, lengths, false);
    return {y, last};
  }
  const variable_list out = ScanNode::apply(lengths, x, gate, decay, inner, state);
  return {out[0], out[1]};
}

// ------------------------------------------------------------------ fused_linear
// The rows of [...,C] in one order: that of the leading axes, or of the first two swapped (a batch-first tensor seen
// time-major), whichever lies in memory with one distance from row to row.
bool one_distance(const Tensor& t, int64_t* ld) {
  const int64_t C = t.size(-1);
  *ld = C;
  int64_t next = -1;  // rows that the axes so far hold, times their distance
  for (int64_t i = t.dim() - 2; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (next < 0) *ld = t.stride(i);
    else if (t.stride(i) != next) return false;
    next = t.stride(i) * t.size(i);
  }
  return *ld >= C;  // (not repeated or overlapping ones)
}
struct Matrix {
  Tensor t;
  int64_t ld;
};
Matrix matrix(Tensor t, bool swapped) {
  if (swapped) t = t.transpose(0, 1);
  int64_t ld;
  if ((t.size(-1) > 1 && t.stride(-1) != 1) || !one_distance(t, &ld)) {
    t = t.contiguous();
    ld = t.size(-1);
  }
  return {t, ld};
}

struct Linear {
  haste_b200_linear a{};
  Tensor weight, bias;
  Matrix x;
  bool swapped = false;
  std::vector<int64_t> sizes;  // of y, in x's order
  Linear(const Tensor& x_, const Tensor& weight_, const OptTensor& bias_, int64_t activation) {
    if (x_.dim() < 1) refuse("x must have a dimension at least, got " + shape_of(x_));
    dims(weight_, "weight", 2);
    const int64_t C = x_.size(-1), H = weight_.size(0);
    a.dtype = a.out_dtype = a.param_dtype = storage(x_);
    if (C < 1 || H < 1 || C >= 1 << 20 || H >= 1 << 20) refuse("weight must have 1 to 2^20 - 1 rows and columns, got " + shape_of(weight_));
    shape(weight_, "weight", {H, C});
    type(weight_, "weight", x_.scalar_type());
    bias = given(bias_);
    if (bias.defined()) {
      shape(bias, "bias", {H});
      type(bias, "bias", x_.scalar_type(), at::kFloat);
      if (bias.scalar_type() == at::kFloat) a.param_dtype = HASTE_B200_F32;
    }
    const int64_t M = x_.numel() / C;
    if (M > 1 << 30) refuse("too many rows: " + shape_of(x_));
    devices(x_, {weight_, bias});
    int64_t ld;
    if (x_.dim() == 3 && x_.numel() && (C == 1 || x_.stride(-1) == 1) && !one_distance(x_, &ld))
      swapped = one_distance(x_.transpose(0, 1), &ld);
    x = matrix(x_, swapped);
    weight = weight_.contiguous();
    bias = contiguous(bias);
    a.activation = (int)activation;
    a.M = (int)M; a.C = (int)C; a.H = (int)H;
    a.x = ptr(x.t); a.x_ld = x.ld;
    a.weight = ptr(weight); a.bias = ptr(bias);
    sizes = x.t.sizes().vec();
    sizes.back() = H;
  }
  Tensor back(const Tensor& t) const { return swapped ? t.transpose(0, 1) : t; }
  // A tensor of y's shape, in x's order.
  Matrix like_y(const Tensor& t, const char* name) {
    std::vector<int64_t> want = sizes;
    if (swapped) std::swap(want[0], want[1]);
    if (t.sizes() != at::IntArrayRef(want)) refuse(std::string(name) + " must have y's shape, got " + shape_of(t));
    return matrix(t, swapped);
  }
};
struct Scratch {
  Tensor t;
  Scratch(const Tensor& x, long long bytes) : t(bytes ? at::empty({bytes}, x.options().dtype(at::kByte)) : Tensor()) {}
  void* get() const { return t.defined() ? t.data_ptr() : nullptr; }
};

// (y, p or None): p, the sums with bias in x's type, [M,H] in x's order of rows, where a backward pass will need it.
std::tuple<Tensor, OptTensor> fused_linear_forward(const Tensor& x, const Tensor& weight, const OptTensor& bias, int64_t activation,
                                                   const OptTensor& residual, bool keep) {
  Linear c(x, weight, bias, activation);
  at::ScalarType out = x.scalar_type();
  Matrix r;
  if (residual) {
    type(*residual, "residual", x.scalar_type(), at::kFloat);
    devices(x, {*residual});
    r = c.like_y(*residual, "residual");
    out = residual->scalar_type();
    c.a.residual = ptr(r.t);
    c.a.residual_ld = r.ld;
    if (out == at::kFloat) c.a.out_dtype = HASTE_B200_F32;
  }
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor y = at::empty(c.sizes, x.options().dtype(out)), pre;
  c.a.y = ptr(y);
  c.a.y_ld = c.a.H;
  if (keep && activation) {
    pre = at::empty({c.a.M, c.a.H}, x.options());
    c.a.pre = ptr(pre);
  }
  const Scratch scratch(x, lib.linear_scratch(&c.a, 0));
  c.a.scratch = scratch.get();
  CALL(linear_forward, &c.a, stream());
  return {c.back(y), maybe(pre)};
}

// Gradients of x, weight and bias, those that are wanted.
std::tuple<OptTensor, OptTensor, OptTensor> fused_linear_backward(const Tensor& x, const Tensor& weight, const OptTensor& bias,
                                                                  int64_t activation, const OptTensor& pre_, const Tensor& dy_,
                                                                  bool want_x, bool want_weight, bool want_bias) {
  Linear c(x, weight, bias, activation);
  type(dy_, "dy", x.scalar_type(), at::kFloat);
  if (dy_.scalar_type() == at::kFloat) c.a.out_dtype = HASTE_B200_F32;
  Tensor pre = given(pre_);
  if (activation) {
    if (!pre.defined()) refuse("an activation's backward pass needs the sums that the forward pass kept");
    shape(pre, "pre", {c.a.M, c.a.H});
    type(pre, "pre", x.scalar_type());
    pre = pre.contiguous();
  }
  devices(x, {dy_, pre});
  const c10::cuda::CUDAGuard guard(x.device());
  const Matrix dy = c.like_y(dy_, "dy");
  c.a.pre = ptr(pre);
  c.a.dy = ptr(dy.t);
  c.a.dy_ld = dy.ld;
  Tensor dx, dw, db;
  if (want_x) {
    dx = at::empty(c.x.t.sizes(), x.options());
    c.a.dx = ptr(dx);
    c.a.dx_ld = c.a.C;
  }
  if (want_weight) {
    dw = at::empty_like(c.weight);
    c.a.dweight = ptr(dw);
  }
  if (want_bias && c.bias.defined()) {
    db = at::empty_like(c.bias);
    c.a.dbias = ptr(db);
  }
  const Scratch scratch(x, lib.linear_scratch(&c.a, 1));
  c.a.scratch = scratch.get();
  CALL(linear_backward, &c.a, stream());
  return {dx.defined() ? OptTensor(c.back(dx)) : OptTensor(), maybe(dw), maybe(db)};
}

struct LinearNode : public torch::autograd::Function<LinearNode> {
  static variable_list forward(AutogradContext* ctx, int64_t activation, Tensor x, Tensor weight, OptTensor bias, OptTensor residual) {
    auto [y, pre] = fused_linear_forward(x, weight, bias, activation, residual, true);
    ctx->save_for_backward({x, weight, given(bias), given(pre)});
    ctx->saved_data["activation"] = activation;
    auto wants = [](const Tensor& t) { return t.defined() && t.requires_grad(); };
    ctx->saved_data["wants"] = (int64_t)(wants(x) | wants(weight) << 1 | wants(given(bias)) << 2 | wants(given(residual)) << 3);
    ctx->set_materialize_grads(false);
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    return guarded("fused_linear", [&]() -> variable_list {
      variable_list out(5);
      if (!grad[0].defined()) return out;
      const variable_list v = ctx->get_saved_variables();
      const int64_t wants = ctx->saved_data["wants"].toInt();
      if (wants & 7) {
        auto [dx, dw, db] = fused_linear_backward(v[0], v[1], maybe(v[2]), ctx->saved_data["activation"].toInt(), maybe(v[3]), grad[0],
                                                  wants & 1, wants & 2, wants & 4);
        out[1] = given(dx); out[2] = given(dw); out[3] = given(db);
      }
      if (wants & 8) out[4] = grad[0];
      return out;
    });
  }
};

Tensor fused_linear(const Tensor& x, const Tensor& weight, const OptTensor& bias, int64_t activation, const OptTensor& residual) {
  if (!wants_grad({x, weight, bias, residual})) return std::get<0>(fused_linear_forward(x, weight, bias, activation, residual, false));
  return LinearNode::apply(activation, x, weight, bias, residual)[0];
}

// ------------------------------------------------------------------ gradients
// Tensors whose elements fill one range of memory, in any order of axes.
haste_b200_gradient range_of(const Tensor& t, const char* name) {
  if (t.layout() != at::kStrided) refuse(std::string(name) + " must be dense tensors, got a sparse one");
  const int dtype = storage(t);
  if (!t.is_non_overlapping_and_dense())
    refuse(std::string(name) + " must fill one range of memory each, got strides over " + shape_of(t));
  return {ptr(t), ptr(t), (long long)t.numel(), dtype, dtype};
}
// Whether the elements of two tensors of one shape lie in the same order (an axis of one element has any stride).
bool lies_like(const Tensor& a, const Tensor& b) {
  for (int64_t i = 0; a.numel() > 1 && i < a.dim(); ++i)
    if (a.size(i) > 1 && a.stride(i) != b.stride(i)) return false;
  return true;
}
struct Span {
  const char *from, *to;
  int gradient;  // number, or -1 - number of an output
};
// What is written must be nobody else's: each output its own gradient's memory, or its own.
void refuse_overlaps(const std::vector<haste_b200_gradient>& g) {
  std::vector<Span> spans;
  spans.reserve(2 * g.size());
  auto add = [&](const void* p, int64_t bytes, int who) {
    if (bytes) spans.push_back({static_cast<const char*>(p), static_cast<const char*>(p) + bytes, who});
  };
  for (size_t i = 0; i < g.size(); ++i) {
    add(g[i].data, g[i].numel * (g[i].dtype == HASTE_B200_F32 ? 4 : 2), (int)i);
    if (g[i].out != g[i].data || g[i].out_dtype != g[i].dtype)
      add(g[i].out, g[i].numel * (g[i].out_dtype == HASTE_B200_F32 ? 4 : 2), -1 - (int)i);
  }
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.from < b.from; });
  const char* written = nullptr;  // end of the last written span so far, and of the last read one
  const char* read = nullptr;
  for (const Span& s : spans) {
    const bool writes = s.gradient < 0 || g[s.gradient].out == g[s.gradient].data;
    if ((written && s.from < written) || (writes && read && s.from < read))
      refuse("gradients overlap in memory with one another or with an output");
    const char*& end = writes ? written : read;
    end = std::max(end, s.to);
  }
}

// The norm of all gradients (a float32 scalar).  With max_norm they are scaled into `out`, or where they are; then a tensor
// that is listed twice counts once.
Tensor clip_gradients(const std::vector<Tensor>& gradients, const c10::optional<double>& max_norm,
                      const c10::optional<std::vector<Tensor>>& out) {
  if (gradients.empty()) refuse("there must be a gradient");
  if (max_norm && !(*max_norm >= 0)) refuse("max_norm must not be negative");
  if (out && out->size() != gradients.size())
    refuse("out must hold as many tensors as there are gradients: " + std::to_string(gradients.size()) + ", got " +
           std::to_string(out->size()));
  if (gradients.size() > INT32_MAX / 2) refuse("too many gradients");
  std::vector<haste_b200_gradient> g;
  g.reserve(gradients.size());
  for (size_t i = 0; i < gradients.size(); ++i) {
    g.push_back(range_of(gradients[i], "gradients"));
    if (!out) continue;
    const Tensor& o = (*out)[i];
    if (o.sizes() != gradients[i].sizes()) refuse("out must have the gradients' shapes, got " + shape_of(o) + " for " + shape_of(gradients[i]));
    const haste_b200_gradient to = range_of(o, "out");
    if (!lies_like(o, gradients[i])) refuse("out must lie in memory like the gradients");
    g.back().out = const_cast<void*>(to.data);
    g.back().out_dtype = to.dtype;
  }
  devices(gradients[0], gradients);
  if (out) devices(gradients[0], *out);
  if (max_norm) {
    if (!out) {
      std::vector<void*> seen;
      for (const Tensor& t : gradients) seen.push_back(t.unsafeGetTensorImpl());
      std::sort(seen.begin(), seen.end());
      if (std::adjacent_find(seen.begin(), seen.end()) != seen.end()) {
        seen.clear();
        size_t n = 0;
        for (size_t i = 0; i < gradients.size(); ++i) {
          if (std::find(seen.begin(), seen.end(), gradients[i].unsafeGetTensorImpl()) != seen.end()) continue;
          seen.push_back(gradients[i].unsafeGetTensorImpl());
          g[n++] = g[i];
        }
        g.resize(n);
      }
    }
    refuse_overlaps(g);
    for (const Tensor& t : out ? *out : gradients)
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  }
  const c10::cuda::CUDAGuard guard(gradients[0].device());
  const at::TensorOptions o = gradients[0].options().dtype(at::kFloat).requires_grad(false);
  Tensor norm = at::empty({}, o), scratch = at::empty({std::max<int64_t>(1, lib.grad_norm_scratch(g.data(), (int)g.size()))}, o);
  float *to = static_cast<float*>(norm.data_ptr()), *with = static_cast<float*>(scratch.data_ptr());
  if (max_norm) CALL(clip_gradients, g.data(), (int)g.size(), (float)*max_norm, to, with, stream());
  else CALL(grad_norm, g.data(), (int)g.size(), to, with, stream());
  return norm;
}

void bind(py::module& m) {
  const py::call_guard<py::gil_scoped_release> free;
  m.def("gated_scan", &gated_scan, free);
  m.def("gated_scan_forward", &gated_scan_forward, free);
  m.def("gated_scan_step", &gated_scan_step, free);
  m.def("gated_scan_backward", &gated_scan_backward, free);
  m.def("fused_linear", &fused_linear, free);
  m.def("fused_linear_forward", &fused_linear_forward, free);
  m.def("fused_linear_backward", &fused_linear_backward, free);
  m.def("clip_gradients", &clip_gradients, free);
}

}  // namespace gated
