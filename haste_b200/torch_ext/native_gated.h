// Host path of the operators of a gated linear recurrence block.  Part of native.cc.
#pragma once

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
  if ((!c.a.N || !c.a.D) && ddecay.defined()) ddecay.zero_();
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

void bind(py::module& m) {
  const py::call_guard<py::gil_scoped_release> free;
  m.def("gated_scan", &gated_scan, free);
  m.def("gated_scan_forward", &gated_scan_forward, free);
  m.def("gated_scan_step", &gated_scan_step, free);
  m.def("gated_scan_backward", &gated_scan_backward, free);
}

}  // namespace gated
