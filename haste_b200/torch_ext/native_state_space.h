// Host path of the state space operators: argument checks, allocation and the library call, one C++
// call each.  Part of native.cc.
#pragma once

namespace state_space {

using OptTensor = c10::optional<Tensor>;

[[noreturn]] void refuse(const std::string& what) { throw py::value_error("haste_b200: " + what); }

void shape(const Tensor& t, const char* name, std::initializer_list<int64_t> want, bool step = false) {
  at::IntArrayRef w(want.begin(), want.size());
  if (step) w = w.slice(1);  // without the axis of time
  if (t.sizes() != w) {
    std::string s = "[";
    for (int64_t n : w) s += (s.size() > 1 ? "," : "") + std::to_string(n);
    refuse(std::string(name) + " must be " + s + "], got " + shape_of(t));
  }
}
void dims(const Tensor& t, const char* name, int64_t n) {
  if (t.dim() != n) refuse(std::string(name) + " must have " + std::to_string(n) + " dimensions, got " + shape_of(t));
}
void type(const Tensor& t, const char* name, at::ScalarType a, at::ScalarType b) {
  if (t.scalar_type() != a && t.scalar_type() != b)
    throw py::type_error("haste_b200: " + std::string(name) + " must be " + c10::toString(a) +
                         (a == b ? "" : std::string(" or ") + c10::toString(b)) + ", got " + c10::toString(t.scalar_type()));
}
void type(const Tensor& t, const char* name, at::ScalarType a) { type(t, name, a, a); }

int storage(const Tensor& x) {
  switch (x.scalar_type()) {
    case at::kFloat: return HASTE_B200_F32;
    case at::kBFloat16: return HASTE_B200_BF16;
    case at::kHalf: return HASTE_B200_F16;
    default: throw py::type_error(std::string("haste_b200 supports float32, bfloat16 and float16 sequences, got ") +
                                  c10::toString(x.scalar_type()));
  }
}
int limited(int64_t n, const char* name) {
  if (n > INT32_MAX) refuse(std::string(name) + " is too large");
  return (int)n;
}
// Every tensor on x's device.  (After the shapes, so that a call with wrong shapes says so anywhere.)
void devices(const Tensor& x, at::ArrayRef<Tensor> ts) {
  TORCH_CHECK(x.is_cuda(), "haste_b200: tensor must be a CUDA tensor");
  for (const Tensor& t : ts) {
    if (!t.defined()) continue;
    TORCH_CHECK(t.is_cuda(), "haste_b200: tensor must be a CUDA tensor");
    TORCH_CHECK(t.device() == x.device(), "haste_b200: all tensors must share one device");
  }
}
Tensor given(const OptTensor& t) { return t ? *t : Tensor(); }
OptTensor maybe(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
Tensor contiguous(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
// [T,N,...], or one step of it, [N,...].
haste_b200_sequence view(const Tensor& t, bool step = false) {
  if (!t.defined() || !t.numel()) return {nullptr, 0, 0};
  return {t.data_ptr(), step ? 0 : t.stride(0), t.stride(step ? 0 : 1)};
}
// An output [T,N,...] that lies like `like`: time-major, or batch-first where that one is.
Tensor output(const Tensor& like, std::vector<int64_t> sizes, at::TensorOptions o) {
  if (like.size(0) > 1 && like.size(1) > 1 && like.stride(0) < like.stride(1)) {
    std::swap(sizes[0], sizes[1]);
    return at::empty(sizes, o).transpose(0, 1);
  }
  return at::empty(sizes, o);
}
Tensor output(const Tensor& like) { return output(like, like.sizes().vec(), like.options()); }
// The kernels take any strides but along the last axis.  A copy lies like the original, and so do outputs.
Tensor unit_strided(const Tensor& t) {
  if (!t.defined() || t.size(-1) <= 1 || t.stride(-1) == 1) return t;
  return t.dim() < 3 ? t.contiguous() : output(t).copy_(t);
}
template <typename T>
T* data(const Tensor& t) { return t.defined() && t.numel() ? static_cast<T*>(t.data_ptr()) : nullptr; }
Tensor floats(const Tensor& x, int64_t n) { return at::empty({n}, x.options().dtype(at::kFloat)); }

Tensor row_lengths(const OptTensor& t, int64_t N) {
  if (!t) return {};
  shape(*t, "lengths", {N});
  type(*t, "lengths", at::kLong, at::kInt);
  return t->to(at::kLong).contiguous();
}

// ------------------------------------------------------------------ causal_conv1d
struct Conv {
  haste_b200_causal_conv1d a{};
  Tensor x, weight, bias, state, lengths;
  Conv(const Tensor& x_, const Tensor& weight_, const OptTensor& bias_, const OptTensor& state_,
       const OptTensor& lengths_, bool silu, bool step = false) {
    dims(x_, "x", step ? 2 : 3);
    dims(weight_, "weight", 2);
    const int64_t T = step ? 1 : x_.size(0), N = x_.size(step ? 0 : 1), D = x_.size(-1), W = weight_.size(1);
    a.dtype = storage(x_);
    if (W < 2 || W > 4) refuse("weight must have 2, 3 or 4 taps, got " + shape_of(weight_));
    shape(weight_, "weight", {D, W});
    type(weight_, "weight", x_.scalar_type(), at::kFloat);
    a.param_dtype = weight_.scalar_type() == at::kFloat ? HASTE_B200_F32 : a.dtype;
    bias = given(bias_);
    if (bias.defined()) {
      shape(bias, "bias", {D});
      type(bias, "bias", weight_.scalar_type());
    }
    state = given(state_);
    if (state.defined()) {
      shape(state, "state", {N, W - 1, D});
      type(state, "state", x_.scalar_type());
    }
    lengths = row_lengths(lengths_, N);
    devices(x_, {weight_, bias, state, lengths});
    x = unit_strided(x_);
    weight = weight_.contiguous();
    bias = contiguous(bias);
    state = contiguous(state);
    a.T = limited(T, "T"); a.N = limited(N, "N"); a.D = limited(D, "D"); a.W = (int)W;
    a.silu = silu;
    a.x = view(x, step);
    a.weight = ptr(weight); a.bias = ptr(bias); a.state = ptr(state);
    a.lengths = data<long long>(lengths);
  }
};

void* stream() { return (void*)c10::cuda::getCurrentCUDAStream().stream(); }

// Whether the memory between two tensors' first and last elements overlaps.
bool overlap(const Tensor& a, const Tensor& b) {
  if (!a.defined() || !b.defined() || !a.numel() || !b.numel()) return false;
  auto end = [](const Tensor& t) {
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    return static_cast<char*>(t.data_ptr()) + (last + 1) * t.element_size();
  };
  return static_cast<char*>(a.data_ptr()) < end(b) && static_cast<char*>(b.data_ptr()) < end(a);
}

// The caller's buffer for the new state, or a new one.  It may be the old state's, which every thread reads
// before it writes; it must not lie over anything else that the call reads.
Tensor state_buffer(const OptTensor& out, const Tensor& like, const Tensor& state, at::ArrayRef<Tensor> read,
                    at::IntArrayRef sizes, at::ScalarType t) {
  if (!out) return at::empty(sizes, like.options().dtype(t));
  if (out->sizes() != sizes) refuse("out_state has the wrong shape: " + shape_of(*out));
  type(*out, "out_state", t);
  devices(like, {*out});
  if (!out->is_contiguous()) refuse("out_state must be contiguous");
  bool over = overlap(*out, state) && out->data_ptr() != state.data_ptr();
  for (const Tensor& r : read) over |= overlap(*out, r);
  if (over) refuse("out_state lies over an input other than the whole state");
  if (!out->is_inference()) out->unsafeGetTensorImpl()->bump_version();  // autograd notices that it changed
  return *out;
}

std::tuple<Tensor, Tensor> causal_conv1d_forward(const Tensor& x, const Tensor& weight, const OptTensor& bias,
                                                 const OptTensor& state, const OptTensor& lengths, bool silu,
                                                 const OptTensor& out_state) {
  Conv c(x, weight, bias, state, lengths, silu);
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor y = output(c.x);
  Tensor last = state_buffer(out_state, x, c.state, {c.x, c.weight, c.bias}, {c.a.N, c.a.W - 1, c.a.D}, x.scalar_type());
  c.a.y = view(y);
  c.a.final_state = ptr(last);
  CALL(causal_conv1d_forward, &c.a, stream());
  return {y, last};
}

// One token: x [N,D].
std::tuple<Tensor, Tensor> causal_conv1d_step(const Tensor& x, const Tensor& weight, const OptTensor& bias,
                                              const Tensor& state, bool silu, const OptTensor& out_state) {
  Conv c(x, weight, bias, state, {}, silu, true);
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor y = at::empty({c.a.N, c.a.D}, x.options());
  Tensor last = state_buffer(out_state, x, c.state, {c.x, c.weight, c.bias}, {c.a.N, c.a.W - 1, c.a.D}, x.scalar_type());
  c.a.y = view(y, true);
  c.a.final_state = ptr(last);
  CALL(causal_conv1d_forward, &c.a, stream());
  return {y, last};
}

// Gradients of x, weight, bias, state (the last two only where given).
std::tuple<Tensor, Tensor, OptTensor, OptTensor> causal_conv1d_backward(
    const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& state, const OptTensor& lengths,
    bool silu, const Tensor& dy_, const OptTensor& dfinal_) {
  Conv c(x, weight, bias, state, lengths, silu);
  shape(dy_, "dy", {c.a.T, c.a.N, c.a.D});
  type(dy_, "dy", x.scalar_type());
  Tensor dfinal = given(dfinal_);
  if (dfinal.defined()) {
    shape(dfinal, "dfinal_state", {c.a.N, c.a.W - 1, c.a.D});
    type(dfinal, "dfinal_state", x.scalar_type());
  }
  devices(x, {dy_, dfinal});
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor dy = unit_strided(dy_), dx = output(c.x), dw = at::empty_like(c.weight), db, ds;
  dfinal = contiguous(dfinal);
  if (c.bias.defined()) db = at::empty_like(c.bias);
  if (c.state.defined()) ds = at::empty_like(c.state);
  if (!c.a.N || !c.a.D) {
    dw.zero_();
    if (db.defined()) db.zero_();
  }
  c.a.dy = view(dy);
  c.a.dx = view(dx);
  c.a.dfinal_state = ptr(dfinal);
  c.a.dweight = ptr(dw); c.a.dbias = ptr(db); c.a.dstate = ptr(ds);
  Tensor scratch = floats(x, lib.causal_conv1d_scratch(&c.a));
  c.a.scratch = data<float>(scratch);
  CALL(causal_conv1d_backward, &c.a, stream());
  return {dx, dw, maybe(db), maybe(ds)};
}

// ------------------------------------------------------------------ selective_scan
struct Scan {
  haste_b200_selective_scan a{};
  Tensor x, dt, A, B, C, skip, z, dt_bias, state, lengths;
  Scan(const Tensor& x_, const Tensor& dt_, const Tensor& A_, const Tensor& B_, const Tensor& C_, const OptTensor& skip_,
       const OptTensor& z_, const OptTensor& dt_bias_, const OptTensor& state_, const OptTensor& lengths_, bool softplus,
       bool step = false) {
    dims(x_, "x", step ? 2 : 3);
    dims(A_, "A", 2);
    const bool grouped = !step || B_.dim() == 3;  // a step's B and C may be [N,S]
    dims(B_, "B", grouped ? (step ? 3 : 4) : 2);
    dims(C_, "C", B_.dim());
    const int64_t T = step ? 1 : x_.size(0), N = x_.size(step ? 0 : 1), D = x_.size(-1), S = A_.size(1),
                  G = grouped ? B_.size(-2) : 1;
    a.dtype = storage(x_);
    if (S < 1 || S > 128) refuse("A must have 1 to 128 states a channel, got " + shape_of(A_));
    if (G < 1 || D % G) refuse("the groups of B must divide the channels: " + std::to_string(G) + " and " + std::to_string(D));
    shape(A_, "A", {D, S});
    shape(dt_, "dt", {T, N, D}, step);
    for (const auto& [t, name] : {std::pair<const Tensor&, const char*>(B_, "B"), {C_, "C"}}) {
      if (grouped) shape(t, name, {T, N, G, S}, step);
      else shape(t, name, {T, N, S}, step);
    }
    skip = given(skip_); z = given(z_); dt_bias = given(dt_bias_); state = given(state_);
    const at::ScalarType t = x_.scalar_type();
    type(dt_, "dt", t);
    type(B_, "B", t);
    type(C_, "C", t);
    type(A_, "A", at::kFloat);
    if (skip.defined()) { shape(skip, "D", {D}); type(skip, "D", at::kFloat); }
    if (z.defined()) { shape(z, "z", {T, N, D}, step); type(z, "z", t); }
    if (dt_bias.defined()) { shape(dt_bias, "dt_bias", {D}); type(dt_bias, "dt_bias", at::kFloat); }
    if (state.defined()) { shape(state, "state", {N, D, S}); type(state, "state", at::kFloat); }
    lengths = row_lengths(lengths_, N);
    devices(x_, {dt_, A_, B_, C_, skip, z, dt_bias, state, lengths});
    x = unit_strided(x_); dt = unit_strided(dt_); z = unit_strided(z); B = unit_strided(B_); C = unit_strided(C_);
    A = A_.contiguous(); skip = contiguous(skip); dt_bias = contiguous(dt_bias); state = contiguous(state);
    a.T = limited(T, "T"); a.N = limited(N, "N"); a.D = limited(D, "D"); a.G = limited(G, "G"); a.S = (int)S;
    a.softplus = softplus;
    a.x = view(x, step); a.dt = view(dt, step); a.z = view(z, step); a.B = view(B, step); a.C = view(C, step);
    a.B_g = grouped ? B.stride(-2) : 0;
    a.C_g = grouped ? C.stride(-2) : 0;
    a.A = data<float>(A); a.skip = data<float>(skip); a.dt_bias = data<float>(dt_bias); a.state = data<float>(state);
    a.lengths = data<long long>(lengths);
  }
};

// `checkpoints`: whether a backward pass will follow.
std::tuple<Tensor, Tensor, OptTensor> selective_scan_forward(
    const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const OptTensor& skip,
    const OptTensor& z, const OptTensor& dt_bias, const OptTensor& state, const OptTensor& lengths, bool softplus,
    bool checkpoints, const OptTensor& out_state) {
  Scan c(x, dt, A, B, C, skip, z, dt_bias, state, lengths, softplus);
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor y = output(c.x), saved, scratch;
  Tensor last = state_buffer(out_state, x, c.state, {c.x, c.dt, c.A, c.B, c.C, c.skip, c.z, c.dt_bias}, {c.a.N, c.a.D, c.a.S},
                             at::kFloat);
  c.a.y = view(y);
  c.a.final_state = data<float>(last);
  if (checkpoints) {
    saved = floats(x, lib.selective_scan_checkpoints(&c.a));
    c.a.checkpoints = data<float>(saved);
  }
  if (const long long n = lib.selective_scan_scratch(&c.a, 0)) {
    scratch = floats(x, n);
    c.a.scratch = data<float>(scratch);
  }
  CALL(selective_scan_forward, &c.a, stream());
  return {y, last, saved.defined() ? OptTensor(saved) : OptTensor()};
}

// One token: x, dt, z [N,D], B, C [N,G,S] or [N,S].
std::tuple<Tensor, Tensor> selective_scan_step(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B,
                                               const Tensor& C, const Tensor& state, const OptTensor& skip,
                                               const OptTensor& z, const OptTensor& dt_bias, bool softplus,
                                               const OptTensor& out_state) {
  Scan c(x, dt, A, B, C, skip, z, dt_bias, state, {}, softplus, true);
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor y = at::empty({c.a.N, c.a.D}, x.options());
  Tensor last = state_buffer(out_state, x, c.state, {c.x, c.dt, c.A, c.B, c.C, c.skip, c.z, c.dt_bias}, {c.a.N, c.a.D, c.a.S},
                             at::kFloat);
  c.a.y = view(y, true);
  c.a.final_state = data<float>(last);
  CALL(selective_scan_forward, &c.a, stream());
  return {y, last};
}

// Gradients of x, dt, A, B, C, D, z, dt_bias, state (those of the optional ones where they are given).
std::vector<OptTensor> selective_scan_backward(
    const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const OptTensor& skip,
    const OptTensor& z, const OptTensor& dt_bias, const OptTensor& state, const OptTensor& lengths, bool softplus,
    const Tensor& checkpoints, const Tensor& dy_, const OptTensor& dfinal_) {
  Scan c(x, dt, A, B, C, skip, z, dt_bias, state, lengths, softplus);
  shape(dy_, "dy", {c.a.T, c.a.N, c.a.D});
  type(dy_, "dy", x.scalar_type());
  Tensor dfinal = given(dfinal_);
  if (dfinal.defined()) {
    shape(dfinal, "dfinal_state", {c.a.N, c.a.D, c.a.S});
    type(dfinal, "dfinal_state", at::kFloat);
  }
  type(checkpoints, "checkpoints", at::kFloat);
  shape(checkpoints, "checkpoints", {lib.selective_scan_checkpoints(&c.a)});
  devices(x, {dy_, dfinal, checkpoints});
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor saved = checkpoints.contiguous(), dy = unit_strided(dy_);
  dfinal = contiguous(dfinal);
  Tensor dx = output(c.x), ddt = output(c.x), dB = output(c.B), dC = output(c.C), dz, dA = at::empty_like(c.A), dskip, dbias, ds;
  if (c.z.defined()) dz = output(c.x);
  if (c.skip.defined()) dskip = at::empty_like(c.skip);
  if (c.dt_bias.defined()) dbias = at::empty_like(c.dt_bias);
  if (c.state.defined()) ds = at::empty_like(c.state);
  if (!c.a.N || !c.a.D) {
    for (Tensor t : {dB, dC, dA, dskip, dbias})
      if (t.defined()) t.zero_();
  }
  c.a.dy = view(dy); c.a.dx = view(dx); c.a.ddt = view(ddt); c.a.dz = view(dz); c.a.dB = view(dB); c.a.dC = view(dC);
  c.a.dB_g = dB.stride(2); c.a.dC_g = dC.stride(2);
  c.a.checkpoints = data<float>(saved);
  c.a.dfinal_state = data<float>(dfinal);
  c.a.dA = data<float>(dA); c.a.dskip = data<float>(dskip); c.a.ddt_bias = data<float>(dbias); c.a.dstate = data<float>(ds);
  Tensor scratch = floats(x, lib.selective_scan_scratch(&c.a, 1));
  c.a.scratch = data<float>(scratch);
  CALL(selective_scan_backward, &c.a, stream());
  std::vector<OptTensor> out;
  for (const Tensor& t : {dx, ddt, dA, dB, dC, dskip, dz, dbias, ds}) out.push_back(t.defined() ? OptTensor(t) : OptTensor());
  return out;
}

// ------------------------------------------------------------------ fused_norm
struct Norm {
  haste_b200_fused_norm a{};
  Tensor x, weight, bias, gate, residual, scale;
  Norm(const Tensor& x_, const Tensor& weight_, const OptTensor& bias_, const OptTensor& gate_, const OptTensor& residual_,
       const OptTensor& scale_, double eps, bool layer_norm) {
    dims(x_, "x", 3);
    const int64_t T = x_.size(0), N = x_.size(1), H = x_.size(2);
    a.dtype = storage(x_);
    if (H < 1 || H > 8192) refuse("rows must have 1 to 8192 values, got " + shape_of(x_));
    if (!(eps >= 0)) refuse("eps must not be negative");
    if (T * N >= INT32_MAX - 65536) refuse("too many rows: " + shape_of(x_));
    shape(weight_, "weight", {H});
    type(weight_, "weight", x_.scalar_type(), at::kFloat);
    bias = given(bias_); gate = given(gate_); residual = given(residual_); scale = given(scale_);
    if (bias.defined()) { shape(bias, "bias", {H}); type(bias, "bias", weight_.scalar_type()); }
    if (gate.defined()) { shape(gate, "gate", {T, N, H}); type(gate, "gate", x_.scalar_type()); }
    if (residual.defined()) { shape(residual, "residual", {T, N, H}); type(residual, "residual", x_.scalar_type(), at::kFloat); }
    if (scale.defined()) {
      if (!residual.defined()) refuse("scale needs a residual");
      shape(scale, "scale", {H});
      type(scale, "scale", weight_.scalar_type());
    }
    devices(x_, {weight_, bias, gate, residual, scale});
    x = unit_strided(x_); gate = unit_strided(gate); residual = unit_strided(residual);
    weight = weight_.contiguous(); bias = contiguous(bias); scale = contiguous(scale);
    a.param_dtype = weight.scalar_type() == at::kFloat ? HASTE_B200_F32 : a.dtype;
    a.residual_dtype = residual.defined() && residual.scalar_type() == at::kFloat ? HASTE_B200_F32 : a.dtype;
    a.T = limited(T, "T"); a.N = limited(N, "N"); a.H = (int)H;
    a.layer_norm = layer_norm;
    a.eps = (float)eps;
    a.x = view(x); a.gate = view(gate); a.residual = view(residual);
    a.weight = ptr(weight); a.bias = ptr(bias); a.scale = ptr(scale);
  }
};

// (y, r or None, statistics or None): r = residual + scale x silu(gate) where there is a residual.
std::tuple<Tensor, OptTensor, OptTensor> fused_norm_forward(const Tensor& x, const Tensor& weight, const OptTensor& bias,
                                                            const OptTensor& gate, const OptTensor& residual,
                                                            const OptTensor& scale, double eps, bool layer_norm,
                                                            bool statistics) {
  Norm c(x, weight, bias, gate, residual, scale, eps, layer_norm);
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor y = output(c.x), r, stats;
  if (c.residual.defined()) r = output(c.residual);
  if (statistics) stats = floats(x, 2 * x.size(0) * x.size(1));
  c.a.y = view(y);
  c.a.r = view(r);
  c.a.stats = data<float>(stats);
  CALL(fused_norm_forward, &c.a, stream());
  return {y, maybe(r), maybe(stats)};
}

// Gradients of x, weight, bias, gate, residual, scale (where given).
std::vector<OptTensor> fused_norm_backward(const Tensor& x, const Tensor& weight, const OptTensor& bias,
                                           const OptTensor& gate, const OptTensor& residual, const OptTensor& scale,
                                           double eps, bool layer_norm, const Tensor& stats_, const Tensor& dy_,
                                           const OptTensor& dr_) {
  Norm c(x, weight, bias, gate, residual, scale, eps, layer_norm);
  shape(dy_, "dy", {c.a.T, c.a.N, c.a.H});
  type(dy_, "dy", x.scalar_type());
  Tensor dr = given(dr_);
  if (dr.defined()) {
    if (!c.residual.defined()) refuse("dr needs a residual");
    shape(dr, "dr", {c.a.T, c.a.N, c.a.H});
    type(dr, "dr", c.residual.scalar_type());
  }
  shape(stats_, "statistics", {2 * x.size(0) * x.size(1)});
  type(stats_, "statistics", at::kFloat);
  devices(x, {dy_, dr, stats_});
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor dy = unit_strided(dy_), stats = stats_.contiguous();
  dr = unit_strided(dr);
  Tensor dx = output(c.x), dw = at::empty_like(c.weight), db, dg, dres, ds;
  if (c.bias.defined()) db = at::empty_like(c.bias);
  if (c.gate.defined()) dg = output(c.x);
  if (c.residual.defined()) dres = output(c.residual);
  if (c.scale.defined()) ds = at::empty_like(c.scale);
  c.a.stats = data<float>(stats);
  c.a.dy = view(dy); c.a.dr = view(dr); c.a.dx = view(dx); c.a.dgate = view(dg); c.a.dresidual = view(dres);
  c.a.dweight = ptr(dw); c.a.dbias = ptr(db); c.a.dscale = ptr(ds);
  Tensor scratch = floats(x, lib.fused_norm_scratch(&c.a));
  c.a.scratch = data<float>(scratch);
  CALL(fused_norm_backward, &c.a, stream());
  std::vector<OptTensor> out;
  for (const Tensor& t : {dx, dw, db, dg, dres, ds}) out.push_back(t.defined() ? OptTensor(t) : OptTensor());
  return out;
}

// ------------------------------------------------------------------ with gradients
// One autograd node a call.  The backward pass of a Python function costs a hundred microseconds of host
// work, more than the kernels of a small batch.

bool wants_grad(std::initializer_list<const OptTensor> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const OptTensor& t : ts)
    if (t && t->defined() && t->requires_grad()) return true;
  return false;
}

// Gradients that may be used but not differentiated again: that raises an error instead of giving zeros.
variable_list once(variable_list grads, const char* name) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list some;
  for (const Tensor& t : grads)
    if (t.defined()) some.push_back(t.detach().requires_grad_(true));
  auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string("haste_b200: ") + name + " cannot be differentiated twice", (int64_t)some.size());
  some = (*error)(std::move(some));
  size_t i = 0;
  for (Tensor& t : grads)
    if (t.defined()) t = some[i++];
  return grads;
}

// Runs a backward pass; the library's errors keep their Python type on the way through the engine.
template <typename F>
variable_list guarded(const char* name, const F& f) {
  try {
    variable_list grads;
    {
      const at::AutoGradMode off(false);
      grads = f();
    }
    return once(std::move(grads), name);
  } catch (const LibraryError& e) {
    py::gil_scoped_acquire gil;
    PyErr_SetString(haste_error, e.what());
    python_error error;
    error.persist();
    throw error;
  }
}

struct ConvNode : public torch::autograd::Function<ConvNode> {
  static variable_list forward(AutogradContext* ctx, bool silu, OptTensor lengths, Tensor x, Tensor weight, OptTensor bias,
                               OptTensor state) {
    auto [y, last] = causal_conv1d_forward(x, weight, bias, state, lengths, silu, {});
    ctx->save_for_backward({x, weight, given(bias), given(state), given(lengths)});
    ctx->saved_data["silu"] = silu;
    ctx->set_materialize_grads(false);
    return {y, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    return guarded("causal_conv1d", [&]() -> variable_list {
      const variable_list v = ctx->get_saved_variables();
      const Tensor dy = grad[0].defined() ? grad[0] : at::zeros_like(v[0]);
      auto [dx, dw, db, ds] = causal_conv1d_backward(v[0], v[1], maybe(v[2]), maybe(v[3]), maybe(v[4]),
                                                     ctx->saved_data["silu"].toBool(), dy, maybe(grad[1]));
      return {Tensor(), Tensor(), dx, dw, given(db), given(ds)};
    });
  }
};

std::tuple<Tensor, Tensor> causal_conv1d(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& state,
                                         const OptTensor& lengths, bool silu) {
  if (!wants_grad({x, weight, bias, state})) return causal_conv1d_forward(x, weight, bias, state, lengths, silu, {});
  const variable_list out = ConvNode::apply(silu, lengths, x, weight, bias, state);
  return {out[0], out[1]};
}

struct ScanNode : public torch::autograd::Function<ScanNode> {
  static variable_list forward(AutogradContext* ctx, bool softplus, OptTensor lengths, Tensor x, Tensor dt, Tensor A, Tensor B,
                               Tensor C, OptTensor skip, OptTensor z, OptTensor dt_bias, OptTensor state) {
    auto [y, last, saved] = selective_scan_forward(x, dt, A, B, C, skip, z, dt_bias, state, lengths, softplus, true, {});
    ctx->save_for_backward({x, dt, A, B, C, given(skip), given(z), given(dt_bias), given(state), given(lengths), given(saved)});
    ctx->saved_data["softplus"] = softplus;
    ctx->set_materialize_grads(false);
    return {y, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    return guarded("selective_scan", [&]() -> variable_list {
      const variable_list v = ctx->get_saved_variables();
      const Tensor dy = grad[0].defined() ? grad[0] : at::zeros_like(v[0]);
      variable_list out(2);
      for (const OptTensor& t :
           selective_scan_backward(v[0], v[1], v[2], v[3], v[4], maybe(v[5]), maybe(v[6]), maybe(v[7]), maybe(v[8]),
                                   maybe(v[9]), ctx->saved_data["softplus"].toBool(), v[10], dy, maybe(grad[1])))
        out.push_back(given(t));
      return out;
    });
  }
};

std::tuple<Tensor, Tensor> selective_scan(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C,
                                          const OptTensor& skip, const OptTensor& z, const OptTensor& dt_bias,
                                          const OptTensor& state, const OptTensor& lengths, bool softplus) {
  if (!wants_grad({x, dt, A, B, C, skip, z, dt_bias, state})) {
    auto [y, last, saved] = selective_scan_forward(x, dt, A, B, C, skip, z, dt_bias, state, lengths, softplus, false, {});
    return {y, last};
  }
  const variable_list out = ScanNode::apply(softplus, lengths, x, dt, A, B, C, skip, z, dt_bias, state);
  return {out[0], out[1]};
}

struct NormNode : public torch::autograd::Function<NormNode> {
  static variable_list forward(AutogradContext* ctx, double eps, bool layer_norm, Tensor x, Tensor weight, OptTensor bias,
                               OptTensor gate, OptTensor residual, OptTensor scale) {
    auto [y, r, stats] = fused_norm_forward(x, weight, bias, gate, residual, scale, eps, layer_norm, true);
    ctx->save_for_backward({x, weight, given(bias), given(gate), given(residual), given(scale), given(stats)});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["layer_norm"] = layer_norm;
    ctx->set_materialize_grads(false);
    if (r) return {y, *r};
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    return guarded("fused_norm", [&]() -> variable_list {
      const variable_list v = ctx->get_saved_variables();
      const Tensor dy = grad[0].defined() ? grad[0] : at::zeros_like(v[0]);
      variable_list out(2);
      for (const OptTensor& t :
           fused_norm_backward(v[0], v[1], maybe(v[2]), maybe(v[3]), maybe(v[4]), maybe(v[5]), ctx->saved_data["eps"].toDouble(),
                               ctx->saved_data["layer_norm"].toBool(), v[6], dy, grad.size() > 1 ? maybe(grad[1]) : OptTensor()))
        out.push_back(given(t));
      return out;
    });
  }
};

std::tuple<Tensor, OptTensor> fused_norm(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& gate,
                                         const OptTensor& residual, const OptTensor& scale, double eps, bool layer_norm) {
  if (!wants_grad({x, weight, bias, gate, residual, scale})) {
    auto [y, r, stats] = fused_norm_forward(x, weight, bias, gate, residual, scale, eps, layer_norm, false);
    return {y, r};
  }
  const variable_list out = NormNode::apply(eps, layer_norm, x, weight, bias, gate, residual, scale);
  return {out[0], out.size() > 1 ? OptTensor(out[1]) : OptTensor()};
}

void bind(py::module& m) {
  const py::call_guard<py::gil_scoped_release> free;
  m.def("causal_conv1d_forward", &causal_conv1d_forward, free);
  m.def("causal_conv1d", &causal_conv1d, free);
  m.def("selective_scan", &selective_scan, free);
  m.def("fused_norm", &fused_norm, free);
  m.def("causal_conv1d_step", &causal_conv1d_step, free);
  m.def("selective_scan_step", &selective_scan_step, free);
  m.def("causal_conv1d_backward", &causal_conv1d_backward, free);
  m.def("selective_scan_forward", &selective_scan_forward, free);
  m.def("selective_scan_backward", &selective_scan_backward, free);
  m.def("fused_norm_forward", &fused_norm_forward, free);
  m.def("fused_norm_backward", &fused_norm_backward, free);
}

}  // namespace state_space
