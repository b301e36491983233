"""Operators of state space and gated linear recurrence blocks, with gradients, and for single tokens.

    x = ssm.causal_conv1d(x, w, b)[0]              # short causal convolution and SiLU
    y, h = ssm.selective_scan(x, dt, A, B, C, D=D, z=z, dt_bias=dt_bias)
    y, h = ssm.gated_scan(x, gate, decay=decay, input_gate=i)     # one state a channel, gates as inputs
    y = ssm.fused_norm(y, weight, gate=z)[0]       # norm behind a block, or in front of one
    r = ssm.fused_linear(y, w, b, activation="silu", residual=r)  # projection into a block, or back

and `causal_conv1d_step` / `selective_scan_step` / `gated_scan_step` where tokens come one at a time.  The state that a
call returns is what the next one takes, so a prompt may be cut anywhere and followed by steps.

Sequences are [T,N,...] in float32, bfloat16 or float16; a batch-first tensor goes in as a transposed
view, halves of a projection as slices, and outputs lie like their inputs.  Arithmetic, sums and the
scan's state are float32.  `lengths` ([N] integers) ends rows early: from there on nothing is read,
outputs and gradients are zero, and the returned state is the one at the row's own end.  The
operators run on CUDA only, on the current stream, deterministically, and may be captured in graphs.
The reference has no counterpart of them.
"""
import torch
import torch.autograd.forward_ad as _forward_ad
from torch.autograd.function import once_differentiable

from . import _C, ops

__all__ = ["causal_conv1d", "causal_conv1d_step", "selective_scan", "selective_scan_step", "gated_scan", "gated_scan_step", "fused_norm",
           "fused_linear"]


_tracing_state = torch._C._get_tracing_state


def _shown():
    """Whether the tracer or forward-mode AD looks on: the compiled nodes do not show them what they
    do, the autograd functions below say what can be recorded or differentiated."""
    return _forward_ad._current_level >= 0 or _tracing_state() is not None


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _lengths(lengths, x):
    return torch.as_tensor(lengths, device=x.device)


_native = _C.native


def _float(t):
    return t if t is None or t.dtype == torch.float32 else t.float()


def _pick(ctx, first, grads):
    """The gradients that autograd asked for; `first` arguments in front of them have none."""
    return tuple(g if ctx.needs_input_grad[first + i] else None for i, g in enumerate(grads))


class _CausalConv1d(torch.autograd.Function):
    @staticmethod
    def forward(ctx, silu, lengths, x, weight, bias, state):
        y, last = ops.causal_conv1d_forward(x, weight, bias, state, lengths, silu)
        ctx.save_for_backward(x, weight, bias, state, lengths)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, weight, bias, state, lengths = ctx.saved_tensors
        dy = torch.zeros_like(x) if dy is None else dy
        return (None, None, *_pick(ctx, 2, ops.causal_conv1d_backward(x, weight, bias, state, lengths, ctx.silu, dy, dlast)))


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, softplus, lengths, x, dt, A, B, C, D, z, dt_bias, state):
        y, last, saved = ops.selective_scan_forward(x, dt, A, B, C, D, z, dt_bias, state, lengths, softplus, True)
        ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, state, lengths, saved)
        ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        *inputs, lengths, saved = ctx.saved_tensors
        dy = torch.zeros_like(inputs[0]) if dy is None else dy
        return (None, None, *_pick(ctx, 2, ops.selective_scan_backward(*inputs, lengths, ctx.softplus, saved, dy, dlast)))


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, lengths, x, gate, decay, input_gate, state):
        y, last, saved = ops.gated_scan_forward(x, gate, decay, input_gate, state, lengths, True)
        ctx.save_for_backward(x, gate, decay, input_gate, state, lengths, saved)
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        *inputs, lengths, saved = ctx.saved_tensors
        dy = torch.zeros_like(inputs[0]) if dy is None else dy
        return (None, *_pick(ctx, 1, ops.gated_scan_backward(*inputs, lengths, saved, dy, dlast)))


class _FusedNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, eps, layer_norm, x, weight, bias, gate, residual, scale):
        y, r, stats = ops.fused_norm_forward(x, weight, bias, gate, residual, scale, eps, layer_norm, True)
        ctx.save_for_backward(x, weight, bias, gate, residual, scale, stats)
        ctx.how = eps, layer_norm
        ctx.set_materialize_grads(False)
        return y, r

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dr):
        *inputs, stats = ctx.saved_tensors
        dy = torch.zeros_like(inputs[0]) if dy is None else dy
        return (None, None, *_pick(ctx, 2, ops.fused_norm_backward(*inputs, *ctx.how, stats, dy, dr)))


class _FusedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, activation, x, weight, bias, residual):
        y, sums = ops.fused_linear_forward(x, weight, bias, activation, residual, True)
        ctx.save_for_backward(x, weight, bias, sums)
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, sums = ctx.saved_tensors
        return (None, *_pick(ctx, 1, [*ops.fused_linear_backward(x, weight, bias, ctx.activation, sums, dy), dy]))


def causal_conv1d(x, weight, bias=None, initial_state=None, lengths=None, silu=True):
    """Depthwise causal convolution along time: y_t = act(bias + sum_k weight[:,k] x_{t-(W-1)+k}).

    x [T,N,D], weight [D,W] with 2 to 4 taps, bias [D]; `initial_state` [N,W-1,D] holds the inputs
    before the first (zeros without it).  weight and bias have one type, x's or float32.
    Returns (y, final_state): the last W-1 inputs of each row."""
    if lengths is not None:
        lengths = _lengths(lengths, x)
    if _shown():
        return _CausalConv1d.apply(silu, lengths, x, weight, bias, initial_state)
    return _native().causal_conv1d(x, weight, bias, initial_state, lengths, silu)


def causal_conv1d_step(x, state, weight, bias=None, silu=True, out_state=None):
    """One token: x [N,D].  Returns (y [N,D], new state); the new state goes into `out_state` where
    given, which may be `state` itself."""
    if _shown() or _wants_grad(x, state, weight, bias):
        if out_state is not None:
            raise ValueError("haste_b200: out_state is for calls without gradients")
        if x.dim() != 2:
            raise ValueError(f"haste_b200: x must have 2 dimensions, got {list(x.shape)}")
        y, state = causal_conv1d(x[None], weight, bias, state, silu=silu)
        return y[0], state
    return _native().causal_conv1d_step(x, weight, bias, state, silu, out_state)


def _grouped(m, dims):
    return m.unsqueeze(-2) if m.dim() == dims else m


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, initial_state=None, lengths=None, softplus=True):
    """delta = softplus(dt + dt_bias);  h_t = exp(delta_t A) h_{t-1} + delta_t x_t B_t;
    y_t = (C_t . h_t + D x_t) silu(z_t), per channel with S states.

    x, dt, z [T,N,D], A [D,S] (S up to 128), B, C [T,N,S] or, with G groups of D / G channels,
    [T,N,G,S]; D, dt_bias [D]; x, dt, z, B, C have one type, A, D, dt_bias any (they are taken as float32);
    `initial_state` [N,D,S] float32 (zeros without it).  Without
    `softplus`, delta = dt + dt_bias.  Returns (y, final_state)."""
    if lengths is not None:
        lengths = _lengths(lengths, x)
    A, D, dt_bias = _float(A), _float(D), _float(dt_bias)
    B, C = _grouped(B, 3), _grouped(C, 3)
    if _shown():
        return _SelectiveScan.apply(softplus, lengths, x, dt, A, B, C, D, z, dt_bias, initial_state)
    return _native().selective_scan(x, dt, A, B, C, D, z, dt_bias, initial_state, lengths, softplus)


def selective_scan_step(x, dt, A, B, C, state, D=None, z=None, dt_bias=None, softplus=True, out_state=None):
    """One token: x, dt, z [N,D], B, C [N,S] or [N,G,S], state [N,D,S] float32.  Returns (y [N,D], new
    state); the new state goes into `out_state` where given, which may be `state` itself."""
    A, D, dt_bias = _float(A), _float(D), _float(dt_bias)
    if _shown() or _wants_grad(x, dt, A, B, C, state, D, z, dt_bias):
        if out_state is not None:
            raise ValueError("haste_b200: out_state is for calls without gradients")
        if x.dim() != 2:
            raise ValueError(f"haste_b200: x must have 2 dimensions, got {list(x.shape)}")
        y, state = selective_scan(x[None], dt[None], A, _grouped(B, 2)[None], _grouped(C, 2)[None], D,
                                  None if z is None else z[None], dt_bias, state, softplus=softplus)
        return y[0], state
    return _native().selective_scan_step(x, dt, A, B, C, state, D, z, dt_bias, softplus, out_state)


def gated_scan(x, gate, decay=None, input_gate=None, initial_state=None, lengths=None):
    """r = sigmoid(gate);  with `decay`: log a = decay r, w = sqrt(1 - a^2);  without: a = r, w = 1 - a;
    h_t = a_t h_{t-1} + w_t x_t sigmoid(input_gate_t).  Returns (h of every step, final_state).

    x, gate, input_gate [T,N,D] have one type; decay [D] has any and is taken as float32, values above zero count as
    zero; `initial_state` [N,D] float32 (zeros without it).  In gradients 1 / w is taken as 1 / sqrt(w^2 + 1e-30), and a
    decay of zero leaves w constant."""
    if lengths is not None:
        lengths = _lengths(lengths, x)
    decay = _float(decay)
    if _shown():
        return _GatedScan.apply(lengths, x, gate, decay, input_gate, initial_state)
    return _native().gated_scan(x, gate, decay, input_gate, initial_state, lengths)


def gated_scan_step(x, gate, state, decay=None, input_gate=None, out_state=None):
    """One token: x, gate, input_gate [N,D], state [N,D] float32.  Returns (y [N,D], new state); the new state goes
    into `out_state` where given, which may be `state` itself."""
    decay = _float(decay)
    if _shown() or _wants_grad(x, gate, state, decay, input_gate):
        if out_state is not None:
            raise ValueError("haste_b200: out_state is for calls without gradients")
        if x.dim() != 2:
            raise ValueError(f"haste_b200: x must have 2 dimensions, got {list(x.shape)}")
        y, state = gated_scan(x[None], gate[None], decay, None if input_gate is None else input_gate[None], state)
        return y[0], state
    return _native().gated_scan_step(x, gate, state, decay, input_gate, out_state)


def fused_norm(x, weight, bias=None, gate=None, residual=None, scale=None, eps=1e-5, kind="rms"):
    """u = x silu(gate);  r = residual + scale u;  y = norm(r) weight + bias.

    x, gate, residual [T,N,H] (H up to 8192), the others [H]; each of gate, residual, scale (with a
    residual only) and bias may be absent.  `kind` "rms" divides by the root mean square, "layer" subtracts the mean
    first.  The residual, and r with it, may be float32 beside narrower x; the parameters have one
    type, x's or float32.  Returns (y, r), r None without a residual; r is normalised before it is rounded."""
    if kind not in ("rms", "layer"):
        raise ValueError(f"haste_b200: kind must be 'rms' or 'layer', got {kind!r}")
    layer = kind == "layer"
    if _shown():
        return _FusedNorm.apply(eps, layer, x, weight, bias, gate, residual, scale)
    return _native().fused_norm(x, weight, bias, gate, residual, scale, eps, layer)


def fused_linear(x, weight, bias=None, activation=None, residual=None):
    """act(x weight^T + bias) + residual, in one pass over the product.

    x [...,C], weight [H,C] (as torch.nn.Linear has it) in x's type, bias [H] in that type or float32, residual [...,H]
    in that type or float32, which is then the result's.  `activation` is None, "relu", "silu", "gelu" (x times the
    normal distribution), "tanh" or "sigmoid".  Sums are float32; their gradient is rounded to x's type.
    float32 inputs are multiplied to float32's rounding, those below 2^-110 to within 2^-134; an infinite one makes NaN of
    its row's or column's sums from nine rows on and in gradients, what the formula has in up to eight.  Rows may lie at any
    distance, and time-major views of batch-first tensors are read as they lie."""
    if activation not in ops.ACTIVATIONS:
        raise ValueError(f"haste_b200: activation must be one of {list(ops.ACTIVATIONS)}, got {activation!r}")
    if _shown():
        return _FusedLinear.apply(activation, x, weight, bias, residual)
    return _native().fused_linear(x, weight, bias, ops.ACTIVATIONS[activation], residual)
