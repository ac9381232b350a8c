"""Token-sequence operators: the layer norm of token rows, the short causal convolution and the selective state space
scan, each with its backward pass, and the last two for single tokens.

They are what a state-space restoration block consists of beside its plain matrix products (the reference's training
script builds such a network, model/train.py:35-49; its scan is called at model/basicsr/archs/mambairv2_arch.py:384-390
and mambair_arch.py:356).  Activations are fp32 or bf16 -- all of a call's in one type -- on a ROCm device;
parameters, the scan's state and every sum are fp32.  Sequences are (batch, channel, token) with the tokens contiguous,
which is what an NCHW image is after ``flatten(2)``.  All arithmetic happens in librestormer_hip.so; there is no CPU or
eager fallback.

Inputs of other strides are copied to contiguous ones, as everywhere in this package.  Work goes to the current stream
of the inputs' device, whichever device is current; scratch comes from torch's allocator call by call, so calls on two
streams and captured graphs share none.  Gradients are first-order and reverse-mode only; others are refused.  A
captured backward pass needs what torch needs of any: leaves without a live eager graph (capture a function that calls ``torch.autograd.grad``).
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import ScanDesc, ScanGrads, ScanInputs, check

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
MAX_STATES = 32          # of a channel of the scan
MAX_NORM_WIDTH = 8192
MAX_TOKENS = 1 << 24     # of a row of the scan


# ----------------------------------------------------------------------------
# plumbing
# ----------------------------------------------------------------------------
def _act(t: torch.Tensor, op: str, what: str, like: Optional[torch.Tensor] = None, want: Optional[tuple] = None) -> torch.Tensor:
    """An activation: fp32 or bf16 on a ROCm device, of `like`'s type and device and of the shape `want`."""
    if want is not None and t.shape != want:
        _wrong_shape(t, op, what, want)
    if like is None or t.dtype is not like.dtype or t.device != like.device:     # `like` is one that was looked at
        if not t.is_cuda:
            raise RuntimeError(f"{op} {what}: tensor is on {t.device}; this operator only runs on a ROCm GPU "
                               "(there is no CPU fallback)")
        if t.dtype not in _DTYPES:
            raise RuntimeError(f"{op} {what}: dtype {t.dtype} not supported (fp32 or bf16)")
        if like is not None:
            raise RuntimeError(f"{op} {what}: {t.dtype} on {t.device}, but x is {like.dtype} on {like.device}")
    return t if t.is_contiguous() else t.contiguous()


def _par(t: Optional[torch.Tensor], op: str, what: str, like: torch.Tensor, want: Optional[tuple] = None) -> Optional[torch.Tensor]:
    """A parameter or a state of the scan: fp32 on `like`'s device, of the shape `want`; or None."""
    if t is None:
        return None
    if want is not None and t.shape != want:
        _wrong_shape(t, op, what, want)
    if t.device != like.device:
        raise RuntimeError(f"{op} {what}: tensor is on {t.device}, but x is on {like.device}")
    if t.dtype != torch.float32:
        raise RuntimeError(f"{op} {what}: dtype {t.dtype} not supported (fp32 only)")
    return t if t.is_contiguous() else t.contiguous()


def _wrong_shape(t: torch.Tensor, op: str, what: str, want: tuple) -> None:
    raise RuntimeError(f"{op} {what}: shape {tuple(t.shape)}, expected {tuple(want)}")


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


# (current_stream() and current_device() build objects and look the device up: 2 us a call, 10 us from the autograd thread,
# as much as the smallest kernels)
_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream


def _call(name: str, t: torch.Tensor, *args) -> None:
    """An entry point of the library on `t`'s device and that device's current stream (the last argument)."""
    index = t.device.index
    fn = getattr(_lib.load(), name)
    if index == _device():
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
    if status:
        check(status, name)


def _first_order_only(name: str) -> None:
    if torch.is_grad_enabled():                  # only under create_graph=True
        raise RuntimeError(f"{name}: gradients are first-order only")


def _scratch(nbytes: int, t: torch.Tensor) -> torch.Tensor:
    return torch.empty(nbytes, dtype=torch.uint8, device=t.device)


def _wants_grad(name: str, *tensors) -> bool:
    """Whether a call has to be differentiable.  A dual tensor of forward-mode differentiation has requires_grad == False:
    it is refused, since the way without gradients would drop its tangent."""
    if forward_ad._current_level >= 0:           # inside dual_level(): -1 without one
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{name} has no forward-mode derivative")
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


# tells autograd that a tensor was written to, so that a graph which saved its old values refuses them (torch.autograd.graph's
# increment_version without its argument checks, which take twice as long)
_increment_version = torch._C._increment_version


def _next_state(state: torch.Tensor, state_out: Optional[torch.Tensor], name: str) -> torch.Tensor:
    """Where an update writes the next state: `state` itself, or a tensor of its own."""
    out = state if state_out is None else state_out
    if not out.is_contiguous():
        raise RuntimeError(f"{name}: the state is written in place and has to be contiguous (strides {out.stride()})")
    if state_out is not None:
        if out.shape != state.shape or out.dtype != state.dtype or out.device != state.device:
            raise RuntimeError(f"{name}: state_out is {out.dtype} {tuple(out.shape)} on {out.device}, "
                               f"state {state.dtype} {tuple(state.shape)} on {state.device}")
        gap = abs(out.data_ptr() - state.data_ptr())
        if gap and gap < out.numel() * out.element_size():
            raise RuntimeError(f"{name}: state_out overlaps state")
    return out


# ----------------------------------------------------------------------------
# layer norm of token rows
# ----------------------------------------------------------------------------
def _norm_forward(x, weight, bias, eps):
    y = torch.empty_like(x)
    n, C = x.numel(), x.shape[-1]
    if n:
        _call("rst_rows_norm_fwd", x, x.data_ptr(), _DTYPES[x.dtype], weight.data_ptr(), _ptr(bias), y.data_ptr(), n // C, C, eps)
    return y


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        ctx.save_for_backward(x, weight)
        ctx.with_bias, ctx.eps = bias is not None, eps
        return _norm_forward(x, weight, bias, eps)

    @staticmethod
    def backward(ctx, dy):
        _first_order_only("layernorm")
        x, weight = ctx.saved_tensors
        if x.numel() == 0:
            return torch.zeros_like(x), torch.zeros_like(weight), torch.zeros_like(weight) if ctx.with_bias else None, None
        dy = _act(dy, "layernorm", "dy", x)
        dx, dw = torch.empty_like(x), torch.empty_like(weight)
        db = torch.empty_like(weight) if ctx.with_bias else None
        rows, C = x.numel() // x.shape[-1], x.shape[-1]
        nb = _lib.load().rst_rows_norm_bwd_workspace_bytes(rows, C)
        ws = _scratch(nb, x)
        _call("rst_rows_norm_bwd", x, x.data_ptr(), _DTYPES[x.dtype], weight.data_ptr(), int(ctx.with_bias), dy.data_ptr(),
              dx.data_ptr(), dw.data_ptr(), _ptr(db), rows, C, ctx.eps, ws.data_ptr(), nb)
        return dx, dw, db, None


def layernorm(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over the last dimension of `x` (..., C), C <= 8192: ``(x - mean) / sqrt(var + eps) * weight + bias``, or
    without a `bias` the bias-free norm ``x / sqrt(var + eps) * weight`` (the variance is still the centred one), as
    ``WithBias_LayerNorm`` and ``BiasFree_LayerNorm`` (reference: model/Restromer.py:28-61).  The variance is fp32: rows that
    spread by more than 1e19 are out of range.  `ops.layernorm` is the
    same norm over the channels of an NCHW image."""
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_NORM_WIDTH:
        raise RuntimeError(f"layernorm: x {tuple(x.shape)} (the last dimension: 1 to {MAX_NORM_WIDTH})")
    if not eps >= 0:
        raise RuntimeError(f"layernorm: eps={eps} is negative or no number")
    x, want = _act(x, "layernorm", "x"), x.shape[-1:]
    weight, bias = _par(weight, "layernorm", "weight", x, want), _par(bias, "layernorm", "bias", x, want)
    if _wants_grad("layernorm", x, weight, bias):
        return _LayerNormFn.apply(x, weight, bias, float(eps))
    return _norm_forward(x, weight, bias, float(eps))


# ----------------------------------------------------------------------------
# short causal convolution
# ----------------------------------------------------------------------------
def _conv_forward(x, weight, bias, state, silu, want_state):
    B, D, L = x.shape
    W = weight.shape[1]
    y = torch.empty_like(x)
    end = torch.empty((B, D, W - 1), dtype=x.dtype, device=x.device) if want_state else None
    if x.numel():
        _call("rst_causal_conv1d_fwd", x, x.data_ptr(), _DTYPES[x.dtype], weight.data_ptr(), _ptr(bias), _ptr(state), y.data_ptr(),
              _ptr(end), B, D, L, W, int(silu))
    elif want_state:
        end.zero_() if state is None else end.copy_(state)
    return y, end


class _CausalConvFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, silu, want_state):
        ctx.save_for_backward(x, weight, bias, state)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        y, end = _conv_forward(x, weight, bias, state, silu, want_state)
        return (y, end) if want_state else y

    @staticmethod
    def backward(ctx, dy, dend=None):
        _first_order_only("causal_conv1d")
        x, weight, bias, state = ctx.saved_tensors
        B, D, L = x.shape
        W = weight.shape[1]
        dend = None if dend is None else _act(dend, "causal_conv1d", "final state's gradient", x)
        dstate = None if state is None else torch.empty_like(state)
        if x.numel() == 0:
            if dstate is not None:
                dstate.zero_() if dend is None else dstate.copy_(dend)
            return (torch.zeros_like(x), torch.zeros_like(weight), None if bias is None else torch.zeros_like(bias), dstate, None,
                    None)
        dy = torch.zeros_like(x) if dy is None else _act(dy, "causal_conv1d", "dy", x)
        dx, dw = torch.empty_like(x), torch.empty_like(weight)
        db = None if bias is None else torch.empty_like(bias)
        nb = _lib.load().rst_causal_conv1d_bwd_workspace_bytes(B, D, L)
        ws = _scratch(nb, x)
        _call("rst_causal_conv1d_bwd", x, x.data_ptr(), _DTYPES[x.dtype], weight.data_ptr(), _ptr(bias), _ptr(state), dy.data_ptr(),
              _ptr(dend), dx.data_ptr(), dw.data_ptr(), _ptr(db), _ptr(dstate), B, D, L, W, int(ctx.silu), ws.data_ptr(), nb)
        return dx, dw, db, dstate, None, None


def _conv_args(name, x, weight, bias, activation):
    if activation not in (None, "silu"):
        raise RuntimeError(f"{name}: activation {activation!r} (None or 'silu')")
    x = _act(x, name, "x")
    if weight.dim() == 3 and weight.shape[1] == 1:          # a depthwise nn.Conv1d's
        weight = weight.squeeze(1)
    D = x.shape[1]
    if weight.dim() != 2 or weight.shape[0] != D or not 2 <= weight.shape[1] <= 4:
        raise RuntimeError(f"{name}: weight {tuple(weight.shape)} does not fit {D} channels and 2 to 4 taps")
    return x, _par(weight, name, "weight", x), _par(bias, name, "bias", x, (D,))


def causal_conv1d(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                  initial_state: Optional[torch.Tensor] = None, activation: Optional[str] = None,
                  return_final_state: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Every channel of `x` (B, D, L) convolved with its 2 to 4 taps `weight` (D, W) -- or (D, 1, W), as a depthwise
    ``nn.Conv1d`` has it; the last tap meets the token itself -- plus `bias` (D), then silu if asked.  The tokens before the first are
    `initial_state` (B, D, W-1), or zeros.  With `return_final_state` also the last W-1 inputs, for the next piece or
    `causal_conv1d_update`.  Differentiable in every tensor."""
    if x.dim() != 3:
        raise RuntimeError(f"causal_conv1d: x {tuple(x.shape)} (batch, channel, token)")
    x, weight, bias = _conv_args("causal_conv1d", x, weight, bias, activation)
    if initial_state is not None:
        initial_state = _act(initial_state, "causal_conv1d", "initial_state", x, (x.shape[0], x.shape[1], weight.shape[1] - 1))
    if _wants_grad("causal_conv1d", x, weight, bias, initial_state):
        return _CausalConvFn.apply(x, weight, bias, initial_state, activation == "silu", bool(return_final_state))
    y, end = _conv_forward(x, weight, bias, initial_state, activation == "silu", return_final_state)
    return (y, end) if return_final_state else y


def causal_conv1d_update(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                         activation: Optional[str] = None, state_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """`causal_conv1d` for one token `x` (B, D).  `state` (B, D, W-1) moves on by the token in place, or into
    `state_out` and stays.  Inference only."""
    if x.dim() != 2:
        raise RuntimeError(f"causal_conv1d_update: x {tuple(x.shape)} (batch, channel)")
    if _wants_grad("causal_conv1d_update", x, state, weight, bias, state_out):
        raise RuntimeError("causal_conv1d_update is inference only: call it under torch.no_grad()")
    x, weight, bias = _conv_args("causal_conv1d_update", x, weight, bias, activation)
    B, D, W = x.shape[0], x.shape[1], weight.shape[1]
    out = _next_state(state, state_out, "causal_conv1d_update")
    state = _act(state, "causal_conv1d_update", "state", x, (B, D, W - 1))
    y = torch.empty_like(x)
    if x.numel():
        _call("rst_causal_conv1d_update", x, x.data_ptr(), _DTYPES[x.dtype], state.data_ptr(), out.data_ptr(), weight.data_ptr(),
              _ptr(bias), y.data_ptr(), B, D, W, int(activation == "silu"))
        _increment_version((out,))
    return y


# ----------------------------------------------------------------------------
# selective state space scan
# ----------------------------------------------------------------------------
def _scan_desc(x, A, B, softplus) -> ScanDesc:
    return ScanDesc(x.shape[0], x.shape[1], B.shape[1], A.shape[1], x.shape[2] if x.dim() == 3 else 1, _DTYPES[x.dtype], int(softplus))


def _scan_inputs(x, delta, A, B, C, D, z, delta_bias) -> ScanInputs:
    return ScanInputs(_ptr(x), _ptr(delta), _ptr(A), _ptr(B), _ptr(C), _ptr(D), _ptr(z), _ptr(delta_bias))


def _scan_forward(x, delta, A, B, C, D, z, delta_bias, h0, softplus, want_last, keep):
    """(y, last state or None, states kept for the backward pass or None)"""
    lib = _lib.load()
    y = torch.empty_like(x)
    last = torch.empty((x.shape[0], x.shape[1], A.shape[1]), dtype=torch.float32, device=x.device) if want_last else None
    saved = None
    if x.numel():
        desc, ins = _scan_desc(x, A, B, softplus), _scan_inputs(x, delta, A, B, C, D, z, delta_bias)
        ref = ctypes.byref(desc)
        if keep:
            saved = _scratch(lib.rst_scan_saved_bytes(ref), x)
        nb = lib.rst_scan_workspace_bytes(ref)
        ws = _scratch(nb, x)
        _call("rst_scan_fwd", x, ref, ctypes.byref(ins), _ptr(h0), y.data_ptr(), _ptr(last), _ptr(saved), ws.data_ptr(), nb)
    elif want_last:
        last.zero_() if h0 is None else last.copy_(h0)
    return y, last, saved


class _ScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, delta, A, B, C, D, z, delta_bias, h0, softplus, want_last):
        y, last, saved = _scan_forward(x, delta, A, B, C, D, z, delta_bias, h0, softplus, want_last, True)
        ctx.save_for_backward(x, delta, A, B, C, D, z, delta_bias, saved)
        ctx.has_h0, ctx.softplus = h0 is not None, softplus
        ctx.set_materialize_grads(False)
        return (y, last) if want_last else y

    @staticmethod
    def backward(ctx, dy, dlast=None):
        _first_order_only("selective_scan")
        *ins, saved = ctx.saved_tensors
        x, delta, A, B, C, D, z, delta_bias = ins
        dlast = _par(dlast, "selective_scan", "last state's gradient", x)
        dh0 = torch.empty((x.shape[0], x.shape[1], A.shape[1]), dtype=torch.float32, device=x.device) if ctx.has_h0 else None
        if x.numel() == 0:
            if dh0 is not None:
                dh0.zero_() if dlast is None else dh0.copy_(dlast)
            return tuple(None if t is None else torch.zeros_like(t) for t in ins) + (dh0, None, None)
        dy = torch.zeros_like(x) if dy is None else _act(dy, "selective_scan", "dy", x)
        grads = [None if t is None else torch.empty_like(t) for t in ins]
        desc, inputs, outs = _scan_desc(x, A, B, ctx.softplus), _scan_inputs(*ins), ScanGrads(*[_ptr(g) for g in grads])
        ref = ctypes.byref(desc)
        nb = _lib.load().rst_scan_bwd_workspace_bytes(ref)
        ws = _scratch(nb, x)
        _call("rst_scan_bwd", x, ref, ctypes.byref(inputs), saved.data_ptr(), dy.data_ptr(), _ptr(dlast), ctypes.byref(outs), _ptr(dh0),
              ws.data_ptr(), nb)
        return tuple(grads) + (dh0, None, None)


def _scan_args(name, x, delta, A, B, C, D, z, delta_bias):
    x = _act(x, name, "x")
    size = x.shape
    chan, dims = size[1], len(size)
    if A.dim() != 2 or A.shape[0] != chan or not 1 <= A.shape[1] <= MAX_STATES:
        raise RuntimeError(f"{name}: A {tuple(A.shape)} does not fit {chan} channels and 1 to {MAX_STATES} states")
    if B.dim() == dims:                                      # one group: (B, N, L) for (B, 1, N, L)
        B = B.unsqueeze(1)
    if C.dim() == dims:
        C = C.unsqueeze(1)
    groups = B.shape[1] if B.dim() == dims + 1 else 0
    if groups < 1 or chan % groups:
        raise RuntimeError(f"{name}: B {tuple(B.shape)}: {chan} channels are not divisible into its groups")
    want = (size[0], groups, A.shape[1]) + size[2:]
    return (x, _act(delta, name, "delta", x, size), _par(A, name, "A", x), _act(B, name, "B", x, want),
            _act(C, name, "C", x, want), _par(D, name, "D", x, (chan,)), None if z is None else _act(z, name, "z", x, size),
            _par(delta_bias, name, "delta_bias", x, (chan,)))


def selective_scan(x: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                   D: Optional[torch.Tensor] = None, *, z: Optional[torch.Tensor] = None,
                   delta_bias: Optional[torch.Tensor] = None, delta_softplus: bool = False,
                   initial_state: Optional[torch.Tensor] = None,
                   return_last_state: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """The state space scan with token-dependent step sizes, inputs and outputs: with ``dt = softplus(delta +
    delta_bias)`` (or without the softplus),

        h_t = exp(dt_t A) h_{t-1} + dt_t x_t B_t,     y_t = <C_t, h_t> + D x_t,     times silu(z_t) with a `z`

    `x`, `delta`, `z`: (batch, channel, token).  `A`: (channel, state), up to 32 states.  `B`, `C`: (batch, group, state,
    token), channel d reads group ``d // (channels / groups)`` -- or (batch, state, token) for one group.  `D`,
    `delta_bias`: (channel).  `initial_state` and, with `return_last_state`, the second result: (batch, channel, state),
    fp32.  At most 2^24 tokens a call.  A token leaves the state alone where its step size is zero (`delta` = -inf under the softplus, and finite
    values in the other tensors, `dy` included): that is how sequences of different lengths are padded.  A rate in `A` may be
    -inf, a state that every token with a step size above 1e-28 forgets.  batch x groups: at most 65535.  Differentiable in every tensor; for that the states
    of every 16th token are kept.  Counterpart in the reference: the scan that model/basicsr/archs/mambairv2_arch.py:384-390
    calls, with the same order of its first six arguments."""
    if x.dim() != 3:
        raise RuntimeError(f"selective_scan: x {tuple(x.shape)} (batch, channel, token)")
    if x.shape[2] > MAX_TOKENS:
        raise RuntimeError(f"selective_scan: {x.shape[2]} tokens (at most {MAX_TOKENS}: carry the state on in pieces)")
    args = _scan_args("selective_scan", x, delta, A, B, C, D, z, delta_bias)
    x, A = args[0], args[2]
    h0 = _par(initial_state, "selective_scan", "initial_state", x, (x.shape[0], x.shape[1], A.shape[1]))
    if _wants_grad("selective_scan", *args, h0):
        return _ScanFn.apply(*args, h0, bool(delta_softplus), bool(return_last_state))
    y, last, _ = _scan_forward(*args, h0, delta_softplus, return_last_state, False)
    return (y, last) if return_last_state else y


def selective_scan_update(state: torch.Tensor, x: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor,
                          C: torch.Tensor, D: Optional[torch.Tensor] = None, *, z: Optional[torch.Tensor] = None,
                          delta_bias: Optional[torch.Tensor] = None, delta_softplus: bool = False,
                          state_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """`selective_scan` for one token: `x`, `delta`, `z` (batch, channel), `B`, `C` (batch, group, state) or (batch,
    state).  `state` (batch, channel, state), fp32, moves on in place, or into `state_out` and stays.  Inference only."""
    if x.dim() != 2:
        raise RuntimeError(f"selective_scan_update: x {tuple(x.shape)} (batch, channel)")
    if _wants_grad("selective_scan_update", state, x, delta, A, B, C, D, z, delta_bias, state_out):
        raise RuntimeError("selective_scan_update is inference only: call it under torch.no_grad()")
    x, delta, A, B, C, D, z, delta_bias = _scan_args("selective_scan_update", x, delta, A, B, C, D, z, delta_bias)
    out = _next_state(state, state_out, "selective_scan_update")
    state = _par(state, "selective_scan_update", "state", x, x.shape + A.shape[1:])
    y = torch.empty_like(x)
    if x.numel():
        desc, ins = _scan_desc(x, A, B, delta_softplus), _scan_inputs(x, delta, A, B, C, D, z, delta_bias)
        _call("rst_scan_update", x, ctypes.byref(desc), ctypes.byref(ins), state.data_ptr(), out.data_ptr(), y.data_ptr())
        _increment_version((out,))
    return y
