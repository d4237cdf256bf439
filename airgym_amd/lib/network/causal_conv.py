"""Short causal depthwise convolution on the HIP kernels of csrc/causal_conv.hip, for sequences and for single steps.

    p[b, t, d] = bias[d] + sum_k weight[d, k] x[b, t - W + 1 + k, d]        y = silu(p) or p

The W - 1 inputs before step 0 are `initial_state` (zeros if None); `resets[b, t]` clears what came before step t (an episode ended),
`lengths[b]` is where a padded sequence ends: later steps give zeros, get no gradient and leave the state alone."""
import ctypes

import torch
from torch.autograd.function import once_differentiable

from airgym_amd import _native as N
from airgym_amd.lib.core.native_call import (activation as first_activation, flags_of, in_place_state, lengths_of, moved_on, no_gradient, nothing,
                                             on_device_of, parameter, ptr, same_kind, shape_error, stream_of)

MAX_TAPS = 8


def _activation(activation):
    if activation not in (None, "silu"):
        raise ValueError(f"activation: None or 'silu' expected, got {activation!r}")
    return int(activation == "silu")


def _fill(x, weight, bias, state, lengths, resets, silu):
    B, T, D = x.shape
    a = N.AgConvArgs(ctypes.sizeof(N.AgConvArgs), N.AG_DTYPES[x.dtype], B, T, D, weight.shape[1], silu, x.data_ptr(), weight.data_ptr(),
                     ptr(bias), ptr(state), ptr(lengths), ptr(resets), x.stride(0), x.stride(1))
    if resets is not None:
        a.r_sb, a.r_st = resets.stride()
    return a


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, lengths, resets, silu, want_state):
        B, T, D = x.shape
        y = torch.empty(B, T, D, dtype=x.dtype, device=x.device)
        last = torch.empty(B, weight.shape[1] - 1, D, dtype=x.dtype, device=x.device) if want_state else None
        a = _fill(x, weight, bias, state, lengths, resets, silu)
        a.y_dev, a.state_out_dev = y.data_ptr(), ptr(last)
        with on_device_of(x):
            N.check(N.load().ag_causal_conv_fwd(ctypes.byref(a), stream_of(x)), "ag_causal_conv_fwd")
        ctx.save_for_backward(x, weight, bias, state, lengths, resets)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, weight, bias, state, lengths, resets = ctx.saved_tensors
        lib = N.load()
        B, T, D = x.shape
        W = weight.shape[1]
        dy = torch.zeros(B, T, D, dtype=x.dtype, device=x.device) if dy is None else same_kind("dy", dy, x.shape, x)
        dlast = None if dlast is None else dlast.contiguous()
        dx, dw = torch.empty(B, T, D, dtype=x.dtype, device=x.device), torch.empty_like(weight)
        db = None if bias is None else torch.empty_like(bias)
        ds = torch.empty_like(state) if ctx.needs_input_grad[3] else None
        n = lib.ag_causal_conv_workspace_bytes(B, T, D, W, N.AG_DTYPES[x.dtype])
        ws = torch.empty(n, dtype=torch.uint8, device=x.device)
        a = _fill(x, weight, bias, state, lengths, resets, ctx.silu)
        g = N.AgConvGrads(ctypes.sizeof(N.AgConvGrads), dy.data_ptr(), ptr(dlast), dy.stride(0), dy.stride(1), dx.data_ptr(), dw.data_ptr(),
                          ptr(db), ptr(ds), ws.data_ptr(), n)
        with on_device_of(x):
            N.check(lib.ag_causal_conv_bwd(ctypes.byref(a), ctypes.byref(g), stream_of(x)), "ag_causal_conv_bwd")
        return dx, dw, db, ds, None, None, None, None


def _weight(weight, D, device):
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or not 2 <= weight.shape[1] <= MAX_TAPS:
        raise shape_error("weight", weight, f"[{D}, W] with 2 to {MAX_TAPS} taps")
    return parameter("weight", weight, (D, weight.shape[1]), device)


def causal_conv(x, weight, bias=None, *, activation="silu", initial_state=None, lengths=None, resets=None, return_state=False):
    """x [B, T, D] (float32, bfloat16 or float16; any batch and time strides), weight [D, W] and bias [D] float32 -> y [B, T, D], and
    with return_state the last W - 1 inputs [B, W - 1, D] (oldest first, x's type) to go on from.  initial_state: the same;
    lengths int32 [B]; resets bool or uint8 [B, T].  Gradients reach x, weight, bias, initial_state, also through the returned state."""
    if not isinstance(x, torch.Tensor) or x.dim() != 3:
        raise shape_error("x", x, "[B, T, D]")
    B, T, D = x.shape
    x = first_activation("x", x, x.shape)
    weight, bias = _weight(weight, D, x.device), parameter("bias", bias, (D,), x.device)
    W = weight.shape[1]
    state = None if initial_state is None else same_kind("initial_state", initial_state, (B, W - 1, D), x).contiguous()
    lengths, resets = lengths_of(lengths, B, x.device), flags_of("resets", resets, (B, T), x.device)
    silu = _activation(activation)
    if x.numel() == 0:
        y, last = nothing(x, weight, bias, state), (x.new_zeros(B, W - 1, D) if state is None else state.clone())
    else:
        y, last = _CausalConv.apply(x, weight, bias, state, lengths, resets, silu, return_state)
    return (y, last) if return_state else y


def causal_conv_step(x, state, weight, bias=None, *, activation="silu", resets=None):
    """One step: x [B, D] -> y [B, D]; state [B, W - 1, D] (contiguous, x's type) is moved on in place.  resets [B] clears a row's
    state first.  No gradients."""
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise shape_error("x", x, "[B, D]")
    B, D = x.shape
    no_gradient("causal_conv_step", x, weight, bias)
    x = first_activation("x", x, x.shape)
    device = x.device
    weight, bias = _weight(weight, D, device), parameter("bias", bias, (D,), device)
    W = weight.shape[1]
    state = in_place_state("state", state, (B, W - 1, D), x.dtype, device)
    resets = flags_of("resets", resets, (B,), device)
    silu = _activation(activation)
    y = torch.empty_like(x) if x.is_contiguous() else torch.empty((B, D), dtype=x.dtype, device=device)      # (half a microsecond apart)
    if x.numel() == 0:
        return y
    if resets is not None and not resets.is_contiguous():
        resets = resets.contiguous()
    with on_device_of(x):
        N.check(N.load().ag_causal_conv_step(x.data_ptr(), x.stride(0), state.data_ptr(), weight.data_ptr(), ptr(bias), ptr(resets),
                                             y.data_ptr(), N.AG_DTYPES[x.dtype], B, D, W, silu, stream_of(x)), "ag_causal_conv_step")
    moved_on(state)
    return y


def causal_conv_torch(x, weight, bias=None, *, activation="silu", initial_state=None, resets=None, return_state=False):
    """The same convolution out of torch ops, step by step (any device; autograd derives the backward): the path of CPU tensors."""
    B, T, D = x.shape
    W = weight.shape[1]
    window = list(x.new_zeros(W - 1, B, D) if initial_state is None else initial_state.unbind(1))
    ys = []
    for t in range(T):
        if resets is not None:
            cut = (resets[:, t] != 0)[:, None]
            window = [torch.where(cut, torch.zeros_like(w), w) for w in window]
        window.append(x[:, t])
        p = sum(w * weight[:, k] for k, w in enumerate(window))
        if bias is not None:
            p = p + bias
        ys.append(p * torch.sigmoid(p) if activation == "silu" else p)
        window.pop(0)
    y = torch.stack(ys, 1)
    return (y, torch.stack(window, 1)) if return_state else y
