"""Selective state space scan on the HIP kernels of csrc/selective_scan.hip, for sequences and for single steps.

    dt = softplus(delta + delta_bias)
    h[b, d, n] <- exp(dt[d] A[d, n]) h[b, d, n] + dt[d] B[n] u[d]        y[d] = sum_n C[n] h[d, n] + D[d] u[d]
    out = y z sigmoid(z)                                                  (y without z)

The state before step 0 is `initial_state` (zeros if None); `resets[b, t]` clears it before step t (an episode ended), `lengths[b]` is
where a padded sequence ends: later steps give zeros, get no gradient and leave the state alone."""
import ctypes

import torch
from torch.autograd.function import once_differentiable

from airgym_amd import _native as N
from airgym_amd.lib.core.native_call import (activation, flags_of, in_place_state, lengths_of, moved_on, no_gradient, nothing, on_device_of,
                                             parameter, ptr, same_kind, shape_error, stream_of, wants_gradient)

MAX_STATES = 32
_ARGS, _GRADS = ctypes.sizeof(N.AgScanArgs), ctypes.sizeof(N.AgScanGrads)


def _groups(t, lead=2):
    """Groups of a B or C ([..., G, N], or [..., N]: one) and its leading and group strides."""
    return (t.shape[lead], t.stride()[:lead + 1]) if t.dim() == lead + 2 else (1, (*t.stride()[:lead], 0))


def _fill(u, delta, A, B, C, D, z, bias, state, lengths, resets, softplus):
    """The argument block of sequences [B, T, ...]."""
    b, T, d = u.shape
    z_sb, z_st = (0, 0) if z is None else z.stride()[:2]
    r_sb, r_st = (0, 0) if resets is None else resets.stride()
    G, b_strides = _groups(B)
    _, c_strides = _groups(C)
    return N.AgScanArgs(_ARGS, N.AG_DTYPES[u.dtype], b, T, d, A.shape[1], G, softplus, u.data_ptr(), delta.data_ptr(), ptr(z),
                        B.data_ptr(), C.data_ptr(), A.data_ptr(), ptr(D), ptr(bias), ptr(state), ptr(lengths), ptr(resets),
                        *u.stride()[:2], *delta.stride()[:2], z_sb, z_st, *b_strides, *c_strides, r_sb, r_st)


def _near_rows(t):
    """t with its steps less than 2^25 elements apart: a tile's rows are addressed with 32 bits."""
    return t if t is None or t.stride(1) < 1 << 25 else t.contiguous()


def _workspace(n, device):
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, B, C, D, z, bias, state, lengths, resets, softplus, want_state, train):
        lib = N.load()
        b, T, d = u.shape
        n = A.shape[1]
        out = torch.empty(b, T, d, dtype=u.dtype, device=u.device)
        last = torch.empty(b, d, n, dtype=torch.float32, device=u.device) if want_state else None
        ckpt = None
        if train:
            ckpt = torch.empty(lib.ag_selective_scan_ckpt_floats(b, T, d, n), dtype=torch.float32, device=u.device)
        bytes_ = lib.ag_selective_scan_workspace_bytes(b, T, d, n, _groups(B)[0], 0)
        ws = _workspace(bytes_, u.device)
        a = _fill(u, delta, A, B, C, D, z, bias, state, lengths, resets, softplus)
        a.out_dev, a.state_out_dev, a.workspace_dev, a.workspace_bytes = out.data_ptr(), ptr(last), ptr(ws), bytes_
        a.ckpt_dev = ptr(ckpt)
        with on_device_of(u):
            N.check(lib.ag_selective_scan_fwd(ctypes.byref(a), stream_of(u)), "ag_selective_scan_fwd")
        ctx.save_for_backward(u, delta, A, B, C, D, z, bias, state, lengths, resets, ckpt)
        ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return out, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dlast):
        u, delta, A, B, C, D, z, bias, state, lengths, resets, ckpt = ctx.saved_tensors
        lib = N.load()
        b, T, d = u.shape
        n, G = A.shape[1], _groups(B)[0]

        dout = torch.zeros(b, T, d, dtype=u.dtype, device=u.device) if dout is None else _near_rows(same_kind("dout", dout, u.shape, u))
        dlast = None if dlast is None else dlast.contiguous()
        du, ddelta, dz, dB, dC = u.new_empty(u.shape), u.new_empty(u.shape), None if z is None else u.new_empty(u.shape), \
            u.new_empty(B.shape), u.new_empty(C.shape)
        dA, dD, dbias = torch.empty_like(A), None if D is None else torch.empty_like(D), None if bias is None else torch.empty_like(bias)
        dstate = torch.empty_like(state) if ctx.needs_input_grad[8] else None
        bytes_ = lib.ag_selective_scan_workspace_bytes(b, T, d, n, G, 1)
        ws = _workspace(bytes_, u.device)
        a = _fill(u, delta, A, B, C, D, z, bias, state, lengths, resets, ctx.softplus)
        a.ckpt_dev = ptr(ckpt)
        g = N.AgScanGrads(_GRADS, dout.data_ptr(), dout.stride(0), dout.stride(1), ptr(dlast), du.data_ptr(),
                          ddelta.data_ptr(), ptr(dz), dB.data_ptr(), dC.data_ptr(), dA.data_ptr(), ptr(dD), ptr(dbias), ptr(dstate),
                          ptr(ws), bytes_)
        with on_device_of(u):
            N.check(lib.ag_selective_scan_bwd(ctypes.byref(a), ctypes.byref(g), stream_of(u)), "ag_selective_scan_bwd")
        return du, ddelta, dA, dB, dC, dD, dz, dbias, dstate, None, None, None, None, None


def _parameters(A, D, delta_bias, d, device):
    if not isinstance(A, torch.Tensor) or A.dim() != 2 or not 1 <= A.shape[1] <= MAX_STATES:
        raise shape_error("A", A, f"[{d}, N] with 1 to {MAX_STATES} states per channel")
    return parameter("A", A, (d, A.shape[1]), device), parameter("D", D, (d,), device), parameter("delta_bias", delta_bias, (d,), device)


def _shared(name, t, lead, n, u):
    """B or C, [..., G, N] or [..., N]: one group."""
    if not isinstance(t, torch.Tensor) or t.dim() not in (len(lead) + 1, len(lead) + 2):
        raise shape_error(name, t, f"{[*lead, 'G', n]} or {[*lead, n]}")
    if t.dim() == len(lead) + 1:
        return same_kind(name, t, (*lead, n), u)
    groups = t.shape[-2]
    if groups < 1 or u.shape[-1] % groups:
        raise ValueError(f"{name}: {u.shape[-1]} channels do not split into {groups} groups")
    return same_kind(name, t, (*lead, groups, n), u)


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, *, delta_softplus=True, initial_state=None, lengths=None,
                   resets=None, return_state=False):
    """u, delta, z [B, T, D] and B, C [B, T, G, N] (or [B, T, N]) in one of float32, bfloat16, float16, with any batch, time and group
    strides; A [D, N], D [D], delta_bias [D] and initial_state [B, D, N] float32; lengths int32 [B]; resets bool or uint8 [B, T].
    G groups of D / G consecutive channels share B and C.  -> out [B, T, D], and with return_state the state [B, D, N] (float32) after
    each sequence's last step.  Gradients reach every floating-point argument, also through the returned state."""
    if not isinstance(u, torch.Tensor) or u.dim() != 3:
        raise shape_error("u", u, "[B, T, D]")
    b, T, d = u.shape
    u = activation("u", u, u.shape)
    delta = same_kind("delta", delta, u.shape, u)
    z = None if z is None else same_kind("z", z, u.shape, u)
    A, D, delta_bias = _parameters(A, D, delta_bias, d, u.device)
    B, C = _shared("B", B, (b, T), A.shape[1], u), _shared("C", C, (b, T), A.shape[1], u)
    if _groups(B)[0] != _groups(C)[0]:
        raise ValueError(f"B and C: {list(B.shape)} and {list(C.shape)}")
    state = parameter("initial_state", initial_state, (b, d, A.shape[1]), u.device)
    lengths, resets = lengths_of(lengths, b, u.device), flags_of("resets", resets, (b, T), u.device)
    if u.numel() == 0:
        out = nothing(u, delta, A, B, C, D, z, delta_bias, state)
        last = torch.zeros(b, d, A.shape[1], dtype=torch.float32, device=u.device) if state is None else state.clone()
    else:
        u, delta, z, B, C = (_near_rows(t) for t in (u, delta, z, B, C))
        out, last = _SelectiveScan.apply(u, delta, A, B, C, D, z, delta_bias, state, lengths, resets, int(bool(delta_softplus)), return_state,
                                         wants_gradient(u, delta, A, B, C, D, z, delta_bias, state))
    return (out, last) if return_state else out


def selective_scan_step(u, delta, A, B, C, state, D=None, z=None, delta_bias=None, *, delta_softplus=True, resets=None):
    """One step: u, delta, z [B, D], B, C [B, G, N] (or [B, N]) -> out [B, D]; state [B, D, N] (float32, contiguous) is moved on in
    place.  resets [B] clears a row's state first.  No gradients."""
    if not isinstance(u, torch.Tensor) or u.dim() != 2:
        raise shape_error("u", u, "[B, D]")
    b, d = u.shape
    no_gradient("selective_scan_step", u, delta, A, B, C, D, z, delta_bias)
    u = activation("u", u, u.shape)
    device = u.device
    delta = same_kind("delta", delta, u.shape, u)
    z = None if z is None else same_kind("z", z, u.shape, u)
    A, D, delta_bias = _parameters(A, D, delta_bias, d, device)
    n = A.shape[1]
    B, C = _shared("B", B, (b,), n, u), _shared("C", C, (b,), n, u)
    (groups, (b_sb, b_sg)), (c_groups, (c_sb, c_sg)) = _groups(B, 1), _groups(C, 1)
    if groups != c_groups:
        raise ValueError(f"B and C: {list(B.shape)} and {list(C.shape)}")
    state = in_place_state("state", state, (b, d, n), torch.float32, device)
    resets = flags_of("resets", resets, (b,), device)
    out = torch.empty_like(u) if u.is_contiguous() else torch.empty((b, d), dtype=u.dtype, device=device)
    if u.numel() == 0:
        return out
    at = state.data_ptr()
    a = N.AgScanArgs(_ARGS, N.AG_DTYPES[u.dtype], b, 1, d, n, groups, int(bool(delta_softplus)), u.data_ptr(), delta.data_ptr(), ptr(z),
                     B.data_ptr(), C.data_ptr(), A.data_ptr(), ptr(D), ptr(delta_bias), at, None, ptr(resets), u.stride(0), 0,
                     delta.stride(0), 0, 0 if z is None else z.stride(0), 0, b_sb, 0, b_sg, c_sb, 0, c_sg,
                     0 if resets is None else resets.stride(0), 0, out.data_ptr(), at)
    with on_device_of(u):
        N.check(N.load().ag_selective_scan_step(ctypes.byref(a), stream_of(u)), "ag_selective_scan_step")
    moved_on(state)
    return out


def selective_scan_torch(u, delta, A, B, C, D=None, z=None, delta_bias=None, *, initial_state=None, resets=None, return_state=False):
    """The same scan (one group, softplus) out of torch ops, step by step (any device; autograd derives the backward): the path of CPU
    tensors."""
    b, T, d = u.shape
    h = u.new_zeros(b, d, A.shape[1]) if initial_state is None else initial_state
    dt = torch.nn.functional.softplus(delta if delta_bias is None else delta + delta_bias)
    ys = []
    for t in range(T):
        if resets is not None:
            h = torch.where((resets[:, t] != 0)[:, None, None], torch.zeros_like(h), h)
        h = torch.exp(dt[:, t, :, None] * A) * h + (dt[:, t] * u[:, t])[..., None] * B[:, t, None]
        ys.append((h * C[:, t, None]).sum(-1))
    y = torch.stack(ys, 1)
    if D is not None:
        y = y + D * u
    if z is not None:
        y = y * z * torch.sigmoid(z)
    return (y, h) if return_state else y
