"""What the wrappers of the sequence operators share: argument checks, element strides, the stream and the device of a call."""
import contextlib
import ctypes

import torch

from airgym_amd import _native as N

_SAME = contextlib.nullcontext()


def require(ok, what):
    if not ok:
        raise ValueError(what)


def on_device_of(t):
    """Context in which launches go to t's device (the library launches on the current one)."""
    return _SAME if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


def stream_of(t):
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def ptr(t):
    return None if t is None else t.data_ptr()


def activations(name, t, shape, like=None):
    """t checked against `shape` and, with `like`, against another activation's type and device; its last dimension made dense if it
    is not (an expanded channel, a transposed view)."""
    require(isinstance(t, torch.Tensor) and t.is_cuda, f"{name}: expected a tensor on the GPU")
    require(t.dtype in N.AG_DTYPES, f"{name}: float32, bfloat16 or float16 expected, got {t.dtype}")
    require(tuple(t.shape) == tuple(shape), f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if like is not None:
        require(t.dtype == like.dtype, f"{name}: expected {like.dtype} like the other activations, got {t.dtype}")
        require(t.device == like.device, f"{name}: on {t.device}, the other tensors on {like.device}")
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def parameter(name, t, shape, device):
    """A float32 parameter as a dense tensor, or None."""
    if t is None:
        return None
    require(isinstance(t, torch.Tensor) and t.device == device, f"{name}: expected a tensor on {device}")
    require(t.dtype == torch.float32, f"{name}: parameters and states of the scan are float32, got {t.dtype}")
    require(tuple(t.shape) == tuple(shape), f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    return t.contiguous()


def lengths_of(lengths, batch, device):
    if lengths is None:
        return None
    require(isinstance(lengths, torch.Tensor) and lengths.dtype == torch.int32 and tuple(lengths.shape) == (batch,)
            and lengths.device == device, f"lengths: expected int32 [{batch}] on {device}")
    return lengths.contiguous()


def flags_of(name, flags, shape, device):
    """bool or uint8 flags, read through their strides."""
    if flags is None:
        return None
    require(isinstance(flags, torch.Tensor) and flags.dtype in (torch.bool, torch.uint8) and tuple(flags.shape) == tuple(shape)
            and flags.device == device, f"{name}: expected bool or uint8 {list(shape)} on {device}")
    return flags


def in_place_state(name, t, shape, dtype, device):
    require(isinstance(t, torch.Tensor) and t.device == device and t.dtype == dtype and tuple(t.shape) == tuple(shape) and t.is_contiguous(),
            f"{name}: expected a contiguous {dtype} tensor of shape {list(shape)} on {device} (it is moved on in place)")
    require(not t.requires_grad, f"{name}: moved on in place, cannot require a gradient")
    return t


def no_gradient(what, *tensors):
    require(not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)),
            f"{what} has no backward pass: call it under torch.no_grad(), or the sequence form to train")
