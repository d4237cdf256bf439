"""What the wrappers of the sequence operators share: argument checks, the stream and the device of a call.

A step of a rollout is a few microseconds of GPU work, so the checks are plain comparisons and messages are put together only when one
fails.

Streams and graphs: a call runs on the current stream of its tensors' device and takes its workspaces from torch's allocator, so that
each captured graph has its own.  Nothing synchronises, all calls can be captured.  As with any torch code, a backward pass is captured
only after every eager graph over the same leaves has been dropped: torch ends the process otherwise."""
import contextlib

import torch

from airgym_amd import _native as N

DTYPES = N.AG_DTYPES
_SAME = contextlib.nullcontext()
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


def on_device_of(t):
    """Context in which launches go to t's device (the library launches on the current one)."""
    return _SAME if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


def stream_of(t):
    """The current stream of t's device as the library takes it."""
    if _raw_stream is not None:
        return _raw_stream(t.device.index)
    return torch.cuda.current_stream(t.device).cuda_stream


def ptr(t):
    return None if t is None else t.data_ptr()


def shape_error(name, t, shape):
    got = f"{t.dtype} {list(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
    return ValueError(f"{name}: expected {shape}, got {got}")


def activation(name, t, shape):
    """t as the first activation of a call: its type and device are what the others are held to.  Its last dimension is made dense if it
    is not (an expanded channel, a transposed view)."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise shape_error(name, t, "a tensor on the GPU")
    if t.dtype not in DTYPES:
        raise shape_error(name, t, "float32, bfloat16 or float16")
    if t.shape != shape:
        raise shape_error(name, t, list(shape))
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def same_kind(name, t, shape, like):
    """... and the others."""
    if not isinstance(t, torch.Tensor) or t.dtype != like.dtype or t.device != like.device or t.shape != shape:
        raise shape_error(name, t, f"{like.dtype} {list(shape)} on {like.device}, like the other activations")
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def parameter(name, t, shape, device):
    """A float32 parameter or state as a dense tensor, or None."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.device != device or t.shape != shape:
        raise shape_error(name, t, f"float32 {list(shape)} on {device}")
    return t if t.is_contiguous() else t.contiguous()


def lengths_of(lengths, batch, device):
    if lengths is None:
        return None
    if not isinstance(lengths, torch.Tensor) or lengths.dtype != torch.int32 or lengths.shape != (batch,) or lengths.device != device:
        raise shape_error("lengths", lengths, f"int32 [{batch}] on {device}")
    return lengths.contiguous()


def flags_of(name, flags, shape, device):
    """bool or uint8 flags, read through their strides, or None."""
    if flags is None:
        return None
    if not isinstance(flags, torch.Tensor) or flags.dtype not in (torch.bool, torch.uint8) or flags.shape != shape or flags.device != device:
        raise shape_error(name, flags, f"bool or uint8 {list(shape)} on {device}")
    return flags


def in_place_state(name, t, shape, dtype, device):
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != device or t.shape != shape or not t.is_contiguous():
        raise shape_error(name, t, f"contiguous {dtype} {list(shape)} on {device} (it is moved on in place)")
    if t.requires_grad:
        raise ValueError(f"{name}: moved on in place, cannot require a gradient")
    return t


def moved_on(state):
    """state was written by a kernel: autograd learns of it as of any in-place change (a graph that saved it refuses its backward)."""
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)


def wants_gradient(*tensors):
    return torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors)


def nothing(x, *inputs):
    """An empty output like x, which has no elements; all of the inputs that want a gradient get one of zero."""
    y = x.new_empty(x.shape)
    for t in (x, *inputs):
        if wants_gradient(t):
            y = y + t.sum().to(y.dtype)
    return y


def no_gradient(what, *tensors):
    if wants_gradient(*tensors):
        raise ValueError(f"{what} has no backward pass: call it under torch.no_grad(), or the sequence form to train")
