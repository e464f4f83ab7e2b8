"""Helpers of the layer norm, embedding and token log-probability tests: views with made-up
addresses for the refusals (no GPU), and views of all kinds of strides for the results."""
import ctypes

import numpy as np

import tlcuda

U = 2.0 ** -24  # a rounding to float32 is off by at most this, relative to the value


def view(shape, strides=None, data=1 << 20):
    """A tlc_tensor that is only looked at: for calls that are refused before any launch."""
    t = tlcuda.Tensor()
    t.data, t.ndim = data, len(shape)
    if strides is None:
        strides = [int(np.prod(shape[i + 1:], dtype=object)) for i in range(len(shape))]
    for i in range(min(len(shape), 8)):
        t.sizes[i], t.strides[i] = shape[i], strides[i]
    return t


def index(shape, strides=None, data=1 << 20, bits=64):
    v = view(shape, strides, data)
    t = tlcuda.Index()
    t.data, t.ndim, t.bits = v.data, v.ndim, bits
    for i in range(8):
        t.sizes[i], t.strides[i] = v.sizes[i], v.strides[i]
    return t


def at(t):
    return None if t is None else ctypes.byref(t)


def refused(name, *args):
    """The message and status of a C call that must fail."""
    f = getattr(tlcuda.lib(), name)
    status = f(*[at(a) if isinstance(a, ctypes.Structure) else a for a in args], None)
    assert status != 0, f"{name} took the call"
    return tlcuda.lib().tlc_last_error().decode(), status


def guarded(shape, offset=0, pad=64, fill=7.5, dtype=None):
    """A contiguous output inside a larger buffer of `fill`, `offset` elements off 256-byte
    alignment; returns (output, check) where check() says whether the surroundings are whole."""
    import torch
    n = int(np.prod(shape, dtype=np.int64))
    buf = torch.full((pad + offset + n + pad,), fill, device="cuda", dtype=dtype or torch.float32)
    out = buf[pad + offset:pad + offset + n].view(shape)

    def check():
        torch.cuda.synchronize()
        return bool((buf[:pad + offset] == fill).all()) and bool((buf[pad + offset + n:] == fill).all())

    return out, check


def laid_out(x, how):
    """The values of the CUDA tensor x [..., D] under another layout."""
    import torch
    if how == "dense":
        return x.contiguous()
    if how == "gap":  # rows of a wider buffer, 16-byte aligned
        wide = torch.full((*x.shape[:-1], x.shape[-1] + 8), float("nan"), device=x.device)
        wide[..., :x.shape[-1]] = x
        return wide[..., :x.shape[-1]]
    if how == "odd gap":  # rows at odd offsets
        wide = torch.full((*x.shape[:-1], x.shape[-1] + 5), float("nan"), device=x.device)
        wide[..., 1:1 + x.shape[-1]] = x
        return wide[..., 1:1 + x.shape[-1]]
    if how == "columns":  # the last dim is not the one with stride 1
        return x.transpose(0, -1).contiguous().transpose(0, -1)
    if how == "shift":  # all but the last position of sequences one longer (x: 3-D)
        long = torch.full((x.shape[0], x.shape[1] + 1, x.shape[2]), float("nan"), device=x.device)
        long[:, :-1] = x
        return long[:, :-1]
    raise ValueError(how)
