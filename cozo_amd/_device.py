"""Arrays of a caller, on the host (numpy) or on the GPU (torch tensors), as the C entry points want them."""
from __future__ import annotations

import contextlib
import ctypes as C


def on_gpu(a) -> bool:
    return bool(getattr(a, "is_cuda", False))


def all_on_gpu(*arrays) -> bool:
    """True: every array is a GPU tensor, False: every one is host memory; a mixture is refused"""
    there = [on_gpu(a) for a in arrays if a is not None]
    if any(there) and not all(there):
        raise ValueError("arrays are either all on the GPU or all on the host")
    if any(there):
        dev = {a.device for a in arrays if a is not None}
        if len(dev) > 1:
            raise ValueError(f"tensors on different devices: {sorted(map(str, dev))}")
    return any(there)


@contextlib.contextmanager
def on_stream(like, stream):
    """-> the raw stream a call works on: the caller's, or torch's current one on the tensor's device.  Outputs and scratch allocated
    inside belong to that stream."""
    import torch
    with torch.cuda.device(like.device):
        if stream is None:
            yield C.c_void_p(torch.cuda.current_stream(like.device).cuda_stream)
        else:
            raw = int(stream.cuda_stream) if hasattr(stream, "cuda_stream") else int(stream)
            # handle 0 is the device's default stream, which ExternalStream does not wrap
            s = torch.cuda.ExternalStream(raw, device=like.device) if raw else torch.cuda.default_stream(like.device)
            with torch.cuda.stream(s):
                yield C.c_void_p(raw)

