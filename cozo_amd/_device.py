"""Arrays of a caller, on the host (numpy) or on the GPU (torch tensors), as the C entry points want them."""
from __future__ import annotations

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


def no_graph(*arrays) -> None:
    """refuses tensors that autograd follows: what a call of the C library makes of them has no gradient, and would not say so"""
    if any(getattr(a, "requires_grad", False) for a in arrays):
        import torch
        if torch.is_grad_enabled():
            raise ValueError("a tensor requires a gradient, which the result would not carry: detach it, or call under torch.no_grad()")


class on_stream:
    """with on_stream(tensor, stream) as raw: the raw stream a call works on -- the caller's (a handle or a torch stream), or torch's
    current one on the tensor's device.  Outputs and scratch allocated inside belong to that stream."""

    def __init__(self, like, stream):
        import torch
        self._inner = None
        if stream is None:
            self._raw = torch.cuda.current_stream(like.device).cuda_stream
        else:
            self._raw = int(stream.cuda_stream) if hasattr(stream, "cuda_stream") else int(stream)
            # handle 0 is the device's default stream, which ExternalStream does not wrap
            s = torch.cuda.ExternalStream(self._raw, device=like.device) if self._raw else torch.cuda.default_stream(like.device)
            self._inner = torch.cuda.stream(s)

    def __enter__(self):
        if self._inner is not None:
            self._inner.__enter__()
        return C.c_void_p(self._raw)

    def __exit__(self, *exc):
        if self._inner is not None:
            self._inner.__exit__(*exc)
