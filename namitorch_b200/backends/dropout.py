"""Counter-based dropout with its bias and residual on torch tensors (``nt_dropout_forward``,
``nt_dropout_backward``).

``DropoutCUDAKernels`` takes tensors that ``nn.functional.dropout`` has checked. The mask is
a function of (seed, offset, element) and is computed by both passes; nothing of it is stored.
"""
from __future__ import annotations

import torch

from .. import _native as N


class DropoutCUDAKernels:
    def __init__(self, backend=None):
        self._backend = backend

    @staticmethod
    def forward(input, p, *, seed, offset=0, bias=None, residual=None):
        """residual + keep * (input + bias) / (1 - p), contiguous, in the input's dtype."""
        input = input.contiguous()
        bias = None if bias is None else bias.contiguous()
        residual = None if residual is None else residual.contiguous()
        output = torch.empty_like(input)
        if not input.numel():
            return output
        width = input.shape[-1]
        args = N.DropoutArgs(dtype=N.dtype_code(input.dtype), rows=input.numel() // width, width=width, p=p, seed=seed,
                             offset=offset, input=input.data_ptr(), bias=None if bias is None else bias.data_ptr(),
                             residual=None if residual is None else residual.data_ptr(), output=output.data_ptr())
        with torch.cuda.device(input.device):
            N.call("nt_dropout_forward", N.C.byref(args), N.stream_handle())
        return output

    @staticmethod
    def backward(gradient, p, *, seed, offset=0, needs=(True, True)):
        """(grad_input, grad_bias), None for what ``needs`` leaves out."""
        gradient = gradient.contiguous()
        width = gradient.shape[-1]
        rows = gradient.numel() // width if width else 0
        dx = torch.empty_like(gradient) if needs[0] else None
        db = torch.empty(width, dtype=gradient.dtype, device=gradient.device) if needs[1] else None
        if not (needs[0] or needs[1]) or not width:
            return dx, db
        size = int(N.load().nt_dropout_workspace_size(rows, width)) if needs[1] else 0
        workspace = torch.empty(size, dtype=torch.uint8, device=gradient.device) if size else None
        args = N.DropoutArgs(dtype=N.dtype_code(gradient.dtype), rows=rows, width=width, p=p, seed=seed, offset=offset,
                             input=gradient.data_ptr(), output=None if dx is None else dx.data_ptr(),
                             grad_bias=None if db is None else db.data_ptr(),
                             workspace=None if workspace is None else workspace.data_ptr(), workspace_bytes=size)
        with torch.cuda.device(gradient.device):
            N.call("nt_dropout_backward", N.C.byref(args), N.stream_handle(),
                   launches=int(rows > 0) * (1 + int(needs[1])))
        return dx, db


__all__ = ["DropoutCUDAKernels"]
