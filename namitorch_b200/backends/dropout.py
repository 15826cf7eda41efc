"""Counter-based dropout with its bias and residual on torch tensors (``nt_dropout_forward``,
``nt_dropout_backward``).

``DropoutCUDAKernels`` takes tensors that ``nn.functional.dropout`` has checked. The mask is
a function of (seed, offset, element) and is computed by both passes; nothing of it is stored.
"""
from __future__ import annotations

import torch

from .. import _native as N

_CODES = {torch.float32: N.NT_F32, torch.float16: N.NT_F16, torch.bfloat16: N.NT_BF16}


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
        count = input.numel()
        if count:
            width = input.shape[-1]
            args = N.pack_dropout(_CODES[input.dtype], 0, count // width, width, p, seed, offset, input.data_ptr(),
                                  0 if bias is None else bias.data_ptr(), 0 if residual is None else residual.data_ptr(),
                                  output.data_ptr(), 0, 0, 0)
            N.on_device(input.device, "nt_dropout_forward", args, 1)
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
        args = N.pack_dropout(_CODES[gradient.dtype], 0, rows, width, p, seed, offset, gradient.data_ptr(), 0, 0,
                              0 if dx is None else dx.data_ptr(), 0 if db is None else db.data_ptr(),
                              0 if workspace is None else workspace.data_ptr(), size)
        N.on_device(gradient.device, "nt_dropout_backward", args, int(rows > 0) * (1 + int(needs[1])))
        return dx, db


__all__ = ["DropoutCUDAKernels"]
