"""Sliding-window attention with sinks on torch tensors (``nt_attention_forward``,
``nt_attention_backward``, ``nt_attention_step``).

``AttentionCUDAKernels`` takes tensors that ``nn.functional`` has checked: query [batch,
heads, queries, head_dim], key and value [batch, kv_heads, keys, head_dim] of one dtype on
one device, with any strides of the first three dimensions. Results are laid out [batch,
queries, heads, head_dim] in memory, so that merging the heads for the output projection is
a view. Everything is launched on the current stream; the backward's scratch comes from
torch's stream-ordered allocator and is free again when the call returns.
"""
from __future__ import annotations

import torch

from .. import _native as N


def _rows(tensor):
    """The tensor itself when the kernels take its layout, else a contiguous copy: a dense last
    dimension, no broadcast dimension, and 16-byte aligned rows where the width allows them (a
    tile copy needs them)."""
    size = tensor.element_size()
    if tensor.shape[-1] > 1 and tensor.stride(-1) != 1:
        return tensor.contiguous()
    aligned = tensor.shape[-1] * size % 16 == 0
    if aligned and tensor.data_ptr() % 16:
        return tensor.clone(memory_format=torch.contiguous_format)
    for extent, stride in zip(tensor.shape[:-1], tensor.stride()[:-1]):
        if extent > 1 and (stride == 0 or (aligned and stride * size % 16)):
            return tensor.contiguous()
    return tensor


def _heads_last(batch, heads, tokens, dim, like):
    return torch.empty((batch, tokens, heads, dim), dtype=like.dtype, device=like.device).transpose(1, 2)


class AttentionCUDAKernels:
    def __init__(self, backend=None):
        self._backend = backend
        self._error = None

    def _error_word(self, device):
        if self._error is None:
            self._error = torch.zeros(1, dtype=torch.int32, device=device)
        return self._error

    def check(self) -> None:
        """Raises if a bounded wait inside an attention kernel of this device has ever run out
        (reads one word from the device)."""
        if self._error is not None and int(self._error.item()):
            raise RuntimeError("A wait inside an attention kernel ran out; the results of that call are incomplete.")

    def _args(self, query, key, value, lengths, window, sinks, query_offset, scale, output, low, lse):
        batch, heads, queries, dim = query.shape
        return N.AttentionArgs(
            dtype=N.dtype_code(query.dtype), head_dim=dim, batch=batch, query_heads=heads, kv_heads=key.shape[1],
            queries=queries, keys=key.shape[2], query=query.data_ptr(), key=key.data_ptr(), value=value.data_ptr(),
            query_strides=query.stride()[:3], key_strides=key.stride()[:3], value_strides=value.stride()[:3],
            lengths=None if lengths is None else lengths.data_ptr(), window=window, sinks=sinks,
            query_offset=query_offset, scale=scale, output=output.data_ptr(), output_strides=output.stride()[:3],
            output_low=None if low is None else low.data_ptr(), lse=None if lse is None else lse.data_ptr(), error=self._error_word(query.device).data_ptr())

    def forward(self, query, key, value, lengths=None, *, window=0, sinks=0, query_offset=0, scale, save=True):
        """(output, low, lse). With ``save``, what the backward needs besides the output: lse, float32
        [batch, heads, queries], and for 16-bit types ``low``, the part of the output that its
        rounding took away (the backward subtracts the row sum of gradient * output from dP; over a
        few keys the two nearly cancel, and the rounded output alone would cost the gradients twice
        the error of their own rounding)."""
        query, key, value = _rows(query), _rows(key), _rows(value)
        batch, heads, queries, dim = query.shape
        output = _heads_last(batch, heads, queries, dim, query)
        low = _heads_last(batch, heads, queries, dim, query) if save and query.dtype != torch.float32 else None
        lse = torch.empty((batch, heads, queries), dtype=torch.float32, device=query.device) if save else None
        with torch.cuda.device(query.device):
            args = self._args(query, key, value, lengths, window, sinks, query_offset, scale, output, low, lse)
            N.call("nt_attention_forward", N.C.byref(args), N.stream_handle(), launches=int(batch * queries > 0))
        return output, low, lse

    def backward(self, query, key, value, output, low, lse, gradient, lengths=None, *, window=0, sinks=0, query_offset=0,
                 scale):
        """(grad_query, grad_key, grad_value)."""
        query, key, value, gradient = _rows(query), _rows(key), _rows(value), _rows(gradient)
        batch, heads, queries, dim = query.shape
        kv_heads, keys = key.shape[1], key.shape[2]
        dq = _heads_last(batch, heads, queries, dim, query)
        dk = _heads_last(batch, kv_heads, keys, dim, query)
        dv = _heads_last(batch, kv_heads, keys, dim, query)
        with torch.cuda.device(query.device):
            args = self._args(query, key, value, lengths, window, sinks, query_offset, scale, output, low, lse)
            args.gradient, args.gradient_strides = gradient.data_ptr(), gradient.stride()[:3]
            args.grad_query, args.grad_query_strides = dq.data_ptr(), dq.stride()[:3]
            args.grad_key, args.grad_key_strides = dk.data_ptr(), dk.stride()[:3]
            args.grad_value, args.grad_value_strides = dv.data_ptr(), dv.stride()[:3]
            size = int(N.load().nt_attention_workspace_size(N.C.byref(args)))
            workspace = torch.empty(size, dtype=torch.uint8, device=query.device)
            args.workspace, args.workspace_bytes = workspace.data_ptr(), size
            statistics = (batch * heads * queries * 4 + 255) // 256 * 256
            N.call("nt_attention_backward", N.C.byref(args), N.stream_handle(),
                   launches=int(batch * queries > 0) + int(batch * keys > 0) + int(size > statistics))
        return dq, dk, dv

    def step(self, query, key_cache, value_cache, lengths, *, window=0, sinks=0, scale):
        """query [batch, heads, head_dim] -> [batch, heads, head_dim]."""
        query, key, value = _rows(query).unsqueeze(2), _rows(key_cache), _rows(value_cache)
        batch, heads, _, dim = query.shape
        output = torch.empty((batch, heads, 1, dim), dtype=query.dtype, device=query.device)
        with torch.cuda.device(query.device):
            args = self._args(query, key, value, lengths, window, sinks, 0, scale, output, None, None)
            N.call("nt_attention_step", N.C.byref(args), N.stream_handle(), launches=int(batch > 0))
        return output.squeeze(2)


__all__ = ["AttentionCUDAKernels"]
