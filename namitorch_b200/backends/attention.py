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

_CODES = {torch.float32: N.NT_F32, torch.float16: N.NT_F16, torch.bfloat16: N.NT_BF16}
_NO_STRIDES = (0,) * 12
_NO_SCRATCH = N.pack_attention_scratch(0, 0, 0)


def _rows(tensor):
    """(tensor, address, strides of the first three dimensions): the tensor itself when the kernels
    take its layout, else a contiguous copy. They take a dense last dimension, no broadcast
    dimension, and 16-byte aligned rows where the width allows them (a tile copy needs them)."""
    strides, address = tensor.stride(), tensor.data_ptr()
    if address % 16 == 0 and tensor.is_contiguous():
        return tensor, address, strides[:3]
    shape, size = tensor.shape, tensor.element_size()
    aligned = shape[3] * size % 16 == 0
    good = (shape[3] <= 1 or strides[3] == 1) and not (aligned and address % 16)
    for i in range(3):
        if shape[i] > 1 and (strides[i] == 0 or (aligned and strides[i] * size % 16)):
            good = False
    if not good:
        tensor = tensor.clone(memory_format=torch.contiguous_format)
        strides, address = tensor.stride(), tensor.data_ptr()
    return tensor, address, strides[:3]


def _heads_last(batch, heads, tokens, dim, like):
    return torch.empty_strided((batch, heads, tokens, dim), (tokens * heads * dim, dim, heads * dim, 1),
                               dtype=like.dtype, device=like.device)


def _statistics_bytes(dtype, batch, heads, kv_heads, queries, keys, dim):
    """What the backward keeps at the start of its scratch: delta, and for float16 the norms that the
    scale of dS is taken from; the rest is for partial gradients, which one more kernel joins."""
    rows = [batch * heads * queries]
    if dtype == torch.float16:
        each = 32 if dim <= 64 else 16
        rows += [rows[0], batch * heads * -(-queries // each), batch * kv_heads * -(-keys // each)]
    return sum((4 * n + 255) // 256 * 256 for n in rows)


class _Word:
    """The library's error word of the current device as an array that torch can view."""

    def __init__(self):
        address = N.C.c_void_p()
        N.check(N.load().nt_attention_error_word(N.C.byref(address)), "nt_attention_error_word")
        self.__cuda_array_interface__ = {"shape": (1,), "typestr": "<i4", "data": (address.value, False), "version": 3}


class AttentionCUDAKernels:
    def __init__(self, backend=None):
        self._backend = backend
        self._error = None

    def _error_word(self, device):
        if self._error is None:
            with torch.cuda.device(device):
                self._error = torch.as_tensor(_Word(), device=device)
        return self._error.data_ptr()

    def check(self) -> None:
        """Raises if a bounded wait inside an attention kernel of this device has ever run out
        (waits for the current stream and reads one word)."""
        if self._error is not None and int(self._error.item()):
            raise RuntimeError("A wait inside an attention kernel ran out; the results of that call are incomplete.")

    def forward(self, query, key, value, lengths=None, *, window=0, sinks=0, query_offset=0, scale, save=True):
        """(output, low, lse). With ``save``, what the backward needs besides the output: lse, float32
        [batch, heads, queries], and for 16-bit types ``low``, the part of the output that its
        rounding took away (the backward subtracts the row sum of gradient * output from dP; over a
        few keys the two nearly cancel, and the rounded output alone would cost the gradients twice
        the error of their own rounding)."""
        query, q, q_strides = _rows(query)
        key, k, k_strides = _rows(key)
        value, v, v_strides = _rows(value)
        batch, heads, queries, dim = query.shape
        output = _heads_last(batch, heads, queries, dim, query)
        low = lse = None
        if save:
            if query.dtype != torch.float32:
                low = _heads_last(batch, heads, queries, dim, query)
            lse = torch.empty((batch, heads, queries), dtype=torch.float32, device=query.device)
        args = N.pack_attention(
            _CODES[query.dtype], dim, batch, heads, key.shape[1], queries, key.shape[2], q, k, v, *q_strides, *k_strides,
            *v_strides, 0 if lengths is None else lengths.data_ptr(), window, sinks, query_offset, scale, 0,
            output.data_ptr(), *output.stride()[:3], 0 if low is None else low.data_ptr(),
            0 if lse is None else lse.data_ptr(), 0, 0, 0, 0, *_NO_STRIDES)
        args += N.pack_attention_scratch(0, 0, self._error_word(query.device))
        N.on_device(query.device, "nt_attention_forward", args, int(batch * queries > 0))
        return output, low, lse

    def backward(self, query, key, value, output, low, lse, gradient, lengths=None, *, window=0, sinks=0, query_offset=0,
                 scale):
        """(grad_query, grad_key, grad_value)."""
        query, q, q_strides = _rows(query)
        key, k, k_strides = _rows(key)
        value, v, v_strides = _rows(value)
        gradient, g, g_strides = _rows(gradient)
        batch, heads, queries, dim = query.shape
        kv_heads, keys = key.shape[1], key.shape[2]
        dq = _heads_last(batch, heads, queries, dim, query)
        dk = _heads_last(batch, kv_heads, keys, dim, query)
        dv = _heads_last(batch, kv_heads, keys, dim, query)
        kv_strides = dk.stride()[:3]
        args = N.pack_attention(
            _CODES[query.dtype], dim, batch, heads, kv_heads, queries, keys, q, k, v, *q_strides, *k_strides, *v_strides,
            0 if lengths is None else lengths.data_ptr(), window, sinks, query_offset, scale, 0, output.data_ptr(),
            *output.stride()[:3], 0 if low is None else low.data_ptr(), lse.data_ptr(), g, dq.data_ptr(), dk.data_ptr(),
            dv.data_ptr(), *g_strides, *dq.stride()[:3], *kv_strides, *kv_strides)
        size = N.load().nt_attention_workspace_size(args + _NO_SCRATCH)
        workspace = torch.empty(size, dtype=torch.uint8, device=query.device)
        args += N.pack_attention_scratch(workspace.data_ptr(), size, self._error_word(query.device))
        statistics = _statistics_bytes(query.dtype, batch, heads, kv_heads, queries, keys, dim)
        N.on_device(query.device, "nt_attention_backward", args,
                    int(batch * queries > 0) + int(batch * keys > 0) + int(size > statistics))
        return dq, dk, dv

    def step(self, query, key_cache, value_cache, lengths, *, window=0, sinks=0, scale):
        """query [batch, heads, head_dim] -> [batch, heads, head_dim]."""
        query = query.contiguous()
        key, k, k_strides = _rows(key_cache)
        value, v, v_strides = _rows(value_cache)
        batch, heads, dim = query.shape
        output = torch.empty_like(query)
        strides = (heads * dim, dim, dim)
        args = N.pack_attention(
            _CODES[query.dtype], dim, batch, heads, key.shape[1], 1, key.shape[2], query.data_ptr(), k, v, *strides,
            *k_strides, *v_strides, lengths.data_ptr(), window, sinks, 0, scale, 0, output.data_ptr(), *strides, 0, 0, 0,
            0, 0, 0, *_NO_STRIDES) + N.pack_attention_scratch(0, 0, self._error_word(query.device))
        N.on_device(query.device, "nt_attention_step", args, int(batch > 0))
        return output


__all__ = ["AttentionCUDAKernels"]
