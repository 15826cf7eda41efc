"""Fused softmax cross-entropy (namitorch/nn/functional.py:792-863), sliding-window attention
with sinks and counter-based dropout.

``cross_entropy`` keeps the reference signature and validation. One kernel launch
(``nt_softmax_xent``) reads the logits once and produces both the loss and, when the logits
require grad, the gradient for a unit upstream gradient; the autograd backward only scales
it by the incoming gradient (and skips even that when the incoming gradient is exactly 1).
float16 / bfloat16 logits are read directly and reduced in float32 — the reference promotes
them to float32 first (``float32_function``) — and the gradient comes back in the logits'
dtype. ``softmax_cross_entropy`` exposes the fused forward + backward without autograd.

``sliding_window_attention`` (forward and backward), ``sliding_window_attention_step`` (one
new token over a cache) and ``dropout`` (with the bias before it and the residual after it;
its mask is a function of a seed and an offset and is never stored) run in the kernels of
``backends.attention`` and ``backends.dropout``.
"""
from __future__ import annotations

from numbers import Integral, Real

import numpy as np
import torch
from torch.autograd import forward_ad

from .. import _native as N
from ..backends import get_backend
from ..flat import xent_workspace

_REDUCTIONS = {"none": N.NT_REDUCTION_NONE, "mean": N.NT_REDUCTION_MEAN, "sum": N.NT_REDUCTION_SUM}


def _label_smoothing(value) -> float:
    if isinstance(value, (bool, np.bool_)) or not isinstance(value, Real):
        raise TypeError("label_smoothing must be a real scalar.")
    epsilon = float(value)
    if not 0 <= epsilon < 1:
        raise ValueError("label_smoothing must be in [0, 1).")
    return epsilon


def _arguments(input, target, weight, ignore_index, reduction):
    """namitorch/nn/functional.py:792-816 (the range check runs on the device)."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"Unsupported loss reduction {reduction!r}; expected 'none', 'mean' or 'sum'.")
    if not isinstance(input, torch.Tensor):
        raise TypeError("Loss input must be a NamiTorch Tensor.")
    if not input.dtype.is_floating_point:
        raise TypeError("Classification loss input must be a floating Tensor.")
    if input.ndim < 1 or input.shape[-1] == 0:
        raise ValueError(f"Classification loss input must have shape [..., C] with C > 0, got {tuple(input.shape)}.")
    if not isinstance(target, torch.Tensor) or target.dtype.is_floating_point or target.dtype == torch.bool:
        raise TypeError("Classification loss target must be an integer Tensor.")
    if tuple(target.shape) != tuple(input.shape[:-1]):
        raise ValueError(f"Target shape {tuple(target.shape)} must equal input shape without the last class axis "
                         f"{tuple(input.shape[:-1])}.")
    if isinstance(ignore_index, (bool, np.bool_)) or not isinstance(ignore_index, Integral):
        raise TypeError("ignore_index must be an integer.")
    classes = input.shape[-1]
    if weight is not None:
        if not isinstance(weight, torch.Tensor) or not weight.dtype.is_floating_point:
            raise TypeError("Class weight must be a floating Tensor.")
        if weight.ndim != 1 or weight.shape[0] == 0:
            raise ValueError(f"Class weight must have shape [C] with C > 0, got {tuple(weight.shape)}.")
        if weight.shape != (classes,):
            raise ValueError(f"Class weight must have shape {(classes,)}, got {tuple(weight.shape)}.")
    if input.device.type != "cuda" or target.device != input.device or (weight is not None and weight.device != input.device):
        raise RuntimeError("namitorch_b200 cross_entropy runs on one CUDA device; move logits, targets and weights "
                           "there first.")
    if input.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TypeError(f"cross_entropy supports float32, float16 and bfloat16 logits, got {input.dtype}.")
    logits = input.reshape(-1, classes)
    if not logits.is_contiguous():
        logits = logits.contiguous()
    targets = target.reshape(-1).to(torch.int64).contiguous()
    w = None if weight is None else weight.to(torch.float32).contiguous()
    return logits, targets, w, int(ignore_index), _REDUCTIONS[reduction]


def _launch(logits, targets, weight, ignore_index, reduction, smoothing, want_grad):
    rows, classes = logits.shape
    device = logits.device
    with torch.cuda.device(device):
        loss = torch.empty(rows if reduction == N.NT_REDUCTION_NONE else 1, dtype=torch.float32, device=device)
        row_loss = loss if reduction == N.NT_REDUCTION_NONE else torch.empty(max(rows, 1), dtype=torch.float32,
                                                                             device=device)
        dlogits = torch.empty_like(logits) if want_grad else None
        info = torch.empty(len(N.XENT_INFO_FIELDS), dtype=torch.float64, device=device)   # reset by the call
        ws = xent_workspace(device)
        args = N.XentArgs(
            logits=logits.data_ptr() if rows else None, dtype=N.dtype_code(logits.dtype), rows=rows, classes=classes,
            targets=targets.data_ptr() if rows else None, ignore_index=ignore_index,
            class_weight=None if weight is None else weight.data_ptr(), label_smoothing=float(smoothing),
            reduction=reduction, dlogits=None if dlogits is None or rows == 0 else dlogits.data_ptr(),
            loss=loss.data_ptr(), row_loss=row_loss.data_ptr(), info=info.data_ptr(), workspace=ws.data_ptr(),
            workspace_bytes=ws.numel())
        # One kernel (with a memset of the info record) without class weights; the one-block
        # prepare kernel first with them, or alone for zero rows.
        N.call("nt_softmax_xent", N.C.byref(args), N.stream_handle(),
               launches=(1 if rows else 0) + (0 if weight is None and rows else 1))
    return loss, dlogits, info


def _validate_targets(info: torch.Tensor, classes: int) -> None:
    bad = float(info[N.XENT_INFO_FIELDS.index("bad_targets")].item())
    if bad:
        raise IndexError(f"Every non-ignored target must be in [0, {classes}).")


def softmax_cross_entropy(logits: torch.Tensor, target: torch.Tensor, weight: torch.Tensor | None = None,
                          ignore_index: int = -100, reduction: str = "mean", label_smoothing: float = 0.0,
                          *, validate: bool = True):
    """Fused forward + backward: returns (loss, dlogits) for a unit upstream gradient.

    ``validate=False`` skips the host read that turns out-of-range targets into IndexError
    (those rows then count as ignored)."""
    epsilon = _label_smoothing(label_smoothing)
    x, t, w, ignore, red = _arguments(logits, target, weight, ignore_index, reduction)
    loss, dlogits, info = _launch(x, t, w, ignore, red, epsilon, True)
    if validate:
        _validate_targets(info, x.shape[1])
    out = loss.reshape(target.shape) if red == N.NT_REDUCTION_NONE else loss[0]
    return out, dlogits.reshape(logits.shape)


class _CrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, target, weight, ignore_index, reduction, epsilon, validate):
        want_grad = ctx.needs_input_grad[0]
        loss, dlogits, info = _launch(logits, target, weight, ignore_index, reduction, epsilon, want_grad)
        if validate:
            _validate_targets(info, logits.shape[1])
        ctx.reduction = reduction
        ctx.used = False
        if want_grad:
            ctx.save_for_backward(dlogits)
        return loss if reduction == N.NT_REDUCTION_NONE else loss[0]

    @staticmethod
    def backward(ctx, grad_output):
        # The gradient was computed by the forward launch; it is scaled in place, once.
        if ctx.used:
            raise RuntimeError("The fused cross_entropy gradient can be taken once per forward call.")
        ctx.used = True
        (dlogits,) = ctx.saved_tensors
        rows, classes = dlogits.shape
        g = grad_output.to(torch.float32).contiguous()
        with torch.cuda.device(dlogits.device):
            N.call("nt_xent_backward_scale", dlogits.data_ptr(), N.dtype_code(dlogits.dtype), rows, classes,
                   g.data_ptr(), int(ctx.reduction == N.NT_REDUCTION_NONE), N.stream_handle())
        return dlogits, None, None, None, None, None, None


def cross_entropy(input: torch.Tensor, target: torch.Tensor, weight: torch.Tensor | None = None,
                  ignore_index: int = -100, reduction: str = "mean", label_smoothing: float = 0.0) -> torch.Tensor:
    """namitorch/nn/functional.py:856-863."""
    epsilon = _label_smoothing(label_smoothing)
    x, t, w, ignore, red = _arguments(input, target, weight, ignore_index, reduction)
    loss = _CrossEntropy.apply(x, t, w, ignore, red, epsilon, True)
    return loss.reshape(target.shape) if red == N.NT_REDUCTION_NONE else loss


def linear(input: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    """``input @ weight.T + bias`` with the reference's checks and autocast rule
    (namitorch/nn/functional.py:44-65): inside an enabled autocast context the operands are
    converted to the autocast dtype (``amp.autocast_operands``), which for parameters held in
    an optimizer's ``model_dtype`` copy is no conversion at all. Operands of different dtypes
    outside autocast are promoted, as the reference's matmul promotes them. The product is a
    library GEMM (torch / cuBLAS); it is not part of this package's kernels."""
    from ..amp import autocast_operands
    if not isinstance(input, torch.Tensor) or not isinstance(weight, torch.Tensor):
        raise TypeError("linear input and weight must be NamiTorch Tensors.")
    if weight.ndim != 2:
        raise ValueError(f"linear weight must have rank 2, got shape {tuple(weight.shape)}.")
    if input.ndim < 1 or input.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear input must have rank >= 1 and last dimension {weight.shape[1]}, got shape "
                         f"{tuple(input.shape)}.")
    if bias is not None:
        if not isinstance(bias, torch.Tensor):
            raise TypeError("linear bias must be a NamiTorch Tensor or None.")
        if tuple(bias.shape) != (weight.shape[0],):
            raise ValueError(f"linear bias must have shape {(weight.shape[0],)}, got {tuple(bias.shape)}.")
    if weight.device != input.device or (bias is not None and bias.device != input.device):
        raise RuntimeError("linear operands must be on the same device.")
    input, weight, bias = autocast_operands("linear", input, weight, bias)
    common = torch.promote_types(input.dtype, weight.dtype)
    if bias is not None:
        common = torch.promote_types(common, bias.dtype)
    input, weight = input.to(common), weight.to(common)
    bias = None if bias is None else bias.to(common)
    return torch.nn.functional.linear(input, weight, bias)


def _count(name: str, value, low: int = 0) -> int:
    if type(value) is int and value >= low:
        return value
    if isinstance(value, (bool, np.bool_)) or not isinstance(value, Integral):
        raise TypeError(f"{name} must be an integer.")
    if value < low:
        raise ValueError(f"{name} must be at least {low}, got {value}.")
    return int(value)


_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _attention_arguments(query, key, value, rank, window, sinks, lengths, scale):
    if not (isinstance(query, torch.Tensor) and isinstance(key, torch.Tensor) and isinstance(value, torch.Tensor)):
        raise TypeError("Attention query, key and value must be NamiTorch Tensors.")
    if query.dim() != rank or key.dim() != 4 or value.dim() != 4:
        raise ValueError(f"Attention query must have rank {rank}, key and value rank 4, got shapes "
                         f"{tuple(query.shape)}, {tuple(key.shape)} and {tuple(value.shape)}.")
    shape, kv_shape = query.shape, key.shape
    batch, heads, dim = shape[0], shape[1], shape[-1]
    if kv_shape != value.shape or kv_shape[0] != batch or kv_shape[3] != dim:
        raise ValueError(f"Attention key and value must have shape [{batch}, kv_heads, keys, {dim}], got "
                         f"{tuple(kv_shape)} and {tuple(value.shape)}.")
    if not 1 <= dim <= N.NT_ATTENTION_MAX_HEAD_DIM:
        raise ValueError(f"Attention head dimension must be in [1, {N.NT_ATTENTION_MAX_HEAD_DIM}], got {dim}.")
    if heads < 1 or kv_shape[1] < 1 or heads % kv_shape[1]:
        raise ValueError(f"Attention needs a whole number of query heads per key head, got {heads} and {kv_shape[1]}.")
    dtype, device = query.dtype, query.device
    if dtype not in _DTYPES:
        raise TypeError(f"Attention supports float32, float16 and bfloat16 tensors, got {dtype}.")
    if key.dtype != dtype or value.dtype != dtype:
        raise TypeError(f"Attention query, key and value must have one dtype, got {dtype}, {key.dtype} and "
                        f"{value.dtype}.")
    if device.type != "cuda" or key.device != device or value.device != device:
        raise RuntimeError("namitorch_b200 attention runs on one CUDA device; move query, key and value there first.")
    # (what lies beyond 2^62 is beyond every position)
    window = 0 if window is None else min(_count("window", window, 1), 1 << 62)
    sinks = min(_count("sinks", sinks), 1 << 62)
    if lengths is not None:
        if not isinstance(lengths, torch.Tensor) or lengths.dtype not in (torch.int32, torch.int64):
            raise TypeError("Attention lengths must be an int32 or int64 Tensor or None.")
        if lengths.shape != (batch,):
            raise ValueError(f"Attention lengths must have shape {(batch,)}, got {tuple(lengths.shape)}.")
        if lengths.device != device:
            raise RuntimeError("Attention lengths must be on the device of the query.")
        if lengths.dtype != torch.int32 or not lengths.is_contiguous():
            lengths = lengths.clamp(0, kv_shape[2]).to(torch.int32).contiguous()
    if scale is None:
        scale = dim ** -0.5
    else:
        if isinstance(scale, (bool, np.bool_)) or not isinstance(scale, Real):
            raise TypeError("Attention scale must be a real scalar or None.")
        scale = float(scale)
        if not 0 < scale <= float(np.finfo(np.float32).max):
            raise ValueError("Attention scale must be positive and finite in float32.")
    return window, sinks, lengths, scale


def _differentiated(*tensors) -> bool:
    """Whether a derivative with respect to one of these (tensors or None) may be asked for: such a call
    goes through its autograd function, which computes it or refuses."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    # Outside of every level of forward-mode differentiation (where torch says so: asking each tensor
    # costs a one-token step a tenth of its time) nothing has a tangent.
    if getattr(forward_ad, "_current_level", 0) < 0:
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


class _Once(torch.autograd.Function):
    """Gradients tied to what they were computed from, so that a second derivative is an error
    rather than a term left out."""
    @staticmethod
    def forward(ctx, name, grads, *sources):
        ctx.name = name
        return grads

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"{ctx.name} can be differentiated only once.")


class _SlidingWindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value, lengths, options):
        output, low, lse = get_backend(query).attention.forward(query, key, value, lengths, **options)
        ctx.save_for_backward(query, key, value, output, low, lse, lengths)
        ctx.options = options
        return output

    @staticmethod
    def backward(ctx, grad_output):
        query, key, value, output, low, lse, lengths = ctx.saved_tensors
        grads = get_backend(query).attention.backward(query, key, value, output, low, lse, grad_output, lengths,
                                                      **ctx.options)
        if torch.is_grad_enabled():                    # create_graph=True
            grads = _Once.apply("sliding_window_attention", grads, query, key, value, grad_output)
        return (*grads, None, None)


def sliding_window_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, *, window: int | None = None,
                             sinks: int = 0, lengths: torch.Tensor | None = None, query_position_offset: int = 0,
                             scale: float | None = None) -> torch.Tensor:
    """Causal attention limited to the last ``window`` positions and the first ``sinks`` ones.

    ``query`` is [batch, heads, queries, head_dim], ``key`` and ``value`` [batch, kv_heads,
    keys, head_dim], with heads a multiple of kv_heads (query head h reads key head
    h // (heads // kv_heads)), head_dim at most 128 and any strides. Query i stands at position
    p = query_position_offset + i and sees key j when ``j < lengths[b]``, ``j <= p`` and
    ``p - j < window or j < sinks`` (every earlier key without a window). The weights are
    softmax(scale * query @ key.T) over the keys it sees, ``scale`` 1 / sqrt(head_dim) by
    default; a query that sees none gives zeros. What ``key`` and ``value`` hold at or past
    ``lengths[b]`` (an integer tensor [batch], clamped to the keys) has no effect; a NaN or an
    infinity that some query sees can reach other queries of its block of 256.

    Differentiable once in query, key and value; sums run in float32 in a fixed order.
    ``check_attention`` tells whether every wait inside the kernels completed."""
    window, sinks, lengths, scale = _attention_arguments(query, key, value, 4, window, sinks, lengths, scale)
    offset = min(_count("query_position_offset", query_position_offset), 1 << 62)
    options = {"window": window, "sinks": sinks, "query_offset": offset, "scale": scale}
    if _differentiated(query, key, value):
        return _SlidingWindowAttention.apply(query, key, value, lengths, options)
    return get_backend(query).attention.forward(query, key, value, lengths, save=False, **options)[0]


class _SlidingWindowAttentionStep(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key_cache, value_cache, lengths, options):
        return get_backend(query).attention.step(query, key_cache, value_cache, lengths, **options)

    @staticmethod
    def backward(ctx, grad_output):
        raise RuntimeError("sliding_window_attention_step has no gradient; differentiate sliding_window_attention, or "
                           "call the step under torch.no_grad().")


def sliding_window_attention_step(query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                                  lengths: torch.Tensor, *, window: int | None = None, sinks: int = 0,
                                  scale: float | None = None) -> torch.Tensor:
    """``sliding_window_attention`` for one new token per sequence over a cache.

    ``query`` is [batch, heads, head_dim], the caches [batch, kv_heads, capacity, head_dim].
    Sequence b holds ``lengths[b]`` keys, the new token's among them, and its query stands at
    the last of them. What the other rows of the cache hold has no effect, but up to 15 rows after
    the sinks and after ``lengths[b]`` may be read with those that are seen. A cache is taken as it
    lies when its last dimension is dense, no dimension is broadcast and, where rows are whole
    16-byte vectors, they start on 16-byte boundaries; any other is copied first, all of it. Has no
    gradient: asking for one through the result is an error."""
    if lengths is None:
        raise TypeError("Attention lengths must be an int32 or int64 Tensor.")
    window, sinks, lengths, scale = _attention_arguments(query, key_cache, value_cache, 3, window, sinks, lengths, scale)
    options = {"window": window, "sinks": sinks, "scale": scale}
    if _differentiated(query, key_cache, value_cache):
        return _SlidingWindowAttentionStep.apply(query, key_cache, value_cache, lengths, options)
    return get_backend(query).attention.step(query, key_cache, value_cache, lengths, **options)


def check_attention(device: torch.device | str | None = None) -> None:
    """Raises RuntimeError if a wait inside an attention kernel on ``device`` (the current one by
    default) has ever run out, graph replays included.

    The kernels bound every wait on their own copies and products at about two seconds. One that runs out
    does not stop the program: the call's outputs are incomplete and a word on the device says so. This
    reads it, which waits for the current stream: call it where the program reads a result anyway."""
    get_backend(device).attention.check()


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, bias, residual, p, seed, offset):
        ctx.call = (p, seed, offset)
        return get_backend(input).dropout.forward(input, p, seed=seed, offset=offset, bias=bias, residual=residual)

    @staticmethod
    def backward(ctx, grad_output):
        p, seed, offset = ctx.call
        need_input, need_bias, need_residual = ctx.needs_input_grad[:3]
        grad_input, grad_bias = get_backend(grad_output).dropout.backward(
            grad_output, p, seed=seed, offset=offset, needs=(need_input, need_bias))
        if torch.is_grad_enabled():                    # create_graph=True
            grad_input, grad_bias = _Once.apply("dropout", (grad_input, grad_bias), grad_output)
        return grad_input, grad_bias, grad_output if need_residual else None, None, None, None


def dropout(input: torch.Tensor, p: float, *, seed: int, offset: int = 0, bias: torch.Tensor | None = None,
            residual: torch.Tensor | None = None, training: bool = True) -> torch.Tensor:
    """``residual + keep * (input + bias) / (1 - p)``, each element kept with probability 1 - p.

    Element e of ``input`` in row-major order is dropped when word e % 4 of Philox4x32-7 at the
    counter (e // 4, ``offset``) under the key ``seed`` (both in [0, 2^64)) is below p * 2^32: the
    mask depends on (seed, offset, e) alone, is computed again by the backward and never stored.
    Use another offset for every call that needs a mask of its own. ``bias`` has the shape
    [width] of the last dimension, ``residual`` that of ``input``; all have one dtype, except inside
    ``amp.autocast``, where several are promoted to float32 (a 16-bit projection beside a float32
    bias and residual). With ``training=False`` nothing is dropped."""
    from ..amp import autocast_promoted
    if not isinstance(input, torch.Tensor):
        raise TypeError("dropout input must be a NamiTorch Tensor.")
    if all(t is None or isinstance(t, torch.Tensor) for t in (bias, residual)):
        input, bias, residual = autocast_promoted(input, bias, residual)
    if input.dtype not in _DTYPES:
        raise TypeError(f"dropout supports float32, float16 and bfloat16 tensors, got {input.dtype}.")
    if input.dim() < 1:
        raise ValueError("dropout input must have rank >= 1.")
    if isinstance(p, (bool, np.bool_)) or not isinstance(p, Real):
        raise TypeError("dropout probability must be a real scalar.")
    if not 0 <= p < 1:
        raise ValueError("dropout probability must be in [0, 1).")
    for name, value in (("seed", seed), ("offset", offset)):
        if _count(f"dropout {name}", value) >= 1 << 64:
            raise ValueError(f"dropout {name} must be below 2^64.")
    if type(training) is not bool:
        raise TypeError("training must be a Python bool.")
    for name, tensor, shape in (("bias", bias, input.shape[-1:]), ("residual", residual, input.shape)):
        if tensor is None:
            continue
        if not isinstance(tensor, torch.Tensor):
            raise TypeError(f"dropout {name} must be a NamiTorch Tensor or None.")
        if tensor.shape != shape:
            raise ValueError(f"dropout {name} must have shape {tuple(shape)}, got {tuple(tensor.shape)}.")
        if tensor.dtype != input.dtype:
            raise TypeError(f"dropout {name} must have the dtype of the input, got {tensor.dtype} and {input.dtype}.")
        if tensor.device != input.device:
            raise RuntimeError(f"dropout {name} must be on the device of the input.")
    if input.device.type != "cuda":
        raise RuntimeError("namitorch_b200 dropout runs on a CUDA device; move the input there first.")
    p = float(p) if training else 0.0
    if _differentiated(input, bias, residual):
        return _Dropout.apply(input, bias, residual, p, int(seed), int(offset))
    return get_backend(input).dropout.forward(input, p, seed=int(seed), offset=int(offset), bias=bias, residual=residual)


__all__ = ["check_attention", "cross_entropy", "dropout", "linear", "sliding_window_attention", "sliding_window_attention_step",
           "softmax_cross_entropy"]
