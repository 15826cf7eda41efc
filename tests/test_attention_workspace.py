"""The scratch of the attention backward: partial sums of cut key blocks, which stay few however many keys
are sinks (no GPU needed)."""
import ctypes
import random

import pytest

from namitorch_b200 import _native as N


def _partial(dtype, batch, heads, kv_heads, queries, keys, dim, window, sinks):
    """Bytes beside the statistics."""
    a = N.AttentionArgs(dtype=dtype, head_dim=dim, batch=batch, query_heads=heads, kv_heads=kv_heads, queries=queries,
                        keys=keys, window=window, sinks=sinks, query_offset=max(0, keys - queries), scale=0.125)
    rows = batch * heads * queries * 4 + 256
    if dtype == N.NT_F16:
        rows = 2 * rows + 4 * batch * (heads * (queries // 16 + 1) + kv_heads * (keys // 16 + 1)) + 512
    size = N.load().nt_attention_workspace_size(ctypes.byref(a))
    assert size > 0, N.last_error()
    return max(0, size - rows)


@pytest.mark.parametrize("dtype,heads,tokens,window,sinks", [
    (N.NT_F32, 4, 8192, 1, 8000), (N.NT_BF16, 4, 8192, 1, 8000), (N.NT_BF16, 16, 32768, 128, 16384),
    (N.NT_F16, 16, 32768, 128, 16384), (N.NT_F32, 8, 16384, 64, 2000)])
def test_many_sinks_need_no_more_than_the_gradients(dtype, heads, tokens, window, sinks):
    gradients = 2 * heads * tokens * 128 * 4                  # dk and dv in float32
    assert _partial(dtype, 1, heads, heads, tokens, tokens, 128, window, sinks) <= gradients


def test_pieces_stay_few():
    """At most about two pieces to an SM and pass, a partial one to each block besides: 148 SMs, 640 of them."""
    rng = random.Random(3)
    for _ in range(4000):
        kv_heads, group, batch = 2 ** rng.randrange(7), 2 ** rng.randrange(4), rng.choice((1, 1, 2, 3, 8, 64))
        queries, keys = (int(2 ** rng.uniform(0, 18)) for _ in range(2))
        window, sinks = rng.choice((0, int(2 ** rng.uniform(0, 17)))), rng.choice((0, 1, 4, 130, int(2 ** rng.uniform(0, 18))))
        dtype, dim = rng.choice((N.NT_F32, N.NT_F16, N.NT_BF16)), rng.choice((64, 128))
        case = (dtype, batch, group * kv_heads, kv_heads, queries, keys, dim, window, sinks)
        assert _partial(*case) <= 640 * 2 * 128 * dim * 4, case


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,tokens,dim,window,sinks", [(2, 2, 1500, 64, 5, 1000), (4, 1, 1400, 128, 1, 300),
                                                                    (16, 8, 1000, 64, 30, 700)])
def test_gradients_with_many_sinks(cuda_device, dt, heads, kv_heads, tokens, dim, window, sinks):
    from test_gpu_attention import _case
    _case(dt, 1, heads, kv_heads, tokens, tokens, dim, seed=5, window=window, sinks=sinks)
