"""The forward whose blocks of queries are shared by a cluster (few of them, over many keys), rows
whose maximum rises far into the keys, and long rows, against the 64-bit oracle. Every case runs forward
and backward: the backward reads the log-sum-exp and the rounding remainder that the forward left.

How many blocks share one of queries is chosen from the sizes and the number of SMs; the numbers
beside the cases are those of 148."""
import numpy as np
import pytest
import torch

from test_gpu_attention import _case, _check, _make

pytestmark = pytest.mark.gpu

SHARED = [
    # batch, heads, kv_heads, queries, keys, options; blocks that share at head widths up to 64, above 64
    (1, 2, 1, 130, 2100, {"offset": 1970}),                                             # 8, 8
    (1, 2, 1, 1, 2100, {"offset": 2099}),                                               # 8, 8
    (1, 2, 2, 300, 1300, {"offset": 1000}),                                             # 4, 4
    (1, 3, 1, 700, 700, {}),                                                            # 2, 2
    (1, 2, 1, 300, 2300, {"offset": 2000, "window": 700, "sinks": 130}),                # 2, 4
    (1, 4, 2, 257, 2400, {"offset": 2143, "window": 1900, "sinks": 3}),                 # 4, 8
    (3, 2, 1, 200, 2200, {"offset": 2000, "lengths": (2200, 0, 5)}),                    # 8, 8; blocks without a tile
    (2, 2, 2, 150, 2150, {"offset": 2000, "lengths": (2010, 900), "window": 1500}),     # 4, 4; rows without keys
    (1, 1, 1, 140, 2048, {"offset": 5000, "window": 1900, "sinks": 200}),               # 8; only the sinks are seen
]


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 80, 128, 24])
@pytest.mark.parametrize("index", range(len(SHARED)))
def test_blocks_of_a_cluster_share_the_keys(cuda_device, dt, dim, index):
    batch, heads, kv_heads, queries, keys, options = SHARED[index]
    _case(dt, batch, heads, kv_heads, queries, keys, dim, seed=7 * index, **options)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("dim,heads,tokens", [(128, 1, 1300), (128, 8, 1100), (64, 16, 1500), (40, 3, 2100)])
def test_long_causal_rows(cuda_device, dt, dim, heads, tokens):
    """Up to 17 tiles to a block or cluster; above width 64 a block's two groups of queries end at different tiles."""
    _case(dt, 1, heads, 1, tokens, tokens, dim, seed=3)


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch,heads,queries,keys", [
    (1, 2, 300, 2100),      # clusters of 8 or 4 (above width 64): maxima that rose apart are joined
    (1, 2, 300, 900),       # clusters of 2
    (4, 16, 260, 700),      # a block to itself
])
def test_maxima_that_rise_far_into_the_row(cuda_device, dt, dim, batch, heads, queries, keys):
    """Single keys whose score is 12 above the rest, and one 22 above, tiles after the row's first: the weights'
    sum of one tile passes 2^13 several times along the row."""
    q, g = _make((batch, heads, queries, dim), dt, 1), _make((batch, heads, queries, dim), dt, 2)
    k, v = _make((batch, 1, keys, dim), dt, 3), _make((batch, 1, keys, dim), dt, 4)
    q[..., 0] = 4.0
    k[..., 0] = 0.0
    for place, score in ((150, 12.5), (420, 13.0), (430, 12.2), (560, 22.0), (1150, 13.0), (1600, 12.6), (2000, 22.5)):
        if place < keys:
            k[:, :, place, 0] = score * dim ** 0.5 / 4.0
    arrays = [t.cuda() for t in (q, k, v, g)]
    _check(*arrays, dt, offset=keys - queries)
    _check(*arrays, dt, offset=keys - queries, window=keys // 2, sinks=200)


def test_a_cluster_repeats_bit_for_bit_and_leaves_other_rows(cuda_device):
    """Rows of a block do not depend on how many others are in it, to the rounding of the same sums."""
    q, k, v = (_make((1, 2, n, 64), "bf16", s).cuda() for n, s in ((200, 1), (2200, 2), (2200, 3)))
    from namitorch_b200.nn import functional as F
    whole = F.sliding_window_attention(q, k, v, query_position_offset=2000)
    part = F.sliding_window_attention(q[:, :, 64:], k, v, query_position_offset=2064)
    assert torch.equal(whole, F.sliding_window_attention(q, k, v, query_position_offset=2000))
    np.testing.assert_allclose(part.float().cpu().numpy(), whole[:, :, 64:].float().cpu().numpy(), rtol=2.0 ** -6, atol=2e-3)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_blocks_without_work_beside_full_ones(cuda_device, dt, dim):
    """Every second sequence is empty, so blocks that end at once share the SMs with blocks that compute: the
    same bits, call after call, as of the sequences alone."""
    from namitorch_b200.nn import functional as F
    n = 12
    arrays = [_make((n, h, 500, dim), dt, s).cuda() for h, s in ((4, 1), (2, 2), (2, 3), (4, 4))]
    lengths = torch.tensor([500 * (b % 2) for b in range(n)], dtype=torch.int32, device="cuda")

    def run(tensors, lengths):
        leaves = [t.detach().requires_grad_() for t in tensors[:3]]
        out = F.sliding_window_attention(*leaves, window=200, lengths=lengths)
        return (out.detach(), *torch.autograd.grad(out, leaves, tensors[3]))

    # (with lengths: rows that see few keys hold their scores' gradients more exactly then)
    alone = run([t[1::2].contiguous() for t in arrays], lengths[1::2].contiguous())
    for _ in range(20):
        for a, b in zip(run(arrays, lengths), alone):
            assert torch.all(a[::2] == 0) and torch.equal(a[1::2], b)
