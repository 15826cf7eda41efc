"""Gradients where rows that see few keys carry much of the norm: ragged batches, whose queries past a
sequence's end see its last few keys alone, and short sequences."""
import numpy as np
import pytest
import torch

from namitorch_b200.nn import functional as F
from oracle import attention as O
from test_gpu_attention import TORCH, _make, _np

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("dim,window,sinks", [(64, 100, 0), (128, 100, 0), (80, 60, 3), (64, None, 0)])
def test_rows_with_few_keys_keep_their_precision(cuda_device, dt, dim, window, sinks):
    """Beside the result's own rounding: dS in one 16-bit value (as large an error) only on rows that see more
    than 16 keys, below half of the squared norm here, and delta's error, below a quarter of it. sqrt(1.75)
    is 1.32; 1.35 with the sample's spread. One value everywhere gives 1.47 to 1.53."""
    batch, tokens = 24, 200
    lengths = [1 + (3 if window else 1) * b for b in range(batch)]
    q, k, v, g = (_make((batch, 2, tokens, dim), dt, s) for s in (1, 2, 3, 4))
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    out = F.sliding_window_attention(*leaves, window=window, sinks=sinks, lengths=torch.tensor(lengths, device="cuda"))
    grads = torch.autograd.grad(out, leaves, g.cuda())
    wanted = O.backward(*(_np(t) for t in (q, k, v, g)), window=window or 0, sinks=sinks, lengths=lengths)
    for got, want, bound in zip(grads, wanted, (1.35, 1.35, 1.5)):
        rounded = _np(torch.from_numpy(want).to(TORCH[dt]))
        assert np.linalg.norm(_np(got) - want) <= bound * np.linalg.norm(rounded - want)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("tokens", [17, 40, 64, 200, 400])
@pytest.mark.parametrize("dim", [64, 128])
def test_short_sequences_keep_their_precision(cuda_device, dt, tokens, dim):
    """Causal rows n see n keys and have about 1 / n of the squared norm: those with more than 16, which hold dS
    in one value, have at most log(400 / 16) / log(400) = 0.54 of it, and delta's error is a few hundredths
    beside it. sqrt(1.54) is 1.24, 1.35 with the spread of a single head's sample."""
    for seed in range(6):
        q, k, v, g = (_make((1, 1, tokens, dim), dt, 10 * seed + s) for s in (1, 2, 3, 4))
        leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
        grads = torch.autograd.grad(F.sliding_window_attention(*leaves), leaves, g.cuda())
        wanted = O.backward(*(_np(t) for t in (q, k, v, g)))
        for got, want in list(zip(grads, wanted))[:2]:
            rounded = _np(torch.from_numpy(want).to(TORCH[dt]))
            assert np.linalg.norm(_np(got) - want) <= 1.35 * np.linalg.norm(rounded - want)


@pytest.mark.parametrize("dt", list(TORCH))
@pytest.mark.parametrize("dim", [64, 128, 33])
def test_rows_with_one_key_have_no_gradient(cuda_device, dt, dim):
    """A single key has the weight 1 whatever its score: dq is 0, and dk gets nothing from the row, exactly."""
    def grads(tokens, **options):
        tensors = [_make((2, h, tokens, dim), dt, s).cuda().requires_grad_() for h, s in ((4, 1), (2, 2), (2, 3))]
        g = _make((2, 4, tokens, dim), dt, 4).cuda()
        out = F.sliding_window_attention(*tensors, **options)
        return torch.autograd.grad(out, tensors, g), tensors, g

    for tokens, options in ((1, {}), (300, {"window": 1}), (700, {"window": 1})):
        (dq, dk, dv), tensors, g = grads(tokens, **options)
        assert not dq.any() and not dk.any()
        # dv is the sum of g over the group, to the bound that counts P's own rounding (P is exp(s - lse)).
        arrays, o = [_np(t) for t in tensors], {"window": options.get("window", 0)}
        want = _np(g).reshape(2, 2, 2, tokens, dim).sum(2)
        assert np.all(np.abs(_np(dv) - want) <= O.tolerances(*arrays, dt, _np(g), **o)[4])
    for tokens in (90, 1200):                                      # the first row of a causal sequence
        (dq, dk, _), _, _ = grads(tokens)
        assert not dq[:, :, 0].any() and dq[:, :, 1:].any() and dk[:, :, 0].any()
    lengths = torch.tensor([1, 40], device="cuda")                 # every row of the first, some of the second
    (dq, dk, _), _, _ = grads(100, lengths=lengths, window=30)
    assert not dq[0].any() and not dk[0].any()
    assert not dq[1, :, 68].any() and dq[1, :, 67].any()           # position 68 sees key 39 alone
