"""float16 gradients of attention at upstream gradients and values of any size.

dS = P (dP - delta) is an operand of the products that give dq and dk, in the inputs' type. Whatever the
size of the upstream gradient, its rounding may cost no more than that of the result itself: two
independent errors of the same size, sqrt(2) of one, 1.5 with the sample's spread (the results are
float16 numbers, so below their normal range the rounding of the exact gradient grows too)."""
import numpy as np
import pytest
import torch

from namitorch_b200.nn import functional as F
from oracle import attention as O

pytestmark = pytest.mark.gpu


def _normal(shape, seed, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * size).to(torch.float16)


def _np(t):
    return t.detach().double().cpu().numpy()


def _gradients(q, k, v, g, **options):
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(F.sliding_window_attention(*leaves, **options), leaves, g.cuda())
    wanted = O.backward(*(_np(t) for t in (q, k, v, g)), window=options.get("window") or 0, sinks=options.get("sinks", 0))
    return [_np(t) for t in grads], wanted


def _keeps_precision(got, want, what):
    rounded = want.astype(np.float16).astype(np.float64)
    assert np.all(np.isfinite(rounded)), "the case itself leaves float16"
    assert np.all(np.isfinite(got)), what
    assert np.linalg.norm(got - want) <= 1.5 * np.linalg.norm(rounded - want), what


@pytest.mark.parametrize("tokens,dim,window,size,values", [
    (2048, 64, None, 1.0, 1.0), (2048, 64, None, 1e-3, 1.0), (2048, 64, None, 1e-4, 1.0), (2048, 128, None, 1.0, 1e-3),
    (2048, 128, None, 1e-5, 1.0), (1024, 128, 64, 1000.0, 16.0), (1500, 64, 2, 8192.0, 1.0), (1500, 80, 2, 8192.0, 1.0),
    (1500, 64, 16, 1e-4, 1.0), (1500, 128, 17, 1e-4, 0.1), (2000, 40, None, 8000.0, 1e-3)])
def test_gradients_of_any_size_keep_their_precision(cuda_device, tokens, dim, window, size, values):
    q, k = _normal((1, 4, tokens, dim), 1), _normal((1, 2, tokens, dim), 2)
    v, g = _normal((1, 2, tokens, dim), 3, values), _normal((1, 4, tokens, dim), 4, size)
    for got, want, what in zip(*_gradients(q, k, v, g, window=window), ("dq", "dk", "dv")):
        _keeps_precision(got, want, what)


@pytest.mark.parametrize("small,between", [(1e-1, 0), (1e-3, 128)])
@pytest.mark.parametrize("dim,window,sinks", [(64, 40, 0), (128, 100, 0), (64, 2, 0)])
def test_rows_sequences_and_heads_of_different_sizes_keep_their_precision(cuda_device, dim, window, sinks, small, between):
    """Gradients of 1000 in one stretch of the rows and far smaller ones in the next, values of 8 in one
    sequence and 1e-2 in the other, one head a thousandth of the rest: each part by itself. dk has one scale
    in a block of 128 keys: where its queries' gradients are a millionth of the largest that the block
    sees, that block's keys are left out."""
    tokens, cut = 1600, 800
    q, k, v, g = (_normal((2, h, tokens, dim), s) for h, s in ((4, 1), (4, 2), (4, 3), (4, 4)))
    v[0] *= 8
    v[1] *= 1e-2
    g[:, :, :cut] *= 1000
    g[:, :, cut:] *= small
    g[:, 2] *= 1e-3
    got, wanted = _gradients(q, k, v, g, window=window, sinks=sinks)
    for a, b, what in zip(got, wanted, ("dq", "dk", "dv")):
        for batch in range(2):
            for head in range(4):
                # (keys before the cut see queries after it, their window's, at most 100)
                for part in (slice(0, cut - 128), slice(cut + between, tokens)):
                    _keeps_precision(a[batch, head, part], b[batch, head, part], f"{what} {batch} {head} {part}")


@pytest.mark.parametrize("dim,window", [(64, 60), (128, 9)])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_one_row_that_overflowed_leaves_the_others(cuda_device, dim, window, bad):
    q, k, v, g = (_normal((1, 2, 1500, dim), s) for s in (1, 2, 3, 4))
    g *= 1e-3
    results = []
    for value in (bad, 0.0):
        g[:, :, 700] = value
        leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
        results.append(torch.autograd.grad(F.sliding_window_attention(*leaves, window=window), leaves, g.cuda()))
    # Beyond the blocks of 128 keys and queries around the row and its window.
    far = np.r_[0:384, 960:1500]
    for a, b in zip(*results):
        assert bool(torch.isfinite(a[:, :, far]).all()) and torch.equal(a[:, :, far], b[:, :, far])
