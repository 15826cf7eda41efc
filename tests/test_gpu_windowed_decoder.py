"""The example decoder: attention, dropout, norm, loss and optimizer in one training loop, and the
one-token path of generation against the whole forward."""
import sys

import pytest
import torch

from conftest import REPO

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(REPO / "examples"))


def test_training_lowers_the_loss_and_generation_matches_the_forward(cuda_device):
    import windowed_decoder as W
    p, losses = W.train(steps=40)
    assert all(torch.isfinite(t).all() for t in p.values())
    assert losses[-1] < 0.7 * losses[0]
    prompt = W.batch_of(10_000, 4, 40, "cuda")[:, :-1]
    tokens, scores = W.generate(p, prompt, 16)
    with torch.no_grad():
        whole = W.logits(p, tokens[:, :-1], W.full_attention)[:, prompt.shape[1] - 1:]
    # bf16 activations through two blocks of different orders of summation: a few of their roundings.
    scale = float(whole.float().abs().max())
    assert float((whole.float() - scores.float()).abs().max()) <= 16 * 2.0 ** -8 * scale


def test_a_step_repeats_bit_for_bit(cuda_device):
    import windowed_decoder as W
    (a, la), (b, lb) = W.train(steps=5), W.train(steps=5)
    assert la == lb and all(torch.equal(a[n], b[n]) for n in a)
