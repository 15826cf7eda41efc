"""Gradients of ragged batches, where the queries past a sequence's end see its last few keys alone."""
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
