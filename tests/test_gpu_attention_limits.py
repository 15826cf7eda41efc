"""Windows, sinks and offsets of any size: what reaches past every position hides nothing, an offset past the
limit is refused as such."""
import pytest
import torch

from namitorch_b200.nn import functional as F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("huge", [1 << 31, (1 << 62) + 1, 1 << 63, 1 << 80])
def test_huge_windows_and_sinks(cuda_device, huge):
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(1, 2, 90, 64, generator=g).cuda().requires_grad_() for _ in range(3))
    lengths = torch.tensor([90], device="cuda")
    results = []
    for options in ({}, {"window": huge}, {"window": 5, "sinks": huge}, {"window": huge, "sinks": huge}):
        out = F.sliding_window_attention(q, k, v, **options)
        step = F.sliding_window_attention_step(q[:, :, -1].detach(), k.detach(), v.detach(), lengths, **options)
        results.append((out, step, *torch.autograd.grad(out.square().sum(), (q, k, v))))
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert torch.equal(a, b)


@pytest.mark.parametrize("huge", [1 << 30, 1 << 63, 1 << 80])
def test_offsets_past_the_limit_are_refused(cuda_device, huge):
    q = torch.zeros(1, 1, 3, 16, device="cuda")
    with pytest.raises(ValueError, match="query_offset"):
        F.sliding_window_attention(q, q, q, query_position_offset=huge)
