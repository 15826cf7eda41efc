"""A derivative that attention, its one-token step or dropout does not compute is an error, never a term
left out: gradients through the step, and tangents of forward-mode differentiation."""
import pytest
import torch
from torch.autograd import forward_ad

from namitorch_b200.nn import functional as F

pytestmark = pytest.mark.gpu


def _inputs():
    g = torch.Generator().manual_seed(1)
    return [torch.randn(2, h, 40, 64, generator=g).cuda() for h in (4, 2, 2)]


def _step(q, k, v):
    lengths = torch.tensor([40, 7], dtype=torch.int32, device="cuda")
    return F.sliding_window_attention_step(q[:, :, -1], k, v, lengths, window=10)


@pytest.mark.parametrize("which", range(3))
def test_a_gradient_through_the_step_is_refused(cuda_device, which):
    tensors = _inputs()
    want = _step(*tensors)
    tensors[which].requires_grad_()
    got = _step(*tensors)
    assert torch.equal(got, want)                      # the values are there
    residual = torch.ones(2, 4, 64, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        (got + residual).sum().backward()
    with torch.no_grad():
        assert not _step(*tensors).requires_grad
    assert not _step(*(t.detach() for t in tensors)).requires_grad


CALLS = {
    "attention": lambda q, k, v: F.sliding_window_attention(q, k, v, window=10),
    "step": _step,
    "dropout": lambda q, k, v: F.dropout(q, 0.5, seed=1, residual=q),
    "bias": lambda q, k, v: F.dropout(v, 0.5, seed=1, bias=q[0, 0, 0]),
    "residual": lambda q, k, v: F.dropout(v, 0.5, seed=1, residual=k),
}


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name,which", [("attention", 0), ("attention", 1), ("attention", 2), ("step", 0), ("step", 1),
                                        ("step", 2), ("dropout", 0), ("bias", 0), ("residual", 1)])
def test_a_tangent_is_refused(cuda_device, name, which, grad):
    tensors = _inputs()
    want = CALLS[name](*tensors)
    with forward_ad.dual_level():
        assert torch.equal(CALLS[name](*tensors), want)     # no tangent, no error
        tensors[which] = forward_ad.make_dual(tensors[which].requires_grad_(grad), torch.ones_like(tensors[which]))
        with pytest.raises((RuntimeError, NotImplementedError)):
            CALLS[name](*tensors)
