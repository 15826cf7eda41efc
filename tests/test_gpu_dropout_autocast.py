"""Dropout with its bias and residual inside the package's autocast: a projection there has 16 bits, parameters
and the residual stream float32. The result is that of the float32 call on the promoted operands."""
import pytest
import torch

from namitorch_b200 import amp
from namitorch_b200.nn import functional as F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_block_inside_autocast(cuda_device, dtype):
    g = torch.Generator().manual_seed(1)
    x, w, b = (torch.randn(*s, generator=g).cuda().requires_grad_() for s in ((3, 7, 64), (64, 64), (64,)))
    with amp.autocast("cuda", dtype=dtype):
        y = F.linear(x, w)
        assert y.dtype == dtype
        z = F.dropout(y, 0.3, seed=5, offset=2, bias=b, residual=x)
        same = F.dropout(y, 0.3, seed=5, bias=b.detach().to(dtype))    # one dtype: kept
    want = F.dropout(y.float(), 0.3, seed=5, offset=2, bias=b, residual=x)
    assert z.dtype == torch.float32 and torch.equal(z, want) and same.dtype == dtype
    grad = torch.randn(3, 7, 64, generator=g).cuda()
    for a, c in zip(torch.autograd.grad(z, (x, w, b), grad, retain_graph=True), torch.autograd.grad(want, (x, w, b), grad)):
        assert a.dtype == torch.float32 and torch.equal(a, c)


def test_other_mixtures_stay_refused(cuda_device):
    x, b = torch.ones(3, 8, device="cuda", dtype=torch.float16), torch.ones(8, device="cuda")
    with pytest.raises(TypeError, match="dtype"):
        F.dropout(x, 0.5, seed=1, bias=b)                             # no autocast
    with amp.autocast("cuda"):
        with pytest.raises(TypeError, match="dtype"):
            F.dropout(x, 0.5, seed=1, bias=b.double())
        with pytest.raises(TypeError, match="dtype"):
            F.dropout(x, 0.5, seed=1, bias=b.cpu())
        with pytest.raises(TypeError, match="Tensor"):
            F.dropout(x, 0.5, seed=1, bias=3.0)
