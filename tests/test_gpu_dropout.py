"""GPU dropout against the NumPy oracle. The mask is exact; y = r + (x + b) c has three float32
roundings and the rounding of c = 1 / (1 - p), then that of the stored type; the bias gradient
is a float32 sum of `rows` terms."""
import numpy as np
import pytest
import torch

from namitorch_b200.nn import functional as F
from oracle import dropout as O

pytestmark = pytest.mark.gpu
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0}
U = 2.0 ** -24


def _make(shape, dt, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(TORCH[dt])


def _np(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


@pytest.mark.parametrize("dt", list(TORCH))
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (3, 8), (5, 9), (2, 3, 64), (257, 769), (64, 2048), (9, 4100), (2000, 40),
                                   (3, 6151), (1024, 2056)])
@pytest.mark.parametrize("p,parts", [(0.1, "br"), (0.5, ""), (0.0, "b"), (0.9, "r")])
def test_matches_oracle(cuda_device, dt, shape, p, parts):
    seed, offset = 0x123456789ABCDEF, 0x1_0000_0007
    x, g = _make(shape, dt, 1).cuda().requires_grad_(), _make(shape, dt, 2).cuda()
    bias = _make(shape[-1:], dt, 3).cuda().requires_grad_() if "b" in parts else None
    residual = _make(shape, dt, 4).cuda().requires_grad_() if "r" in parts else None
    y = F.dropout(x, p, seed=seed, offset=offset, bias=bias, residual=residual)
    wanted = [t for t in (x, bias, residual) if t is not None]
    grads = dict(zip(["x"] + ["bias"] * ("b" in parts) + ["residual"] * ("r" in parts),
                     torch.autograd.grad(y, wanted, g)))
    n = lambda t: None if t is None else _np(t)  # noqa: E731
    want = O.forward(n(x), p, seed, offset, n(bias), n(residual))
    dx, db = O.backward(n(g), p, seed, offset)
    t, tiny = UNIT[dt], TINY[dt]
    size = (np.abs(n(x)) + (0 if bias is None else np.abs(n(bias)))) / (1 - p) + (0 if residual is None else np.abs(n(residual)))
    assert np.all(np.abs(_np(y) - want) <= 4 * U * size + t * np.abs(want) * (1 + 4 * U) + tiny)
    assert np.all(np.abs(_np(grads["x"]) - dx) <= (2 * U + t) * np.abs(dx) * (1 + t) + tiny)
    assert np.array_equal(_np(grads["x"]) != 0, dx != 0)          # the mask itself
    if bias is not None:
        rows = x.numel() // shape[-1]
        total = np.abs(dx).reshape(-1, shape[-1]).sum(0)
        assert np.all(np.abs(_np(grads["bias"]) - db) <= (rows + 4) * U * total + t * np.abs(db) * (1 + t) + tiny)
    if residual is not None:
        assert torch.equal(grads["residual"], g)


def test_unaligned_start_uses_the_same_mask(cuda_device):
    flat = _make((1 + 40 * 64,), "bf16", 1).cuda()
    a, b = flat[1:].view(40, 64), flat[1:].view(40, 64).clone()
    assert torch.equal(F.dropout(a, 0.4, seed=5), F.dropout(b, 0.4, seed=5))
    t = b.t()
    assert torch.equal(F.dropout(t, 0.4, seed=5), F.dropout(t.contiguous(), 0.4, seed=5))


def test_repeats_and_differs_by_seed_and_offset(cuda_device):
    x = torch.ones(512, 256, device="cuda")
    a = F.dropout(x, 0.5, seed=1, offset=0)
    assert torch.equal(a, F.dropout(x, 0.5, seed=1, offset=0))
    for options in ({"seed": 2}, {"seed": 1, "offset": 1}, {"seed": 1 + (1 << 32)}, {"seed": 1, "offset": 1 << 32}):
        agree = float((a == F.dropout(x, 0.5, **options)).float().mean())
        assert abs(agree - 0.5) < 6 * 0.5 / (512 * 256) ** 0.5


def test_dropped_values_do_not_reach_the_output(cuda_device):
    x = torch.ones(64, 64, device="cuda")
    dropped = F.dropout(x, 0.5, seed=3) == 0
    for bad in (float("nan"), float("inf")):
        y = F.dropout(torch.where(dropped, torch.full_like(x, bad), x), 0.5, seed=3, residual=x)
        assert bool(torch.isfinite(y).all())


def test_evaluation_and_empty(cuda_device):
    x = _make((5, 8), "f32", 1).cuda()
    assert torch.equal(F.dropout(x, 0.7, seed=1, training=False), x)
    for shape in ((0, 8), (3, 0)):
        x = torch.zeros(*shape, device="cuda", requires_grad=True)
        bias = torch.zeros(shape[-1], device="cuda", requires_grad=True)
        dx, db = torch.autograd.grad(F.dropout(x, 0.5, seed=1, bias=bias).sum(), (x, bias))
        assert dx.shape == shape and torch.all(db == 0)


def test_gradient_matches_differences(cuda_device):
    """y is linear in its inputs: a difference over a step of 1 is the gradient's product, to the
    float32 roundings of the two sums of n values of size at most 8."""
    x, b, r, g, d = (_make(s, "f32", i).cuda() for i, s in enumerate([(37, 50), (50,), (37, 50), (37, 50), (37, 50)]))
    for which in range(3):
        leaves = [t.clone().requires_grad_() for t in (x, b, r)]
        y = F.dropout(leaves[0], 0.3, seed=9, offset=4, bias=leaves[1], residual=leaves[2])
        grad = torch.autograd.grad(y, leaves, g)[which]
        step = d[0] if which == 1 else d
        moved = [t.detach() + step if i == which else t.detach() for i, t in enumerate(leaves)]
        z = F.dropout(moved[0], 0.3, seed=9, offset=4, bias=moved[1], residual=moved[2])
        left = ((z.detach().double() - y.detach().double()) * g.double()).sum()
        right = (grad.double() * step.double()).sum()
        assert abs(float(left - right)) <= 37 * 50 * 64 * 2.0 ** -23


def test_many_rows_repeat(cuda_device):
    x = _make((30001, 96), "bf16", 1).cuda().requires_grad_()
    bias = _make((96,), "bf16", 2).cuda().requires_grad_()
    g = _make((30001, 96), "bf16", 3).cuda()
    first, second = (torch.autograd.grad(F.dropout(x, 0.2, seed=8, bias=bias), (x, bias), g) for _ in range(2))
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    dx, db = O.backward(_np(g), 0.2, 8, 0)
    bound = 30005 * U * np.abs(dx).sum(0) + 2.0 ** -8 * np.abs(db) * (1 + 2.0 ** -8)
    assert np.all(np.abs(_np(first[1]) - db) <= bound)
