"""GPU sliding-window attention against the 64-bit oracle, within the bounds that
``oracle.attention.tolerances`` derives from the arithmetic."""
import numpy as np
import pytest
import torch

from namitorch_b200.backends import get_backend
from namitorch_b200.nn import functional as F
from oracle import attention as O

pytestmark = pytest.mark.gpu
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _make(shape, dt, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(TORCH[dt])


def _np(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def _within(got, want, bound, what):
    got = _np(got)
    assert got.shape == want.shape
    finite = np.isfinite(want)
    assert np.array_equal(finite, np.isfinite(got)), what
    assert np.array_equal(got[~finite], want[~finite]), what
    over = np.abs(got - want)[finite] - bound[finite]
    assert over.size == 0 or over.max() <= 0, f"{what}: over its bound by {over.max():.3g} (bound {bound.max():.3g})"


def _check(q, k, v, g, dt, lengths=None, offset=0, scale=None, **options):
    """Forward and backward of CUDA tensors q, k, v (any strides) against the oracle."""
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out = F.sliding_window_attention(q, k, v, lengths=n, query_position_offset=offset, scale=scale, **options)
    grads = torch.autograd.grad(out, (q, k, v), g)
    again = F.sliding_window_attention(q, k, v, lengths=n, query_position_offset=offset, scale=scale, **options)
    assert torch.equal(out, again)
    for a, b in zip(grads, torch.autograd.grad(again, (q, k, v), g)):
        assert torch.equal(a, b)                       # a fixed order of every sum
    arrays = [_np(t) for t in (q, k, v)]
    o = dict(window=options.get("window") or 0, sinks=options.get("sinks", 0), lengths=lengths, offset=offset, scale=scale)
    want, lse = O.forward(*arrays, **o)
    dq, dk, dv = O.backward(*arrays, _np(g), **o)
    t_out, t_lse, t_dq, t_dk, t_dv = O.tolerances(*arrays, dt, _np(g), **o)
    _within(out, want, t_out, "out")
    for got, w, t, name in zip(grads, (dq, dk, dv), (t_dq, t_dk, t_dv), ("dq", "dk", "dv")):
        _within(got, w, t, name)
    forward_only = F.sliding_window_attention(q.detach(), k.detach(), v.detach(), lengths=n,
                                              query_position_offset=offset, scale=scale, **options)
    assert torch.equal(forward_only, out)
    _, _, got_lse = get_backend(q).attention.forward(q.detach(), k.detach(), v.detach(), n, query_offset=offset,
                                                  window=options.get("window") or 0, sinks=options.get("sinks", 0),
                                                  scale=q.shape[-1] ** -0.5 if scale is None else scale)
    _within(got_lse, lse, t_lse, "lse")
    get_backend(q).attention.check()
    return out, grads


def _case(dt, batch, heads, kv_heads, queries, keys, dim, seed=0, **options):
    q, g = _make((batch, heads, queries, dim), dt, seed).cuda(), _make((batch, heads, queries, dim), dt, seed + 1).cuda()
    k, v = _make((batch, kv_heads, keys, dim), dt, seed + 2).cuda(), _make((batch, kv_heads, keys, dim), dt, seed + 3).cuda()
    return _check(q, k, v, g, dt, **options)


SHAPES = [
    # batch, heads, kv_heads, queries, keys, dim, options
    (1, 1, 1, 1, 1, 64, {}),
    (2, 2, 1, 1, 5, 64, {"offset": 4, "window": 2, "sinks": 1}),
    (1, 2, 2, 64, 64, 64, {}),
    (1, 2, 1, 129, 129, 128, {"window": 1}),
    (1, 2, 1, 129, 129, 128, {"window": 1, "sinks": 1}),
    (2, 3, 3, 200, 200, 64, {"window": 64, "sinks": 4}),
    (1, 4, 2, 257, 257, 80, {"window": 100, "sinks": 3}),
    (1, 6, 2, 300, 300, 128, {"window": 37, "sinks": 130}),
    (1, 2, 2, 385, 385, 40, {"window": 1000, "sinks": 5}),
    (1, 2, 1, 77, 400, 128, {"offset": 323, "window": 128, "sinks": 16}),
    (1, 2, 1, 300, 90, 64, {"window": 50, "sinks": 2}),              # later queries see the sinks alone
    (1, 2, 1, 300, 90, 64, {"window": 50}),                          # later queries see nothing
    (1, 1, 1, 70, 20, 64, {"offset": 5000, "window": 10}),           # no query sees anything
    (4, 2, 1, 150, 150, 64, {"lengths": (150, 0, 1, 131), "window": 60, "sinks": 2}),
    (3, 2, 2, 260, 260, 128, {"lengths": (300, -4, 129)}),           # clamped to [0, keys]
    (1, 8, 1, 140, 140, 64, {"window": 33, "sinks": 33}),
    (1, 4, 4, 256, 256, 32, {"window": 128, "scale": 0.7}),
    (1, 3, 1, 130, 130, 16, {}),
]


@pytest.mark.parametrize("dt", list(TORCH))
@pytest.mark.parametrize("index", range(len(SHAPES)))
def test_matches_oracle(cuda_device, dt, index):
    *shape, options = SHAPES[index]
    _case(dt, *shape, seed=10 * index, **options)


@pytest.mark.parametrize("dt,dim", [("bf16", 33), ("f16", 7), ("f32", 1), ("f32", 65), ("bf16", 100)])
def test_odd_head_widths(cuda_device, dt, dim):
    _case(dt, 1, 2, 1, 97, 97, dim, window=40, sinks=2)


@pytest.mark.parametrize("dt", list(TORCH))
def test_long_rows_split_sinks(cuda_device, dt):
    """Enough queries that the sink keys' queries are cut into pieces, in one and two sink blocks."""
    _case(dt, 1, 2, 1, 1500, 1500, 64, window=70, sinks=4)
    _case(dt, 1, 2, 2, 1400, 1400, 128, window=20, sinks=140)


@pytest.mark.parametrize("dt", list(TORCH))
def test_strides(cuda_device, dt):
    # Views of a packed projection, an unaligned start, broadcast heads and a transposed gradient.
    packed = _make((2, 150, 8, 64), dt, 3).cuda()
    q, k, v = (t.transpose(1, 2) for t in packed.split((4, 2, 2), dim=2))
    g = _make((2, 150, 4, 64), dt, 4).cuda().transpose(1, 2)
    _check(q, k, v, g, dt, window=50, sinks=2)
    flat = _make((2 * 150 * 4 * 64 + 1,), dt, 5).cuda()
    q = flat[1:].view(2, 4, 150, 64)
    _check(q, k, v, g, dt, window=50, sinks=2)
    wide = _make((2, 1, 150, 64), dt, 6).cuda().expand(2, 2, 150, 64)
    _check(q, wide, v, g.transpose(2, 3).contiguous().transpose(2, 3), dt, window=20)
    _check(q, k, v, torch.ones((), dtype=TORCH[dt], device="cuda").expand(2, 4, 150, 64), dt, window=20)


@pytest.mark.parametrize("dt", list(TORCH))
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_lies_past_the_length_has_no_effect(cuda_device, dt, bad):
    q, g = _make((2, 2, 180, 64), dt, 1).cuda(), _make((2, 2, 180, 64), dt, 2).cuda()
    k, v = _make((2, 1, 200, 64), dt, 3).cuda(), _make((2, 1, 200, 64), dt, 4).cuda()
    for b, n in enumerate((133, 70)):
        k[b, :, n:], v[b, :, n:] = bad, -bad
    _, (dq, dk, dv) = _check(q, k, v, g, dt, lengths=(133, 70), window=60, sinks=3)
    assert torch.all(dk[0, :, 133:] == 0) and torch.all(dv[1, :, 70:] == 0)
    # Keys after the last query, and keys that no window reaches any more.
    k, v = _make((1, 1, 300, 64), dt, 5).cuda(), _make((1, 1, 300, 64), dt, 6).cuda()
    k[:, :, 190:], v[:, :, 190:] = bad, bad
    k[:, :, 3:61], v[:, :, 3:61] = bad, bad
    clean_k, clean_v = (torch.where(torch.isfinite(t), t, torch.zeros_like(t)) for t in (k, v))
    q, g = q[:1, :, :90], g[:1, :, :90]
    options = dict(window=40, sinks=3, query_position_offset=100)
    grads = []
    for kk, vv in ((k, v), (clean_k, clean_v)):
        leaves = [t.detach().clone().requires_grad_() for t in (q, kk, vv)]
        out = F.sliding_window_attention(*leaves, **options)
        grads.append((out, *torch.autograd.grad(out, leaves, g)))
    for a, b in zip(*grads):
        assert torch.equal(a, b) and bool(torch.isfinite(a).all())


def test_extreme_scores(cuda_device):
    """Scores of +-30000 neither overflow nor lose the row; the lowest float as a score is a value."""
    for dt in ("f32", "bf16"):
        q = torch.full((1, 1, 4, 64), 60.0, dtype=TORCH[dt], device="cuda")
        k = torch.full((1, 1, 4, 64), 60.0, dtype=TORCH[dt], device="cuda")
        k[:, :, 1] = -60.0
        v = _make((1, 1, 4, 64), dt, 1).cuda()
        out = F.sliding_window_attention(q, k, v)
        assert torch.equal(out[0, 0, 1], v[0, 0, 0])
        assert torch.equal(out[0, 0, 0], v[0, 0, 0])
        big = torch.finfo(torch.float32).max
        qq, kk = torch.zeros_like(q), torch.zeros_like(k)
        qq[..., 0], kk[..., 0] = 1.0, -big if dt == "f32" else float(torch.finfo(torch.bfloat16).min)
        out = F.sliding_window_attention(qq, kk, v, scale=1.0)
        np.testing.assert_allclose(_np(out)[0, 0], np.cumsum(_np(v)[0, 0], 0) / np.arange(1, 5)[:, None], rtol=1e-2,
                                   atol=1e-2)


@pytest.mark.parametrize("dt", list(TORCH))
def test_gradients_match_differences(cuda_device, dt):
    """Directional differences of the 64-bit forward, to the gradients' own bounds."""
    q, g = _make((1, 4, 140, 64), dt, 1).cuda(), _make((1, 4, 140, 64), dt, 2).cuda()
    k, v = _make((1, 2, 140, 64), dt, 3).cuda(), _make((1, 2, 140, 64), dt, 4).cuda()
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = F.sliding_window_attention(*leaves, window=30, sinks=2)
    grads = torch.autograd.grad(out, leaves, g)
    arrays, up = [_np(t) for t in leaves], _np(g)
    bounds = O.tolerances(*arrays, dt, up, window=30, sinks=2)[2:]
    rng, h = np.random.default_rng(0), 1e-5
    for i, (grad, bound) in enumerate(zip(grads, bounds)):
        d = rng.normal(size=bound.shape)
        f = [float((O.forward(*[x + s * h * d if j == i else x for j, x in enumerate(arrays)], window=30,
                              sinks=2)[0] * up).sum()) for s in (1, -1)]
        assert abs((f[0] - f[1]) / (2 * h) - float((_np(grad) * d).sum())) <= float((bound * np.abs(d)).sum()) + 1e-6


def test_partial_gradients_and_no_grad(cuda_device):
    q, k, v = (_make((1, 2, 70, 64), "bf16", s).cuda() for s in (1, 2, 3))
    v.requires_grad_()
    out = F.sliding_window_attention(q, k, v, window=20)
    out.sum().backward()
    assert v.grad is not None and q.grad is None and k.grad is None
    with torch.no_grad():
        assert not F.sliding_window_attention(q, k, v, window=20).requires_grad


def test_empty_sizes(cuda_device):
    q, k = torch.zeros(2, 4, 0, 64, device="cuda"), torch.randn(2, 2, 7, 64, device="cuda")
    assert F.sliding_window_attention(q, k, k).shape == (2, 4, 0, 64)
    q = torch.randn(2, 4, 3, 64, device="cuda", requires_grad=True)
    empty = torch.zeros(2, 2, 0, 64, device="cuda", requires_grad=True)
    for dt in TORCH.values():
        out = F.sliding_window_attention(q.to(dt), empty.to(dt), empty.to(dt))
        assert torch.all(out == 0)
        dq, dk = torch.autograd.grad(out.float().sum(), (q, empty))
        assert torch.all(dq == 0) and dk.shape == empty.shape
    none = torch.zeros(2, 4, 0, 64, device="cuda", requires_grad=True)
    keys = torch.randn(2, 2, 7, 64, device="cuda", requires_grad=True)
    grads = torch.autograd.grad(F.sliding_window_attention(none, keys, keys).sum(), (none, keys))
    assert torch.all(grads[1] == 0)
    assert F.sliding_window_attention(torch.zeros(0, 4, 3, 64, device="cuda"), k[:0], k[:0]).shape == (0, 4, 3, 64)


def test_another_stream(cuda_device):
    q, k, v = (_make((2, 4, 300, 64), "bf16", s).cuda() for s in (1, 2, 3))
    want = F.sliding_window_attention(q, k, v, window=64, sinks=2)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = F.sliding_window_attention(q, k, v, window=64, sinks=2)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want)


STEPS = [
    # batch, heads, kv_heads, capacity, dim, lengths, options
    (1, 1, 1, 1, 64, (1,), {}),
    (3, 4, 2, 50, 64, (50, 1, 0), {"window": 10, "sinks": 2}),
    (2, 12, 12, 700, 64, (700, 333), {"window": 256, "sinks": 4}),
    (2, 16, 2, 1000, 128, (999, 64), {}),
    (2, 6, 2, 300, 80, (300, 7), {"window": 33, "sinks": 130}),
    (1, 5, 1, 2000, 40, (1999,), {"window": 1, "sinks": 0}),
    (1, 8, 8, 513, 33, (513,), {"window": 300, "sinks": 1, "scale": 0.3}),
    (2, 7, 7, 90, 1, (90, 45), {}),
    (9, 2, 1, 260, 128, (260, 0, -3, 400, 1, 2, 3, 129, 255), {"window": 128}),
]


@pytest.mark.parametrize("dt", list(TORCH))
@pytest.mark.parametrize("index", range(len(STEPS)))
def test_step_matches_oracle(cuda_device, dt, index):
    batch, heads, kv_heads, capacity, dim, lengths, options = STEPS[index]
    q, k, v = _make((batch, heads, dim), dt, index), _make((batch, kv_heads, capacity, dim), dt, index + 50), _make(
        (batch, kv_heads, capacity, dim), dt, index + 90)
    for b, n in enumerate(lengths):                    # whatever an unused slot holds
        k[b, :, max(0, n):], v[b, :, max(0, n):] = float("nan"), float("inf")
    n = torch.tensor(lengths, dtype=torch.int64, device="cuda")
    got = F.sliding_window_attention_step(q.cuda(), k.cuda(), v.cuda(), n, **options)
    assert torch.equal(got, F.sliding_window_attention_step(q.cuda(), k.cuda(), v.cuda(), n, **options))
    for b, length in enumerate(lengths):
        length = min(max(length, 0), capacity)
        arrays = [_np(t) for t in (q[b:b + 1, :, None], k[b:b + 1, :, :length], v[b:b + 1, :, :length])]
        o = dict(window=options.get("window", 0), sinks=options.get("sinks", 0), offset=max(0, length - 1),
                 scale=options.get("scale"))
        want, _ = O.forward(*arrays, **o)
        t_out, _ = O.tolerances(*arrays, dt, **o)
        _within(got[b:b + 1, :, None], want, t_out, f"sequence {b}")


def test_step_equals_the_last_row_of_the_forward(cuda_device):
    """One rounding of the stored type apart (two orders of the same float32 sums)."""
    q, k, v = (_make((2, 4, 400, 64), "f32", s).cuda() for s in (1, 2, 3))
    whole = F.sliding_window_attention(q, k, v, window=100, sinks=4)
    n = torch.full((2,), 400, dtype=torch.int32, device="cuda")
    got = F.sliding_window_attention_step(q[:, :, -1], k, v, n, window=100, sinks=4)
    np.testing.assert_allclose(_np(got), _np(whole[:, :, -1]), rtol=2e-5, atol=2e-6)


def test_offsets_past_32_bits(cuda_device):
    """A cache whose last rows lie more than 2^31 elements behind its start."""
    capacity, dim, n = (1 << 24) + 1000, 128, 200
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GB of free device memory")
    cache = [torch.empty(1, 1, capacity, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    tail = [_make((1, 1, n, dim), "bf16", s).cuda() for s in (1, 2)]
    for c, t in zip(cache, tail):
        c[:, :, -n:] = t
    q = _make((1, 4, 1, dim), "bf16", 3).cuda()
    length = torch.tensor([capacity], dtype=torch.int32, device="cuda")
    got = F.sliding_window_attention_step(q[:, :, 0], *cache, length, window=n - 1)
    short = torch.tensor([n], dtype=torch.int32, device="cuda")
    assert torch.equal(got, F.sliding_window_attention_step(q[:, :, 0], *tail, short, window=n - 1))
    many = _make((1, 4, 150, dim), "bf16", 4).cuda()
    far = F.sliding_window_attention(many, *cache, window=50, query_position_offset=capacity - 150)
    near = F.sliding_window_attention(many, *tail, window=50, query_position_offset=n - 150)
    assert torch.equal(far, near)


def test_refusals_on_the_device(cuda_device):
    q, k = torch.zeros(2, 4, 5, 16, device="cuda"), torch.zeros(2, 2, 7, 16, device="cuda")
    n = torch.tensor([1, 2], device="cuda")
    for options, error, text in (
            ({"window": 0}, ValueError, "window"), ({"window": 1.5}, TypeError, "window"), ({"window": True}, TypeError, "window"),
            ({"sinks": -1}, ValueError, "sinks"), ({"query_position_offset": -1}, ValueError, "offset"),
            ({"query_position_offset": 1 << 30}, ValueError, "query_offset"),
            ({"scale": 0.0}, ValueError, "scale"), ({"scale": float("nan")}, ValueError, "scale"),
            ({"scale": "1"}, TypeError, "scale"), ({"lengths": n[:1]}, ValueError, "lengths"),
            ({"lengths": n.float()}, TypeError, "lengths"), ({"lengths": n.cpu()}, RuntimeError, "lengths")):
        with pytest.raises(error, match=text):
            F.sliding_window_attention(q, k, k, **options)
    with pytest.raises(ValueError, match="rank 3"):
        F.sliding_window_attention_step(q, k, k, n)
    with pytest.raises(RuntimeError, match="CUDA"):
        F.sliding_window_attention(q, k.cpu(), k)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("dim,window,sinks", [(64, 2, 0), (128, 2, 1), (64, 3, 0), (128, 16, 0), (128, 17, 0), (64, 100, 0)])
def test_gradients_of_narrow_windows_keep_their_precision(cuda_device, dt, dim, window, sinks):
    """Beside the result's own rounding one operand is rounded, of the same size and independent of it:
    at most sqrt(2) times the error of rounding the exact gradient, and 1.5 with the sample's spread."""
    q, k, v, g = (_make((1, 4, 1500, dim), dt, s) for s in (1, 2, 3, 4))
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(F.sliding_window_attention(*leaves, window=window, sinks=sinks), leaves, g.cuda())
    wanted = O.backward(*(_np(t) for t in (q, k, v, g)), window=window, sinks=sinks, lengths=None, offset=0, scale=None)
    for got, want in zip(grads, wanted):
        rounded = _np(torch.from_numpy(want).to(TORCH[dt]))
        assert np.linalg.norm(_np(got) - want) <= 1.5 * np.linalg.norm(rounded - want)


@pytest.mark.parametrize("dt", list(TORCH))
def test_masked_keys_of_a_narrow_window(cuda_device, dt):
    q, g = _make((2, 4, 180, 64), dt, 1).cuda(), _make((2, 4, 180, 64), dt, 2).cuda()
    k, v = _make((2, 2, 200, 64), dt, 3).cuda(), _make((2, 2, 200, 64), dt, 4).cuda()
    for b, n in enumerate((133, 1)):
        k[b, :, n:], v[b, :, n:] = float("nan"), float("-inf")
    _, (_, dk, dv) = _check(q, k, v, g, dt, lengths=(133, 1), window=4, sinks=1)
    assert torch.all(dk[0, :, 133:] == 0) and torch.all(dv[1, :, 1:] == 0)


def test_a_graph_replays_what_the_calls_compute(cuda_device):
    """Forward, backward and the one-token step captured once and replayed on new inputs and lengths."""
    shape = dict(q=(2, 8, 600, 64), k=(2, 2, 600, 64), v=(2, 2, 600, 64), g=(2, 8, 600, 64), one=(2, 8, 64))
    inputs = {name: _make(s, "bf16", i).cuda() for i, (name, s) in enumerate(shape.items())}
    lengths = torch.tensor([600, 411], dtype=torch.int32, device="cuda")

    def run(t, n):
        leaves = [t[name].detach().requires_grad_() for name in "qkv"]
        out = F.sliding_window_attention(*leaves, window=90, sinks=4, lengths=n)
        kept = F.dropout(out, 0.3, seed=7, offset=9)
        grads = torch.autograd.grad(kept, leaves, t["g"])
        step = F.sliding_window_attention_step(t["one"], t["k"], t["v"], n, window=90, sinks=4)
        return [out.detach(), kept.detach(), *grads, step]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(inputs, lengths)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = run(inputs, lengths)
    for seed, n in ((20, (600, 411)), (30, (3, 0))):
        for i, (name, s) in enumerate(shape.items()):
            inputs[name].copy_(_make(s, "bf16", seed + i))
        lengths.copy_(torch.tensor(n, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in results]
        for a, b in zip(got, run(inputs, lengths)):
            assert torch.equal(a, b)


def test_second_derivatives_are_refused(cuda_device):
    q, k, v = (_make((1, 2, 40, 64), "f32", s).cuda().requires_grad_() for s in (1, 2, 3))
    want = torch.autograd.grad(F.sliding_window_attention(q, k, v).sum(), (q, k, v))
    grads = torch.autograd.grad(F.sliding_window_attention(q, k, v).sum(), (q, k, v), create_graph=True)
    for a, b in zip(want, grads):
        assert torch.equal(a, b)
    for grad in grads:
        with pytest.raises(RuntimeError, match="only once"):
            torch.autograd.grad(grad.sum() + k.sum(), k, retain_graph=True)
    grad, = torch.autograd.grad(F.dropout(q, 0.5, seed=1).square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="only once"):
        torch.autograd.grad(grad.sum(), q)


@pytest.mark.parametrize("lengths", [(3000, 40), (1, 2900, 700), (0, 0), (1500, 0, 1500, 3), (900, 3000, 0, 20, 2200)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1100, 5)])
def test_step_of_sequences_of_very_different_lengths(cuda_device, lengths, window, sinks):
    """Few sequences over a long cache: many blocks to each, dealt by the lengths."""
    batch, heads, kv_heads, capacity, dim = len(lengths), 32 // len(lengths) * 2, 32 // len(lengths), 3001, 128
    q, k, v = _make((batch, heads, dim), "bf16", 1), _make((batch, kv_heads, capacity, dim), "bf16", 2), _make(
        (batch, kv_heads, capacity, dim), "bf16", 3)
    got = F.sliding_window_attention_step(q.cuda(), k.cuda(), v.cuda(), torch.tensor(lengths, device="cuda"), window=window,
                                          sinks=sinks)
    for b, length in enumerate(lengths):
        arrays = [_np(t) for t in (q[b:b + 1, :, None], k[b:b + 1, :, :length], v[b:b + 1, :, :length])]
        o = dict(window=window or 0, sinks=sinks, offset=max(0, length - 1))
        _within(got[b:b + 1, :, None], O.forward(*arrays, **o)[0], O.tolerances(*arrays, "bf16", **o)[0], f"sequence {b}")
