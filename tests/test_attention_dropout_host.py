"""Host side of the attention and dropout operators, without a GPU: the oracles against known
answers and differences, the C entry points' refusals, struct layouts and the Python checks."""
import ctypes
import shutil
import subprocess

import numpy as np
import pytest
import torch

from conftest import REPO
from namitorch_b200 import _native as N
from namitorch_b200.nn import functional as F
from oracle import attention as OA
from oracle import dropout as OD


def test_philox_known_answers():
    """The authors' published vectors for a zero and an all-ones counter and key."""
    zeros, ones = np.zeros((1, 4), np.uint64), np.full((1, 4), 0xFFFFFFFF, np.uint64)
    assert [hex(int(w)) for w in OD.philox4x32(zeros, (0, 0), 7)[0]] == ["0x5f6fb709", "0xd893f64", "0x4f121f81",
                                                                         "0x4f730a48"]
    assert [hex(int(w)) for w in OD.philox4x32(zeros, (0, 0), 10)[0]] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c",
                                                                          "0x9b00dbd8"]
    assert [hex(int(w)) for w in OD.philox4x32(ones, (0xFFFFFFFF, 0xFFFFFFFF), 10)[0]] == [
        "0x408f276d", "0x41c83b0e", "0xa20bc7c6", "0x6d5451fd"]


def test_keep_rate_and_independence_of_offsets():
    n, p = 1 << 18, 0.3
    a, b = OD.keep_mask((n,), p, 12345, 0), OD.keep_mask((n,), p, 12345, 1)
    sigma = (p * (1 - p) / n) ** 0.5
    for mask in (a, b, OD.keep_mask((n,), p, 12346, 0)):
        assert abs(mask.mean() - (1 - p)) < 6 * sigma
    # Two independent masks agree with probability p^2 + (1 - p)^2.
    agree = p * p + (1 - p) ** 2
    assert abs((a == b).mean() - agree) < 6 * (agree * (1 - agree) / n) ** 0.5


@pytest.mark.parametrize("window,sinks,lengths,offset", [(0, 0, None, 0), (3, 0, None, 2), (4, 2, (5, 0), 0),
                                                         (2, 1, (9, 3), 1)])
def test_oracle_gradients_match_differences(window, sinks, lengths, offset):
    rng = np.random.default_rng(5)
    q, g = rng.normal(size=(2, 4, 6, 5)), rng.normal(size=(2, 4, 6, 5))
    k, v = rng.normal(size=(2, 2, 9, 5)), rng.normal(size=(2, 2, 9, 5))
    options = dict(window=window, sinks=sinks, lengths=lengths, offset=offset)
    grads = OA.backward(q, k, v, g, **options)
    h = 1e-5
    for which, grad in enumerate(grads):
        d = rng.normal(size=grad.shape)
        moved = [[x + s * h * d if i == which else x for i, x in enumerate((q, k, v))] for s in (1, -1)]
        up, down = (float((OA.forward(*m, **options)[0] * g).sum()) for m in moved)
        assert abs((up - down) / (2 * h) - float((grad * d).sum())) < 1e-7


def test_oracle_rows_without_keys_are_zero():
    rng = np.random.default_rng(0)
    q, k = rng.normal(size=(1, 1, 4, 3)), rng.normal(size=(1, 1, 2, 3))
    out, lse = OA.forward(q, k, k, window=1, offset=0)      # queries 2 and 3 see no key
    assert np.all(out[0, 0, 2:] == 0) and np.all(np.isneginf(lse[0, 0, 2:])) and np.all(np.isfinite(lse[0, 0, :2]))


def _attention(**changes):
    a = N.AttentionArgs(dtype=N.NT_BF16, head_dim=64, batch=1, query_heads=4, kv_heads=2, queries=8, keys=8, query=16,
                        key=16, value=16, output=16, scale=0.125)
    for name, value in changes.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("changes,message", [
    ({"head_dim": 0}, b"head_dim"), ({"head_dim": 129}, b"head_dim"), ({"kv_heads": 3}, b"multiple"),
    ({"kv_heads": 0}, b"multiple"), ({"batch": -1}, b"nonnegative"), ({"batch": 70000}, b"65536"),
    ({"keys": 1 << 30}, b"2^30"), ({"window": -1}, b"window"), ({"sinks": -2}, b"sinks"),
    ({"query_offset": 1 << 30}, b"query_offset"), ({"scale": 0.0}, b"scale"), ({"scale": float("nan")}, b"scale"),
    ({"scale": float("inf")}, b"scale"), ({"key": None}, b"NULL")])
def test_attention_entry_points_refuse(changes, message):
    lib = N.load()
    for entry in (lib.nt_attention_forward, lib.nt_attention_backward, lib.nt_attention_step):
        a = _attention(**changes)
        if entry is lib.nt_attention_backward:
            a.gradient = a.grad_query = a.grad_key = a.grad_value = a.lse = 16
        if entry is lib.nt_attention_step:
            a.queries, a.lengths = 1, 16
        assert entry(ctypes.byref(a), None) == N.NT_EINVAL
        assert message in lib.nt_last_error(), lib.nt_last_error()
    assert lib.nt_attention_forward(ctypes.byref(_attention(dtype=9)), None) == N.NT_EUNSUPPORTED


def test_attention_entry_points_refuse_missing_parts_and_accept_empty_calls():
    lib = N.load()
    for entry in (lib.nt_attention_forward, lib.nt_attention_backward, lib.nt_attention_step):
        assert entry(None, None) == N.NT_EINVAL
    assert lib.nt_attention_step(ctypes.byref(_attention(queries=2, lengths=16)), None) == N.NT_EINVAL
    assert lib.nt_attention_step(ctypes.byref(_attention(queries=1)), None) == N.NT_EINVAL   # no lengths
    a = _attention(gradient=16, grad_query=16, grad_key=16, grad_value=16, lse=16)
    assert lib.nt_attention_backward(ctypes.byref(a), None) == N.NT_EINVAL
    assert b"workspace" in lib.nt_last_error()
    assert lib.nt_attention_forward(ctypes.byref(_attention(batch=0)), None) == N.NT_OK
    assert lib.nt_attention_forward(ctypes.byref(_attention(queries=0)), None) == N.NT_OK
    assert lib.nt_attention_backward(ctypes.byref(_attention(batch=0)), None) == N.NT_OK
    assert lib.nt_attention_workspace_size(None) == 0
    assert lib.nt_attention_workspace_size(ctypes.byref(_attention())) >= 4 * 8 * 4
    # A window with sinks cuts the sink keys' queries into pieces, whose sums need room.
    plain = lib.nt_attention_workspace_size(ctypes.byref(_attention(queries=8192, keys=8192, window=256)))
    sinks = lib.nt_attention_workspace_size(ctypes.byref(_attention(queries=8192, keys=8192, window=256, sinks=4)))
    assert sinks > plain


def test_dropout_entry_points_refuse():
    lib = N.load()
    make = lambda **c: N.DropoutArgs(**{**dict(dtype=N.NT_F32, rows=2, width=8, p=0.5, input=16, output=16), **c})  # noqa: E731
    for entry in (lib.nt_dropout_forward, lib.nt_dropout_backward):
        assert entry(None, None) == N.NT_EINVAL
        for changes in ({"p": 1.0}, {"p": -0.1}, {"p": float("nan")}, {"rows": -1}, {"width": -1},
                        {"rows": 1 << 40, "width": 1 << 30}, {"input": None}):
            assert entry(ctypes.byref(make(**changes)), None) == N.NT_EINVAL, changes
        assert entry(ctypes.byref(make(dtype=5)), None) == N.NT_EUNSUPPORTED
        assert entry(ctypes.byref(make(rows=0)), None) == N.NT_OK
        assert entry(ctypes.byref(make(width=0)), None) == N.NT_OK
    assert lib.nt_dropout_backward(ctypes.byref(make(grad_bias=16)), None) == N.NT_EINVAL
    assert b"workspace" in lib.nt_last_error()
    assert lib.nt_dropout_workspace_size(0, 8) == 0 and lib.nt_dropout_workspace_size(2, 8) >= 64


def test_attention_arguments_are_checked():
    q, k = torch.zeros(2, 4, 5, 16), torch.zeros(2, 2, 7, 16)
    cases = [
        ((q[0], k, k), {}, ValueError, "rank 4"), ((q, k, k[:, :, :6]), {}, ValueError, "shape"),
        ((q, k[:1], k[:1]), {}, ValueError, "shape"), ((q[:, :3], k, k), {}, ValueError, "whole number"),
        ((q, k.double(), k), {}, TypeError, "one dtype"), ((q.double(), k, k), {}, TypeError, "supports"),
        ((torch.zeros(2, 4, 5, 200), torch.zeros(2, 2, 7, 200), torch.zeros(2, 2, 7, 200)), {}, ValueError, "dimension"),
        ((None, k, k), {}, TypeError, "Tensor"), ((q, k, k), {}, RuntimeError, "CUDA")]
    for arrays, options, error, text in cases:
        with pytest.raises(error, match=text):
            F.sliding_window_attention(*arrays, **options)
    with pytest.raises(TypeError, match="lengths"):
        F.sliding_window_attention_step(q[:, :, 0], k, k, None)
    x = torch.zeros(3, 8)
    for options, error in (({"p": 1.0}, ValueError), ({"p": True}, TypeError), ({"seed": -1}, ValueError),
                           ({"seed": 1 << 64}, ValueError), ({"offset": 1.5}, TypeError), ({"training": 1}, TypeError),
                           ({"bias": torch.zeros(7)}, ValueError), ({"residual": torch.zeros(8)}, ValueError),
                           ({"bias": torch.zeros(8, dtype=torch.float16)}, TypeError), ({}, RuntimeError)):
        with pytest.raises(error):
            F.dropout(x, **{**dict(p=0.1, seed=1), **options})
    with pytest.raises(TypeError):
        F.dropout(x.double(), 0.1, seed=1)


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_struct_layouts_match_the_c_compiler(tmp_path):
    structs = {"nt_attention_args": N.AttentionArgs, "nt_dropout_args": N.DropoutArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "namitorch_b200.h"', "int main(void) {"]
    for cname, cls in structs.items():
        lines.append(f'  printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, *_ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-I", str(REPO / "include"), str(src), "-o", str(exe)], check=True)
    out = dict(line.rsplit(" ", 1) for line in
               subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for cname, cls in structs.items():
        assert int(out[cname]) == ctypes.sizeof(cls)
        for f, *_ in cls._fields_:
            assert int(out[f"{cname}.{f}"]) == getattr(cls, f).offset, f
