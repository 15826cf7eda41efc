"""The word that says that a wait inside an attention kernel ran out: it is reported, it starts as 0 without
a launch, and a graph that holds the first call of a process does not clear it."""
import subprocess
import sys
import textwrap

import pytest
import torch

from conftest import REPO
from namitorch_b200 import _native as N
from namitorch_b200.backends.attention import AttentionCUDAKernels


@pytest.mark.parametrize("word", [0, 1, 5])
def test_a_set_word_is_an_error(word):
    kernels = AttentionCUDAKernels()
    kernels._error = torch.tensor([word], dtype=torch.int32)
    if word:
        with pytest.raises(RuntimeError, match="ran out"):
            kernels.check()
    else:
        kernels.check()


def test_the_entry_point_refuses_a_null_pointer():
    assert N.load().nt_attention_error_word(None) == N.NT_EINVAL


CHILD = """
    import torch
    from namitorch_b200.backends import get_backend
    from namitorch_b200.nn import functional as F
    q = torch.randn(1, 2, 70, 64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = F.sliding_window_attention(q, q, q, window=9)
    kernels = get_backend(q).attention
    word = kernels._error
    from namitorch_b200 import _native as N
    address = N.C.c_void_p()
    assert N.load().nt_attention_error_word(N.C.byref(address)) == 0 and address.value == word.data_ptr()
    graph.replay()
    torch.cuda.synchronize()
    kernels.check()
    assert torch.equal(out, F.sliding_window_attention(q, q, q, window=9))
    word.fill_(1)
    graph.replay()
    torch.cuda.synchronize()
    try:
        kernels.check()
    except RuntimeError as error:
        assert "ran out" in str(error)
    else:
        raise AssertionError("the replay cleared the word")
    try:
        F.check_attention("cuda")
    except RuntimeError as error:
        assert "ran out" in str(error)
    else:
        raise AssertionError("check_attention passed")
    word.zero_()
    F.check_attention()
    F.check_attention(q.device)
    print("done")
"""


@pytest.mark.gpu
def test_a_graph_with_the_first_call_keeps_the_word(cuda_device):
    run = subprocess.run([sys.executable, "-c", textwrap.dedent(CHILD)], cwd=REPO, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip().endswith("done"), run.stderr[-2000:]
