"""The status word when a process's first call is captured: it belongs to no
graph, so it is clear before the first replay and a replay does not clear it."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest
import torch

import vllm_rlt_b200 as rb
from vllm_rlt_b200 import _lib

pytestmark = pytest.mark.gpu

FIRST_USE = """
import torch, vllm_rlt_b200 as rb
from vllm_rlt_b200 import _lib
device = torch.device("cuda", 0)
junk = [torch.full((n,), -1, dtype=torch.int32, device=device) for n in (1, 128, 1 << 20)]
x = torch.randn(4, 128, device=device).bfloat16()
w = torch.randn(256, 128, device=device).bfloat16()
tokens = torch.tensor([1, 2, 3, 300], device=device)
fine = torch.tensor([1, 2, 3, 4], device=device)
torch.cuda.synchronize()
del junk
graph = torch.cuda.CUDAGraph()
%s
    with torch.cuda.graph(graph):
        scored = rb.token_logprobs(x, w, tokens)
bad = [_lib.STATUS_BITS[128]]
assert _lib.read_status(device) == []
rb.token_logprobs(x, w, tokens)
held = tokens.clone()
tokens.copy_(fine)
graph.replay()
assert _lib.read_status(device) == bad
graph.replay()
assert _lib.read_status(device) == []
tokens.copy_(held)
graph.replay()
assert _lib.read_status(device) == bad
assert _lib.read_status(device) == []
assert scored.isnan().tolist() == [False, False, False, True]
del graph, scored
torch.cuda.empty_cache()
junk = [torch.full((n,), -1, dtype=torch.int32, device=device) for n in (1, 128, 1 << 20)]
assert _lib.read_status(device) == []
"""


@pytest.mark.parametrize("context", ["if True:", "with torch.inference_mode():"])
def test_first_requested_while_capturing(context):
    subprocess.run([sys.executable, "-c", FIRST_USE % context], check=True,
                   cwd=Path(__file__).resolve().parents[1], timeout=300)


def test_it_is_one_tensor_per_device():
    device = torch.device("cuda", 0)
    word = _lib.status_word(device)
    assert word is _lib.status_word(torch.device("cuda"))
    assert word.shape == (1,) and word.dtype == torch.int32 and word.device == device
    word.fill_(2)
    assert _lib.read_status(device) == [_lib.STATUS_BITS[2]] and word.item() == 0


def test_every_entry_reports_into_the_same_word():
    """Whoever asked first: the extension's calls, and a tensor made anew."""
    h = torch.randn(2, 64, device="cuda").bfloat16()
    w = torch.randn(100, 64, device="cuda").bfloat16()
    bad = torch.tensor([5, 100], device="cuda")
    rb.token_logprobs(h, w, bad)
    _lib._status.pop(0, None)
    assert rb.check_errors() == [_lib.STATUS_BITS[128]]
    rb.token_logprobs(h, w, bad)
    assert rb.check_errors() == [_lib.STATUS_BITS[128]] and rb.check_errors() == []
