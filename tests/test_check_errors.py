"""check_errors: the public look at what kernels report."""

from __future__ import annotations

import pytest
import torch

import vllm_rlt_b200 as rb
from vllm_rlt_b200 import _lib


def test_a_cpu_device_is_refused():
    for device in ("cpu", torch.device("cpu")):
        with pytest.raises(ValueError, match="requires a CUDA device"):
            rb.check_errors(device)


@pytest.mark.gpu
def test_a_reported_token_is_seen_once():
    h = torch.randn(3, 64, device="cuda").bfloat16()
    w = torch.randn(100, 64, device="cuda").bfloat16()
    rb.check_errors()
    rb.token_logprobs(h, w, torch.tensor([5, 99, -1], device="cuda"))
    assert rb.check_errors() == []
    for device in (None, "cuda", 0, "cuda:0", h.device):
        rb.token_logprobs(h, w, torch.tensor([5, 100, -1], device="cuda"))
        assert rb.check_errors(device) == [_lib.STATUS_BITS[128]]
        assert rb.check_errors(device) == []
