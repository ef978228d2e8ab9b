"""Tensors whose memory does not hold their values are refused: the kernels read
memory."""

from __future__ import annotations

import pytest
import torch

import vllm_rlt_b200 as rb


def negated(*shape):
    """The imaginary part of a conjugate: values -1 where memory holds 1."""
    t = torch.complex(torch.zeros(shape), torch.ones(shape)).conj().imag
    assert t.is_neg() and t.sum() < 0
    return t


def lazy_zeros(*shape):
    return torch._efficientzerotensor(shape)


@pytest.mark.parametrize("bad", [negated, lazy_zeros])
def test_refused(bad):
    x, w = torch.zeros(2, 8), torch.zeros(4, 8)
    calls = [lambda: rb.linear(bad(2, 8), w), lambda: rb.linear(x, bad(4, 8)),
             lambda: rb.linear(x, w, bad(4)), lambda: rb.linear(x, w, residual=bad(2, 4)),
             lambda: rb.linear(x, w, out=bad(2, 4)), lambda: rb.gated_linear(bad(2, 8), w),
             lambda: rb.gated_linear(x, w, out=bad(2, 2)), lambda: rb.greedy_tokens(x, bad(4, 8)),
             lambda: rb.token_logprobs(bad(2, 8), w, torch.zeros(2, dtype=torch.int64))]
    for call in calls:
        with pytest.raises(ValueError, match="does not hold its values"):
            call()
    with pytest.raises(ValueError, match="requires a CUDA device"):
        rb.linear(negated(2, 8).resolve_neg(), w)
