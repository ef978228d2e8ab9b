"""Sizes near 2^31 are refused before any launch: the kernels and their tilings
step past a size in 32 bits. Meta tensors have such sizes without the memory."""

from __future__ import annotations

import pytest
import torch

import vllm_rlt_b200 as rb
from vllm_rlt_b200 import _lib

MOST = 2 ** 31 - 2 ** 16


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("size", [2 ** 31 - 1, MOST + 1, 2 ** 31 + 8])
def test_python_calls(size):
    tokens = meta(size, dtype=torch.int64)
    for call in (lambda: rb.linear(meta(size, 8), meta(4, 8)),
                 lambda: rb.linear(meta(2, size), meta(4, size)),
                 lambda: rb.linear(meta(2, 8), meta(size, 8)),
                 lambda: rb.gated_linear(meta(size, 8), meta(4, 8)),
                 lambda: rb.greedy_tokens(meta(2, 8), meta(size, 8)),
                 lambda: rb.token_logprobs(meta(size, 8), meta(4, 8), tokens)):
        with pytest.raises(ValueError, match="at most 2147418112"):
            call()


def test_the_largest_size_is_refused_for_its_device_alone():
    with pytest.raises(ValueError, match="requires a CUDA device"):
        rb.linear(meta(MOST, 8), meta(MOST, 8))


@pytest.mark.parametrize("size", [2 ** 31 - 1, MOST + 1])
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_c_entries(size, dtype):
    lib = _lib.load()
    p = None
    for rows, inner, outer in ((size, 8, 4), (2, size, 4), (2, 8, size)):
        assert lib.rlt_linear_workspace_bytes(16, 16, dtype, rows, inner, outer, 0, 9, 9, 1) == 0
        assert lib.rlt_vocab_head_workspace_bytes(16, 16, dtype, rows, inner, outer, 9, 9, 1) == 0
        assert lib.rlt_linear(p, p, p, p, p, p, 0, p, dtype, rows, inner, outer, 0, inner, inner, 1,
                              0, outer, p) == -5
        assert lib.rlt_gated_linear(p, p, p, p, 0, p, dtype, rows, inner, outer, 0, inner, inner, 1,
                                    outer, p) == -5
        assert lib.rlt_vocab_head(p, p, p, p, p, p, 0, p, dtype, rows, inner, outer, inner, inner,
                                  1, p) == -5
