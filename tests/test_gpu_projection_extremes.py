"""Projection operators on numbers at the ends of their types."""

from __future__ import annotations

import pytest
import torch

import vllm_rlt_b200 as rb
from test_gpu_projections import generator, normal

pytestmark = pytest.mark.gpu


def time_of(call):
    call()
    torch.cuda.synchronize()
    best = float("inf")
    for _ in range(3):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        call()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


@pytest.mark.parametrize("rows", [40, 600])
def test_one_infinite_weight_costs_its_own_entry_alone(rows):
    """fp32 recomputes what its parts cannot carry: here one vocabulary entry of
    each row (2000 others stay), 1 of the 64 that a thread holds. The clean call
    reads x and the weights once; rows of 5632 recomputed one feature after the
    other may take some of that time again, all 64 entries took 150 of it."""
    g = generator(81)
    x, w = normal(g, rows, 5632), normal(g, 2000, 5632, std=0.02)
    clean = time_of(lambda: rb.greedy_tokens(x, w))
    before, _ = rb.greedy_tokens(x, w)
    w[700, 3] = float("inf")
    assert time_of(lambda: rb.greedy_tokens(x, w)) < 40 * clean
    tokens, logprobs = rb.greedy_tokens(x, w)
    up = x[:, 3] > 0
    assert tokens[up].eq(700).all() and logprobs[up].isnan().all()
    rest = ~up & before.ne(700)
    assert rest.any() and torch.equal(tokens[rest], before[rest]) and logprobs[rest].isfinite().all()
