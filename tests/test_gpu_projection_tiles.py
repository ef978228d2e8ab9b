"""Projection operators at the sizes where their kernels take wide tiles, pairs
of CTAs, several tiles per CTA and several partial sums per output, against
their 64-bit forms (tests/projection_oracle.py derives every tolerance).

Tilings named here are those of a device with 148 SMs."""

from __future__ import annotations

import pytest
import torch

import projection_oracle as po
import vllm_rlt_b200 as rb
from test_gpu_projections import TYPES, assert_within, generator, make_weight, normal, peaked

pytestmark = pytest.mark.gpu

WIDE = [  # rows, in, out
    (4096, 192, 2048),   # pairs, 160 (weights [in, out]: 128) features wide, 3 (4) tiles each
    (1030, 328, 4104),   # the same with a last tile of few rows and features
    (700, 1088, 5000),   # pairs, 224 (256) wide, 17 slices of input features
    (300, 1000, 20011),  # pairs, 192 wide; [in, out]: single CTAs, 256 wide, two tiles each
    (70, 5632, 600),     # single CTAs, 32 (64) wide, a long sum
]


@pytest.mark.parametrize("layout", ["out_in", "in_out"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner,outer", WIDE)
def test_linear_on_wide_tiles(rows, inner, outer, dtype, layout):
    g = generator(rows + outer)
    x = normal(g, rows, inner, dtype=dtype)
    w = make_weight(g, outer, inner, dtype, layout)
    bias = normal(g, outer, dtype=dtype)
    residual = normal(g, rows, outer, dtype=dtype)
    got = rb.linear(x, w, bias, activation="silu", residual=residual)
    assert_within(got, *po.linear(x, w, bias, "silu", residual))
    again = [rb.linear(x, w, bias, activation="silu", residual=residual) for _ in range(5)]
    assert all(torch.equal(a, got) for a in again)


@pytest.mark.parametrize("layout", ["out_in", "in_out"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner,outer", WIDE)
def test_gated_linear_on_wide_tiles(rows, inner, outer, dtype, layout):
    g = generator(rows - outer)
    x = normal(g, rows, inner, dtype=dtype)
    w = make_weight(g, 2 * outer, inner, dtype, layout)
    got = rb.gated_linear(x, w)
    assert_within(got, *po.gated(x, w))
    assert all(torch.equal(rb.gated_linear(x, w), got) for _ in range(5))


@pytest.mark.parametrize("layout", ["out_in", "in_out"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner,vocab", [
    (1, 2048, 49152), (64, 2048, 49152), (256, 2048, 49152), (33, 1088, 20483), (300, 1000, 20483),
    (700, 2048, 20011), (64, 768, 3001), (20, 704, 20483)])
def test_head_over_several_sums_and_tiles(rows, inner, vocab, dtype, layout):
    g = generator(rows + inner)
    h, w, target = peaked(g, rows, inner, vocab, dtype, layout)
    chosen = torch.randint(vocab, (rows,), device="cuda", generator=g)
    chosen[::2] = target[::2]
    tokens, logprobs = rb.greedy_tokens(h, w)
    scored = rb.token_logprobs(h, w, chosen)
    z, e, lp, bound = po.vocab(h, w)
    picked = z.gather(1, tokens[:, None])[:, 0]
    top = z.topk(2, -1).values
    assert bool((picked >= top[:, 0] - 2 * e[:, 0]).all())
    clear = top[:, 0] - top[:, 1] > 2 * e[:, 0]
    assert torch.equal(tokens[clear], z.argmax(-1)[clear])
    for at, got in ((tokens[:, None], logprobs), (chosen[:, None], scored)):
        assert_within(got, lp.gather(1, at)[:, 0], bound.gather(1, at)[:, 0])
