"""Long sums of the 16-bit projection operators. The tensor core truncates as it
accumulates, so operands of one sign come out too small by an amount that grows
with the number of input features added there: the kernels may add some hundreds,
and have to add those sums rounding to nearest.

The measure is the mean relative error over all outputs. What a sum of 512
features loses is taken from a call of that length (on more than 64 rows, where
nothing is split), and what a longer one may lose is twice that, and a rounding
(2^-24) for each of its sums."""

from __future__ import annotations

import pytest
import torch

import projection_oracle as po
import vllm_rlt_b200 as rb
from test_gpu_projections import assert_within, generator, make_weight, normal

pytestmark = pytest.mark.gpu

HALVES = [torch.bfloat16, torch.float16]


def one_sign(g, lines, inner, dtype, scale=1.0):
    """Values in [0.5, 1.5) times a factor of the line's own in [1, 2): sums that
    spread over more than an octave, so that their roundings average out."""
    spread = torch.rand(lines, 1, device="cuda", generator=g) + 1
    return ((torch.rand(lines, inner, device="cuda", generator=g) + 0.5) * spread * scale).to(dtype)


def mean_error(rows, inner, outer, dtype, layout):
    g = generator(rows + inner)
    x = one_sign(g, rows, inner, dtype)
    w = one_sign(g, inner, outer, dtype).t() if layout == "in_out" else one_sign(g, outer, inner, dtype)
    y = rb.linear(x, w)
    left = rb.linear(x, w, residual=-y)  # what the first rounding took: exact in fp32
    want = x.double() @ w.double().t()
    return ((y.double() + left.double() - want) / want).mean().item()


@pytest.mark.parametrize("layout", ["out_in", "in_out"])
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rows,inner,outer", [
    (300, 8192, 2000), (100, 8192, 600), (64, 8192, 2048), (33, 8192, 700), (1, 8192, 2000),
    (64, 2048, 20000), (16, 8192, 20000), (64, 4160, 20000)])
def test_linear(rows, inner, outer, dtype, layout):
    least = abs(mean_error(300, 512, 2000, dtype, layout))
    # each output's remainder is rounded to half a step of at most half a step
    noise = 5 * (torch.finfo(dtype).eps / 2) ** 2 / (rows * outer) ** 0.5
    assert abs(mean_error(rows, inner, outer, dtype, layout)) <= (
        2 * least + inner / 512 * 2.0 ** -24 + noise)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rows,inner,outer", [(300, 8192, 2000), (64, 8192, 5000), (16, 8192, 20000)])
def test_gated_linear(rows, inner, outer, dtype):
    def error(rows, inner, outer):
        """The mean error, and what the outputs' own roundings, half a step each,
        may leave of it. Products beyond fp16's largest number (65504) are
        infinite and count for nothing."""
        g = generator(rows * 3 + inner)
        x = one_sign(g, rows, inner, dtype, 1 / 64)
        w = one_sign(g, 2 * outer, inner, dtype)
        got = rb.gated_linear(x, w, activation=None).double()
        want = (x.double() @ w[:outer].double().t()) * (x.double() @ w[outer:].double().t())
        small = want < 65000
        assert bool(got[want > 66000].isinf().all()) or dtype == torch.bfloat16
        off = ((got - want) / want)[small]
        return off.mean().abs().item(), 5 * torch.finfo(dtype).eps / 2 / off.numel() ** 0.5

    least, short = error(300, 512, 4000)
    most, noise = error(rows, inner, outer)
    assert most <= 2 * (least + short) + inner / 256 * 2.0 ** -24 + noise


@pytest.mark.parametrize("layout", ["out_in", "in_out"])
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rows,inner,outer", [
    (16, 4096, 20000), (64, 2048, 20000), (64, 2112, 20000), (3, 8256, 20000), (33, 1000, 20011)])
def test_few_rows_of_wide_weights(rows, inner, outer, dtype, layout):
    """One CTA for a tile's whole sum: in several accumulators, or, where they
    cannot hold it, by the kernel for many rows."""
    g = generator(rows + outer)
    x = normal(g, rows, inner, dtype=dtype)
    w = make_weight(g, outer, inner, dtype, layout)
    assert_within(rb.linear(x, w), *po.linear(x, w))
    del w
    w = make_weight(g, 2 * outer, inner, dtype, layout)
    assert_within(rb.gated_linear(x, w), *po.gated(x, w))
