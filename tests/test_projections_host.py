"""Refusals of the projection operators: every one is made before any launch,
so they are tested without a GPU."""

from __future__ import annotations

import pytest
import torch

import vllm_rlt_b200 as rb
from vllm_rlt_b200 import _lib
from vllm_rlt_b200.kernels import projections


class FakeCuda:
    """A CPU tensor that reports a CUDA device, to reach the checks behind the
    device check; the calls below are refused before anything touches a GPU."""

    def __init__(self, t, device="cuda:0"):
        self.t, self.device = t, torch.device(device)

    def __getattr__(self, name):
        return getattr(self.t, name)

    def __getitem__(self, index):
        return FakeCuda(self.t[index], self.device)

    def t_(self):
        return FakeCuda(self.t.t(), self.device)


def fake(*shape, dtype=torch.bfloat16, device="cuda:0"):
    return FakeCuda(torch.zeros(shape, dtype=dtype), device)


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 8), torch.zeros(4, 8)
    for call in (lambda: rb.linear(x, w), lambda: rb.gated_linear(x, w),
                 lambda: rb.greedy_tokens(x, w),
                 lambda: rb.token_logprobs(x, w, torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(ValueError, match="requires a CUDA device"):
            call()


@pytest.mark.parametrize("call", [rb.linear, rb.gated_linear, rb.greedy_tokens])
def test_operands(call):
    x, w = fake(2, 8), fake(4, 8)
    for bad_x, bad_w, words in [
        (fake(8), w, "expected x"), (x, fake(8), "expected x"), (x, fake(4, 9), "expected x"),
        (fake(2, 3, 8), w, "expected x"), (fake(2, 8, dtype=torch.float64), w, "dtype"),
        (x, fake(4, 8, dtype=torch.float16), "dtype"), (x, fake(4, 8, device="cuda:1"), "device"),
        (fake(2, 0), fake(4, 0), "in_features"),
    ]:
        with pytest.raises(ValueError, match=words):
            call(bad_x, bad_w)
    strided = FakeCuda(torch.zeros(4, 16, dtype=torch.bfloat16)[:, ::2])
    with pytest.raises(ValueError, match="contiguous"):
        call(x, strided)


def test_epilogue_arguments():
    x, w = fake(2, 8), fake(4, 8)
    for kwargs, words in [
        (dict(bias=fake(5)), "bias"), (dict(bias=fake(4, dtype=torch.float32)), "bias"),
        (dict(bias=fake(4, device="cuda:1")), "bias"), (dict(residual=fake(2, 5)), "residual"),
        (dict(residual=fake(2, 4, dtype=torch.float16)), "residual"),
        (dict(activation="tanh"), "activation"), (dict(activation=["silu"]), "activation"),
        (dict(out=fake(3, 4)), "out"), (dict(out=fake(2, 4, dtype=torch.float32)), "out"),
        (dict(out=FakeCuda(torch.zeros(2, 8, dtype=torch.bfloat16)[:, ::2])), "out"),
        (dict(out=FakeCuda(torch.zeros(1, 4, dtype=torch.bfloat16).expand(2, 4))), "out"),
    ]:
        with pytest.raises(ValueError, match=words):
            rb.linear(x, w, **kwargs)
    with pytest.raises(ValueError, match="gate rows"):
        rb.gated_linear(x, fake(5, 8))
    with pytest.raises(ValueError, match="activation"):
        rb.gated_linear(x, w, activation="swish")


def test_head_arguments():
    h, w = fake(2, 8), fake(4, 8)
    for tokens in (fake(2, dtype=torch.int32), fake(3, dtype=torch.int64),
                   fake(2, 1, dtype=torch.int64), fake(2, dtype=torch.int64, device="cuda:1")):
        with pytest.raises(ValueError, match="tokens|device"):
            rb.token_logprobs(h, w, tokens)
    with pytest.raises(ValueError, match="vocabulary"):
        rb.greedy_tokens(h, fake(0, 8))


def test_weight_layouts():
    def strides(w):
        w = FakeCuda(w)
        return projections._operands(fake(2, w.shape[1], dtype=w.dtype), w, "")[5:7]

    assert strides(torch.zeros(4, 8)) == (8, 1)
    assert strides(torch.zeros(8, 4).t()) == (1, 4)
    assert strides(torch.zeros(4, 16)[:, ::16]) == (16, 1)  # one input feature
    assert strides(torch.zeros(1, 16)[:, ::2]) == (1, 2)  # one output feature


def test_c_entries_refuse_before_any_launch():
    lib = _lib.load()
    p = None

    def linear(dtype=2, rows=2, inner=8, outer=4, act=0, xs=8, ns=8, ks=1):
        return lib.rlt_linear(p, p, p, p, p, p, 0, p, dtype, rows, inner, outer, act, xs, ns, ks,
                              0, 4, p)

    def gated(dtype=2, rows=2, inner=8, outer=4, act=0, xs=8, ns=8, ks=1):
        return lib.rlt_gated_linear(p, p, p, p, 0, p, dtype, rows, inner, outer, act, xs, ns, ks,
                                    4, p)

    def head(dtype=2, rows=2, inner=8, outer=4, xs=8, ns=8, ks=1, act=0):
        return lib.rlt_vocab_head(p, p, p, p, p, p, 0, p, dtype, rows, inner, outer, xs, ns, ks, p)

    for call in (linear, gated, head):
        assert call(dtype=3) == -1
        assert call(rows=-1) == -5
        assert call(inner=0) == -5
        assert call(outer=-1) == -5
        assert call(ns=16, ks=2) == -5
        assert call(rows=0) == 0
    for call in (linear, gated):
        assert call(act=6) == -5 and call(act=-1) == -5
        assert call(outer=0) == 0
    assert head(outer=0) == -5
    assert head() == -4  # no workspace
