"""Refusals of the projection operators. Every one is made before any launch,
the CUDA device last, so CPU (and meta) tensors meet all the others."""

from __future__ import annotations

import pytest
import torch

import vllm_rlt_b200 as rb
from vllm_rlt_b200 import _lib


def zeros(*shape, dtype=torch.bfloat16, device="cpu"):
    return torch.zeros(shape, dtype=dtype, device=device)


def test_cpu_tensors_are_refused():
    x, w = zeros(2, 8), zeros(4, 8)
    for call in (lambda: rb.linear(x, w), lambda: rb.gated_linear(x, w),
                 lambda: rb.linear(x, w, zeros(4), activation="gelu", residual=zeros(2, 4),
                                   out=zeros(2, 4)),
                 lambda: rb.linear(x, w.t().contiguous().t()),
                 lambda: rb.greedy_tokens(x, w),
                 lambda: rb.token_logprobs(x, w, zeros(2, dtype=torch.int64))):
        with pytest.raises(ValueError, match="requires a CUDA device"):
            call()


@pytest.mark.parametrize("call", [
    rb.linear, rb.gated_linear, rb.greedy_tokens,
    lambda x, w: rb.token_logprobs(x, w, zeros(2, dtype=torch.int64))])
def test_operands(call):
    x, w = zeros(2, 8), zeros(4, 8)
    for bad_x, bad_w, words in [
        (zeros(8), w, "expected x"), (x, zeros(8), "expected x"), (x, zeros(4, 9), "expected x"),
        (zeros(2, 3, 8), w, "expected x"), (zeros(2, 8, dtype=torch.float64), w, "dtype"),
        (x, zeros(4, 8, dtype=torch.float16), "dtype"), (x, zeros(4, 8, device="meta"), "device"),
        (zeros(2, 0), zeros(4, 0), "in_features"), (x, zeros(4, 16)[:, ::2], "contiguous"),
        (x, w.to_sparse(), "dense"),
    ]:
        with pytest.raises(ValueError, match=words):
            call(bad_x, bad_w)
    for bad in (None, 3, [[1.0]]):
        with pytest.raises(TypeError, match="must be a tensor"):
            call(bad, w)
        with pytest.raises(TypeError, match="must be a tensor"):
            call(x, bad)


def test_epilogue_arguments():
    x, w = zeros(2, 8), zeros(4, 8)
    for kwargs, words in [
        (dict(bias=zeros(5)), "bias"), (dict(bias=zeros(4, dtype=torch.float32)), "bias"),
        (dict(bias=zeros(4, device="meta")), "bias"), (dict(bias=zeros(1, 4)), "bias"),
        (dict(residual=zeros(2, 5)), "residual"),
        (dict(residual=zeros(2, 4, dtype=torch.float16)), "residual"),
        (dict(residual=zeros(2, 4, device="meta")), "residual"),
        (dict(activation="tanh"), "activation"),
        (dict(out=zeros(3, 4)), "out"), (dict(out=zeros(2, 4, dtype=torch.float32)), "out"),
        (dict(out=zeros(2, 8)[:, ::2]), "out"), (dict(out=zeros(1, 4).expand(2, 4)), "out"),
    ]:
        with pytest.raises(ValueError, match=words):
            rb.linear(x, w, **kwargs)
    with pytest.raises(TypeError, match="must be a tensor"):
        rb.linear(x, w, residual=1.0)
    with pytest.raises(ValueError, match="gate rows"):
        rb.gated_linear(x, zeros(5, 8))
    with pytest.raises(ValueError, match="activation"):
        rb.gated_linear(x, w, activation="swish")
    with pytest.raises(ValueError, match="out"):
        rb.gated_linear(x, w, out=zeros(2, 4))


def test_head_arguments():
    h, w = zeros(2, 8), zeros(4, 8)
    for tokens in (zeros(2, dtype=torch.int32), zeros(3, dtype=torch.int64),
                   zeros(2, 1, dtype=torch.int64), zeros(2, dtype=torch.int64, device="meta"),
                   None):
        with pytest.raises(ValueError, match="tokens|device"):
            rb.token_logprobs(h, w, tokens)
    with pytest.raises(ValueError, match="vocabulary"):
        rb.greedy_tokens(h, zeros(0, 8))


def test_weights_of_one_feature_have_any_stride():
    """A dimension of size one has no stride to speak of: these are refused
    for their device alone."""
    for w in (zeros(4, 16)[:, ::16], zeros(1, 16)[:, ::2]):
        with pytest.raises(ValueError, match="requires a CUDA device"):
            rb.linear(zeros(2, w.shape[1]), w)


def test_a_missing_extension_raises(monkeypatch, tmp_path):
    monkeypatch.setattr(_lib, "_native", None)
    monkeypatch.setattr(_lib, "BINDING_PATH", tmp_path / "_rlt_torch.so")
    with pytest.raises(RuntimeError, match="no fallback"):
        rb.linear(zeros(2, 8), zeros(4, 8))


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
        assert call(xs=9) == -4  # operands that TMA cannot address need scratch
    for call in (linear, gated):
        assert call(act=6) == -5 and call(act=-1) == -5
        assert call(outer=0) == 0
    assert head(outer=0) == -5
    assert head() == -4  # no workspace


def test_workspace_sizes():
    """Copies in rows of whole 16-byte units, only where TMA asks for them."""
    lib = _lib.load()

    def size(x=16, w=16, dtype=2, rows=3, inner=8, outer=4, gated=0, xs=8, ns=8, ks=1):
        return lib.rlt_linear_workspace_bytes(x, w, dtype, rows, inner, outer, gated, xs, ns, ks)

    assert size() == 0
    assert size(x=18) == 3 * 8 * 2
    assert size(xs=9) == 3 * 8 * 2
    assert size(xs=0) == 3 * 8 * 2  # a broadcast row
    assert size(rows=1, xs=9) == 0
    assert size(inner=9, xs=9, ns=16) == 3 * 16 * 2
    assert size(w=8) == 4 * 8 * 2
    assert size(ns=12) == 4 * 8 * 2
    assert size(ns=1, ks=4) == 8 * 8 * 2
    assert size(ns=1, ks=8) == 0
    assert size(ns=12, gated=1) == 2 * 4 * 8 * 2
    assert size(ns=1, ks=8, gated=1) == 2 * 8 * 8 * 2  # up columns start off a 16-byte boundary
    assert size(dtype=0, xs=10) == 3 * 8 * 4
    assert size(dtype=0, xs=12) == 0
