"""Projections with what follows them on sm_100a: the matrix product with
bias, activation and residual, the gated product of a feed-forward block, and
the language-model head reduced to tokens and log-probabilities.

They stand in for the reference's torch products and the separate steps after
them (vllm_rlt/models/ouro.py:96-123, the exit gate :209-217, the greedy choice
vllm_rlt/worker/model_runner.py:602-618). Each computes in fp32 and rounds once
to the tensors' dtype, where the torch expressions round at every step.

Activations are ``[rows, features]``; weights ``[out, in]`` with either
dimension contiguous, so a ``torch.nn.Linear`` weight and the decoder's
transposed views (``OuroWeights``) both serve as they are. Calls launch on the
current stream of the tensors' device, allocate only through torch and never
synchronise, so they can be captured in a CUDA graph. A wait inside a kernel that
gives up leaves its output void and is reported by
``vllm_rlt_b200.check_errors()``. There is no backward pass: outputs carry no
gradient.
"""

from __future__ import annotations

from .. import _lib

ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2, "gelu_tanh": 3, "relu": 4, "sigmoid": 5}


_UNKNOWN = f"activation must be one of {list(ACTIVATIONS)}"


def linear(x, weight, bias=None, *, activation=None, residual=None, out=None):
    """``act(x @ weight.t() + bias) + residual`` in one kernel.

    x ``[rows, in]``, weight ``[out, in]``, bias ``[out]``, residual and the
    result ``[rows, out]``. ``activation``: None, "silu", "gelu" (erf),
    "gelu_tanh", "relu" or "sigmoid". ``out`` may be ``residual`` itself and
    must not overlap any other argument."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"linear: {_UNKNOWN}")
    return _lib.native().linear(x, weight, bias, ACTIVATIONS[activation], residual, out)


def gated_linear(x, weight, *, activation="silu", out=None):
    """``act(x @ gate.t()) * (x @ up.t())`` in one kernel, ``weight`` being
    ``[gate; up]``, ``[2 * features, in]``. Returns ``[rows, features]``."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"gated linear: {_UNKNOWN}")
    return _lib.native().gated_linear(x, weight, ACTIVATIONS[activation], out)


def greedy_tokens(hidden, weight):
    """Each row's likeliest token and its log-probability, without storing
    ``logits = hidden @ weight.t()`` (kept in fp32, reduced tile by tile).

    hidden ``[rows, in]``, weight ``[vocab, in]``. Returns int64 ``[rows]`` (the
    lowest token on a tie, as ``torch.argmax``) and fp32 ``[rows]``."""
    return _lib.native().vocab_head(hidden, weight, None)


def token_logprobs(hidden, weight, tokens):
    """``log_softmax(hidden @ weight.t())`` at ``tokens``, int64 ``[rows]``,
    without storing the logits; 0 where a token is negative (nothing to score).
    A token beyond the vocabulary gives NaN and is reported by
    ``vllm_rlt_b200.check_errors()``. Returns fp32 ``[rows]``."""
    if tokens is None:
        raise ValueError("token logprobs: tokens must be int64 [rows]")
    return _lib.native().vocab_head(hidden, weight, tokens)
