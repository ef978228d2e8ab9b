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
synchronise, so they can be captured in a CUDA graph. There is no backward
pass: outputs carry no gradient.
"""

from __future__ import annotations

import torch

from .. import _lib

ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2, "gelu_tanh": 3, "relu": 4, "sigmoid": 5}


def _operands(x, weight, what):
    """Check x [rows, in] and weight [out, in]; returns x with contiguous rows."""
    if x.ndim != 2 or weight.ndim != 2 or x.shape[1] != weight.shape[1]:
        raise ValueError(f"{what}: expected x [rows, in] and weight [out, in]")
    if x.device.type != "cuda":
        raise ValueError(f"{what} requires a CUDA device")
    if x.dtype not in _lib.DTYPE_CODES or weight.dtype != x.dtype:
        raise ValueError(f"{what}: x and weight must share a float32, float16 or bfloat16 dtype")
    if weight.device != x.device:
        raise ValueError(f"{what}: all tensors must live on the same device")
    if x.shape[1] == 0:
        raise ValueError(f"{what}: in_features must be positive")
    return x if x.stride(1) == 1 else x.contiguous()


def _weight_strides(weight, what):
    """(between output features, between input features), one of them 1."""
    ns, ks = weight.stride()
    if ks == 1 or weight.shape[1] == 1:
        return ns, 1
    if ns == 1 or weight.shape[0] == 1:
        return 1, ks
    raise ValueError(f"{what}: one dimension of weight must be contiguous")


def _rows_like(t, x, outer, name, what):
    if t.shape != (x.shape[0], outer) or t.dtype != x.dtype or t.device != x.device:
        raise ValueError(f"{what}: {name} must be [rows, out] of x's dtype and device")


def _output(out, x, outer, what):
    if out is None:
        return torch.empty((x.shape[0], outer), device=x.device, dtype=x.dtype)
    _rows_like(out, x, outer, "out", what)
    if outer > 1 and out.stride(1) != 1 or x.shape[0] > 1 and out.stride(0) < outer:
        raise ValueError(f"{what}: rows of out must be contiguous and apart")
    return out


def _activation(name, what):
    try:
        return ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError(f"{what}: activation must be one of {list(ACTIVATIONS)}") from None


def _scratch(need, device):
    return torch.empty(need, dtype=torch.uint8, device=device) if need else None


def linear(x, weight, bias=None, *, activation=None, residual=None, out=None):
    """``act(x @ weight.t() + bias) + residual`` in one kernel.

    x ``[rows, in]``, weight ``[out, in]``, bias ``[out]``, residual and the
    result ``[rows, out]``. ``activation``: None, "silu", "gelu" (erf),
    "gelu_tanh", "relu" or "sigmoid". ``out`` may be ``residual`` itself and
    must not overlap any other argument."""
    what = "linear"
    x = _operands(x, weight, what)
    rows, inner = x.shape
    outer = weight.shape[0]
    act = _activation(activation, what)
    ns, ks = _weight_strides(weight, what)
    if bias is not None:
        if bias.shape != (outer,) or bias.dtype != x.dtype or bias.device != x.device:
            raise ValueError(f"{what}: bias must be [out] of x's dtype and device")
        bias = bias.contiguous()
    if residual is not None:
        _rows_like(residual, x, outer, "residual", what)
        if residual.stride(1) != 1:
            residual = residual.contiguous()
    result = _output(out, x, outer, what)
    if rows == 0 or outer == 0:
        return result
    lib, device, code = _lib.load(), x.device, _lib.DTYPE_CODES[x.dtype]
    with torch.cuda.device(device):
        xp, wp, xs = x.data_ptr(), weight.data_ptr(), x.stride(0)
        need = lib.rlt_linear_workspace_bytes(xp, wp, code, rows, inner, outer, 0, xs, ns, ks)
        scratch = _scratch(need, device)
        rc = lib.rlt_linear(
            xp, wp, _lib.ptr(bias), _lib.ptr(residual), result.data_ptr(), _lib.ptr(scratch), need,
            _lib.status_word(device).data_ptr(), code, rows, inner, outer, act, xs, ns, ks,
            0 if residual is None else residual.stride(0), result.stride(0),
            _lib.stream_of(device))
    _lib.check(rc, what)
    return result


def gated_linear(x, weight, *, activation="silu", out=None):
    """``act(x @ gate.t()) * (x @ up.t())`` in one kernel, ``weight`` being
    ``[gate; up]``, ``[2 * features, in]``. Returns ``[rows, features]``."""
    what = "gated linear"
    x = _operands(x, weight, what)
    if weight.shape[0] % 2:
        raise ValueError(f"{what}: weight must hold as many gate rows as up rows")
    rows, inner = x.shape
    outer = weight.shape[0] // 2
    act = _activation(activation, what)
    ns, ks = _weight_strides(weight, what)
    result = _output(out, x, outer, what)
    if rows == 0 or outer == 0:
        return result
    lib, device, code = _lib.load(), x.device, _lib.DTYPE_CODES[x.dtype]
    with torch.cuda.device(device):
        xp, wp, xs = x.data_ptr(), weight.data_ptr(), x.stride(0)
        need = lib.rlt_linear_workspace_bytes(xp, wp, code, rows, inner, outer, 1, xs, ns, ks)
        scratch = _scratch(need, device)
        rc = lib.rlt_gated_linear(
            xp, wp, result.data_ptr(), _lib.ptr(scratch), need,
            _lib.status_word(device).data_ptr(), code, rows, inner, outer, act, xs, ns, ks,
            result.stride(0), _lib.stream_of(device))
    _lib.check(rc, what)
    return result


def _vocab_head(hidden, weight, tokens, what):
    hidden = _operands(hidden, weight, what)
    rows, inner = hidden.shape
    vocab = weight.shape[0]
    if vocab == 0:
        raise ValueError(f"{what}: the vocabulary must not be empty")
    ns, ks = _weight_strides(weight, what)
    device = hidden.device
    chosen = None
    if tokens is None:
        chosen = torch.empty(rows, dtype=torch.int64, device=device)
    logprobs = torch.empty(rows, dtype=torch.float32, device=device)
    if rows == 0:
        return chosen, logprobs
    lib, code = _lib.load(), _lib.DTYPE_CODES[hidden.dtype]
    with torch.cuda.device(device):
        hp, wp, hs = hidden.data_ptr(), weight.data_ptr(), hidden.stride(0)
        need = lib.rlt_vocab_head_workspace_bytes(hp, wp, code, rows, inner, vocab, hs, ns, ks)
        scratch = _scratch(need, device)
        rc = lib.rlt_vocab_head(
            hp, wp, _lib.ptr(tokens), _lib.ptr(chosen), logprobs.data_ptr(), _lib.ptr(scratch),
            need, _lib.status_word(device).data_ptr(), code, rows, inner, vocab, hs, ns, ks,
            _lib.stream_of(device))
    _lib.check(rc, what)
    return chosen, logprobs


def greedy_tokens(hidden, weight):
    """Each row's likeliest token and its log-probability, without storing
    ``logits = hidden @ weight.t()`` (kept in fp32, reduced tile by tile).

    hidden ``[rows, in]``, weight ``[vocab, in]``. Returns int64 ``[rows]`` (the
    lowest token on a tie, as ``torch.argmax``) and fp32 ``[rows]``."""
    return _vocab_head(hidden, weight, None, "greedy tokens")


def token_logprobs(hidden, weight, tokens):
    """``log_softmax(hidden @ weight.t())`` at ``tokens``, int64 ``[rows]``,
    without storing the logits; 0 where a token is negative (nothing to score).
    A token beyond the vocabulary gives NaN and is reported by the backend's
    ``check_errors()``. Returns fp32 ``[rows]``."""
    what = "token logprobs"
    if tokens.ndim != 1 or tokens.dtype != torch.int64 or tokens.shape[0] != hidden.shape[0]:
        raise ValueError(f"{what}: tokens must be int64 [rows]")
    if tokens.device != hidden.device:
        raise ValueError(f"{what}: all tensors must live on the same device")
    return _vocab_head(hidden, weight, tokens.contiguous(), what)[1]
