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
    """Check x [rows, in] and weight [out, in]; returns x with contiguous rows,
    rows, in, out, x's row stride, the weight's strides (one of them 1), the
    dtype's code and the device."""
    shape, wshape = x.shape, weight.shape
    if len(shape) != 2 or len(wshape) != 2 or shape[1] != wshape[1]:
        raise ValueError(f"{what}: expected x [rows, in] and weight [out, in]")
    device, dtype = x.device, x.dtype
    if device.type != "cuda":
        raise ValueError(f"{what} requires a CUDA device")
    code = _lib.DTYPE_CODES.get(dtype)
    if code is None or weight.dtype != dtype:
        raise ValueError(f"{what}: x and weight must share a float32, float16 or bfloat16 dtype")
    if weight.device != device:
        raise ValueError(f"{what}: all tensors must live on the same device")
    rows, inner = shape
    if inner == 0:
        raise ValueError(f"{what}: in_features must be positive")
    ns, ks = weight.stride()
    if ks == 1 or inner == 1:
        ks = 1
    elif ns == 1 or wshape[0] == 1:
        ns = 1
    else:
        raise ValueError(f"{what}: one dimension of weight must be contiguous")
    xs, unit = x.stride()
    if unit != 1:
        x, xs = x.contiguous(), inner
    return x, rows, inner, wshape[0], xs, ns, ks, code, device


def _rows_like(t, rows, outer, x, name, what):
    if t.shape != (rows, outer) or t.dtype != x.dtype or t.device != x.device:
        raise ValueError(f"{what}: {name} must be [rows, out] of x's dtype and device")


def _output(out, x, rows, outer, what):
    """The result tensor and its row stride."""
    if out is None:
        return torch.empty_strided((rows, outer), (outer, 1), dtype=x.dtype,
                                   device=x.device), outer
    _rows_like(out, rows, outer, x, "out", what)
    stride, unit = out.stride()
    if outer > 1 and unit != 1 or rows > 1 and stride < outer:
        raise ValueError(f"{what}: rows of out must be contiguous and apart")
    return out, stride


def _activation(name, what):
    try:
        return ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError(f"{what}: activation must be one of {list(ACTIVATIONS)}") from None


def _run(device, what, entry, head, tail, need, operands):
    """``entry(*head, workspace, bytes, status, *tail, stream)`` on ``device``.
    Scratch is asked for, and allocated, only by calls that are refused without:
    the vocabulary head, and operands that have to be copied into aligned rows."""
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _run(device, what, entry, head, tail, need, operands)
    status, stream = _lib.status_ptr(device), _lib.stream_of(device)
    rc = entry(*head, None, 0, status, *tail, stream)
    if rc == _lib.E_WORKSPACE:
        size = need(*operands)
        scratch = torch.empty(size, dtype=torch.uint8, device=device)
        rc = entry(*head, scratch.data_ptr(), size, status, *tail, stream)
    if rc:
        _lib.check(rc, what)


def linear(x, weight, bias=None, *, activation=None, residual=None, out=None):
    """``act(x @ weight.t() + bias) + residual`` in one kernel.

    x ``[rows, in]``, weight ``[out, in]``, bias ``[out]``, residual and the
    result ``[rows, out]``. ``activation``: None, "silu", "gelu" (erf),
    "gelu_tanh", "relu" or "sigmoid". ``out`` may be ``residual`` itself and
    must not overlap any other argument."""
    what = "linear"
    x, rows, inner, outer, xs, ns, ks, code, device = _operands(x, weight, what)
    act = _activation(activation, what)
    bias_ptr = residual_ptr = None
    rs = 0
    if bias is not None:
        if bias.shape != (outer,) or bias.dtype != x.dtype or bias.device != device:
            raise ValueError(f"{what}: bias must be [out] of x's dtype and device")
        if bias.stride(0) != 1:
            bias = bias.contiguous()
        bias_ptr = bias.data_ptr()
    if residual is not None:
        _rows_like(residual, rows, outer, x, "residual", what)
        rs, unit = residual.stride()
        if unit != 1:
            residual, rs = residual.contiguous(), outer
        residual_ptr = residual.data_ptr()
    result, os = _output(out, x, rows, outer, what)
    if rows == 0 or outer == 0:
        return result
    lib, xp, wp = _lib.load(), x.data_ptr(), weight.data_ptr()
    _run(device, what, lib.rlt_linear, (xp, wp, bias_ptr, residual_ptr, result.data_ptr()),
         (code, rows, inner, outer, act, xs, ns, ks, rs, os),
         lib.rlt_linear_workspace_bytes, (xp, wp, code, rows, inner, outer, 0, xs, ns, ks))
    return result


def gated_linear(x, weight, *, activation="silu", out=None):
    """``act(x @ gate.t()) * (x @ up.t())`` in one kernel, ``weight`` being
    ``[gate; up]``, ``[2 * features, in]``. Returns ``[rows, features]``."""
    what = "gated linear"
    x, rows, inner, outer, xs, ns, ks, code, device = _operands(x, weight, what)
    if outer % 2:
        raise ValueError(f"{what}: weight must hold as many gate rows as up rows")
    outer //= 2
    act = _activation(activation, what)
    result, os = _output(out, x, rows, outer, what)
    if rows == 0 or outer == 0:
        return result
    lib, xp, wp = _lib.load(), x.data_ptr(), weight.data_ptr()
    _run(device, what, lib.rlt_gated_linear, (xp, wp, result.data_ptr()),
         (code, rows, inner, outer, act, xs, ns, ks, os),
         lib.rlt_linear_workspace_bytes, (xp, wp, code, rows, inner, outer, 1, xs, ns, ks))
    return result


def _vocab_head(hidden, weight, tokens, what):
    hidden, rows, inner, vocab, hs, ns, ks, code, device = _operands(hidden, weight, what)
    if vocab == 0:
        raise ValueError(f"{what}: the vocabulary must not be empty")
    chosen = chosen_ptr = tokens_ptr = None
    if tokens is None:
        chosen = torch.empty(rows, dtype=torch.int64, device=device)
        chosen_ptr = chosen.data_ptr()
    else:
        tokens_ptr = tokens.data_ptr()
    logprobs = torch.empty(rows, dtype=torch.float32, device=device)
    if rows == 0:
        return chosen, logprobs
    lib, hp, wp = _lib.load(), hidden.data_ptr(), weight.data_ptr()
    _run(device, what, lib.rlt_vocab_head, (hp, wp, tokens_ptr, chosen_ptr, logprobs.data_ptr()),
         (code, rows, inner, vocab, hs, ns, ks),
         lib.rlt_vocab_head_workspace_bytes, (hp, wp, code, rows, inner, vocab, hs, ns, ks))
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
