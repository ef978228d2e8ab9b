"""64-bit forms of the projection operators, with bounds on an fp32 kernel's
error against them.

Sums. A dot product of K terms, S = sum |x_k w_k|, is accumulated in fp32 in
some order. Every rounding is at most 2^-24 of a partial sum (<= S). With
roundings to nearest the errors are unbiased, and by Hoeffding's inequality the
total exceeds 7 sqrt(K) 2^-24 S with probability below 1e-10. A tensor core
may instead truncate (one-sided, at most 2^-23 of the partial sum) once for
each 16 input features: K / 16 such steps add at most (K / 8) 2^-24 S.

Activations. Each has a slope of at most 1.13. Its own fp32 evaluation: the
exponential's argument is rounded (relative error of the result |argument|
2^-23, the argument of gelu_tanh being 1.6 (z + 0.045 z^3)), the hardware
exponential and reciprocal are good to 2^-22, gelu's 1 + erf to 2^-22 absolute.

Rounding to the output's type is half a step, eps / 2 of the value (and half
of fp16's smallest subnormal, 2^-25)."""

from __future__ import annotations

import torch

F = torch.nn.functional
ACTIVATE = {None: lambda t: t, "silu": F.silu, "gelu": F.gelu,
            "gelu_tanh": lambda t: F.gelu(t, approximate="tanh"), "relu": F.relu,
            "sigmoid": torch.sigmoid}


def product(x, w, bias=None):
    """(x w^T + bias, bound on its fp32 error), both fp64."""
    x, w = x.double(), w.double()
    k = x.shape[1]
    y, s = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        y = y + bias.double()
        s = s + bias.double().abs()
    return y, (7 * k ** 0.5 + k / 8 + 1) * 2.0 ** -24 * s


def activated(z, e, name):
    """(act(z), bound) for z known to within e."""
    if name is None:
        return z, e
    a = z.abs()
    own = torch.zeros_like(z) if name == "relu" else 2.0 ** -22 * (a + 1) * (8 + 2 * a + 0.1 * a ** 3)
    return ACTIVATE[name](z), 1.13 * e + own.clamp(max=1e30)


def rounded(y, e, dtype):
    """Bound after rounding to dtype."""
    half = torch.finfo(dtype).eps / 2
    return e + half * (y.abs() + e) + (2.0 ** -25 if dtype == torch.float16 else 0.0)


def linear(x, w, bias=None, activation=None, residual=None):
    z, e = product(x, w, bias)
    y, e = activated(z, e, activation)
    if residual is not None:
        y = y + residual.double()
        e = e + 2.0 ** -24 * (y.abs() + residual.double().abs())
    return y, rounded(y, e, x.dtype)


def gated(x, w, activation="silu"):
    half = w.shape[0] // 2
    g, eg = product(x, w[:half])
    u, eu = product(x, w[half:])
    a, ea = activated(g, eg, activation)
    e = ea * u.abs() + eu * (a.abs() + ea) + 2.0 ** -23 * (a * u).abs()
    return a * u, rounded(a * u, e, x.dtype)


def vocab(h, w):
    """(logits, bound on a logit's error, log-probabilities, bound on theirs).

    A log-probability moves by at most the errors of its own logit and of the
    largest; the sum of V exponentials carries their relative errors (2^-20)
    and its own roundings (7 sqrt(V) 2^-24); its logarithm and the differences
    round relative to their size."""
    z, e = product(h, w)
    worst = e.amax(-1, keepdim=True)
    lp = torch.log_softmax(z, -1)
    v = w.shape[0]
    own = 2.0 ** -20 + 7 * v ** 0.5 * 2.0 ** -24
    return z, worst, lp, 2 * worst + own + 2.0 ** -22 * (lp.abs() + z.abs().amax(-1, keepdim=True))
