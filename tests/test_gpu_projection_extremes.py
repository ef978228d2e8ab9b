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


# ------------------------------------------------------- fp32 as three bf16 parts


def test_single_precision_products():
    """Products of two numbers. The parts of a number leave out at most 2^-24
    (1 + 2^-10) of a product; the sum of the large and the small ones is rounded
    once (2^-24), and the five small products, 2^-7 of it together, truncate when
    they meet (a step of each other at most, 5 x 2^-23 x 2^-7)."""
    g = generator(82)
    bits = torch.cat([torch.tensor([0x3f80ffff, 0x3f808000, 0x3f818000, 0x3fffffff, 0x3f800001]),
                      torch.randint(0x3f800000, 0x40000000, (251,), generator=torch.Generator().manual_seed(82))])
    x = bits.int().view(torch.float32).cuda()[:, None]
    w = torch.cat([x, normal(g, 256, 1), -x])
    got, want = rb.linear(x, w).double(), x.double() @ w.double().t()
    bound = (2 + 2.0 ** -9 + 5 * 2.0 ** -6) * 2.0 ** -24
    assert (((got - want) / want).abs() <= bound).all()


@pytest.mark.parametrize("rows", [40, 300])
def test_single_precision_sums_are_not_biased(rows):
    """Sums of 64 products in [1, 4): the large ones add up exactly (16 bits above
    2^-14, less than 2^8 together), so an output's error is that of the parts left
    out and of one rounding, each within 2^-24 and of both signs. Over the outputs
    of 40 x 64 or more independent numbers its mean stays below 5 x 2^-23 /
    sqrt(2560), which is below 2^-26; parts left out with one sign leave 4e-8."""
    g = generator(83)
    x, w = (torch.rand(n, 64, device="cuda", generator=g) + 1 for n in (rows, 400))
    got, want = rb.linear(x, w).double(), x.double() @ w.double().t()
    assert abs(((got - want) / want).mean().item()) < 2.0 ** -26


def test_single_precision_near_the_largest_number():
    """Numbers that round up to infinity as bf16, and products whose large parts
    overflow although the product does not, come out as fp32 multiply-adds give
    them; the head sees the same."""
    most = torch.finfo(torch.float32).max
    for a, b in ((most, 1.0), (most, 0.5), (-3.4e38, 0.9999), (1.8446e19, 1.8446e19),
                 (1.8446e19, -1.8446e19), (3.3961e38, 1.0), (2.0 ** 127 * 1.999, 1.0)):
        for rows in (3, 200):
            x = torch.full((rows, 1), a, device="cuda")
            w = torch.full((70, 1), b, device="cuda")
            want = x.double() @ w.double().t()
            got = rb.linear(x, w).double()
            assert torch.equal(got.isinf(), want.abs() > most) and not got.isnan().any()
            fine = got.isfinite()
            assert ((got - want)[fine].abs() <= 2.0 ** -22 * want[fine].abs()).all()


# ----------------------------------------------------------------- activations


@pytest.mark.parametrize("op", ["linear", "gated"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_gelu_of_negative_numbers(op, dtype):
    """Relative to the result: x / sqrt 2 is rounded twice (2^-24 and 2^-25 of it),
    which moves erfc by up to 2 u^2 = x^2 times as much, at most 36 x 1.5 x 2^-24 on
    [-6, 0]; erfc itself is good to 4 steps of 2^-23, the products and the output
    to half a step each. fp16 adds half of its smallest subnormal, 2^-25."""
    x = torch.linspace(-6, 0, 16384, device="cuda").to(dtype).reshape(256, 64)
    for rows in (40, 256):
        z = x[:rows]
        w = torch.eye(64, device="cuda", dtype=dtype)
        if op == "linear":
            got = rb.linear(z, w, activation="gelu")
        else:  # up rows that give each row's last number: 1
            z = torch.cat([z, torch.ones_like(z[:, :8])], 1)
            w = torch.cat([torch.eye(72, device="cuda", dtype=dtype)[:64],
                           torch.eye(72, device="cuda", dtype=dtype)[64:65].expand(64, 72)])
            got = rb.gated_linear(z, w, activation="gelu")
        z = z[:, :64].double()
        want = 0.5 * z * torch.special.erfc(-z * 0.5 ** 0.5)
        bound = (54 + 8 + 3) * 2.0 ** -24 + torch.finfo(dtype).eps / 2
        small = 2.0 ** -25 if dtype == torch.float16 else 0.0
        assert ((got.double() - want).abs() <= bound * want.abs() * (1 + bound) + small).all()


# ------------------------------------------------------------- vocabulary head


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [4, 70, 300])
def test_logits_near_the_largest_number(rows, dtype):
    """Logits of 3e38 and 1e38 beside zeros, and a row of -3e38: finite, far apart,
    and times log2 e not a number. The likeliest entry has all of the probability
    (shared where it is reached twice)."""
    h = torch.zeros(rows, 64, device="cuda", dtype=dtype)
    w = torch.zeros(900, 64, device="cuda", dtype=dtype)
    h[:, 0] = 1e38
    h[1, 0] = -1e38
    w[:, 0], w[77, 0], w[500, 0], w[333, 0] = 1, 3, 3, 0
    logits = h.double() @ w.double().t()
    want = torch.log_softmax(logits, -1)
    tokens, logprobs = rb.greedy_tokens(h, w)
    assert torch.equal(tokens, logits.argmax(-1))
    best = want.gather(1, tokens[:, None])[:, 0]
    assert ((logprobs.double() - best).abs() <= 2.0 ** -20).all()  # of an exponential's error
    scored = rb.token_logprobs(h, w, torch.full_like(tokens, 500)).double()
    assert (scored[0] - best[0]).abs() <= 2.0 ** -20
    assert (scored[1] / want[1, 500] - 1).abs() <= 2.0 ** -20


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", [1e4, 1e8, 1e9, 1e10, 1e20, 1e30])
def test_large_logits(size, dtype):
    """Entries at size, at the next smaller number of the type and at half of it:
    from 2^28 on, where log2 e times a logit is only known to 16, the head takes
    differences of logits first."""
    h = torch.zeros(70, 64, device="cuda", dtype=dtype)
    w = torch.zeros(900, 64, device="cuda", dtype=dtype)
    h[:, 0] = 1
    w[:, 0] = size / 2
    w[200:, 0] = size
    w[300, 0] = torch.nextafter(w[300, 0].cpu(), torch.zeros((), dtype=dtype)).item()
    logits = h.double() @ w.double().t()
    want = torch.log_softmax(logits, -1)
    tokens, logprobs = rb.greedy_tokens(h, w)
    assert tokens.eq(200).all()
    # an exponential (2^-20), the roundings of a sum of 900 and of a logarithm below 7
    assert ((logprobs.double() - want[:, 200]).abs() <= 2.0 ** -20 + 250 * 2.0 ** -24).all()
    for token in (0, 300, 899):
        got = rb.token_logprobs(h, w, torch.full_like(tokens, token)).double()
        bound = 2.0 ** -20 + 250 * 2.0 ** -24 + 2.0 ** -23 * want[:, token].abs()
        assert ((got - want[:, token]).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(5, 1), (70, 1), (70, 300), (200, 5000)])
def test_probabilities_are_at_most_one(rows, vocab, dtype):
    """Rows that are all but certain: their log-probability rounds to 0, never above."""
    g = generator(84)
    w = normal(g, vocab, 64, dtype=dtype)
    h = normal(g, rows, 64) + 60 * w[torch.randint(vocab, (rows,), device="cuda", generator=g)].float()
    h = h.to(dtype)
    tokens, logprobs = rb.greedy_tokens(h, w)
    assert (logprobs <= 0).all() and (rb.token_logprobs(h, w, tokens) <= 0).all()
    assert torch.equal(rb.token_logprobs(h, w, tokens), logprobs)
    if vocab == 1:
        assert logprobs.eq(0).all()
