"""Projection operators against their 64-bit forms (tests/projection_oracle.py
derives every tolerance)."""

from __future__ import annotations

import pytest
import torch

import projection_oracle as po
import vllm_rlt_b200 as rb
from vllm_rlt_b200 import _lib

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
ACTS = [None, "silu", "gelu", "gelu_tanh", "relu", "sigmoid"]


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *size, std=1.0, dtype=torch.float32):
    return (torch.randn(size, device="cuda", generator=g) * std).to(dtype)


def make_weight(g, outer, inner, dtype, layout):
    if layout == "in_out":
        return normal(g, inner, outer, std=0.05, dtype=dtype).t()
    return normal(g, outer, inner, std=0.05, dtype=dtype)


def assert_within(got, want, bound):
    assert got.shape == want.shape
    off = (got.double() - want).abs() - bound
    worst = off.max().item() if off.numel() else -1.0
    assert worst <= 0, f"{int((off > 0).sum())} of {off.numel()} beyond the bound, by {worst}"


SIZES = [  # rows, in, out
    (1, 1, 1), (1, 64, 128), (2, 7, 3), (1, 2048, 64), (3, 40, 100), (16, 64, 64), (17, 72, 129),
    (33, 100, 136), (64, 520, 257), (65, 128, 1), (64, 2048, 1), (128, 256, 384), (129, 1000, 100),
    (200, 1001, 77), (300, 576, 1231), (513, 192, 640), (1030, 328, 520),
]


@pytest.mark.parametrize("layout", ["out_in", "in_out"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner,outer", SIZES)
def test_linear(rows, inner, outer, dtype, layout):
    g = generator(rows * 7 + inner)
    x = normal(g, rows, inner, dtype=dtype)
    w = make_weight(g, outer, inner, dtype, layout)
    assert_within(rb.linear(x, w), *po.linear(x, w))


@pytest.mark.parametrize("activation", ACTS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner,outer", [(5, 96, 70), (70, 264, 200), (400, 128, 392)])
def test_linear_epilogue(rows, inner, outer, dtype, activation):
    g = generator(3)
    x = normal(g, rows, inner, std=3.0, dtype=dtype)
    w = make_weight(g, outer, inner, dtype, "out_in")
    bias = normal(g, outer, dtype=dtype)
    residual = normal(g, rows, outer, dtype=dtype)
    for b, r in ((bias, None), (None, residual), (bias, residual)):
        got = rb.linear(x, w, b, activation=activation, residual=r)
        assert_within(got, *po.linear(x, w, b, activation, r))


@pytest.mark.parametrize("layout", ["out_in", "in_out"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner,outer", SIZES)
def test_gated_linear(rows, inner, outer, dtype, layout):
    g = generator(rows + inner * 5)
    x = normal(g, rows, inner, dtype=dtype)
    w = make_weight(g, 2 * outer, inner, dtype, layout)
    assert_within(rb.gated_linear(x, w), *po.gated(x, w))


@pytest.mark.parametrize("activation", ACTS)
@pytest.mark.parametrize("dtype", TYPES)
def test_gated_activations(dtype, activation):
    g = generator(11)
    for rows, inner, outer in ((7, 128, 72), (150, 200, 264)):
        x = normal(g, rows, inner, std=3.0, dtype=dtype)
        w = make_weight(g, 2 * outer, inner, dtype, "out_in")
        assert_within(rb.gated_linear(x, w, activation=activation), *po.gated(x, w, activation))


VOCAB = [(1, 64, 1), (1, 128, 97), (3, 33, 300), (16, 256, 1000), (64, 128, 2000), (65, 72, 777),
         (130, 512, 4096), (300, 100, 5001), (700, 64, 1537)]


def peaked(g, rows, inner, vocab, dtype, layout):
    w = make_weight(g, vocab, inner, dtype, layout)
    target = torch.randint(vocab, (rows,), device="cuda", generator=g)
    h = normal(g, rows, inner) + w[target].float() * torch.rand(
        rows, 1, device="cuda", generator=g) * 40
    return h.to(dtype), w, target


@pytest.mark.parametrize("layout", ["out_in", "in_out"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner,vocab", VOCAB)
def test_greedy_tokens(rows, inner, vocab, dtype, layout):
    h, w, _ = peaked(generator(rows + vocab), rows, inner, vocab, dtype, layout)
    tokens, logprobs = rb.greedy_tokens(h, w)
    z, e, lp, bound = po.vocab(h, w)
    assert tokens.dtype == torch.int64 and logprobs.dtype == torch.float32
    best = z.amax(-1)
    picked = z.gather(1, tokens[:, None])[:, 0]
    assert bool((picked >= best - 2 * e[:, 0]).all())
    top = z.topk(min(2, vocab), -1).values
    clear = top[:, 0] - top[:, -1] > 2 * e[:, 0] if vocab > 1 else torch.ones_like(best).bool()
    assert torch.equal(tokens[clear], z.argmax(-1)[clear])
    at = tokens[:, None]
    assert_within(logprobs, lp.gather(1, at)[:, 0], bound.gather(1, at)[:, 0])


@pytest.mark.parametrize("layout", ["out_in", "in_out"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner,vocab", VOCAB)
def test_token_logprobs(rows, inner, vocab, dtype, layout):
    g = generator(rows * 3 + vocab)
    h, w, target = peaked(g, rows, inner, vocab, dtype, layout)
    tokens = torch.randint(vocab, (rows,), device="cuda", generator=g)
    tokens[::3] = target[::3]
    tokens[rows // 2] = vocab - 1
    tokens[1::7] = -1
    got = rb.token_logprobs(h, w, tokens)
    _, _, lp, bound = po.vocab(h, w)
    at = tokens.clamp(min=0)[:, None]
    keep = tokens >= 0
    want = torch.where(keep, lp.gather(1, at)[:, 0], torch.zeros_like(lp[:, 0]))
    assert_within(got, want, torch.where(keep, bound.gather(1, at)[:, 0], torch.zeros_like(want)))
    assert _lib.read_status(h.device) == []


@pytest.mark.parametrize("dtype", TYPES)
def test_ties_go_to_the_lowest_token(dtype):
    """Equal vocabulary rows give equal logits; their copies lie in the same
    tile, in neighbouring ones and in the last."""
    g = generator(5)
    for rows, vocab in ((4, 1500), (200, 3001)):
        h = normal(g, rows, 64, dtype=dtype)
        w = normal(g, vocab, 64, std=0.02, dtype=dtype)
        best = (normal(g, 1, 64) * 0.02).to(dtype)
        best = best + h[:1] * 0.5
        h[:] = h[:1]
        for first in (0, 3, 70, 500):
            v = w.clone()
            for at in (first, first + 1, first + 40, first + 300, vocab - 1):
                v[at] = best[0]
            tokens, _ = rb.greedy_tokens(h, v)
            assert tokens.eq(first).all()


def test_a_token_beyond_the_vocabulary_is_reported():
    g = generator(9)
    h, w = normal(g, 4, 64, dtype=torch.bfloat16), normal(g, 100, 64, dtype=torch.bfloat16)
    tokens = torch.tensor([5, 100, -7, 2 ** 40], device="cuda")
    got = rb.token_logprobs(h, w, tokens)
    assert _lib.read_status(h.device) == [_lib.STATUS_BITS[128]]
    assert got.isnan().tolist() == [False, True, False, True] and got[2].item() == 0.0


# ------------------------------------------------------- layouts and strides


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [3, 64, 300])
@pytest.mark.parametrize("inner,outer", [(64, 128), (200, 96), (77, 51)])
def test_slices_of_wider_tensors(rows, inner, outer, dtype):
    """x, residual and out are column slices whose neighbours hold NaN; the
    neighbours of out stay as they were."""
    g = generator(21)

    def inside(r, c, left, right, fill=float("nan")):
        wide = torch.full((r + 2, left + c + right), fill, device="cuda", dtype=dtype)
        return wide, wide[1 : r + 1, left : left + c]

    for left, right in ((8, 8), (1, 2)):
        _, x = inside(rows, inner, left, right)
        x.copy_(normal(g, rows, inner))
        _, w = inside(outer, inner, left, right)
        w.copy_(normal(g, outer, inner, std=0.05))
        _, residual = inside(rows, outer, left, right)
        residual.copy_(normal(g, rows, outer))
        wide, out = inside(rows, outer, left, right, fill=7.0)
        got = rb.linear(x, w, residual=residual, out=out)
        assert got is out
        assert_within(out, *po.linear(x, w, residual=residual))
        out.fill_(7.0)
        assert bool((wide == 7.0).all())
        _, w_t = inside(inner, outer, left, right)
        w_t.copy_(w.t())
        assert_within(rb.linear(x, w_t.t()), *po.linear(x, w))
        _, w2 = inside(2 * outer, inner, left, right)
        w2.copy_(normal(g, 2 * outer, inner, std=0.05))
        rb.gated_linear(x, w2, out=out)
        assert_within(out, *po.gated(x, w2))
        out.fill_(7.0)
        assert bool((wide == 7.0).all())
        _, w2_t = inside(inner, 2 * outer, left, right)
        w2_t.copy_(w2.t())
        assert_within(rb.gated_linear(x, w2_t.t()), *po.gated(x, w2))


@pytest.mark.parametrize("dtype", TYPES)
def test_broadcast_and_transposed_inputs(dtype):
    g = generator(22)
    one = normal(g, 1, 128, dtype=dtype)
    w = normal(g, 72, 128, std=0.05, dtype=dtype)
    res = normal(g, 1, 72, dtype=dtype)
    x = one.expand(40, 128)
    assert_within(rb.linear(x, w, residual=res.expand(40, 72)),
                  *po.linear(x, w, residual=res.expand(40, 72)))
    shared = normal(g, 1, 128, std=0.05, dtype=dtype).expand(72, 128)  # every output alike
    assert_within(rb.linear(x, shared), *po.linear(x, shared))
    xt = normal(g, 128, 40, dtype=dtype).t()
    assert_within(rb.linear(xt, w), *po.linear(xt, w))
    rt = normal(g, 72, 40, dtype=dtype).t()
    assert_within(rb.linear(xt, w, residual=rt), *po.linear(xt, w, residual=rt))
    wide_bias = normal(g, 72, 2, dtype=dtype)[:, 0]
    assert_within(rb.linear(xt, w, wide_bias), *po.linear(xt, w, wide_bias))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [5, 200])
def test_residual_in_place(rows, dtype):
    g = generator(23)
    x, w = normal(g, rows, 320, dtype=dtype), normal(g, 136, 320, std=0.05, dtype=dtype)
    hidden = normal(g, rows, 136, dtype=dtype)
    want, bound = po.linear(x, w, residual=hidden)
    assert rb.linear(x, w, residual=hidden, out=hidden) is hidden
    assert_within(hidden, want, bound)


@pytest.mark.parametrize("dtype", TYPES)
def test_empty_calls(dtype):
    x = torch.zeros(0, 64, device="cuda", dtype=dtype)
    w = torch.zeros(32, 64, device="cuda", dtype=dtype)
    assert rb.linear(x, w).shape == (0, 32)
    assert rb.gated_linear(x, w).shape == (0, 16)
    assert rb.linear(torch.zeros(3, 64, device="cuda", dtype=dtype), w[:0]).shape == (3, 0)
    tokens, logprobs = rb.greedy_tokens(x, w)
    assert tokens.shape == (0,) and logprobs.shape == (0,)
    assert rb.token_logprobs(x, w, tokens).shape == (0,)


# --------------------------------------------------- not-numbers, infinities


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [9, 150])
def test_not_numbers_stay_in_their_row_and_column(rows, dtype):
    g = generator(31)
    x, w = normal(g, rows, 200, dtype=dtype), normal(g, 260, 200, std=0.05, dtype=dtype)
    clean = rb.linear(x, w, activation="silu")
    x[4, 17] = float("nan")
    w[100, 3] = float("nan")
    got = rb.linear(x, w, activation="silu")
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[4], hit[:, 100] = True, True
    assert torch.equal(got.isnan(), hit)
    assert torch.equal(got[~hit], clean[~hit])
    got = rb.gated_linear(x, w)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[4], hit[:, 100] = True, True
    assert torch.equal(got.isnan(), hit)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", ACTS)
def test_infinite_sums(dtype, activation):
    """One infinite input feature makes whole rows of plus and minus infinity;
    the activations take their limits there, as torch's formulas do."""
    g = generator(32)
    x, w = normal(g, 6, 64, dtype=dtype), normal(g, 40, 64, std=0.05, dtype=dtype)
    x[2, 5] = float("inf")
    got = rb.linear(x, w, activation=activation).float()
    z = x.float() @ w.float().t()
    want = {None: lambda t: t, "silu": lambda t: t / (1 + torch.exp(-t)),
            "gelu": lambda t: 0.5 * t * (1 + torch.erf(t)),
            "gelu_tanh": lambda t: 0.5 * t * (1 + torch.tanh(t)), "relu": torch.relu,
            "sigmoid": torch.sigmoid}[activation](z[2])
    assert torch.equal(got[2].isnan(), want.isnan())
    assert torch.equal(got[2][~want.isnan()], want[~want.isnan()])


@pytest.mark.parametrize("dtype", TYPES)
def test_vocabulary_head_with_not_numbers_and_infinities(dtype):
    g = generator(33)
    h, w = normal(g, 40, 64, dtype=dtype), normal(g, 900, 64, std=0.05, dtype=dtype)
    h[3, 0] = float("nan")
    h[5, 1] = float("inf")
    tokens, logprobs = rb.greedy_tokens(h, w)
    z = h.float() @ w.float().t()
    assert logprobs.isnan().nonzero()[:, 0].tolist() == [3, 5]
    assert tokens[3].item() == 0
    assert torch.isinf(z[5, tokens[5]]) and z[5, tokens[5]] > 0
    assert tokens[5].item() == int(torch.argmax(z[5]))
    w[700, 2] = float("nan")  # one vocabulary entry: the largest of every row
    tokens, logprobs = rb.greedy_tokens(h, w)
    keep = torch.ones(40, dtype=torch.bool, device="cuda")
    keep[3] = False
    assert tokens[keep].eq(700).all() and logprobs.isnan().all()


# ------------------------------------------------------ streams, graphs, repeats


def calls(dtype, rows):
    g = generator(41)
    x = normal(g, rows, 320, dtype=dtype)
    w = normal(g, 192, 320, std=0.05, dtype=dtype)
    v = normal(g, 320, 3000, std=0.05, dtype=dtype).t()
    bias = normal(g, 192, dtype=dtype)
    tokens = torch.randint(3000, (rows,), device="cuda", generator=g)
    return x, lambda: (rb.linear(x, w, bias, activation="silu"), rb.gated_linear(x, w),
                       *rb.greedy_tokens(x, v), rb.token_logprobs(x, v, tokens))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 64, 260])
def test_repeats_bit_for_bit_and_in_graphs(rows, dtype):
    """Eager calls repeat; two graphs captured from the same calls and replayed
    in turn on new inputs give what eager calls give."""
    x, call = calls(dtype, rows)
    first = call()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(call(), first))
    graphs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs = call()
        graphs.append((graph, outputs))
    for seed in (1, 2):
        x.copy_(normal(generator(seed), *x.shape))
        want = call()
        for graph, outputs in graphs:
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(outputs, want))
        for graph, _ in graphs:  # back to back, nothing in between
            graph.replay()
        assert all(torch.equal(a, b) for _, o in graphs for a, b in zip(o, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_two_streams_at_once(dtype):
    x, call = calls(dtype, 70)
    want = call()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(call())
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_another_device():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    g = torch.Generator(device="cuda:1").manual_seed(0)
    x = torch.randn(30, 64, device="cuda:1", generator=g).bfloat16()
    w = torch.randn(40, 64, device="cuda:1", generator=g).bfloat16()
    assert torch.cuda.current_device() == 0
    assert_within(rb.linear(x, w), *po.linear(x, w))


# ------------------------------------------------------------- used together


@pytest.mark.parametrize("layout", ["out_in", "in_out"])
@pytest.mark.parametrize("rows", [1, 40, 300])
def test_feed_forward_block_and_head(rows, layout):
    """A block as a decoder runs it: gated product, down projection added to
    the residual stream in place, then the next token's choice and its score.
    Each step is checked against the 64-bit form of its own input."""
    g = generator(51)
    dtype = torch.bfloat16
    x = normal(g, rows, 256, dtype=dtype)
    wgu = make_weight(g, 2 * 384, 256, dtype, layout)
    wdown = make_weight(g, 256, 384, dtype, layout)
    head = make_weight(g, 2500, 256, dtype, layout)
    h = rb.gated_linear(x, wgu)
    assert_within(h, *po.gated(x, wgu))
    hidden = x.clone()
    want = po.linear(h, wdown, residual=hidden)
    rb.linear(h, wdown, residual=hidden, out=hidden)
    assert_within(hidden, *want)
    tokens, logprobs = rb.greedy_tokens(hidden, head)
    _, _, lp, bound = po.vocab(hidden, head)
    at = tokens[:, None]
    assert_within(logprobs, lp.gather(1, at)[:, 0], bound.gather(1, at)[:, 0])
    assert torch.equal(rb.token_logprobs(hidden, head, tokens), logprobs)


# ------------------------------------------------- together on one device, extremes


@pytest.mark.parametrize("rows", [3, 64])
def test_types_on_two_streams_at_once(rows):
    """fp32 and 16-bit calls split their sums over clusters of CTAs that wait for
    one another; both kinds run at once without holding each other up."""
    made = [calls(torch.bfloat16, rows)[1], calls(torch.float32, rows)[1]]
    want = [call() for call in made]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(40):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(made[i]())
    torch.cuda.synchronize()
    assert _lib.read_status(torch.device("cuda", 0)) == []
    for i in range(2):
        for result in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(result, want[i]))


FIRST_CALL_CAPTURED = """
import torch, vllm_rlt_b200 as rb
x = torch.randn(%d, 128, device="cuda").to(torch.%s)
w = torch.randn(256, 128, device="cuda").to(torch.%s)
torch.cuda.synchronize()
rb._lib.status_word(x.device)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y, h, t = rb.linear(x, w), rb.gated_linear(x, w), rb.greedy_tokens(x, w)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(y, rb.linear(x, w)) and torch.equal(h, rb.gated_linear(x, w))
assert all(torch.equal(a, b) for a, b in zip(t, rb.greedy_tokens(x, w)))
"""


@pytest.mark.parametrize("rows,dtype", [(5, "bfloat16"), (300, "bfloat16"), (5, "float32")])
def test_the_first_call_may_be_captured(rows, dtype):
    import subprocess
    import sys
    from pathlib import Path

    subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED % (rows, dtype, dtype)], check=True,
                   cwd=Path(__file__).resolve().parents[1], timeout=300)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inner,outer", [(40000, 3), (20011, 70)])
def test_long_sums(inner, outer, dtype):
    g = generator(61)
    for rows in (2, 90):
        x = normal(g, rows, inner, dtype=dtype)
        w = normal(g, outer, inner, std=0.05, dtype=dtype)
        assert_within(rb.linear(x, w), *po.linear(x, w))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_offsets_beyond_32_bits(dtype):
    """Rows of x, residual and out lie 2^31 and more elements apart."""
    g = generator(62)
    gap = 2 ** 30 + 16
    room = torch.zeros(3 * gap + 4096, device="cuda", dtype=dtype)
    rows = [room.as_strided((4, n), (gap, 1), at) for n, at in ((128, 0), (64, 1024), (64, 2048))]
    x, residual, out = rows
    x.copy_(normal(g, 4, 128))
    residual.copy_(normal(g, 4, 64))
    w = normal(g, 64, 128, std=0.05, dtype=dtype)
    rb.linear(x, w, residual=residual, out=out)
    assert_within(out, *po.linear(x, w, residual=residual))
    head = room.as_strided((4, 128), (gap, 1), 3200)  # weights far apart as well
    head.copy_(normal(g, 4, 128))
    assert_within(rb.linear(x, head), *po.linear(x, head))


def test_a_row_of_infinities_and_not_numbers_in_single_precision():
    """fp32 splits its operands; what the split cannot carry is recomputed."""
    g = generator(63)
    for rows in (4, 150):
        x, w = normal(g, rows, 96), normal(g, 130, 96, std=0.05)
        x[0, 3], x[1, 4], x[2] = float("inf"), -float("inf"), float("nan")
        x[3, 0], x[3, 1] = float("inf"), float("nan")
        w[7, 3], w[9, 4], w[11] = 0.0, 0.5, float("inf")
        got = rb.linear(x, w)
        want = (x.double()[:, None] * w.double()[None]).sum(-1)
        assert torch.equal(got.isnan(), want.isnan())
        inf = want.isinf()
        assert torch.equal(got[inf].double(), want[inf])
        fine = want.isfinite()
        assert fine.any() or rows == 4
        close = po.linear(torch.nan_to_num(x, 0, 0, 0), torch.nan_to_num(w, 0, 0, 0))
        off = (got.double() - close[0]).abs() - close[1]
        assert bool((off[fine] <= 0).all())


@pytest.mark.parametrize("rows", [4, 200])
def test_captured_behind_copies_and_other_streams(rows):
    """In a captured graph the kernels follow memory copies, memsets, kernels of
    other libraries and a joined side stream, and read what those wrote."""
    g = generator(71)
    source = normal(g, rows, 256, dtype=torch.bfloat16)
    x, y = torch.zeros_like(source), torch.zeros_like(source)
    w = normal(g, 256, 256, std=0.05, dtype=torch.bfloat16)
    v = torch.empty_like(w)
    side = torch.cuda.Stream()

    def work():
        x.copy_(source)  # a copy of device memory
        a = rb.linear(x, w)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y.copy_(source)
            b = rb.gated_linear(y, w)
        v.zero_()
        v.add_(w)  # weights written by the kernel just before
        c = rb.linear(x, v, residual=a)
        torch.cuda.current_stream().wait_stream(side)
        d = rb.linear(b, v[:, :128].contiguous())
        x.zero_()  # after their last reader
        y.zero_()
        return a, b, c, d, *rb.greedy_tokens(a, v)

    want = [t.clone() for t in work()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for _ in range(20):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    for _ in range(20):  # and eagerly, without a wait in between
        got = work()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
