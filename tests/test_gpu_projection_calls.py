"""Calls of the projection operators that their documentation allows beyond the
plain ones: rows far apart on many rows, tokens of any stride, subnormal numbers,
other kernels of the package on another stream, threads."""

from __future__ import annotations

import threading

import pytest
import torch

import projection_oracle as po
import vllm_rlt_b200 as rb
from test_gpu_projections import TYPES, assert_within, generator, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,outer", [(70, 64), (200, 96)])
def test_many_rows_far_apart(rows, outer, dtype):
    """Rows of x, residual, out and the weights reach past 2^32 elements."""
    g = generator(91)
    gap = 2 ** 32 // rows + 2 ** 16 // 16 * 16
    gap -= gap % 16
    room = torch.zeros((rows + 1) * gap, device="cuda", dtype=dtype)
    x, residual, out = (room.as_strided((rows, n), (gap, 1), at)
                        for n, at in ((128, 0), (outer, 1024), (outer, 2048)))
    w = room.as_strided((outer, 128), (gap, 1), 3200)
    assert (rows - 1) * gap + 3200 > 2 ** 32 - gap
    x.copy_(normal(g, rows, 128))
    residual.copy_(normal(g, rows, outer))
    w.copy_(normal(g, outer, 128, std=0.05))
    rb.linear(x, w, residual=residual, out=out)
    assert_within(out, *po.linear(x, w, residual=residual))
    rb.gated_linear(x, w, out=out[:, : outer // 2])
    assert_within(out[:, : outer // 2], *po.gated(x, w))
    tokens, logprobs = rb.greedy_tokens(x, w)
    want = rb.greedy_tokens(x.contiguous(), w.contiguous())
    assert torch.equal(tokens, want[0]) and torch.equal(logprobs, want[1])


@pytest.mark.parametrize("rows", [5, 90])
def test_tokens_of_any_stride(rows):
    g = generator(92)
    h, w = normal(g, rows, 64, dtype=torch.bfloat16), normal(g, 300, 64, dtype=torch.bfloat16)
    tokens = torch.randint(300, (rows, 3), device="cuda", generator=g)
    for t in (tokens[:, 1], tokens[:1, 0].expand(rows), tokens[:, 2].flip(0)):
        assert torch.equal(rb.token_logprobs(h, w, t), rb.token_logprobs(h, w, t.contiguous()))


@pytest.mark.parametrize("dtype,least", [(torch.bfloat16, -133), (torch.float16, -24),
                                         (torch.float32, -133)])
@pytest.mark.parametrize("rows", [3, 150])
def test_subnormal_operands_count(rows, dtype, least):
    """Powers of two down to the type's smallest (fp32: to the smallest that its
    parts hold) times one, summed exactly: fp32 outputs hold 24 bits from any of
    them up, 16-bit ones their own."""
    x = torch.ones(rows, 64, device="cuda", dtype=dtype)
    powers = torch.tensor([2.0 ** e for e in range(least, least + 40)], dtype=torch.float64).cuda()
    w = torch.zeros(40, 64, device="cuda", dtype=dtype)
    w[:, 7] = powers.to(dtype)
    assert torch.equal(w[:, 7].double(), powers)
    got = rb.linear(x, w)
    assert torch.equal(got.double(), powers.expand(rows, 40))
    assert torch.equal(rb.linear(w, x), got.t())


def test_beside_prefill_attention():
    """Tensor-core kernels of both kinds take TMEM on the same SMs: calls on one
    stream and packed prefill on another give what they give alone."""
    g = generator(93)
    heads, d, page, tokens = 16, 128, 16, 1024
    pool = normal(g, 2, 2 * tokens // page, page, heads, d, dtype=torch.bfloat16)
    tables = torch.arange(2 * tokens // page, device="cuda", dtype=torch.int32).view(2, -1)
    lengths = torch.full((2,), tokens, device="cuda", dtype=torch.int32)
    cu = torch.tensor([0, tokens, 2 * tokens], device="cuda", dtype=torch.int32)
    q = normal(g, 2 * tokens, heads, d, dtype=torch.bfloat16)
    made = {rows: (normal(g, rows, 1024, dtype=torch.bfloat16),
                   normal(g, 2048, 1024, std=0.05, dtype=torch.bfloat16)) for rows in (3, 64, 600)}
    single = (normal(g, 40, 512), normal(g, 400, 512, std=0.05))

    def attention():
        return rb.paged_prefill(q, pool[0], pool[1], tables, lengths, cu, tokens)

    def projections():
        result = []
        for x, w in made.values():
            result += [rb.linear(x, w, activation="silu"), rb.gated_linear(x, w),
                       *rb.greedy_tokens(x, w)]
        return [*result, rb.linear(*single), *rb.greedy_tokens(*single)]

    want_attention, want = attention(), projections()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    attended, projected = [], []
    for _ in range(20):
        with torch.cuda.stream(streams[0]):
            attended.append(attention())
        for s in streams[1:]:
            with torch.cuda.stream(s):
                projected.append(projections())
    torch.cuda.synchronize()
    assert rb.check_errors() == []
    assert all(torch.equal(a, want_attention) for a in attended)
    assert all(torch.equal(a, b) for r in projected for a, b in zip(r, want))


def test_calls_from_several_threads():
    g = generator(94)
    x, w = normal(g, 70, 320, dtype=torch.bfloat16), normal(g, 192, 320, std=0.05, dtype=torch.bfloat16)
    want = [rb.linear(x, w), rb.gated_linear(x, w), *rb.greedy_tokens(x, w)]
    torch.cuda.synchronize()
    failed = []

    def work():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(50):
                    got = [rb.linear(x, w), rb.gated_linear(x, w), *rb.greedy_tokens(x, w)]
                torch.cuda.current_stream().synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        except BaseException as error:  # noqa: BLE001
            failed.append(error)

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert failed == []
