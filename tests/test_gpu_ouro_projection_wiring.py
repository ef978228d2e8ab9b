"""The decoder's 16-bit step on the projection kernels: each product has the
weights that the layer's has, and is held to the 64-bit form of its own input
(tests/projection_oracle.py derives the bounds)."""

from __future__ import annotations

import pytest
import torch

import projection_oracle as po
from test_gpu_ouro import make_decoder
from test_gpu_projections import assert_within
from vllm_rlt_b200 import ouro

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["last_exited", "shared"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_projection_of_a_step(dtype, layout, monkeypatch):
    dec, sched = make_decoder(dtype, layout, seed=5)
    dec.projections = "kernels"
    seen = []
    linear, gated_linear, greedy_tokens = ouro.linear, ouro.gated_linear, ouro.greedy_tokens

    def checked_linear(x, w, bias=None, *, activation=None):
        y = linear(x, w, bias, activation=activation)
        assert_within(y, *po.linear(x, w, bias, activation))
        seen.append(("linear", w.data_ptr()))
        return y

    def checked_gated(x, w):
        y = gated_linear(x, w)
        assert_within(y, *po.gated(x, w))
        seen.append(("gated", w.data_ptr()))
        return y

    def checked_greedy(h, w):
        tokens, logprobs = greedy_tokens(h, w)
        z, e, lp, bound = po.vocab(h, w)
        at = tokens[:, None]
        assert bool((z.gather(1, at) >= z.amax(-1, keepdim=True) - 2 * e).all())
        assert_within(logprobs, lp.gather(1, at)[:, 0], bound.gather(1, at)[:, 0])
        seen.append(("greedy", w.data_ptr()))
        return tokens, logprobs

    monkeypatch.setattr(ouro, "linear", checked_linear)
    monkeypatch.setattr(ouro, "gated_linear", checked_gated)
    monkeypatch.setattr(ouro, "greedy_tokens", checked_greedy)
    w = dec.w
    step = []
    for i in range(dec.shape.layers):
        step += [("linear", w.wqkv[i].data_ptr()), ("linear", w.wo[i].data_ptr()),
                 ("gated", w.wgu[i].data_ptr()), ("linear", w.wdown[i].data_ptr())]
    step += [("linear", w.gate_w.data_ptr()), ("greedy", w.lm_head.data_ptr())]
    for _ in range(6):
        seen.clear()
        exiting = sched.prepare()
        before, kept = dec.tokens.clone(), dec.logprobs.clone()
        dec.run(graphed=False)
        assert seen == step
        out = ~dec.exit_mask
        assert torch.equal(dec.tokens[out], before[out])
        assert torch.equal(dec.logprobs[out], kept[out])
        sched.advance(exiting)
    assert dec.attention.check_errors() == []
