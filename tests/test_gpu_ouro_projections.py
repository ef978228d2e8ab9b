"""The decoder with its projections, exit gate and next tokens on the package's
kernels, against the dense fp32 reference and its own graph replay."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_ouro import DenseOuro, make_decoder
from vllm_rlt_b200.ouro import OuroDecoder

pytestmark = pytest.mark.gpu


def on_kernels(*args, **kwargs):
    dec, sched = make_decoder(*args, **kwargs)
    dec.projections = "kernels"
    return dec, sched


@pytest.mark.parametrize("layout", ["last_exited", "shared"])
def test_decode_matches_dense_reference(layout):
    """The bound of the same comparison with library products: both sum in fp32."""
    dec, sched = on_kernels(torch.float32, layout)
    dense = DenseOuro(dec)
    for _ in range(14):
        depth, pos = sched.depth.copy(), sched.pos.copy()
        exiting = sched.prepare()
        dec.run(graphed=False)
        expected = dense.step(depth, pos, exiting)
        torch.cuda.synchronize()
        torch.testing.assert_close(dec.hidden_state, expected, atol=2e-4, rtol=2e-4)
        assert torch.equal(dec.tokens, dense.tokens)
        gate = torch.sigmoid(expected @ dec.w.gate_w.t() + dec.w.gate_b)[:, 0]
        torch.testing.assert_close(dec.gate, gate, atol=2e-4, rtol=2e-4)
        ex = np.nonzero(exiting)[0]
        lp = torch.log_softmax(expected @ dec.w.lm_head.t(), -1).amax(-1)
        torch.testing.assert_close(dec.logprobs[ex], lp[ex], atol=2e-4, rtol=2e-4)
        sched.advance(exiting)
    assert dec.attention.check_errors() == []


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_graph_replay_matches_eager_steps(dtype):
    eager, s1 = on_kernels(dtype, seed=3)
    graphed, s2 = on_kernels(dtype, seed=3)
    exiting = s2.prepare()
    graphed.capture()
    for step in range(10):
        e1 = s1.prepare()
        eager.run(graphed=False)
        if step:
            exiting = s2.prepare()
        graphed.run(graphed=True)
        torch.cuda.synchronize()
        for name in ("hidden_state", "tokens", "logprobs"):
            assert torch.equal(getattr(eager, name), getattr(graphed, name))
        s1.advance(e1)
        s2.advance(exiting)
    assert torch.equal(eager.key_cache, graphed.key_cache)


def test_choices_of_projections():
    dec, _ = make_decoder(torch.bfloat16)
    assert dec.projections == "library"
    with pytest.raises(ValueError, match="projections"):
        OuroDecoder(dec.shape, dec.w, [16], "cuda", torch.bfloat16, projections="own")
    with pytest.raises(ValueError, match="fused"):
        OuroDecoder(dec.shape, dec.w, [16], "cuda", torch.bfloat16, fused=False,
                    projections="kernels")
