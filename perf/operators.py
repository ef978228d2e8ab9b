"""Timed cases of the projection operators: the matrix product with its
epilogue, the gated product, and the vocabulary head that never stores logits.

``run`` computes a case in plain torch operations (fp32, one rounding at the
end), or, with ``own`` set, through this package's operators.

  linear           act(x W^T + bias) + residual
  gated_linear     act(x Wg^T) * (x Wu^T), W = [Wg; Wu]
  greedy_tokens    argmax_v h.w_v and its log-probability
  token_logprobs   log softmax(h W^T)[token], 0 where the token is negative
"""

import math

import torch

own = False

HIDDEN, INTERMEDIATE, VOCAB = 2048, 5632, 49152  # the decoder's geometry (ouro.OuroShape)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def linear(name, rows, inner, outer, dtype, act="none", bias=False, residual=False,
           layout="out_in"):
    return {"name": name, "op": "linear", "rows": rows, "in": inner, "out": outer, "dtype": dtype,
            "act": act, "bias": bias, "residual": residual, "layout": layout}


def gated(name, rows, inner, outer, dtype, act="silu", layout="out_in"):
    return {"name": name, "op": "gated_linear", "rows": rows, "in": inner, "out": outer,
            "dtype": dtype, "act": act, "layout": layout}


def head(name, op, rows, inner, outer, dtype, layout="out_in"):
    return {"name": name, "op": op, "rows": rows, "in": inner, "out": outer, "dtype": dtype,
            "layout": layout}


def listed():
    return [
        # the exit gate of a decode step: one output feature for 64 resident requests
        linear("gate 64 rows", 64, HIDDEN, 1, "bf16", "sigmoid", bias=True),
        # one request's new token through the down projection, weights as the decoder holds them
        linear("down 1 row", 1, INTERMEDIATE, HIDDEN, "bf16", residual=True, layout="in_out"),
        # a decode batch's attention output projection
        linear("out 64 rows", 64, HIDDEN, HIDDEN, "bf16", residual=True),
        # a packed prompt chunk through the down projection
        linear("down 4096 rows", 4096, INTERMEDIATE, HIDDEN, "bf16", bias=True, residual=True),
        # a ragged batch, sizes that no tile divides
        linear("odd 777 rows fp16", 777, 1000, 1231, "fp16", "gelu", bias=True, residual=True),
        # a parity run in single precision
        linear("fp32 300 rows", 300, HIDDEN, HIDDEN, "fp32", "silu", bias=True, residual=True),
        # one request's new token through the gate and up projections
        gated("gated 1 row fp16", 1, HIDDEN, INTERMEDIATE, "fp16"),
        # a decode batch, weights as the decoder holds them
        gated("gated 64 rows", 64, HIDDEN, INTERMEDIATE, "bf16", layout="in_out"),
        # a packed prompt chunk
        gated("gated 4096 rows", 4096, HIDDEN, INTERMEDIATE, "bf16"),
        # the next tokens of a decode batch, weights as the decoder holds them
        head("greedy 64 rows", "greedy_tokens", 64, HIDDEN, VOCAB, "bf16", layout="in_out"),
        # scoring a packed prompt: the log-probability of each next token
        head("score 4096 rows", "token_logprobs", 4096, HIDDEN, VOCAB, "bf16"),
        # a parity run of the head, a vocabulary that no tile divides
        head("fp32 greedy 33 rows", "greedy_tokens", 33, 1000, 32003, "fp32"),
    ]


def spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["linear", "gated_linear", "greedy_tokens", "token_logprobs"])
    case = {"op": op, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
            "layout": rng.choice(["out_in", "out_in", "in_out"])}
    inner = spread(rng, 256, INTERMEDIATE)
    outer = spread(rng, 1000, VOCAB) if op.endswith(("tokens", "logprobs")) else spread(rng, 64, 8192)
    kind = rng.random()
    if kind < 0.6:  # whole tiles, as model geometries have them
        inner, outer = -(-inner // 64) * 64, -(-outer // 64) * 64
    elif kind < 0.9:  # whole 16-byte rows only
        inner, outer = -(-inner // 8) * 8, -(-outer // 8) * 8
    case["in"], case["out"] = min(inner, INTERMEDIATE), min(outer, VOCAB)
    # decode batches and prompt chunks; single tokens by themselves. A greedy
    # call has a row for each request, a scoring call one for each token.
    rows = 1 if rng.random() < 0.15 else spread(rng, 2, 256 if op == "greedy_tokens" else 4096)
    if case["dtype"] == "fp32":
        rows = min(rows, 600)
    most = 4096 * HIDDEN * VOCAB
    case["rows"] = max(1, min(rows, most // (case["in"] * case["out"] * 2)))
    if op == "linear":
        case["act"] = rng.choice(["none", "none", "silu", "gelu", "gelu_tanh", "relu", "sigmoid"])
        case["bias"], case["residual"] = rng.random() < 0.5, rng.random() < 0.5
    if op == "gated_linear":
        case["act"] = rng.choice(["silu", "silu", "gelu_tanh", "gelu", "relu", "sigmoid"])
    return case


def prepare(case, seed):
    """Activations as a norm leaves them (unit variance), weights as the model
    initialises them (standard deviation 0.02). The head's activations lean
    towards one vocabulary entry by a different amount in each row, as a
    trained model's do."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    rows, inner, outer = case["rows"], case["in"], case["out"]
    features = 2 * outer if case["op"] == "gated_linear" else outer

    def normal(*size, std=1.0):
        return (torch.randn(size, device="cuda", generator=g) * std).to(dtype)

    if case["layout"] == "in_out":  # [out, in] held as the view of a contiguous [in, out]
        weight = normal(inner, features, std=0.02).t()
    else:
        weight = normal(features, inner, std=0.02)
    state = {"case": case, "weight": weight}
    if case["op"] in ("greedy_tokens", "token_logprobs"):
        target = torch.randint(outer, (rows,), device="cuda", generator=g)
        towards = weight[target].float()
        lean = torch.rand(rows, 1, device="cuda", generator=g) * 12 + 2
        x = torch.randn(rows, inner, device="cuda", generator=g)
        state["x"] = (x + lean * towards / towards.norm(dim=-1, keepdim=True)).to(dtype)
        if case["op"] == "token_logprobs":
            # most rows are scored on the likely token, some on another, and a
            # row at a sequence's end has no next token (-1)
            other = torch.randint(outer, (rows,), device="cuda", generator=g)
            u = torch.rand(rows, device="cuda", generator=g)
            tokens = torch.where(u < 0.25, other, target)
            state["tokens"] = torch.where(u > 0.98, torch.full_like(tokens, -1), tokens)
        return state
    state["x"] = normal(rows, inner)
    if case.get("bias"):
        state["bias"] = normal(outer, std=0.1)
    if case.get("residual"):
        state["residual"] = normal(rows, outer)
    return state


def activate(x, act):
    if act == "silu":
        return x / (1 + torch.exp(-x))
    if act == "gelu":
        return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))
    if act == "relu":
        return torch.clamp(x, min=0)
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-x))
    return x


def run(state):
    case, x, weight = state["case"], state["x"], state["weight"]
    op = case["op"]
    if own:
        import vllm_rlt_b200 as rb

        if op == "linear":
            act = case["act"]
            return rb.linear(x, weight, state.get("bias"), activation=None if act == "none" else act,
                             residual=state.get("residual"))
        if op == "gated_linear":
            return rb.gated_linear(x, weight, activation=case["act"])
        if op == "greedy_tokens":
            return rb.greedy_tokens(x, weight)
        return rb.token_logprobs(x, weight, state["tokens"])
    y = x.float() @ weight.float().t()
    if op == "linear":
        if "bias" in state:
            y = y + state["bias"].float()
        y = activate(y, case["act"])
        if "residual" in state:
            y = y + state["residual"].float()
        return y.to(x.dtype)
    if op == "gated_linear":
        gate, up = y[:, : case["out"]], y[:, case["out"] :]
        return (activate(gate, case["act"]) * up).to(x.dtype)
    most = y.amax(-1)
    total = torch.exp(y - most[:, None]).sum(-1)
    if op == "greedy_tokens":
        return torch.argmax(y, dim=-1), -torch.log(total)
    tokens = state["tokens"]
    chosen = y.gather(1, tokens.clamp(min=0)[:, None])[:, 0]
    return torch.where(tokens < 0, torch.zeros_like(chosen), chosen - most - torch.log(total))


def work(case):
    rows, inner, outer, es = case["rows"], case["in"], case["out"], SIZE[case["dtype"]]
    features = 2 * outer if case["op"] == "gated_linear" else outer
    moved = (rows * inner + features * inner) * es
    if case["op"] in ("linear", "gated_linear"):
        moved += rows * outer * es * (2 if case.get("residual") else 1)
        moved += outer * es if case.get("bias") else 0
    else:
        moved += rows * 12  # a token id (int64) and its log-probability (fp32)
    return {"bytes": moved, "flops": 2 * rows * inner * features}


def exact(case, seed):
    """The definition in 64 bits."""
    state = prepare(case, seed)
    x, w = state["x"].double(), state["weight"].double()
    if case["op"] == "gated_linear":
        gate = torch.einsum("rk,nk->rn", x, w[: case["out"]])
        up = torch.einsum("rk,nk->rn", x, w[case["out"] :])
        return activation64(gate, case["act"]).mul_(up)
    y = torch.einsum("rk,nk->rn", x, w)
    if case["op"] == "linear":
        if case["bias"]:
            y += state["bias"].double()
        y = activation64(y, case["act"])
        return y + state["residual"].double() if case["residual"] else y
    if case["op"] == "greedy_tokens":
        return None, y.amax(-1) - torch.logsumexp(y, -1)
    tokens = state["tokens"]
    scored = torch.nonzero(tokens >= 0)[:, 0]
    result = torch.zeros(case["rows"], dtype=torch.float64, device="cuda")
    result[scored] = y[scored, tokens[scored]] - torch.logsumexp(y, -1)[scored]
    return result


def activation64(x, act):
    f = torch.nn.functional
    return {"none": lambda t: t, "silu": f.silu, "gelu": f.gelu,
            "gelu_tanh": lambda t: f.gelu(t, approximate="tanh"), "relu": f.relu,
            "sigmoid": torch.sigmoid}[act](x)
