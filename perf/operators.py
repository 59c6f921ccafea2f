"""What is measured of the dense operators beside the packed expert layer.

Four operators, the parts of a model layer that stay outside the packed experts:

``int8_linear``   y = x W^T + b with both operands in 8-bit integers: one scale a token, one a weight row
``int8_gated``    h = silu(x Wg^T) * (x Wu^T) with the same operands (the first half of an 8-bit feed-forward block)
``ffn``           y = (silu(x Wg^T) * (x Wu^T)) Wd^T in 16 bits, as it is served
``ffn_train``     the same block and the gradients of x and of the three weights

``run`` computes them in elementary torch operations in 32 bits where ``own`` is false, and through the package's public
functions where it is true.  ``exact`` computes them from their definitions in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one token through a projection of the 35B-A3B-like layer (hidden 2048): decode, latency counts
        {"name": "int8_linear t1", "op": "int8_linear", "tokens": 1, "k": 2048, "n": 4096, "dtype": "bf16", "bias": False},
        # a ragged batch through a biased projection with an odd number of outputs (a classifier or value head)
        {"name": "int8_linear ragged", "op": "int8_linear", "tokens": 333, "k": 2064, "n": 1001, "dtype": "fp16", "bias": True},
        # prefill of eight sequences of 2048 tokens through a square projection of a dense model
        {"name": "int8_linear prefill", "op": "int8_linear", "tokens": 16384, "k": 4096, "n": 4096, "dtype": "bf16", "bias": False},
        # the shared expert of the 35B-A3B-like layer at a decode batch of 16
        {"name": "int8_gated t16", "op": "int8_gated", "tokens": 16, "k": 2048, "n": 512, "dtype": "bf16"},
        # a ragged chunk of a prompt through a dense block whose sizes are multiples of no tile
        {"name": "int8_gated ragged", "op": "int8_gated", "tokens": 1111, "k": 4112, "n": 10936, "dtype": "fp16"},
        # the shared expert of the 35B-A3B-like layer over the benchmark's batch (16 sequences x 2048 tokens)
        {"name": "int8_gated prefill", "op": "int8_gated", "tokens": 32768, "k": 2048, "n": 512, "dtype": "bf16"},
        # one token through an unpacked shared expert
        {"name": "ffn t1", "op": "ffn", "tokens": 1, "k": 2048, "n": 512, "dtype": "bf16"},
        # a decode batch of 64 through a dense block: bound by reading the weights
        {"name": "ffn t64", "op": "ffn", "tokens": 64, "k": 5120, "n": 13824, "dtype": "fp16"},
        # the unpacked shared expert over the benchmark's batch
        {"name": "ffn prefill", "op": "ffn", "tokens": 32768, "k": 2048, "n": 512, "dtype": "bf16"},
        # tuning a small block on a short ragged batch
        {"name": "ffn_train ragged", "op": "ffn_train", "tokens": 257, "k": 1032, "n": 2728, "dtype": "fp16"},
        # tuning the shared expert of a packed layer: few weights, many tokens (the weight gradients sum over a long axis)
        {"name": "ffn_train shared", "op": "ffn_train", "tokens": 8192, "k": 2048, "n": 512, "dtype": "bf16"},
        # a training step of a dense block
        {"name": "ffn_train dense", "op": "ffn_train", "tokens": 8192, "k": 4096, "n": 14336, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["int8_linear", "int8_gated", "ffn", "ffn_train"])
    case = {"op": op, "dtype": rng.choice(["bf16", "fp16"])}
    case["k"] = 16 * _log_int(rng, 16, 320)                       # 256 .. 5120
    if op == "int8_linear":
        case["n"] = _log_int(rng, 128, 16384)                     # any number of outputs, odd ones among them
        case["bias"] = rng.random() < 0.5
    elif op == "int8_gated":
        case["n"] = _log_int(rng, 128, 14336)
    else:
        case["n"] = 8 * _log_int(rng, 16, 1792)                   # 128 .. 14336
    tokens = _log_int(rng, 1, 32768 if op != "ffn_train" else 8192)
    # at most half the work of the largest listed case
    most = 9 * 8192 * 4096 * 14336
    case["tokens"] = max(1, min(tokens, most // (_products(op) * case["k"] * case["n"])))
    return case


def _products(op):
    """Multiply-adds of a pass over tokens x k x n."""
    return {"int8_linear": 1, "int8_gated": 2, "ffn": 3, "ffn_train": 9}[op]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    t, k, n, dt = case["tokens"], case["k"], case["n"], DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    # activations: N(0, 1) with one channel in a hundred twenty times as large, as in the benchmark's layers
    wide = torch.rand(k, generator=g, device=DEV) < 0.01
    x = (normal(t, k) * torch.where(wide, 20.0, 1.0)).to(dt)
    state = {"op": case["op"], "x": x}

    def int8_weight(rows):
        codes = (normal(rows, k) * 32).round().clamp(-127, 127).to(torch.int8)
        scale = 0.02 / 32 * torch.exp(0.3 * normal(rows))
        return codes, scale

    if case["op"] == "int8_linear":
        state["w"], state["w_scale"] = int8_weight(n)
        state["bias"] = normal(n).to(dt) if case["bias"] else None
    elif case["op"] == "int8_gated":
        state["w_gate"], state["gate_scale"] = int8_weight(n)
        state["w_up"], state["up_scale"] = int8_weight(n)
    else:
        train = case["op"] == "ffn_train"
        state["w_gate"] = (0.02 * normal(n, k)).to(dt)
        state["w_up"] = (0.02 * normal(n, k)).to(dt)
        state["w_down"] = (0.02 * normal(k, n)).to(dt)
        if train:
            state["dy"] = normal(t, k).to(dt)
            for name in ("x", "w_gate", "w_up", "w_down"):
                state[name].requires_grad_(True)
    return state


def run(state):
    if own:
        return _own(state)
    return _plain(state)


def _own(state):
    from dartmoq_b200 import dense

    op, x = state["op"], state["x"]
    if op == "int8_linear":
        return dense.int8_linear(x, state["w"], state["w_scale"], state["bias"])
    if op == "int8_gated":
        return dense.int8_gated_linear(x, state["w_gate"], state["gate_scale"], state["w_up"], state["up_scale"])
    weights = (state["w_gate"], state["w_up"], state["w_down"])
    y = dense.gated_feed_forward(x, *weights)
    if op == "ffn":
        return y
    grads = torch.autograd.grad(y, (x,) + weights, state["dy"])
    return {"y": y.detach(), "dx": grads[0], "dw_gate": grads[1], "dw_up": grads[2], "dw_down": grads[3]}


def _codes(x):
    """8-bit codes of each row, as whole numbers in 32-bit floats, and the row's scale.  127 x has at most 18
    significant bits and the row's largest value 11, so the 32-bit quotient is a tie only where the exact one is."""
    x = x.float()
    top = x.abs().amax(dim=1, keepdim=True)
    codes = torch.where(top > 0, torch.round(127.0 * x / torch.where(top > 0, top, 1.0)), 0.0)
    return codes, top / 127.0


@torch.no_grad()
def _plain(state):
    op, x = state["op"], state["x"]
    dt = x.dtype
    if op == "int8_linear":
        codes, scale = _codes(x)
        y = (codes @ state["w"].float().t()) * scale * state["w_scale"]
        if state["bias"] is not None:
            y = y + state["bias"].float()
        return y.to(dt)
    if op == "int8_gated":
        codes, scale = _codes(x)
        gate = (codes @ state["w_gate"].float().t()) * scale * state["gate_scale"]
        up = (codes @ state["w_up"].float().t()) * scale * state["up_scale"]
        return (gate / (1.0 + torch.exp(-gate)) * up).to(dt)
    x = x.float()
    w_gate, w_up, w_down = (state[name].float() for name in ("w_gate", "w_up", "w_down"))
    gate, up = x @ w_gate.t(), x @ w_up.t()
    sig = 1.0 / (1.0 + torch.exp(-gate))
    hidden = gate * sig * up
    y = (hidden @ w_down.t()).to(dt)
    if op == "ffn":
        return y
    dy = state["dy"].float()
    dhidden = dy @ w_down
    dgate = dhidden * up * sig * (1.0 + gate * (1.0 - sig))
    dup = dhidden * gate * sig
    return {"y": y, "dx": (dgate @ w_gate + dup @ w_up).to(dt), "dw_gate": (dgate.t() @ x).to(dt),
            "dw_up": (dup.t() @ x).to(dt), "dw_down": (dy.t() @ hidden).to(dt)}


def work(case):
    t, k, n, op = case["tokens"], case["k"], case["n"], case["op"]
    flops = 2 * _products(op) * t * k * n
    if op == "int8_linear":
        byts = 2 * t * k + n * k + 4 * n + 2 * t * n + (2 * n if case["bias"] else 0)
    elif op == "int8_gated":
        byts = 2 * t * k + 2 * n * k + 8 * n + 2 * t * n
    elif op == "ffn":
        byts = 2 * (2 * t * k + 3 * n * k)
    else:
        byts = 2 * (4 * t * k + 6 * n * k)      # x, dy, y, dx; three weights and their gradients
    return {"bytes": byts, "flops": flops}


@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    op = state["op"]
    v = {name: t.detach().double() for name, t in state.items() if torch.is_tensor(t)}
    if op in ("int8_linear", "int8_gated"):
        largest = torch.linalg.vector_norm(v["x"], ord=math.inf, dim=-1)
        step = largest / 127
        whole = (127 * v["x"]).div_(largest.clamp(min=1e-300).unsqueeze(-1)).round_()

        def product(w, scale):
            return torch.einsum("tk,nk->tn", whole, v[w]) * torch.outer(step, v[scale])

        if op == "int8_linear":
            y = product("w", "w_scale")
            return y + v["bias"] if "bias" in v else y
        return torch.nn.functional.silu(product("w_gate", "gate_scale")) * product("w_up", "up_scale")
    a = torch.einsum("tk,nk->tn", v["x"], v["w_gate"])
    b = torch.einsum("tk,nk->tn", v["x"], v["w_up"])
    s = torch.sigmoid(a)
    y = torch.einsum("tn,kn->tk", a * s * b, v["w_down"])
    if op == "ffn":
        return y
    d = torch.einsum("tk,kn->tn", v["dy"], v["w_down"])
    da, db = d * b * (s + a * s * (1 - s)), d * a * s
    return {"y": y,
            "dx": torch.einsum("tn,nk->tk", da, v["w_gate"]) + torch.einsum("tn,nk->tk", db, v["w_up"]),
            "dw_gate": torch.einsum("tn,tk->nk", da, v["x"]),
            "dw_up": torch.einsum("tn,tk->nk", db, v["x"]),
            "dw_down": torch.einsum("tk,tn->kn", v["dy"], a * s * b)}
