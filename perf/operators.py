"""The dense feed-forward operators that stand beside the mixture-of-experts layer, as measurable cases.

  gated   ``torch_ops.gated_linear``: act(x Wg^T + bg) * (x Wu^T + bu), the two projections stacked as the layer stacks its
          experts' ([2 * ispp, hidden], gate rows, then up rows), and ``torch_ops.gated_linear_backward``
  linear  ``torch_ops.fused_linear``: act(x W^T + b) + residual, and ``torch_ops.fused_linear_backward``

A dense layer of a mixture-of-experts model, or its always-on expert where the checkpoint keeps that one in 16 bits, is the
first followed by the second. Shapes are those of the benchmark configurations (2880 x 2880, 7168 x 2048) and generic ones.
Where ``own`` is false a pass is made of elementary torch operations in 32 bits, rounded once at the end.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
# SiTU's two constants, as the layer takes them
BETA, LINEAR_BETA = 4.0, 25.0


def _case(op, tokens, n_in, n_out, *, dtype="bf16", train=False, bias=False, act="none", limit=0.0, residual=False, gap=0):
    """``n_out``: features of the result (gated: of the product, so the weight has twice as many rows). ``gap``: elements between
    one token's row and the next one's beyond ``n_in`` (x is a slice of a wider tensor)."""
    return dict(op=op, tokens=tokens, n_in=n_in, n_out=n_out, dtype=dtype, train=train, bias=bias, act=act, limit=limit,
                residual=residual, gap=gap)


def listed():
    named = {
        # one user's decode step: latency and the rate at which the weights arrive
        "gated_1": _case("gated", 1, 2880, 2880, act="swiglu", limit=7.0),
        # a decode batch through the always-on expert of the wide model
        "gated_64_wide": _case("gated", 64, 7168, 2048, act="swiglu"),
        # decode tokens and a prompt's tail in one batch, with biases and the other activation; half precision
        "gated_333_fp16": _case("gated", 333, 2880, 2880, dtype="fp16", bias=True, act="situ"),
        # prefill through the always-on expert of the wide model
        "gated_8192_wide": _case("gated", 8192, 7168, 2048, act="swiglu"),
        # a training step of a dense layer
        "gated_train_4096": _case("gated", 4096, 2880, 2880, train=True, bias=True, act="swiglu", limit=7.0),
        # a short, ragged training batch of a model whose sizes are not multiples of anything
        "gated_train_1001_odd": _case("gated", 1001, 1500, 1027, dtype="fp16", train=True, act="swiglu"),
        # the second projection of a decode step: bias, and the residual stream added
        "linear_1": _case("linear", 1, 2880, 2880, bias=True, residual=True),
        # the wide model's second projection for a decode batch, added to the routed experts' result
        "linear_64_wide": _case("linear", 64, 2048, 7168, residual=True),
        # one chunk of a chunked prefill through a projection with an activation of its own
        "linear_2047_gelu": _case("linear", 2047, 2880, 2880, bias=True, act="gelu"),
        # the largest prefill batch: second projection of the wide model, residual added
        "linear_16384_wide": _case("linear", 16384, 2048, 7168, residual=True),
        # a training step of a projection with everything in its epilogue
        "linear_train_4096": _case("linear", 4096, 2880, 2880, train=True, bias=True, act="gelu_tanh", residual=True),
        # odd features, rows that start anywhere, half precision
        "linear_train_517_odd": _case("linear", 517, 1023, 770, dtype="fp16", train=True, bias=True, act="silu", residual=True, gap=2),
    }
    return [dict(case, name=name) for name, case in named.items()]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """1 to 16384 tokens, 64 to 8192 features on either side (three in four multiples of 8), either type, forward alone or with
    the backward pass, every activation, with and without bias, residual and a gap between the rows."""
    op, train = rng.choice(["gated", "linear"]), rng.random() < 0.4
    tokens, n_in, n_out = (_log_int(rng, *r) for r in ((1, 16384), (64, 8192), (64, 8192)))
    if rng.random() < 0.75:
        n_in, n_out = (n_in + 4) // 8 * 8, (n_out + 4) // 8 * 8
    most = 2.0 * 8192 * 7168 * 4096      # no more products than the largest listed case has
    products = 2.0 * n_in * n_out * (2 if op == "gated" else 1) * (3 if train else 1)
    tokens = max(1, min(tokens, int(most / products)))
    act = rng.choice(["swiglu", "swiglu", "situ"] if op == "gated" else ["none", "none", "silu", "gelu", "gelu_tanh"])
    return _case(op, tokens, n_in, n_out, dtype=rng.choice(["bf16", "bf16", "bf16", "fp16"]), train=train, bias=rng.random() < 0.5,
                 act=act, limit=7.0 if act == "swiglu" and rng.random() < 0.5 else 0.0, residual=op == "linear" and rng.random() < 0.5,
                 gap=rng.choice([0, 0, 0, 8, 64, 3]))


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed((seed & 0x3FFFFFFF) * 7919 + 11)
    dtype, T, K, N = DTYPES[case["dtype"]], case["tokens"], case["n_in"], case["n_out"]
    rows = 2 * N if case["op"] == "gated" else N

    def normal(*shape, std=1.0):
        return (std * torch.randn(shape, generator=g, device=DEVICE)).to(dtype)

    # activations as they leave a norm; weights that give pre-activations a spread of 1.5
    return {"op": case["op"], "train": case["train"], "act": case["act"], "limit": case["limit"],
            "x": normal(T, K + case["gap"])[:, :K],
            "w": normal(rows, K, std=1.5 / math.sqrt(K)),
            "bias": normal(rows, std=0.2) if case["bias"] else None,
            "residual": normal(T, N) if case["residual"] else None,
            "dy": normal(T, N) if case["train"] else None}


def _own(s):
    from vkernels_b200 import torch_ops as ops

    if s["op"] == "gated":
        kw = dict(activation=ops.SITU if s["act"] == "situ" else ops.SWIGLU, swiglu_limit=s["limit"], beta=BETA, linear_beta=LINEAR_BETA)
        if not s["train"]:
            return {"y": ops.gated_linear(s["x"], s["w"], s["bias"], **kw)}
        y, preact = ops.gated_linear(s["x"], s["w"], s["bias"], return_preact=True, **kw)
        dx, dw, db = ops.gated_linear_backward(s["dy"], s["x"], s["w"], preact, bias_grad=s["bias"] is not None, **kw)
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    act = None if s["act"] == "none" else s["act"]
    if not s["train"]:
        return {"y": ops.fused_linear(s["x"], s["w"], s["bias"], activation=act, residual=s["residual"])}
    y, preact = ops.fused_linear(s["x"], s["w"], s["bias"], activation=act, residual=s["residual"], return_preact=True)
    dx, dw, db = ops.fused_linear_backward(s["dy"], s["x"], s["w"], preact, activation=act, bias_grad=s["bias"] is not None)
    return {"y": y, "dx": dx, "dw": dw, "db": db}


def _projected(s):
    z = s["x"].float() @ s["w"].float().t()
    return z if s["bias"] is None else z + s["bias"].float()


def _gradients(s, y, dz):
    dtype = s["x"].dtype
    return {"y": y.to(dtype), "dx": (dz @ s["w"].float()).to(dtype), "dw": (dz.t() @ s["x"].float()).to(dtype),
            "db": None if s["bias"] is None else dz.sum(0).to(dtype)}


def _plain_gated(s):
    g0, u0 = _projected(s).chunk(2, dim=1)
    if s["act"] == "situ":
        a, b, p = torch.tanh(g0 / BETA), torch.tanh(u0 / LINEAR_BETA), torch.sigmoid(g0)
        gate, up = BETA * a * p, LINEAR_BETA * b
    else:
        g, up = (g0.clamp(max=s["limit"]), u0.clamp(-s["limit"], s["limit"])) if s["limit"] > 0 else (g0, u0)
        p = torch.sigmoid(g)
        gate = g * p
    y = gate * up
    if not s["train"]:
        return {"y": y.to(s["x"].dtype)}
    dy = s["dy"].float()
    if s["act"] == "situ":
        dg = dy * up * ((1 - a * a) * p + BETA * a * p * (1 - p))
        du = dy * gate * (1 - b * b)
    else:
        dg, du = dy * up * (p + gate * (1 - p)), dy * gate
        if s["limit"] > 0:
            dg, du = dg * (g0 <= s["limit"]), du * (u0.abs() <= s["limit"])
    return _gradients(s, y, torch.cat([dg, du], dim=1))


def _plain_linear(s):
    z, act = _projected(s), s["act"]
    if act == "none":
        y, slope = z, None
    elif act == "silu":
        p = torch.sigmoid(z)
        y, slope = z * p, p + z * p * (1 - p)
    elif act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        y, slope = z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    else:
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        y, slope = 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    if not s["train"]:
        return {"y": y.to(s["x"].dtype)}
    dz = s["dy"].float()
    return _gradients(s, y, dz if slope is None else dz * slope)


def run(state):
    if own:
        return _own(state)
    return _plain_gated(state) if state["op"] == "gated" else _plain_linear(state)


def exact(case, seed):
    """The definition in 64 bits; the gradients by differentiation of it."""
    s = prepare(case, seed)
    x, w, b = (None if s[n] is None else s[n].double().requires_grad_(case["train"]) for n in ("x", "w", "bias"))
    z = x @ w.mT
    if b is not None:
        z = z + b
    f = torch.nn.functional
    if case["op"] == "gated":
        n = case["n_out"]
        g, u = z[:, :n], z[:, n:]
        if case["act"] == "situ":
            y = BETA * torch.tanh(g / BETA) / (1 + torch.exp(-g)) * LINEAR_BETA * torch.tanh(u / LINEAR_BETA)
        else:
            if case["limit"] > 0:
                top = torch.full((), case["limit"], dtype=torch.float64, device=z.device)
                g = torch.where(g > top, top, g)
                u = torch.where(u > top, top, torch.where(u < -top, -top, u))
            y = f.silu(g) * u
    else:
        act = case["act"]
        y = z if act == "none" else f.silu(z) if act == "silu" else f.gelu(z, approximate="tanh" if act == "gelu_tanh" else "none")
        if s["residual"] is not None:
            y = y + s["residual"].double()
    if not case["train"]:
        return {"y": y}
    leaves = [x, w] if b is None else [x, w, b]
    grads = torch.autograd.grad(y, leaves, s["dy"].double())
    return {"y": y.detach(), "dx": grads[0], "dw": grads[1], "db": grads[2] if b is not None else None}


def work(case):
    """Inputs in and results out once, at two bytes a value; one product for the forward pass, two more for the backward pass."""
    T, K, N = case["tokens"], case["n_in"], case["n_out"]
    rows = 2 * N if case["op"] == "gated" else N
    x, w, y, b = T * K, rows * K, T * N, rows if case["bias"] else 0
    values = x + w + b + y + (y if case["residual"] else 0)
    if case["train"]:
        values += y + x + w + b      # the result's gradient in; the gradients of x, w and the bias out
    return {"bytes": 2 * values, "flops": 2 * T * K * rows * (3 if case["train"] else 1)}
