"""What is measured of the layer-norm backward pass and of the fused linear layer: cases, inputs, one pass, its work.

A case is one call of one operator.  ``run`` computes it in elementary torch operations, or, with ``own`` set, through
the package's own entry points.  The operators are the parts of one pre-norm feed-forward block, trained and served:

    layernorm_backward      dx, dgamma, dbeta of y = (x - mean) * rsqrt(var + eps) * gamma + beta  (dx + residual gradient)
    linear                  y = act(x w^T + bias) + residual, and the pre-activation when it is kept for the backward pass
    linear_backward_input   dx = (dy w) * act'(pre): the gradient of the layer before, through its activation
    linear_backward_weight  dw = dy^T x (+ c) and dbias = the column sums of dy
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu")
_MAX_FLOPS = 2.0 * 16384 * 4096 * 1024      # no drawn product is larger than the largest listed one
_MAX_ROW_BYTES = 32768 * 4096 * 2           # nor one array of a drawn layer norm


def listed():
    return [
        # the encoder layer norm of the benchmark configuration (FP32, 16384 tokens of width 768)
        {"name": "ln_bwd_f32_16384x768", "op": "layernorm_backward", "dtype": "f32", "rows": 16384, "cols": 768,
         "gamma": True, "residual": False, "ddof": 0},
        # a wide pre-norm block in BF16: the gradient of the skip connection is added in the same pass; the largest norm
        {"name": "ln_bwd_bf16_32768x4096", "op": "layernorm_backward", "dtype": "bf16", "rows": 32768, "cols": 4096,
         "gamma": True, "residual": True, "ddof": 0},
        # a short odd-width batch, where no row starts on a vector boundary and latency counts
        {"name": "ln_bwd_f16_333x1001", "op": "layernorm_backward", "dtype": "f16", "rows": 333, "cols": 1001,
         "gamma": True, "residual": False, "ddof": 0},
        # training, up projection: bias and GELU in the epilogue, pre-activation kept
        {"name": "linear_bf16_16384x4096x1024_gelu", "op": "linear", "dtype": "bf16", "out": "bf16", "tokens": 16384,
         "n": 4096, "k": 1024, "activation": "gelu", "bias": True, "residual": False, "pre": True},
        # training, down projection: bias and the skip connection in the epilogue
        {"name": "linear_bf16_16384x1024x4096_residual", "op": "linear", "dtype": "bf16", "out": "bf16", "tokens": 16384,
         "n": 1024, "k": 4096, "activation": "none", "bias": True, "residual": True, "pre": False},
        # serving, one new token: the weights are read once, latency is everything
        {"name": "linear_f16_1x4096x4096_silu", "op": "linear", "dtype": "f16", "out": "f16", "tokens": 1, "n": 4096,
         "k": 4096, "activation": "silu", "bias": True, "residual": False, "pre": False},
        # serving, a handful of sequences decoded together, down projection with the skip connection
        {"name": "linear_bf16_20x2000x8192_residual", "op": "linear", "dtype": "bf16", "out": "bf16", "tokens": 20,
         "n": 2000, "k": 8192, "activation": "none", "bias": True, "residual": True, "pre": False},
        # a ragged prompt into an output head kept in FP32: odd number of tokens and of columns
        {"name": "linear_bf16_1021x2053x1096_f32", "op": "linear", "dtype": "bf16", "out": "f32", "tokens": 1021,
         "n": 2053, "k": 1096, "activation": "relu", "bias": True, "residual": False, "pre": False},
        # training, back through the down projection and the GELU before it
        {"name": "dgrad_bf16_16384x1024x4096_gelu", "op": "linear_backward_input", "dtype": "bf16", "out": "bf16",
         "tokens": 16384, "n": 1024, "k": 4096, "activation": "gelu"},
        # a small fine-tuning batch in FP16
        {"name": "dgrad_f16_250x1000x776_silu", "op": "linear_backward_input", "dtype": "f16", "out": "f16",
         "tokens": 250, "n": 1000, "k": 776, "activation": "silu"},
        # training, weight and bias gradients of the up projection over a whole batch, FP32 for the optimiser
        {"name": "wgrad_bf16_16384x4096x1024", "op": "linear_backward_weight", "dtype": "bf16", "out": "f32",
         "tokens": 16384, "n": 4096, "k": 1024, "bias": True, "c": False},
        # one micro-batch of odd length added to the gradient gathered so far
        {"name": "wgrad_f16_777x1000x520_add", "op": "linear_backward_weight", "dtype": "f16", "out": "f32", "tokens": 777,
         "n": 1000, "k": 520, "bias": True, "c": True},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["layernorm_backward", "layernorm_backward", "linear", "linear", "linear_backward_input",
                     "linear_backward_weight"])
    if op == "layernorm_backward":
        # widths from short odd ones to rows beyond one block's registers; odd, or a multiple of 8 as real widths are
        cols = _log_uniform(rng, 64, 20480)
        if rng.random() < 0.6:
            cols = (cols + 7) // 8 * 8
        dtype = rng.choice(["f32", "f16", "bf16"])
        rows = min(_log_uniform(rng, 1, 65536), _MAX_ROW_BYTES // (_SIZE[dtype] * cols) - 1)
        return {"op": op, "dtype": dtype, "rows": rows, "cols": cols,
                "gamma": rng.random() < 0.8, "residual": rng.random() < 0.5, "ddof": int(rng.random() < 0.2)}
    n, k = _log_uniform(rng, 64, 8192), _log_uniform(rng, 64, 8192) // 8 * 8
    tokens = _log_uniform(rng, 1, 16384)
    tokens = max(1, min(tokens, int(_MAX_FLOPS / (2.0 * n * k)), 100_000_000 // max(n, k)))
    dtype = rng.choice(["f16", "bf16"])
    out = rng.choice([dtype, dtype, "f32"])
    if op == "linear":
        return {"op": op, "dtype": dtype, "out": out, "tokens": tokens, "n": n, "k": k, "activation": rng.choice(_ACTIVATIONS),
                "bias": rng.random() < 0.8, "residual": rng.random() < 0.4, "pre": rng.random() < 0.4}
    n = n // 8 * 8
    if op == "linear_backward_input":
        return {"op": op, "dtype": dtype, "out": out, "tokens": tokens, "n": n, "k": k, "activation": rng.choice(_ACTIVATIONS)}
    return {"op": op, "dtype": dtype, "out": out, "tokens": tokens, "n": n, "k": k, "bias": rng.random() < 0.7,
            "c": rng.random() < 0.4}


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, to=dtype):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(scale).add_(shift).to(to)

    if case["op"] == "layernorm_backward":
        rows, cols = case["rows"], case["cols"]
        # activations of a residual stream: rows of different size and offset
        x = torch.randn(rows, cols, generator=gen, device="cuda")
        x.mul_(torch.rand(rows, 1, generator=gen, device="cuda").mul_(2.0).add_(0.25))
        x.add_(torch.randn(rows, 1, generator=gen, device="cuda").mul_(0.5))
        return {"case": case, "x": x.to(dtype), "dy": normal(rows, cols), "eps": 1e-5,
                "gamma": normal(cols, scale=0.2, shift=1.0) if case["gamma"] else None,
                "residual": normal(rows, cols) if case["residual"] else None}
    m, n, k = case["tokens"], case["n"], case["k"]
    out = _DTYPES[case["out"]]
    if case["op"] == "linear":
        return {"case": case, "x": normal(m, k), "w": normal(n, k, scale=k ** -0.5),
                "bias": normal(n, scale=0.5) if case["bias"] else None,
                "residual": normal(m, n, to=out) if case["residual"] else None}
    if case["op"] == "linear_backward_input":
        return {"case": case, "dy": normal(m, n), "w": normal(n, k, scale=n ** -0.5),
                "pre": normal(m, k, scale=1.5) if case["activation"] != "none" else None}
    return {"case": case, "dy": normal(m, n), "x": normal(m, k), "c": normal(n, k, to=out) if case["c"] else None}


def _activation(z, kind):
    if kind == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if kind == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if kind == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if kind == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _activation_slope(z, kind):
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if kind == "gelu_tanh":
        t = torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * math.sqrt(2.0 / math.pi) * (1.0 + 3 * 0.044715 * z * z)
    s = 1.0 / (1.0 + torch.exp(-z))
    return s * (1.0 + z * (1.0 - s))


def _plain(state):
    case = state["case"]
    dtype = _DTYPES[case["dtype"]]
    if case["op"] == "layernorm_backward":
        x, dy = state["x"].float(), state["dy"].float()
        count = case["cols"] - case["ddof"]
        centred = x - x.mean(dim=1, keepdim=True)
        rstd = 1.0 / torch.sqrt((centred * centred).sum(dim=1, keepdim=True) / count + state["eps"])
        normed = centred * rstd
        g = dy * state["gamma"].float() if state["gamma"] is not None else dy
        dx = rstd * (g - g.mean(dim=1, keepdim=True) - normed * ((g * normed).sum(dim=1, keepdim=True) / count))
        if state["residual"] is not None:
            dx = dx + state["residual"].float()
        return dx.to(dtype), (dy * normed).sum(dim=0), dy.sum(dim=0)
    out = _DTYPES[case["out"]]
    if case["op"] == "linear":
        z = state["x"].float() @ state["w"].float().t()
        if state["bias"] is not None:
            z = z + state["bias"].float()
        y = _activation(z, case["activation"])
        if state["residual"] is not None:
            y = y + state["residual"].float()
        return (y.to(out), z.to(dtype)) if case["pre"] else y.to(out)
    if case["op"] == "linear_backward_input":
        dx = state["dy"].float() @ state["w"].float()
        if state["pre"] is not None:
            dx = dx * _activation_slope(state["pre"].float(), case["activation"])
        return dx.to(out)
    dy = state["dy"].float()
    dw = dy.t() @ state["x"].float()
    if state["c"] is not None:
        dw = dw + state["c"].float()
    return (dw.to(out), dy.sum(dim=0)) if case["bias"] else dw.to(out)


def _own(state):
    import kernel_optimization_b200 as ko

    case = state["case"]
    if case["op"] == "layernorm_backward":
        return ko.layernorm_backward(state["dy"], state["x"], state["eps"], state["gamma"], case["ddof"],
                                     residual=state["residual"])
    out = _DTYPES[case["out"]]
    if case["op"] == "linear":
        return ko.linear(state["x"], state["w"], state["bias"], activation=case["activation"], residual=state["residual"],
                         out_dtype=out, return_pre=case["pre"])
    if case["op"] == "linear_backward_input":
        return ko.linear_backward_input(state["dy"], state["w"], state["pre"], activation=case["activation"], out_dtype=out)
    return ko.linear_backward_weight(state["dy"], state["x"], c=state["c"], out_dtype=out, return_bias=case["bias"])


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    size = _SIZE[case["dtype"]]
    if case["op"] == "layernorm_backward":
        rows, cols = case["rows"], case["cols"]
        read = (3 if case["residual"] else 2) * rows * cols * size + (cols * size if case["gamma"] else 0)
        return {"bytes": read + rows * cols * size + 2 * cols * 4, "flops": 16 * rows * cols}
    m, n, k = case["tokens"], case["n"], case["k"]
    out = _SIZE[case["out"]]
    if case["op"] == "linear":
        moved = (m * k + n * k) * size + m * n * out + (n * size if case["bias"] else 0)
        moved += (m * n * out if case["residual"] else 0) + (m * n * size if case["pre"] else 0)
    elif case["op"] == "linear_backward_input":
        moved = (m * n + n * k) * size + m * k * out + (m * k * size if case["activation"] != "none" else 0)
    else:
        moved = (m * n + m * k) * size + n * k * out * (2 if case["c"] else 1) + (n * 4 if case["bias"] else 0)
    return {"bytes": moved, "flops": 2 * m * n * k}


def exact(case, seed):
    """The definition in 64 bits: statistics by row, products as blocks of inner products."""
    state = prepare(case, seed)
    f64 = torch.float64

    def dot(a, b):
        # rows of a times rows of b, over the last dimension, a few thousand rows at a time
        return torch.cat([torch.einsum("ik,jk->ij", part, b) for part in a.split(4096)]) if len(a) else a @ b.t()

    if case["op"] == "layernorm_backward":
        gamma = torch.ones(case["cols"], dtype=f64, device="cuda") if state["gamma"] is None else state["gamma"].to(f64)
        free = case["cols"] - case["ddof"]
        dgamma = torch.zeros(case["cols"], dtype=f64, device="cuda")
        dbeta = torch.zeros_like(dgamma)
        pieces = []
        for r0 in range(0, case["rows"], 4096):
            x, dy = state["x"][r0:r0 + 4096].to(f64), state["dy"][r0:r0 + 4096].to(f64)
            mean = x.sum(1) / case["cols"]
            inv = ((x - mean[:, None]).pow(2).sum(1) / free + state["eps"]).pow(-0.5)
            xhat = (x - mean[:, None]) * inv[:, None]
            # d y_i / d x_j = inv * gamma_i * (delta_ij - 1 / cols - xhat_i * xhat_j / free)
            upstream = dy * gamma
            along = torch.einsum("rc,rc->r", upstream, xhat) / free
            dx = inv[:, None] * (upstream - upstream.sum(1, keepdim=True) / case["cols"] - along[:, None] * xhat)
            pieces.append(dx if state["residual"] is None else dx + state["residual"][r0:r0 + 4096].to(f64))
            dgamma += torch.einsum("rc,rc->c", dy, xhat)
            dbeta += dy.sum(0)
        return torch.cat(pieces), dgamma, dbeta

    kind = case.get("activation", "none")
    root_half, root_2_over_pi = math.sqrt(0.5), math.sqrt(2.0 / math.pi)
    if case["op"] == "linear":
        z = dot(state["x"].to(f64), state["w"].to(f64))
        if state["bias"] is not None:
            z += state["bias"].to(f64)
        if kind == "relu":
            y = z.clamp(min=0.0)
        elif kind == "gelu":
            y = 0.5 * z * torch.erfc(-z * root_half)
        elif kind == "gelu_tanh":
            y = z * torch.sigmoid(2.0 * root_2_over_pi * (z + 0.044715 * z.pow(3)))
        elif kind == "silu":
            y = z * torch.sigmoid(z)
        else:
            y = z
        if state["residual"] is not None:
            y = y + state["residual"].to(f64)
        return (y, z) if case["pre"] else y
    if case["op"] == "linear_backward_input":
        dx = dot(state["dy"].to(f64), state["w"].to(f64).t())
        if state["pre"] is not None:
            z = state["pre"].to(f64)
            if kind == "relu":
                slope = torch.sign(z).clamp(min=0.0)
            elif kind == "gelu":
                slope = 0.5 * torch.erfc(-z * root_half) + z * torch.exp(-z.pow(2) / 2.0) * (0.5 * root_2_over_pi)
            elif kind == "gelu_tanh":
                s = torch.sigmoid(2.0 * root_2_over_pi * (z + 0.044715 * z.pow(3)))
                slope = s + z * s * (1.0 - s) * 2.0 * root_2_over_pi * (1.0 + 3.0 * 0.044715 * z.pow(2))
            else:
                slope = torch.sigmoid(z) + z * torch.sigmoid(z) * torch.sigmoid(-z)
            dx = dx * slope
        return dx
    dw = dot(state["dy"].to(f64).t(), state["x"].to(f64).t())
    if state["c"] is not None:
        dw = dw + state["c"].to(f64)
    return (dw, state["dy"].to(f64).sum(0)) if case["bias"] else dw
