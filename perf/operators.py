"""The operators of a transformer's feed-forward sublayer and of its training step, as cases to be measured.

Six kinds of pass, the three operators in each direction:

    ln_forward      layernorm_rows_stats       y = (x - mean) * rstd * gamma + beta, with mean and rstd kept for the backward pass
    ln_backward     layernorm_rows_backward    dx, dgamma, dbeta
    gemm_forward    gemm_bias_act_residual     c = act(a @ b + bias) + residual, with a @ b + bias kept where a backward pass follows
    gemm_backward   gemm_bias_act_backward     da, db, dbias
    gated_forward   gated_gemm                 h = act(x @ w_gate + bias_gate) * (x @ w_up + bias_up), with both projections kept
    gated_backward  gated_gemm_backward        dx, dw_gate, dw_up and the gradients of the biases

`run` computes a pass in elementary torch operations in 32 bits, or, where `own` is true, makes the framework's call.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the norm in front of one decoding step of a few sequences: all latency
        {"name": "ln_forward_decode", "kind": "ln_forward", "type": "bf16", "rows": 8, "cols": 4096},
        # the norm of a training micro-batch of 16384 tokens
        {"name": "ln_forward_train", "kind": "ln_forward", "type": "bf16", "rows": 16384, "cols": 4096},
        # the backward pass over the benchmark's layer-norm size
        {"name": "ln_backward_train", "kind": "ln_backward", "type": "bf16", "rows": 65536, "cols": 8192},
        # fp32 training with a row length that is no whole number of 16-byte vectors
        {"name": "ln_backward_odd", "kind": "ln_backward", "type": "f32", "rows": 4099, "cols": 1001},
        # output projection of one token with the residual stream added
        {"name": "gemm_forward_decode", "kind": "gemm_forward", "rows": 1, "k": 4096, "n": 4096, "act": "none", "bias": False,
         "residual": True, "save": False},
        # an ungated feed-forward layer on a few short prompts of odd lengths, packed
        {"name": "gemm_forward_odd", "kind": "gemm_forward", "rows": 1003, "k": 1000, "n": 2728, "act": "silu", "bias": True,
         "residual": False, "save": False},
        # the benchmark's contraction with everything its epilogue can carry in a training step
        {"name": "gemm_forward_train", "kind": "gemm_forward", "rows": 8192, "k": 8192, "n": 8192, "act": "gelu", "bias": True,
         "residual": True, "save": True},
        # the backward pass of an ungated feed-forward layer's first projection
        {"name": "gemm_backward_train", "kind": "gemm_backward", "rows": 4096, "k": 4096, "n": 11008, "act": "gelu", "bias": True},
        # a small layer on an odd number of tokens
        {"name": "gemm_backward_odd", "kind": "gemm_backward", "rows": 515, "k": 1032, "n": 2056, "act": "relu", "bias": True},
        # one decoding step of sixteen sequences through the gated projections
        {"name": "gated_forward_decode", "kind": "gated_forward", "rows": 16, "k": 4096, "n": 11008, "act": "silu", "bias": False,
         "save": False},
        # a training micro-batch through the gated projections
        {"name": "gated_forward_train", "kind": "gated_forward", "rows": 8192, "k": 4096, "n": 11008, "act": "silu", "bias": False,
         "save": True},
        # its backward pass on half the tokens
        {"name": "gated_backward_train", "kind": "gated_backward", "rows": 4096, "k": 4096, "n": 11008, "act": "silu", "bias": False},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["ln_forward", "ln_backward", "gemm_forward", "gemm_backward", "gated_forward", "gated_backward"])
    if kind.startswith("ln"):
        # rows from one token to a large micro-batch, columns from a head's to a large model's, any remainder
        cols = _log_uniform(rng, 64, 16384)
        if rng.random() < 0.6:
            cols = max(64, cols // 64 * 64)
        rows = _log_uniform(rng, 1, min(65536, (1 << 28) // cols))
        return {"kind": kind, "type": rng.choice(["bf16", "bf16", "f32"]), "rows": rows, "cols": cols}
    # contractions: k and n in whole 16-byte vectors, any number of tokens
    k = 8 * _log_uniform(rng, 8, 1024)
    n = 8 * _log_uniform(rng, 8, 1376)
    most = (1 << 37) // (k * n)
    rows = _log_uniform(rng, 1, max(1, min(8192, most)))
    case = {"kind": kind, "rows": rows, "k": k, "n": n, "bias": rng.random() < 0.5}
    if kind.startswith("gemm"):
        case["act"] = rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"])
        if kind == "gemm_forward":
            case["residual"] = rng.random() < 0.5
            case["save"] = rows > 64 and rng.random() < 0.5
    else:
        case["act"] = rng.choice(["silu", "gelu", "gelu_tanh", "sigmoid", "relu"])
        if kind == "gated_forward":
            case["save"] = rows > 64 and rng.random() < 0.5
    return case


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape, scale=1.0, dtype=torch.bfloat16):
        # generated in pieces, so that a large tensor does not need a 32-bit copy of itself
        t = torch.empty(shape, device="cuda", dtype=dtype)
        flat = t.view(-1)
        step = 1 << 27
        for i in range(0, flat.numel(), step):
            part = flat[i:i + step]
            part.copy_(torch.randn(part.numel(), device="cuda", generator=g).mul_(scale))
        return t

    s = {"case": case}
    if case["kind"].startswith("ln"):
        dtype, rows, cols = _TYPES[case["type"]], case["rows"], case["cols"]
        # a residual stream: off centre, a few columns much larger than the others
        x = normal(rows, cols, scale=2.0, dtype=dtype)
        x += 0.5
        x[:, ::97] *= 8
        s["x"] = x
        s["gamma"] = normal(cols, scale=0.2, dtype=dtype).add_(1)
        s["beta"] = normal(cols, scale=0.1, dtype=dtype)
        s["eps"] = 1e-5
        if case["kind"] == "ln_backward":
            s["dy"] = normal(rows, cols, scale=0.02, dtype=dtype)
            # what the forward pass has kept
            mean, rstd = _ln_statistics(x, 1e-5)
            s["mean"], s["rstd"] = mean.view(rows), rstd.view(rows)
        return s
    rows, k, n = case["rows"], case["k"], case["n"]
    s["x"] = normal(rows, k)  # the output of a norm
    names = ["b"] if case["kind"].startswith("gemm") else ["w_gate", "w_up"]
    for name in names:
        s[name] = normal(k, n, scale=k ** -0.5)
    if case["kind"].endswith("forward"):
        for name in (["bias"] if len(names) == 1 else ["bias_gate", "bias_up"]):
            s[name] = normal(n, scale=0.2, dtype=torch.float32) if case["bias"] else None
        s["residual"] = normal(rows, n, scale=2.0) if case.get("residual") else None
    else:
        s["dy"] = normal(rows, n, scale=0.02)
        # the projections that the forward pass has kept
        if len(names) == 1:
            s["z"] = normal(rows, n) if case["act"] != "none" else None
        else:
            s["gate"], s["up"] = normal(rows, n), normal(rows, n)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass: the framework's calls, or the plain form
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    return (_RUN_OWN if own else _RUN_PLAIN)[case["kind"]](s, case)


def _framework():
    import tcacomp_b200
    return tcacomp_b200


def _own_ln_forward(s, case):
    y, mean, rstd = _framework().layernorm_rows_stats(s["x"], s["gamma"], s["beta"], s["eps"])
    return {"y": y, "mean": mean, "rstd": rstd}


def _own_ln_backward(s, case):
    dx, dgamma, dbeta = _framework().layernorm_rows_backward(s["dy"], s["x"], s["gamma"], s["mean"], s["rstd"])
    return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}


def _own_gemm_forward(s, case):
    z = torch.empty((case["rows"], case["n"]), device="cuda", dtype=torch.bfloat16) if case["save"] else None
    c = _framework().gemm_bias_act_residual(s["x"], s["b"], s["bias"], s["residual"], case["act"], preact=z)
    return {"c": c, "z": z} if case["save"] else {"c": c}


def _own_gemm_backward(s, case):
    want = ("da", "db", "dbias") if case["bias"] else ("da", "db")
    return _framework().gemm_bias_act_backward(s["dy"], s["x"], s["b"], s["z"], case["act"], want=want)


def _own_gated_forward(s, case):
    if not case["save"]:
        return {"h": _framework().gated_gemm(s["x"], s["w_gate"], s["w_up"], s["bias_gate"], s["bias_up"], case["act"])}
    gate, up = (torch.empty((case["rows"], case["n"]), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    h = _framework().gated_gemm(s["x"], s["w_gate"], s["w_up"], s["bias_gate"], s["bias_up"], case["act"], gate=gate, up=up)
    return {"h": h, "gate": gate, "up": up}


def _own_gated_backward(s, case):
    want = ("dx", "dw_gate", "dw_up") + (("dbias_gate", "dbias_up") if case["bias"] else ())
    return _framework().gated_gemm_backward(s["dy"], s["x"], s["w_gate"], s["w_up"], s["gate"], s["up"], case["act"], want=want)


def _ln_statistics(x, eps):
    x = x.float()
    mean = x.mean(-1, keepdim=True)
    var = (x - mean).square().mean(-1, keepdim=True)
    return mean, (var + eps).rsqrt()


def _plain_ln_forward(s, case):
    mean, rstd = _ln_statistics(s["x"], s["eps"])
    y = (s["x"].float() - mean) * rstd * s["gamma"].float() + s["beta"].float()
    return {"y": y.to(s["x"].dtype), "mean": mean.view(-1), "rstd": rstd.view(-1)}


def _plain_ln_backward(s, case):
    dy = s["dy"].float()
    rstd = s["rstd"].view(-1, 1)
    xhat = (s["x"].float() - s["mean"].view(-1, 1)) * rstd
    wdy = dy * s["gamma"].float()
    dx = rstd * (wdy - wdy.mean(-1, keepdim=True) - xhat * (wdy * xhat).mean(-1, keepdim=True))
    return {"dx": dx.to(s["x"].dtype), "dgamma": (dy * xhat).sum(0), "dbeta": dy.sum(0)}


def _normal_cdf(z):
    return 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))


def _act(z, act):
    if act == "none":
        return z
    if act == "relu":
        return z * (z > 0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    if act == "gelu":
        return z * _normal_cdf(z)
    return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))  # gelu_tanh


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    if act == "sigmoid":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 - p)
    if act == "gelu":
        return _normal_cdf(z) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    c = math.sqrt(2 / math.pi)  # gelu_tanh
    t = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def _project(x, w, bias):
    z = x.float() @ w.float()
    return z if bias is None else z + bias


def _plain_gemm_forward(s, case):
    z = _project(s["x"], s["b"], s["bias"])
    c = _act(z, case["act"])
    if s["residual"] is not None:
        c = c + s["residual"].float()
    return {"c": c.bfloat16(), "z": z.bfloat16()} if case["save"] else {"c": c.bfloat16()}


def _plain_gemm_backward(s, case):
    dz = s["dy"].float()
    if case["act"] != "none":
        dz = dz * _act_slope(s["z"].float(), case["act"])
    grads = {"da": (dz @ s["b"].float().t()).bfloat16(), "db": (s["x"].float().t() @ dz).bfloat16()}
    if case["bias"]:
        grads["dbias"] = dz.sum(0)
    return grads


def _plain_gated_forward(s, case):
    gate = _project(s["x"], s["w_gate"], s["bias_gate"])
    up = _project(s["x"], s["w_up"], s["bias_up"])
    h = _act(gate, case["act"]) * up
    return {"h": h.bfloat16(), "gate": gate.bfloat16(), "up": up.bfloat16()} if case["save"] else {"h": h.bfloat16()}


def _plain_gated_backward(s, case):
    dh, gate, up, x = s["dy"].float(), s["gate"].float(), s["up"].float(), s["x"].float()
    dgate = dh * up * _act_slope(gate, case["act"])
    dup = dh * _act(gate, case["act"])
    grads = {"dx": (dgate @ s["w_gate"].float().t() + dup @ s["w_up"].float().t()).bfloat16(),
             "dw_gate": (x.t() @ dgate).bfloat16(), "dw_up": (x.t() @ dup).bfloat16()}
    if case["bias"]:
        grads["dbias_gate"], grads["dbias_up"] = dgate.sum(0), dup.sum(0)
    return grads


_RUN_OWN = {"ln_forward": _own_ln_forward, "ln_backward": _own_ln_backward, "gemm_forward": _own_gemm_forward,
            "gemm_backward": _own_gemm_backward, "gated_forward": _own_gated_forward, "gated_backward": _own_gated_backward}
_RUN_PLAIN = {"ln_forward": _plain_ln_forward, "ln_backward": _plain_ln_backward, "gemm_forward": _plain_gemm_forward,
              "gemm_backward": _plain_gemm_backward, "gated_forward": _plain_gated_forward,
              "gated_backward": _plain_gated_backward}


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without: every input read once, every output written once
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind.startswith("ln"):
        rows, cols = case["rows"], case["cols"]
        es = 2 if case["type"] == "bf16" else 4
        if kind == "ln_forward":
            return {"bytes": 2 * rows * cols * es + 2 * cols * es + 8 * rows, "flops": 8 * rows * cols}
        return {"bytes": 3 * rows * cols * es + cols * es + 8 * rows + 8 * cols, "flops": 14 * rows * cols}
    rows, k, n = case["rows"], case["k"], case["n"]
    if kind == "gemm_forward":
        tiles = rows * k + k * n + rows * n * (1 + case["residual"] + case["save"])
        return {"bytes": 2 * tiles + 4 * n * case["bias"], "flops": 2 * rows * k * n}
    if kind == "gemm_backward":
        tiles = 2 * rows * k + 2 * k * n + rows * n * (1 + (case["act"] != "none"))
        return {"bytes": 2 * tiles + 4 * n * case["bias"], "flops": 4 * rows * k * n}
    if kind == "gated_forward":
        tiles = rows * k + 2 * k * n + rows * n * (3 if case["save"] else 1)
        return {"bytes": 2 * tiles + 8 * n * case["bias"], "flops": 4 * rows * k * n}
    tiles = 2 * rows * k + 4 * k * n + 3 * rows * n
    return {"bytes": 2 * tiles + 8 * n * case["bias"], "flops": 8 * rows * k * n}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = {name: t.double() if isinstance(t, torch.Tensor) else t for name, t in prepare(case, seed).items()}
    kind, x = case["kind"], s["x"]
    if kind == "ln_forward":
        var, mean = torch.var_mean(x, dim=1, correction=0)
        deviation = torch.sqrt(var + s["eps"])
        y = torch.addcmul(s["beta"], x.sub(mean[:, None]).div_(deviation[:, None]), s["gamma"])
        return {"y": y, "mean": mean, "rstd": deviation.reciprocal()}
    if kind == "ln_backward":
        # y = g * u + b with u = (x - mean) * rstd: du/dx is rstd * (1 - 1/n - u u^T / n)
        u = x.sub_(s["mean"][:, None]).mul_(s["rstd"][:, None])
        dgamma = torch.einsum("rc,rc->c", s["dy"], u)
        dbeta = torch.einsum("rc->c", s["dy"])
        du = s["dy"].mul_(s["gamma"])
        along_one = du.sum(1) / case["cols"]
        along_u = torch.einsum("rc,rc->r", du, u) / case["cols"]
        dx = du.sub_(along_one[:, None]).sub_(u.mul_(along_u[:, None])).mul_(s["rstd"][:, None])
        return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}

    def value_and_slope(z):
        act = case["act"]
        if act == "none":
            return z, torch.ones_like(z)
        if act == "relu":
            return torch.clamp(z, min=0), torch.heaviside(z, torch.zeros((), dtype=z.dtype, device=z.device))
        if act in ("silu", "sigmoid"):
            p = torch.special.expit(z)
            q = p * torch.special.expit(-z)
            return (z * p, p + z * q) if act == "silu" else (p, q)
        if act == "gelu":
            phi = torch.special.erfc(z * -math.sqrt(0.5)) / 2
            return z * phi, phi + z * torch.exp(z * z / -2) / math.sqrt(2 * math.pi)
        w = math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3)  # gelu_tanh: (1 + tanh(w / 2)) / 2 = expit(w)
        p = torch.special.expit(w)
        return z * p, p + z * p * torch.special.expit(-w) * math.sqrt(8 / math.pi) * (1 + 0.134145 * z ** 2)

    if kind == "gemm_forward":
        z = x.matmul(s["b"])
        if s["bias"] is not None:
            z += s["bias"]
        c = value_and_slope(z)[0]
        if s["residual"] is not None:
            c = c + s["residual"]
        return {"c": c, "z": z} if case["save"] else {"c": c}
    if kind == "gemm_backward":
        dz = s["dy"]
        if s["z"] is not None:
            dz = value_and_slope(s["z"])[1].mul_(dz)
        grads = {"da": torch.einsum("rn,kn->rk", dz, s["b"]), "db": torch.einsum("rk,rn->kn", x, dz)}
        if case["bias"]:
            grads["dbias"] = torch.einsum("rn->n", dz)
        return grads
    if kind == "gated_forward":
        gate, up = x.matmul(s["w_gate"]), x.matmul(s["w_up"])
        if s["bias_gate"] is not None:
            gate += s["bias_gate"]
            up += s["bias_up"]
        h = value_and_slope(gate)[0] * up
        return {"h": h, "gate": gate, "up": up} if case["save"] else {"h": h}
    value, slope = value_and_slope(s["gate"])
    dgate, dup = slope.mul_(s["dy"]).mul_(s["up"]), value.mul_(s["dy"])
    grads = {"dx": torch.einsum("rn,kn->rk", dgate, s["w_gate"]).add_(torch.einsum("rn,kn->rk", dup, s["w_up"])),
             "dw_gate": torch.einsum("rk,rn->kn", x, dgate), "dw_up": torch.einsum("rk,rn->kn", x, dup)}
    if case["bias"]:
        grads["dbias_gate"], grads["dbias_up"] = torch.einsum("rn->n", dgate), torch.einsum("rn->n", dup)
    return grads
