"""Float operators around the 8-bit path, as timed cases: products with an epilogue, layer normalization with its gradient, and the
log probabilities of given tokens with theirs.

Every case is a dict of plain values; `kind` names the operator:

  linear         y = act(x w^T + b) + r, or act(x w^T + b + r)
  layernorm      LayerNormalization with the statistics a gradient needs
  layernorm_grad its gradient by the input, the scale and the bias
  logprobs       log probability of one token per row, entropy, log of the sum, and the best alternatives
  logprobs_grad  the gradient by the logits, given those of the log probability and of the entropy

`own` chooses between the package's operators and their plain forms in elementary torch operations.
"""
import importlib
import math

import torch

own = False

_DEV = "cuda:0"
_TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_ACTIVATIONS = [None, "Relu", "Gelu", "GeluTanh", "Swish", "Sigmoid", "Tanh"]
_EPS = 1e-5


def _ops(found=[]):
    if not found:
        found.append(importlib.import_module("chainer-compiler_b200.ops"))  # the folder's name is not an identifier
    return found[0]


def listed():
    return [
        # one token through the first product of a feed-forward block
        {"name": "linear_token", "kind": "linear", "m": 1, "o": 4096, "k": 1024, "dtype": "bfloat16", "act": "GeluTanh", "residual": "none", "bias": True, "pad": 0},
        # the hidden layer of a classifier head kept in 32 bits, at the classifier's own batch and width
        {"name": "linear_head_f32", "kind": "linear", "m": 256, "o": 1000, "k": 2048, "dtype": "float32", "act": "Relu", "residual": "none", "bias": True, "pad": 0},
        # odd extents, rows cut out of a wider buffer, residual joined before the activation
        {"name": "linear_ragged", "kind": "linear", "m": 509, "o": 2999, "k": 1283, "dtype": "float16", "act": "Swish", "residual": "first", "bias": True, "pad": 13},
        # the largest product of the integer sweep, in 16 bits: second product of a feed-forward block over a long prompt
        {"name": "linear_8192", "kind": "linear", "m": 8192, "o": 8192, "k": 8192, "dtype": "bfloat16", "act": None, "residual": "last", "bias": True, "pad": 0},
        # the tokens of one decoding step of a batch
        {"name": "layernorm_batch", "kind": "layernorm", "rows": 64, "d": 1000, "dtype": "float32", "affine": "float32", "bias": True},
        # a long prompt, or a training batch
        {"name": "layernorm_16384", "kind": "layernorm", "rows": 16384, "d": 4096, "dtype": "bfloat16", "affine": "bfloat16", "bias": True},
        # odd extents, parameters in 32 bits beside 16-bit activations
        {"name": "layernorm_grad_ragged", "kind": "layernorm_grad", "rows": 4099, "d": 1283, "dtype": "float16", "affine": "float32"},
        # the training batch
        {"name": "layernorm_grad_8192", "kind": "layernorm_grad", "rows": 8192, "d": 8192, "dtype": "bfloat16", "affine": "float32"},
        # one decoding step of one sequence, with alternatives
        {"name": "logprobs_token", "kind": "logprobs", "rows": 1, "v": 131072, "dtype": "bfloat16", "top": 20, "masked": False, "pad": 0},
        # scoring a batch of prompts; a vocabulary of odd size in padded rows, some tokens forbidden
        {"name": "logprobs_ragged", "kind": "logprobs", "rows": 4096, "v": 50001, "dtype": "float32", "top": 5, "masked": True, "pad": 47},
        # the image networks' classes
        {"name": "logprobs_grad_classes", "kind": "logprobs_grad", "rows": 256, "v": 1000, "dtype": "float32", "masked": False, "pad": 0},
        # the loss of a training batch of tokens
        {"name": "logprobs_grad_4096", "kind": "logprobs_grad", "rows": 4096, "v": 131072, "dtype": "bfloat16", "masked": False, "pad": 0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _extent(rng, lo, hi):
    """An extent between lo and hi, spread over the logarithm: as it falls, or rounded to a multiple of 16 as often."""
    v = _log_int(rng, lo, hi)
    return v if rng.random() < 0.5 else max(16, (v + 8) // 16 * 16)


def draw(rng):
    kind = rng.choice(["linear", "linear", "layernorm", "layernorm_grad", "logprobs", "logprobs_grad"])
    dtype = rng.choice(["bfloat16", "float16", "float32"])
    if kind == "linear":
        most = 8192 ** 3 if dtype != "float32" else 2048 ** 3
        while True:
            m, o, k = _extent(rng, 1, 8192), _extent(rng, 16, 8192), _extent(rng, 16, 8192)
            if m * o * k <= most:
                break
        return {"kind": kind, "m": m, "o": o, "k": k, "dtype": dtype, "act": rng.choice(_ACTIVATIONS), "residual": rng.choice(["none", "none", "last", "first"]),
                "bias": rng.random() < 0.8, "pad": rng.choice([0, 0, 0, 16, rng.randint(1, 64)])}
    if kind in ("layernorm", "layernorm_grad"):
        while True:
            rows, d = _log_int(rng, 1, 65536), _extent(rng, 16, 16384)
            if rows * d <= 8192 * 8192:
                break
        case = {"kind": kind, "rows": rows, "d": d, "dtype": dtype, "affine": rng.choice([dtype, "float32"])}
        if kind == "layernorm":
            case["bias"] = rng.random() < 0.8
        return case
    while True:
        rows, v = _log_int(rng, 1, 16384), _extent(rng, 128, 262144)
        if rows * v * (2 if dtype == "float32" else 1) <= 4096 * 131072:
            break
    case = {"kind": kind, "rows": rows, "v": v, "dtype": dtype, "masked": rng.random() < 0.3, "pad": rng.choice([0, 0, rng.randint(1, 64)])}
    if kind == "logprobs":
        case["top"] = rng.choice([0, 1, 5, 20, rng.randint(2, 32)])
    return case


# ---- inputs -------------------------------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=_DEV).manual_seed(int(seed))


def _normal(shape, dtype, gen, scale=1.0, shift=0.0):
    return (torch.randn(shape, device=_DEV, generator=gen) * scale + shift).to(_TYPES[dtype])


def _chunks(rows, cols, limit=1 << 26):
    step = max(1, limit // max(1, cols))
    return [(r, min(rows, r + step)) for r in range(0, rows, step)]


def _logits(case, gen):
    """Logits [rows, v] in rows of v + pad values: a spread of about three, a few likely tokens a row; `masked`: three in ten forbidden."""
    rows, v = case["rows"], case["v"]
    buf = torch.zeros((rows, v + case["pad"]), dtype=_TYPES[case["dtype"]], device=_DEV)
    logits = buf[:, :v]
    tokens = torch.empty(rows, dtype=torch.int64, device=_DEV)
    for a, b in _chunks(rows, v):
        x = torch.randn((b - a, v), device=_DEV, generator=gen) * 2.5
        x.scatter_add_(1, torch.randint(0, v, (b - a, 8), device=_DEV, generator=gen), torch.full((b - a, 8), 6.0, device=_DEV))
        if case["masked"]:
            x.masked_fill_(torch.rand((b - a, v), device=_DEV, generator=gen) < 0.3, float("-inf"))
        logits[a:b] = x.to(logits.dtype)
        x = logits[a:b].float()
        x -= torch.log(-torch.log(torch.rand((b - a, v), device=_DEV, generator=gen).clamp_(1e-30, 1 - 1e-7)))
        tokens[a:b] = x.argmax(dim=1)  # a token drawn with the probabilities that the logits give
    return logits, tokens


def _prepare_linear(case, seed):
    g = _gen(seed)
    m, o, k, dt = case["m"], case["o"], case["k"], case["dtype"]
    x = _normal((m, k + case["pad"]), dt, g)[:, :k]
    state = {"x": x, "w": _normal((o, k), dt, g, 1.0 / math.sqrt(k)), "b": _normal((o,), dt, g, 0.2) if case["bias"] else None,
             "r": _normal((m, o), dt, g) if case["residual"] != "none" else None}
    return state


def _prepare_layernorm(case, seed):
    g = _gen(seed)
    rows, d = case["rows"], case["d"]
    state = {"x": _normal((rows, d), case["dtype"], g, 1.7, 0.3), "scale": _normal((d,), case["affine"], g, 0.2, 1.0)}
    if case["kind"] == "layernorm":
        state["bias"] = _normal((d,), case["affine"], g, 0.2) if case["bias"] else None
    else:
        state["dy"] = _normal((rows, d), case["dtype"], g)
        x = state["x"].float()
        mean = x.mean(dim=1, keepdim=True)
        state["mean"], state["inv"] = mean, torch.rsqrt((x - mean).square_().mean(dim=1, keepdim=True) + _EPS)
    return state


def _prepare_logprobs(case, seed):
    g = _gen(seed)
    logits, tokens = _logits(case, g)
    state = {"logits": logits, "tokens": tokens}
    if case["kind"] == "logprobs_grad":
        rows = case["rows"]
        state["dlp"] = torch.full((rows,), -1.0 / rows, device=_DEV) * (1 + torch.rand(rows, device=_DEV, generator=g))
        state["dent"] = torch.full((rows,), -0.01 / rows, device=_DEV)
        lse, ent = torch.empty(rows, device=_DEV), torch.empty(rows, device=_DEV)
        for a, b in _chunks(rows, case["v"]):
            lse[a:b], ent[a:b] = _lse_entropy(logits[a:b].float())
        state["lse"], state["ent"] = lse, ent
    return state


def prepare(case, seed):
    f = {"linear": _prepare_linear, "layernorm": _prepare_layernorm, "layernorm_grad": _prepare_layernorm}.get(case["kind"], _prepare_logprobs)
    return dict(f(case, seed), case=dict(case))


# ---- plain forms ----------------------------------------------------------------------------------------------------------


def _activate(z, act):
    if act is None:
        return z
    if act == "Relu":
        return torch.clamp(z, min=0)
    if act == "Gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "GeluTanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "Swish":
        return z / (1 + torch.exp(-z))
    if act == "Sigmoid":
        return 1 / (1 + torch.exp(-z))
    return torch.tanh(z)


def _plain_linear(s):
    c = s["case"]
    z = s["x"].float() @ s["w"].float().t()
    if s["b"] is not None:
        z += s["b"].float()
    if c["residual"] == "first":
        z += s["r"].float()
    y = _activate(z, c["act"])
    if c["residual"] == "last":
        y = y + s["r"].float()
    return y.to(s["x"].dtype)


def _plain_layernorm(s):
    x = s["x"].float()
    mean = x.mean(dim=1, keepdim=True)
    x = x - mean
    inv = 1 / torch.sqrt((x * x).mean(dim=1, keepdim=True) + _EPS)
    y = x * inv * s["scale"].float()
    if s["bias"] is not None:
        y += s["bias"].float()
    return y.to(s["x"].dtype), mean, inv


def _plain_layernorm_grad(s):
    xh = (s["x"].float() - s["mean"]) * s["inv"]
    dy = s["dy"].float()
    gd = dy * s["scale"].float()
    dx = s["inv"] * (gd - gd.mean(dim=1, keepdim=True) - xh * (gd * xh).mean(dim=1, keepdim=True))
    t = s["scale"].dtype
    return dx.to(s["x"].dtype), (dy * xh).sum(dim=0).to(t), dy.sum(dim=0).to(t)


def _lse_entropy(x):
    m = x.amax(dim=1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(dim=1)
    log_total = torch.log(total)
    # a forbidden token has probability zero and adds nothing, whatever its logit
    mean = torch.where(e > 0, e * (x - m), 0.0).sum(dim=1) / total
    return m[:, 0] + log_total, log_total - mean


def _sortable(x):
    """Whole numbers that order as (value, then lower index first)."""
    bits = (x + 0.0).view(torch.int32)  # -0 counts as 0
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64)
    return (order << 32) + (0xFFFFFFFF - torch.arange(x.shape[1], device=x.device))


def _plain_logprobs(s):
    c = s["case"]
    parts = []
    for a, b in _chunks(c["rows"], c["v"], 1 << 28):
        x = s["logits"][a:b].float()
        lse, ent = _lse_entropy(x)
        lp = x.gather(1, s["tokens"][a:b, None])[:, 0] - lse
        keys = torch.topk(_sortable(x), c["top"], dim=1)[0]
        idx = 0xFFFFFFFF - (keys & 0xFFFFFFFF)
        parts.append((lp, ent, lse, x.gather(1, idx) - lse[:, None], idx))
    return tuple(torch.cat(p) if len(p) > 1 else p[0] for p in zip(*parts))


def _plain_logprobs_grad(s):
    c = s["case"]
    out = torch.empty((c["rows"], c["v"]), dtype=s["logits"].dtype, device=_DEV)
    for a, b in _chunks(c["rows"], c["v"], 1 << 28):
        logp = s["logits"][a:b].float() - s["lse"][a:b, None]
        p = torch.exp(logp)
        d = -s["dlp"][a:b, None] * p - torch.where(p > 0, s["dent"][a:b, None] * p * (logp + s["ent"][a:b, None]), 0.0)
        d.scatter_add_(1, s["tokens"][a:b, None], s["dlp"][a:b, None])
        out[a:b] = d.to(out.dtype)
    return out


_PLAIN = {"linear": _plain_linear, "layernorm": _plain_layernorm, "layernorm_grad": _plain_layernorm_grad, "logprobs": _plain_logprobs,
          "logprobs_grad": _plain_logprobs_grad}


# ---- the package's operators ------------------------------------------------------------------------------------------------


def _own_linear(s):
    c = s["case"]
    return _ops().Linear(s["x"], s["w"], s["b"], activation=c["act"], residual=s["r"], residual_first=c["residual"] == "first")


def _own_layernorm(s):
    return _ops().LayerNormalization(s["x"], s["scale"], s["bias"], epsilon=_EPS, stats=True)


def _own_layernorm_grad(s):
    return _ops().LayerNormalizationGrad(s["dy"], s["x"], s["scale"], s["mean"], s["inv"])


def _own_logprobs(s):
    return _ops().TokenLogProbs(s["logits"], s["tokens"], s["case"]["top"])


def _own_logprobs_grad(s):
    return _ops().TokenLogProbsGrad(s["dlp"], s["dent"], s["logits"], s["tokens"], s["lse"], s["ent"])


_OWN = {"linear": _own_linear, "layernorm": _own_layernorm, "layernorm_grad": _own_layernorm_grad, "logprobs": _own_logprobs,
        "logprobs_grad": _own_logprobs_grad}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["kind"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------


def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "linear":
        m, o, k = case["m"], case["o"], case["k"]
        return {"bytes": e * (m * k + o * k + m * o * (1 if case["residual"] == "none" else 2) + (o if case["bias"] else 0)), "flops": 2 * m * o * k}
    if case["kind"] in ("layernorm", "layernorm_grad"):
        rows, d, p = case["rows"], case["d"], 4 if case["affine"] == "float32" else 2
        if case["kind"] == "layernorm":
            return {"bytes": 2 * e * rows * d + 8 * rows + p * d * (2 if case["bias"] else 1), "flops": 7 * rows * d}
        return {"bytes": 3 * e * rows * d + 8 * rows + 3 * p * d, "flops": 13 * rows * d}
    rows, v = case["rows"], case["v"]
    if case["kind"] == "logprobs":
        return {"bytes": e * rows * v + rows * (8 + 12 + 12 * case["top"]), "flops": 5 * rows * v}
    return {"bytes": 2 * e * rows * v + rows * (8 + 16), "flops": 7 * rows * v}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------


def _exact_linear(case, s):
    x, w = s["x"].double(), s["w"].double()
    z = torch.matmul(x, w.T)
    del x, w
    if case["bias"]:
        z = z + s["b"].double()
    if case["residual"] == "first":
        z = z + s["r"].double()
    act = case["act"]
    if act == "Relu":
        z = torch.where(z > 0, z, torch.zeros_like(z))
    elif act == "Gelu":
        z = z * torch.special.ndtr(z)
    elif act == "GeluTanh":
        z = z * torch.special.expit(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))  # (1 + tanh u) / 2 = 1 / (1 + exp(-2 u))
    elif act == "Swish":
        z = z * torch.special.expit(z)
    elif act == "Sigmoid":
        z = torch.special.expit(z)
    elif act == "Tanh":
        z = 2 * torch.special.expit(2 * z) - 1
    return z + s["r"].double() if case["residual"] == "last" else z


def _exact_layernorm(case, s):
    x = s["x"].double()
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    inv = (var + _EPS) ** -0.5
    y = (x - mean) / torch.sqrt(var + _EPS) * s["scale"].double()
    return (y if s["bias"] is None else y + s["bias"].double()), mean, inv


def _exact_layernorm_grad(case, s):
    d = case["d"]
    mean, inv, scale = s["mean"].double(), s["inv"].double(), s["scale"].double()
    dx, dscale, dbias = [], torch.zeros_like(scale), torch.zeros_like(scale)
    for a, b in _chunks(case["rows"], d):
        x, dy = s["x"][a:b].double(), s["dy"][a:b].double()
        xh = (x - mean[a:b]) * inv[a:b]
        c1 = dy @ scale / d
        c2 = (dy * xh) @ scale / d
        dx.append((dy * scale - c1[:, None] - c2[:, None] * xh) * inv[a:b])
        dscale += torch.einsum("rd,rd->d", dy, xh)
        dbias += torch.einsum("rd->d", dy)
    return torch.cat(dx), dscale, dbias


def _exact_logprobs(case, s):
    lp, ent, lse, top_lp, top = [], [], [], [], []
    for a, b in _chunks(case["rows"], case["v"], 1 << 25):
        logp = torch.log_softmax(s["logits"][a:b].double(), dim=1)
        p = torch.exp(logp)
        ent.append(torch.special.entr(p).sum(dim=1))
        t = s["tokens"][a:b]
        picked = logp[torch.arange(b - a, device=_DEV), t]
        lp.append(picked)
        lse.append(s["logits"][torch.arange(a, b, device=_DEV), t].double() - picked)
        order = torch.sort(s["logits"][a:b], dim=1, descending=True, stable=True)[1][:, :case["top"]]
        top.append(order)
        top_lp.append(torch.gather(logp, 1, order))
    return tuple(torch.cat(v) for v in (lp, ent, lse, top_lp, top))


def _exact_logprobs_grad(case, s):
    out = []
    for a, b in _chunks(case["rows"], case["v"], 1 << 25):
        logp = s["logits"][a:b].double() - s["lse"][a:b].double()[:, None]
        p = torch.exp(logp)
        onehot = torch.zeros_like(p)
        onehot[torch.arange(b - a, device=_DEV), s["tokens"][a:b]] = 1
        inner = torch.nan_to_num(p * logp, nan=0.0) + p * s["ent"][a:b].double()[:, None]
        out.append(s["dlp"][a:b].double()[:, None] * (onehot - p) - s["dent"][a:b].double()[:, None] * inner)
    return torch.cat(out)


def exact(case, seed):
    s = prepare(case, seed)
    f = {"linear": _exact_linear, "layernorm": _exact_layernorm, "layernorm_grad": _exact_layernorm_grad, "logprobs": _exact_logprobs,
         "logprobs_grad": _exact_logprobs_grad}[case["kind"]]
    return f(case, s)
