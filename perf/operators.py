"""Cases of the dense and the expert-grouped linear products, forward and
backward, in their plain form (elementary torch operations, fp32) and through
the package's entry points:

* ``linear``: y = act(x W^T + b) + r for x [T, in], W [out, in];
* ``linear_backward``: dx, dW and db of act(x W^T + b) from dy;
* ``grouped_linear``: the same product with one W per expert, the rows of x in
  expert order (``offsets`` from the dispatch);
* ``grouped_linear_backward``: its dx, dW and db.

``act`` is none, relu, silu, gelu, gelu_tanh, or a gated pair: swiglu and
geglu take W [2 * out, in] with the gate rows first, y = act(gate) * up.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.abspath(os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
GATED = ("swiglu", "geglu")
ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh", "swiglu", "geglu")
MAX_FLOPS = 4.2e11  # the largest listed case's


def _linear(name, op, rows, inner, out, act="none", bias=False, residual=False, save=False, dtype="bf16"):
    return {"name": name, "op": op, "rows": rows, "in": inner, "out": out, "act": act, "bias": bias,
            "residual": residual, "save": save, "dtype": dtype}


def _grouped(name, op, tokens, experts, top_k, inner, out, act="none", bias=False, save=False, skew=False,
             dtype="bf16"):
    return {"name": name, "op": op, "tokens": tokens, "experts": experts, "top_k": top_k, "in": inner, "out": out,
            "act": act, "bias": bias, "save": save, "skew": skew, "dtype": dtype}


def listed():
    return [
        # one decoded token through a hidden-size projection with bias
        _linear("linear 1 token", "linear", 1, 2048, 2048, bias=True),
        # a decode batch: the shared expert's down projection added to the residual stream
        _linear("linear 64 residual", "linear", 64, 512, 2048, residual=True),
        # an odd prompt through a dense feed-forward block's gated half, tanh GeLU
        _linear("linear 1031 geglu", "linear", 1031, 2816, 2112, act="geglu"),
        # training forward of a wide feed-forward projection, pre-activation kept
        _linear("linear 8192 gelu fp16", "linear", 8192, 2048, 8192, act="gelu", bias=True, save=True, dtype="fp16"),
        # a short fine-tuning batch of the same projection as the decoded token's
        _linear("linear backward 333", "linear_backward", 333, 2048, 2048, bias=True, dtype="fp16"),
        # a training batch: tanh-GeLU projection, every gradient
        _linear("linear backward 4096 gelu", "linear_backward", 4096, 2816, 2112, act="gelu_tanh", bias=True),
        # one decoded token: its 8 experts' gate and up
        _grouped("grouped 1 token swiglu", "grouped_linear", 1, 128, 8, 2048, 768, act="swiglu"),
        # a decode batch: the down projection of 128 experts
        _grouped("grouped 64 tokens down", "grouped_linear", 64, 128, 8, 768, 2048),
        # many small experts under skewed routing, several left empty, odd row count
        _grouped("grouped 2049 skewed fp16", "grouped_linear", 2049, 512, 10, 2048, 512, act="swiglu", skew=True,
                 dtype="fp16"),
        # a training prompt's gate and up, pre-activations kept for the backward pass
        _grouped("grouped 4096 swiglu", "grouped_linear", 4096, 128, 8, 2048, 768, act="swiglu", save=True),
        # gradients of a down projection with bias, 704 inner columns, odd row count
        _grouped("grouped backward 1031 down", "grouped_linear_backward", 1031, 128, 8, 704, 2816, bias=True),
        # gradients of the training prompt's gate and up
        _grouped("grouped backward 4096 swiglu", "grouped_linear_backward", 4096, 128, 8, 2048, 768, act="swiglu"),
    ]


def _log_int(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    """Rows over the whole range and odd; features in steps of 8, as models have them."""
    while True:
        op = rng.choice(["linear", "linear_backward", "grouped_linear", "grouped_linear_backward"])
        act, bias, dtype = rng.choice(ACTS), rng.random() < 0.5, rng.choice(["bf16", "fp16"])
        if op.startswith("linear"):
            c = _linear("", op, _log_int(rng, 1, 8192), _log_int(rng, 128, 8192, 8), _log_int(rng, 128, 8192, 8), act,
                        bias, op == "linear" and rng.random() < 0.5, op == "linear" and rng.random() < 0.3, dtype)
        else:
            experts = _log_int(rng, 8, 512)
            c = _grouped("", op, _log_int(rng, 1, 4096), experts, min(experts, rng.choice([1, 2, 4, 6, 8, 10])),
                         _log_int(rng, 256, 2816, 8), _log_int(rng, 64, 2816, 8), act, bias,
                         op == "grouped_linear" and rng.random() < 0.3, rng.random() < 0.3, dtype)
            blocks = _rows(c) // _block(c) + min(experts, _rows(c))
            if max(blocks, experts) * _wide(c) * c["in"] * 4 > 8e9:
                continue
        del c["name"]
        if work(c)["flops"] <= MAX_FLOPS:
            return c


# ------------------------------------------------------------------ sizes
def _wide(c):
    """Rows of W: the gate's and the up's for a gated pair."""
    return c["out"] * (2 if c["act"] in GATED else 1)


def _rows(c):
    return c["rows"] if "rows" in c else c["tokens"] * c["top_k"]


def _touched(c):
    """Experts that receive rows, expected (all of a token's experts differ)."""
    if "rows" in c:
        return 1.0
    E, K, T = c["experts"], c["top_k"], c["tokens"]
    if not c["skew"]:
        return E * (1.0 - (1.0 - K / E) ** T)
    p = [1.0 / (i + 1) ** 1.2 for i in range(E)]
    s = sum(p)
    return sum(1.0 - (1.0 - min(1.0, K * v / s)) ** T for v in p)


def work(case):
    """Each input read and each output written once; multiply-adds count two."""
    c = case
    S, n, wide, k, two = _rows(c), c["out"], _wide(c), c["in"], 2
    E = c.get("experts", 1)
    touched = _touched(c)
    offsets = 4 * (E + 1) if "experts" in c else 0
    if not c["op"].endswith("backward"):
        b = S * k + touched * wide * k + S * n + (touched * wide if c["bias"] else 0)
        b += S * n if c.get("residual") else 0
        b += S * wide if c["save"] else 0
        return {"bytes": two * b + offsets, "flops": 2.0 * S * wide * k}
    b = S * n + S * k + touched * wide * k + S * k + E * wide * k + (E * wide if c["bias"] else 0)
    b += S * wide if c["act"] != "none" else 0
    return {"bytes": two * b + offsets, "flops": 4.0 * S * wide * k}


# ----------------------------------------------------------------- inputs
def prepare(case, seed):
    c, dt = case, DTYPES[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dt)

    S, k, n, wide = _rows(c), c["in"], c["out"], _wide(c)
    s = {"case": c, "x": normal(S, k)}
    lead = () if "rows" in c else (c["experts"],)
    std = 0.9 / math.sqrt(k)  # pre-activations of about unit size
    if lead:  # expert by expert: no fp32 copy of a whole layer's weights
        s["w"] = torch.empty(*lead, wide, k, dtype=dt, device="cuda")
        step = max(1, (1 << 26) // (wide * k))
        for e in range(0, lead[0], step):
            s["w"][e:e + step] = normal(min(step, lead[0] - e), wide, k, std=std)
        scores = torch.randn(c["tokens"], lead[0], generator=g, device="cuda")
        if c["skew"]:  # Zipf(1.2) over the experts, by perturbed scores
            rank = torch.randperm(lead[0], generator=g, device="cuda") + 1
            gumbel = -torch.log(-torch.log(torch.rand(scores.shape, generator=g, device="cuda").clamp(1e-9, 1 - 1e-7)))
            scores = gumbel - 1.2 * torch.log(rank.float())
        ids = torch.topk(scores, c["top_k"], dim=1).indices.flatten()
        counts = torch.bincount(ids, minlength=lead[0])
        s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    else:
        s["w"] = normal(wide, k, std=std)
    if c["op"].endswith("backward"):
        s["dy"] = normal(S, n, std=0.1)
        s["preact"] = normal(S, wide, std=0.9) if c["act"] != "none" else None
    else:
        s["b"] = normal(*lead, wide, std=0.1) if c["bias"] else None
        s["r"] = normal(S, n) if c.get("residual") else None
    return s


# ------------------------------------------------------------- plain form
def _act(act, z):
    if act in GATED:
        g, u = z.chunk(2, dim=-1)
        return _act("silu" if act == "swiglu" else "gelu_tanh", g) * u
    if act == "relu":
        return z * (z > 0)
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _slope(act, z):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 0.134145 * z * z)


def _dz(act, dy, preact):
    dy = dy.float()
    if act == "none":
        return dy
    z = preact.float()
    if act not in GATED:
        return dy * _slope(act, z)
    inner = "silu" if act == "swiglu" else "gelu_tanh"
    g, u = z.chunk(2, dim=-1)
    return torch.cat([dy * u * _slope(inner, g), dy * _act(inner, g)], dim=-1)


def _block(c):
    """Rows of a block of the grouped form: near the mean group, so little is padded."""
    mean = _rows(c) / c["experts"]
    return 128 if mean >= 64 else 32 if mean >= 8 else 8


def _blocks(c, offsets):
    """Expert, rows and validity of blocks that together hold every group, none shared by two."""
    S, E, n = _rows(c), c["experts"], _block(c)
    o = offsets.long()
    per = (o[1:] - o[:-1] + n - 1) // n
    end = per.cumsum(0)
    b = torch.arange(S // n + min(E, S), device=o.device)
    e = torch.searchsorted(end, b, right=True).clamp(max=E - 1)
    row = (o[e] + (b - end[e] + per[e]) * n)[:, None] + torch.arange(n, device=o.device)
    return e, row, (b < end[-1])[:, None] & (row < o[e + 1][:, None])


def _gather(v, row, live):
    return v.float()[torch.where(live, row, 0)] * live[..., None]


def _scatter(S, row, live, v):
    out = torch.zeros(S + 1, v.shape[-1], device=v.device)
    out[torch.where(live, row, S).flatten()] = v.flatten(0, 1)
    return out[:S]


def _plain(s):
    c, x, w = s["case"], s["x"], s["w"]
    dt, S = x.dtype, _rows(c)
    if c["op"] == "linear":
        z = x.float() @ w.float().t()
        z = z + s["b"].float() if c["bias"] else z
        y = _act(c["act"], z)
        y = y + s["r"].float() if c["residual"] else y
        return (y.to(dt), z.to(dt)) if c["save"] else y.to(dt)
    if c["op"] == "linear_backward":
        dz = _dz(c["act"], s["dy"], s["preact"])
        out = (dz @ w.float()).to(dt), (dz.t() @ x.float()).to(dt)
        return (*out, dz.sum(0).to(dt)) if c["bias"] else out
    e, row, live = _blocks(c, s["offsets"])
    if c["op"] == "grouped_linear":
        z = torch.bmm(_gather(x, row, live), w[e].float().transpose(1, 2))
        z = z + s["b"].float()[e][:, None] if c["bias"] else z
        z = _scatter(S, row, live, z)
        y = _act(c["act"], z)
        return (y.to(dt), z.to(dt)) if c["save"] else y.to(dt)
    dz = _gather(_dz(c["act"], s["dy"], s["preact"]), row, live)
    dx = _scatter(S, row, live, torch.bmm(dz, w[e].float())).to(dt)
    dw = torch.zeros(w.shape, device=w.device).index_add_(0, e, torch.bmm(dz.transpose(1, 2), _gather(x, row, live)))
    if not c["bias"]:
        return dx, dw.to(dt)
    return dx, dw.to(dt), torch.zeros(w.shape[:2], device=w.device).index_add_(0, e, dz.sum(1)).to(dt)


def _package():
    if "senmoe" not in sys.modules:
        sys.path.insert(0, os.path.join(ROOT, "sen-mlx_b200"))
    import senmoe
    return senmoe


def _kernels(s):
    m, c = _package(), s["case"]
    if c["op"] == "linear":
        return m.linear(s["x"], s["w"], bias=s["b"], residual=s["r"], activation=c["act"], save_preact=c["save"])
    if c["op"] == "grouped_linear":
        return m.grouped_linear(s["x"], s["w"], s["offsets"], bias=s["b"], activation=c["act"], save_preact=c["save"])
    if c["op"] == "linear_backward":
        out = m.linear_backward(s["dy"], s["x"], s["w"], preact=s["preact"], activation=c["act"], bias=c["bias"])
    else:
        out = m.grouped_linear_backward(s["dy"], s["x"], s["w"], s["offsets"], preact=s["preact"],
                                        activation=c["act"], bias=c["bias"])
    return out if c["bias"] else out[:2]


def run(state):
    return _kernels(state) if own else _plain(state)


# ---------------------------------------------------------- in 64 bits
def _exact_act(act, z):
    if act in GATED:
        half = z.shape[-1] // 2
        return _exact_act({"swiglu": "silu", "geglu": "gelu_tanh"}[act], z[..., :half]) * z[..., half:]
    if act == "relu":
        return z.clamp(min=0)
    if act == "silu":
        return z * torch.special.expit(z)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    if act == "gelu_tanh":  # 0.5 (1 + tanh(a)) = expit(2a)
        return z * torch.special.expit(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3))
    return z


def exact(case, seed):
    """One group at a time in float64; the activation's gradient by differentiating its definition."""
    s = prepare(case, seed)
    c, x, w = case, s["x"], s["w"]
    ends = s["offsets"].tolist() if "offsets" in s else [0, _rows(c)]
    ws = w if "offsets" in s else w[None]
    if not c["op"].endswith("backward"):
        z = torch.zeros(_rows(c), _wide(c), dtype=torch.float64, device="cuda")
        for e in range(len(ends) - 1):
            part = slice(ends[e], ends[e + 1])
            if ends[e + 1] > ends[e]:
                z[part] = x[part].double() @ ws[e].double().t()
                if c["bias"]:
                    z[part] += (s["b"][e] if "offsets" in s else s["b"]).double()
        y = _exact_act(c["act"], z)
        if c.get("residual"):
            y = y + s["r"].double()
        return (y, z) if c["save"] else y
    dz = s["dy"].double()
    if c["act"] != "none":
        with torch.enable_grad():
            z = s["preact"].double().requires_grad_(True)
            dz = torch.autograd.grad(_exact_act(c["act"], z), z, dz)[0]
    dx = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    dw = torch.zeros(ws.shape, dtype=torch.float64, device="cuda")
    db = torch.zeros(ws.shape[:2], dtype=torch.float64, device="cuda")
    for e in range(len(ends) - 1):
        part = slice(ends[e], ends[e + 1])
        if ends[e + 1] > ends[e]:
            dx[part] = dz[part] @ ws[e].double()
            dw[e] = dz[part].t() @ x[part].double()
            db[e] = dz[part].sum(0)
    if "offsets" not in s:
        dw, db = dw[0], db[0]
    return (dx, dw, db) if c["bias"] else (dx, dw)
