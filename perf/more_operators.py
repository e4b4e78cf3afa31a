"""Cases of the RMS norm and of the products over 8-bit rows, forward and
backward, in their plain form (elementary torch operations, fp32) and through
the package's entry points:

* ``rms_norm``: h = x + residual in 16 bits, y = h / sqrt(mean(h^2) + eps) * g,
  with g the weight (or 1 + weight), y in 16 bits, in 8 bits with scales, or
  both from one reading;
* ``rms_norm_backward``: dx and dweight from dy and the residual stream's dh;
* ``linear8`` / ``grouped_linear8``: y = act(x W^T + b) + r over 8-bit x and W
  with a scale for every 32 elements along the contraction, dense or one W per
  expert over rows in expert order; a gated pair (swiglu, geglu: W holds the
  gate's rows, then the up's) with its output in 8 bits with scales is the
  first half of a feed-forward block;
* ``linear8_input_grad`` / ``grouped_linear8_input_grad``: dx = dz W with
  dz = dy act'(z) in 8 bits with scales and W^T in 8 bits.

8 bits: elements in e4m3, and for every 32 of a row the scale 2^e with the
smallest e for which the largest magnitude is at most 448 * 2^e.  Outputs in 8
bits are returned as they are held: the elements, and the scales.
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
BLOCK = 32  # elements of a scale
EPS = 1e-6
MAX_FLOPS = 2.8e11  # the largest listed case's
MAX_NORM = 1.0e8    # elements of the largest listed norm


def _norm(name, op, rows, hidden, residual=False, eight=False, sixteen=True, unit=False, dtype="bf16"):
    return {"name": name, "op": op, "rows": rows, "hidden": hidden, "residual": residual, "eight": eight,
            "sixteen": sixteen, "unit": unit, "dtype": dtype}


def _linear(name, op, rows, inner, out, act="none", bias=False, residual=False, save=False, eight=False,
            dtype="bf16"):
    return {"name": name, "op": op, "rows": rows, "in": inner, "out": out, "act": act, "bias": bias,
            "residual": residual, "save": save, "eight": eight, "dtype": dtype}


def _grouped(name, op, tokens, experts, top_k, inner, out, act="none", bias=False, save=False, eight=False,
             skew=False, dtype="bf16"):
    return {"name": name, "op": op, "tokens": tokens, "experts": experts, "top_k": top_k, "in": inner, "out": out,
            "act": act, "bias": bias, "residual": False, "save": save, "eight": eight, "skew": skew, "dtype": dtype}


def listed():
    return [
        # one decoded token: the residual add and the norm before the block, for the router and for its 8-bit experts
        _norm("norm 1 token", "rms_norm", 1, 2048, residual=True, eight=True),
        # a prompt's tokens at the same place, every output
        _norm("norm 4096 tokens", "rms_norm", 4096, 2048, residual=True, eight=True),
        # a long batch of a wider model with weights stored around zero, 16 bits only, odd row count
        _norm("norm 32767 fp16", "rms_norm", 32767, 2816, unit=True, dtype="fp16"),
        # a short fine-tuning batch, the residual stream's gradient added
        _norm("norm backward 1031", "rms_norm_backward", 1031, 2816, residual=True, unit=True),
        # a training batch
        _norm("norm backward 32768", "rms_norm_backward", 32768, 2048, residual=True, dtype="fp16"),
        # a decode batch: the shared expert's down projection added to the residual stream
        _linear("linear8 64 residual", "linear8", 64, 512, 2048, residual=True),
        # an odd prompt through a dense feed-forward block's first half, pre-activations kept
        _linear("linear8 1031 geglu fp16", "linear8", 1031, 2816, 2112, act="geglu", save=True, eight=True, dtype="fp16"),
        # a wide feed-forward projection with bias over a long batch
        _linear("linear8 8192 gelu", "linear8", 8192, 2048, 8192, act="gelu", bias=True),
        # one decoded token: its 8 experts' gate and up
        _grouped("grouped8 1 token swiglu", "grouped_linear8", 1, 128, 8, 2048, 768, act="swiglu", eight=True),
        # a training prompt's gate and up, pre-activations kept for the backward pass
        _grouped("grouped8 4096 swiglu", "grouped_linear8", 4096, 128, 8, 2048, 768, act="swiglu", save=True, eight=True),
        # a short fine-tuning batch: input gradient of a dense block's first half, fp16
        _linear("input grad 333 geglu", "linear8_input_grad", 333, 2816, 2112, act="geglu", dtype="fp16"),
        # input gradient of the training prompt's gate and up
        _grouped("input grad 4096 swiglu", "grouped_linear8_input_grad", 4096, 128, 8, 2048, 768, act="swiglu"),
    ]


def _log_int(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    """Rows over the whole range and odd; features in whole scale blocks where
    they are held in 8 bits, in steps of 8 or odd elsewhere."""
    while True:
        op = rng.choice(["rms_norm", "rms_norm_backward", "linear8", "grouped_linear8", "linear8_input_grad",
                         "grouped_linear8_input_grad"])
        dtype = rng.choice(["bf16", "fp16"])
        if op.startswith("rms_norm"):
            eight = op == "rms_norm" and rng.random() < 0.5
            step = BLOCK if eight else rng.choice([8, 8, 1])
            c = _norm("", op, _log_int(rng, 1, 32768), _log_int(rng, 64, 8192, step), rng.random() < 0.6, eight,
                      not eight or rng.random() < 0.5, rng.random() < 0.4, dtype)
            del c["name"]
            if c["rows"] * c["hidden"] > MAX_NORM:
                continue
            return c
        grad = op.endswith("grad")
        act, bias, save = rng.choice(ACTS + GATED), not grad and rng.random() < 0.3, not grad and rng.random() < 0.3
        eight = not grad and rng.random() < 0.5
        # what is contracted is in whole blocks: in for the product, the rows of W for its gradient
        out_step = BLOCK if eight or grad else rng.choice([8, 1])
        in_step = 8 if grad else BLOCK
        if op.startswith("linear8"):
            c = _linear("", op, _log_int(rng, 1, 8192), _log_int(rng, 128, 8192, in_step),
                        _log_int(rng, 128, 8192, out_step), act, bias, not grad and rng.random() < 0.4, save, eight,
                        dtype)
        else:
            experts = _log_int(rng, 8, 512)
            c = _grouped("", op, _log_int(rng, 1, 4096), experts, min(experts, rng.choice([1, 2, 4, 6, 8, 10])),
                         _log_int(rng, 256, 2816, in_step), _log_int(rng, 64, 2816, out_step), act, bias, save, eight,
                         rng.random() < 0.3, dtype)
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
    c, held8 = case, 1.0 + 1.0 / BLOCK
    if c["op"].startswith("rms_norm"):
        n, h = c["rows"] * c["hidden"], c["hidden"]
        if c["op"] == "rms_norm":  # x, (residual and h), y, y8
            each = 2 + (4 if c["residual"] else 0) + (2 if c["sixteen"] else 0) + (held8 if c["eight"] else 0)
            return {"bytes": each * n + 2 * h, "flops": 5.0 * n}
        # dy, h, (dh), dx; dweight
        return {"bytes": (6 + (2 if c["residual"] else 0)) * n + 4 * h, "flops": 10.0 * n}
    S, n, wide, k = _rows(c), c["out"], _wide(c), c["in"]
    weights = _touched(c) * wide * k * held8
    offsets = 4 * (c["experts"] + 1) if "experts" in c else 0
    flops = 2.0 * S * wide * k
    if c["op"].endswith("grad"):  # dy, z, W^T, dx
        return {"bytes": 2 * S * n + (2 * S * wide if c["act"] != "none" else 0) + weights + 2 * S * k + offsets,
                "flops": flops}
    b = S * k * held8 + weights + S * n * (held8 if c["eight"] else 2)
    b += 2 * _touched(c) * wide if c["bias"] else 0
    b += 2 * S * n if c["residual"] else 0
    b += 2 * S * wide if c["save"] else 0
    return {"bytes": b + offsets, "flops": flops}


# ----------------------------------------------------------------- inputs
def _to8(v):
    """v [..., n] -> (elements e4m3 [..., n], scales e8m0 [..., n / 32])."""
    g = v.unflatten(-1, (-1, BLOCK))
    m, e = torch.frexp(g.abs().amax(-1))            # largest = m * 2^e, 1/2 <= m < 1; 448 = 7/8 * 2^9
    e = (e - 9 + (m > 0.875)).clamp(min=-127)
    codes = (g * torch.exp2(-e.to(v.dtype))[..., None]).flatten(-2).to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _from8(codes, scales, dtype=torch.float32):
    return (codes.to(dtype).unflatten(-1, (-1, BLOCK)) * scales.to(dtype)[..., None]).flatten(-2)


def prepare(case, seed):
    c, dt = case, DTYPES[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dt)

    s = {"case": c}
    if c["op"].startswith("rms_norm"):
        n, h = c["rows"], c["hidden"]
        s["x"] = normal(n, h, std=1.5)
        s["weight"] = (normal(h, std=0.2).float() + (0.0 if c["unit"] else 1.0)).to(dt)
        if c["op"] == "rms_norm":
            s["residual"] = normal(n, h) if c["residual"] else None
        else:
            s["dy"] = normal(n, h, std=0.1)
            s["dh"] = normal(n, h, std=0.1) if c["residual"] else None
        return s
    S, k, n, wide = _rows(c), c["in"], c["out"], _wide(c)
    grad = c["op"].endswith("grad")
    lead = () if "rows" in c else (c["experts"],)
    # W [wide, in], or its transpose for the gradient; pre-activations of about unit size
    shape, std = ((k, wide), 0.9 / math.sqrt(wide)) if grad else ((wide, k), 0.9 / math.sqrt(k))
    if lead:  # some experts at a time: no fp32 copy of a whole layer's weights
        codes = torch.empty(*lead, *shape, dtype=torch.float8_e4m3fn, device="cuda")
        scales = torch.empty(*lead, shape[0], shape[1] // BLOCK, dtype=torch.float8_e8m0fnu, device="cuda")
        step = max(1, (1 << 26) // (wide * k))
        for e in range(0, lead[0], step):
            part = _to8(normal(min(step, lead[0] - e), *shape, std=std).float())
            codes[e:e + step], scales[e:e + step] = part
        s["w"] = codes, scales
        scores = torch.randn(c["tokens"], lead[0], generator=g, device="cuda")
        if c["skew"]:  # Zipf(1.2) over the experts, by perturbed scores
            rank = torch.randperm(lead[0], generator=g, device="cuda") + 1
            gumbel = -torch.log(-torch.log(torch.rand(scores.shape, generator=g, device="cuda").clamp(1e-9, 1 - 1e-7)))
            scores = gumbel - 1.2 * torch.log(rank.float())
        ids = torch.topk(scores, c["top_k"], dim=1).indices.flatten()
        counts = torch.bincount(ids, minlength=lead[0])
        s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    else:
        s["w"] = _to8(normal(*shape, std=std).float())
    if grad:
        s["dy"] = normal(S, n, std=0.1)
        s["preact"] = normal(S, wide, std=0.9) if c["act"] != "none" else None
    else:
        s["x"] = _to8(normal(S, k).float())
        s["b"] = normal(*lead, wide, std=0.1) if c["bias"] else None
        s["r"] = normal(S, n) if c["residual"] else None
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


def _product(c, x, w, offsets):
    """x [S, n] times each row's W^T, in fp32."""
    if offsets is None:
        return x @ _from8(*w).t()
    # blocks that together hold every group, none shared by two: expert, rows, validity
    S, E, n = _rows(c), c["experts"], _block(c)
    o = offsets.long()
    per = (o[1:] - o[:-1] + n - 1) // n
    end = per.cumsum(0)
    b = torch.arange(S // n + min(E, S), device=o.device)
    e = torch.searchsorted(end, b, right=True).clamp(max=E - 1)
    row = (o[e] + (b - end[e] + per[e]) * n)[:, None] + torch.arange(n, device=o.device)
    live = (b < end[-1])[:, None] & (row < o[e + 1][:, None])
    xs = x[torch.where(live, row, 0)] * live[..., None]
    ws = _from8(w[0].view(torch.uint8)[e].view(torch.float8_e4m3fn), w[1].view(torch.uint8)[e].view(torch.float8_e8m0fnu))
    z = torch.bmm(xs, ws.transpose(1, 2))
    out = torch.zeros(S + 1, z.shape[-1], device=z.device)
    out[torch.where(live, row, S).flatten()] = z.flatten(0, 1)
    return out[:S], e, row, live


def _plain(s):
    c = s["case"]
    dt = DTYPES[c["dtype"]]
    if c["op"] == "rms_norm":
        h = (s["x"].float() + s["residual"].float()).to(dt) if c["residual"] else s["x"]
        hf, g = h.float(), s["weight"].float() + (1.0 if c["unit"] else 0.0)
        y = hf * torch.rsqrt((hf * hf).mean(-1, keepdim=True) + EPS) * g
        return (y.to(dt) if c["sixteen"] else None, *(_to8(y) if c["eight"] else ()), h if c["residual"] else None)
    if c["op"] == "rms_norm_backward":
        hf, g = s["x"].float(), s["weight"].float() + (1.0 if c["unit"] else 0.0)
        r = torch.rsqrt((hf * hf).mean(-1, keepdim=True) + EPS)
        dy = s["dy"].float()
        dn = dy * g
        dx = r * (dn - hf * r * r * (dn * hf).mean(-1, keepdim=True))
        dx = dx + s["dh"].float() if c["residual"] else dx
        return dx.to(dt), (dy * hf * r).sum(0).to(dt)
    offsets = s.get("offsets")
    if c["op"].endswith("grad"):
        dz = _from8(*_to8(_dz(c["act"], s["dy"], s["preact"])))
        dx = _product(c, dz, s["w"], offsets)
        return (dx if offsets is None else dx[0]).to(dt)
    z = _product(c, _from8(*s["x"]), s["w"], offsets)
    b = s["b"].float() if c["bias"] else None
    if offsets is not None:
        z, e, row, live = z
        if c["bias"]:
            expert = torch.zeros(_rows(c) + 1, dtype=torch.long, device=z.device)
            expert[torch.where(live, row, _rows(c)).flatten()] = e[:, None].expand(row.shape).flatten()
            b = b[expert[:-1]]
    z = z + b if c["bias"] else z
    y = _act(c["act"], z)
    y = y + s["r"].float() if c["residual"] else y
    return (*(_to8(y) if c["eight"] else (y.to(dt),)), *((z.to(dt),) if c["save"] else ()))


def _package():
    if "senmoe" not in sys.modules:
        sys.path.insert(0, os.path.join(ROOT, "sen-mlx_b200"))
    import senmoe
    return senmoe


def _kernels(s):
    m, c = _package(), s["case"]
    if c["op"] == "rms_norm":
        n = m.rms_norm(s["x"], s["weight"], EPS, residual=s["residual"], unit_offset=c["unit"],
                       sixteen_bit=c["sixteen"], eight_bit=c["eight"])
        return (n.y, *(n.y8 if c["eight"] else ()), n.h if c["residual"] else None)
    if c["op"] == "rms_norm_backward":
        return m.rms_norm_backward(s["dy"], s["x"], s["weight"], EPS, dh=s["dh"], unit_offset=c["unit"])
    w = m.Rows8(*s["w"])
    if c["op"] == "linear8_input_grad":
        return m.linear8_input_grad(s["dy"], w, preact=s["preact"], activation=c["act"])
    if c["op"] == "grouped_linear8_input_grad":
        return m.grouped_linear8_input_grad(s["dy"], w, s["offsets"], preact=s["preact"], activation=c["act"])
    x, dt = m.Rows8(*s["x"]), DTYPES[c["dtype"]]
    if c["op"] == "linear8":
        y = m.linear8(x, w, bias=s["b"], residual=s["r"], activation=c["act"], save_preact=c["save"],
                      eight_bit=c["eight"], dtype=dt)
    else:
        y = m.grouped_linear8(x, w, s["offsets"], bias=s["b"], activation=c["act"], save_preact=c["save"],
                              eight_bit=c["eight"], dtype=dt)
    y, z = y if c["save"] else (y, None)
    return (*(y if c["eight"] else (y,)), *((z,) if c["save"] else ()))


def run(state):
    return _kernels(state) if own else _plain(state)


# ---------------------------------------------------------- in 64 bits
def _exact8(v):
    """The elements and the scales that stand for v, from the definition, in float64."""
    groups = v.reshape(*v.shape[:-1], -1, BLOCK)
    largest = groups.abs().max(-1).values
    e = torch.ceil(torch.log2(largest / 448.0))
    e = torch.where(448.0 * torch.exp2(e - 1) >= largest, e - 1, e)  # the logarithm's last bit
    e = torch.where(448.0 * torch.exp2(e) < largest, e + 1, e).clamp(min=-127)
    scaled = groups / torch.exp2(e)[..., None]
    step = torch.exp2(torch.floor(torch.log2(scaled.abs().clamp(min=2.0 ** -6))) - 3)  # 3 bits behind the leading one
    return (torch.round(scaled / step) * step).reshape(v.shape), torch.exp2(e)


def _exact_held(codes, scales):
    return (codes.double().reshape(*scales.shape, BLOCK) * scales.double()[..., None]).reshape(codes.shape)


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
    """One group at a time in float64; gradients by differentiating the definitions."""
    c, s = case, prepare(case, seed)
    if c["op"].startswith("rms_norm"):
        g = s["weight"].double() + (1.0 if c["unit"] else 0.0)
        if c["op"] == "rms_norm":
            h = s["x"].double()
            if c["residual"]:  # h is held in 16 bits, and its norm taken
                h = (h + s["residual"].double()).to(DTYPES[c["dtype"]]).double()
            y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + EPS) * g
            return (y if c["sixteen"] else None, *(_exact8(y) if c["eight"] else ()), h if c["residual"] else None)
        with torch.enable_grad():
            h, g = s["x"].double().requires_grad_(True), g.requires_grad_(True)
            y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + EPS) * g
            dx, dw = torch.autograd.grad(y, (h, g), s["dy"].double())
        return (dx + s["dh"].double() if c["residual"] else dx), dw
    S, grouped = _rows(c), "offsets" in s
    ends = s["offsets"].tolist() if grouped else [0, S]
    codes, scales = s["w"] if grouped else (s["w"][0][None], s["w"][1][None])
    if c["op"].endswith("grad"):
        a = s["dy"].double()
        if c["act"] != "none":
            with torch.enable_grad():
                z = s["preact"].double().requires_grad_(True)
                a = torch.autograd.grad(_exact_act(c["act"], z), z, a)[0]
        a = _exact_held(*_exact8(a))
    else:
        a = _exact_held(*s["x"])
    out = torch.zeros(S, codes.shape[1], dtype=torch.float64, device="cuda")
    for e in range(len(ends) - 1):
        if ends[e + 1] > ends[e]:
            out[ends[e]:ends[e + 1]] = a[ends[e]:ends[e + 1]] @ _exact_held(codes[e], scales[e]).t()
            if not c["op"].endswith("grad") and c["bias"]:
                out[ends[e]:ends[e + 1]] += (s["b"][e] if grouped else s["b"]).double()
    if c["op"].endswith("grad"):
        return out
    y = _exact_act(c["act"], out)
    if c["residual"]:
        y = y + s["r"].double()
    return (*(_exact8(y) if c["eight"] else (y,)), *((out,) if c["save"] else ()))
