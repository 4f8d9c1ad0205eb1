"""The operators of the feed-forward sublayer as cases that can be timed and checked.

* ``norm``    root-mean-square norm of a residual stream: ``h = x + r``, ``y = h / rms(h) * w``; forward, or a
              training step (the gradients of x, which are r's too, and of w);
* ``linear``  ``y = act(x W^T + b) + r``, forward or a training step (the gradients of x, W and b; r's is the
              given one itself);
* ``quant``   the serving form in 8 bits: the norm's output as e4m3 with one scale a row, times an e4m3 weight with one
              scale an output channel, bias, activation and residual: ``h`` and ``y``.

``run`` computes them in plain torch operations in 32 bits, or, where ``own`` is set, through the package's entry points.
"""
import math

import torch

own = False

EPS = 1e-6
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
E4M3_MAX = 448.0
SMALLEST = 2.0 ** -100  # a row whose largest value is less takes this one's scale


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one token's norm between two layers: a launch
        {"name": "norm_token", "kind": "norm", "rows": 1, "width": 4096, "dtype": "bf16", "step": False},
        # the norms of a long ragged batch, evaluated
        {"name": "norm_forward", "kind": "norm", "rows": 8191, "width": 4096, "dtype": "bf16", "step": False},
        # node features of a batch of molecules, each degree's channels a row: 1280 nodes x 25 rows of 128, in training
        {"name": "norm_nodes_fp32_step", "kind": "norm", "rows": 32000, "width": 128, "dtype": "fp32", "step": True},
        # wide rows in training
        {"name": "norm_wide_step", "kind": "norm", "rows": 4093, "width": 8192, "dtype": "bf16", "step": True},
        # one token through the first layer of a feed-forward block: the weights are read once
        {"name": "linear_token", "kind": "linear", "rows": 1, "inner": 4096, "outer": 16384, "dtype": "bf16",
         "act": "silu", "bias": True, "residual": False, "step": False},
        # a few sequences a step, the layer that adds to the residual stream
        {"name": "linear_few_rows", "kind": "linear", "rows": 24, "inner": 5120, "outer": 5120, "dtype": "fp16",
         "act": "none", "bias": True, "residual": True, "step": False},
        # no size a multiple of anything, in training
        {"name": "linear_ragged_step", "kind": "linear", "rows": 777, "inner": 1234, "outer": 1531, "dtype": "fp16",
         "act": "gelu", "bias": True, "residual": True, "step": True},
        # the radial function's wide first layer over a batch's edges, in the model's own precision
        {"name": "linear_edges_fp32_step", "kind": "linear", "rows": 36800, "inner": 384, "outer": 128, "dtype": "fp32",
         "act": "silu", "bias": True, "residual": False, "step": True},
        # the first layer of a feed-forward block over a long batch, evaluated
        {"name": "linear_forward", "kind": "linear", "rows": 8192, "inner": 4096, "outer": 16384, "dtype": "bf16",
         "act": "gelu", "bias": True, "residual": False, "step": False},
        # a square layer with its residual in training, a ragged batch
        {"name": "linear_step", "kind": "linear", "rows": 4133, "inner": 4096, "outer": 4096, "dtype": "bf16",
         "act": "silu", "bias": True, "residual": True, "step": True},
        # one token served in 8 bits
        {"name": "quant_token", "kind": "quant", "rows": 1, "inner": 4096, "outer": 16384, "dtype": "bf16",
         "act": "silu", "bias": True, "residual": False},
        # a long batch served in 8 bits
        {"name": "quant_forward", "kind": "quant", "rows": 8192, "inner": 4096, "outer": 16384, "dtype": "bf16",
         "act": "silu", "bias": True, "residual": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {}
    for c in listed():
        w, m = work(c), most.setdefault((c["kind"], c["dtype"] == "fp32"), {"bytes": 0, "flops": 0})
        m.update(bytes=max(m["bytes"], w["bytes"]), flops=max(m["flops"], w["flops"]))
    while True:
        kind = rng.choice(["norm", "norm", "linear", "linear", "linear", "quant"])
        case = {"kind": kind, "rows": _log(rng, 1, 40000), "dtype": rng.choice(["fp32", "bf16", "fp16"])}
        if kind == "norm":
            case.update(width=_log(rng, 16, 16384), step=rng.random() < 0.5)
            if rng.random() < 0.5:
                case["width"] = max(16, case["width"] // 16 * 16)
        else:
            case.update(inner=_log(rng, 64, 16384), outer=_log(rng, 64, 16384), bias=rng.random() < 0.7,
                        act=rng.choice(["none", "relu", "silu", "gelu"]), residual=rng.random() < 0.5)
            if rng.random() < 0.6:  # most widths are round, some are not
                case.update(inner=max(64, case["inner"] // 64 * 64), outer=max(64, case["outer"] // 64 * 64))
            if kind == "linear":
                case["step"] = rng.random() < 0.5
            elif case["dtype"] == "fp32":
                case["dtype"] = "bf16"
        w, m = work(case), most[kind, case["dtype"] == "fp32"]
        if w["bytes"] <= m["bytes"] and w["flops"] <= m["flops"]:
            return case


# ----------------------------------------------------------------- inputs
def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def prepare(case, seed):
    dev, dt = _device(), TYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=gen, device=dev) * scale + shift).to(dt)

    rows = case["rows"]
    if case["kind"] == "norm":
        c = case["width"]
        s = {"case": case, "x": normal(rows, c), "r": normal(rows, c, scale=2.0), "w": normal(c, scale=0.2, shift=1.0)}
        if case["step"]:
            s.update(g=normal(rows, c), gh=normal(rows, c))
            s.update({k: s[k].requires_grad_() for k in ("x", "r", "w")})
        return s
    k, n = case["inner"], case["outer"]
    s = {"case": case, "x": normal(rows, k), "w": normal(n, k, scale=k ** -0.5),
         "b": normal(n, scale=0.2) if case["bias"] else None, "r": normal(rows, n) if case["residual"] else None}
    if case["kind"] == "quant":  # the weights are quantised once, as a serving program does
        s["rx"], s["wn"] = normal(rows, k, scale=2.0), normal(k, scale=0.2, shift=1.0)
        s["wq"], s["ws"] = _to_e4m3(s.pop("w").float())
    elif case["step"]:
        s["g"] = normal(rows, n)
        s.update({k: s[k].requires_grad_() for k in ("x", "w", "b", "r") if s[k] is not None})
    return s


def _to_e4m3(y):
    """Rows of y as e4m3 numbers and one fp32 scale a row: the largest of a row becomes 448."""
    scale = y.abs().amax(-1).clamp_min(SMALLEST) / E4M3_MAX
    return (y / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale.float()


# ------------------------------------------------------------------- runs
def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"norm": _plain_norm, "linear": _plain_linear, "quant": _plain_quant}[state["case"]["kind"]](state)


def _run_own(s):
    from maloq_amd.dense import linear_act, linear_quantized
    from maloq_amd.norm import rms_norm, rms_norm_quantized
    case = s["case"]
    if case["kind"] == "norm":
        y, h = rms_norm(s["x"], s["w"], EPS, residual=s["r"])
        if not case["step"]:
            return {"y": y, "h": h}
        gx, gw = torch.autograd.grad((y, h), (s["x"], s["w"]), (s["g"], s["gh"]))
        return {"y": y, "h": h, "gx": gx, "gw": gw}
    if case["kind"] == "quant":
        q, scale, h = rms_norm_quantized(s["x"], s["wn"], EPS, residual=s["rx"])
        y = linear_quantized(q, scale, s["wq"], s["ws"], s["b"], act=case["act"], residual=s["r"],
                             dtype=TYPES[case["dtype"]])
        return {"y": y, "h": h}
    y = linear_act(s["x"], s["w"], s["b"], act=case["act"], residual=s["r"])
    if not case["step"]:
        return {"y": y}
    names = [k for k in ("x", "w", "b") if s[k] is not None]
    return {"y": y, **{"g" + k: v for k, v in zip(names, torch.autograd.grad(y, [s[k] for k in names], s["g"]))}}


def _act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return z * 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return torch.ones_like(z)


def _plain_norm(s):
    dt = s["x"].dtype
    h, w = s["x"].float() + s["r"].float(), s["w"].float()
    rstd = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
    n = h * rstd
    out = {"y": (n * w).to(dt), "h": h.to(dt)}
    if s["case"]["step"]:
        g = s["g"].float()
        u = g * w
        out["gx"] = (rstd * (u - n * (u * n).mean(-1, keepdim=True)) + s["gh"].float()).to(dt)
        out["gw"] = (g * n).sum(0).to(dt)
    return out


def _plain_linear(s):
    act, dt = s["case"]["act"], s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.T
    if s["b"] is not None:
        z = z + s["b"].float()
    y = _act(z, act)
    if s["r"] is not None:
        y = y + s["r"].float()
    out = {"y": y.to(dt)}
    if s["case"]["step"]:
        dz = s["g"].float() * _act_slope(z, act)
        out.update(gx=(dz @ w).to(dt), gw=(dz.T @ x).to(dt))
        if s["b"] is not None:
            out["gb"] = dz.sum(0).to(dt)
    return out


def _plain_quant(s):
    act, dt = s["case"]["act"], s["x"].dtype
    h = s["x"].float() + s["rx"].float()
    # which of two e4m3 numbers a value falls to is settled in 64 bits
    h64 = h.double()
    q, scale = _to_e4m3(h64 * torch.rsqrt(h64.square().mean(-1, keepdim=True) + EPS) * s["wn"].double())
    z = (q.float() @ s["wq"].float().T) * scale[:, None] * s["ws"]
    if s["b"] is not None:
        z = z + s["b"].float()
    y = _act(z, act)
    if s["r"] is not None:
        y = y + s["r"].float()
    return {"y": y.to(dt), "h": h.to(dt)}


# ------------------------------------------------------------------- work
def work(case):
    rows, b = case["rows"], BYTES[case["dtype"]]
    if case["kind"] == "norm":
        c = case["width"]
        if case["step"]:  # x, r, g, gh and w in; y, h, gx and gw out
            return {"bytes": b * (7 * rows * c + 2 * c), "flops": 16 * rows * c}
        return {"bytes": b * (4 * rows * c + c), "flops": 5 * rows * c}
    k, n = case["inner"], case["outer"]
    each = rows * n * (1 + case["residual"]) + n * case["bias"]
    if case["kind"] == "quant":
        return {"bytes": b * (3 * rows * k + k + each) + n * k + 4 * n, "flops": 2 * rows * n * k}
    if case["step"]:  # the gradients beside what the forward moves
        return {"bytes": b * (2 * rows * k + 2 * n * k + each + rows * n + n * case["bias"]), "flops": 6 * rows * n * k}
    return {"bytes": b * (rows * k + n * k + each), "flops": 2 * rows * n * k}


# ------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.detach().double() for k, v in s.items() if torch.is_tensor(v)}
    act = {"none": lambda z: z, "relu": torch.nn.functional.relu, "silu": torch.nn.functional.silu,
           "gelu": torch.nn.functional.gelu}[case.get("act", "none")]

    def norm(h, w):
        return w * h / (h.pow(2).sum(-1, keepdim=True) / h.shape[-1] + EPS).sqrt()

    if case["kind"] == "norm":
        x, w = d["x"].requires_grad_(), d["w"].requires_grad_()
        h = x + d["r"]
        y = norm(h, w)
        out = {"y": y.detach(), "h": h.detach()}
        if case["step"]:
            out["gx"], out["gw"] = torch.autograd.grad([y, h], [x, w], [d["g"], d["gh"]])
        return out
    if case["kind"] == "quant":
        h = d["x"] + d["rx"]
        y = norm(h, d["wn"])
        step = y.abs().max(-1, keepdim=True).values / E4M3_MAX
        z = (_nearest_e4m3(y / step) * step) @ (d["wq"] * d["ws"][:, None]).T
        y = act(z if s["b"] is None else z + d["b"])
        return {"y": y if s["r"] is None else y + d["r"], "h": h}
    leaves = [d[k].requires_grad_() for k in ("x", "w", "b") if k in d]
    y = act(torch.nn.functional.linear(d["x"], d["w"], d.get("b")))
    y = y + d["r"] if "r" in d else y
    if not case["step"]:
        return {"y": y.detach()}
    grads = torch.autograd.grad(y, leaves, d["g"])
    return {"y": y.detach(), **{"g" + k: v for k, v in zip([k for k in ("x", "w", "b") if k in d], grads)}}


def _nearest_e4m3(v):
    """v (of at most 448) at four significant bits, ties to the even one, in steps of 2^-9 at the least."""
    e = torch.frexp(v)[1].clamp_min(-5) - 4  # v = m 2^e', 1/2 <= m < 1: steps of 2^(e' - 4)
    return torch.ldexp(torch.round(torch.ldexp(v, -e)), e)
