"""Dense layers in 8 bits and the norm over groups of channels, as cases that can be timed and checked.

* ``group``       group norm with an activation, channels last: ``act((x - mean) rstd w + b)`` with the statistics of a
                  sample's positions and of a group's channels; forward, or a training step (gradients of x, w and b);
* ``int8``        a linear layer of 8-bit integers, one scale a row of x and one a row of the weight:
                  ``act(s t (q p^T) + b) + r``; the rows are x's, or those of x's norm with a residual;
* ``checkpoint``  a training step of a linear layer, ``act(x W^T + b) + r`` and the gradients of x, W and b, that keeps x
                  and the activation's argument in 8 bits: blocks of 32 values with a power of two as their step.

``run`` computes them in plain torch operations in 32 bits, or, where ``own`` is set, through the package's entry points.
"""
import math

import torch

own = False

GROUP_EPS = 1e-5
RMS_EPS = 1e-6
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
SMALLEST = 2.0 ** -100  # an 8-bit row whose largest value is less takes this one's scale
ACTS = ("none", "relu", "silu", "gelu")


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one small sample between two layers: launches
        {"name": "group_small", "kind": "group", "samples": 1, "places": 16, "channels": 64, "groups": 8, "dtype": "bf16",
         "act": "silu", "step": False},
        # node features of a batch of molecules, 40 nodes x 25 rows of 128 channels each, in training
        {"name": "group_nodes_fp32_step", "kind": "group", "samples": 32, "places": 1000, "channels": 128, "groups": 8,
         "dtype": "fp32", "act": "silu", "step": True},
        # no size a multiple of anything, groups of 30 channels, in training
        {"name": "group_ragged_step", "kind": "group", "samples": 5, "places": 777, "channels": 330, "groups": 11,
         "dtype": "fp16", "act": "gelu", "step": True},
        # grids of 64 x 64, evaluated
        {"name": "group_forward", "kind": "group", "samples": 8, "places": 4096, "channels": 512, "groups": 32,
         "dtype": "bf16", "act": "silu", "step": False},
        # grids of 128 x 128 in training
        {"name": "group_step", "kind": "group", "samples": 4, "places": 16384, "channels": 512, "groups": 32,
         "dtype": "bf16", "act": "silu", "step": True},
        # one token through norm and first layer of a feed-forward block: the weights are read once
        {"name": "int8_token", "kind": "int8", "rows": 1, "inner": 4096, "outer": 16384, "dtype": "bf16", "act": "silu",
         "bias": True, "residual": False, "norm": True},
        # no size a multiple of anything, results in 32 bits
        {"name": "int8_ragged", "kind": "int8", "rows": 777, "inner": 1234, "outer": 1531, "dtype": "fp32", "act": "gelu",
         "bias": True, "residual": True, "norm": False},
        # a long batch through norm and first layer
        {"name": "int8_forward", "kind": "int8", "rows": 8192, "inner": 4096, "outer": 16384, "dtype": "bf16",
         "act": "silu", "bias": True, "residual": False, "norm": True},
        # a small step: launches
        {"name": "checkpoint_small_step", "kind": "checkpoint", "rows": 48, "inner": 256, "outer": 512, "dtype": "bf16",
         "act": "silu", "bias": True, "residual": False},
        # no size a multiple of anything
        {"name": "checkpoint_ragged_step", "kind": "checkpoint", "rows": 777, "inner": 1234, "outer": 1531,
         "dtype": "fp16", "act": "gelu", "bias": True, "residual": True},
        # a linear layer over a batch's edges, in the model's own precision
        {"name": "checkpoint_edges_fp32_step", "kind": "checkpoint", "rows": 36800, "inner": 384, "outer": 128,
         "dtype": "fp32", "act": "none", "bias": True, "residual": False},
        # the first layer of a feed-forward block over a long batch
        {"name": "checkpoint_step", "kind": "checkpoint", "rows": 8192, "inner": 4096, "outer": 16384, "dtype": "bf16",
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
        kind = rng.choice(["group", "int8", "checkpoint"])
        case = {"kind": kind, "dtype": rng.choice(["fp32", "bf16", "fp16"]), "act": rng.choice(ACTS)}
        if kind == "group":
            groups = _log(rng, 1, 64)
            each = _log(rng, 1, 256)
            if rng.random() < 0.5:  # most groups are of round sizes, some are not
                each = max(8, each // 8 * 8)
            case.update(samples=_log(rng, 1, 128), places=_log(rng, 1, 40000), channels=groups * each, groups=groups,
                        step=rng.random() < 0.6)
            if case["places"] * each < 32:  # statistics of a few values: gradients that cancel
                continue
            if case["step"] and case["act"] == "relu":  # (of many values some lie within a rounding of its corner)
                continue
        else:
            case.update(rows=_log(rng, 1, 40000), inner=_log(rng, 64, 16384), outer=_log(rng, 64, 16384),
                        bias=rng.random() < 0.7, residual=rng.random() < 0.5)
            if rng.random() < 0.6:
                case.update(inner=max(64, case["inner"] // 64 * 64), outer=max(64, case["outer"] // 64 * 64))
            if kind == "int8":  # (the norm's rounding may take a value across an integer's border: no 32-bit results)
                case["norm"] = case["dtype"] != "fp32" and rng.random() < 0.5
            elif case["dtype"] == "fp32":  # (nor with arguments kept in steps: the product's rounding may take one to the next)
                case["act"] = "none"
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

    if case["kind"] == "group":
        n, p, c = case["samples"], case["places"], case["channels"]
        spread, mean = normal(c, scale=0.3, shift=1.0), normal(c)  # channels have their own ranges
        s = {"case": case, "x": normal(n, p, c) * spread + mean, "w": normal(c, scale=0.2, shift=1.0), "b": normal(c, scale=0.2)}
        if case["step"]:
            s["g"] = normal(n, p, c)
            s.update({k: s[k].requires_grad_() for k in ("x", "w", "b")})
        return s
    rows, k, n = case["rows"], case["inner"], case["outer"]
    s = {"case": case, "x": normal(rows, k), "w": normal(n, k, scale=k ** -0.5),
         "b": normal(n, scale=0.2) if case["bias"] else None, "r": normal(rows, n) if case["residual"] else None}
    if case["kind"] == "int8":  # the weights are quantised once, as a serving program does
        if case["norm"]:
            s["rx"], s["wn"] = normal(rows, k, scale=2.0), normal(k, scale=0.2, shift=1.0)
        s["wq"], s["ws"] = _to_int8(s.pop("w").double())
    else:
        s["g"] = normal(rows, n)
        s.update({k: s[k].requires_grad_() for k in ("x", "w", "b", "r") if s[k] is not None})
    return s


def _to_int8(y):
    """Rows of y (64 bits: which integer a value falls to) as integers of -127 to 127 and one fp32 scale a row."""
    most = y.abs().amax(-1).clamp_min(SMALLEST)
    return torch.round(127 * y / most[:, None]).to(torch.int8), (most / 127).float()


# ------------------------------------------------------------------- runs
def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"group": _plain_group, "int8": _plain_int8, "checkpoint": _plain_checkpoint}[state["case"]["kind"]](state)


def _run_own(s):
    from maloq_amd.dense import linear_act, linear_quantized, quantize_rows
    from maloq_amd.norm import group_norm, rms_norm_quantized
    case = s["case"]
    if case["kind"] == "group":
        y = group_norm(s["x"], case["groups"], s["w"], s["b"], GROUP_EPS, act=case["act"])
        if not case["step"]:
            return {"y": y}
        return {"y": y, **dict(zip(("gx", "gw", "gb"), torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["g"])))}
    if case["kind"] == "int8":
        out = {}
        if case["norm"]:
            q, scale, out["h"] = rms_norm_quantized(s["x"], s["wn"], RMS_EPS, residual=s["rx"], dtype=torch.int8)
        else:
            q, scale = quantize_rows(s["x"], dtype=torch.int8)
        return {"y": linear_quantized(q, scale, s["wq"], s["ws"], s["b"], act=case["act"], residual=s["r"],
                                      dtype=TYPES[case["dtype"]]), **out}
    y = linear_act(s["x"], s["w"], s["b"], act=case["act"], residual=s["r"], checkpoint=torch.int8)
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


def _plain_group(s):
    case, dt = s["case"], s["x"].dtype
    n, p, c, g = case["samples"], case["places"], case["channels"], case["groups"]
    x, w, b = s["x"].float().view(n, p, g, c // g), s["w"].float().view(g, -1), s["b"].float().view(g, -1)
    x = x - x.mean((1, 3), keepdim=True)
    rstd = torch.rsqrt(x.square().mean((1, 3), keepdim=True) + GROUP_EPS)
    xh = x * rstd
    z = xh * w + b
    out = {"y": _act(z, case["act"]).view(n, p, c).to(dt)}
    if case["step"]:
        u = s["g"].float().view(n, p, g, c // g) * _act_slope(z, case["act"])
        uw = u * w
        gx = rstd * (uw - uw.mean((1, 3), keepdim=True) - xh * (uw * xh).mean((1, 3), keepdim=True))
        out.update(gx=gx.view(n, p, c).to(dt), gw=(u * xh).sum((0, 1)).view(c).to(dt), gb=u.sum((0, 1)).view(c).to(dt))
    return out


def _plain_int8(s):
    act, dt, out = s["case"]["act"], s["x"].dtype, {}
    x = s["x"].double()
    if s["case"]["norm"]:
        x = x + s["rx"].double()
        out["h"] = x.to(dt)
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + RMS_EPS) * s["wn"].double()
    q, scale = _to_int8(x)
    z = (q.float() @ s["wq"].float().T) * scale[:, None] * s["ws"]
    if s["b"] is not None:
        z = z + s["b"].float()
    y = _act(z, act)
    if s["r"] is not None:
        y = y + s["r"].float()
    return {"y": y.to(dt), **out}


def _kept(v, sign=False):
    """v (fp32 rows) as 8 bits give it back: blocks of 32 in steps of a power of two, the largest between 63 and 126
    steps; sign: what is not zero stays so."""
    rows, n = v.shape
    b = torch.nn.functional.pad(v, (0, -n % 32)).view(rows, -1, 32)
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True))  # m of 1/2 to 1
    e = e + (m >= 126.5 / 128).to(e.dtype) - 7
    q = torch.round(torch.ldexp(b, -e))
    if sign:
        q = torch.where((q == 0) & (b > 0), 1.0, q)
    return torch.ldexp(q, e).view(rows, -1)[:, :n]


def _plain_checkpoint(s):
    act, dt = s["case"]["act"], s["x"].dtype
    x, w, g = s["x"].float(), s["w"].float(), s["g"].float()
    z = x @ w.T
    if s["b"] is not None:
        z = z + s["b"].float()
    y = _act(z, act)
    if s["r"] is not None:
        y = y + s["r"].float()
    dz = g * _act_slope(_kept(z, act == "relu"), act)
    out = {"y": y.to(dt), "gx": (dz @ w).to(dt), "gw": (dz.T @ _kept(x)).to(dt)}
    if s["b"] is not None:
        out["gb"] = dz.sum(0).to(dt)
    return out


# ------------------------------------------------------------------- work
def work(case):
    b = BYTES[case["dtype"]]
    if case["kind"] == "group":
        values, c = case["samples"] * case["places"] * case["channels"], case["channels"]
        if case["step"]:  # x, g, w and b in; y, gx, gw and gb out
            return {"bytes": b * (4 * values + 4 * c), "flops": 30 * values}
        return {"bytes": b * (2 * values + 2 * c), "flops": 12 * values}
    rows, k, n = case["rows"], case["inner"], case["outer"]
    each = rows * n * (1 + case["residual"]) + n * case["bias"]
    if case["kind"] == "int8":  # x, the residual stream and its sum, the weights and their scales
        norm = 2 * rows * k + k if case["norm"] else 0
        return {"bytes": b * (rows * k + norm + each) + n * k + 4 * n, "flops": 2 * rows * n * k}
    return {"bytes": b * (2 * rows * k + 2 * n * k + each + rows * n + n * case["bias"]), "flops": 6 * rows * n * k}


# ------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.detach().double() for k, v in s.items() if torch.is_tensor(v)}
    act = {"none": lambda z: z, "relu": torch.nn.functional.relu, "silu": torch.nn.functional.silu,
           "gelu": torch.nn.functional.gelu}[case["act"]]
    if case["kind"] == "group":
        x, w, b = (d[k].requires_grad_(case["step"]) for k in ("x", "w", "b"))
        y = act(torch.nn.functional.group_norm(x.transpose(1, 2), case["groups"], w, b, GROUP_EPS)).transpose(1, 2)
        if not case["step"]:
            return {"y": y}
        grads = torch.autograd.grad(y, (x, w, b), d["g"])
        return {"y": y.detach(), **dict(zip(("gx", "gw", "gb"), grads))}
    if case["kind"] == "int8":
        x, out = d["x"], {}
        if case["norm"]:
            out["h"] = x = x + d["rx"]
            x = d["wn"] * x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + RMS_EPS).sqrt()
        most = x.abs().max(-1, keepdim=True).values.clamp_min(SMALLEST)
        q = torch.round(127 * x / most)
        y = torch.nn.functional.linear(q * most / 127, d["wq"] * d["ws"][:, None], d.get("b"))
        y = act(y)
        return {"y": y + d["r"] if "r" in d else y, **out}
    z = torch.nn.functional.linear(d["x"], d["w"], d.get("b"))
    y = act(z) + d["r"] if "r" in d else act(z)
    at = _in_steps(z)
    if case["act"] == "relu":
        at = torch.where(z > 0, 1.0, 0.0).double()
    at.requires_grad_()
    dz = torch.autograd.grad(act(at), at, d["g"])[0]
    out = {"y": y, "gx": torch.mm(dz, d["w"]), "gw": torch.mm(dz.mT.contiguous(), _in_steps(d["x"]))}
    if "b" in d:
        out["gb"] = dz.sum(0)
    return out


def _in_steps(v):
    """Each 32 of a row at the nearest multiples of 2^(E - 6), the largest of them in 2^E (126.5 / 128) [1, 2)."""
    out = []
    for block in v.split(32, -1):
        top = block.abs().max(-1, keepdim=True).values
        step = torch.exp2(torch.floor(torch.log2((top * (128 / 126.5)).clamp_min(1e-300))) - 6)
        out.append(torch.round(block / step) * step)
    return torch.cat(out, -1)
