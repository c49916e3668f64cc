"""Operators around feature tables: decoding features by dense layers, and keeping them in 8 bits.

Seven kinds of calls on three operators:

  linear        act(x W^T + b) + residual, forward alone (serving)
  linear_train  the same with the gradients of x, W, b and the residual
  linear8       the same from e4m3 rows of x and W, a scale each
  norm          root-mean-square norm of x + residual, in the input's type or as e4m3 rows with scales
  norm_train    the same with the gradients of x, residual and weight
  cache_write   an emptied hash map takes keys and their rows, which it keeps in 8 bits with a scale a row
  cache_read    rows of such a map by key, zeros for keys that it does not hold

With ``own`` false everything is computed by elementary torch operations in 32 bits; with ``own`` true by the calls that a
user makes of the ``ash`` package.
"""
import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
ACTIVATIONS = ("none", "relu", "silu", "gelu", "sin")
MOST_FLOPS = 2 * 8192 * 4096 * 4096
EPS = 1e-6


# ----------------------------------------------------------------------------------------- cases
def listed():
    return [
        # One query point of a decoder head: the smallest call, nothing but latency.
        {"name": "linear_point", "kind": "linear", "rows": 1, "inputs": 256, "outputs": 256, "type": "bf16",
         "activation": "relu", "bias": True, "residual": False, "omega": 1.0},
        # A handful of points through a wide layer: the weights are all there is to read.
        {"name": "linear_few", "kind": "linear", "rows": 4, "inputs": 4096, "outputs": 4096, "type": "bf16",
         "activation": "silu", "bias": True, "residual": True, "omega": 1.0},
        # A sine layer over a million sampled positions, in the type of the feature tables.
        {"name": "linear_sine_1m", "kind": "linear", "rows": 1_000_000, "inputs": 64, "outputs": 64, "type": "f32",
         "activation": "sin", "bias": True, "residual": False, "omega": 30.0},
        # A wide hidden layer over a batch: bound by the tensor cores.
        {"name": "linear_wide", "kind": "linear", "rows": 8192, "inputs": 4096, "outputs": 4096, "type": "bf16",
         "activation": "gelu", "bias": True, "residual": True, "omega": 1.0},
        # Training the first layer of a head on 16 features of the grid, an odd number of samples.
        {"name": "train_features", "kind": "linear_train", "rows": 262_147, "inputs": 16, "outputs": 64, "type": "f32",
         "activation": "silu", "bias": True, "residual": False, "omega": 1.0},
        # Training a residual hidden layer of that head over half a million samples.
        {"name": "train_hidden", "kind": "linear_train", "rows": 500_003, "inputs": 128, "outputs": 128, "type": "bf16",
         "activation": "relu", "bias": True, "residual": True, "omega": 1.0},
        # Training a layer that widens four times.
        {"name": "train_wide", "kind": "linear_train", "rows": 4096, "inputs": 1024, "outputs": 4096, "type": "f16",
         "activation": "gelu", "bias": True, "residual": False, "omega": 1.0},
        # The wide hidden layer served in 8 bits.
        {"name": "linear8_wide", "kind": "linear8", "rows": 8192, "inputs": 4096, "outputs": 4096, "type": "bf16",
         "activation": "gelu", "bias": True, "residual": False, "omega": 1.0},
        # The norm before it, adding the residual and writing its 8-bit operand.
        {"name": "norm_8bit", "kind": "norm", "rows": 8192, "width": 4096, "type": "bf16", "residual": True,
         "quantize": True},
        # Training the norm between two layers of a head, an odd number of samples, in 32 bits.
        {"name": "norm_train", "kind": "norm_train", "rows": 300_001, "width": 128, "type": "f32", "residual": True},
        # Feature rows of a scan's voxels into an emptied map, kept as e4m3.
        {"name": "cache_write_1m", "kind": "cache_write", "keys": 1_000_000, "capacity": 2_000_000, "dim": 3, "width": 32,
         "format": "e4m3", "hits": 1.0},
        # A large batch of look-ups in such a map, int8, half of them of voxels that were never seen.
        {"name": "cache_read_4m", "kind": "cache_read", "keys": 2_000_000, "queries": 4_000_003, "capacity": 2_500_000,
         "dim": 3, "width": 64, "format": "int8", "hits": 0.5},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, uniform over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "linear_train", "linear_train", "linear8", "norm", "norm_train",
                       "cache_write", "cache_read"])
    if kind.startswith("linear"):
        train = kind == "linear_train"
        inputs, outputs = _spread(rng, 3, 4096), _spread(rng, 1, 4096)
        if rng.random() < 0.5:      # as layers mostly are: whole multiples
            inputs, outputs = max(16, inputs // 16 * 16), max(16, outputs // 16 * 16)
        rows = _spread(rng, 1, 600_000)
        most = min(MOST_FLOPS // (6 if train else 2), 60_000_000_000)
        rows = max(1, min(rows, most // (inputs * outputs), 256_000_000 // (inputs + outputs)))
        kept = rng.choice(["bf16", "f16"]) if kind == "linear8" else rng.choice(["f32", "bf16", "f16"])
        activation = rng.choice(ACTIVATIONS)
        if train and kept == "f32" and activation == "relu":
            activation = "silu"     # a sum that 32 bits put on the other side of zero turns a whole gradient on or off
        omega = 30.0 if activation == "sin" and kept != "f16" and rng.random() < 0.5 else 1.0    # 30 leaves the range of f16 in sums
        return {"kind": kind, "rows": rows, "inputs": inputs, "outputs": outputs, "type": kept, "activation": activation,
                "bias": rng.random() < 0.7, "residual": rng.random() < 0.5, "omega": omega}
    if kind.startswith("norm"):
        width = _spread(rng, 8, 8192)
        case = {"kind": kind, "rows": min(_spread(rng, 1, 500_000), max(1, 40_000_000 // width)), "width": width,
                "type": rng.choice(["f32", "bf16", "f16"]), "residual": rng.random() < 0.6}
        if kind == "norm":
            case["quantize"] = rng.random() < 0.5
        return case
    width = rng.choice([1, 3, 4, 8, 16, 31, 32, 64, 100, 128, 256])
    keys = min(_spread(rng, 1, 2_000_000), 100_000_000 // width)
    case = {"kind": kind, "keys": keys, "capacity": int(keys * rng.uniform(1.0, 2.0)), "dim": rng.choice([1, 2, 3, 3, 3, 4]),
            "width": width, "format": rng.choice(["e4m3", "int8"]), "hits": 1.0}
    if kind == "cache_read":
        case["queries"] = min(_spread(rng, 1, 4_000_000), 200_000_000 // width)
        case["hits"] = round(rng.uniform(0.0, 1.0), 2)
    return case


# ----------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE)


def _layer(case, g):
    """Weights as layers are initialised: sine layers by the bound that keeps their phases of order one."""
    k, n = case["inputs"], case["outputs"]
    bound = math.sqrt(6.0 / k) / case["omega"] if case["activation"] == "sin" else math.sqrt(3.0 / k)
    uniform = lambda *shape: torch.rand(*shape, generator=g, device=DEVICE) * 2.0 - 1.0
    return uniform(n, k) * bound, uniform(n) * bound


def _quantized(v):
    """Rows as e4m3 codes and a scale each."""
    scale = (v.abs().amax(1) / 448.0).clamp_min(2.0**-126)
    return (v * (1.0 / scale)[:, None]).to(torch.float8_e4m3fn), scale


def _edge(n, dim):
    return max(2, math.ceil(n ** (1.0 / dim)))


def _distinct_keys(n, dim, g):
    """n different voxels in no order: a lattice block, its edge by the dimension."""
    i = torch.randperm(n, generator=g, device=DEVICE)
    edge = _edge(n, dim)
    columns = []
    for d in range(dim):
        columns.append(i % edge if d < dim - 1 else i)
        i = i // edge
    return torch.stack(columns, 1).int() - edge // 2


def _ash():
    at = os.path.abspath("torch-ash_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import ash
    import ash.mlp
    import ash.quant

    return ash


def prepare(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    s = {"case": case}
    if kind.startswith("linear"):
        m, k, n, t = case["rows"], case["inputs"], case["outputs"], TYPES[case["type"]]
        weight, bias = _layer(case, g)
        x = _normal(g, m, k)
        if kind == "linear8":
            s["x"], s["x_scale"] = _quantized(x)
            s["weight"], s["weight_scale"] = _quantized(weight)
        else:
            s["x"], s["weight"] = x.to(t), weight.to(t)
        s["bias"] = bias.to(t) if case["bias"] else None
        s["residual"] = _normal(g, m, n).to(t) if case["residual"] else None
        if kind == "linear_train":
            s["grad"] = _normal(g, m, n).to(t)
            for name in ("x", "weight", "bias", "residual"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
    elif kind.startswith("norm"):
        m, d, t = case["rows"], case["width"], TYPES[case["type"]]
        s["x"] = (_normal(g, m, d) * torch.exp(_normal(g, m, 1))).to(t)
        s["weight"] = (1.0 + 0.2 * _normal(g, d)).to(t)
        s["residual"] = _normal(g, m, d).to(t) if case["residual"] else None
        if kind == "norm_train":
            s["grad"] = _normal(g, m, d).to(t)
            s["grad_sum"] = _normal(g, m, d).to(t) if case["residual"] else None
            for name in ("x", "weight", "residual"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
    else:
        n, w = case["keys"], case["width"]
        s["keys"] = _distinct_keys(n, case["dim"], g)
        s["values"] = _normal(g, n, w) * torch.exp(_normal(g, n, 1))
        if kind == "cache_read":
            q = case["queries"]
            pick = torch.randint(0, n, (q,), generator=g, device=DEVICE)
            s["queries"] = s["keys"][pick].contiguous()
            absent = torch.rand(q, generator=g, device=DEVICE) >= case["hits"]
            s["queries"][:, 0] += absent.int() * (_edge(n, case["dim"]) + 7)      # beyond the block
        if own:
            ash = _ash()
            s["map"] = ash.HashMap(case["dim"], w, case["capacity"], torch.device(DEVICE, torch.cuda.current_device()),
                                   value_formats=case["format"])
            if kind == "cache_read":
                s["map"].insert(s["keys"], s["values"])
        elif kind == "cache_read":
            s["table"] = _plain_store(s["keys"], s["values"], case["format"])
        if kind == "cache_read":
            del s["keys"], s["values"]
    return s


# ----------------------------------------------------------------------------------------- plain forms
def _activation(z, name, omega):
    """act(z) and act'(z)."""
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).to(z.dtype)
    if name == "silu":
        p = 1.0 / (1.0 + torch.exp(-z))
        return z * p, p * (1.0 + z * (1.0 - p))
    if name == "gelu":
        c = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * c, c + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if name == "sin":
        return torch.sin(omega * z), omega * torch.cos(omega * z)
    return z, torch.ones_like(z)


def _float(t):
    return None if t is None else t.detach().float()


def _plain_linear(s):
    case = s["case"]
    x, weight, bias, residual = (_float(s[name]) for name in ("x", "weight", "bias", "residual"))
    if case["kind"] == "linear8":
        x, weight = x * s["x_scale"][:, None], weight * s["weight_scale"][:, None]
    t = TYPES[case["type"]]
    z = x @ weight.T
    if bias is not None:
        z = z + bias
    y, slope = _activation(z, case["activation"], case["omega"])
    if residual is not None:
        y = y + residual
    if case["kind"] != "linear_train":
        return {"y": y.to(t)}
    dz = _float(s["grad"]) * slope
    out = {"y": y.to(t), "grad_x": (dz @ weight).to(t), "grad_weight": (dz.T @ x).to(t)}
    if bias is not None:
        out["grad_bias"] = dz.sum(0).to(t)
    if residual is not None:
        out["grad_residual"] = s["grad"]
    return out


def _plain_norm(s):
    case = s["case"]
    t = TYPES[case["type"]]
    x, weight, residual = _float(s["x"]), _float(s["weight"]), _float(s["residual"])
    v = x if residual is None else x + residual
    rstd = torch.rsqrt((v * v).mean(1, keepdim=True) + EPS)
    y = v * rstd * weight
    out = {}
    if case["kind"] == "norm" and case["quantize"]:
        out["codes"], out["scales"] = _quantized(y)
    else:
        out["y"] = y.to(t)
    if residual is not None:
        out["sum"] = v.to(t)
    if case["kind"] == "norm_train":
        dy = _float(s["grad"])
        gw = dy * weight
        dx = rstd * (gw - v * rstd * rstd * (gw * v).mean(1, keepdim=True))
        if residual is not None:
            dx = dx + _float(s["grad_sum"])
            out["grad_residual"] = dx.to(t)
        out["grad_x"] = dx.to(t)
        out["grad_weight"] = (dy * v * rstd).sum(0).to(t)
    return out


def _packed(keys):
    """One whole number a key, alike for alike keys only."""
    p = torch.zeros(keys.shape[0], dtype=torch.int64, device=keys.device)
    bits = 64 // keys.shape[1] if keys.shape[1] > 1 else 32
    for d in range(keys.shape[1]):
        p = (p << bits) + keys[:, d].long()
    return p


def _plain_store(keys, values, fmt):
    most = 448.0 if fmt == "e4m3" else 127.0
    scale = (values.abs().amax(1) / most).clamp_min(2.0**-126)
    v = values * (1.0 / scale)[:, None]
    codes = v.to(torch.float8_e4m3fn) if fmt == "e4m3" else torch.round(v).to(torch.int8)
    packed, order = torch.sort(_packed(keys))
    return packed, order, codes, scale


def _plain_fetch(table, queries):
    packed, order, codes, scale = table
    q = _packed(queries)
    at = torch.searchsorted(packed, q).clamp_max(packed.shape[0] - 1)
    found = packed[at] == q
    row = order[at]
    rows = codes.view(torch.uint8)[row].view(codes.dtype).float() * scale[row][:, None]
    return {"rows": torch.where(found[:, None], rows, torch.zeros_like(rows)), "found": found}


# ----------------------------------------------------------------------------------------- a pass
def run(state):
    s, case = state, state["case"]
    kind = case["kind"]
    if not own:
        if kind.startswith("linear"):
            return _plain_linear(s)
        if kind.startswith("norm"):
            return _plain_norm(s)
        table = _plain_store(s["keys"], s["values"], case["format"]) if kind == "cache_write" else s["table"]
        return _plain_fetch(table, s["keys"] if kind == "cache_write" else s["queries"])
    ash = _ash()
    if kind in ("linear", "linear_train"):
        y = ash.mlp.fused_linear(s["x"], s["weight"], s["bias"], activation=case["activation"], residual=s["residual"],
                                 omega=case["omega"])
        if kind == "linear":
            return {"y": y}
        names = [name for name in ("x", "weight", "bias", "residual") if s[name] is not None]
        grads = torch.autograd.grad(y, [s[name] for name in names], s["grad"])
        return {"y": y.detach(), **{"grad_" + name: grad for name, grad in zip(names, grads)}}
    if kind == "linear8":
        y = ash.mlp.fused_linear(ash.quant.QuantizedRows(s["x"], s["x_scale"]),
                                 ash.quant.QuantizedRows(s["weight"], s["weight_scale"]), s["bias"],
                                 activation=case["activation"], residual=s["residual"], omega=case["omega"],
                                 dtype=TYPES[case["type"]])
        return {"y": y}
    if kind.startswith("norm"):
        quantize = kind == "norm" and case["quantize"]
        got = ash.mlp.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS, quantize=quantize)
        y, v = got if s["residual"] is not None else (got, None)
        out = {"codes": y.codes, "scales": y.scales} if quantize else {"y": y.detach()}
        if v is not None:
            out["sum"] = v.detach()
        if kind == "norm_train":
            names = [name for name in ("residual", "x", "weight") if s[name] is not None]
            outputs, upstream = ([y], [s["grad"]]) if v is None else ([y, v], [s["grad"], s["grad_sum"]])
            grads = torch.autograd.grad(outputs, [s[name] for name in names], upstream)
            out.update({"grad_" + name: grad for name, grad in zip(names, grads)})
        return out
    m = s["map"]
    if kind == "cache_write":
        m.clear()
        m.insert(s["keys"], s["values"])
    found, rows = m.find(s["keys"] if kind == "cache_write" else s["queries"], return_indices=False, return_values=True)
    return {"rows": rows, "found": found}


# ----------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind.startswith("linear"):
        m, k, n, e = case["rows"], case["inputs"], case["outputs"], BYTES[case["type"]]
        train, extra = kind == "linear_train", n * case["bias"] + m * n * case["residual"]
        if kind == "linear8":
            nbytes = m * k + n * k + 4 * (m + n) + e * (m * n + extra)
        else:
            nbytes = e * (m * k + n * k + m * n + extra)
        if train:       # the upstream gradient is read; each input's gradient is written, the residual's is the upstream one
            nbytes += e * (m * n + m * k + n * k + n * case["bias"])
        return {"bytes": nbytes, "flops": (6 if train else 2) * m * n * k}
    if kind.startswith("norm"):
        m, d, e = case["rows"], case["width"], BYTES[case["type"]]
        nbytes = e * (m * d * (3 if case["residual"] else 1) + d)                       # x, residual, sum; weight
        nbytes += m * d + 4 * m if kind == "norm" and case["quantize"] else e * m * d    # the normed rows
        if kind == "norm_train":     # upstream gradients read; the gradient of x, which the residual's is too, and the weight's
            nbytes += e * (m * d * (3 if case["residual"] else 2) + d)
        return {"bytes": nbytes, "flops": (10 if kind == "norm_train" else 4) * m * d}
    w, key = case["width"], 4 * case["dim"]
    slot = 16 if case["dim"] < 4 else 32
    if kind == "cache_write":        # keys, rows, slots and their emptying, codes and scales written; all of it read back
        n = case["keys"]
        return {"bytes": n * (key + 4 * w + 2 * slot + 4 + w + 4) + n * (key + slot + w + 4 + 4 * w + 1), "flops": 4 * n * w}
    q, hit = case["queries"], int(case["queries"] * case["hits"])
    return {"bytes": q * (key + slot + 4 * w + 1) + hit * (w + 4), "flops": hit * w}


# ----------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """What a pass returns for these inputs, from the definitions in 64 bits."""
    s = prepare(case, seed)
    kind = case["kind"]
    wide = lambda t: None if t is None else t.detach().to(torch.float64)
    if kind.startswith("linear"):
        x, w = wide(s["x"]), wide(s["weight"])
        if kind == "linear8":
            x, w = x * wide(s["x_scale"]).unsqueeze(1), w * wide(s["weight_scale"]).unsqueeze(1)
        z = torch.einsum("mk,nk->mn", x, w)
        if s["bias"] is not None:
            z += wide(s["bias"])
        a, om = case["activation"], case["omega"]
        y = {"none": lambda: z, "relu": lambda: z.clamp_min(0.0), "silu": lambda: z * torch.sigmoid(z),
             "gelu": lambda: z * 0.5 * torch.erfc(-z / math.sqrt(2.0)), "sin": lambda: torch.sin(z * om)}[a]()
        if s["residual"] is not None:
            y = y + wide(s["residual"])
        out = {"y": y}
        if kind == "linear_train":
            sig = torch.sigmoid(z)
            d = {"none": lambda: 1.0, "relu": lambda: (z > 0).double(), "silu": lambda: sig + z * sig * (1.0 - sig),
                 "gelu": lambda: 0.5 * torch.erfc(-z / math.sqrt(2.0)) + z * torch.exp(-z * z / 2.0) / math.sqrt(2.0 * math.pi),
                 "sin": lambda: torch.cos(z * om) * om}[a]()
            dz = wide(s["grad"]) * d
            out["grad_x"] = torch.einsum("mn,nk->mk", dz, w)
            out["grad_weight"] = torch.einsum("mn,mk->nk", dz, x)
            if s["bias"] is not None:
                out["grad_bias"] = dz.sum(0)
            if s["residual"] is not None:
                out["grad_residual"] = wide(s["grad"])
        return out
    if kind.startswith("norm"):
        v = wide(s["x"]) if s["residual"] is None else wide(s["x"]) + wide(s["residual"])
        rms = torch.sqrt(v.square().sum(1) / case["width"] + EPS).unsqueeze(1)
        unit, w = v / rms, wide(s["weight"])
        out = {}
        if kind == "norm" and case["quantize"]:
            out["codes"], out["scales"] = None, ((unit * w).abs().max(1).values / 448.0).clamp_min(2.0**-126)
        else:
            out["y"] = unit * w
        if s["residual"] is not None:
            out["sum"] = v
        if kind == "norm_train":
            gu = wide(s["grad"]) * w
            dx = (gu - unit * (gu * unit).sum(1, keepdim=True) / case["width"]) / rms
            if s["residual"] is not None:
                dx = dx + wide(s["grad_sum"])
                out["grad_residual"] = dx
            out["grad_x"] = dx
            out["grad_weight"] = (wide(s["grad"]) * unit).sum(0)
        return out
    return None      # codes of stored rows are whole numbers by 32-bit rules: nothing that 64 bits would say better
