"""Cases of the INT8 decoder-layer operators: the root-mean-square norm that answers in 8 bits, the codes of
a tensor's rows, the 8-bit matrix product with a scale for each token and channel, and cross attention to an
encoder's states.

A decoder that reads image features runs them in this order: norm -> product (queries) -> cross attention
over the features' keys and values (made once for each image by the same product) -> codes -> product.
Every case is one pass through one of them.  `own` chooses between the plain form, in elementary torch
operations of 32 bits, and the calls of spinnv2_b200.transformer.
"""

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6


# ------------------------------------------------------------------ cases
def _norm(name, rows, width, dtype, residual):
    return {"name": name, "op": "rms_norm_i8", "rows": rows, "width": width, "dtype": dtype, "residual": residual}


def _codes(name, rows, width, dtype):
    return {"name": name, "op": "quantize_rows_i8", "rows": rows, "width": width, "dtype": dtype}


def _linear(name, m, k, n, dtype, bias, act):
    return {"name": name, "op": "linear_i8", "m": m, "k": k, "n": n, "dtype": dtype, "bias": bias, "act": act}


def _cross(name, batch, queries, heads, kv_heads, width, grid_h, grid_w, dtype, mask):
    return {"name": name, "op": "cross_attention", "batch": batch, "queries": queries, "heads": heads,
            "kv_heads": kv_heads, "width": width, "grid_h": grid_h, "grid_w": grid_w, "dtype": dtype, "mask": mask}


def listed():
    return [
        # One token of one request enters a layer: latency.
        _norm("norm one token", 1, 2048, "bf16", True),
        # The prompts of a batch enter a layer: memory bandwidth.
        _norm("norm prompts", 16384, 4096, "bf16", True),
        # The attention's answer of one step of an odd batch, on its way into the output product.
        _codes("codes one step", 37, 1000, "fp16"),
        # The encoder's features of 256 images (7 x 7 pixels, 2048 channels, as ResNet-50 and ResNet-101
        # leave them in this runtime), on their way into the product that makes keys and values.
        _codes("codes image features", 12544, 2048, "fp32"),
        # One token's projection: the weights' bytes and the launch.
        _linear("linear one token", 1, 2048, 2048, "bf16", False, "none"),
        # The classifier of the ResNets (2048 -> 1000) for an odd batch, in 32 bits.
        _linear("linear classifier", 37, 2048, 1000, "fp32", True, "none"),
        # Keys and values of 256 images' features in one product.
        _linear("linear image features", 12544, 2048, 4096, "bf16", True, "none"),
        # One token looks at one image: latency.
        _cross("attention one token", 1, 1, 16, 16, 64, 7, 7, "bf16", "none"),
        # One step of a batch with shared key heads, over encoder states of every length from none to 4096.
        _cross("attention batch step", 64, 1, 32, 8, 128, 1, 4096, "fp16", "lengths"),
        # Prompts over images of several sizes, padded to one grid: the valid keys have holes.
        _cross("attention padded grids", 16, 77, 12, 12, 64, 14, 14, "bf16", "grid"),
        # A detection decoder's object queries over a feature map, in 32 bits.
        _cross("attention object queries", 2, 100, 8, 8, 32, 25, 34, "fp32", "none"),
        # Long prompts over a large feature map with shared key heads: matrix units.
        _cross("attention long", 8, 2048, 16, 4, 128, 64, 64, "bf16", "none"),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _cost(case):
    w = work(case)
    rate = 60e12 if case["op"] == "cross_attention" and case["dtype"] == "fp32" else 1.6e15
    return max(w["bytes"] / 6.5e12, w["flops"] / rate)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["rms_norm_i8", "quantize_rows_i8", "linear_i8", "linear_i8", "cross_attention",
                         "cross_attention", "cross_attention"])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        if op == "rms_norm_i8":
            case = _norm("", _spread(rng, 1, 16384), _spread(rng, 64, 16384), dtype, rng.random() < 0.7)
        elif op == "quantize_rows_i8":
            case = _codes("", _spread(rng, 1, 16384), _spread(rng, 64, 16384), dtype)
        elif op == "linear_i8":
            case = _linear("", _spread(rng, 1, 16384), _spread(rng, 64, 16384), _spread(rng, 64, 16384), dtype,
                           rng.random() < 0.5, rng.choice(["none", "none", "relu", "silu"]))
        else:
            kv_heads = rng.choice([1, 2, 4, 8, 12, 16])
            case = _cross("", _spread(rng, 1, 64), rng.choice([1, _spread(rng, 1, 2048), _spread(rng, 1, 2048)]),
                          kv_heads * rng.choice([1, 1, 2, 4, 8]), kv_heads, rng.choice([32, 40, 64, 64, 80, 96, 128, 128]),
                          _spread(rng, 1, 64), _spread(rng, 1, 128), dtype, rng.choice(["none", "lengths", "grid"]))
            scores = case["batch"] * case["heads"] * case["queries"] * case["grid_h"] * case["grid_w"]
            if scores > 8 * 16 * 2048 * 4096:  # what the plain form has to hold
                continue
        del case["name"]
        if _cost(case) <= most:
            return case


# ------------------------------------------------------------------ what a pass cannot do without
def _lengths(case):
    """Valid keys of each batch entry, before their order is drawn: from none (where the batch has more than
    one entry) to all of them."""
    b, n = case["batch"], case["grid_h"] * case["grid_w"]
    return [n] if b == 1 else [i * n // (b - 1) for i in range(b)]


def _extents(case):
    """Valid rows and columns of each entry's grid, before their order is drawn; one entry has nothing."""
    b, h, w = case["batch"], case["grid_h"], case["grid_w"]
    if b == 1:
        return [(h, max(1, w - w // 4))]
    return [(0, 0)] + [(1 + (7 * i) % h, 1 + (5 * i) % w) for i in range(1, b)]


def _keys(case):
    """Valid keys of the whole batch."""
    if case["mask"] == "lengths":
        return sum(_lengths(case))
    if case["mask"] == "grid":
        return sum(h * w for h, w in _extents(case))
    return case["batch"] * case["grid_h"] * case["grid_w"]


def work(case):
    op, size = case["op"], SIZE[case["dtype"]]
    if op == "rms_norm_i8":
        n = case["rows"] * case["width"]
        return {"bytes": n * (size * (3 if case["residual"] else 1) + 1) + 4 * case["rows"] + size * case["width"],
                "flops": 6 * n}
    if op == "quantize_rows_i8":
        n = case["rows"] * case["width"]
        return {"bytes": n * (size + 1) + 4 * case["rows"], "flops": 3 * n}
    if op == "linear_i8":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": m * k + n * k + m * n * size + 4 * m + 4 * n + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    q = case["batch"] * case["queries"] * case["heads"] * case["width"]
    kv = _keys(case) * case["kv_heads"] * case["width"]
    return {"bytes": size * (2 * q + 2 * kv),
            "flops": 4 * case["queries"] * case["heads"] * case["width"] * _keys(case)}


# ------------------------------------------------------------------ inputs
def _activations(rows, width, dtype, g):
    """Rows as a residual stream has them: unit spread, a few channels eight times as wide."""
    x = torch.randn(rows, width, generator=g, device="cuda")
    wide = torch.randperm(width, generator=g, device="cuda")[: max(1, width // 512)]
    x[:, wide] *= 8.0
    return x.to(dtype)


def _pitched(rows, width):
    """Codes as the framework's quantisers lay them out: rows start on 16-byte boundaries."""
    return torch.empty(rows, (width + 15) // 16 * 16, dtype=torch.int8, device="cuda")[:, :width]


def _random_codes(rows, width, g):
    q = _pitched(rows, width)
    q.copy_((torch.randn(rows, width, generator=g, device="cuda") * 32.0).round_().clamp_(-127, 127))
    return q


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype, op = TYPES[case["dtype"]], case["op"]
    s = {"case": case, "dtype": dtype}
    if op in ("rms_norm_i8", "quantize_rows_i8"):
        rows, width = case["rows"], case["width"]
        s["x"] = _activations(rows, width, dtype, g)
        s["codes"] = _pitched(rows, width)
        s["scale"] = torch.empty(rows, device="cuda")
        s["values"] = torch.empty(rows, width, dtype=torch.bfloat16, device="cuda")
        if op == "rms_norm_i8":
            s["weight"] = (1.0 + 0.1 * torch.randn(width, generator=g, device="cuda")).to(dtype)
            s["residual"] = torch.randn(rows, width, generator=g, device="cuda").to(dtype) if case["residual"] else None
            s["sum"] = torch.empty_like(s["x"]) if case["residual"] else None
    elif op == "linear_i8":
        m, k, n = case["m"], case["k"], case["n"]
        s["a"], s["w"] = _random_codes(m, k, g), _random_codes(n, k, g)
        s["a_scale"] = 0.02 + 0.03 * torch.rand(m, generator=g, device="cuda")
        s["w_scale"] = (0.5 + torch.rand(n, generator=g, device="cuda")) / (32.0 * math.sqrt(k))
        s["bias"] = torch.randn(n, generator=g, device="cuda") if case["bias"] else None
        s["out"] = torch.empty(m, n, dtype=dtype, device="cuda")
    else:
        b, lq, hq, hk, d = case["batch"], case["queries"], case["heads"], case["kv_heads"], case["width"]
        gh, gw = case["grid_h"], case["grid_w"]
        lk = gh * gw
        s["q"] = (1.5 * torch.randn(b, lq, hq, d, generator=g, device="cuda")).to(dtype)
        # Keys and values lie side by side, as one product leaves them.
        kv = torch.randn(b, lk, 2, hk, d, generator=g, device="cuda").to(dtype)
        s["lengths"] = s["mask"] = None
        if case["mask"] == "lengths":
            order = torch.randperm(b, generator=g, device="cuda")
            s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")[order].contiguous()
            # What lies behind an entry's last state was never written.
            behind = torch.arange(lk, device="cuda")[None, :] >= s["lengths"][:, None]
            kv.masked_fill_(behind[:, :, None, None, None], float("nan"))
        elif case["mask"] == "grid":
            order = torch.randperm(b, generator=g, device="cuda")
            ext = torch.tensor(_extents(case), dtype=torch.int32, device="cuda")[order]
            rows = torch.arange(gh, device="cuda")[None, :, None] < ext[:, 0, None, None]
            cols = torch.arange(gw, device="cuda")[None, None, :] < ext[:, 1, None, None]
            s["mask"] = (rows & cols).reshape(b, lk).contiguous()
        s["k"], s["v"] = kv[:, :, 0], kv[:, :, 1]
        s["out"] = torch.empty_like(s["q"])
    return s


# ------------------------------------------------------------------ one pass
def _own(s):
    from spinnv2_b200 import transformer as T

    op = s["case"]["op"]
    if op == "rms_norm_i8":
        T.rms_norm_i8(s["x"], s["weight"], s["residual"], eps=EPS, out=s["codes"], scale_out=s["scale"], sum_out=s["sum"])
        T.dequantize_rows_i8(s["codes"], s["scale"], out=s["values"])
        out = {"values": s["values"], "scale": s["scale"]}
        return out if s["sum"] is None else {**out, "sum": s["sum"]}
    if op == "quantize_rows_i8":
        T.quantize_rows_i8(s["x"], out=s["codes"], scale_out=s["scale"])
        T.dequantize_rows_i8(s["codes"], s["scale"], out=s["values"])
        return {"values": s["values"], "scale": s["scale"]}
    if op == "linear_i8":
        return T.linear_i8(s["a"], s["a_scale"], s["w"], s["w_scale"], bias=s["bias"], activation=s["case"]["act"], out=s["out"])
    return T.cross_attention(s["q"], s["k"], s["v"], lengths=s["lengths"], key_mask=s["mask"], out=s["out"])


def _act(y, act):
    if act == "relu":
        return torch.relu(y)
    return y * torch.sigmoid(y) if act == "silu" else y


def _plain_codes(y):
    scale = y.abs().amax(dim=1, keepdim=True) / 127.0
    q = torch.round(y / torch.where(scale > 0, scale, 1.0))
    return {"values": (q * scale).to(torch.bfloat16), "scale": scale[:, 0]}


def _valid(s):
    """[batch, keys] truth values, or None where every key counts."""
    if s["lengths"] is not None:
        return torch.arange(s["k"].shape[1], device="cuda")[None, :] < s["lengths"][:, None]
    return s["mask"]


def _plain(s):
    op, dtype = s["case"]["op"], s["dtype"]
    if op == "rms_norm_i8":
        x = s["x"].float()
        if s["residual"] is not None:
            x = x + s["residual"].float()
        y = x * torch.rsqrt(x.square().mean(dim=1, keepdim=True) + EPS) * s["weight"].float()
        out = _plain_codes(y)
        return out if s["residual"] is None else {**out, "sum": x.to(dtype)}
    if op == "quantize_rows_i8":
        return _plain_codes(s["x"].float())
    if op == "linear_i8":
        y = (s["a"].float() @ s["w"].float().t()) * s["a_scale"][:, None] * s["w_scale"][None, :]
        if s["bias"] is not None:
            y = y + s["bias"][None, :]
        return _act(y, s["case"]["act"]).to(dtype)
    b, lq, hq, d = s["q"].shape
    hk = s["k"].shape[2]
    q = s["q"].float().reshape(b, lq, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, hq // hk * lq, d)
    k = s["k"].float().permute(0, 2, 3, 1)
    v = s["v"].float().permute(0, 2, 1, 3)
    scores = (q @ k) * (1.0 / math.sqrt(d))
    valid = _valid(s)
    if valid is not None:
        scores = torch.where(valid[:, None, None, :], scores, -math.inf)
        v = torch.where(valid[:, None, :, None], v, 0.0)
    top = scores.amax(dim=-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(dim=-1, keepdim=True)
    o = (p @ v) / torch.where(total > 0, total, 1.0)
    return o.reshape(b, hk, hq // hk, lq, d).permute(0, 3, 1, 2, 4).reshape(b, lq, hq, d).to(dtype)


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_codes(y):
    top = y.abs().max(dim=1).values
    step = top / 127
    codes = torch.zeros_like(y)
    some = step > 0
    codes[some] = (y[some] / step[some, None]).round()
    return {"values": codes * step[:, None], "scale": step}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rms_norm_i8":
        t = s["x"].double()
        if case["residual"]:
            t += s["residual"].double()
        mean = (t * t).sum(dim=1) / case["width"]
        out = _exact_codes(t / (mean + EPS).sqrt()[:, None] * s["weight"].double())
        return {**out, "sum": t} if case["residual"] else out
    if op == "quantize_rows_i8":
        return _exact_codes(s["x"].double())
    if op == "linear_i8":
        w = s["w"].double().t().contiguous()
        y = torch.empty(case["m"], case["n"], dtype=torch.float64, device="cuda")
        for at in range(0, case["m"], 2048):
            part = torch.mm(s["a"][at: at + 2048].double(), w)
            part *= s["a_scale"][at: at + 2048].double()[:, None]
            part *= s["w_scale"].double()
            if case["bias"]:
                part += s["bias"].double()
            if case["act"] == "relu":
                part.clamp_(min=0)
            elif case["act"] == "silu":
                part = part / (1 + (-part).exp())
            y[at: at + 2048] = part
        return y
    b, lq, hq, d = s["q"].shape
    hk, lk = s["k"].shape[2], s["k"].shape[1]
    o = torch.zeros(b, lq, hq, d, dtype=torch.float64, device="cuda")
    valid = _valid(s)
    for i in range(b):
        at = torch.arange(lk, device="cuda") if valid is None else valid[i].nonzero()[:, 0]
        if not len(at):
            continue  # no key: the answer is zero
        for h in range(hq):
            k = s["k"][i, at, h * hk // hq].double()
            v = s["v"][i, at, h * hk // hq].double()
            p = torch.softmax(s["q"][i, :, h].double() @ k.t() / math.sqrt(d), dim=1)
            o[i, :, h] = p @ v
    return o
