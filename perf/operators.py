"""The quantised linears' few-bit and routed forms: what is computed, on which sizes, and how the framework is called for it.

Four operators of one family, in the order a routed feed-forward layer or a memory-bound linear uses them:

* ``int4``     few activation rows (int8 codes, one scale a row) times a weight held in 4 bits with one scale
               for each group of input channels;
* ``route``    the router: each token's ``top_k`` experts, their weights, and the rows sorted by expert;
* ``grouped``  the int8 linear with one weight per expert over ragged groups of rows;
* ``combine``  each token's weighted sum of its experts' rows.

``run`` computes them in plain torch (``own = False``) or by the framework's entry points (``own = True``).
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"fp32": 4, "fp16": 2, "bf16": 2}


def listed():
    return [
        # One token through a small projection: the call is all latency.
        {"name": "int4 1x2048x1536 g64", "op": "int4", "m": 1, "k": 2048, "n": 1536, "group": 64, "scale": "fp16", "bias": False, "out": "fp16"},
        # One token through a video transformer block's qkv projection.
        {"name": "int4 1x5120x15360 g128", "op": "int4", "m": 1, "k": 5120, "n": 15360, "group": 128, "scale": "fp16", "bias": True, "out": "fp16"},
        # A batch of single tokens through the long inner dimension of the block's second feed-forward product.
        {"name": "int4 16x13824x5120 g256", "op": "int4", "m": 16, "k": 13824, "n": 5120, "group": 256, "scale": "fp32", "bias": False, "out": "bf16"},
        # The most rows the operator takes, the finest groups, an odd width.
        {"name": "int4 61x5120x13823 g32", "op": "int4", "m": 61, "k": 5120, "n": 13823, "group": 32, "scale": "bf16", "bias": True, "out": "fp32"},
        # A single token is routed.
        {"name": "route 1x64 top8", "op": "route", "t": 1, "e": 64, "top_k": 8, "renormalize": True, "masked": False, "in": "fp32"},
        # An image's tokens, many experts.
        {"name": "route 4096x128 top8", "op": "route", "t": 4096, "e": 128, "top_k": 8, "renormalize": True, "masked": False, "in": "bf16"},
        # A video's tokens (65520) over few experts, with padded tokens that no expert gets.
        {"name": "route 65520x31 top2 padded", "op": "route", "t": 65520, "e": 31, "top_k": 2, "renormalize": False, "masked": True, "in": "fp32"},
        # Eight single tokens: most experts get one row or none, and the weights' bytes are the work.
        {"name": "grouped 8 of 64 top8 2048x1536", "op": "grouped", "t": 8, "e": 64, "top_k": 8, "k": 2048, "n": 1536, "gather": True, "bias": False, "out": "bf16"},
        # A thousand tokens through the second product: rows already in the experts' order, about ninety each.
        {"name": "grouped 1000 of 64 top6 1536x5120", "op": "grouped", "t": 1000, "e": 64, "top_k": 6, "k": 1536, "n": 5120, "gather": False, "bias": True, "out": "fp16"},
        # An image's tokens through a wide first product, gathered: matrix products by the thousand rows.
        {"name": "grouped 4096 of 8 top2 5120x13824", "op": "grouped", "t": 4096, "e": 8, "top_k": 2, "k": 5120, "n": 13824, "gather": True, "bias": False, "out": "fp16"},
        # One token's rows are brought together.
        {"name": "combine 1 top8 5120", "op": "combine", "t": 1, "top_k": 8, "n": 5120, "residual": True, "masked": False, "out": "bf16"},
        # An image's tokens, on to the residual stream.
        {"name": "combine 4096 top2 5120", "op": "combine", "t": 4096, "top_k": 2, "n": 5120, "residual": True, "masked": True, "out": "fp16"},
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["int4", "route", "grouped", "combine"])
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    if op == "int4":
        group = rng.choice([32, 64, 128, 256])
        step = max(128, group)
        return {"op": op, "m": _log(rng, 1, 64), "k": step * _log(rng, 1, 14000 // step), "n": _log(rng, 1, 16384), "group": group,
                "scale": rng.choice(["fp32", "fp16", "bf16"]), "bias": rng.random() < 0.5, "out": dtype}
    if op == "route":
        e = _log(rng, 2, 256)
        return {"op": op, "t": _log(rng, 1, 65536), "e": e, "top_k": rng.randint(1, min(e, 16)), "renormalize": rng.random() < 0.5,
                "masked": rng.random() < 0.5, "in": dtype}
    if op == "grouped":
        e, t = _log(rng, 2, 128), _log(rng, 1, 8192)
        top_k = rng.randint(1, min(e, 8))
        k, n = 16 * _log(rng, 4, 320), 8 * _log(rng, 4, 1700)
        n = min(n, 8 * max(4, int(min(4e8 / (e * k), 5e11 / (t * top_k * k)) // 8)))
        return {"op": op, "t": t, "e": e, "top_k": top_k, "k": k, "n": n, "gather": rng.random() < 0.5, "bias": rng.random() < 0.5, "out": dtype}
    return {"op": op, "t": _log(rng, 1, 8192), "top_k": rng.randint(1, 12), "n": _log(rng, 1, 8192), "residual": rng.random() < 0.5,
            "masked": rng.random() < 0.5, "out": dtype}


# ---------------------------------------------------------------- inputs
def _codes(shape, spread, limit, g):
    """Integer codes as a quantiser leaves them: rounded normal values, clipped to the range."""
    out = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat = out.view(-1)
    for at in range(0, flat.numel(), 1 << 28):
        part = flat[at:at + (1 << 28)]
        part.copy_((torch.randn(part.numel(), generator=g, device="cuda") * spread).round_().clamp_(-limit, limit))
    return out


def _pack(codes):
    """Codes in [-8, 7], [n, k] with k a multiple of 128, in the framework's 4-bit layout, [n, k / 2] bytes: of
    each 128 codes, byte 16 t + 4 j + b holds code 32 j + 8 t + b in its low and 32 j + 8 t + 4 + b in its high half."""
    n, k = codes.shape
    c = codes.view(n, k // 128, 4, 4, 2, 4).permute(0, 1, 3, 2, 4, 5).to(torch.uint8) & 15
    return (c[..., 0, :] | (c[..., 1, :] << 4)).reshape(n, k // 2).contiguous()


def _unpack(packed):
    """The codes of ``_pack``'s bytes as fp32."""
    n, half = packed.shape
    c = packed.view(n, half // 64, 4, 4, 4)
    c = torch.stack([c & 15, c >> 4], dim=-2).permute(0, 1, 3, 2, 4, 5).reshape(n, half * 2).float()
    return c - 16 * (c >= 8)


def _logits(t, e, masked, dtype, g):
    """Router logits: some experts are liked better; ``masked``: an eighth of the tokens are padding (every logit
    -inf) and one expert of the last quarter of them is closed."""
    x = torch.randn(t, e, generator=g, device="cuda") + 0.5 * torch.randn(e, generator=g, device="cuda")
    if masked:
        x[torch.rand(t, generator=g, device="cuda") < 0.125] = -math.inf
        x[3 * t // 4:, e - 1] = -math.inf
    return x.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    st, op = dict(case), case["op"]
    if op == "int4":
        m, k, n = case["m"], case["k"], case["n"]
        st["xq"] = _codes((m, k), 32, 127, g)
        st["xs"] = torch.rand(m, generator=g, device="cuda") * 0.02 + 0.01
        st["w4"] = _pack(_codes((n, k), 2.6, 7, g))
        st["ws"] = (torch.rand(n, k // case["group"], generator=g, device="cuda") * 0.005 + 0.005).to(DTYPES[case["scale"]])
        st["b"] = torch.randn(n, generator=g, device="cuda") if case["bias"] else None
    elif op == "route":
        st["logits"] = _logits(case["t"], case["e"], case["masked"], DTYPES[case["in"]], g)
    elif op == "grouped":
        t, e, k, n = case["t"], case["e"], case["k"], case["n"]
        _, ids, offsets, rows, _ = _route(_logits(t, e, False, torch.float32, g), case["top_k"], True)
        m = t if case["gather"] else t * case["top_k"]
        st["offsets"], st["rows"] = offsets, rows if case["gather"] else None
        st["most"] = int((offsets[1:] - offsets[:-1]).max())
        st["xq"] = _codes((m, k), 32, 127, g)
        st["xs"] = torch.rand(m, generator=g, device="cuda") * 0.02 + 0.01
        st["wq"] = _codes((e, n, k), 36, 127, g)
        st["ws"] = torch.rand(e, n, generator=g, device="cuda") * 0.0005 + 0.0005
        st["b"] = torch.randn(e, n, generator=g, device="cuda") if case["bias"] else None
    else:
        t, n, top_k, dtype = case["t"], case["n"], case["top_k"], DTYPES[case["out"]]
        logits = _logits(t, 4 * top_k, case["masked"], torch.float32, g)
        st["weights"], _, _, _, st["place"] = _route(logits, top_k, True)
        st["y"] = torch.randn(t * top_k, n, generator=g, device="cuda").to(dtype)
        st["residual"] = torch.randn(t, n, generator=g, device="cuda").to(dtype) if case["residual"] else None
    return st


# ---------------------------------------------------------------- the plain forms
def _int4(xq, xs, w4, ws, b, group, dtype):
    n, k = w4.shape[0], xq.shape[1]
    w = (_unpack(w4).view(n, k // group, group) * ws.float()[:, :, None]).view(n, k)
    y = (xq.float() @ w.t()) * xs[:, None]
    return (y if b is None else y + b).to(dtype)


def _route(logits, top_k, renormalize):
    """(weights [t, k], ids [t, k], offsets [e + 1], rows [t k], place [t, k]): the experts with the largest logits
    (ties: the lower index first), their softmax weights over the chosen or over all experts, and the slots
    sorted by expert.  A slot whose logit is -inf is left out: weight 0, id and place -1."""
    t, e = logits.shape
    x = logits.float()
    value, ids = torch.sort(x, dim=1, descending=True, stable=True)
    top = torch.where(torch.isneginf(value[:, :1]), 0.0, value[:, :1])
    value, ids = value[:, :top_k], ids[:, :top_k]
    weight = torch.exp(value - top)
    total = (weight if renormalize else torch.exp(x - top)).sum(1, keepdim=True)
    live = ~torch.isneginf(value)
    weight = torch.where(live, weight / total, 0.0)
    key = torch.where(live, ids, e).reshape(-1)
    counts = (key[:, None] == torch.arange(e, device=key.device)).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    order = torch.sort(key, stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(t * top_k, device=order.device)
    dead = key == e
    rows = torch.where(dead[order], -1, order // top_k)
    place = torch.where(dead, -1, place).view(t, top_k)
    ids = torch.where(live, ids, -1)
    return weight, ids.int(), offsets.int(), rows.int(), place.int()


def _grouped(xq, xs, wq, ws, b, offsets, rows, most, dtype):
    e, n, k = wq.shape
    x = xq.float() * xs[:, None]
    x = x if rows is None else x[rows.long()]
    r = torch.arange(x.shape[0], device=x.device)
    expert = (r[:, None] >= offsets[1:-1]).sum(1)
    within = r - offsets.long()[expert]
    padded = x.new_zeros(e, most, k)
    padded[expert, within] = x
    y = torch.bmm(padded, wq.float().transpose(1, 2)) * ws[:, None, :]
    y = y if b is None else y + b[:, None, :]
    return y[expert, within].to(dtype)


def _combine(y, place, weights, residual, dtype):
    live = place >= 0
    out = torch.where(live, weights, 0.0)[:, :, None] * y[place.clamp(min=0).long()].float()
    out = out.sum(1)
    return (out if residual is None else out + residual.float()).to(dtype)


def run(st):
    op = st["op"]
    if own:
        from tilegen_b200 import ops

        if op == "int4":
            return ops.int4_gemv_dequant(st["xq"], st["xs"], st["w4"], st["ws"], st["b"], DTYPES[st["out"]])
        if op == "route":
            return tuple(ops.route_experts(st["logits"], st["top_k"], renormalize=st["renormalize"]))
        if op == "grouped":
            return ops.int8_grouped_gemm_dequant(st["xq"], st["xs"], st["wq"], st["ws"], st["b"], st["offsets"], DTYPES[st["out"]],
                                                 rows=st["rows"])
        return ops.combine_experts(st["y"], st["place"], st["weights"], residual=st["residual"])
    if op == "int4":
        return _int4(st["xq"], st["xs"], st["w4"], st["ws"], st["b"], st["group"], DTYPES[st["out"]])
    if op == "route":
        return _route(st["logits"], st["top_k"], st["renormalize"])
    if op == "grouped":
        return _grouped(st["xq"], st["xs"], st["wq"], st["ws"], st["b"], st["offsets"], st["rows"], st["most"], DTYPES[st["out"]])
    return _combine(st["y"], st["place"], st["weights"], st["residual"], DTYPES[st["out"]])


def work(case):
    op = case["op"]
    if op == "int4":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": m * k + 4 * m + n * k // 2 + n * (k // case["group"]) * SIZES[case["scale"]] + 4 * n * case["bias"] + m * n * SIZES[case["out"]],
                "flops": 2 * m * n * k}
    if op == "route":
        t, e, slots = case["t"], case["e"], case["t"] * case["top_k"]
        return {"bytes": t * e * SIZES[case["in"]] + 16 * slots + 4 * (e + 1), "flops": t * e + 4 * slots}
    if op == "grouped":
        t, e, k, n, r = case["t"], case["e"], case["k"], case["n"], case["t"] * case["top_k"]
        m = t if case["gather"] else r
        used = e * (1 - (1 - case["top_k"] / e) ** t)  # the experts that get a row, where all are liked the same
        return {"bytes": m * (k + 4) + used * n * (k + 4 + 4 * case["bias"]) + r * n * SIZES[case["out"]] + 4 * r * case["gather"], "flops": 2 * r * n * k}
    t, n, r = case["t"], case["n"], case["t"] * case["top_k"]
    return {"bytes": (r + t + t * case["residual"]) * n * SIZES[case["out"]] + 8 * r, "flops": 2 * r * n}


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "int4":
        m, k, n, group = case["m"], case["k"], case["n"], case["group"]
        byte = st["w4"].view(n, k // 128, 64).long()
        at = torch.arange(128, device="cuda")  # code `at` of a block: its byte, and which half of it
        byte = byte[:, :, (at % 32) // 8 * 16 + at // 32 * 4 + at % 4]
        code = (byte >> (4 * (at % 8 // 4))) & 15
        code = torch.where(code > 7, code - 16, code).view(n, k).double()
        y = torch.zeros(m, n, dtype=torch.float64, device="cuda")
        for i in range(k // group):
            cut = slice(i * group, (i + 1) * group)
            y += (st["xq"][:, cut].double() @ code[:, cut].t()) * st["ws"][:, i].double()
        y *= st["xs"].double()[:, None]
        return y if st["b"] is None else y + st["b"].double()
    if op == "route":
        x = st["logits"].double()
        value, _ = torch.topk(x, case["top_k"], dim=1)
        norm = torch.logsumexp(value if case["renormalize"] else x, dim=1, keepdim=True)
        weight = torch.exp(value - torch.where(torch.isneginf(norm), 0.0, norm))
        return weight, None, None, None, None
    if op == "grouped":
        bounds = st["offsets"].tolist()
        out = torch.empty(bounds[-1], case["n"], dtype=torch.float64, device="cuda")
        for e in range(case["e"]):
            cut = slice(bounds[e], bounds[e + 1])
            at = st["rows"][cut].long() if case["gather"] else cut
            y = (st["xq"][at].double() @ st["wq"][e].double().t()) * st["xs"][at].double()[:, None] * st["ws"][e].double()
            out[cut] = y if st["b"] is None else y + st["b"][e].double()
        return out
    out = torch.zeros(case["t"], case["n"], dtype=torch.float64, device="cuda")
    for j in range(case["top_k"]):
        at = st["place"][:, j].long()
        out += torch.where(at < 0, 0.0, st["weights"][:, j].double())[:, None] * st["y"][at.clamp(min=0)].double()
    return out if st["residual"] is None else out + st["residual"].double()
