"""Measured cases of the feed-forward operators: root-mean-square norm with the residual's addition
(and its form with an 8-bit output), matrix product with bias, activation and residual (and its form
with 8-bit operands), and the exchange of rows between token order and expert order.

``run`` computes them with elementary torch operations, or, with ``own`` set, with this package's
kernels; ``exact`` gives the same outputs from the definitions in 64 bits.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
_ACTS = ("none", "relu", "leaky_relu", "elu", "gelu", "silu")
_SLOPE = 0.2
_EPS = 1e-6
_E4M3_MAX = 448.0
_FLT_MIN = 2.0 ** -126


# ---- cases -----------------------------------------------------------------------------------------
def _norm(rows, width, dtype, residual, train):
    return {"op": "norm", "rows": rows, "width": width, "dtype": dtype, "residual": residual, "train": train}


def _norm8(rows, width, dtype, residual, block):
    return {"op": "norm8", "rows": rows, "width": width, "dtype": dtype, "residual": residual, "block": block}


def _linear(rows, inner, outer, dtype, act, bias, residual, train):
    return {"op": "linear", "rows": rows, "in": inner, "out": outer, "dtype": dtype, "act": act, "bias": bias,
            "residual": residual, "train": train}


def _linear8(rows, inner, outer, dtype, act, bias, residual):
    return {"op": "linear8", "rows": rows, "in": inner, "out": outer, "dtype": dtype, "act": act, "bias": bias,
            "residual": residual}


def _experts(tokens, k, experts, width, dtype, dropped, train):
    return {"op": "experts", "tokens": tokens, "k": k, "experts": experts, "width": width, "dtype": dtype,
            "dropped": dropped, "train": train}


def listed():
    return [
        # one generated token enters a block: latency
        {"name": "norm_token", **_norm(1, 4096, "bf16", True, False)},
        # a training batch of sequences, forward and backward, with a ragged number of rows
        {"name": "norm_train", **_norm(16381, 2048, "bf16", True, True)},
        # the input features of the power-law graph's nodes, in the framework's own type; rows of 602
        # floats are not whole 16-byte units
        {"name": "norm_nodes", **_norm(232965, 602, "fp32", False, True)},
        # a few sequences decoding, a scale for every 128 columns
        {"name": "norm8_tokens", **_norm8(8, 5120, "bf16", True, 128)},
        # a long prompt, one scale a row, as the product with 8-bit operands takes it
        {"name": "norm8_prompt", **_norm8(16384, 4096, "bf16", True, 0)},
        # one generated token through a layer: bound by the weights' bytes
        {"name": "linear_token", **_linear(1, 4096, 8192, "bf16", "silu", True, False, False)},
        # the wide layer of a feed-forward block in training
        {"name": "linear_train", **_linear(8192, 2048, 8192, "bf16", "gelu", True, True, True)},
        # node features projected in 32 bits, forward and backward
        {"name": "linear_nodes", **_linear(232965, 602, 256, "fp32", "elu", True, False, True)},
        # 19 sequences decoding with 8-bit weights
        {"name": "linear8_tokens", **_linear8(19, 4096, 8192, "bf16", "silu", True, False)},
        # a long prompt with 8-bit weights, closing a residual branch
        {"name": "linear8_prompt", **_linear8(8192, 8192, 4096, "bf16", "none", True, True)},
        # a few sequences decoding through a layer of experts
        {"name": "experts_tokens", **_experts(16, 4, 64, 2048, "bf16", 0.0, False)},
        # a training batch through a layer of experts; an eighth of the tokens are padding
        {"name": "experts_train", **_experts(16411, 8, 128, 2048, "bf16", 0.125, True)},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _multiple(rng, n, of):
    """n, or for half of the draws the multiple of ``of`` next below it."""
    return n if rng.random() < 0.5 else max(of, n // of * of)


def draw(rng):
    op = rng.choice(["norm", "norm8", "linear", "linear", "linear8", "experts"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op in ("norm", "norm8"):
        width = _multiple(rng, _log(rng, 16, 16384), 64)
        rows = _log(rng, 1, min(262144, (1 << 26) // width))
        if op == "norm":
            return _norm(rows, width, dtype, rng.random() < 0.7, rng.random() < 0.5)
        return _norm8(rows, width, dtype, rng.random() < 0.7, rng.choice([0, 0, 128]))
    if op == "experts":
        experts = _log(rng, 4, 256)
        k = rng.randint(1, min(8, experts))
        width = _multiple(rng, _log(rng, 32, 8192), 64)
        tokens = _log(rng, 1, min(65536, (1 << 28) // (width * k)))
        return _experts(tokens, k, experts, width, dtype, rng.choice([0.0, 0.0, 0.2]), rng.random() < 0.5)
    inner = _multiple(rng, _log(rng, 32, 8192), 64)
    outer = _multiple(rng, _log(rng, 8, 8192), 64)
    act = rng.choice(_ACTS)
    bias, residual = rng.random() < 0.7, rng.random() < 0.5
    most = (1 << 37) // (inner * outer)  # multiply-adds of linear_train's forward product
    if op == "linear8":
        rows = _log(rng, 1, min(32768, most))
        return _linear8(rows, inner, outer, dtype, act, bias, residual)
    train = rng.random() < 0.5
    if train and dtype == "fp32" and act in ("relu", "leaky_relu"):
        act = "elu"  # a gradient with a step at zero hangs on the last bit of its argument
    rows = _log(rng, 1, min(262144 if dtype == "fp32" else 32768, most, (1 << 27) // (inner + outer)))
    return _linear(rows, inner, outer, dtype, act, bias, residual, train)


def _seeded(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def prepare(case, seed):
    gen = _seeded(seed)
    op, dt = case["op"], _DT[case["dtype"]]
    s = {"case": case}
    if op in ("norm", "norm8"):
        n, d = case["rows"], case["width"]
        s["x"] = _randn(gen, n, d).to(dt)
        s["weight"] = (1 + 0.1 * _randn(gen, d)).to(dt)
        # the residual stream is larger than what a block adds to it
        s["residual"] = (2 * _randn(gen, n, d)).to(dt) if case["residual"] else None
        if case.get("train"):
            s["grad_y"] = _randn(gen, n, d).to(dt)
            s["grad_h"] = _randn(gen, n, d).to(dt) if case["residual"] else None
    elif op == "linear":
        m, k, n = case["rows"], case["in"], case["out"]
        s["x"] = _randn(gen, m, k).to(dt)
        s["weight"] = (_randn(gen, n, k) / math.sqrt(k)).to(dt)
        s["bias"] = (0.1 * _randn(gen, n)).to(dt) if case["bias"] else None
        s["residual"] = _randn(gen, m, n).to(dt) if case["residual"] else None
        if case["train"]:
            s["grad_y"] = _randn(gen, m, n).to(dt)
    elif op == "linear8":
        m, k, n = case["rows"], case["in"], case["out"]
        s["x8"], s["x_scale"] = _to_8_bits(_randn(gen, m, k))
        s["weight8"], s["weight_scale"] = _to_8_bits(_randn(gen, n, k) / math.sqrt(k))
        s["bias"] = (0.1 * _randn(gen, n)).to(dt) if case["bias"] else None
        s["residual"] = _randn(gen, m, n).to(dt) if case["residual"] else None
    else:
        t, k, e, d = case["tokens"], case["k"], case["experts"], case["width"]
        # a router's choice: distinct experts for a token, some experts liked better than others
        liked = _randn(gen, e)
        top = torch.topk(_randn(gen, t, e) + liked, k, dim=1)
        ids = top.indices.to(torch.int32)
        if case["dropped"] > 0:  # padding tokens go to no expert
            ids[torch.rand(t, generator=gen, device="cuda") < case["dropped"]] = -1
        s["ids"], s["weights"] = ids, torch.softmax(top.values, dim=1)
        s["x"] = _randn(gen, t, d).to(dt)
        s["expert_out"] = _randn(gen, t * k, d).to(dt)  # what the experts make of the sorted rows
        if case["train"]:
            s["grad_sorted"] = _randn(gen, t * k, d).to(dt)
            s["grad_out"] = _randn(gen, t, d).to(dt)
    if case.get("train"):
        for name in ("x", "weight", "bias", "residual", "weights", "expert_out"):
            if isinstance(s.get(name), torch.Tensor):
                s[name].requires_grad_(True)
    return s


def _to_8_bits(v):
    scale = (v.abs().amax(1, keepdim=True) / _E4M3_MAX).clamp_min(_FLT_MIN)
    return (v / scale).to(torch.float8_e4m3fn), scale


# ---- this package's kernels ----------------------------------------------------------------------------
def _run_own(s):
    case = s["case"]
    op, train = case["op"], case.get("train", False)
    if op == "norm":
        from ae_mlsys_gnn_b200.operators.rms_norm import add_rms_norm

        y, h = add_rms_norm(s["x"], s["weight"], s["residual"], _EPS)
        if not train:
            return {"y": y, "h": h} if case["residual"] else {"y": y}
        if case["residual"]:
            gx, gw = torch.autograd.grad((y, h), (s["x"], s["weight"]), (s["grad_y"], s["grad_h"]))
            return {"y": y, "h": h, "gx": gx, "gw": gw}
        gx, gw = torch.autograd.grad(y, (s["x"], s["weight"]), s["grad_y"])
        return {"y": y, "gx": gx, "gw": gw}
    if op == "norm8":
        from ae_mlsys_gnn_b200.operators.rms_norm import add_rms_norm_fp8

        q, scale, h = add_rms_norm_fp8(s["x"], s["weight"], s["residual"], _EPS, case["block"])
        return {"q": q, "scale": scale, "h": h} if case["residual"] else {"q": q, "scale": scale}
    act = None if case.get("act") == "none" else case.get("act")
    if op == "linear":
        from ae_mlsys_gnn_b200.operators.linear_act import linear_act

        y = linear_act(s["x"], s["weight"], s["bias"], act, s["residual"], _SLOPE)
        if not train:
            return {"y": y}
        if case["bias"]:
            gx, gw, gb = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["grad_y"])
            return {"y": y, "gx": gx, "gw": gw, "gb": gb}
        gx, gw = torch.autograd.grad(y, (s["x"], s["weight"]), s["grad_y"])
        return {"y": y, "gx": gx, "gw": gw}
    if op == "linear8":
        from ae_mlsys_gnn_b200.operators.linear_act import linear_act_fp8

        return {"y": linear_act_fp8(s["x8"], s["x_scale"], s["weight8"], s["weight_scale"], s["bias"], act,
                                    s["residual"], _SLOPE, _DT[case["dtype"]])}
    from ae_mlsys_gnn_b200.operators.experts import expert_combine, expert_dispatch, expert_sort

    order = expert_sort(s["ids"], case["experts"])
    xs = expert_dispatch(s["x"], order)
    out = expert_combine(s["expert_out"], s["weights"], order)
    got = {"offsets": order.offsets, "slots": order.slots, "sorted": xs, "out": out}
    if train:
        got["gx"], = torch.autograd.grad(xs, s["x"], s["grad_sorted"])
        got["gye"], got["gw"] = torch.autograd.grad(out, (s["expert_out"], s["weights"]), s["grad_out"])
    return got


# ---- plain forms ------------------------------------------------------------------------------------------
def _act(z, name):
    if name == "relu":
        return z.clamp_min(0)
    if name == "leaky_relu":
        return torch.where(z > 0, z, _SLOPE * z)
    if name == "elu":
        return torch.where(z > 0, z, torch.expm1(z.clamp_max(0)))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "leaky_relu":
        return torch.where(z > 0, 1.0, _SLOPE).to(z.dtype)
    if name == "elu":
        return torch.exp(z.clamp_max(0))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "silu":
        sig = 1 / (1 + torch.exp(-z))
        return sig * (1 + z * (1 - sig))
    return torch.ones_like(z)


def _plain_norm(s):
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    rstd = torch.rsqrt((h * h).mean(1, keepdim=True) + _EPS)
    return h, rstd, h * rstd * s["weight"].float()


def _run_plain(s):
    case = s["case"]
    op, dt = case["op"], _DT[case["dtype"]]
    if op == "norm":
        h, rstd, y = _plain_norm(s)
        got = {"y": y.to(dt)}
        if case["residual"]:
            got["h"] = h.to(dt)
        if case["train"]:
            gy, xhat = s["grad_y"].float(), h * rstd
            gw = gy * s["weight"].float()
            gx = rstd * (gw - xhat * (gw * xhat).mean(1, keepdim=True))
            if case["residual"]:
                gx = gx + s["grad_h"].float()
            got["gx"] = gx.to(dt)
            got["gw"] = (gy * xhat).sum(0, dtype=torch.float64).to(dt)
        return got
    if op == "norm8":
        h, _, y = _plain_norm(s)
        n, d = y.shape
        block = case["block"] or d
        parts = (d + block - 1) // block
        yb = torch.nn.functional.pad(y, (0, parts * block - d)).view(n, parts, block)
        scale = (yb.abs().amax(2) / _E4M3_MAX).clamp_min(_FLT_MIN)
        q = (yb / scale[:, :, None]).view(n, parts * block)[:, :d].contiguous().to(torch.float8_e4m3fn)
        return {"q": q, "scale": scale, "h": h.to(dt)} if case["residual"] else {"q": q, "scale": scale}
    if op in ("linear", "linear8"):
        if op == "linear":
            x, w = s["x"].float(), s["weight"].float()
        else:
            x, w = s["x8"].float() * s["x_scale"], s["weight8"].float() * s["weight_scale"]
        z = x @ w.t()
        if s["bias"] is not None:
            z = z + s["bias"].float()
        y = _act(z, case["act"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        got = {"y": y.to(dt)}
        if case.get("train"):
            gz = s["grad_y"].float() * _act_slope(z, case["act"])
            got["gx"] = (gz @ w).to(dt)
            got["gw"] = (gz.t() @ x).to(dt)
            if case["bias"]:
                got["gb"] = gz.sum(0, dtype=torch.float64).to(dt)
        return got
    t, k, e = case["tokens"], case["k"], case["experts"]
    ids = s["ids"].reshape(-1).long()
    valid = (ids >= 0) & (ids < e)
    key = torch.where(valid, ids, e)
    order = torch.argsort(key, stable=True)
    slots = torch.empty_like(order)
    slots[order] = torch.arange(t * k, device=order.device)
    counts = torch.bincount(key, minlength=e + 1)[:e]
    offsets = torch.nn.functional.pad(torch.cumsum(counts, 0), (1, 0)).to(torch.int32)
    used = valid[order][:, None]  # rows behind the last expert's hold zeros
    ok = valid.view(t, k, 1)
    at = slots.view(t, k)
    x, ye, w = s["x"], s["expert_out"].float(), s["weights"].unsqueeze(2)
    picked = torch.where(ok, ye[at], 0.0)
    got = {"offsets": offsets, "slots": torch.where(valid, slots, -1).to(torch.int32).view(t, k),
           "sorted": torch.where(used, x[order // k], torch.zeros((), dtype=dt, device=x.device)),
           "out": (picked * w).sum(1).to(dt)}
    if case["train"]:
        got["gx"] = torch.where(ok, s["grad_sorted"].float()[at], 0.0).sum(1).to(dt)
        go = s["grad_out"].float().unsqueeze(1)
        got["gw"] = (picked * go).sum(2)
        got["gye"] = torch.where(used, (go * w).reshape(t * k, -1)[order], 0.0).to(dt)
    return got


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():  # the plain gradients are formulas, nothing is recorded
        return _run_plain(state)


# ---- definitions in 64 bits ---------------------------------------------------------------------------------
def _activation64(z, name):
    f = torch.nn.functional
    table = {"none": lambda v: v, "relu": f.relu, "leaky_relu": lambda v: f.leaky_relu(v, _SLOPE), "elu": f.elu,
             "gelu": f.gelu, "silu": f.silu}
    return table[name](z)


def _leaf(t):
    return None if t is None else t.detach().double().requires_grad_(True)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("norm", "norm8"):
        x, w, r = _leaf(s["x"]), _leaf(s["weight"]), _leaf(s["residual"])
        h = x if r is None else x + r
        y = w * (h / torch.sqrt(h.square().mean(-1, keepdim=True) + _EPS))
        got = {"h": h.detach()} if case["residual"] else {}
        if op == "norm":
            got["y"] = y.detach()
            if case["train"]:
                outs, grads = ((y, h), (s["grad_y"].double(), s["grad_h"].double())) if case["residual"] else (
                    (y,), (s["grad_y"].double(),))
                got["gx"], got["gw"] = torch.autograd.grad(outs, (x, w), grads)
            return got
        y = y.detach()
        chunks = torch.split(y, case["block"] or y.shape[1], dim=1)
        scales = [torch.clamp(c.abs().max(1, keepdim=True).values / _E4M3_MAX, min=_FLT_MIN) for c in chunks]
        got["scale"] = torch.cat(scales, 1)
        # the value itself: how far the 8 bits are from it is what their rounding costs
        got["q"] = torch.cat([c / v for c, v in zip(chunks, scales)], 1)
        return got
    if op in ("linear", "linear8"):
        if op == "linear":
            x, w = _leaf(s["x"]), _leaf(s["weight"])
        else:
            x = s["x8"].to(torch.float64) * s["x_scale"].double()
            w = s["weight8"].to(torch.float64) * s["weight_scale"].double()
        b = _leaf(s["bias"])
        z = torch.nn.functional.linear(x, w, b)
        y = _activation64(z, case["act"])
        if s["residual"] is not None:
            y = y + s["residual"].detach().double()
        got = {"y": y.detach()}
        if case.get("train"):
            grads = torch.autograd.grad(y, (x, w) if b is None else (x, w, b), s["grad_y"].double())
            got["gx"], got["gw"] = grads[0], grads[1]
            if b is not None:
                got["gb"] = grads[2]
        return got
    t, k, e, d = case["tokens"], case["k"], case["experts"], case["width"]
    ids = s["ids"].long().view(-1)
    dev = ids.device
    # a pair's place: the pairs of lower experts, and those of its own expert that come before it
    onehot = (ids[:, None] == torch.arange(e, device=dev)).to(torch.int32)
    counts = onehot.sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    valid = onehot.any(1)
    before = torch.gather(onehot.cumsum(0), 1, ids.clamp_min(0)[:, None]).squeeze(1) - 1
    slots = torch.where(valid, offsets[ids.clamp_min(0)] + before, torch.full_like(before, -1))
    pairs = torch.nonzero(valid).squeeze(1)
    to, token = slots[pairs], pairs // k
    x, ye, w = _leaf(s["x"]), _leaf(s["expert_out"]), _leaf(s["weights"])
    xs = torch.zeros(t * k, d, dtype=torch.float64, device=dev).index_add(0, to, x[token])
    out = torch.zeros(t, d, dtype=torch.float64, device=dev).index_add(0, token, ye[to] * w.view(-1)[pairs, None])
    got = {"offsets": offsets.to(torch.int32), "slots": slots.to(torch.int32).view(t, k), "sorted": xs.detach(),
           "out": out.detach()}
    if case["train"]:
        got["gx"], = torch.autograd.grad(xs, x, s["grad_sorted"].double())
        got["gye"], got["gw"] = torch.autograd.grad(out, (ye, w), s["grad_out"].double())
    return got


# ---- what a pass cannot do without -----------------------------------------------------------------------------
def work(case):
    op, b = case["op"], _SIZE[case["dtype"]]
    if op in ("norm", "norm8"):
        n, d = case["rows"], case["width"]
        read = n * d * b * (2 if case["residual"] else 1) + d * b
        kept = n * d * b if case["residual"] else 0  # h
        if op == "norm8":
            return {"bytes": read + kept + n * d + 4 * n * (-(-d // (case["block"] or d))), "flops": 6 * n * d}
        total = read + kept + n * d * b
        if case["train"]:
            # grad_y (and grad_h) come in, grad_x and the weight's gradient go out
            total += n * d * b * (3 if case["residual"] else 2) + d * b
        return {"bytes": total, "flops": n * d * (14 if case["train"] else 5)}
    if op in ("linear", "linear8"):
        m, k, n = case["rows"], case["in"], case["out"]
        e = b if op == "linear" else 1
        total = (m * k + n * k) * e + m * n * b * (2 if case["residual"] else 1) + (n * b if case["bias"] else 0)
        if op == "linear8":
            return {"bytes": total + 4 * (m + n), "flops": 2 * m * n * k}
        if case["train"]:
            total += m * n * b + (m * k + n * k) * b + (n * b if case["bias"] else 0)
        return {"bytes": total, "flops": 2 * m * n * k * (3 if case["train"] else 1)}
    t, k, e, d = case["tokens"], case["k"], case["experts"], case["width"]
    kept = t * k * (1 - case["dropped"])
    total = 4 * t * k * 3 + 4 * (e + 1)          # ids, slots, weights, offsets
    total += t * d * b + t * k * d * b           # rows to expert order
    total += kept * d * b + t * d * b            # and back
    flops = 2 * kept * d
    if case["train"]:
        total += kept * d * b + t * d * b        # gradient of the rows' way out
        total += t * d * b + t * k * d * b + 4 * t * k  # gradients of the way back (the experts' rows are read above)
        flops += 4 * kept * d
    return {"bytes": total, "flops": flops}
