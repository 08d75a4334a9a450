"""Measured calls of the 8-bit linear layers, the 8-bit routed experts and the grouped router.

Four operators, each as a serving program calls it on one GPU:

* ``linear``       x (bf16) -> rows quantised to 8 bits -> 8-bit product, epilogue -> bf16
* ``norm_linear``  residual add + RMSNorm + quantisation in one call -> 8-bit gate/up product with SwiGLU
* ``experts``      routed rows gathered and quantised -> grouped gate/up (SwiGLU) -> quantised -> grouped down
* ``route``        router logits -> expert ids and weights (softmax or sigmoid, bias, groups, top-k)

Where ``own`` is false they run in elementary torch operations; where it is true through the C ABI of the package.
"""

import math

import torch

own = False

EPILOGUE = {"none": 0, "bias": 1, "residual": 2, "swiglu": 3, "bias_gelu": 4, "bias_residual": 5}


# ------------------------------------------------------------------ cases


def _linear(m, n, k, epi):
    return {"kind": "linear", "m": m, "n": n, "k": k, "epi": epi}


def _norm(m, n, k):
    return {"kind": "norm_linear", "m": m, "n": n, "k": k}


def _experts(t, top, e, h, i):
    return {"kind": "experts", "t": t, "top": top, "e": e, "h": h, "i": i}


def _route(t, e, top, score, bias, groups, keep, best, renorm, scale):
    return {"kind": "route", "t": t, "e": e, "top": top, "score": score, "bias": bias, "groups": groups, "keep": keep,
            "best": best, "renorm": renorm, "scale": scale}


def listed():
    cases = [
        # one sequence decoding: the attention output projection of a 4096-wide decoder, added onto the residual stream
        ("linear decode 1", _linear(1, 4096, 4096, "residual")),
        # a full decode batch: the fused q/k/v projection of the same decoder
        ("linear decode 64", _linear(64, 6144, 4096, "none")),
        # one image's patches through a vision block's first MLP projection (odd patch count)
        ("linear ragged 777", _linear(777, 4096, 1024, "bias_gelu")),
        # packed prefill of 8 x 2048 tokens: the down projection
        ("linear prefill 16384", _linear(16384, 4096, 12288, "residual")),
        # a full decode batch through the second half of a layer: residual, norm, gate/up
        ("norm gate/up 64", _norm(64, 24576, 4096)),
        # the same for a packed prefill
        ("norm gate/up 8192", _norm(8192, 24576, 4096)),
        # decode batch over many small experts (64 experts, 6 a token)
        ("experts 64 x 1408 decode", _experts(32, 6, 64, 2048, 1408)),
        # decode batch over few large experts (8 experts, 2 a token)
        ("experts 8 x 14336 decode", _experts(32, 2, 8, 4096, 14336)),
        # packed prefill over the many small experts
        ("experts 64 x 1408 prefill", _experts(8192, 6, 64, 2048, 1408)),
        # router of a decode batch: plain softmax top-6 of 64
        ("route decode 64", _route(64, 64, 6, "softmax", False, 1, 1, 1, False, 1.0)),
        # router of a packed prefill: sigmoid scores, balance bias, 4 of 8 groups by their two best, top-8 of 256
        ("route prefill 16384", _route(16384, 256, 8, "sigmoid", True, 8, 4, 2, True, 2.5)),
        # softmax scores, 3 of 8 groups by their best expert, top-6 of 160, an odd number of tokens
        ("route groups 4099", _route(4099, 160, 6, "softmax", False, 8, 3, 1, False, 16.0)),
    ]
    return [{"name": name, **c} for name, c in cases]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _mult(rng, lo, hi, step):
    return max(1, int(round(_log(rng, lo, hi) / step))) * step


def draw(rng):
    kind = rng.choice(["linear", "linear", "norm_linear", "experts", "experts", "route"])
    if kind == "linear":
        m, n, k = _log(rng, 1, 16384), _mult(rng, 256, 16384, 8), _mult(rng, 256, 14336, 16)
        most = 16384 * 4096 * 12288
        if m * n * k > most:
            m = max(1, most // (n * k))
        return _linear(m, n, k, rng.choice(["none", "bias", "residual", "bias_gelu", "bias_residual"]))
    if kind == "norm_linear":
        m, n, k = _log(rng, 1, 8192), _mult(rng, 1024, 24576, 16), _mult(rng, 512, 8192, 16)
        most = 8192 * 24576 * 4096
        if m * n * k > most:
            m = max(1, most // (n * k))
        return _norm(m, n, k)
    if kind == "experts":
        e = rng.choice([4, 8, 16, 32, 60, 64, 128])
        top = rng.randint(1, min(8, e))
        h = _mult(rng, 512, 4096, 16)
        i = min(_mult(rng, 256, 14336, 16), 8 * 4096 * 14336 // (e * h) // 16 * 16)
        t = _log(rng, 1, 8192)
        most = 8192 * 6 * 2048 * 1408
        if t * top * h * i > most:
            t = max(1, most // (top * h * i))
        return _experts(t, top, e, h, i)
    groups = rng.choice([1, 1, 2, 4, 8])
    size = rng.randint(2, 256 // groups)
    keep = rng.randint(1, groups)
    top = rng.randint(1, min(8, keep * size))
    return _route(_log(rng, 1, 16384), groups * size, top, rng.choice(["softmax", "sigmoid"]), rng.random() < 0.5, groups,
                  keep, rng.choice([1, 2]), rng.random() < 0.5, rng.choice([1.0, 2.5, 16.0]))


def work(case):
    c = case
    if c["kind"] == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        extra = 2 * m * n * ("residual" in c["epi"]) + 2 * n * ("bias" in c["epi"])
        return {"bytes": 2 * m * k + n * k + 4 * n + 2 * m * n + extra, "flops": 2 * m * n * k}
    if c["kind"] == "norm_linear":  # x and residual in, the sum and the activation out
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": 6 * m * k + 2 * k + n * k + 4 * n + m * n, "flops": 2 * m * n * k}
    if c["kind"] == "experts":  # weights of the experts that random routing reaches
        t, e, h, i = c["t"], c["e"], c["h"], c["i"]
        rows, reached = t * c["top"], e * (1 - (1 - c["top"] / e) ** t)
        return {"bytes": reached * (3 * h * i + 4 * (2 * i + h)) + 2 * t * h + 2 * rows * h, "flops": 6 * rows * h * i}
    return {"bytes": 4 * c["t"] * c["e"] + 8 * c["t"] * c["top"], "flops": 8 * c["t"] * c["e"]}


# ----------------------------------------------------------------- inputs


def _activations(g, rows, dim):
    """Normal rows with a few channels an order of magnitude larger, as hidden states have them."""
    gain = torch.where(torch.rand(dim, generator=g, device="cuda") < 0.01, 8.0, 1.0)
    return (torch.randn(rows, dim, generator=g, device="cuda") * gain).to(torch.bfloat16)


def _weights(g, rows, dim):
    """8-bit rows of normal weights and their channel scales (standard deviation about 0.02)."""
    q = torch.empty(rows, dim, dtype=torch.int8, device="cuda")
    for r in range(0, rows, 32768):
        q[r:r + 32768] = torch.randn(min(32768, rows - r), dim, generator=g, device="cuda").mul_(32).round_().clamp_(-127, 127)
    return q, 0.02 / 32 * (0.5 + torch.rand(rows, generator=g, device="cuda"))


def _normal(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(torch.bfloat16)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c = dict(case)
    s = {"case": c}
    new = lambda *shape, t=torch.bfloat16: torch.empty(*shape, dtype=t, device="cuda")  # noqa: E731
    if c["kind"] == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        s["x"] = _activations(g, m, k)
        s["w"], s["ws"] = _weights(g, n, k)
        s["bias"] = _normal(g, n) if "bias" in c["epi"] else None
        s["res"] = _normal(g, m, n) if "residual" in c["epi"] else None
        s["q"], s["qs"], s["out"] = new(m, k, t=torch.int8), new(m, t=torch.float32), new(m, n)
    elif c["kind"] == "norm_linear":
        m, n, k = c["m"], c["n"], c["k"]
        s["x"], s["res"] = _activations(g, m, k), _normal(g, m, k)
        s["norm"] = (1 + 0.1 * torch.randn(k, generator=g, device="cuda")).to(torch.bfloat16)
        s["w"], s["ws"] = _weights(g, n, k)  # gate and up rows interleaved
        s["q"], s["qs"], s["sum"], s["out"] = new(m, k, t=torch.int8), new(m, t=torch.float32), new(m, k), new(m, n // 2)
    elif c["kind"] == "experts":
        t, top, e, h, i = c["t"], c["top"], c["e"], c["h"], c["i"]
        rows = t * top
        s["x"] = _activations(g, t, h)
        ids = torch.rand(t, e, generator=g, device="cuda").topk(top, 1).indices.reshape(-1)
        order = torch.sort(ids, stable=True).indices
        s["src"] = (order // top).to(torch.int32)  # the token of each routed row, rows grouped by expert
        counts = torch.bincount(ids, minlength=e)
        s["off"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        s["most"] = int(counts.max())
        s["w1"], s["s1"] = _weights(g, e * 2 * i, h)
        s["w2"], s["s2"] = _weights(g, e * h, i)
        s["q1"], s["qs1"], s["act"] = new(rows, h, t=torch.int8), new(rows, t=torch.float32), new(rows, i)
        s["q2"], s["qs2"], s["out"] = new(rows, i, t=torch.int8), new(rows, t=torch.float32), new(rows, h)
    else:
        t, e, top = c["t"], c["e"], c["top"]
        s["logits"] = torch.randn(t, e, generator=g, device="cuda") * 1.5
        s["bias"] = torch.randn(e, generator=g, device="cuda") * 0.05 if c["bias"] else None
        s["ids"], s["wts"] = new(t, top, t=torch.int32), new(t, top, t=torch.float32)
    return s


# ------------------------------------------------------------- plain forms


def _quant(x):
    """Rows of x (fp32) as integers in -127..127 and their fp32 scales; 127 x is exact for bf16 values, so ties are too."""
    amax = x.abs().amax(1, keepdim=True)
    q = torch.where(amax > 0, torch.round(x * 127 / amax), torch.zeros_like(x))
    return q, amax / torch.full_like(amax, 127)


def _silu(x):
    return x / (1 + torch.exp(-x))


def _gelu(x):
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))


def _plain_linear(s):
    q, qs = _quant(s["x"].float())
    y = (q @ s["w"].float().T) * qs * s["ws"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["case"]["epi"] == "bias_gelu":
        y = _gelu(y)
    if s["res"] is not None:
        y = y + s["res"].float()
    return y.to(torch.bfloat16)


def _plain_norm_linear(s):
    h = s["x"].float() + s["res"].float()
    n = h * torch.rsqrt((h * h).mean(1, keepdim=True) + 1e-6) * s["norm"].float()
    q, qs = _quant(n.to(torch.bfloat16).float())
    y = (q @ s["w"].float().T) * qs * s["ws"]
    return h.to(torch.bfloat16), (_silu(y[:, 0::2]) * y[:, 1::2]).to(torch.bfloat16)


def _plain_experts(s):
    c = s["case"]
    e, h, i = c["e"], c["h"], c["i"]
    at = s["off"][:-1, None].long() + torch.arange(s["most"], device="cuda")  # [e, most] rows of each expert, padded
    real = at < s["off"][1:, None]
    at = torch.where(real, at, torch.zeros_like(at))
    q, qs = _quant(s["x"].float()[s["src"].long()])
    y = torch.bmm(q[at], s["w1"].view(e, 2 * i, h).float().transpose(1, 2)) * qs[at] * s["s1"].view(e, 1, 2 * i)
    a = (_silu(y[:, :, 0::2]) * y[:, :, 1::2]).to(torch.bfloat16).float()
    q, qs = _quant(a.view(-1, i))
    y = torch.bmm(q.view(e, -1, i), s["w2"].view(e, h, i).float().transpose(1, 2)) * qs.view(e, -1, 1) * s["s2"].view(e, 1, h)
    out = torch.zeros(c["t"] * c["top"], h, dtype=torch.bfloat16, device="cuda")
    out[at[real]] = y[real].to(torch.bfloat16)
    return out


def _plain_route(s):
    c = s["case"]
    t, e, groups = c["t"], c["e"], c["groups"]
    x = s["logits"].double()  # neighbours in rank can be closer than fp32 scores tell apart
    if c["score"] == "softmax":
        p = torch.exp(x - x.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
    else:
        p = 1 / (1 + torch.exp(-x))
    choice = p if s["bias"] is None else p + s["bias"].double()
    if groups > 1:
        best = torch.sort(choice.view(t, groups, -1), dim=2, descending=True).values[:, :, :c["best"]].sum(2)
        kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :c["keep"]]
        mask = torch.zeros(t, groups, dtype=torch.bool, device="cuda").scatter_(1, kept, True)
        choice = torch.where(mask.repeat_interleave(e // groups, 1), choice, torch.full_like(choice, -math.inf))
    ids = torch.sort(choice, dim=1, descending=True, stable=True).indices[:, :c["top"]]
    w = p.gather(1, ids)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True)
    return ids.to(torch.int32), (w * c["scale"]).float()


# --------------------------------------------------------- framework calls


def _own_linear(L, check, st, s):
    c = s["case"]
    m, n, k = c["m"], c["n"], c["k"]
    q, qs, out = s["q"].data_ptr(), s["qs"].data_ptr(), s["out"]
    check(L.b200_quant_rows_int8(s["x"].data_ptr(), k, m, None, None, q, k, qs, m, k, st), "quant_rows_int8")
    check(L.b200_gemm_int8(q, k, qs, s["w"].data_ptr(), k, s["ws"].data_ptr(), out.data_ptr(), n, m, n, k,
                           EPILOGUE[c["epi"]], None if s["bias"] is None else s["bias"].data_ptr(),
                           None if s["res"] is None else s["res"].data_ptr(), n, st), "gemm_int8")
    return out


def _own_norm_linear(L, check, st, s):
    c = s["case"]
    m, n, k = c["m"], c["n"], c["k"]
    q, qs = s["q"].data_ptr(), s["qs"].data_ptr()
    check(L.b200_rmsnorm_quant_int8(s["x"].data_ptr(), s["res"].data_ptr(), s["norm"].data_ptr(), q, k, qs, None,
                                    s["sum"].data_ptr(), m, k, k, 1e-6, st), "rmsnorm_quant_int8")
    check(L.b200_gemm_int8(q, k, qs, s["w"].data_ptr(), k, s["ws"].data_ptr(), s["out"].data_ptr(), n // 2, m, n, k,
                           EPILOGUE["swiglu"], None, None, 0, st), "gemm_int8")
    return s["sum"], s["out"]


def _own_experts(L, check, st, s):
    c = s["case"]
    e, h, i = c["e"], c["h"], c["i"]
    rows = c["t"] * c["top"]
    off, act, out = s["off"].data_ptr(), s["act"].data_ptr(), s["out"]
    q1, qs1, q2, qs2 = s["q1"].data_ptr(), s["qs1"].data_ptr(), s["q2"].data_ptr(), s["qs2"].data_ptr()
    check(L.b200_quant_rows_int8(s["x"].data_ptr(), h, c["t"], s["src"].data_ptr(), off + 4 * e, q1, h, qs1, rows, h, st),
          "quant_rows_int8")
    check(L.b200_grouped_gemm_int8(q1, h, qs1, s["w1"].data_ptr(), h, s["s1"].data_ptr(), act, i, off, e, rows, 2 * i, h,
                                   EPILOGUE["swiglu"], st), "grouped_gemm_int8")
    check(L.b200_quant_rows_int8(act, i, rows, None, off + 4 * e, q2, i, qs2, rows, i, st), "quant_rows_int8")
    check(L.b200_grouped_gemm_int8(q2, i, qs2, s["w2"].data_ptr(), i, s["s2"].data_ptr(), out.data_ptr(), h, off, e, rows, h,
                                   i, EPILOGUE["none"], st), "grouped_gemm_int8")
    return out


def _own_route(L, check, st, s):
    c = s["case"]
    check(L.b200_moe_topk_grouped(s["logits"].data_ptr(), c["e"], None if s["bias"] is None else s["bias"].data_ptr(),
                                  c["t"], c["e"], c["top"], 0 if c["score"] == "softmax" else 1, c["groups"], c["keep"],
                                  c["best"], int(c["renorm"]), c["scale"], s["ids"].data_ptr(), s["wts"].data_ptr(), st),
          "moe_topk_grouped")
    return s["ids"], s["wts"]


def run(state):
    kind = state["case"]["kind"]
    if own:
        from atb_llm_study_b200 import capi

        call = {"linear": _own_linear, "norm_linear": _own_norm_linear, "experts": _own_experts, "route": _own_route}[kind]
        return call(capi.lib(), capi.check, torch.cuda.current_stream().cuda_stream, state)
    return {"linear": _plain_linear, "norm_linear": _plain_norm_linear, "experts": _plain_experts, "route": _plain_route}[kind](state)


# --------------------------------------------------------- 64-bit reference


def _rows64(x):
    """Row scales and integers of float64 rows (round half to even)."""
    top = x.abs().max(1).values
    scale = top / 127
    return torch.nan_to_num(torch.round(127 * x / top[:, None]), nan=0.0), scale


def _product64(q, scale, w, ws):
    return torch.matmul(q, w.double().t()) * torch.outer(scale, ws.double())


def _swish64(v):
    gate, up = v.unflatten(1, (-1, 2)).unbind(2)
    return gate * torch.sigmoid(gate) * up


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "linear":
        v = _product64(*_rows64(s["x"].double()), s["w"], s["ws"])
        if "bias" in case["epi"]:
            v += s["bias"].double()
        if "gelu" in case["epi"]:
            v = v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v.pow(3)))
        if "residual" in case["epi"]:
            v += s["res"].double()
        return v
    if kind == "norm_linear":
        total = s["x"].double() + s["res"].double()
        unit = total / (total.pow(2).sum(1, keepdim=True) / case["k"] + 1e-6).sqrt()
        stored = (unit * s["norm"].double()).to(torch.bfloat16).double()  # the norm's output is a bf16 value
        return total, _swish64(_product64(*_rows64(stored), s["w"], s["ws"]))
    if kind == "experts":
        h, i = case["h"], case["i"]
        out = torch.zeros(case["t"] * case["top"], h, dtype=torch.float64, device="cuda")
        off = s["off"].tolist()
        for n in range(case["e"]):
            lo, hi = off[n], off[n + 1]
            if lo == hi:
                continue
            up = slice(n * 2 * i, (n + 1) * 2 * i)
            down = slice(n * h, (n + 1) * h)
            x = s["x"].double().index_select(0, s["src"][lo:hi].long())
            act = _swish64(_product64(*_rows64(x), s["w1"][up], s["s1"][up])).to(torch.bfloat16).double()
            out[lo:hi] = _product64(*_rows64(act), s["w2"][down], s["s2"][down])
        return out
    x = s["logits"].double().cpu().numpy()
    import numpy as np

    if case["score"] == "softmax":
        p = np.exp(x - x.max(axis=1)[:, None])
        p /= p.sum(axis=1)[:, None]
    else:
        p = np.reciprocal(1 + np.exp(-x))
    key = p + (s["bias"].double().cpu().numpy() if case["bias"] else 0.0)
    if case["groups"] > 1:
        parts = np.sort(key.reshape(case["t"], case["groups"], -1), axis=2)[:, :, ::-1]
        rank = np.argsort(-parts[:, :, :case["best"]].sum(axis=2), axis=1, kind="stable")
        out_of = np.ones((case["t"], case["groups"]), bool)
        np.put_along_axis(out_of, rank[:, :case["keep"]], False, 1)
        key = np.where(np.repeat(out_of, case["e"] // case["groups"], axis=1), -np.inf, key)
    ids = np.argsort(-key, axis=1, kind="stable")[:, :case["top"]]
    w = np.take_along_axis(p, ids, 1)
    if case["renorm"]:
        w = w / w.sum(axis=1)[:, None]
    return ids.astype(np.int32), w * case["scale"]
