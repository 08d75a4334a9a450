"""Measured calls of a serving step around the paged KV cache: block tables, window and shared-prefix attention, logits.

Operators, each as a serving program calls it on one GPU:

* ``extend``   block tables, context lengths, positions and cache slots of a step from request lengths
* ``release``  blocks of finished or shortened requests back to the free list
* ``prompt``   packed prompts, causal attention with a sliding window and a few first tokens that stay visible
* ``token``    the same for one token a sequence, over the paged cache
* ``shared``   one token a sequence of a batch whose sequences share a long prefix, over the paged cache
* ``logits``   penalties for repeated tokens, biases and grammar masks on logits, and the greedy token

Where ``own`` is false they run in elementary torch operations; where it is true through the C ABI of the package.
"""

import math
import random

import torch

own = False

# ------------------------------------------------------------------ cases


def _extend(seqs, cached, new, block, idle):
    return {"kind": "extend", "seqs": seqs, "cached": cached, "new": new, "block": block, "idle": idle}


def _release(seqs, cached, block, finished):
    return {"kind": "release", "seqs": seqs, "cached": cached, "block": block, "finished": finished}


def _prompt(seqs, longest, ragged, nq, nkv, d, window, sinks):
    return {"kind": "prompt", "seqs": seqs, "longest": longest, "ragged": ragged, "nq": nq, "nkv": nkv, "d": d,
            "window": window, "sinks": sinks}


def _token(batch, longest, ragged, nq, nkv, d, block, window, sinks):
    return {"kind": "token", "batch": batch, "longest": longest, "ragged": ragged, "nq": nq, "nkv": nkv, "d": d,
            "block": block, "window": window, "sinks": sinks}


def _shared(batch, prefix, longest, nq, nkv, d, block):
    return {"kind": "shared", "batch": batch, "prefix": prefix, "longest": longest, "nq": nq, "nkv": nkv, "d": d,
            "block": block}


def _logits(rows, vocab, history, biases, masks):
    return {"kind": "logits", "rows": rows, "vocab": vocab, "history": history, "biases": biases, "masks": masks}


def listed():
    cases = [
        # one decode step of a full batch: 64 sequences of up to 4096 cached tokens, one new token each
        ("extend decode 64", _extend(64, 4096, 1, 128, 0.0)),
        # many slots, some idle, chunks of prompts beside single tokens: about 130 thousand new tokens
        ("extend prompts 2048", _extend(2048, 8192, 127, 64, 0.2)),
        # the end of a step: a third of 300 sequences finished, others lose rejected draft tokens
        ("release 300", _release(300, 4096, 64, 0.33)),
        # packed prompts of the benchmark's prefill shape, half of each prompt inside the window
        ("prompt 8 x 2048", _prompt(8, 2048, False, 32, 8, 128, 1024, 4)),
        # many short ragged prompts with narrow heads and a short window, no sinks
        ("prompt ragged 17 x 900", _prompt(17, 900, True, 12, 4, 64, 128, 0)),
        # one long document under a long window
        ("prompt 1 x 32768", _prompt(1, 32768, False, 32, 8, 128, 4096, 4)),
        # one conversation, long past its window: latency
        ("token 1", _token(1, 20000, False, 32, 8, 128, 128, 1024, 4)),
        # a full decode batch of ragged contexts under a long window
        ("token 64", _token(64, 32768, True, 32, 8, 128, 128, 4096, 4)),
        # a few requests behind a middling system prompt of odd length
        ("shared 5 x 1001", _shared(5, 1001, 300, 32, 8, 128, 64)),
        # a full decode batch behind one long document
        ("shared 64 x 16384", _shared(64, 16384, 1024, 32, 8, 128, 128)),
        # one sequence: penalties over its history, then the greedy token
        ("logits 1", _logits(1, 151936, 700, 0, False)),
        # a full decode batch with everything: penalties, 300 biases and a grammar on every other row
        ("logits 64", _logits(64, 151936, 4000, 300, True)),
    ]
    return [{"name": name, **c} for name, c in cases]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["extend", "release", "prompt", "prompt", "token", "token", "shared", "shared", "logits"])
    if kind == "extend":
        seqs = _log(rng, 1, 4096)
        return _extend(seqs, _log(rng, 1, 16384), min(_log(rng, 1, 2048), max(1, 250000 // seqs)), rng.choice([16, 32, 64, 128]),
                       rng.choice([0.0, 0.1, 0.5]))
    if kind == "release":
        return _release(_log(rng, 1, 4096), _log(rng, 1, 16384), rng.choice([16, 32, 64, 128]), rng.choice([0.05, 0.3, 1.0]))
    if kind == "prompt":
        nq, nkv, d = rng.choice([(32, 8, 128), (16, 8, 128), (16, 16, 64), (12, 4, 64), (32, 32, 128), (8, 2, 32), (4, 4, 16)])
        seqs, longest = _log(rng, 1, 24), _log(rng, 1, 16384)
        longest = min(longest, max(1, 65536 // seqs))
        window, sinks = _log(rng, 1, 8192), rng.choice([0, 1, 4, 64, 130])
        most = 32 * 32768 * 4096
        while seqs * longest * min(longest, window + sinks) * nq > most:
            longest = longest * 3 // 4
        return _prompt(seqs, longest, rng.random() < 0.7, nq, nkv, d, window, sinks)
    if kind == "token":
        nq, nkv, d = rng.choice([(32, 8, 128), (16, 8, 128), (28, 4, 128), (32, 32, 128), (12, 4, 64), (40, 2, 64), (8, 1, 128)])
        batch, longest = _log(rng, 1, 256), _log(rng, 1, 65536)
        window, sinks = _log(rng, 1, 16384), rng.choice([0, 1, 4, 64, 130])
        most = 64 * 4096 * 8 * 128
        if batch * min(longest, window + sinks) * nkv * d > most:
            batch = max(1, most // (min(longest, window + sinks) * nkv * d))
        return _token(batch, longest, rng.random() < 0.7, nq, nkv, d, rng.choice([64, 128]), window, sinks)
    if kind == "shared":
        nq, nkv, d = rng.choice([(32, 8, 128), (16, 8, 128), (28, 4, 128), (32, 32, 128), (12, 4, 64), (40, 2, 64), (8, 1, 128)])
        batch, prefix, longest = _log(rng, 1, 256), _log(rng, 1, 32768), _log(rng, 1, 2048)
        most = 64 * 16384 * 32
        if batch * prefix * nq > most:
            prefix = max(1, most // (batch * nq))
        if batch * longest * nkv * d > 64 * 1024 * 8 * 128:
            longest = max(1, 64 * 1024 * 8 * 128 // (batch * nkv * d))
        return _shared(batch, prefix, longest, nq, nkv, d, rng.choice([64, 128]))
    rows, vocab = _log(rng, 1, 64), _log(rng, 1000, 151936)
    return _logits(rows, vocab, _log(rng, 1, 4000), rng.choice([0, 1, 30, 300]), rng.random() < 0.5)


def _lengths(case):
    """The lengths of a case's sequences, the same for every seed: cached, kept and new tokens, or tokens of a prompt or a context.
    (Inputs of another seed have them in another order.)"""
    c = case
    r = random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))
    if c["kind"] == "extend":
        return [(r.randint(0, c["cached"]), 0 if r.random() < c["idle"] else (1 if c["new"] == 1 else r.randint(1, c["new"])))
                for _ in range(c["seqs"])]
    if c["kind"] == "release":
        cached = [r.randint(0, c["cached"]) for _ in range(c["seqs"])]
        return [(n, 0 if r.random() < c["finished"] else max(0, n - r.choice([0, 0, 1, 3]))) for n in cached]
    if c["kind"] == "shared":
        return [r.randint(0, c["longest"]) for _ in range(c["batch"])]
    count = c["seqs"] if c["kind"] == "prompt" else c["batch"]
    return [c["longest"]] + [r.randint(1, c["longest"]) if c["ragged"] else c["longest"] for _ in range(count - 1)]


def _visible(length, window, sinks):
    """Key positions that the last of ``length`` tokens attends to."""
    return min(length, min(sinks, max(0, length - window)) + window)


def _pairs(length, window, sinks):
    """The same, summed over all tokens of a prompt."""
    full = min(length, window + sinks)
    near = min(length, window)
    return near * (near + 1) // 2 + sum(range(near + 1, full + 1)) + (length - full) * (window + sinks)


def work(case):
    c = case
    kind = c["kind"]
    if kind == "logits":
        r, v = c["rows"], c["vocab"]
        extra = 4 * c["history"] / 2 + 8 * c["biases"] + (v / 16 if c["masks"] else 0)
        return {"bytes": r * (4 * v + extra), "flops": r * v}
    lens = _lengths(c)
    if kind in ("extend", "release"):
        s, bs = len(lens), c["block"]
        if kind == "extend":
            tokens = sum(m for _, m in lens)
            need = sum(-(-(n + m) // bs) - -(-n // bs) for n, m in lens)
            return {"bytes": 8 * s + 4 * s + 8 * need + 8 * s + 16 * tokens, "flops": 4 * tokens}
        drop = sum(-(-n // bs) - -(-k // bs) for n, k in lens)
        return {"bytes": 12 * s + 8 * drop, "flops": 2 * drop + s}
    nq, nkv, d = c["nq"], c["nkv"], c["d"]
    if kind == "prompt":
        return {"bytes": 2 * sum(lens) * d * (2 * nq + 2 * nkv),
                "flops": 4 * d * nq * sum(_pairs(n, c["window"], c["sinks"]) for n in lens)}
    b = c["batch"]
    if kind == "token":
        seen = sum(_visible(n, c["window"], c["sinks"]) for n in lens)
        return {"bytes": 4 * seen * nkv * d + 4 * b * nq * d, "flops": 4 * d * nq * seen}
    return {"bytes": 4 * (c["prefix"] + sum(lens)) * nkv * d + 4 * b * nq * d, "flops": 4 * d * nq * (b * c["prefix"] + sum(lens))}


# ----------------------------------------------------------------- inputs


def _normal(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(torch.bfloat16)


def _cache(g, blocks, nkv, block, d):
    """A cache half [blocks, nkv, block, d] of normal values, made in parts."""
    out = torch.empty(blocks, nkv, block, d, dtype=torch.bfloat16, device="cuda")
    part = max(1, (1 << 28) // (nkv * block * d))
    for at in range(0, blocks, part):
        n = min(part, blocks - at)
        out[at:at + n] = torch.randn(n, nkv, block, d, generator=g, device="cuda", dtype=torch.bfloat16)
    return out


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    r = random.Random(seed)
    c = dict(case)
    s = {"case": c}
    new = lambda *shape, t=torch.bfloat16: torch.empty(*shape, dtype=t, device="cuda")  # noqa: E731
    kind = c["kind"]
    if kind in ("extend", "release"):
        n, bs = c["seqs"], c["block"]
        lens = _lengths(case)
        r.shuffle(lens)
        cached = [x for x, _ in lens]
        more = [y for _, y in lens] if kind == "extend" else [0] * n
        if kind == "release":
            s["keep"], s["lens"] = _i32([y for _, y in lens]), new(n, t=torch.int32)
        held = [-(-x // bs) for x in cached]
        width = -(-(c["cached"] + (c["new"] if kind == "extend" else 0)) // bs)
        taken, blocks = sum(held), n * width + 64
        order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
        col = torch.arange(width, device="cuda")
        held_t = torch.tensor(held, device="cuda")
        first = held_t.cumsum(0) - held_t
        at = (first[:, None] + col).clamp(max=blocks - 1)
        s["tables"] = torch.where(col < held_t[:, None], order[at], torch.full_like(order[at], -1))
        s["free"] = torch.zeros(blocks, dtype=torch.int32, device="cuda")
        s["free"][:blocks - taken] = order[taken:]
        s["count"] = _i32([blocks - taken])
        s["cached"], s["left"], s["blocks"], s["width"] = _i32(cached), new(1, t=torch.int32), blocks, width
        if kind == "extend":
            cap = sum(more) + 3  # a batch padded to a few tokens more than there are
            s["more"], s["cap"] = _i32(more), cap
            s["ctx"], s["cu"], s["missing"] = new(n, t=torch.int32), new(n + 1, t=torch.int32), new(1, t=torch.int32)
            s["pos"], s["slots"] = new(cap, t=torch.int64), new(cap, t=torch.int64)
        return s
    if kind == "logits":
        rows, v, h = c["rows"], c["vocab"], c["history"]
        s["logits"] = _normal(g, rows, v, scale=2.0)
        lens = [r.randint(1, h) for _ in range(rows)]
        s["lens"], s["prompt"] = _i32(lens), _i32([r.randint(0, x) for x in lens])
        # repeated tokens as text has them: a skewed draw over the vocabulary
        s["history"] = (torch.rand(rows, h, generator=g, device="cuda") ** 4 * v).to(torch.int32).clamp_(max=v - 1)
        s["history"][:, ::3] = s["logits"][:, :].float().topk(min(v, 50), 1).indices[:, torch.randint(
            0, min(v, 50), (len(range(0, h, 3)),), generator=g, device="cuda")].to(torch.int32)
        s["rep"] = 1 + 0.3 * torch.rand(rows, generator=g, device="cuda")
        s["freq"] = 0.5 * torch.rand(rows, generator=g, device="cuda")
        s["pres"] = 0.5 * torch.rand(rows, generator=g, device="cuda")
        if c["biases"]:
            counts = [r.choice([0, c["biases"], c["biases"]]) for _ in range(rows)]
            starts = [0]
            for x in counts:
                starts.append(starts[-1] + x)
            n = max(1, starts[-1])
            s["starts"] = _i32(starts)
            s["bias_ids"] = torch.randint(0, v, (n,), generator=g, device="cuda").to(torch.int32)
            s["bias"] = 3 * torch.randn(n, generator=g, device="cuda")
            s["bias_row"] = torch.repeat_interleave(torch.arange(rows, device="cuda"), torch.tensor(counts, device="cuda"))
        if c["masks"]:
            words = (v + 31) // 32
            s["mask"] = torch.randint(-2**31, 2**31, ((rows + 1) // 2, words), generator=g, device="cuda").to(torch.int32)
            s["mask_rows"] = _i32([x // 2 if x % 2 == 0 else -1 for x in range(rows)])
        s["out"], s["next"] = new(rows, v), new(rows, t=torch.int64)
        return s
    nq, nkv, d = c["nq"], c["nkv"], c["d"]
    if kind == "prompt":
        lens = _lengths(case)
        r.shuffle(lens)
        cu = [0]
        for x in lens:
            cu.append(cu[-1] + x)
        # the fused projection's output, as the attention finds it: q heads, k heads, v heads side by side
        s["qkv"] = _normal(g, cu[-1], (nq + 2 * nkv) * d)
        s["qkv"][:, :nq * d] *= 2
        s["lens"], s["cu"], s["out"] = lens, _i32(cu), new(cu[-1], nq * d)
        return s
    b, bs = c["batch"], c["block"]
    lens = _lengths(case)
    r.shuffle(lens)
    s["q"] = _normal(g, b, nq * d, scale=2.0)
    s["out"] = new(b, nq * d)
    if kind == "token":
        # a cache that keeps only what the window still needs: other entries of the tables are stale
        entries = []
        for n in lens:
            lo, first = max(0, n - c["window"]), min(n, c["sinks"])
            entries.append(sorted(set(range(-(-first // bs))) | set(range(lo // bs, -(-n // bs)))))
        blocks = sum(len(e) for e in entries) + 1
        order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32).cpu().tolist()
        width = -(-c["longest"] // bs)
        tables, at = torch.full((b, width), -1, dtype=torch.int32), 0
        for i, e in enumerate(entries):
            tables[i, torch.tensor(e)] = torch.tensor(order[at:at + len(e)], dtype=torch.int32)
            at += len(e)
        s["tables"], s["ctx"] = tables.cuda(), _i32(lens)
    else:
        held, head = [-(-x // bs) for x in lens], -(-c["prefix"] // bs)
        width = max(max(held), 1)
        blocks = sum(held) + head + 1
        order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
        col, held_t = torch.arange(width, device="cuda"), torch.tensor(held, device="cuda")
        at = (head + (held_t.cumsum(0) - held_t)[:, None] + col).clamp(max=blocks - 1)
        s["tables"] = torch.where(col < held_t[:, None], order[at], torch.full_like(order[at], -1))
        s["prefix"], s["prefix_len"], s["ctx"] = order[:head].contiguous(), _i32([c["prefix"]]), _i32(lens)
        if own:
            from atb_llm_study_b200 import capi

            s["ws_bytes"] = capi.lib().b200_paged_decode_shared_workspace_bytes(b, nq, nkv, d, c["prefix"])
            s["ws"] = new(max(16, s["ws_bytes"]), t=torch.uint8)
    s["blocks"], s["width"] = blocks, width
    s["k"], s["v"] = _cache(g, blocks, nkv, bs, d), _cache(g, blocks, nkv, bs, d)
    return s


# ------------------------------------------------------------- plain forms


def _plain_extend(s):
    c, bs = s["case"], s["case"]["block"]
    cached, more, count = s["cached"].long(), s["more"].long(), s["count"].long()
    held, total = (cached + bs - 1) // bs, (cached + more + bs - 1) // bs
    need = total - held
    first = need.cumsum(0) - need
    missing = (need.sum() - count).clamp(min=0)
    fits = missing == 0
    more = more * fits
    col = torch.arange(s["width"], device="cuda")
    fresh = (col >= held[:, None]) & (col < total[:, None]) & fits
    take = (count - 1 - first[:, None] - (col - held[:, None])).clamp(0, s["free"].numel() - 1)
    tables = torch.where(fresh, s["free"][take], s["tables"])
    cu = torch.cat([more.new_zeros(1), more.cumsum(0)])
    t = torch.arange(s["cap"], device="cuda")
    starts = torch.zeros(s["cap"] + 1, dtype=torch.int64, device="cuda").index_add_(0, cu[1:], torch.ones_like(more))
    seq = starts.cumsum(0)[:-1].clamp(max=c["seqs"] - 1)  # sequences that end at or before each token
    real = (t < cu[-1]) & fits
    pos = torch.where(real, cached[seq] + t - cu[seq], torch.zeros_like(t))
    block = tables[seq, (pos // bs).clamp(max=s["width"] - 1)].long()
    slots = torch.where(real, block * bs + pos % bs, torch.full_like(pos, -1))
    ctx = cached + more
    left = torch.where(fits, count - need.sum(), count)
    i32 = torch.int32
    return tables, ctx.to(i32), cu.to(i32), pos, slots, left.to(i32), missing.to(i32)


def _plain_release(s):
    bs = s["case"]["block"]
    cached, count = s["cached"].long(), s["count"].long()
    lens = torch.minimum(cached, s["keep"].long())
    kept, held = (lens + bs - 1) // bs, (cached + bs - 1) // bs
    drop = held - kept
    first = drop.cumsum(0) - drop
    col = torch.arange(s["width"], device="cuda")
    goes = (col >= kept[:, None]) & (col < held[:, None])
    size = s["free"].numel()
    to = torch.where(goes, count + first[:, None] + col - kept[:, None], torch.full_like(goes, size, dtype=torch.int64))
    free = torch.cat([s["free"], s["free"][:1]])
    free = free.scatter(0, to.reshape(-1), s["tables"].reshape(-1))[:size]
    return free, lens.to(torch.int32), (count + drop.sum()).to(torch.int32)


def _softmax_parts(scores, mask):
    """exp(scores - max) and their sums under a mask; rows with nothing visible give zeros."""
    low = torch.where(mask, scores, torch.full_like(scores, -math.inf))
    top = low.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, torch.zeros_like(top))
    p = torch.exp(low - top)
    return p, p.sum(-1, keepdim=True)


def _plain_prompt(s):
    c = s["case"]
    nq, nkv, d, w, sinks = c["nq"], c["nkv"], c["d"], c["window"], c["sinks"]
    rep = nq // nkv
    out, at = s["out"], 0
    for n in s["lens"]:
        x = s["qkv"][at:at + n].float()
        q = x[:, :nq * d].reshape(n, nkv, rep, d).permute(1, 2, 0, 3)
        k = x[:, nq * d:(nq + nkv) * d].reshape(n, nkv, d).transpose(0, 1)
        v = x[:, (nq + nkv) * d:].reshape(n, nkv, d).transpose(0, 1)
        for i0 in range(0, n, 1024):
            i1 = min(n, i0 + 1024)
            lo = max(0, i0 - w + 1)
            j = torch.cat([torch.arange(min(sinks, lo), device="cuda"), torch.arange(lo, i1, device="cuda")])
            i = torch.arange(i0, i1, device="cuda")[:, None]
            mask = (j <= i) & ((i - j < w) | (j < sinks))
            scores = q[:, :, i0:i1].reshape(nkv, -1, d) @ k[:, j].transpose(1, 2) / math.sqrt(d)
            p, total = _softmax_parts(scores.reshape(nkv, rep, i1 - i0, -1), mask)
            o = (p.reshape(nkv, -1, p.shape[-1]) @ v[:, j]).reshape(nkv, rep, i1 - i0, d) / total
            out[at + i0:at + i1] = o.permute(2, 0, 1, 3).reshape(i1 - i0, nq * d).to(torch.bfloat16)
        at += n
    return out


def _rows(cache, table, pos, bs):
    """Cached rows (fp32) of positions ``pos`` [b, n] of the tables' sequences: [b, nkv, n, d]."""
    block = table.gather(1, pos // bs).long().clamp(min=0)
    return cache[block, :, pos % bs].float().transpose(1, 2)


def _plain_token(s):
    c = s["case"]
    nq, nkv, d, w, sinks, bs = c["nq"], c["nkv"], c["d"], c["window"], c["sinks"], c["block"]
    width = _visible(c["longest"], w, sinks)
    out = s["out"]
    part = max(1, (1 << 28) // (width * nkv * d))
    for at in range(0, c["batch"], part):
        ctx = s["ctx"][at:at + part].long()[:, None]
        j = torch.arange(width, device="cuda")
        gap = torch.minimum(torch.full_like(ctx, sinks), (ctx - w).clamp(min=0))  # first tokens that lie before the window
        pos = torch.where(j < gap, j, (ctx - w).clamp(min=0) + j - gap)
        mask = (pos < ctx)[:, None, None]
        pos = torch.minimum(pos, ctx - 1)
        k, v = (_rows(s[x], s["tables"][at:at + part], pos, bs) for x in "kv")
        q = s["q"][at:at + part].float().view(-1, nkv, nq // nkv, d)
        p, total = _softmax_parts(q @ k.transpose(2, 3) / math.sqrt(d), mask)
        out[at:at + part] = (p @ v / total).reshape(-1, nq * d).to(torch.bfloat16)
    return out


def _plain_shared(s):
    c = s["case"]
    b, nq, nkv, d, bs, n = c["batch"], c["nq"], c["nkv"], c["d"], c["block"], c["prefix"]
    rep = nq // nkv
    q = s["q"].float().view(b, nkv, rep, d)
    pos = torch.arange(n, device="cuda")[None]
    k, v = (_rows(s[x], s["prefix"][None], pos, bs)[0] for x in "kv")  # [nkv, n, d]
    head = q.transpose(0, 1).reshape(nkv, b * rep, d) @ k.transpose(1, 2) / math.sqrt(d)
    head = head.view(nkv, b, rep, n).transpose(0, 1)
    j = torch.arange(max(1, c["longest"]), device="cuda")
    ctx = s["ctx"].long()[:, None]
    ko, vo = (_rows(s[x], s["tables"], torch.minimum(j, (ctx - 1).clamp(min=0)), bs) for x in "kv")
    own_scores = q @ ko.transpose(2, 3) / math.sqrt(d)
    mask = torch.cat([torch.ones(b, n, dtype=torch.bool, device="cuda"), j < ctx], 1)[:, None, None]
    p, total = _softmax_parts(torch.cat([head, own_scores], 3), mask)
    o = (p[..., :n].transpose(0, 1).reshape(nkv, b * rep, n) @ v).view(nkv, b, rep, d).transpose(0, 1)
    return ((o + p[..., n:] @ vo) / total).reshape(b, nq * d).to(torch.bfloat16)


def _plain_logits(s):
    c = s["case"]
    rows, v, h = c["rows"], c["vocab"], c["history"]
    x = s["logits"].double()  # values next to each other decide the greedy token
    at = torch.arange(h, device="cuda")
    ids = s["history"].long()
    nowhere = torch.full_like(ids, v)
    spoken = torch.where(at < s["lens"][:, None], ids, nowhere)
    answer = torch.where(at >= s["prompt"][:, None], spoken, nowhere)
    ones = torch.ones_like(ids, dtype=torch.float64)
    seen = torch.zeros(rows, v + 1, dtype=torch.float64, device="cuda").scatter_add_(1, spoken, ones)[:, :v] > 0
    said = torch.zeros(rows, v + 1, dtype=torch.float64, device="cuda").scatter_add_(1, answer, ones)[:, :v]
    rep, freq, pres = (s[n].double()[:, None] for n in ("rep", "freq", "pres"))
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - freq * said - pres * (said > 0)
    if c["biases"]:
        n = s["bias_row"].numel()
        x.view(-1).index_add_(0, s["bias_row"] * v + s["bias_ids"][:n].long(), s["bias"][:n].double())
    if c["masks"]:
        col = torch.arange(v, device="cuda")
        bit = (s["mask"][s["mask_rows"].clamp(min=0).long()][:, col // 32] >> (col % 32)) & 1
        allowed = (bit == 1) | (s["mask_rows"] < 0)[:, None]
        x = torch.where(allowed, x, torch.full_like(x, -math.inf))
    top = x.amax(1, keepdim=True)
    first = torch.where(x == top, torch.arange(v, device="cuda"), torch.full((1, 1), v, device="cuda")).amin(1)
    return x.to(torch.bfloat16), first


# --------------------------------------------------------- framework calls


def _own_extend(L, check, st, s):
    c = s["case"]
    check(L.b200_block_tables_extend(s["cached"].data_ptr(), s["more"].data_ptr(), c["seqs"], c["block"],
                                     s["tables"].data_ptr(), s["width"], s["free"].data_ptr(), s["count"].data_ptr(),
                                     s["blocks"], s["ctx"].data_ptr(), s["cu"].data_ptr(), s["pos"].data_ptr(),
                                     s["slots"].data_ptr(), s["cap"], s["left"].data_ptr(), s["missing"].data_ptr(), st),
          "block_tables_extend")
    return s["tables"], s["ctx"], s["cu"], s["pos"], s["slots"], s["left"], s["missing"]


def _own_release(L, check, st, s):
    c = s["case"]
    check(L.b200_block_tables_release(s["cached"].data_ptr(), s["keep"].data_ptr(), c["seqs"], c["block"],
                                      s["tables"].data_ptr(), s["width"], s["free"].data_ptr(), s["free"].numel(),
                                      s["count"].data_ptr(), s["blocks"], s["lens"].data_ptr(), s["left"].data_ptr(), st),
          "block_tables_release")
    return s["free"], s["lens"], s["left"]


def _own_prompt(L, check, st, s):
    c = s["case"]
    nq, nkv, d = c["nq"], c["nkv"], c["d"]
    x, row = s["qkv"].data_ptr(), (nq + 2 * nkv) * d
    check(L.b200_flash_prefill_window(x, row, d, x + 2 * nq * d, row, d, x + 2 * (nq + nkv) * d, row, d,
                                      s["out"].data_ptr(), nq * d, d, s["cu"].data_ptr(), c["seqs"], c["longest"],
                                      s["out"].shape[0], nq, nkv, d, d, 1 / math.sqrt(d), c["window"], c["sinks"], st),
          "flash_prefill_window")
    return s["out"]


def _own_token(L, check, st, s):
    c = s["case"]
    nq, nkv, d = c["nq"], c["nkv"], c["d"]
    check(L.b200_paged_decode_window(s["q"].data_ptr(), nq * d, s["k"].data_ptr(), s["v"].data_ptr(),
                                     s["tables"].data_ptr(), s["width"], s["ctx"].data_ptr(), c["batch"], nq, nkv, d,
                                     c["block"], s["blocks"], 1 / math.sqrt(d), c["window"], c["sinks"],
                                     s["out"].data_ptr(), nq * d, c["longest"], st), "paged_decode_window")
    return s["out"]


def _own_shared(L, check, st, s):
    c = s["case"]
    nq, nkv, d = c["nq"], c["nkv"], c["d"]
    check(L.b200_paged_decode_shared(s["q"].data_ptr(), nq * d, s["k"].data_ptr(), s["v"].data_ptr(),
                                     s["prefix"].data_ptr(), s["prefix_len"].data_ptr(), c["prefix"],
                                     s["tables"].data_ptr(), s["width"], s["ctx"].data_ptr(),
                                     min(c["longest"], s["width"] * c["block"]), c["batch"],
                                     nq, nkv, d, c["block"], s["blocks"], 1 / math.sqrt(d), s["out"].data_ptr(), nq * d,
                                     s["ws"].data_ptr(), s["ws_bytes"], st), "paged_decode_shared")
    return s["out"]


def _own_logits(L, check, st, s):
    c = s["case"]
    v = c["vocab"]
    at = lambda name: s[name].data_ptr() if name in s else None  # noqa: E731
    check(L.b200_logits_process(s["logits"].data_ptr(), v, c["rows"], v, at("history"), c["history"], at("prompt"),
                                at("lens"), at("rep"), at("freq"), at("pres"), at("starts"), at("bias_ids"), at("bias"),
                                at("mask"), (v + 31) // 32, s["mask"].shape[0] if "mask" in s else 0, at("mask_rows"),
                                s["out"].data_ptr(), v, s["next"].data_ptr(), st), "logits_process")
    return s["out"], s["next"]


def run(state):
    kind = state["case"]["kind"]
    if own:
        from atb_llm_study_b200 import capi

        call = {"extend": _own_extend, "release": _own_release, "prompt": _own_prompt, "token": _own_token,
                "shared": _own_shared, "logits": _own_logits}[kind]
        return call(capi.lib(), capi.check, torch.cuda.current_stream().cuda_stream, state)
    return {"extend": _plain_extend, "release": _plain_release, "prompt": _plain_prompt, "token": _plain_token,
            "shared": _plain_shared, "logits": _plain_logits}[kind](state)


# --------------------------------------------------------- 64-bit reference


def _attend64(q, k, v, seen=None):
    """q [m, d] over k, v [n, d] (float64), keys where ``seen`` [m, n] is true."""
    x = torch.einsum("md,nd->mn", q, k) * q.shape[1] ** -0.5
    if seen is not None:
        x = x.masked_fill(~seen, -math.inf)
    return torch.exp(x - torch.logsumexp(x, 1, keepdim=True)) @ v


def _history64(s, c):
    """Lists of the rows' prompt and answer tokens."""
    ids, lens, prompt = (s[n].cpu().tolist() for n in ("history", "lens", "prompt"))
    return [(ids[i][:prompt[i]], ids[i][prompt[i]:lens[i]]) for i in range(c["rows"])]


def exact(case, seed):
    s = prepare(case, seed)
    c, kind = case, case["kind"]
    if kind in ("extend", "release"):
        import numpy as np

        bs, count = c["block"], int(s["count"])
        cached, tables, free = (s[n].cpu().numpy().copy() for n in ("cached", "tables", "free"))
        if kind == "release":
            keep, top = s["keep"].cpu().numpy(), count
            for i in range(c["seqs"]):
                for j in range(-(-int(min(keep[i], cached[i])) // bs), -(-int(cached[i]) // bs)):
                    free[top] = tables[i, j]
                    top += 1
            return free, np.minimum(cached, keep), np.array([top], np.int32)
        more, pos, slots = s["more"].cpu().numpy(), [], []
        for i in range(c["seqs"]):
            for j in range(-(-int(cached[i]) // bs), -(-int(cached[i] + more[i]) // bs)):
                count -= 1  # prepare leaves enough free blocks
                tables[i, j] = free[count]
            p = np.arange(cached[i], cached[i] + more[i], dtype=np.int64)
            pos.append(p)
            slots.append(tables[i, p // bs].astype(np.int64) * bs + p % bs)
        pad = s["cap"] - int(more.sum())
        pos, slots = np.concatenate(pos + [np.zeros(pad, np.int64)]), np.concatenate(slots + [np.full(pad, -1, np.int64)])
        return (tables, (cached + more).astype(np.int32), np.concatenate([[0], np.cumsum(more)]).astype(np.int32), pos, slots,
                np.array([count], np.int32), np.zeros(1, np.int32))
    if kind == "logits":
        x = s["logits"].double()
        v = c["vocab"]
        for i, (prompt, answer) in enumerate(_history64(s, c)):
            counts = torch.bincount(torch.tensor(answer, dtype=torch.int64), minlength=v).double().cuda()
            both = torch.tensor(sorted(set(prompt) | set(answer)), dtype=torch.int64, device="cuda")
            value = x[i, both]
            x[i, both] = value * torch.where(value > 0, 1 / s["rep"][i].double(), s["rep"][i].double())
            x[i] -= counts * s["freq"][i].double() + counts.clamp(max=1) * s["pres"][i].double()
            if c["biases"]:
                lo, hi = int(s["starts"][i]), int(s["starts"][i + 1])
                for token, value in zip(s["bias_ids"][lo:hi].tolist(), s["bias"][lo:hi].tolist()):
                    x[i, token] += value
            if c["masks"] and i % 2 == 0:
                words = s["mask"][i // 2].cpu().numpy().view("uint8")
                import numpy as np

                bits = np.unpackbits(words, bitorder="little")[:v]
                x[i, torch.from_numpy(bits == 0).cuda()] = -math.inf
        return x, x.max(1, keepdim=True).values.eq(x).int().argmax(1)
    nq, nkv, d = c["nq"], c["nkv"], c["d"]
    rep = nq // nkv
    out = torch.empty(s["out"].shape, dtype=torch.float64, device="cuda")
    if kind == "prompt":
        at = 0
        for n in s["lens"]:
            x = s["qkv"][at:at + n].double().view(n, nq + 2 * nkv, d)
            for i0 in range(0, n, 2048):
                i = torch.arange(i0, min(n, i0 + 2048), device="cuda")[:, None]
                lo = max(0, i0 - c["window"] + 1)
                keys = torch.tensor([*range(min(lo, c["sinks"])), *range(lo, int(i[-1]) + 1)], device="cuda")
                seen = (keys <= i) & ((keys > i - c["window"]) | (keys < c["sinks"]))
                for h in range(nq):
                    kv = nq + h // rep
                    out[at + i0:at + i0 + len(i), h * d:(h + 1) * d] = _attend64(x[i0:i0 + len(i), h], x[keys, kv], x[keys, kv + nkv],
                                                                                seen)
            at += n
        return out
    bs = c["block"]
    q = s["q"].double().view(-1, nkv, rep, d)
    for b, n in enumerate(s["ctx"].tolist()):
        if kind == "token":
            pos = [p for p in range(n) if p >= n - c["window"] or p < c["sinks"]] if n < 4096 else [
                *range(min(c["sinks"], max(0, n - c["window"]))), *range(max(0, n - c["window"]), n)]
            pos = torch.tensor(pos, device="cuda")
            block, off = s["tables"][b, pos // bs].long(), pos % bs
        else:
            pos, head = torch.arange(n, device="cuda"), torch.arange(c["prefix"], device="cuda")
            block = torch.cat([s["prefix"][head // bs], s["tables"][b, pos // bs]]).long()
            off = torch.cat([head % bs, pos % bs])
        for h in range(nkv):
            k, v = s["k"][block, h, off].double(), s["v"][block, h, off].double()
            out[b, h * rep * d:(h + 1) * rep * d] = _attend64(q[b, h], k, v).reshape(-1)
    return out
