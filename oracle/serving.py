"""float64 restatements of a serving step's operators: block tables from request
lengths, window and shared-prefix attention, logits processing.

The reference only declares a KV-cache manager
(atb_cpp_llm/src/core/kv_cache_manager.h:25-76), masks with the causal rule
alone (atb_cpp_llm/src/runners/text_runner.cpp:74-85) and chooses no token
(atb_cpp_llm/include/atb_llm/model.h:47-50), so these follow the definitions in
include/b200_llm.h.  Attention comes with ``weight``, the softmax-weighted mean
of |v|, which error bounds are relative to.
"""

import numpy as np


def attend(q, k, v, seen, scale):
    """q [m, d], k [n, d], v [n, dv], seen [m, n] -> (out [m, dv], weight [m, dv]); rows that see nothing give zeros."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    out, weight = np.zeros((q.shape[0], v.shape[1])), np.zeros((q.shape[0], v.shape[1]))
    for cols in np.unique(seen, axis=0):  # what no row of a kind sees takes no part, NaN included
        rows = (seen == cols).all(1)
        if not cols.any():
            continue
        s = q[rows] @ k[cols].T * scale
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        out[rows], weight[rows] = p @ v[cols], p @ np.abs(v[cols])
    return out, weight


def window_mask(n, window, sinks):
    i, j = np.arange(n)[:, None], np.arange(n)[None]
    return (j <= i) & ((i - j < window) | (j < sinks))


def window_prompt(q, k, v, lens, window, sinks, scale):
    """q [T, nq, d], k / v [T, nkv, .] of packed prompts."""
    nq, nkv = q.shape[1], k.shape[1]
    out, weight = (np.zeros((q.shape[0], nq, v.shape[2])) for _ in range(2))
    at = 0
    for n in lens:
        s = slice(at, at + n)
        mask = window_mask(n, window, sinks)
        for h in range(nq):
            out[s, h], weight[s, h] = attend(q[s, h], k[s, h * nkv // nq], v[s, h * nkv // nq], mask, scale)
        at += n
    return out, weight


def cached_rows(cache, table, positions):
    """cache [blocks, nkv, bs, d] -> [len(positions), nkv, d]"""
    bs = cache.shape[2]
    positions = np.asarray(positions, np.int64)
    return cache[np.asarray(table, np.int64)[positions // bs], :, positions % bs]


def paged(q, rows):
    """q [nq, d] over (k, v) rows [n, nkv, d] -> (out, weight) [nq, d]"""
    k, v = rows
    nq, nkv = q.shape[0], k.shape[1]
    pairs = [attend(q[h:h + 1], k[:, h * nkv // nq], v[:, h * nkv // nq], np.ones((1, len(k)), bool), q.shape[1] ** -0.5)
             for h in range(nq)]
    return np.concatenate([o for o, _ in pairs]), np.concatenate([w for _, w in pairs])


def window_decode(q, kc, vc, tables, context, window, sinks):
    """q [B, nq, d]; only visible positions are looked up."""
    out = []
    for b, n in enumerate(context):
        pos = [j for j in range(n) if j >= n - window or j < sinks]
        out.append(paged(q[b], [cached_rows(c, tables[b], pos) for c in (kc, vc)]))
    return np.stack([o for o, _ in out]), np.stack([w for _, w in out])


def shared_decode(q, kc, vc, prefix, prefix_len, tables, context):
    out = []
    for b, n in enumerate(context):
        rows = [np.concatenate([cached_rows(c, prefix, np.arange(prefix_len)), cached_rows(c, tables[b], np.arange(n))])
                for c in (kc, vc)]
        out.append(paged(q[b], rows))
    return np.stack([o for o, _ in out]), np.stack([w for _, w in out])


def extend(cached, new, bs, tables, free, count, capacity):
    """-> tables, context, cu, positions, slots, free_left, missing (arguments in range)"""
    cached, new, tables = np.asarray(cached), np.asarray(new), np.array(tables)
    ceil = lambda x: -(-x // bs)  # noqa: E731
    need = int((ceil(cached + new) - ceil(cached)).sum())
    pos, slots = np.zeros(capacity, np.int64), np.full(capacity, -1, np.int64)
    if need > count:
        return tables, cached, np.zeros(len(new) + 1, np.int32), pos, slots, count, need - count
    t = 0
    for i in range(len(new)):
        for p in range(cached[i], cached[i] + new[i]):
            if p % bs == 0:
                count -= 1
                tables[i, p // bs] = free[count]
            pos[t], slots[t] = p, np.int64(tables[i, p // bs]) * bs + p % bs
            t += 1
    return tables, cached + new, np.concatenate([[0], np.cumsum(new)]), pos, slots, count, 0


def release(cached, keep, bs, tables, free, count):
    """-> free, lens, free_left"""
    free, lens = np.array(free), np.minimum(cached, keep)
    for i in range(len(lens)):
        for j in range(-(-int(lens[i]) // bs), -(-int(cached[i]) // bs)):
            free[count] = tables[i, j]
            count += 1
    return free, lens, count


def logits(x, prompts=None, answers=None, repetition=None, frequency=None, presence=None, biases=None, allowed=None):
    """One row: x [V]; token lists; biases [(token, value)]; allowed [V] bool -> (values, next)"""
    x = np.array(x, np.float64)
    if prompts is not None:
        said = {}
        for t in answers:
            said[t] = said.get(t, 0) + 1
        for t in set(prompts) | set(answers):
            if repetition is not None:
                x[t] = x[t] / np.float64(repetition) if x[t] > 0 else x[t] * np.float64(repetition)
            if frequency is not None:
                x[t] = x[t] - np.float64(frequency) * said.get(t, 0)
            if presence is not None and t in said:
                x[t] = x[t] - np.float64(presence)
    sums = {}
    for t, v in biases or []:
        sums[t] = sums[t] + np.float64(v) if t in sums else np.float64(v)
    for t, v in sums.items():
        x[t] += v
    if allowed is not None:
        x[~allowed] = -np.inf
    best = np.where(np.isnan(x), -np.inf, x)
    return x, int(best.argmax()) if best.max() > -np.inf else -1
