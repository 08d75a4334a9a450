"""GPU parity of block tables from request lengths and of logits processing with
the float64 restatements in oracle.serving, and a run of a serving step's calls
together.

Tables and tokens are whole numbers: equal.  Logits are computed in double and
rounded once: within half a step of bf16, 2^-8 relative (and bit for bit where
nothing touches a token)."""

import numpy as np
import pytest
import torch

from oracle import serving
from test_gpu_window import close

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import gpu_util as G

BAD_INDEX = 2
I32 = torch.int32


# ------------------------------------------------------------ block tables


def pool(seed, cached, width, bs, blocks):
    """Tables of the cached tokens and the free list, blocks shuffled."""
    rng = np.random.default_rng(seed)
    order = rng.permutation(blocks).astype(np.int32)
    held = -(-np.asarray(cached, np.int64) // bs)
    tables, at = np.full((len(cached), width), -1, np.int32), 0
    for i, n in enumerate(held):
        tables[i, :n] = order[at:at + n]
        at += n
    return tables, np.concatenate([order[at:], np.full(at, -7, np.int32)]), blocks - at


def extend_call(cached, new, bs, tables, free, count, blocks, capacity, in_place=False):
    n = len(cached)
    d = dict(cached=G.i32(cached), new=G.i32(new), tables=G.i32(tables), free=G.i32(free), count=G.i32([count]),
             cu=torch.full((n + 2,), -9, dtype=I32, device=G.DEV), missing=torch.full((1,), -9, dtype=I32, device=G.DEV),
             pos=torch.full((capacity + 1,), -9, dtype=torch.int64, device=G.DEV),
             slots=torch.full((capacity + 1,), -9, dtype=torch.int64, device=G.DEV))
    d["ctx"] = d["cached"] if in_place else torch.full((n,), -9, dtype=I32, device=G.DEV)
    d["left"] = d["count"] if in_place else torch.full((1,), -9, dtype=I32, device=G.DEV)
    G.check(G.L().b200_block_tables_extend(d["cached"].data_ptr(), d["new"].data_ptr(), n, bs, d["tables"].data_ptr(),
                                           tables.shape[1], d["free"].data_ptr(), d["count"].data_ptr(), blocks,
                                           d["ctx"].data_ptr(), d["cu"].data_ptr(), d["pos"].data_ptr(), d["slots"].data_ptr(),
                                           capacity, d["left"].data_ptr(), d["missing"].data_ptr(), G.stream()), "extend")
    return {k: v.cpu().numpy() for k, v in d.items()}


def check_extend(cached, new, bs, width, capacity, blocks=None, in_place=False, seed=0):
    cached, new = np.asarray(cached, np.int32), np.asarray(new, np.int32)
    blocks = blocks or int((-(-(cached.astype(np.int64) + new) // bs)).sum()) + 2
    tables, free, count = pool(seed, cached, width, bs, blocks)
    got = extend_call(cached, new, bs, tables, free, count, blocks, capacity, in_place)
    want = serving.extend(cached, new, bs, tables, free, count, capacity)
    for name, w in zip(("tables", "ctx", "cu", "pos", "slots", "left", "missing"), want):
        g = got[name]
        if name in ("cu", "pos", "slots"):
            assert g[-1] == -9
            g = g[:-1]
        np.testing.assert_array_equal(g, np.broadcast_to(w, g.shape), err_msg=name)
    np.testing.assert_array_equal(got["free"], free)
    assert G.device_errors() == 0
    return got


@pytest.mark.parametrize("bs", [1, 7, 16, 64, 128])
@pytest.mark.parametrize("n,most,new,pad", [(1, 0, 1, 0), (1, 200, 300, 5), (3, 50, 0, 2), (64, 300, 1, 0), (500, 100, 9, 1000),
                                            (1024, 20, 3, 1), (1025, 20, 3, 0), (2500, 9, 5, 77)])
@pytest.mark.parametrize("in_place", [False, True], ids=["", "in-place"])
def test_extend(bs, n, most, new, pad, in_place):
    rng = np.random.default_rng(n + bs)
    cached, more = rng.integers(0, most + 1, n), rng.integers(0, new + 1, n)
    more[rng.random(n) < 0.3] = 0
    check_extend(cached, more, bs, -(-(most + new) // bs) + 1, int(more.sum()) + pad, in_place=in_place, seed=n)


def test_extend_lengths_at_the_ends():
    check_extend([0] * 8192, [0] * 8191 + [5], 4, 3, 5)  # long runs without tokens
    check_extend([0] + [0] * 8191, [700] + [0] * 8190 + [1], 16, 50, 900)
    check_extend([63, 64, 65, 127, 128], [1, 1, 1, 1, 1], 64, 3, 5)
    check_extend([0, 100], [40000, 3], 64, 700, 50000)  # one long prompt: many entries in a row
    check_extend([], [], 64, 1, 3, blocks=5)


def test_extend_without_enough_blocks_takes_nothing():
    cached, new = np.array([10, 0, 5], np.int32), np.array([60, 100, 0], np.int32)
    for spare, missing in ((3, 0), (2, 1), (0, 3)):
        tables, free, _ = pool(1, cached, 4, 64, 12)
        got = extend_call(cached, new, 64, tables, free, spare, 12, 200)
        want = serving.extend(cached, new, 64, tables, free, spare, 200)
        assert got["missing"] == missing == want[6]
        for name, w in zip(("tables", "ctx", "cu", "pos", "slots", "left"), want):
            g = got[name][:-1] if name in ("cu", "pos", "slots") else got[name]
            np.testing.assert_array_equal(g, np.broadcast_to(w, g.shape), err_msg=name)
        assert G.device_errors() == 0


@pytest.mark.parametrize("cached,new,count,capacity", [([10, -1], [1, 1], 5, 9), ([10, 0], [1, -2], 5, 9), ([250, 0], [7, 1], 5, 9),
                                                       ([10, 0], [5, 5], 5, 9), ([10, 0], [1, 1], -1, 9), ([10, 0], [1, 1], 99, 9),
                                                       ([2**31 - 1, 0], [2**31 - 1, 1], 5, 9)])
def test_extend_refuses_lengths_on_the_device(cached, new, count, capacity):
    tables, free, _ = pool(2, [10, 0], 4, 64, 12)
    for in_place in (False, True):
        got = extend_call(cached, new, 64, tables, free, count, 12, capacity, in_place)
        assert G.device_errors() == BAD_INDEX and got["missing"] == -1 and got["left"] == count
        np.testing.assert_array_equal(got["tables"], tables)
        np.testing.assert_array_equal(got["ctx"], cached)
        assert (got["slots"][:-1] == -1).all() and (got["pos"][:-1] == 0).all() and (got["cu"][:-1] == 0).all()


def test_extend_bad_blocks_give_no_slots():
    tables, free, count = pool(3, [10, 0], 2, 64, 12)
    tables[0, 0], free[count - 1] = 12, -3
    got = extend_call([10, 0], [2, 2], 64, tables, free, count, 12, 4)
    assert G.device_errors() == BAD_INDEX and (got["slots"][:4] == -1).all() and got["tables"][1, 0] == -1


def test_extend_without_optional_outputs():
    cached, new = G.i32([10, 0]), G.i32([60, 3])
    tables, free, count = pool(4, [10, 0], 2, 64, 12)
    t, f, c, left = G.i32(tables), G.i32(free), G.i32([count]), G.i32([0])
    ctx = G.i32([0, 0])
    G.check(G.L().b200_block_tables_extend(cached.data_ptr(), new.data_ptr(), 2, 64, t.data_ptr(), 2, f.data_ptr(), c.data_ptr(), 12,
                                           ctx.data_ptr(), None, None, None, 1000, left.data_ptr(), None, G.stream()))
    want = serving.extend(np.array([10, 0]), np.array([60, 3]), 64, tables, free, count, 1000)
    np.testing.assert_array_equal(t.cpu().numpy(), want[0])
    assert ctx.tolist() == [70, 3] and left.item() == want[5]


def release_call(cached, keep, bs, tables, free, count, blocks, in_place=False, capacity=None):
    d = dict(cached=G.i32(cached), keep=G.i32(keep), tables=G.i32(tables), free=G.i32(free), count=G.i32([count]))
    d["lens"] = d["cached"] if in_place else torch.full((len(cached),), -9, dtype=I32, device=G.DEV)
    d["left"] = d["count"] if in_place else torch.full((1,), -9, dtype=I32, device=G.DEV)
    G.check(G.L().b200_block_tables_release(d["cached"].data_ptr(), d["keep"].data_ptr(), len(cached), bs, d["tables"].data_ptr(),
                                            tables.shape[1], d["free"].data_ptr(), len(free) if capacity is None else capacity,
                                            d["count"].data_ptr(), blocks, d["lens"].data_ptr(), d["left"].data_ptr(),
                                            G.stream()), "release")
    return {k: v.cpu().numpy() for k, v in d.items()}


@pytest.mark.parametrize("bs", [1, 16, 64])
@pytest.mark.parametrize("n,most", [(1, 100), (3, 0), (300, 200), (1024, 9), (5000, 30)])
@pytest.mark.parametrize("in_place", [False, True], ids=["", "in-place"])
def test_release(bs, n, most, in_place):
    rng = np.random.default_rng(n + bs)
    cached = rng.integers(0, most + 1, n)
    keep = np.where(rng.random(n) < 0.4, 0, cached - rng.integers(-2, 4, n)).clip(0)
    blocks = int((-(-cached // bs)).sum()) + 3
    tables, free, count = pool(n, cached, -(-most // bs) + 1, bs, blocks)
    got = release_call(cached, keep, bs, tables, free, count, blocks, in_place)
    want = serving.release(cached, keep, bs, tables, free, count)
    np.testing.assert_array_equal(got["free"], want[0])
    np.testing.assert_array_equal(got["lens"], want[1])
    assert got["left"] == want[2] and (got["tables"] == tables).all() and G.device_errors() == 0


def test_release_refuses_on_the_device():
    tables, free, count = pool(5, [100, 30], 2, 64, 12)
    for cached, keep, c, cap in (([100, -3], [0, 0], count, 12), ([100, 30], [0, -1], count, 12), ([129, 30], [0, 0], count, 12),
                                 ([100, 30], [0, 0], 10, 12), ([100, 30], [0, 0], -1, 12), ([100, 30], [0, 0], count, 11)):
        got = release_call(cached, keep, 64, tables, free, c, 12, capacity=cap)
        assert G.device_errors() == BAD_INDEX and got["left"] == c
        np.testing.assert_array_equal(got["free"], free)
        np.testing.assert_array_equal(got["lens"], cached)
    tables[0, 1] = 50  # a block that is none is handed on with an error
    got = release_call([100, 30], [0, 0], 64, tables, free, count, 12)
    assert G.device_errors() == BAD_INDEX and got["free"][count:].tolist() == [tables[0, 0], 50, tables[1, 0]]


# ------------------------------------------------------------------ logits


def logits_case(seed, rows, vocab, history, biases, masks, spread=2.0):
    rng = np.random.default_rng(seed)
    c = dict(x=G.rounded(rng.standard_normal((rows, vocab)) * spread), history=None, biases=None, allowed=None)
    if history:
        lens = rng.integers(0, history + 1, rows)
        c["history"] = [np.where(rng.random(n) < 0.5, rng.integers(0, vocab, n), c["x"][i].argsort()[-1 - rng.integers(0, min(vocab, 9), n)])
                        for i, n in enumerate(lens)]
        c["prompt"] = [int(rng.integers(0, n + 1)) for n in lens]
        c["rep"], c["freq"], c["pres"] = (rng.random((3, rows)) * [[1], [0.6], [0.6]] + [[0.6], [0], [0]]).astype(np.float32)
    if biases:
        c["biases"] = [[(int(t), np.float32(v)) for t, v in zip(rng.integers(0, vocab, n), rng.standard_normal(n) * 4)]
                       for n in rng.integers(0, biases + 1, rows)]
    if masks:
        c["allowed"] = [rng.random(vocab) < 0.5 if i % 3 else None for i in range(rows)]
    return c


def logits_call(c, pad=0, shift=0, in_place=False, want_next=True, want_out=True, use=("rep", "freq", "pres"), prompts=True):
    x = c["x"]
    rows, vocab = x.shape
    ld = vocab + pad
    buf = torch.full((rows * ld + shift + 8,), float("nan"), dtype=torch.bfloat16, device=G.DEV)
    view = buf[shift:shift + rows * ld].view(rows, ld)
    view[:, :vocab] = G.bf16(x)
    a = dict(history=None, prompt=None, lens=None, rep=None, freq=None, pres=None, off=None, ids=None, vals=None, mask=None, mrow=None)
    hld, words, num = 0, (vocab + 31) // 32, 0
    if c["history"] is not None:
        hld = max(map(len, c["history"])) + 2
        h = np.full((rows, hld), -99, np.int32)
        for i, t in enumerate(c["history"]):
            h[i, :len(t)] = t
        a.update(history=G.i32(h), lens=G.i32([len(t) for t in c["history"]]))
        if prompts:
            a["prompt"] = G.i32(c["prompt"])
        a.update({k: G.f32(c[k]) for k in use})
    if c["biases"] is not None:
        flat = [e for r in c["biases"] for e in r] or [(0, 0.0)]
        a.update(off=G.i32(np.concatenate([[0], np.cumsum([len(r) for r in c["biases"]])])), ids=G.i32([t for t, _ in flat]),
                 vals=G.f32([v for _, v in flat]))
    if c["allowed"] is not None:
        which = [i for i, m in enumerate(c["allowed"]) if m is not None]
        num = max(1, len(which))
        bits = np.ones((num, words * 32), bool)
        for k, i in enumerate(which):
            bits[k, :vocab] = c["allowed"][i]
        m = np.packbits(bits, axis=1, bitorder="little").view(np.int32)
        a.update(mask=G.i32(m), mrow=G.i32([which.index(i) if i in which else -1 for i in range(rows)]))
    out = view if in_place else torch.full((rows, ld), -5.0, dtype=torch.bfloat16, device=G.DEV) if want_out else None
    nxt = torch.full((rows + 1,), -9, dtype=torch.int64, device=G.DEV) if want_next else None
    p = {k: None if v is None else v.data_ptr() for k, v in a.items()}
    G.check(G.L().b200_logits_process(view.data_ptr(), ld, rows, vocab, p["history"], hld, p["prompt"], p["lens"], p["rep"],
                                      p["freq"], p["pres"], p["off"], p["ids"], p["vals"], p["mask"], words, num, p["mrow"],
                                      G.ptr(out), ld, G.ptr(nxt), G.stream()), "logits_process")
    if out is not None and pad:
        assert torch.isnan(out[:, vocab:]).all() if in_place else (out[:, vocab:] == -5).all()
    return None if out is None else out[:, :vocab].double().cpu().numpy(), None if nxt is None else nxt.cpu().numpy()


def logits_want(c, use=("rep", "freq", "pres"), prompts=True):
    want = []
    for i, x in enumerate(c["x"]):
        h, n = (c["history"][i].tolist(), c["prompt"][i] if prompts else 0) if c["history"] is not None else (None, 0)
        args = [c[k][i] if h is not None and k in use else None for k in ("rep", "freq", "pres")]
        want.append(serving.logits(x, None if h is None else h[:n], None if h is None else h[n:], *args,
                                   None if c["biases"] is None else c["biases"][i],
                                   None if c["allowed"] is None else c["allowed"][i]))
    return np.stack([w for w, _ in want]), np.array([n for _, n in want])


def check_logits(c, use=("rep", "freq", "pres"), prompts=True, **kw):
    c = dict(c, x=G.rounded(c["x"]))  # the values that the kernel sees
    out, nxt = logits_call(c, use=use, prompts=prompts, **kw)
    want, token = logits_want(c, use, prompts)
    if nxt is not None:
        assert nxt[-1] == -9
        np.testing.assert_array_equal(nxt[:-1], token)
    if out is not None:
        same = (want == c["x"]) | (np.isnan(want) & np.isnan(c["x"]))
        np.testing.assert_array_equal(out[same], want[same])  # untouched, or back at a bf16 value
        np.testing.assert_allclose(out, want, rtol=2.0 ** -8, atol=1e-40)
    assert G.device_errors() == 0


VOCABS = [1, 2, 31, 33, 1000, 1024, 1025, 4096, 32000, 50257, 151936]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("history,biases,masks", [(0, 0, 0), (300, 0, 0), (0, 40, 0), (0, 0, 1), (300, 40, 1)])
def test_logits(vocab, history, biases, masks):
    check_logits(logits_case(vocab, 5, vocab, history, biases, masks))


@pytest.mark.parametrize("pad,shift,in_place", [(8, 0, False), (3, 0, False), (0, 1, False), (5, 3, True), (0, 0, True), (64, 8, True)])
def test_logits_strides_and_in_place(pad, shift, in_place):
    check_logits(logits_case(1, 4, 5003, 100, 20, 1), pad=pad, shift=shift, in_place=in_place)


@pytest.mark.parametrize("use", [(), ("rep",), ("freq",), ("pres",), ("freq", "pres")])
@pytest.mark.parametrize("prompts", [True, False])
def test_logits_parts(use, prompts):
    check_logits(logits_case(2, 6, 3000, 200, 0, 0), use=use, prompts=prompts)
    c = logits_case(2, 6, 3000, 200, 30, 1)
    check_logits(c, use=use, prompts=prompts, want_out=False)
    check_logits(c, use=use, prompts=prompts, want_next=False)


def test_logits_long_history_and_many_rows():
    check_logits(logits_case(3, 2, 200, 40000, 0, 0))  # tokens that occur hundreds of times
    check_logits(logits_case(4, 300, 777, 20, 3, 1))
    # more tokens of one CTA touched than it computes at a time (a row a CTA, thousands of different tokens)
    c = logits_case(4, 150, 13000, 5, 2, 1)
    rng = np.random.default_rng(4)
    c["history"][7], c["history"][8] = rng.permutation(13000), rng.integers(0, 13000, 9000)
    c["prompt"][7], c["prompt"][8] = 6000, 0
    c["biases"][8] = [(int(t), np.float32(t % 7 - 3)) for t in rng.integers(0, 13000, 700)]
    check_logits(c)


def test_logits_tokens_listed_twice():
    c = logits_case(5, 3, 2000, 50, 0, 0)
    c["biases"] = [[(7, np.float32(0.1))] * 50 + [(9, np.float32(1e8)), (9, np.float32(1)), (9, np.float32(-1e8))],
                   [(1999, np.float32(3)), (0, np.float32(1)), (1999, np.float32(-2.5))], []]
    check_logits(c)


def test_logits_ties_go_to_the_lowest_token():
    c = logits_case(6, 4, 9000, 0, 0, 0)
    c["x"][:] = 1.0
    c["x"][1, [8999, 4500, 600]] = 2.0
    c["x"][2, :] = -np.inf
    c["x"][2, 70] = -3.0
    c["x"][3, 5:] = 3.0
    check_logits(c)
    # a penalty that brings a token level with others: the lowest of them
    c = logits_case(6, 2, 9000, 0, 0, 0)
    c["x"][:] = 0.0
    c["x"][0, [30, 20, 10]] = [2.0, 4.0, 2.0]
    c["x"][1, [30, 20, 10]] = [2.0, 4.0, 2.0]
    c.update(history=[np.array([20]), np.array([20])], prompt=[1, 1], rep=np.array([2, 2.0000002], np.float32),
             freq=np.zeros(2, np.float32), pres=np.zeros(2, np.float32))
    check_logits(c)


def test_logits_differences_below_32_bits_decide():
    # 3 / 1.1f and 3 / 1.1f + 1e-9 round to one fp32 value
    c = logits_case(7, 1, 5000, 0, 0, 0)
    c["x"][:] = 0.0
    c["x"][0, [100, 200]] = 3.0
    c.update(history=[np.array([100, 200])], prompt=[2], rep=np.array([1.1], np.float32), freq=np.zeros(1, np.float32),
             pres=np.zeros(1, np.float32), biases=[[(200, np.float32(1e-9))]])
    _, nxt = logits_call(c)
    assert nxt[0] == 200
    check_logits(c)


def test_logits_special_values():
    c = logits_case(8, 6, 4000, 60, 10, 0)
    c["x"][0, :] = np.nan
    c["x"][1, :] = -np.inf
    c["x"][2, ::2] = np.nan
    c["x"][3, 5], c["x"][3, 6] = np.inf, np.inf
    c["x"][4, 1:] = -np.finfo(np.float32).max / 2
    c["x"][5] = -0.0
    for i in range(6):  # a history token of each row is special too
        c["history"][i] = np.concatenate([c["history"][i], [5, 6, 5]]).astype(np.int64)
    c["biases"] = [[] for _ in range(6)]
    check_logits(c)
    nothing = logits_case(9, 3, 4000, 60, 10, 0)
    nothing["allowed"] = [np.zeros(4000, bool)] * 3
    out, nxt = logits_call(nothing)
    assert (out == -np.inf).all() and (nxt[:3] == -1).all()


def test_logits_bad_ids_and_lengths():
    c = logits_case(10, 2, 3000, 50, 10, 0)
    want, token = logits_want(c)
    x = G.bf16(c["x"])
    hist = np.concatenate([np.full((2, 1), v) for v in (3000, -1, 2**31 - 1)] + [np.full((2, 49), 7)], 1).astype(np.int32)
    out, nxt = torch.empty_like(x), torch.empty(2, dtype=torch.int64, device=G.DEV)
    rep, off = G.f32([1.5, 1.5]), G.i32([0, 2, 2])
    ids, vals = G.i32([3000, -5]), G.f32([100, 100])
    L = G.L()
    h = G.i32(hist)
    want = c["x"].astype(np.float64)
    want[:, 7] = np.where(want[:, 7] > 0, want[:, 7] / 1.5, want[:, 7] * 1.5)
    for lens, prompt in (([52, 52], [1, 60]), ([1000, 52], [0, -3])):
        n, p = G.i32(lens), G.i32(prompt)
        G.check(L.b200_logits_process(x.data_ptr(), 3000, 2, 3000, h.data_ptr(), 52, p.data_ptr(), n.data_ptr(), rep.data_ptr(), None,
                                      None, off.data_ptr(), ids.data_ptr(), vals.data_ptr(), None, 0, 0, None, out.data_ptr(), 3000,
                                      nxt.data_ptr(), G.stream()))
        np.testing.assert_allclose(out.double().cpu().numpy(), want, rtol=2.0 ** -8)
        assert G.device_errors() == BAD_INDEX
    mask, rows = G.i32(np.zeros((2, 94))), G.i32([2, -2])
    G.check(L.b200_logits_process(x.data_ptr(), 3000, 2, 3000, None, 0, None, None, None, None, None, None, None, None,
                                  mask.data_ptr(), 94, 2, rows.data_ptr(), out.data_ptr(), 3000, nxt.data_ptr(), G.stream()))
    assert torch.equal(out, x) and G.device_errors() == BAD_INDEX


def test_logits_equal_argmax_without_changes():
    c = logits_case(11, 7, 151936, 0, 0, 0)
    out, nxt = logits_call(c)
    want = torch.empty(7, dtype=torch.int64, device=G.DEV)
    G.check(G.L().b200_argmax(G.bf16(c["x"]).data_ptr(), 7, 151936, 151936, want.data_ptr(), G.stream()))
    assert nxt[:7].tolist() == want.tolist() and (out == c["x"]).all()


def test_logits_of_the_largest_vocabulary():
    check_logits(logits_case(12, 2, 1 << 23, 300, 40, 1))


def test_logits_offsets_past_32_bits():
    rows, ld, vocab = 1100, 1 << 21, 1000  # 2.3e9 elements
    rng = np.random.default_rng(13)
    x = torch.full((rows, ld), 7.0, dtype=torch.bfloat16, device=G.DEV)
    values = G.rounded(rng.standard_normal((rows, vocab)))
    x[:, :vocab] = G.bf16(values)
    history = G.i32(values.argmax(1)[:, None])
    one, rep, nxt = G.i32([1] * rows), G.f32([1.5] * rows), torch.zeros(rows, dtype=torch.int64, device=G.DEV)
    G.check(G.L().b200_logits_process(x.data_ptr(), ld, rows, vocab, history.data_ptr(), 1, None, one.data_ptr(), rep.data_ptr(), None,
                                      None, None, None, None, None, 0, 0, None, x.data_ptr(), ld, nxt.data_ptr(), G.stream()))
    want = [serving.logits(r, [], [int(r.argmax())], np.float32(1.5)) for r in values]
    assert nxt.tolist() == [t for _, t in want]
    np.testing.assert_allclose(G.host(x[:, :vocab]), np.stack([w for w, _ in want]), rtol=2.0 ** -8)
    x[:, :vocab] = 7
    assert bool((x == 7).all()) and G.device_errors() == 0
    del x
    torch.cuda.empty_cache()


# --------------------------------------------------------- a step of it all


@pytest.mark.parametrize("shared", [False, True], ids=["window", "shared"])
def test_steps_of_a_captured_serving_loop(shared):
    """extend -> cache write -> attention -> logits -> release, captured once and replayed while requests grow, end, lose
    tokens and run out of blocks; each step against the restatements."""
    L, rng = G.L(), np.random.default_rng(12)
    B, nq, nkv, d, bs, width, vocab, cap = 6, 8, 2, 128, 64, 5, 1000, 6
    window, sinks, plen = 100, 4, 150 if shared else 0
    head = -(-plen // bs)
    blocks = 8 + head  # fewer than six sequences come to want
    kc, vc = (G.bf16(np.full((blocks, nkv, bs, d), np.nan)) for _ in range(2))
    hk, hv = (np.full((blocks, nkv, bs, d), np.nan, np.float32) for _ in range(2))
    prefix = np.arange(blocks - head, blocks)
    for c, dev in ((hk, kc), (hv, vc)):
        for j in range(plen):
            c[prefix[j // bs], :, j % bs] = G.rounded(rng.standard_normal((nkv, d)))
        dev.copy_(G.bf16(c))
    lens, new, keep = G.i32([0] * B), G.i32([0] * B), G.i32([0] * B)
    tables, free, count = G.i32(np.full((B, width), -1)), G.i32(np.arange(blocks)), G.i32([blocks - head])
    cu, pos = G.i32([0] * (B + 1)), G.i64([0] * cap)
    slots, missing = G.i64([-1] * cap), G.i32([0])
    qkv = torch.zeros(cap, (nq + 2 * nkv) * d, dtype=torch.bfloat16, device=G.DEV)
    ones, zeros = torch.ones(cap, d, device=G.DEV), torch.zeros(cap, d, device=G.DEV)  # a rotation by nothing
    out = torch.zeros(B, nq * d, dtype=torch.bfloat16, device=G.DEV)
    x, y = (torch.zeros(B, vocab, dtype=torch.bfloat16, device=G.DEV) for _ in range(2))
    hist, hlen, rep, nxt = G.i32(np.zeros((B, 400))), G.i32([0] * B), G.f32([1.3] * B), G.i64([0] * B)
    q = torch.zeros(B, nq * d, dtype=torch.bfloat16, device=G.DEV)
    pre, pl = G.i32(prefix if shared else [0]), G.i32([plen])
    ws = torch.empty(max(4, L.b200_paged_decode_shared_workspace_bytes(B, nq, nkv, d, max(plen, 1))), dtype=torch.uint8, device=G.DEV)

    def step(st):
        G.check(L.b200_block_tables_extend(lens.data_ptr(), new.data_ptr(), B, bs, tables.data_ptr(), width, free.data_ptr(),
                                           count.data_ptr(), blocks, lens.data_ptr(), cu.data_ptr(), pos.data_ptr(),
                                           slots.data_ptr(), cap, count.data_ptr(), missing.data_ptr(), st))
        G.check(L.b200_qk_norm_rope(qkv.data_ptr(), cap, nq, nkv, d, qkv.shape[1], None, None, 1e-6, ones.data_ptr(),
                                    zeros.data_ptr(), slots.data_ptr(), kc.data_ptr(), vc.data_ptr(), blocks, bs, st))
        if shared:
            G.check(L.b200_paged_decode_shared(q.data_ptr(), nq * d, kc.data_ptr(), vc.data_ptr(), pre.data_ptr(), pl.data_ptr(), plen,
                                               tables.data_ptr(), width, lens.data_ptr(), width * bs, B, nq, nkv, d, bs, blocks,
                                               d ** -0.5, out.data_ptr(), nq * d, ws.data_ptr(), ws.numel(), st))
        else:
            G.check(L.b200_paged_decode_window(q.data_ptr(), nq * d, kc.data_ptr(), vc.data_ptr(), tables.data_ptr(), width,
                                               lens.data_ptr(), B, nq, nkv, d, bs, blocks, d ** -0.5, window, sinks,
                                               out.data_ptr(), nq * d, width * bs, st))
        G.check(L.b200_logits_process(x.data_ptr(), vocab, B, vocab, hist.data_ptr(), 400, None, hlen.data_ptr(), rep.data_ptr(), None,
                                      None, None, None, None, None, 0, 0, None, y.data_ptr(), vocab, nxt.data_ptr(), st))
        G.check(L.b200_block_tables_release(lens.data_ptr(), keep.data_ptr(), B, bs, tables.data_ptr(), width, free.data_ptr(),
                                            blocks, count.data_ptr(), blocks, lens.data_ptr(), count.data_ptr(), st))

    step(G.stream())  # no tokens yet
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(G.stream())
    h_lens, h_tables, h_free = np.zeros(B, np.int64), tables.cpu().numpy(), free.cpu().numpy()
    h_count, history, seen_short = blocks - head, [[] for _ in range(B)], False
    for i in range(260):
        more = (rng.random(B) < 0.93).astype(np.int64)
        rows = G.rounded(rng.standard_normal((cap, (nq + 2 * nkv) * d)))
        qn = G.rounded(rng.standard_normal((B, nq * d)) * 2)
        xn = G.rounded(rng.standard_normal((B, vocab)) * 2)
        want = serving.extend(h_lens, more, bs, h_tables, h_free, h_count, cap)
        cut = np.where(rng.random(B) < 0.015, 0, want[1] - (rng.random(B) < 0.05)).clip(0)
        cut = np.where(want[1] >= width * bs - 1, 0, cut)
        if want[6]:  # out of blocks: the longest goes
            cut[want[1].argmax()] = 0
            seen_short = True
        h = np.zeros((B, 400), np.int32)
        for b in range(B):
            h[b, :len(history[b])] = history[b]
        for dev, val in ((new, more), (keep, cut), (hlen, [len(t) for t in history]), (hist, h)):
            dev.copy_(torch.from_numpy(np.ascontiguousarray(np.asarray(val, np.int32))))
        for dev, val in ((qkv, rows), (q, qn), (x, xn)):
            dev.copy_(torch.from_numpy(val))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        h_tables, ctx = want[0], want[1]
        kv = rows.reshape(cap, nq + 2 * nkv, d)
        for t, s in enumerate(want[4]):
            if s >= 0:
                hk[s // bs, :, s % bs], hv[s // bs, :, s % bs] = kv[t, nq:nq + nkv], kv[t, nq + nkv:]
        if i % 13 == 0 or want[6]:
            qh = qn.reshape(B, nq, d)
            ref = serving.shared_decode(qh, hk, hv, prefix, plen, h_tables, ctx) if shared else \
                serving.window_decode(qh, hk, hv, h_tables, ctx, window, sinks)
            close(G.host(out).reshape(B, nq, d), *ref)
        tokens = [serving.logits(xn[b], [], history[b], 1.3)[1] for b in range(B)]
        assert nxt.tolist() == tokens and missing.item() == want[6]
        np.testing.assert_array_equal(cu.cpu().numpy(), want[2])
        h_free, h_lens, h_count = serving.release(ctx, cut, bs, h_tables, h_free, want[5])
        np.testing.assert_array_equal(lens.cpu().numpy(), h_lens)
        np.testing.assert_array_equal(tables.cpu().numpy(), h_tables)
        assert count.item() == h_count and sorted(h_free[:h_count].tolist() + [
            t for b in range(B) for t in h_tables[b, :-(-int(h_lens[b]) // bs)]]) == list(range(blocks - head))
        for b in range(B):
            history[b] = (history[b] + [tokens[b]])[-399:] if h_lens[b] else []
    assert G.device_errors() == 0 and seen_short


FIRST_CALL = """
import sys
sys.path.insert(0, {root!r}); sys.path.insert(0, {tests!r})
import numpy as np, torch
from atb_llm_study_b200 import capi
torch.zeros(1, device="cuda")
import gpu_util as G, test_gpu_window as T, test_gpu_serving as S
from oracle import serving
kind = sys.argv[1]
g = torch.cuda.CUDAGraph()
if kind in ("token", "shared"):
    c = T.Cache(1, [70, 130], 2, 64, 64, spare=4)
    c.fill_fast(c.order[:2], 100)
    q, qd = T.queries(1, 2, 4, 64)
    dev, pre, plen = c.device(), G.i32(c.order[:2]), G.i32([100])
    out = torch.zeros(2, 256, dtype=torch.bfloat16, device=G.DEV)
    ws = torch.zeros(1 << 20, device=G.DEV)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        T.token_call(qd, dev, c, 4, 50, 2, out=out) if kind == "token" else T.shared_call(qd, dev, c, 4, pre, plen, 100, ws=ws, out=out)
    g.replay()
    want = serving.window_decode(q, c.k, c.v, c.tables, c.lens, 50, 2) if kind == "token" else \\
        serving.shared_decode(q, c.k, c.v, c.order[:2], 100, c.tables, c.lens)
    T.close(G.host(out).reshape(2, 4, 64), *want)
elif kind == "prompt":
    q, k, v = T.prompt_inputs(1, 200, 4, 2, 64, 64)
    dq, dk, dv = (G.bf16(x.reshape(200, -1)) for x in (q, k, v))
    out, cu = torch.zeros(200, 256, dtype=torch.bfloat16, device=G.DEV), G.i32([0, 200])
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        G.check(G.L().b200_flash_prefill_window(dq.data_ptr(), 256, 64, dk.data_ptr(), 128, 64, dv.data_ptr(), 128, 64, out.data_ptr(),
                                                256, 64, cu.data_ptr(), 1, 200, 200, 4, 2, 64, 64, 0.125, 60, 3, G.stream()))
    g.replay()
    T.close(G.host(out).reshape(200, 4, 64), *serving.window_prompt(q, k, v, [200], 60, 3, 0.125))
elif kind == "logits":
    x = G.bf16(np.arange(2000)[None] % 700)
    nxt = torch.zeros(1, dtype=torch.int64, device=G.DEV)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        G.check(G.L().b200_logits_process(x.data_ptr(), 2000, 1, 2000, None, 0, None, None, None, None, None, None, None, None, None, 0,
                                          0, None, None, 0, nxt.data_ptr(), G.stream()))
    g.replay()
    assert nxt.item() == int(G.host(x)[0].argmax())
else:
    lens, new, ctx = G.i32([3]), G.i32([2]), G.i32([0])
    tables, free, count, left = G.i32([[4, -1]]), G.i32([0, 1, 2, 3, 5, 6]), G.i32([6]), G.i32([0])
    slots = G.i64([0, 0])
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        G.check(G.L().b200_block_tables_extend(lens.data_ptr(), new.data_ptr(), 1, 4, tables.data_ptr(), 2, free.data_ptr(),
                                               count.data_ptr(), 7, ctx.data_ptr(), None, None, slots.data_ptr(), 2, left.data_ptr(),
                                               None, G.stream()))
        G.check(G.L().b200_block_tables_release(ctx.data_ptr(), lens.data_ptr(), 1, 4, tables.data_ptr(), 2, free.data_ptr(), 6,
                                                left.data_ptr(), 7, ctx.data_ptr(), left.data_ptr(), G.stream()))
    g.replay()
    assert slots.tolist() == [19, 24] and left.item() == 6 and ctx.item() == 3 and free.tolist()[5] == 6
torch.cuda.synchronize()
print("fine")
"""


@pytest.mark.parametrize("kind", ["prompt", "token", "shared", "logits", "tables"])
def test_first_call_of_a_process_may_be_captured(kind):
    import os
    import subprocess
    import sys

    tests = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL.format(root=os.path.dirname(tests), tests=tests), kind], capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("fine"), r.stdout[-500:] + r.stderr[-2000:]
