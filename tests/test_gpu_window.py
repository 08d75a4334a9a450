"""GPU parity of window attention (prompts and single tokens) and of shared-prefix
decode attention with the float64 restatements in oracle.serving.

Tolerance, per element, with A the softmax-weighted mean of |v| and half a step
of bf16 2^-8: the output's rounding 2^-8 |o|, the weights' rounding to bf16
2^-8 A, and the scores' error in both the weight and the sum: a score is a sum
of d <= 192 products in fp32, off by at most d 2^-24 sum |q_i k_i| scale, and
sum |q_i k_i| scale is below 60 for the inputs here (d = 192, |q| = 2), so p is
off by 192 x 60 x 2^-24 = 7e-4 relative at the very most; the exponential
(2^-22) and the sums are far below that.  Hence 2^-8 |o| + (2^-8 + 1.4e-3) A,
and 1e-6 for outputs near zero.
"""

import numpy as np
import pytest
import torch

from oracle import serving

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import gpu_util as G

BAD_INDEX = 2


def close(got, want, weight):
    got = np.asarray(got, np.float64)
    err = np.abs(got - want)
    bound = 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 1.4e-3) * weight + 1e-6
    assert np.isfinite(got).all()
    worst = np.unravel_index((err - bound).argmax(), err.shape)
    assert (err <= bound).all(), (worst, got[worst], want[worst], bound[worst])


# ---------------------------------------------------------------- prompts


def prompt(q, k, v, lens, window, sinks, pad_rows=0, longest=None, fused=True):
    """q [T, nq, d], k [T, nkv, d], v [T, nkv, dv] (numpy) -> out [T + pad_rows, nq, dv] (numpy); pad rows are NaN on the way
    in and -5 in the output's buffer."""
    T, nq, d = q.shape
    nkv, dv = k.shape[1], v.shape[2]
    widths = [nq * d, nkv * d, nkv * dv]
    rows = T + pad_rows
    gap = 0 if fused else 8  # elements between heads
    parts = []
    for x, n, w in ((q, nq, d), (k, nkv, d), (v, nkv, dv)):
        y = np.full((rows, n, w + gap), np.nan, np.float32)
        y[:T, :, :w] = x
        parts.append(y.reshape(rows, -1))
    dev = G.bf16(np.concatenate(parts, 1))
    row, at = dev.shape[1], dev.data_ptr()
    qo, ko, vo = at, at + 2 * parts[0].shape[1], at + 2 * (parts[0].shape[1] + parts[1].shape[1])
    out = torch.full((rows, nq * dv + 8), -5.0, dtype=torch.bfloat16, device=G.DEV)
    cu = G.i32(np.concatenate([[0], np.cumsum(lens)]))
    G.check(G.L().b200_flash_prefill_window(qo, row, d + gap, ko, row, d + gap, vo, row, dv + gap, out.data_ptr(), nq * dv + 8, dv,
                                            cu.data_ptr(), len(lens), max(lens) if longest is None else longest, rows, nq, nkv,
                                            d, dv, d ** -0.5, window, sinks, G.stream()), "flash_prefill_window")
    got = G.host(out)
    assert (got[:, nq * dv:] == -5).all() and (got[T:] == -5).all()
    del widths
    return got[:, :nq * dv].reshape(rows, nq, dv)[:T]


def prompt_inputs(seed, T, nq, nkv, d, dv, scale=1.0):
    rng = np.random.default_rng(seed)
    q, k, v = rng.standard_normal((T, nq, d)) * 2 * scale, rng.standard_normal((T, nkv, d)), rng.standard_normal((T, nkv, dv))
    return [G.rounded(x) for x in (q, k, v)]


def check_prompt(lens, nq, nkv, d, dv, window, sinks, **kw):
    q, k, v = prompt_inputs(sum(lens) + window, sum(lens), nq, nkv, d, dv)
    want, weight = serving.window_prompt(q, k, v, lens, window, sinks, d ** -0.5)
    close(prompt(q, k, v, lens, window, sinks, **kw), want, weight)
    assert G.device_errors() == 0


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 0), (63, 4), (64, 0), (127, 0), (128, 0), (128, 4), (129, 1),
                                          (130, 128), (200, 129), (300, 300), (256, 0), (384, 64), (5000, 0), (1, 5000)])
def test_prompt_windows(window, sinks):
    check_prompt([515], 4, 2, 128, 128, window, sinks)


@pytest.mark.parametrize("lens", [[1], [0, 1, 0], [2, 127, 128, 129, 1], [0, 0, 257, 0, 640, 33], [1] * 20, [700, 3]],
                         ids=lambda x: "-".join(map(str, x)))
@pytest.mark.parametrize("window,sinks", [(1, 0), (100, 3), (128, 0)])
def test_prompt_lengths(lens, window, sinks):
    check_prompt(lens, 2, 1, 64, 64, window, sinks)


@pytest.mark.parametrize("nq,nkv,d,dv", [(4, 4, 16, 16), (6, 2, 32, 32), (12, 4, 64, 64), (7, 1, 128, 128), (8, 8, 128, 128),
                                         (4, 4, 192, 128), (1, 1, 64, 64)])
@pytest.mark.parametrize("fused", [True, False], ids=["fused", "spaced"])
def test_prompt_heads(nq, nkv, d, dv, fused):
    check_prompt([130, 300, 5], nq, nkv, d, dv, 150, 2, fused=fused, pad_rows=70)


@pytest.mark.parametrize("nq", [4, 2])  # two heads an item, or two row tiles
def test_prompt_many_lengths(nq):
    rng = np.random.default_rng(nq)
    lens = [int(n) for n in rng.choice([0, 0, 1, 3, 100, 127, 128, 129, 255, 256, 257, 400], 60)]
    check_prompt(lens, nq, 2, 64, 64, 90, 2)


def test_prompt_longer_limit_and_rows_behind():
    check_prompt([200, 100], 4, 2, 128, 128, 64, 4, pad_rows=300, longest=1000)
    check_prompt([200, 100, 0], 4, 2, 128, 128, 64, 4, pad_rows=5000, longest=100000)
    q, k, v = prompt_inputs(1, 300, 2, 2, 64, 64)  # a sequence longer than max_seqlen: its first tiles, the rest as it was
    got = prompt(q, k, v, [300], 64, 0, longest=128)
    want, weight = serving.window_prompt(q, k, v, [300], 64, 0, 0.125)
    close(got[:128], want[:128], weight[:128])
    assert (got[128:] == -5).all()


def test_prompt_sequence_outside_the_rows():
    q, k, v = prompt_inputs(2, 100, 2, 2, 64, 64)
    dev = [G.bf16(x.reshape(100, -1)) for x in (q, k, v)]
    out = torch.full((100, 128), -5.0, dtype=torch.bfloat16, device=G.DEV)
    for cu, left in (([0, 60, 120], 60), ([-4, 60, 100], 0)):
        out.fill_(-5)
        c = G.i32(cu)
        G.check(G.L().b200_flash_prefill_window(dev[0].data_ptr(), 128, 64, dev[1].data_ptr(), 128, 64, dev[2].data_ptr(), 128,
                                                64, out.data_ptr(), 128, 64, c.data_ptr(), 2, 120, 100, 2, 2, 64, 64, 0.125,
                                                30, 0, G.stream()))
        got = G.host(out)
        assert G.device_errors() == BAD_INDEX
        assert (got[:60] != -5).all() == (left == 60) and (got[60:] == -5).all() == (left == 60)


@pytest.mark.parametrize("window,sinks,bad", [(40, 0, 0), (40, 4, 2), (40, 4, 5), (130, 0, 200), (130, 0, 299), (128, 130, 129),
                                              (128, 130, 131), (300, 0, 128)])
@pytest.mark.parametrize("value", [np.nan, np.inf, 3e38])
def test_prompt_hidden_values_stay_hidden(window, sinks, bad, value):
    lens = [300, 300]
    q, k, v = prompt_inputs(3, 600, 4, 2, 64, 64)
    want, weight = serving.window_prompt(q, k, v, lens, window, sinks, 0.125)
    k2, v2 = k.copy(), v.copy()
    v2[bad, 0, 7] = value
    sees = serving.window_mask(300, window, sinks)[:, bad]
    for kk, vv in ((k, v2), (np.where(np.arange(600)[:, None, None] == bad, np.float32(np.nan), k2), v2)):
        got = prompt(q, kk, vv, lens, window, sinks)
        close(got[300:], want[300:], weight[300:])
        close(got[:300][~sees], want[:300][~sees], weight[:300][~sees])
        if not np.isfinite(value) or kk is not k:
            assert not np.isfinite(got[:300][sees][:, :2, 7]).any()
        if kk is k:  # the other kv head's query heads
            close(got[:300, 2:], want[:300, 2:], weight[:300, 2:])


# heads in pairs and (odd groups) row tiles in pairs; four, two and one stages of V
@pytest.mark.parametrize("nq,nkv,d,dv", [(3, 1, 64, 64), (4, 2, 128, 128), (3, 1, 128, 128), (4, 2, 192, 128), (2, 2, 192, 128),
                                         (2, 1, 32, 32)])
@pytest.mark.parametrize("window,sinks,bad", [(40, 4, 2), (130, 0, 200), (128, 130, 131), (200, 3, 255), (300, 0, 128)])
@pytest.mark.parametrize("value", [np.nan, -np.inf])
def test_prompt_hidden_values_of_all_widths(nq, nkv, d, dv, window, sinks, bad, value):
    lens = [400, 90]
    q, k, v = prompt_inputs(7, 490, nq, nkv, d, dv)
    want, weight = serving.window_prompt(q, k, v, lens, window, sinks, d ** -0.5)
    v = v.copy()
    v[bad, 0, dv - 1] = value
    sees = serving.window_mask(400, window, sinks)[:, bad]
    got = prompt(q, k, v, lens, window, sinks)
    group = nq // nkv
    assert not np.isfinite(got[:400][sees][:, :group, dv - 1]).any()
    close(got[:400][~sees], want[:400][~sees], weight[:400][~sees])
    if nkv > 1:
        close(got[:, group:], want[:, group:], weight[:, group:])
    close(got[400:], want[400:], weight[400:])


@pytest.mark.parametrize("nq,nkv,d,dv,seqs", [(4, 4, 192, 128, 500), (4, 2, 192, 128, 700), (8, 4, 128, 128, 900), (16, 8, 64, 64, 900)])
def test_prompt_records_of_many_short_items(nq, nkv, d, dv, seqs):
    """A CTA walks a dozen items of one key tile and more, several times what the ring of zeroed values' records holds;
    some sequences and heads have a value that is no number, the items around them do not."""
    rng = np.random.default_rng(d + nq)
    lens = rng.integers(1, 9, seqs).tolist()
    total = sum(lens)
    q, k, v = prompt_inputs(8, total, nq, nkv, d, dv)
    want, weight = serving.window_prompt(q, k, v, lens, 6, 1, d ** -0.5)
    v = v.copy()
    poisoned = np.zeros((total, nq), bool)
    at = 0
    for n in lens:
        for h in np.nonzero(rng.random(nkv) < 0.3)[0]:
            bad = int(rng.integers(0, n))
            v[at + bad, h, int(rng.integers(0, dv))] = rng.choice([np.nan, np.inf])
            sees = serving.window_mask(n, 6, 1)[:, bad]
            poisoned[at:at + n, h * nq // nkv:(h + 1) * nq // nkv] |= sees[:, None]
        at += n
    for _ in range(3):
        got = prompt(q, k, v, lens, 6, 1)
        finite = np.isfinite(got).all(2)
        np.testing.assert_array_equal(finite, ~poisoned)
        close(got[finite], want[finite], weight[finite])
    assert G.device_errors() == 0


def test_a_query_that_is_nan_is_alone():
    q, k, v = prompt_inputs(6, 200, 4, 2, 64, 64)
    want, weight = serving.window_prompt(q, k, v, [200], 70, 2, 0.125)
    q[130, 1, 5] = np.nan
    got = prompt(q, k, v, [200], 70, 2)
    assert np.isnan(got[130, 1]).all()
    got[130, 1] = want[130, 1]
    close(got, want, weight)
    c = Cache(9, [100, 100], 2, 64, 64, spare=4)
    c.fill_fast(c.order[:2], 100)
    q, _ = queries(9, 2, 4, 64)
    qn = q.reshape(2, 256).copy()
    qn[1, 64] = np.nan
    qd = G.bf16(np.concatenate([qn, np.zeros((2, 8), np.float32)], 1))
    for got, (want, weight) in (
            (token_call(qd, c.device(), c, 4, 80, 0), serving.window_decode(q, c.k, c.v, c.tables, c.lens, 80, 0)),
            (shared_call(qd, c.device(), c, 4, G.i32(c.order[:2]), G.i32([100]), 100),
             serving.shared_decode(q, c.k, c.v, c.order[:2], 100, c.tables, c.lens))):
        got = G.host(got)[:2, :256].reshape(2, 4, 64)
        assert np.isnan(got[1, 1]).all()
        got[1, 1] = want[1, 1]
        close(got, want, weight)


@pytest.mark.parametrize("nq,nkv,d,dv", [(4, 2, 64, 64), (3, 1, 128, 128), (2, 2, 192, 128), (2, 2, 16, 16)])
def test_prompt_infinite_scores(nq, nkv, d, dv):
    """Scores of -inf alone are 0 / 0, and one of +inf is inf / inf; one of -inf beside finite ones has no weight."""
    q, k, v = prompt_inputs(11, 300, nq, nkv, d, dv)
    k[:, :, 0] = G.rounded(np.abs(k[:, :, 0]) + 0.5)  # the values that the kernel sees
    q[:, :, 0] = G.rounded(np.abs(q[:, :, 0]) + 0.5)
    for bad, value in ((170, -np.inf), (170, np.inf), (0, -np.inf), (299, np.inf)):
        qq = q.copy()
        qq[bad, 0, 0] = value  # all scores of one query's head
        want, weight = serving.window_prompt(q, k, v, [300], 140, 2, d ** -0.5)
        got = prompt(qq, k, v, [300], 140, 2)
        assert np.isnan(got[bad, 0]).all()
        got[bad, 0] = want[bad, 0]
        close(got, want, weight)
    for bad in (1, 100, 200):
        kk = k.copy()
        kk[bad, :, 0] = -np.inf
        want, weight = serving.window_prompt(q, kk, v, [300], 140, 2, d ** -0.5)
        close(prompt(q, kk, v, [300], 140, 2), want, weight)
        kk[bad, :, 0] = np.inf
        sees = serving.window_mask(300, 140, 2)[:, bad]
        got = prompt(q, kk, v, [300], 140, 2)
        assert np.isnan(got[sees]).all()
        close(got[~sees], want[~sees], weight[~sees])


@pytest.mark.parametrize("lens", [[100, 0, 100], [2000, 0, 2000]], ids=["short", "long"])  # one CTA a pair, and a cluster
@pytest.mark.parametrize("d", [64, 128])
def test_token_infinite_scores(lens, d):
    c = Cache(12, lens, 2, d, 64, spare=2)
    c.k[..., 0] = G.rounded(np.abs(c.k[..., 0]) + 0.5)
    q, _ = queries(12, 3, 4, d)
    want, weight = serving.window_decode(q, c.k, c.v, c.tables, lens, 5000, 0)
    for value in (-np.inf, np.inf):
        qq = q.copy()
        qq[:2, 1, 0] = value  # one head of the first sequence, and of the empty one
        for longest in (1, max(lens)):
            got = G.host(token_call(G.bf16(qq.reshape(3, -1)), c.device(), c, 4, 5000, 0, longest))[:3, :4 * d].reshape(3, 4, d)
            assert np.isnan(got[0, 1]).all() and (got[1] == 0).all()
            got[0, 1] = want[0, 1]
            close(got, want, weight)


@pytest.mark.parametrize("plen", [0, 1, 300])
def test_shared_infinite_scores(plen):
    lens = [100, 0, 100]
    c = Cache(13, lens, 2, 64, 64, spare=6)
    prefix = c.order[:5]
    c.fill_fast(prefix, plen)
    c.k[..., 0] = G.rounded(np.abs(c.k[..., 0]) + 0.5)
    q, _ = queries(13, 3, 4, 64)
    want, weight = serving.shared_decode(q, c.k, c.v, prefix, plen, c.tables, lens)
    for value in (-np.inf, np.inf):
        qq = q.copy()
        qq[:2, 1, 0] = value
        got = G.host(shared_call(G.bf16(qq.reshape(3, -1)), c.device(), c, 4, G.i32(prefix), G.i32([plen]), 320))[:3, :256]
        got = got.reshape(3, 4, 64)
        assert np.isnan(got[0, 1]).all()
        assert np.isnan(got[1, 1]).all() if plen else (got[1] == 0).all()
        got[:2, 1] = want[:2, 1]
        close(got, want, weight)


def test_prompt_growing_and_flat_scores():
    lens = [400]
    q, k, v = prompt_inputs(4, 400, 2, 1, 128, 128, scale=0.0)
    want, weight = serving.window_prompt(q, k, v, lens, 150, 2, 128 ** -0.5)  # all scores equal: means
    close(prompt(q, k, v, lens, 150, 2), want, weight)
    q = G.rounded(np.ones((400, 2, 128)))
    k = G.rounded(np.arange(400)[:, None, None] * np.ones((1, 1, 128)) * 0.05)  # 0.57 a key: the maximum moves many times
    want, weight = serving.window_prompt(q, k, v, lens, 390, 0, 128 ** -0.5)
    close(prompt(q, k, v, lens, 390, 0), want, weight)


def test_prompt_matches_causal_kernel_without_a_window():
    lens = [500, 277]
    x = prompt_inputs(5, 777, 8, 2, 128, 128)
    q, k, v = (G.bf16(a.reshape(777, -1)) for a in x)
    cu = G.i32([0, 500, 777])
    outs = [torch.empty(777, 1024, dtype=torch.bfloat16, device=G.DEV) for _ in range(2)]
    args = (q.data_ptr(), 1024, 128, k.data_ptr(), 256, 128, v.data_ptr(), 256, 128)
    tail = (cu.data_ptr(), 2, 500, 777, 8, 2, 128, 128, 128 ** -0.5)
    G.check(G.L().b200_flash_prefill_packed(*args, outs[0].data_ptr(), 1024, 128, *tail, 1, G.stream()))
    G.check(G.L().b200_flash_prefill_window(*args, outs[1].data_ptr(), 1024, 128, *tail, 777, 0, G.stream()))
    want, weight = serving.window_prompt(*x, lens, 777, 0, 128 ** -0.5)
    for out in outs:
        close(G.host(out).reshape(777, 8, 128), want, weight)


# ------------------------------------------------------------ single tokens


class Cache:
    """A paged cache whose unused blocks and block rests are `rest`, with tables of shuffled blocks."""

    def __init__(self, seed, lens, nkv, d, bs, window=None, sinks=0, spare=3, width=None, rest=np.nan):
        rng = self.rng = np.random.default_rng(seed)
        self.nkv, self.d, self.bs, self.lens = nkv, d, bs, lens
        self.width = width or max(1, -(-max([*lens, 1]) // bs))
        need = [[c for c in range(-(-n // bs)) if window is None or (c + 1) * bs > n - window or c * bs < sinks] for n in lens]
        self.blocks = sum(map(len, need)) + spare
        order = rng.permutation(self.blocks)
        self.tables = np.full((len(lens), self.width), -1, np.int32)
        at = 0
        for i, cols in enumerate(need):
            self.tables[i, cols] = order[at:at + len(cols)]
            at += len(cols)
        shape = (self.blocks, nkv, bs, d)
        self.k, self.v = np.full(shape, rest, np.float32), np.full(shape, rest, np.float32)
        for i, n in enumerate(lens):
            self.fill(self.tables[i], [j for j in range(n) if window is None or j >= n - window or j < sinks])
        self.order = order[at:]

    def fill(self, table, positions):
        for j in positions:
            for c in (self.k, self.v):
                c[table[j // self.bs], :, j % self.bs] = G.rounded(self.rng.standard_normal((self.nkv, self.d)))

    def fill_fast(self, table, n):
        for c in (self.k, self.v):
            x = G.rounded(self.rng.standard_normal((n, self.nkv, self.d)))
            for b in range(-(-n // self.bs)):
                part = x[b * self.bs:(b + 1) * self.bs]
                c[table[b], :, :len(part)] = part.transpose(1, 0, 2)

    def device(self):
        return G.bf16(self.k), G.bf16(self.v), G.i32(self.tables), G.i32(self.lens)


def token_call(q, dev, c, nq, window, sinks, longest=None, out=None, qs=None):
    B = q.shape[0]
    k, v, tables, ctx = dev
    out = torch.full((B + 1, nq * c.d + 3), -5.0, dtype=torch.bfloat16, device=G.DEV) if out is None else out
    G.check(G.L().b200_paged_decode_window(q.data_ptr(), q.stride(0), k.data_ptr(), v.data_ptr(), tables.data_ptr(), c.width,
                                           ctx.data_ptr(), B, nq, c.nkv, c.d, c.bs, c.blocks, c.d ** -0.5, window, sinks,
                                           out.data_ptr(), out.stride(0), max(c.lens) if longest is None else longest,
                                           G.stream()), "paged_decode_window")
    return out


def queries(seed, B, nq, d, pad=0):
    x = G.rounded(np.random.default_rng(seed).standard_normal((B, nq * d)) * 2)
    dev = G.bf16(np.concatenate([x, np.full((B, pad), np.nan, np.float32)], 1))
    return x.reshape(B, nq, d), dev


def check_token(lens, nq, nkv, d, bs, window, sinks, longest=None, seed=0, rest=np.nan):
    c = Cache(seed + len(lens), lens, nkv, d, bs, window, sinks, rest=rest)
    q, qd = queries(seed, len(lens), nq, d, pad=8)
    got = G.host(token_call(qd, c.device(), c, nq, window, sinks, longest))
    assert (got[-1] == -5).all() and (got[:, nq * d:] == -5).all()
    want, weight = serving.window_decode(q, c.k, c.v, c.tables, lens, window, sinks)
    close(got[:-1, :nq * d].reshape(want.shape), want, weight)
    assert G.device_errors() == 0


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 64), (63, 0), (64, 0), (64, 4), (65, 130), (200, 1), (5000, 0),
                                          (1, 5000)])
@pytest.mark.parametrize("bs", [64, 128])
def test_token_windows(window, sinks, bs):
    check_token([0, 1, 2, 63, 64, 65, 127, 128, 129, 200, 333, 513], 8, 2, 128, bs, window, sinks)


@pytest.mark.parametrize("nq,nkv,d", [(1, 1, 64), (12, 4, 64), (28, 4, 128), (16, 1, 128), (17, 1, 64), (40, 2, 128), (8, 8, 128),
                                      (64, 1, 64)])
def test_token_heads(nq, nkv, d):
    check_token([300, 7, 150], nq, nkv, d, 64, 100, 3)


@pytest.mark.parametrize("lens,window,longest", [([1], 1, 1), ([1500], 1024, 1500), ([1500], 1024, 4), ([1500], 5000, 1500),
                                                 ([700] * 40, 300, 700), ([90, 900] * 30, 128, 900)])
def test_token_sharing_of_a_sequence(lens, window, longest):
    # one sequence in a cluster of eight CTAs, or in one when the longest is understated; many in one CTA each
    check_token(lens, 16, 8, 128, 128, window, 4, min(longest, -(-max(lens) // 128) * 128))


@pytest.mark.parametrize("rest", [3e38, -3e38, np.inf])
def test_rests_of_blocks_do_not_matter(rest):
    check_token([1, 65, 300], 8, 2, 128, 64, 70, 3, rest=rest)
    for bs in (64, 128):
        check_shared([5, 0, 130], 777, 8, 2, 128, bs, rest=rest)
        check_shared([5, 0, 130], 65, 8, 2, 64, bs, rest=rest)


def test_token_bad_entries():
    c = Cache(1, [100, 100], 2, 64, 64)
    q, qd = queries(1, 2, 4, 64)
    want, weight = serving.window_decode(q, c.k, c.v, c.tables, c.lens, 80, 0)
    for entry in (-1, c.blocks, 2**31 - 1):
        k, v, tables, ctx = c.device()
        tables[0, 1] = entry
        got = G.host(token_call(qd, (k, v, tables, ctx), c, 4, 80, 0))[:2, :256].reshape(2, 4, 64)
        assert G.device_errors() == BAD_INDEX
        close(got[1], want[1], weight[1])
    for n, seen in ((-3, 0), (1000, 128)):
        k, v, tables, ctx = c.device()
        ctx[0] = n
        k.nan_to_num_(0), v.nan_to_num_(0)
        got = G.host(token_call(qd, (k, v, tables, ctx), c, 4, 80, 0))[:2, :256].reshape(2, 4, 64)
        assert G.device_errors() == BAD_INDEX
        close(got[1], want[1], weight[1])
        clamped, w = serving.window_decode(q[:1], np.nan_to_num(c.k), np.nan_to_num(c.v), c.tables, [seen], 80, 0)
        close(got[:1], clamped, w)


def test_token_visible_nan_is_not_lost():
    c = Cache(2, [100, 100], 2, 64, 64)
    c.v[c.tables[0, 0], 0, 50, 3] = np.nan
    c.k[c.tables[1, 1], 1, 5, 3] = np.nan
    _, qd = queries(2, 2, 4, 64)
    got = G.host(token_call(qd, c.device(), c, 4, 80, 0))[:2, :256].reshape(2, 4, 64)
    assert np.isnan(got[0, :2, 3]).all() and np.isfinite(got[0, 2:]).all()
    assert np.isnan(got[1, 2:]).all() and np.isfinite(got[1, :2]).all()


def test_token_offsets_past_32_bits():
    nkv, d, bs = 8, 128, 128
    blocks = (1 << 31) // (nkv * bs * d) + 40  # more than 2^31 elements in each half
    k, v = (torch.zeros(blocks, nkv, bs, d, dtype=torch.bfloat16, device=G.DEV) for _ in range(2))
    c = Cache(3, [300], nkv, d, bs)
    high = blocks - 1 - np.arange(3)
    kk, vv = (np.nan_to_num(x[c.tables[0]]) for x in (c.k, c.v))
    k[torch.from_numpy(high).to(G.DEV)], v[torch.from_numpy(high).to(G.DEV)] = G.bf16(kk), G.bf16(vv)
    q, qd = queries(3, 1, 8, d)
    want, weight = serving.window_decode(q, c.k, c.v, c.tables, [300], 200, 4)
    c.blocks = blocks
    got = G.host(token_call(qd, (k, v, G.i32([high]), G.i32([300])), c, 8, 200, 4))[:1, :1024].reshape(1, 8, d)
    close(got, want, weight)
    del k, v
    torch.cuda.empty_cache()


def test_token_captured_calls_follow_their_lengths_on_two_streams():
    lens = [[500, 20, 300], [1, 0, 128], [77, 513, 64]]
    c = Cache(4, [513] * 3, 8, 128, 64)
    q, qd = queries(4, 3, 16, 128)
    k, v, tables, ctx = c.device()
    outs = [torch.empty(3, 2048, dtype=torch.bfloat16, device=G.DEV) for _ in range(2)]
    torch.cuda.synchronize()
    graphs = []
    for out, (window, sinks) in zip(outs, ((100, 4), (600, 0))):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            token_call(qd, (k, v, tables, ctx), c, 16, window, sinks, out=out)
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for n in lens:
        ctx.copy_(torch.tensor(n, dtype=torch.int32))
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for out, (window, sinks) in zip(outs, ((100, 4), (600, 0))):
            want, weight = serving.window_decode(q, c.k, c.v, c.tables, n, window, sinks)
            close(G.host(out).reshape(want.shape), want, weight)


# ---------------------------------------------------------- shared prefixes


def shared_call(qd, dev, c, nq, prefix, plen, pmax, ws=None, out=None, longest=None):
    k, v, tables, ctx = dev
    B = qd.shape[0]
    size = G.L().b200_paged_decode_shared_workspace_bytes(B, nq, c.nkv, c.d, pmax)
    if ws is None:
        ws = torch.full((max(size, 64) // 4,), float("nan"), device=G.DEV)
    out = torch.full((B + 1, nq * c.d + 5), -5.0, dtype=torch.bfloat16, device=G.DEV) if out is None else out
    G.check(G.L().b200_paged_decode_shared(qd.data_ptr(), qd.stride(0), k.data_ptr(), v.data_ptr(), G.ptr(prefix),
                                           G.ptr(plen), pmax, tables.data_ptr(), c.width, ctx.data_ptr(),
                                           max(c.lens) if longest is None else longest, B, nq, c.nkv, c.d, c.bs, c.blocks,
                                           c.d ** -0.5, out.data_ptr(), out.stride(0), ws.data_ptr(), ws.numel() * 4,
                                           G.stream()), "paged_decode_shared")
    return out


def check_shared(lens, plen, nq, nkv, d, bs, pmax=None, seed=0, rest=np.nan):
    pmax = plen if pmax is None else pmax
    c = Cache(seed + plen, lens, nkv, d, bs, spare=-(-pmax // bs) + 2, rest=rest)
    prefix = c.order[:-(-pmax // bs)]
    c.fill_fast(prefix, plen)
    q, qd = queries(seed, len(lens), nq, d, pad=8)
    got = G.host(shared_call(qd, c.device(), c, nq, G.i32(prefix) if pmax else None, G.i32([plen]) if pmax else None, pmax))
    assert (got[-1] == -5).all() and (got[:, nq * d:] == -5).all()
    want, weight = serving.shared_decode(q, c.k, c.v, prefix, plen, c.tables, lens)
    close(got[:-1, :nq * d].reshape(want.shape), want, weight)
    assert G.device_errors() == 0


@pytest.mark.parametrize("plen", [0, 1, 63, 64, 65, 127, 128, 129, 191, 193, 1000, 2049])
@pytest.mark.parametrize("bs", [64, 128])
def test_shared_prefix_lengths(plen, bs):
    check_shared([5, 0, 64, 130, 1], plen, 8, 2, 128, bs)


@pytest.mark.parametrize("batch,nq,nkv,d", [(1, 8, 2, 128), (32, 8, 2, 128), (33, 8, 2, 64), (65, 8, 2, 128), (50, 6, 2, 64),
                                            (19, 7, 1, 128), (9, 16, 1, 128), (7, 17, 1, 64), (3, 40, 1, 128), (2, 64, 1, 64),
                                            (3, 128, 1, 64), (140, 8, 8, 64)])
def test_shared_heads_and_batches(batch, nq, nkv, d):
    rng = np.random.default_rng(batch)
    check_shared(rng.integers(0, 150, batch).tolist(), 300, nq, nkv, d, 64)


@pytest.mark.parametrize("plen,pmax", [(0, 1000), (1, 3000), (130, 3000), (700, 701), (384, 20000)])
def test_shared_prefix_shorter_than_its_limit(plen, pmax):
    check_shared([3, 100, 0], plen, 8, 4, 128, 128, pmax)


def test_shared_nothing_at_all():
    c = Cache(5, [0, 0], 2, 64, 64, spare=4)
    _, qd = queries(5, 2, 4, 64)
    prefix = G.i32(c.order[:2])
    for plen, pmax in ((0, 100), (-7, 100)):
        got = G.host(shared_call(qd, c.device(), c, 4, prefix, G.i32([plen]), pmax, longest=64))
        assert (got[:2, :256] == 0).all()
    got = G.host(shared_call(qd, c.device(), c, 4, None, None, 0, longest=64))
    assert (got[:2, :256] == 0).all() and G.device_errors() == 0


def test_shared_bad_entries():
    c = Cache(6, [70, 30], 2, 64, 64, spare=6)
    c.fill_fast(c.order[:2], 128)
    q, qd = queries(6, 2, 4, 64)
    k, v, tables, ctx = c.device()
    k.nan_to_num_(0), v.nan_to_num_(0)
    for bad in (-1, c.blocks, 2**31 - 1):
        got = G.host(shared_call(qd, (k, v, tables, ctx), c, 4, G.i32([c.order[0], bad]), G.i32([128]), 128))
        assert G.device_errors() == BAD_INDEX and np.isfinite(got).all()
    # a prefix length behind the limit is clamped to it
    want, weight = serving.shared_decode(q, c.k, c.v, c.order[:2], 100, c.tables, c.lens)
    got = G.host(shared_call(qd, (k, v, tables, ctx), c, 4, G.i32(c.order[:2]), G.i32([5000]), 100))
    close(got[:2, :256].reshape(want.shape), want, weight)


def test_shared_visible_nan_is_not_lost():
    for at in (10, 127, 129):  # in a whole tile, and in the last one
        c = Cache(7, [70, 30], 2, 64, 64, spare=6)
        c.fill_fast(c.order[:3], 130)
        c.v[c.order[at // 64], 1, at % 64, 3] = np.nan
        _, qd = queries(7, 2, 4, 64)
        got = G.host(shared_call(qd, c.device(), c, 4, G.i32(c.order[:3]), G.i32([130]), 130))[:2, :256].reshape(2, 4, 64)
        assert np.isnan(got[:, 2:, 3]).all() and np.isfinite(got[:, :2]).all()


def far_below(c, table, positions):
    """Keys of -inf in the first dim: with queries above zero there, scores of -inf."""
    for j in positions:
        c.k[table[j // c.bs], :, j % c.bs, 0] = -np.inf


@pytest.mark.parametrize("plen,positions", [(1, [0]), (128, range(128)), (129, [128]), (300, range(128, 256)), (1000, range(1000)),
                                            (1000, range(5, 1000))], ids=["1", "128", "last", "tile", "1000", "but-5"])
@pytest.mark.parametrize("d", [64, 128])
def test_shared_prefix_without_weight(plen, positions, d):
    # stretches of the prefix whose every score is -inf weigh nothing beside the rest
    lens = [70, 1, 30]
    c = Cache(10, lens, 2, d, 64, spare=20)
    prefix = c.order[:-(-plen // 64)]
    c.fill_fast(prefix, plen)
    far_below(c, prefix, positions)
    q = G.rounded(np.random.default_rng(10).standard_normal((3, 8 * d)) * 2)
    q[:, ::d] = G.rounded(np.abs(q[:, ::d]) + 1)
    want, weight = serving.shared_decode(q.reshape(3, 8, d), c.k, c.v, prefix, plen, c.tables, lens)
    got = G.host(shared_call(G.bf16(q), c.device(), c, 8, G.i32(prefix), G.i32([plen]), plen))[:3, :8 * d]
    close(got.reshape(want.shape), want, weight)


def test_shared_captured_calls_with_workspaces_of_their_own():
    c = Cache(8, [200] * 9, 4, 128, 64, spare=20)
    prefix = c.order[:16]
    c.fill_fast(prefix, 1000)
    q, qd = queries(8, 9, 16, 128)
    dev = c.device()
    plen, pre = G.i32([1000]), G.i32(prefix)
    calls = []
    torch.cuda.synchronize()
    for _ in range(2):
        size = G.L().b200_paged_decode_shared_workspace_bytes(9, 16, 4, 128, 1000)
        ws = torch.full((size // 4,), float("nan"), device=G.DEV)
        out = torch.empty(9, 2048, dtype=torch.bfloat16, device=G.DEV)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            shared_call(qd, dev, c, 16, pre, plen, 1000, ws=ws, out=out)
        calls.append((g, out, ws, torch.cuda.Stream()))
    for n, own in ((1000, 200), (65, 1), (0, 200), (777, 0)):
        plen.fill_(n)
        dev[3].fill_(own)
        torch.cuda.synchronize()
        for _ in range(3):
            for g, _, _, s in calls:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        want, weight = serving.shared_decode(q, c.k, c.v, prefix, n, c.tables, [own] * 9)
        for _, out, _, _ in calls:
            close(G.host(out).reshape(want.shape), want, weight)


# ------------------------------------------------- many tiles, far offsets


@pytest.mark.parametrize("nq,nkv,d,dv,window,sinks", [(4, 2, 128, 128, 4600, 5), (3, 1, 128, 128, 6000, 0), (2, 2, 192, 128, 3000, 200),
                                                      (4, 2, 64, 64, 2500, 1), (4, 4, 32, 32, 5000, 4)])
def test_prompt_items_of_many_tiles(nq, nkv, d, dv, window, sinks):
    lens = [5777, 1500]
    q, k, v = prompt_inputs(14, sum(lens), nq, nkv, d, dv)
    got = prompt(q, k, v, lens, window, sinks)
    rng, at = np.random.default_rng(14), 0
    for n in lens:
        rows = np.unique(np.concatenate([rng.integers(0, n, 60), [0, n - 1, min(n - 1, window), min(n - 1, window + 127)]]))
        j = np.arange(n)[None]
        sees = (j <= rows[:, None]) & ((rows[:, None] - j < window) | (j < sinks))
        for h in range(nq):
            kv = h * nkv // nq
            want, weight = serving.attend(q[at + rows, h], k[at:at + n, kv], v[at:at + n, kv], sees, d ** -0.5)
            close(got[at + rows, h], want, weight)
        at += n
    assert np.isfinite(got).all() and G.device_errors() == 0


@pytest.mark.parametrize("nq,nkv,d,bs", [(8, 2, 128, 128), (8, 2, 64, 64)])
def test_shared_prefix_of_many_tiles(nq, nkv, d, bs):
    check_shared([300, 0, 1, 2000, 77], 20011, nq, nkv, d, bs)


def test_prompt_offsets_past_32_bits():
    rows, stride, n, nq, nkv, d = 33000, 70000, 300, 4, 2, 64  # 2.3e9 elements in inputs and outputs
    q, k, v = prompt_inputs(15, n, nq, nkv, d, d)
    x = torch.zeros(rows, stride, dtype=torch.bfloat16, device=G.DEV)
    out = torch.full((rows, stride), -5.0, dtype=torch.bfloat16, device=G.DEV)
    cols = (0, 40000, 69800)
    for y, c in zip((q, k, v), cols):
        x[rows - n:, c:c + y.shape[1] * d] = G.bf16(y.reshape(n, -1))
    cu = G.i32([rows - n, rows])
    at = [x.data_ptr() + 2 * c for c in cols]
    G.check(G.L().b200_flash_prefill_window(at[0], stride, d, at[1], stride, d, at[2], stride, d, out.data_ptr() + 2 * 60000, stride,
                                            d, cu.data_ptr(), 1, n, rows, nq, nkv, d, d, d ** -0.5, 130, 3, G.stream()))
    want, weight = serving.window_prompt(q, k, v, [n], 130, 3, d ** -0.5)
    close(G.host(out[rows - n:, 60000:60000 + nq * d]).reshape(want.shape), want, weight)
    out[rows - n:, 60000:60000 + nq * d] = -5
    assert bool((out == -5).all()) and G.device_errors() == 0
    del x, out
    torch.cuda.empty_cache()


def test_shared_offsets_past_32_bits():
    nkv, d, bs, plen, lens = 8, 128, 128, 500, [300, 0]
    blocks = (1 << 31) // (nkv * bs * d) + 40  # more than 2^31 elements in each half
    k, v = (torch.zeros(blocks, nkv, bs, d, dtype=torch.bfloat16, device=G.DEV) for _ in range(2))
    c = Cache(16, lens, nkv, d, bs, spare=5)
    c.fill_fast(c.order[:4], plen)
    used = np.concatenate([c.tables[0], c.order[:4]])
    high = torch.from_numpy(blocks - 1 - np.arange(len(used))).to(G.DEV)
    k[high], v[high] = G.bf16(np.nan_to_num(c.k[used])), G.bf16(np.nan_to_num(c.v[used]))
    q, qd = queries(16, 2, 16, d)
    want, weight = serving.shared_decode(q, c.k, c.v, c.order[:4], plen, c.tables, lens)
    c.blocks = blocks
    tables = torch.stack([high[:3], high[:3]]).to(torch.int32)
    got = G.host(shared_call(qd, (k, v, tables, G.i32(lens)), c, 16, high[3:].to(torch.int32), G.i32([plen]), plen))
    close(got[:2, :2048].reshape(want.shape), want, weight)
    del k, v
    torch.cuda.empty_cache()
