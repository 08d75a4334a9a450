"""Host-side checks (no GPU) of the serving step's operators: every documented
refusal returns its status before anything touches a device, the restatements
hold their defining properties, and the stretches of a shared prefix cover it."""

import os

import numpy as np
import pytest

import oracle
from atb_llm_study_b200 import capi
from oracle import serving

INVALID, UNSUPPORTED = -1, -7
P = 1 << 20  # an aligned address no call reads: every case below is refused on the host

needs_lib = pytest.mark.skipif(not os.path.exists(capi.LIB_PATH), reason="library not built")

EXTEND = dict(cached=P, new=P, n=4, bs=64, tables=P, width=8, free=P, count=P, blocks=64, ctx=P, cu=P, pos=P, slots=P, cap=64,
              left=P, missing=P, st=None)
RELEASE = dict(cached=P, keep=P, n=4, bs=64, tables=P, width=8, free=P, cap=64, count=P, blocks=64, lens=P, left=P, st=None)
PROMPT = dict(q=P, qs=256, qh=64, k=P, ks=128, kh=64, v=P, vs=128, vh=64, o=P, os=256, oh=64, cu=P, n=1, longest=8, total=8,
              nq=4, nkv=2, d=64, dv=64, scale=0.1, window=4, sinks=0, st=None)
TOKEN = dict(q=P, qs=256, k=P, v=P, tables=P, width=4, ctx=P, b=2, nq=4, nkv=2, d=64, bs=64, blocks=8, scale=0.1, window=4,
             sinks=0, o=P, os=256, longest=64, st=None)
SHARED = dict(q=P, qs=256, k=P, v=P, prefix=P, plen=P, pmax=100, tables=P, width=4, ctx=P, longest=64, b=2, nq=4, nkv=2, d=64,
              bs=64, blocks=8, scale=0.1, o=P, os=256, ws=P, wsb=1 << 30, st=None)
LOGITS = dict(x=P, ld=1000, rows=2, vocab=1000, hist=P, hld=10, prompt=P, lens=P, rep=P, freq=P, pres=P, boff=P, bid=P, bval=P,
              mask=P, mld=32, masks=2, mrow=P, out=P, ldo=1000, next=P, st=None)

REFUSED = [
    ("b200_block_tables_extend", EXTEND, [
        dict(cached=None), dict(new=None), dict(tables=None), dict(free=None), dict(count=None), dict(ctx=None), dict(left=None),
        dict(n=-1), dict(bs=0), dict(width=0), dict(blocks=0), dict(cap=-1), dict(cached=P + 2), dict(slots=P + 4),
        dict(pos=P + 4), dict(missing=P + 1)]),
    ("b200_block_tables_release", RELEASE, [
        dict(cached=None), dict(keep=None), dict(tables=None), dict(free=None), dict(count=None), dict(lens=None),
        dict(left=None), dict(n=-1), dict(bs=0), dict(width=0), dict(blocks=0), dict(cap=-1), dict(free=P + 2)]),
    ("b200_flash_prefill_window", PROMPT, [
        dict(q=None), dict(k=None), dict(v=None), dict(o=None), dict(cu=None), dict(n=-1), dict(longest=-1), dict(total=-1),
        dict(nq=0), dict(nkv=0), dict(nq=3), dict(window=0), dict(window=-1), dict(sinks=-1), dict(scale=0.0),
        dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(qs=252), dict(qs=192), dict(kh=60),
        dict(os=248), dict(q=P + 8), dict(o=P + 2), dict(cu=P + 2)]),
    ("b200_paged_decode_window", TOKEN, [
        dict(q=None), dict(k=None), dict(v=None), dict(tables=None), dict(ctx=None), dict(o=None), dict(b=-1), dict(nq=0),
        dict(nkv=3), dict(width=0), dict(blocks=0), dict(longest=-1), dict(longest=257), dict(window=0), dict(sinks=-1),
        dict(scale=0.0), dict(scale=float("nan")), dict(qs=252), dict(qs=248), dict(os=248), dict(q=P + 8), dict(k=P + 8),
        dict(v=P + 4), dict(o=P + 1), dict(tables=P + 2), dict(ctx=P + 2)]),
    ("b200_paged_decode_shared", SHARED, [
        dict(q=None), dict(k=None), dict(tables=None), dict(ctx=None), dict(o=None), dict(b=-1), dict(nkv=3), dict(pmax=-1),
        dict(prefix=None), dict(plen=None), dict(prefix=P + 2), dict(plen=P + 1), dict(ws=None), dict(ws=P + 16),
        dict(wsb=100), dict(longest=257), dict(scale=-0.1), dict(qs=252), dict(os=248)]),
    ("b200_logits_process", LOGITS, [
        dict(x=None), dict(out=None, next=None), dict(rows=-1), dict(vocab=0), dict(ld=999), dict(ldo=999), dict(out=P, x=P, ldo=1008),
        dict(hist=None), dict(lens=None), dict(hld=0), dict(boff=None), dict(bid=None), dict(bval=None), dict(mask=None),
        dict(mld=31), dict(masks=0), dict(mrow=None, masks=1), dict(hist=P + 2), dict(rep=P + 1), dict(x=P + 1),
        dict(out=P + 1), dict(next=P + 4)]),
]
TOO_MUCH = [
    ("b200_block_tables_extend", EXTEND, [dict(n=8193), dict(blocks=1 << 31), dict(cap=1 << 31), dict(width=1 << 30)]),
    ("b200_block_tables_release", RELEASE, [dict(n=8193), dict(blocks=1 << 31), dict(cap=1 << 31), dict(width=1 << 30)]),
    ("b200_flash_prefill_window", PROMPT, [dict(d=96, dv=96), dict(d=64, dv=128), dict(total=(1 << 31) - 2)]),
    ("b200_paged_decode_window", TOKEN, [dict(d=32), dict(d=96), dict(bs=32), dict(bs=256), dict(blocks=1 << 30),
                                         dict(width=1 << 29)]),
    ("b200_paged_decode_shared", SHARED, [dict(d=96), dict(bs=16), dict(nq=258, nkv=2, qs=258 * 64, os=258 * 64),
                                          dict(pmax=(1 << 31) - 1)]),
    ("b200_logits_process", LOGITS, [dict(vocab=(1 << 23) + 1, ld=1 << 24, ldo=1 << 24, mld=1 << 19), dict(rows=1 << 28)]),
]


@needs_lib
@pytest.mark.parametrize("name,base,change,status",
                         [(n, b, c, s) for s, table in ((INVALID, REFUSED), (UNSUPPORTED, TOO_MUCH)) for n, b, cs in table for c in cs],
                         ids=lambda x: "" if isinstance(x, dict) and len(x) > 9 else str(x))
def test_refused(name, base, change, status):
    assert getattr(capi.lib(), name)(*{**base, **change}.values()) == status


@needs_lib
@pytest.mark.parametrize("name,base,change,status", [
    # products that would wrap in 64 bits: 2^62 blocks x 2 heads x 64 tokens = 2^69, 3 heads x 2^62 elements
    ("b200_paged_decode_window", TOKEN, dict(blocks=1 << 62, b=0), UNSUPPORTED),
    ("b200_paged_decode_shared", SHARED, dict(blocks=1 << 62, b=0), UNSUPPORTED),
    ("b200_flash_prefill_window", PROMPT, dict(qh=1 << 62), INVALID),
    ("b200_flash_prefill_window", PROMPT, dict(oh=1 << 62), INVALID),
    # the largest cache that 32-bit rows reach, and one block more
    ("b200_paged_decode_window", TOKEN, dict(blocks=((1 << 31) - 1) // 128, b=0), 0),
    ("b200_paged_decode_window", TOKEN, dict(blocks=((1 << 31) - 1) // 128 + 1, b=0), UNSUPPORTED),
], ids=lambda x: "" if isinstance(x, dict) and len(x) > 9 else str(x))
def test_sizes_whose_products_wrap(name, base, change, status):
    assert getattr(capi.lib(), name)(*{**base, **change}.values()) == status


@needs_lib
def test_nothing_to_do():
    L = capi.lib()
    assert L.b200_flash_prefill_window(*{**PROMPT, "n": 0}.values()) == 0
    assert L.b200_flash_prefill_window(*{**PROMPT, "total": 0}.values()) == 0
    assert L.b200_paged_decode_window(*{**TOKEN, "b": 0}.values()) == 0
    assert L.b200_paged_decode_shared(*{**SHARED, "b": 0}.values()) == 0
    assert L.b200_logits_process(*{**LOGITS, "rows": 0}.values()) == 0
    ws = L.b200_paged_decode_shared_workspace_bytes
    assert ws(0, 4, 2, 64, 100) == ws(2, 4, 3, 64, 100) == ws(2, 4, 2, 96, 100) == ws(2, 4, 2, 64, 0) == 0
    # 2 sequences of 2 heads: one row tile a kv head; 1 key tile each: 2 CTAs, 4 slots of 2 x 128 x (64 + 1)
    assert ws(2, 4, 2, 64, 100) == 4 * 256 * 65 * 4
    assert ws(64, 32, 8, 128, 16384) >= (148 + 8) * 256 * 129 * 4


@pytest.mark.parametrize("workers", [1, 2, 7, 148])
@pytest.mark.parametrize("items,K", [(1, 1), (1, 300), (3, 1), (16, 9), (64, 128), (5, 77), (200, 2)])
def test_stretches_cover_every_item_once(workers, items, K):
    """shared_prefix.h: W = min(workers, U) stretches of U / W units or, the first U mod W, one more; the formulas for a
    stretch's first unit and a unit's stretch agree, and every stretch from an item's first to its last has a part of it, in a
    slot of its own."""
    U = items * K
    W = min(workers, U)
    each, longer = divmod(U, W)
    first = [c * each + min(c, longer) for c in range(W + 1)]
    assert first[0] == 0 and first[W] == U and all(a < b for a, b in zip(first, first[1:]))
    owner = [c for c in range(W) for _ in range(first[c], first[c + 1])]
    cut = longer * (each + 1)
    assert owner == [u // (each + 1) if u < cut else longer + (u - cut) // each for u in range(U)]
    slots = set()
    for i in range(items):
        parts = sorted(set(owner[i * K:(i + 1) * K]))
        assert parts == list(range(parts[0], parts[-1] + 1))
        for c in parts:
            assert c + i < workers + items and c + i not in slots
            slots.add(c + i)


STRETCHES = """
#include <stdint.h>
#include <stdio.h>
#include <algorithm>
#define B200_DEV inline
typedef void* cudaStream_t;
using std::max;
using std::min;
"""
STRETCHES_MAIN = """
#include "shared_prefix.h"
// length max_length workers row_tiles per_tile group batch nkv -> stretches, then the slots that each sequence's head 0 reads
int main() {
  int length, batch, nkv;
  b200::PrefixParts p{};
  while (scanf("%d %d %d %d %d %d %d %d", &length, &p.max_length, &p.workers, &p.row_tiles, &p.per_tile, &p.group, &batch, &nkv) == 8) {
    p.length = &length;
    const int K = (b200::prefix_length(p) + 127) / 128, units = K * nkv * b200::prefix_pairs(p);
    const b200::PrefixDeal deal(p, units);
    printf("%d %d", K, units ? deal.W : 0);
    for (int c = 0; units && c <= deal.W; ++c) printf(" %d", deal.first_unit(c));
    printf("\\n");
    for (int b = 0; b < batch; ++b)
      for (int kh = 0; kh < nkv; ++kh) {
        const b200::PrefixSpan s = b200::prefix_span(p, b, kh, nkv, 0, 64);
        printf("%d %lld ", s.count, s.count ? (long long)(s.lse - p.lse) : -1);
        if (s.count && (s.parts - p.parts) != (s.lse - p.lse) * 64) return 1;
      }
    printf("\\n");
  }
  return 0;
}
"""


def test_stretches_and_parts_of_the_header(tmp_path):
    """shared_prefix.h itself, compiled for the host: the stretches cover all units in order, every part that a stretch
    leaves lies in a slot of its own inside the workspace, and a sequence reads the parts that hold its rows, no others."""
    import shutil
    import subprocess

    csrc = os.path.join(os.path.dirname(os.path.abspath(capi.__file__)), "csrc")
    shutil.copy(os.path.join(csrc, "shared_prefix.h"), tmp_path)
    (tmp_path / "common.cuh").write_text("#pragma once\n" + STRETCHES)
    (tmp_path / "main.cpp").write_text(STRETCHES_MAIN)
    subprocess.run(["g++", "-std=c++17", "-O1", "-o", tmp_path / "main", tmp_path / "main.cpp"], check=True)
    cases = []
    for batch, group, nkv in ((1, 1, 1), (5, 4, 8), (64, 4, 8), (65, 4, 2), (9, 17, 1), (256, 8, 1), (3, 128, 2), (140, 1, 8)):
        for length, most in ((0, 100), (1, 1), (128, 128), (129, 1000), (1001, 1001), (16384, 16384), (500, 300), (-3, 10)):
            per = 128 // group
            tiles = -(-batch // per)
            items = nkv * -(-tiles // 2)
            workers = max(1, min(items * -(-most // 128), 148))
            cases.append((length, most, workers, tiles, per, group, batch, nkv))
    out = subprocess.run([tmp_path / "main"], input="\n".join(" ".join(map(str, c)) for c in cases), capture_output=True, text=True,
                         check=True).stdout.splitlines()
    assert len(out) == 2 * len(cases)
    for (length, most, workers, tiles, per, group, batch, nkv), head, spans in zip(cases, out[::2], out[1::2]):
        K, W, *first = map(int, head.split())
        items = nkv * -(-tiles // 2)
        assert K == -(-max(0, min(length, most)) // 128) and W == min(workers, K * items)
        spans = np.array(spans.split(), np.int64).reshape(batch, nkv, 2)
        if K == 0:
            assert (spans[..., 0] == 0).all()
            continue
        assert first[0] == 0 and first[W] == K * items and (np.diff(first) > 0).all()
        parts = {}  # item -> the slots of its parts, as the kernel numbers them
        for c in range(W):
            for item in range(first[c] // K, (first[c + 1] - 1) // K + 1):
                parts.setdefault(item, []).append(2 * (c + item))
        slots = [s for ss in parts.values() for s in ss]
        assert len(set(slots)) == len(slots) and max(slots) + 1 < 2 * (workers + items)
        for b in range(batch):
            for kh in range(nkv):
                mine = parts[kh * -(-tiles // 2) + b // per // 2]
                assert mine == list(range(mine[0], mine[0] + 2 * len(mine), 2))
                assert spans[b, kh].tolist() == [len(mine), (mine[0] + b // per % 2) * 128 + b % per * group]


def test_window_without_an_end_is_causal_attention():
    rng = np.random.default_rng(0)
    q, k, v = (rng.standard_normal((9, h, 16)).astype(np.float32) for h in (4, 2, 2))
    want = oracle.varlen_causal_attention(q, k, v, [0, 5, 9], 4, 2)
    got, _ = serving.window_prompt(q, k, v, [5, 4], 9, 0, 0.25)
    np.testing.assert_allclose(got, want, atol=1e-5)
    got, _ = serving.window_prompt(q, k, v, [5, 4], 2, 9, 0.25)
    np.testing.assert_allclose(got, want, atol=1e-5)


def test_window_decode_is_the_last_row_of_a_prompt():
    rng = np.random.default_rng(1)
    q, k, v = (rng.standard_normal((50, h, 16)) for h in (4, 2, 2))
    kc, vc = (np.ascontiguousarray(x[:48].reshape(6, 8, 2, 16).transpose(0, 2, 1, 3)) for x in (k, v))
    for n, window, sinks in ((48, 5, 3), (17, 40, 0), (30, 1, 0), (30, 28, 4)):
        want, _ = serving.window_prompt(q[:n], k[:n], v[:n], [n], window, sinks, 0.25)
        got, _ = serving.window_decode(q[n - 1:n], kc, vc, [np.arange(6)], [n], window, sinks)
        np.testing.assert_allclose(got[0], want[-1], atol=1e-12)


def test_shared_prefix_is_attention_over_both():
    rng = np.random.default_rng(2)
    q = rng.standard_normal((2, 4, 16))
    kc, vc = (rng.standard_normal((9, 2, 8, 16)) for _ in range(2))
    got, _ = serving.shared_decode(q, kc, vc, [3, 1], 13, [[4, 5], [0, 2]], [9, 0])
    keys = np.concatenate([serving.cached_rows(kc, [3, 1], range(13)), serving.cached_rows(kc, [4, 5], range(9))])
    vals = np.concatenate([serving.cached_rows(vc, [3, 1], range(13)), serving.cached_rows(vc, [4, 5], range(9))])
    s = np.einsum("hd,nhd->hn", q[0], np.repeat(keys, 2, 1)) * 0.25
    p = np.exp(s) / np.exp(s).sum(1, keepdims=True)
    np.testing.assert_allclose(got[0], np.einsum("hn,nhd->hd", p, np.repeat(vals, 2, 1)), atol=1e-12)


def test_released_blocks_come_back_in_order():
    tables, ctx, cu, pos, slots, left, missing = serving.extend([0, 5], [9, 2], 4, [[-1] * 4, [7, 8, -1, -1]],
                                                                np.array([3, 1, 4, 6]), 4, 12)
    assert tables.tolist() == [[6, 4, 1, -1], [7, 8, -1, -1]] and left == 1 and missing == 0
    assert slots.tolist() == [24, 25, 26, 27, 16, 17, 18, 19, 4, 33, 34, -1] and cu.tolist() == [0, 9, 11]
    free, lens, count = serving.release(ctx, np.array([4, 0]), 4, tables, np.array([3, 0, 0, 0, 0]), left)
    assert free.tolist() == [3, 4, 1, 7, 8] and lens.tolist() == [4, 0] and count == 5
    assert serving.extend([0], [9], 4, [[-1] * 4], np.array([1, 2]), 2, 3)[5:] == (2, 1)
