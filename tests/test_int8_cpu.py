"""Host-side checks (no GPU) of the 8-bit linear layers and the grouped router:
every documented refusal returns its status before anything touches a device,
and the numpy restatements hold their defining properties."""

import os

import numpy as np
import pytest

from atb_llm_study_b200 import capi
from oracle import int8, moe

INVALID, UNSUPPORTED = -1, -7
P = 1 << 20  # an aligned address no call reads: every case below is refused on the host

needs_lib = pytest.mark.skipif(not os.path.exists(capi.LIB_PATH), reason="library not built")

QUANT = dict(x=P, ldx=64, src_rows=4, src=None, count=None, q=P, ldq=64, scale=P, rows=4, dim=64, st=None)
NORM = dict(x=P, res=None, w=P, q=P, ldq=64, scale=P, out=None, res_out=None, rows=4, dim=64, stride=64, eps=1e-6, st=None)
GEMM = dict(A=P, lda=64, sa=P, B=P, ldb=64, sb=P, C=P, ldc=32, M=4, N=32, K=64, epi=0, bias=None, R=None, ldr=0, st=None)
GROUPED = dict(A=P, lda=64, sa=P, B=P, ldb=64, sb=P, C=P, ldc=32, off=P, groups=2, rows=4, N=32, K=64, epi=0, st=None)
TOPK = dict(logits=P, ld=64, bias=None, T=4, E=64, k=6, score=0, groups=8, keep=3, best=1, renorm=0, scale=1.0, ids=P,
            w=P, st=None)

ROUTE = dict(x=P, ldx=64, gate=P, bias=None, T=4, H=64, E=64, k=6, score=0, groups=8, keep=3, best=1, renorm=0, scale=1.0,
             ids=P, w=P, logits=P, st=None)

REFUSED = [
    ("b200_quant_rows_int8", QUANT, [
        dict(x=None), dict(q=None), dict(scale=None), dict(rows=-1), dict(dim=0), dict(dim=24), dict(ldx=48), dict(ldx=65),
        dict(ldq=48), dict(ldq=72), dict(src_rows=3), dict(src_rows=-1, src=P), dict(x=P + 8), dict(q=P + 4),
        dict(scale=P + 2), dict(src=P + 1), dict(count=P + 2)]),
    ("b200_rmsnorm_quant_int8", NORM, [
        dict(x=None), dict(w=None), dict(q=None), dict(scale=None), dict(rows=-1), dict(dim=24), dict(stride=48),
        dict(stride=68), dict(ldq=48), dict(ldq=72), dict(out=P + 2), dict(res=P + 2), dict(res_out=P + 8)]),
    ("b200_gemm_int8", GEMM, [
        dict(A=None), dict(B=None), dict(sa=None), dict(sb=None), dict(C=None), dict(M=-1), dict(N=-8), dict(K=0),
        dict(K=40), dict(lda=48), dict(lda=72), dict(ldb=48), dict(ldb=72), dict(N=28, ldc=32), dict(ldc=24), dict(ldc=36),
        dict(epi=6), dict(epi=-1), dict(epi=1), dict(epi=4), dict(epi=5, bias=P), dict(epi=2), dict(epi=2, R=P, ldr=24),
        dict(epi=2, R=P, ldr=33), dict(epi=3, N=24, ldc=16), dict(A=P + 8), dict(B=P + 1), dict(sa=P + 4), dict(sb=P + 8),
        dict(C=P + 2), dict(epi=1, bias=P + 2)]),
    ("b200_grouped_gemm_int8", GROUPED, [
        dict(A=None), dict(off=None), dict(off=P + 2), dict(groups=0), dict(groups=257), dict(rows=-1), dict(N=0),
        dict(K=40), dict(epi=1), dict(epi=2), dict(epi=3, N=24, ldc=16), dict(lda=48), dict(ldc=24), dict(sb=P + 4)]),
    ("b200_moe_topk_grouped", TOPK, [
        dict(logits=None), dict(ids=None), dict(w=None), dict(T=-1), dict(E=0), dict(ld=63), dict(score=2), dict(score=-1),
        dict(groups=0), dict(groups=7), dict(keep=0), dict(keep=9), dict(best=0), dict(best=3), dict(groups=64, best=2),
        dict(k=0), dict(k=9), dict(keep=1, groups=16), dict(logits=P + 2), dict(bias=P + 1)]),
    ("b200_moe_route_grouped", ROUTE, [
        dict(x=None), dict(gate=None), dict(logits=None), dict(H=60), dict(ldx=56), dict(ldx=68), dict(x=P + 8),
        dict(gate=P + 2), dict(logits=P + 4), dict(T=-1), dict(E=0), dict(groups=7), dict(k=9), dict(score=3)]),
]


@needs_lib
@pytest.mark.parametrize("name,base,change", [(n, b, c) for n, b, cs in REFUSED for c in cs],
                         ids=[f"{n[5:]}-{','.join(c)}-{i}" for n, b, cs in REFUSED for i, c in enumerate(cs)])
def test_refused(name, base, change):
    assert getattr(capi.lib(), name)(*{**base, **change}.values()) == INVALID


@needs_lib
@pytest.mark.parametrize("name,base,change", [
    ("b200_quant_rows_int8", QUANT, dict(rows=1 << 31, src_rows=1 << 31)),
    ("b200_rmsnorm_quant_int8", NORM, dict(rows=1 << 31)),
    ("b200_rmsnorm_quant_int8", NORM, dict(dim=8208, stride=8208, ldq=8208)),
    ("b200_gemm_int8", GEMM, dict(K=131072, lda=131072, ldb=131072)),  # 128 * 128 * K passes 31 bits
    ("b200_gemm_int8", GEMM, dict(M=1 << 31)),
    ("b200_grouped_gemm_int8", GROUPED, dict(K=131072, lda=131072, ldb=131072)),
    ("b200_grouped_gemm_int8", GROUPED, dict(rows=1 << 30)),
    ("b200_moe_topk_grouped", TOPK, dict(E=264, ld=264)),
    ("b200_moe_topk_grouped", TOPK, dict(groups=64, keep=8)),
    ("b200_moe_route_grouped", ROUTE, dict(E=264)),
    ("b200_moe_route_grouped", ROUTE, dict(T=1 << 24)),
], ids=str)
def test_unsupported(name, base, change):
    assert getattr(capi.lib(), name)(*{**base, **change}.values()) == UNSUPPORTED


@needs_lib
@pytest.mark.parametrize("name,base,change", [
    ("b200_quant_rows_int8", QUANT, dict(rows=0)), ("b200_rmsnorm_quant_int8", NORM, dict(rows=0)),
    ("b200_gemm_int8", GEMM, dict(M=0)), ("b200_gemm_int8", GEMM, dict(N=0)),
    ("b200_grouped_gemm_int8", GROUPED, dict(rows=0)), ("b200_moe_topk_grouped", TOPK, dict(T=0)),
    ("b200_moe_route_grouped", ROUTE, dict(T=0))], ids=str)
def test_nothing_to_do(name, base, change):
    assert getattr(capi.lib(), name)(*{**base, **change}.values()) == 0


def test_oracle_quant_rows():
    q, s = int8.quant_rows(np.array([[1.0, -2.0, 0.5, 2.0], [0, 0, 0, 0], [np.inf, 1, 2, 3], [1, np.nan, 2, 3]]))
    # 127 * 1 / 2 = 63.5 is a tie: to the even 64; 127 * 0.5 / 2 = 31.75
    np.testing.assert_array_equal(q, [[64, -127, 32, 127], [0] * 4, [0] * 4, [0] * 4])
    assert s[0] == np.float32(2) / np.float32(127) and s[1] == 0 and np.isnan(s[2:]).all()


def test_oracle_route_grouped():
    rng = np.random.default_rng(0)
    lg = rng.standard_normal((50, 64)).astype(np.float32)
    ids, w = moe.route_grouped(lg, 6, renormalize=False, scale=1.5)
    rid, rw = moe.route_topk(lg, 6, renormalize=False, scale=1.5)  # one group, no bias: the ungrouped gate
    np.testing.assert_array_equal(ids, rid)
    np.testing.assert_allclose(w, rw, rtol=1e-5)
    ids, w = moe.route_grouped(lg, 4, sigmoid=True, groups=8, keep=2, best=2)
    assert all(len(set(r // 8)) <= 2 for r in ids)
    np.testing.assert_allclose(w.sum(1), 1, rtol=1e-12)
    # a bias moves the choice and not the weights
    b = np.zeros(64)
    b[63] = 10
    ids, w = moe.route_grouped(lg, 2, sigmoid=True, bias=b, renormalize=False)
    assert (ids[:, 0] == 63).all()
    np.testing.assert_allclose(w[:, 0], 1 / (1 + np.exp(-lg[:, 63].astype(np.float64))))
    # a row with nothing left is uniform and takes the lowest experts
    ids, w = moe.route_grouped(np.full((1, 8), -np.inf, np.float32), 2, renormalize=False)
    assert list(ids[0]) == [0, 1] and np.allclose(w, 1 / 8)
