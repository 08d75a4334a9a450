"""GPU parity of b200_moe_topk_grouped against the float64 restatement.

Expert ids are equal, ties and near-ties included: the definition ranks scores
in 64 bits, and the kernel decides in double whatever fp32 cannot tell apart.
Weights: fp32 scores are within 1.8e-6 of the largest one (expf 2 ulp, at most
21 roundings of the sum, the division), renormalising adds as much again.
"""

import numpy as np
import pytest
import torch

from oracle import moe

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import gpu_util as G

F = np.float32


def route(lg, k, sigmoid=False, bias=None, groups=1, keep=1, best=1, renorm=True, scale=1.0, pad=0):
    T, E = lg.shape
    d = G.f32(np.concatenate([lg, np.full((T, pad), 1e9, F)], 1) if pad else lg)
    ids = torch.full((T + 1, k), -5, dtype=torch.int32, device=G.DEV)
    w = torch.full((T + 1, k), -5.0, dtype=torch.float32, device=G.DEV)
    G.check(G.L().b200_moe_topk_grouped(d.data_ptr(), E + pad, G.ptr(None if bias is None else G.f32(bias)), T, E, k,
                                        int(sigmoid), groups, keep, best, int(renorm), scale, ids.data_ptr(), w.data_ptr(),
                                        G.stream()), "moe_topk_grouped")
    ids, w = ids.cpu().numpy(), G.host(w)
    assert (ids[T] == -5).all() and (w[T] == -5).all()
    return ids[:T], w[:T]


def check(lg, k, **kw):
    ids, w = route(lg, k, **kw)
    kw.pop("pad", None)
    rid, rw = moe.route_grouped(lg, k, kw.get("sigmoid", False), kw.get("bias"), kw.get("groups", 1), kw.get("keep", 1),
                                kw.get("best", 1), kw.get("renorm", True), kw.get("scale", 1.0))
    np.testing.assert_array_equal(ids, rid)
    np.testing.assert_allclose(w, rw, rtol=1e-5, atol=2e-6 * kw.get("scale", 1.0))
    return ids, w


CASES = [(1, 1, 1, 1, 1, 1), (5, 2, 1, 1, 1, 1), (777, 8, 2, 1, 1, 1), (64, 64, 6, 1, 1, 1), (1000, 128, 8, 1, 1, 1),
         (2049, 256, 8, 8, 4, 2), (300, 160, 6, 8, 3, 1), (301, 160, 6, 5, 2, 2), (100, 64, 8, 8, 1, 2), (100, 64, 8, 32, 4, 2),
         (99, 96, 5, 3, 2, 2), (98, 255, 7, 17, 3, 2), (97, 252, 8, 18, 9, 1), (96, 7, 3, 7, 4, 1), (95, 30, 4, 3, 3, 2),
         (94, 250, 8, 2, 1, 2), (93, 6, 6, 2, 2, 1), (92, 34, 2, 17, 1, 2)]


@pytest.mark.parametrize("T,E,k,groups,keep,best", CASES)
@pytest.mark.parametrize("sigmoid", [False, True], ids=["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True], ids=["", "bias"])
def test_choice(T, E, k, groups, keep, best, sigmoid, biased):
    rng = np.random.default_rng(T + E)
    lg = (rng.standard_normal((T, E)) * 1.5).astype(F)
    bias = (rng.standard_normal(E) * 0.05).astype(F) if biased else None
    for renorm in (False, True):
        check(lg, k, sigmoid=sigmoid, bias=bias, groups=groups, keep=keep, best=best, renorm=renorm,
              scale=2.5 if renorm else 1.0, pad=E % 3)


@pytest.mark.parametrize("sigmoid", [False, True], ids=["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,keep,best", [(1, 1, 1), (8, 3, 1), (8, 4, 2)])
def test_ties(sigmoid, groups, keep, best):
    rng = np.random.default_rng(groups)
    lg = (rng.integers(-3, 4, (400, 128)) * 0.5).astype(F)
    lg[0] = 0
    check(lg, 8, sigmoid=sigmoid, groups=groups, keep=keep, best=best)
    b = (rng.integers(-2, 3, 128) * 0.25).astype(F)
    check(lg, 8, sigmoid=sigmoid, bias=b, groups=groups, keep=keep, best=best)


@pytest.mark.parametrize("sigmoid", [False, True], ids=["softmax", "sigmoid"])
def test_scores_that_fp32_cannot_tell_apart(sigmoid):
    # logits one ulp apart, under a bias that hides the difference in fp32
    rng = np.random.default_rng(5)
    lg = np.full((64, 64), 0.5, F)
    up = rng.integers(0, 20, lg.shape)
    lg = (lg.view(np.int32) + up.astype(np.int32)).view(F)
    bias = np.full(64, 1.0, F)
    check(lg, 8, sigmoid=sigmoid, bias=bias, groups=8, keep=4, best=2)
    check(lg, 8, sigmoid=sigmoid, bias=bias)
    check(lg, 8, sigmoid=sigmoid, groups=8, keep=4, best=2)


def test_masked_and_extreme_logits():
    big = float(np.finfo(F).max)
    lg = np.zeros((10, 32), F)
    lg[0] = -np.inf  # nothing left: uniform, the lowest experts
    lg[1] = -big
    lg[2, :] = -np.inf
    lg[2, 30] = 1.0  # one expert left
    lg[3, 4] = np.inf
    lg[4, 4], lg[4, 9] = np.inf, np.inf
    lg[5] = np.nan
    lg[6, 3], lg[6, 20] = np.nan, 2.0
    lg[7] = np.linspace(-80, 80, 32)
    lg[8, ::2] = -big
    lg[6, ::2] = np.where(lg[6, ::2] == 0, -0.0, lg[6, ::2])  # zeros of both signs are equal
    lg[9] = -1 - np.arange(32)
    lg[9, :4] = -0.0, 0.0, -3.0, -0.0
    for sigmoid in (False, True):
        for groups, keep, best in ((1, 1, 1), (4, 2, 1), (4, 2, 2)):
            for renorm in (False, True):
                check(lg, 4, sigmoid=sigmoid, groups=groups, keep=keep, best=best, renorm=renorm)
    # sigmoids below fp32's range are renormalised in double
    ids, w = route(np.linspace(-120, -100, 32, dtype=F)[None], 4, sigmoid=True)
    rid, rw = moe.route_grouped(np.linspace(-120, -100, 32, dtype=F)[None], 4, True)
    np.testing.assert_array_equal(ids, rid)
    np.testing.assert_allclose(w, rw, rtol=1e-5)


def test_large_biases_move_the_choice_alone():
    rng = np.random.default_rng(6)
    lg = rng.standard_normal((50, 64)).astype(F)
    b = (rng.standard_normal(64) * 1000).astype(F)
    for sigmoid in (False, True):
        ids, w = check(lg, 6, sigmoid=sigmoid, bias=b, groups=8, keep=4, best=2, renorm=False)
        assert (w <= 1).all()


def test_matches_the_ungrouped_selection():
    rng = np.random.default_rng(7)
    lg = rng.standard_normal((500, 64)).astype(F)
    ids, w = route(lg, 6, renorm=False, scale=1.5)
    d = G.f32(lg)
    i2 = torch.empty(500, 6, dtype=torch.int32, device=G.DEV)
    w2 = torch.empty(500, 6, dtype=torch.float32, device=G.DEV)
    G.check(G.L().b200_moe_topk(d.data_ptr(), 500, 64, 6, 0, 1.5, i2.data_ptr(), w2.data_ptr(), G.stream()))
    np.testing.assert_array_equal(ids, i2.cpu().numpy())
    np.testing.assert_allclose(w, G.host(w2), rtol=1e-5, atol=2e-6)


@pytest.mark.parametrize("T,E,H,pad", [(1, 64, 2048, 0), (5, 7, 64, 8), (200, 60, 512, 16), (130, 252, 1024, 0), (33, 256, 7168, 0),
                                       (129, 255, 264, 0), (700, 256, 520, 8), (300, 8, 4096, 0), (3000, 160, 136, 0)])
def test_route_from_hidden_states(T, E, H, pad):
    """b200_moe_route_grouped: logits within fp32 accumulation of the float64 ones (H terms of two bf16 factors each,
    2^-24 sqrt(H) of their sizes typically, 2^-24 H bounded), then the selection of those very logits."""
    rng = np.random.default_rng(T + E)
    x, wg = G.rounded(rng.standard_normal((T, H))), G.rounded(rng.standard_normal((E, H)) * 0.05)
    groups = 4 if E % 4 == 0 and E >= 8 else 1
    keep, best, k = max(1, groups // 2), 2 if groups > 1 else 1, min(6, max(1, E // 2))
    bias = (rng.standard_normal(E) * 0.05).astype(F)
    X = G.bf16(np.concatenate([x, np.full((T, pad), 1e30)], 1) if pad else x)
    ids = torch.empty(T, k, dtype=torch.int32, device=G.DEV)
    w = torch.empty(T, k, dtype=torch.float32, device=G.DEV)
    lg = torch.full((T + 1, E), 7.0, dtype=torch.float32, device=G.DEV)
    G.check(G.L().b200_moe_route_grouped(X.data_ptr(), H + pad, G.bf16(wg).data_ptr(), G.f32(bias).data_ptr(), T, H, E, k, 1,
                                         groups, keep, best, 1, 2.0, ids.data_ptr(), w.data_ptr(), lg.data_ptr(), G.stream()))
    got = G.host(lg)
    assert (got[T] == 7).all()
    ref = x.astype(np.float64) @ wg.astype(np.float64).T
    size = np.abs(x.astype(np.float64)) @ np.abs(wg.astype(np.float64)).T
    assert (np.abs(got[:T] - ref) <= 2.0**-24 * H * size + 1e-30).all()
    rid, rw = moe.route_grouped(got[:T], k, True, bias, groups, keep, best, True, 2.0)
    np.testing.assert_array_equal(ids.cpu().numpy(), rid)
    np.testing.assert_allclose(G.host(w), rw, rtol=1e-5, atol=4e-6)
    assert G.device_errors() == 0


@pytest.mark.parametrize("sigmoid", [False, True], ids=["softmax", "sigmoid"])
@pytest.mark.parametrize("size", [2.0**14, 2.0**20], ids=["2^14", "2^20"])
@pytest.mark.parametrize("groups", [(0,), (2, 7)], ids=str)
def test_group_scores_whose_terms_cancel(sigmoid, size, groups):
    """Groups of two experts, some biased by +size and -size: such a group's score is of the others' size, but in fp32 it
    carries the rounding of `size` (2^-10 and 2^-4), at whatever rank it comes out and far from the cut too."""
    rng = np.random.default_rng(17)
    lg = rng.standard_normal((400000, 16)).astype(F)
    bias = np.zeros(16, F)
    for g in groups:
        bias[2 * g:2 * g + 2] = size, -size
    check(lg, 8, sigmoid=sigmoid, bias=bias, groups=8, keep=4, best=2)


@pytest.mark.parametrize("T", [8, 64, 300], ids=["warps", "weights on the M side", "weights on the N side"])
def test_gate_weights_written_right_before_the_call(T):
    """A gate merged (base + U V^T) by a GEMM just before on the stream, in place and many times over: each call's logits
    are those of the gate that was merged for it."""
    rng = np.random.default_rng(T)
    E, H, k, R = 256, 2048, 8, 64
    L = G.L()
    X = G.bf16(rng.standard_normal((T, H)))
    U, V = G.bf16(rng.standard_normal((E, R)) * 0.1), G.bf16(rng.standard_normal((H, R)) * 0.1)
    bases = [G.bf16(rng.standard_normal((E, H))) for _ in range(3)]
    gate = torch.zeros(E, H, dtype=torch.bfloat16, device=G.DEV)
    out = lambda: (torch.empty(T, k, dtype=torch.int32, device=G.DEV), torch.empty(T, k, device=G.DEV),  # noqa: E731
                   torch.empty(T, E, device=G.DEV))

    def merge(base):
        G.check(L.b200_gemm_bf16(U.data_ptr(), R, V.data_ptr(), R, gate.data_ptr(), H, E, H, R, 2, None, base.data_ptr(), H,
                                 None, 0, G.stream()))

    def route_to(o):
        G.check(L.b200_moe_route_grouped(X.data_ptr(), H, gate.data_ptr(), None, T, H, E, k, 0, 1, 1, 1, 1, 1.0,
                                         o[0].data_ptr(), o[1].data_ptr(), o[2].data_ptr(), G.stream()))

    want = []
    for base in bases:
        merge(base)
        torch.cuda.synchronize()
        want.append(out())
        route_to(want[-1])
        torch.cuda.synchronize()
    assert not any(torch.equal(want[0][2], w[2]) for w in want[1:])
    got = [out() for _ in range(60)]
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        merge(bases[i % 3])
        route_to(o)
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        for a, b in zip(o, want[i % 3]):
            assert torch.equal(a, b), i
    assert G.device_errors() == 0
