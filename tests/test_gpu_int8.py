"""GPU parity of the 8-bit linear layers through the C ABI: row quantisation
(bit-exact), its fused RMSNorm form (bit-exact against the two calls), the
8-bit products, plain and grouped, against float64, and a routed expert MLP
run through all of them.

Tolerances.  The integer sums are exact, so a product carries: the conversion
of the sum to fp32, two scale products, and the bias / residual additions (at
most 6 roundings of 2^-24 of the terms), then one rounding to bf16 (2^-8 of the
value).  SwiGLU's and GELU's exponential is the fast one: (2 + 1.2 |w|) 2^-23
relative for e^-w, 1.3e-5 for |w| <= 90, below which the value vanishes, and
the division is within 2 ulp.  GELU's w = 2 sqrt(2/pi) (x + 0.044715 x^3) adds
its own roundings, which the cases here keep small (|w| of a few units; far
values have a test and a bound of their own).  So |out - ref| <= 2^-8 |ref| +
2e-5 (|ref| + |terms|) for all of them.
"""

import os
import subprocess
import sys
import textwrap

import numpy as np
import pytest
import torch

from oracle import int8, moe

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import gpu_util as G

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F = np.float32
NONE, BIAS, RESIDUAL, SWIGLU, BIAS_GELU, BIAS_RESIDUAL = range(6)


def i8(a):
    return G._keep(torch.from_numpy(np.ascontiguousarray(np.asarray(a, np.int8))).to(G.DEV))


def all_bf16_up_to(top_bits):
    """Every non-negative bf16 value up to the one with these bits, as float32."""
    return (np.arange(top_bits + 1, dtype=np.uint32) << 16).view(F)


def quant(x, ldx=None, ldq=None, src=None, count=None, rows=None):
    """b200_quant_rows_int8 of a bf16 device tensor's first columns."""
    n, dim = x.shape
    rows = rows if rows is not None else (len(src) if src is not None else n)
    ldq = ldq or dim
    q = torch.full((rows, ldq), 99, dtype=torch.int8, device=G.DEV)
    s = torch.full((rows,), 77.0, dtype=torch.float32, device=G.DEV)
    G.check(G.L().b200_quant_rows_int8(x.data_ptr(), ldx or x.stride(0), n, G.ptr(None if src is None else G.i32(src)),
                                       G.ptr(None if count is None else G.i32([count])), q.data_ptr(), ldq, s.data_ptr(),
                                       rows, dim, G.stream()), "quant_rows_int8")
    torch.cuda.synchronize()
    return q.cpu().numpy(), G.host(s)


# ------------------------------------------------------------ quantisation


@pytest.mark.parametrize("rows,dim", [(1, 16), (3, 48), (777, 1408), (64, 2048), (5, 2064), (33, 4096), (2, 8208), (7, 14336),
                                      (2, 16384), (3, 16400), (2, 131056)])
def test_quant_rows(rows, dim):
    rng = np.random.default_rng(dim)
    x = G.rounded(rng.standard_normal((rows, dim)).astype(F) * np.exp2(rng.integers(-20, 20, (rows, 1))).astype(F))
    q, s = quant(G.bf16(x))
    rq, rs = int8.quant_rows(x)
    np.testing.assert_array_equal(q, rq)
    np.testing.assert_array_equal(s, rs)


@pytest.mark.parametrize("top", [0x0001, 0x0002, 0x0003, 0x007f, 0x0080, 0x00ff, 0x0d80, 0x0dff, 0x0e00, 0x3f7f, 0x3f80,
                                 0x3f81, 0x3faa, 0x3ffd, 0x4213, 0x7180, 0x71ff, 0x7200, 0x7f00, 0x7f7e, 0x7f7f],
                         ids=hex)
def test_quant_every_value_below_a_maximum(top):
    # ties, subnormals and both ends of the range: every bf16 magnitude up to the row's largest, both signs
    v = all_bf16_up_to(top)
    dim = -(-len(v) // 16) * 16
    x = np.zeros((2, dim), F)
    x[0, :len(v)] = v
    x[1, :len(v)] = -v
    q, s = quant(G.bf16(x))
    rq, rs = int8.quant_rows(x)
    np.testing.assert_array_equal(q, rq)
    np.testing.assert_array_equal(s, rs)


def test_quant_empty_and_non_finite_rows():
    x = np.ones((6, 64), F)
    x[1] = 0
    x[2, 5] = np.inf
    x[3, 63] = -np.inf
    x[4, 0] = np.nan
    x[5, 7] = -0.0
    q, s = quant(G.bf16(x))
    rq, rs = int8.quant_rows(x)
    np.testing.assert_array_equal(q, rq)
    np.testing.assert_array_equal(s, rs)
    assert s[1] == 0 and np.isnan(s[2:5]).all() and not q[1:5].any()


def test_quant_strides_gather_and_count():
    rng = np.random.default_rng(1)
    wide = G.bf16(rng.standard_normal((40, 112)).astype(F))
    x = wide[:, 16:80]  # 64 columns of 112-wide rows
    rx = G.host(x)
    q, s = quant(x, ldx=112, ldq=96)
    rq, rs = int8.quant_rows(rx)
    np.testing.assert_array_equal(q[:, :64], rq)
    assert (q[:, 64:] == 99).all()  # what lies between the rows is left alone
    np.testing.assert_array_equal(s, rs)
    src = rng.integers(0, 40, 101)
    q, s = quant(x, ldx=112, src=src, count=90)
    np.testing.assert_array_equal(q[:90], rq[src[:90]])
    np.testing.assert_array_equal(s[:90], rs[src[:90]])
    assert (q[90:] == 99).all() and (s[90:] == 77).all()
    assert G.device_errors() == 0
    src[[3, 50]] = [40, -1]  # out of range: reported, their rows left alone
    q, s = quant(x, ldx=112, src=src)
    ok = np.ones(101, bool)
    ok[[3, 50]] = False
    np.testing.assert_array_equal(q[ok], rq[src[ok]])
    assert (q[~ok] == 99).all() and (s[~ok] == 77).all()
    assert G.device_errors() == 2


@pytest.mark.parametrize("rows,dim,stride", [(1, 16, 16), (64, 4096, 4096), (333, 1408, 1424), (3, 2064, 2064), (5, 8192, 8192)])
@pytest.mark.parametrize("residual", [False, True])
def test_rmsnorm_quant_is_the_two_calls(rows, dim, stride, residual):
    rng = np.random.default_rng(rows + dim)
    L = G.L()
    x = G.bf16(rng.standard_normal((rows, stride)).astype(F) * 3)
    x[rows // 2] = 0  # a row of zeros
    r = G.bf16(rng.standard_normal((rows, stride)).astype(F)) if residual else None
    if residual:
        r[rows // 2] = 0
    w = G.bf16(1 + 0.1 * rng.standard_normal(dim).astype(F))
    out, ro, out2, ro2 = (torch.zeros(rows, stride, dtype=torch.bfloat16, device=G.DEV) for _ in range(4))
    q = torch.zeros(rows, dim, dtype=torch.int8, device=G.DEV)
    s = torch.zeros(rows, dtype=torch.float32, device=G.DEV)
    G.check(L.b200_rmsnorm(x.data_ptr(), G.ptr(r), w.data_ptr(), out.data_ptr(), ro.data_ptr() if residual else None, rows,
                           dim, stride, 1e-6, G.stream()))
    for with_out in (True, False):
        q.fill_(99)
        G.check(L.b200_rmsnorm_quant_int8(x.data_ptr(), G.ptr(r), w.data_ptr(), q.data_ptr(), dim, s.data_ptr(),
                                          out2.data_ptr() if with_out else None, ro2.data_ptr() if residual else None, rows,
                                          dim, stride, 1e-6, G.stream()))
        torch.cuda.synchronize()
        rq, rs = int8.quant_rows(G.host(out)[:, :dim])
        np.testing.assert_array_equal(q.cpu().numpy(), rq)
        np.testing.assert_array_equal(G.host(s), rs)
        if residual:
            np.testing.assert_array_equal(G.host(ro2), G.host(ro))
    np.testing.assert_array_equal(G.host(out2), G.host(out))
    if residual:  # the sum written over the residual
        G.check(L.b200_rmsnorm_quant_int8(x.data_ptr(), r.data_ptr(), w.data_ptr(), q.data_ptr(), dim, s.data_ptr(), None,
                                          r.data_ptr(), rows, dim, stride, 1e-6, G.stream()))
        torch.cuda.synchronize()
        np.testing.assert_array_equal(G.host(r)[:, :dim], G.host(ro)[:, :dim])
        np.testing.assert_array_equal(q.cpu().numpy(), rq)


# ----------------------------------------------------------------- products


def near(out, ref, terms=0.0):
    """The bound of the module's docstring; NaN where the reference is NaN."""
    out, ref = np.asarray(out, np.float64), np.asarray(ref, np.float64)
    bad = np.isnan(ref)
    assert (np.isnan(out) == bad).all()
    err = np.abs(out - ref)
    lim = 2.0**-8 * np.abs(ref) + 2e-5 * (np.abs(ref) + terms) + 1e-30
    worst = np.where(bad, 0, err - lim)
    assert (worst <= 0).all(), (float(worst.max()), np.unravel_index(worst.argmax(), worst.shape))


def operands(rng, M, N, K, epi, full=False):
    a = rng.integers(-128 if full else -127, 128, (M, K)).astype(np.int8)
    b = rng.integers(-128 if full else -127, 128, (N, K)).astype(np.int8)
    unit = 1.0 / (73 * np.sqrt(K))  # products of about one standard deviation
    sa = (rng.uniform(0.5, 2, M) * unit).astype(F)
    sb = (rng.uniform(0.5, 2, N) / 73 * 40).astype(F)
    bias = G.rounded(rng.standard_normal(N)) if epi in (BIAS, BIAS_GELU, BIAS_RESIDUAL) else None
    res = G.rounded(rng.standard_normal((M, N))) if epi in (RESIDUAL, BIAS_RESIDUAL) else None
    return a, sa, b, sb, bias, res


def gemm(a, sa, b, sb, epi, bias=None, res=None, pad=0, out=None, inplace=False):
    """b200_gemm_int8 on numpy operands; pad: extra columns in every row stride."""
    M, K = a.shape
    N = b.shape[0]
    outN = N // 2 if epi == SWIGLU else N
    wide = lambda m, fill: np.concatenate([m, np.full((len(m), pad), fill, m.dtype)], 1)  # noqa: E731
    A, B = i8(wide(a, 55)), i8(wide(b, -77))
    R = G.bf16(wide(np.asarray(res, F), 1e30)) if res is not None else None
    C = R if inplace else torch.full((M, outN + pad), 7.0, dtype=torch.bfloat16, device=G.DEV)
    G.check(G.L().b200_gemm_int8(A.data_ptr(), K + pad, G.f32(sa).data_ptr(), B.data_ptr(), K + pad, G.f32(sb).data_ptr(),
                                 C.data_ptr(), outN + pad, M, N, K, epi, G.ptr(None if bias is None else G.bf16(bias)),
                                 G.ptr(R), N + pad, G.stream()), "gemm_int8")
    torch.cuda.synchronize()
    assert G.device_errors() == 0
    h = G.host(C)
    if pad and not inplace:
        assert (h[:, outN:] == 7).all()
    return h[:, :outN]


SHAPES = [(1, 8, 16), (1, 4096, 4096), (2, 136, 144), (8, 256, 48), (15, 520, 1040), (16, 128, 128), (17, 264, 272),
          (32, 6144, 512), (33, 1032, 2064), (64, 512, 4096), (65, 2056, 128), (96, 24, 4112), (128, 640, 1408),
          (129, 128, 256), (130, 136, 272), (200, 1408, 2048), (257, 264, 1040), (300, 8, 16), (512, 4096, 1024),
          (777, 520, 1040), (1025, 1288, 400), (2049, 2568, 144), (2300, 2312, 1040), (257, 20000, 272), (5000, 1160, 4112)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gemm_shapes(M, N, K):
    rng = np.random.default_rng(M * 7 + N + K)
    a, sa, b, sb, _, _ = operands(rng, M, N, K, NONE)
    near(gemm(a, sa, b, sb, NONE), int8.gemm(a, sa, b, sb))


@pytest.mark.parametrize("epi", range(6))
@pytest.mark.parametrize("M,N,K", [(1, 144, 272), (20, 528, 1040), (50, 272, 4112), (128, 1040, 512), (131, 144, 272),
                                   (700, 1296, 528), (2100, 2576, 400)])
def test_gemm_epilogues(M, N, K, epi):
    rng = np.random.default_rng(M + epi)
    a, sa, b, sb, bias, res = operands(rng, M, N, K, epi)
    ref = int8.gemm(a, sa, b, sb, epi, bias, res)
    out = gemm(a, sa, b, sb, epi, bias, res, pad=16)
    if epi == SWIGLU:
        v = int8.gemm(a, sa, b, sb)
        near(out, ref, 0.0 * v[:, ::2])
    else:
        terms = np.abs(int8.gemm(a, sa, b, sb)) + (0 if bias is None else np.abs(bias)) + (0 if res is None else np.abs(res))
        near(out, ref, terms)
    if epi == RESIDUAL:  # the residual stream updated in place
        near(gemm(a, sa, b, sb, epi, bias, res, pad=16, inplace=True), ref, terms)


@pytest.mark.parametrize("M,K", [(3, 131056), (140, 131056)])
def test_gemm_longest_sums_of_extremes(M, K):
    # -128 * -128 over the longest K: 2^31 - 2^18, exact in 32 bits
    a, b = np.full((M, K), -128, np.int8), np.full((16, K), -128, np.int8)
    b[1::2] = 127
    sa, sb = np.full(M, 2.0**-20, F), np.full(16, 1.0, F)
    near(gemm(a, sa, b, sb, NONE), int8.gemm(a, sa, b, sb))


@pytest.mark.parametrize("M", [5, 64, 150])
def test_gemm_integers_are_exact(M):
    # sums small enough for bf16 come back as themselves, so every partial product is in its place
    rng = np.random.default_rng(M)
    N, K = 264, 2064
    a, b = np.zeros((M, K), np.int8), np.zeros((N, K), np.int8)
    a[np.arange(M), rng.permutation(K)[:M]] = rng.integers(-8, 9, M)
    b[:] = rng.integers(-8, 9, (N, K))
    out = gemm(a, np.ones(M, F), b, np.ones(N, F), NONE)
    np.testing.assert_array_equal(out, a.astype(np.int64) @ b.astype(np.int64).T)


def test_gemm_non_finite_scales_stay_in_their_rows():
    rng = np.random.default_rng(9)
    for M, N in ((6, 272), (200, 272), (6100, 528)):
        for epi in (NONE, SWIGLU):
            a, sa, b, sb, _, _ = operands(rng, M, N, 528, epi)
            sa[3] = np.nan
            a[3] = 0
            sa[4] = 0
            near(gemm(a, sa, b, sb, epi), int8.gemm(a, sa, b, sb, epi))


def test_gemm_swiglu_of_large_gates():
    rng = np.random.default_rng(10)
    for M, N in ((6, 272), (200, 272), (6100, 528)):
        a, sa, b, sb, _, _ = operands(rng, M, N, 528, SWIGLU)
        out = gemm(a, sa * 200, b, sb, SWIGLU)
        assert np.isfinite(out).all()
        ref = int8.gemm(a, sa * 200, b, sb, SWIGLU)
        gate = int8.gemm(a, sa * 200, b, sb)[:, ::2]
        seen = gate > -80  # below, the gate's e^g leaves the fast division's range: less than 1e-30 of the up value
        near(np.where(seen, out, 0), np.where(seen, ref, 0))
        assert np.abs(np.where(seen, 0, out)).max() < 1e-25


def test_gemm_same_bits_twice_and_on_two_streams():
    rng = np.random.default_rng(11)
    for M, N, K in [(8, 4096, 4096), (300, 1024, 2048)]:
        a, sa, b, sb, _, _ = operands(rng, M, N, K, NONE)
        want = gemm(a, sa, b, sb, NONE)
        A, B, SA, SB = i8(a), i8(b), G.f32(sa), G.f32(sb)
        outs = [torch.zeros(M, N, dtype=torch.bfloat16, device=G.DEV) for _ in range(6)]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for i, o in enumerate(outs):
            G.check(G.L().b200_gemm_int8(A.data_ptr(), K, SA.data_ptr(), B.data_ptr(), K, SB.data_ptr(), o.data_ptr(), N, M,
                                         N, K, NONE, None, None, 0, streams[i % 2].cuda_stream))
        torch.cuda.synchronize()
        for o in outs:
            np.testing.assert_array_equal(G.host(o), want)


@pytest.mark.parametrize("epi", [NONE, RESIDUAL, SWIGLU, BIAS_GELU])
def test_gemm_rows_aligned_to_16_bytes_only(epi):
    # the widest stores want 32-byte rows: an odd start and an odd stride of 8 elements each
    rng = np.random.default_rng(13 + epi)
    M, N, K = 6100, 528, 272
    a, sa, b, sb, bias, res = operands(rng, M, N, K, epi)
    outN = N // 2 if epi == SWIGLU else N
    ref = int8.gemm(a, sa, b, sb, epi, bias, res)
    terms = np.abs(int8.gemm(a, sa, b, sb)).max() + 4 if epi in (RESIDUAL, BIAS_GELU) else 0.0
    for start, pad in ((8, 0), (0, 8), (8, 24)):
        C = torch.full((M * (outN + pad) + 16,), 7.0, dtype=torch.bfloat16, device=G.DEV)
        R = G.bf16(np.concatenate([np.zeros(start), np.concatenate([res, np.zeros((M, pad))], 1).ravel()])) if res is not None else None
        G.check(G.L().b200_gemm_int8(i8(a).data_ptr(), K, G.f32(sa).data_ptr(), i8(b).data_ptr(), K, G.f32(sb).data_ptr(),
                                     C.data_ptr() + 2 * start, outN + pad, M, N, K, epi,
                                     G.ptr(None if bias is None else G.bf16(bias)), 0 if R is None else R.data_ptr() + 2 * start,
                                     N + pad, G.stream()))
        torch.cuda.synchronize()
        h = G.host(C)
        assert (h[:start] == 7).all() and (h[start + M * (outN + pad):] == 7).all()
        h = h[start:start + M * (outN + pad)].reshape(M, outN + pad)
        assert (h[:, outN:] == 7).all()
        near(h[:, :outN], ref, terms)


def test_offsets_past_32_bits():
    """More than 2^31 elements in x, q and C: the last rows are quantised, read and written where they belong."""
    M, K, N = 70001, 32768, 32776
    g = torch.Generator(device=G.DEV)
    g.manual_seed(3)
    last = [0, 1, 65535, 65536, M - 2, M - 1]
    x = torch.zeros(M, K, dtype=torch.bfloat16, device=G.DEV)
    x[last] = torch.randn(len(last), K, generator=g, device=G.DEV).bfloat16()
    q = torch.full((M, K), 99, dtype=torch.int8, device=G.DEV)
    s = torch.full((M,), 7.0, device=G.DEV)
    L = G.L()
    G.check(L.b200_quant_rows_int8(x.data_ptr(), K, M, None, None, q.data_ptr(), K, s.data_ptr(), M, K, G.stream()))
    rq, rs = int8.quant_rows(G.host(x[last]))
    np.testing.assert_array_equal(q[last].cpu().numpy(), rq)
    np.testing.assert_array_equal(G.host(s[last]), rs)
    assert int(q[2:65535].abs().max()) == 0
    del x
    b = torch.randint(-127, 128, (264, K), generator=g, device=G.DEV).to(torch.int8)
    sb = torch.rand(264, generator=g, device=G.DEV) + 0.5
    C = torch.full((M, 264), 7.0, dtype=torch.bfloat16, device=G.DEV)
    G.check(L.b200_gemm_int8(q.data_ptr(), K, s.data_ptr(), b.data_ptr(), K, sb.data_ptr(), C.data_ptr(), 264, M, 264, K,
                             NONE, None, None, 0, G.stream()))
    near(G.host(C[last]), int8.gemm(rq, rs, b.cpu().numpy(), G.host(sb)))
    assert float(C[2:65535].abs().max()) == 0
    del C
    b = torch.randint(-127, 128, (N, 32), generator=g, device=G.DEV).to(torch.int8)
    sb = torch.rand(N, generator=g, device=G.DEV) + 0.5
    q[:, :32] = torch.randint(-127, 128, (M, 32), generator=g, device=G.DEV).to(torch.int8)
    s = torch.rand(M, generator=g, device=G.DEV) + 0.5
    C = torch.full((M, N), 7.0, dtype=torch.bfloat16, device=G.DEV)
    G.check(L.b200_gemm_int8(q.data_ptr(), K, s.data_ptr(), b.data_ptr(), 32, sb.data_ptr(), C.data_ptr(), N, M, N, 32,
                             NONE, None, None, 0, G.stream()))
    near(G.host(C[last]), int8.gemm(q[last][:, :32].cpu().numpy(), G.host(s[last]), b.cpu().numpy(), G.host(sb)))
    assert G.device_errors() == 0


def test_forms_side_by_side_on_streams():
    """The pair, split and grouped forms and the bf16 GEMM running at once on four streams give what they give alone."""
    rng = np.random.default_rng(14)
    L = G.L()
    jobs = []

    def plain(M, N, K):
        a, sa, b, sb, _, _ = operands(rng, M, N, K, NONE)
        A, B, SA, SB = i8(a), i8(b), G.f32(sa), G.f32(sb)
        return lambda st, o: G.check(L.b200_gemm_int8(A.data_ptr(), K, SA.data_ptr(), B.data_ptr(), K, SB.data_ptr(),
                                                      o.data_ptr(), N, M, N, K, NONE, None, None, 0, st)), (M, N)

    def experts(rows, n, N, K):
        a, sa, b, sb, _, _ = operands(rng, rows, n * N, K, NONE)
        A, B, SA, SB = i8(a), i8(b), G.f32(sa), G.f32(sb)
        off = G.i32(np.linspace(0, rows, n + 1).astype(np.int32))
        return lambda st, o: G.check(L.b200_grouped_gemm_int8(A.data_ptr(), K, SA.data_ptr(), B.data_ptr(), K, SB.data_ptr(),
                                                              o.data_ptr(), N, off.data_ptr(), n, rows, N, K, NONE, st)), (rows, N)

    X, W = G.bf16(rng.standard_normal((300, 1024))), G.bf16(rng.standard_normal((2048, 1024)))
    bf = lambda st, o: G.check(L.b200_gemm_bf16(X.data_ptr(), 1024, W.data_ptr(), 1024, o.data_ptr(), 2048, 300, 2048, 1024,  # noqa: E731
                                                NONE, None, None, 0, None, 0, st))
    jobs = [plain(2048, 2048, 2048), plain(16, 4096, 4096), experts(900, 8, 512, 1024), (bf, (300, 2048)), plain(100, 1024, 4096),
            experts(24, 8, 1024, 1024), experts(4000, 8, 512, 512)]
    new = lambda shape: torch.zeros(*shape, dtype=torch.bfloat16, device=G.DEV)  # noqa: E731
    alone = []
    for f, shape in jobs:
        o = new(shape)
        f(G.stream(), o)
        torch.cuda.synchronize()
        alone.append(G.host(o))
    streams = [torch.cuda.Stream() for _ in range(4)]
    outs = [(i, new(shape)) for r in range(8) for i, (_, shape) in enumerate(jobs)]
    torch.cuda.synchronize()
    for n, (i, o) in enumerate(outs):
        jobs[i][0](streams[(n * 3 + n // 7) % 4].cuda_stream, o)
    torch.cuda.synchronize()
    for i, o in outs:
        np.testing.assert_array_equal(G.host(o), alone[i])
    assert G.device_errors() == 0


def test_first_calls_of_a_process_under_capture():
    code = textwrap.dedent("""
        import sys; sys.path[:0] = [%r, %r]
        import torch
        from atb_llm_study_b200 import capi
        L = capi.lib()
        one = lambda *s, t: torch.ones(*s, device="cuda").to(t)
        x, w = one(8, 512, t=torch.bfloat16), one(256, 512, t=torch.int8)
        q, s, ws = one(8, 512, t=torch.int8), one(8, t=torch.float32), one(256, t=torch.float32)
        out, lg = one(8, 256, t=torch.bfloat16), one(8, 64, t=torch.float32)
        ids, wt = one(8, 4, t=torch.int32), one(8, 4, t=torch.float32)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            st = torch.cuda.current_stream().cuda_stream
            capi.check(L.b200_quant_rows_int8(x.data_ptr(), 512, 8, None, None, q.data_ptr(), 512, s.data_ptr(), 8, 512, st))
            capi.check(L.b200_gemm_int8(q.data_ptr(), 512, s.data_ptr(), w.data_ptr(), 512, ws.data_ptr(), out.data_ptr(), 256,
                                        8, 256, 512, 0, None, None, 0, st))
            capi.check(L.b200_moe_topk_grouped(lg.data_ptr(), 64, None, 8, 64, 4, 0, 8, 2, 1, 1, 1.0, ids.data_ptr(),
                                               wt.data_ptr(), st))
        out.zero_(); ids.zero_()
        g.replay(); torch.cuda.synchronize()
        assert (out == 512).all(), out
        assert ids.tolist() == [[0, 1, 2, 3]] * 8, ids
    """ % (ROOT, os.path.join(ROOT, "tests")))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


# ------------------------------------------------------------ grouped product


def grouped(a, sa, b, sb, sizes, N, epi, extra=0):
    K = a.shape[1]
    off = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    rows = int(off[-1]) + extra
    outN = N // 2 if epi == SWIGLU else N
    pad = np.zeros((rows - len(a), K), np.int8)
    C = torch.full((rows, outN), 7.0, dtype=torch.bfloat16, device=G.DEV)
    SA = G.f32(np.concatenate([sa, np.ones(rows - len(sa), F)]))
    G.check(G.L().b200_grouped_gemm_int8(i8(np.concatenate([a, pad])).data_ptr(), K, SA.data_ptr(), i8(b).data_ptr(), K,
                                         G.f32(sb).data_ptr(), C.data_ptr(), outN, G.i32(off).data_ptr(), len(sizes), rows,
                                         N, K, epi, G.stream()), "grouped_gemm_int8")
    torch.cuda.synchronize()
    assert G.device_errors() == 0
    h = G.host(C)
    assert (h[off[-1]:] == 7).all()  # rows behind the last group stay as they were
    return h[:off[-1]], off


GROUPS = [
    ([3, 0, 17, 64, 1, 0, 100, 7], 256, 512), ([3, 0, 17, 64, 1, 0, 100, 7], 208, 528), ([1], 128, 128), ([0, 1, 0], 24, 16),
    ([2] * 64, 176, 256), ([0, 0, 0, 40], 128, 144), ([300, 0, 513, 129], 512, 256), ([300, 0, 513, 129], 144, 272),
    ([128, 256, 1, 700], 1296, 144), ([0, 0, 900], 2816, 400), ([97] * 5, 272, 1040), ([5, 700, 3, 0, 2, 1], 544, 256),
    ([0] * 40 + [9], 144, 272), ([1000] + [0] * 255, 48, 48), ([700] + [1] * 63, 144, 272),
    ([300, 0, 513, 129], 520, 272), ([100, 60, 0, 130], 520, 272)]


@pytest.mark.parametrize("epi", [NONE, SWIGLU])
@pytest.mark.parametrize("sizes,N,K", GROUPS, ids=[str(i) for i in range(len(GROUPS))])
def test_grouped_gemm(sizes, N, K, epi):
    if epi == SWIGLU:
        N = -(-N // 16) * 16  # gate / up pairs of 8 (others are refused, tests/test_int8_cpu.py)
    rng = np.random.default_rng(sum(sizes) + N + epi)
    rows, n = int(sum(sizes)), len(sizes)
    a, sa, b, sb, _, _ = operands(rng, rows, n * N, K, epi)
    out, off = grouped(a, sa, b, sb, sizes, N, epi, extra=37)
    for g in range(n):
        r, w = slice(off[g], off[g + 1]), slice(g * N, (g + 1) * N)
        near(out[r], int8.gemm(a[r], sa[r], b[w], sb[w], epi))


def test_grouped_gemm_without_rows_and_with_bad_offsets():
    rng = np.random.default_rng(4)
    a, sa, b, sb, _, _ = operands(rng, 20, 3 * 128, 256, NONE)
    L = G.L()

    def call(off, rows=20):
        C = torch.full((20, 128), 7.0, dtype=torch.bfloat16, device=G.DEV)
        G.check(L.b200_grouped_gemm_int8(i8(a).data_ptr(), 256, G.f32(sa).data_ptr(), i8(b).data_ptr(), 256,
                                         G.f32(sb).data_ptr(), C.data_ptr(), 128, G.i32(off).data_ptr(), 3, rows, 128, 256,
                                         NONE, G.stream()))
        torch.cuda.synchronize()
        return G.host(C), G.device_errors()

    out, err = call([0, 0, 0, 0])
    assert (out == 7).all() and err == 0
    for off in ([0, 10, 5, 20], [0, 10, 15, 30], [-3, 5, 10, 20], [4, 5, 10, 20]):
        assert call(off)[1] == 2, off


# ----------------------------------------------------------- used together


@pytest.mark.parametrize("T,E,k,H,I,groups", [(1, 8, 2, 256, 272, 1), (33, 64, 6, 512, 176, 8), (700, 16, 4, 272, 144, 4)])
def test_routed_experts(T, E, k, H, I, groups):
    """Router selection -> permutation -> gather + quantise -> gate/up -> quantise -> down -> combine, each stage
    against float64 on its own inputs, and the same bits from a captured graph and from two graphs replayed in turn."""
    rng = np.random.default_rng(T)
    L = G.L()
    R = T * k
    x = G.rounded(rng.standard_normal((T, H)))
    lg = (rng.standard_normal((T, E)) * 1.5).astype(F)
    b1, sb1 = rng.integers(-127, 128, (E * 2 * I, H)).astype(np.int8), rng.uniform(1, 3, E * 2 * I).astype(F) * 3e-4
    b2, sb2 = rng.integers(-127, 128, (E * H, I)).astype(np.int8), rng.uniform(1, 3, E * H).astype(F) * 3e-4
    X, LG, B1, S1, B2, S2 = G.bf16(x), G.f32(lg), i8(b1), G.f32(sb1), i8(b2), G.f32(sb2)
    new = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device=G.DEV)  # noqa: E731

    def buffers():
        return dict(ids=new(T, k, t=torch.int32), w=new(T, k, t=torch.float32), off=new(E + 1, t=torch.int32),
                    pos=new(R, t=torch.int32), src=new(R, t=torch.int32),
                    ws=new(max(16, L.b200_moe_permute_workspace_bytes(T, k, E)), t=torch.uint8), q1=new(R, H, t=torch.int8),
                    s1=new(R, t=torch.float32), act=new(R, I), q2=new(R, I, t=torch.int8), s2=new(R, t=torch.float32),
                    y=new(R, H), out=new(T, H))

    def run(d, st):
        p = {n: t.data_ptr() for n, t in d.items()}
        G.check(L.b200_moe_topk_grouped(LG.data_ptr(), E, None, T, E, k, 1, groups, max(1, groups // 2),
                                        2 if groups > 1 else 1, 1, 1.0, p["ids"], p["w"], st))
        G.check(L.b200_moe_permute(p["ids"], T, k, E, None, 0, 0, None, p["off"], p["pos"], p["src"], p["ws"],
                                   d["ws"].numel(), st))
        total = p["off"] + 4 * E
        G.check(L.b200_quant_rows_int8(X.data_ptr(), H, T, p["src"], total, p["q1"], H, p["s1"], R, H, st))
        G.check(L.b200_grouped_gemm_int8(p["q1"], H, p["s1"], B1.data_ptr(), H, S1.data_ptr(), p["act"], I, p["off"], E, R,
                                         2 * I, H, SWIGLU, st))
        G.check(L.b200_quant_rows_int8(p["act"], I, R, None, total, p["q2"], I, p["s2"], R, I, st))
        G.check(L.b200_grouped_gemm_int8(p["q2"], I, p["s2"], B2.data_ptr(), I, S2.data_ptr(), p["y"], H, p["off"], E, R, H,
                                         I, NONE, st))
        G.check(L.b200_moe_combine(p["y"], p["pos"], p["w"], T, k, H, X.data_ptr(), None, p["out"], None, None, 1e-6, st))

    d = buffers()
    run(d, G.stream())
    torch.cuda.synchronize()
    assert G.device_errors() == 0
    ids, w = moe.route_grouped(lg, k, True, None, groups, max(1, groups // 2), 2 if groups > 1 else 1)
    np.testing.assert_array_equal(d["ids"].cpu().numpy(), ids)
    off, pos, src = moe.permute(ids, E)
    np.testing.assert_array_equal(d["src"].cpu().numpy(), src)
    q1, s1 = int8.quant_rows(x[src])
    np.testing.assert_array_equal(d["q1"].cpu().numpy(), q1)
    act, y = G.host(d["act"]), G.host(d["y"])
    q2, s2 = int8.quant_rows(act)
    np.testing.assert_array_equal(d["q2"].cpu().numpy(), q2)
    np.testing.assert_array_equal(G.host(d["s2"]), s2)
    for e in range(E):
        r = slice(off[e], off[e + 1])
        up, down = slice(e * 2 * I, (e + 1) * 2 * I), slice(e * H, (e + 1) * H)
        near(act[r], int8.gemm(q1[r], s1[r], b1[up], sb1[up], SWIGLU))
        near(y[r], int8.gemm(q2[r], s2[r], b2[down], sb2[down]))
    routed = (y[pos].reshape(T, k, H) * w[:, :, None]).sum(1)
    # fp32 sums of k + 1 terms and fp32 weights, one rounding to bf16
    near(G.host(d["out"]), x + routed, 2 * np.abs(y[pos]).reshape(T, k, H).max(1))

    # captured, with the weights shared and the buffers each graph's own
    graphs = []
    for _ in range(2):
        g, b = torch.cuda.CUDAGraph(), buffers()
        st = torch.cuda.Stream()
        with torch.cuda.graph(g, stream=st):
            run(b, torch.cuda.current_stream().cuda_stream)
        graphs.append((g, b))
    for _ in range(3):
        for g, _b in graphs:
            g.replay()
    torch.cuda.synchronize()
    for _g, b in graphs:
        np.testing.assert_array_equal(G.host(b["out"]), G.host(d["out"]))
    assert G.device_errors() == 0


def test_weights_quantised_right_before_the_product():
    """The product's weights made by the kernels just before it, back to back on one stream, many times over."""
    rng = np.random.default_rng(12)
    M, N, K = 16, 2048, 4096
    L = G.L()
    x = G.bf16(rng.standard_normal((M, K)).astype(F))
    q, s = torch.zeros(M, K, dtype=torch.int8, device=G.DEV), torch.zeros(M, dtype=torch.float32, device=G.DEV)
    wq, ws = torch.zeros(N, K, dtype=torch.int8, device=G.DEV), torch.zeros(N, dtype=torch.float32, device=G.DEV)
    weights = [G.bf16(rng.standard_normal((N, K)).astype(F)) for _ in range(3)]
    outs = [torch.zeros(M, N, dtype=torch.bfloat16, device=G.DEV) for _ in range(30)]
    for i, o in enumerate(outs):
        w = weights[i % 3]
        if i % 2:
            G.check(L.b200_quant_rows_int8(w.data_ptr(), K, N, None, None, wq.data_ptr(), K, ws.data_ptr(), N, K, G.stream()))
            G.check(L.b200_quant_rows_int8(x.data_ptr(), K, M, None, None, q.data_ptr(), K, s.data_ptr(), M, K, G.stream()))
        else:
            G.check(L.b200_quant_rows_int8(x.data_ptr(), K, M, None, None, q.data_ptr(), K, s.data_ptr(), M, K, G.stream()))
            G.check(L.b200_quant_rows_int8(w.data_ptr(), K, N, None, None, wq.data_ptr(), K, ws.data_ptr(), N, K, G.stream()))
        G.check(L.b200_gemm_int8(q.data_ptr(), K, s.data_ptr(), wq.data_ptr(), K, ws.data_ptr(), o.data_ptr(), N, M, N, K,
                                 NONE, None, None, 0, G.stream()))
    torch.cuda.synchronize()
    qa, sa = int8.quant_rows(G.host(x))
    for i in range(3):
        qb, sb = int8.quant_rows(G.host(weights[i]))
        near(G.host(outs[i]), int8.gemm(qa, sa, qb, sb))
        for j in range(i, 30, 3):
            np.testing.assert_array_equal(G.host(outs[j]), G.host(outs[i]))


# ------------------------------------- grouped products of many tiles a worker

# Sizes of 64 groups and the form that their average takes (tokens a tile, features a tile, workers: CTAs or pairs).
MANY_TILES = {
    "16 tokens": ([1, 3, 9, 0, 17, 2, 15, 16], 16, 128, 148),
    "32 tokens": ([20, 1, 33, 0, 5, 32, 7, 8], 32, 128, 148),
    "64 tokens": ([40, 64, 65, 1, 0, 90, 30, 20], 64, 128, 148),
    "pairs, tokens on the N side": ([1, 20, 33, 100, 200, 300, 256, 0], 256, 256, 74),
    "pairs, tokens on the M side": ([300, 513, 1, 256, 299, 420, 0, 280], 256, 256, 74),
}


@pytest.mark.parametrize("K", [272, 1680], ids=["K inside the ring", "K past the ring"])
@pytest.mark.parametrize("epi", [NONE, SWIGLU], ids=["none", "swiglu"])
@pytest.mark.parametrize("form", MANY_TILES)
def test_grouped_gemm_of_many_tiles_a_worker(form, epi, K):
    """Each worker walks five tiles and more: accumulators handed back and taken again, barriers through several phases,
    tiles of other extents and other groups one after another, with a short K the next tile's loads under this one's sums."""
    sizes, tok, feat, workers = MANY_TILES[form]
    rng = np.random.default_rng(tok + epi + K)
    sizes = np.concatenate([rng.permutation(sizes) for _ in range(8)])
    N = 1040 if "M side" in form else 1568
    rows, n = int(sizes.sum()), len(sizes)
    mean = (rows + 5) / n
    assert {16: mean <= 8, 32: 8 < mean <= 16, 64: 16 < mean <= 56, 256: mean > 56}[tok]
    assert feat == 128 or (mean <= 160) == ("N side" in form)
    assert (-(-sizes // tok) * -(-N // feat)).sum() >= 5 * workers
    a, sa, b, sb, _, _ = operands(rng, rows, n * N, K, epi)
    out, off = grouped(a, sa, b, sb, sizes, N, epi, extra=5)
    for g in range(n):
        r, w = slice(off[g], off[g + 1]), slice(g * N, (g + 1) * N)
        near(out[r], int8.gemm(a[r], sa[r], b[w], sb[w], epi))


@pytest.mark.parametrize("K", [272, 1680], ids=["K inside the ring", "K past the ring"])
@pytest.mark.parametrize("epi", [NONE, SWIGLU, BIAS_RESIDUAL], ids=["none", "swiglu", "bias, residual"])
def test_gemm_of_many_tiles_a_pair(epi, K):
    M, N = 3001, 8208
    assert -(-M // 256) * -(-N // 256) >= 5 * 74
    rng = np.random.default_rng(epi + K)
    a, sa, b, sb, bias, res = operands(rng, M, N, K, epi)
    terms = 0.0 if epi != BIAS_RESIDUAL else np.abs(int8.gemm(a, sa, b, sb)) + np.abs(bias) + np.abs(res)
    near(gemm(a, sa, b, sb, epi, bias, res), int8.gemm(a, sa, b, sb, epi, bias, res), terms)


# ------------------------------------------------------------- GELU of far values


@pytest.mark.parametrize("M,N", [(6, 272), (200, 272), (6100, 528)], ids=["cluster", "cluster, many tokens", "pairs"])
def test_gemm_gelu_of_large_values(M, N):
    """GELU as x / (1 + e^-w), w = 2 sqrt(2/pi) (x + 0.044715 x^3), with the fast exponential and division.

    x carries the conversion of the sum, two scale products and the bias addition: dx <= (3 |v| + |x|) 2^-24.  The
    result's relative error is dx / |x| (1 + 3 |w|), as w grows no faster than x^3; 8 |w| 2^-24 from w's own roundings
    and constants; (2 + 1.2 |w|) 2^-23 from the exponential; 3 2^-23 from the sum and the division; 2^-8 from bf16.
    Below w = -80 the value vanishes (under 1e-30)."""
    rng = np.random.default_rng(21)
    K = 528
    a, sa, b, sb, bias, _ = operands(rng, M, N, K, BIAS_GELU)
    sa = sa * np.exp2(rng.uniform(-3, 3, M)).astype(F)  # rows of all sizes: products of a few units up to hundreds
    out = gemm(a, sa, b, sb, BIAS_GELU, bias).astype(np.float64)
    v = int8.gemm(a, sa, b, sb)
    x = v + bias
    assert x.min() < -200 and x.max() > 200 and (np.abs(x) < 6).mean() > 0.01
    w = 2 * np.sqrt(2 / np.pi) * (x + 0.044715 * x**3)
    with np.errstate(over="ignore"):
        ref = x / (1 + np.exp(-w))
    assert np.isfinite(out).all()
    seen = w > -80
    # where w is above 20 the value is x itself, to less than the other terms
    aw = np.minimum(np.abs(w), np.where(w > 0, 20, np.inf))
    dx = (3 * np.abs(v) + np.abs(x)) * 2.0**-24 / np.maximum(np.abs(x), 1e-30)
    lim = np.abs(ref) * (2.0**-8 + dx * (1 + 3 * aw) + 8 * aw * 2.0**-24 + (5 + 1.2 * aw) * 2.0**-23) + 1e-30
    assert (np.abs(out - ref) <= lim)[seen].all(), float((np.abs(out - ref) / lim)[seen].max())
    assert np.abs(out[~seen]).max() < 1e-30 and (~seen).any()
