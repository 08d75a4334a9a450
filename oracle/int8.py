"""8-bit quantisation and products restated in numpy (64-bit).

The reference runs fp16 throughout (atb_cpp_llm/src/io/weight_helpers.cpp:16-76),
so parity is unpinned by it; this follows the definitions the C ABI documents:
symmetric rows, ``scale = amax / 127``, round half to even, exact integer sums.
"""

import numpy as np


def quant_rows(x):
    """``x [rows, dim]`` (bf16 values) -> ``(q int8, scale fp32)``.  127 x / amax
    is exact in float64 where it is a half integer, and at least 2^-17 away
    from one where it is not, so ``rint`` decides every tie as the definition."""
    x = np.asarray(x, np.float64)
    bad = ~np.isfinite(x).all(1)
    xf = np.where(bad[:, None], 0.0, x)
    amax = np.abs(xf).max(1)
    q = np.rint(127 * xf / np.where(amax > 0, amax, 1.0)[:, None]).astype(np.int8)
    scale = amax.astype(np.float32) / np.float32(127)
    scale[bad] = np.nan
    return q, scale


def silu(v):
    with np.errstate(over="ignore"):
        return v / (1 + np.exp(-v))


def gelu_tanh(v):
    return 0.5 * v * (1 + np.tanh(np.sqrt(2 / np.pi) * (v + 0.044715 * v**3)))


def gemm(a, a_scale, b, b_scale, epi=0, bias=None, residual=None):
    """``epi(a_scale b_scale (a @ b^T))`` in float64 (the integer sums are exact
    below 2^53); epilogue numbers as in the C ABI."""
    v = a.astype(np.float64) @ b.astype(np.float64).T
    v = v * np.asarray(a_scale, np.float64)[:, None] * np.asarray(b_scale, np.float64)
    if epi in (1, 4, 5):
        v = v + np.asarray(bias, np.float64)
    if epi == 4:
        v = gelu_tanh(v)
    if epi in (2, 5):
        v = v + np.asarray(residual, np.float64)
    if epi == 3:
        v = silu(v[:, 0::2]) * v[:, 1::2]
    return v
