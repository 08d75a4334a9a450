"""Kernels whose waits run out: a copy that never lands ends the call within the waits' limit (two seconds each), with the
error word set, what it does not concern right, and the GPU as it was.  The kernels are compiled with a problem of the
test's own, in which one copy is announced and not issued; nothing of it is in flight."""

import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

from oracle import serving

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import gpu_util as G
    from test_gpu_window import Cache, close, queries

TESTS = os.path.dirname(os.path.abspath(__file__))
WAIT_TIMEOUT = 1


def compiled(folder, name):
    from atb_llm_study_b200 import build

    if not shutil.which(build.NVCC):
        pytest.skip("no nvcc")
    lib = os.path.join(folder, name + ".so")
    subprocess.run([build.NVCC, *build.CU_FLAGS, "-shared", os.path.join(TESTS, "cuda", name + ".cu"), "-o", lib], check=True)
    return ctypes.CDLL(lib)


@pytest.fixture(scope="module")
def items(tmp_path_factory):
    return compiled(str(tmp_path_factory.mktemp("lost")), "lost_copies")


def address(t):
    return ctypes.c_void_p(t.data_ptr())


NONE, Q, K, V = range(4)


@pytest.mark.parametrize("lost,item,tile", [(NONE, 0, 0), (Q, 2, 1), (K, 0, 1), (V, 0, 0), (V, 2, 2)],
                         ids=["none", "Q", "K", "V-first", "V-later"])
def test_items_kernel_ends_when_a_copy_is_lost(items, lost, item, tile):
    n, keys = 5, 300  # CTA 0 walks items 0, 2, 4 and CTA 1 items 1, 3, three key tiles each
    rng = np.random.default_rng(1)
    q, k, v = (G.rounded(rng.standard_normal((m, 64)) * s) for m, s in ((n * 256, 2), (keys, 1), (keys, 1)))
    want, weight = serving.attend(q, k, v, np.ones((n * 256, keys), bool), 0.125)
    dq, dk, dv = G.bf16(q), G.bf16(k), G.bf16(v)
    for now in (lost, NONE):
        out = torch.full((n * 256, 64), -5.0, dtype=torch.bfloat16, device=G.DEV)
        err = torch.zeros(1, dtype=torch.int32, device=G.DEV)
        assert items.lost_copy(address(dq), address(dk), address(dv), address(out), n, keys, 2, now, item, tile, address(err),
                               ctypes.c_void_p(G.stream())) == 0
        torch.cuda.synchronize()
        got = G.host(out)
        if now == NONE:
            assert err.item() == 0
            close(got, want, weight)
            continue
        assert err.item() == WAIT_TIMEOUT
        for i in range(n):
            rows = slice(i * 256, i * 256 + 256)
            sides = [slice(rows.start, rows.start + 128), slice(rows.start + 128, rows.stop)]
            for side in sides:  # stored as it should be, or not at all
                if i % 2 == 1 or not (got[side] == -5).all():
                    close(got[side], want[side], weight[side])
            if i % 2 == 0 and i >= item:
                assert any((got[side] == -5).all() for side in sides)


@pytest.fixture(scope="module")
def token(tmp_path_factory):
    return compiled(str(tmp_path_factory.mktemp("lost")), "lost_token_copies")


@pytest.mark.parametrize("lens", [[100, 1], [700, 30]], ids=["two-tiles", "ring-wraps"])
@pytest.mark.parametrize("ctas", [1, 2])
def test_token_kernel_ends_when_copies_are_lost(token, lens, ctas):
    c = Cache(3, lens, 2, 64, 64)
    q, qd = queries(3, 2, 4, 64)
    k, v, tables, ctx = c.device()
    want, weight = serving.window_decode(q, c.k, c.v, c.tables, lens, 1 << 20, 0)
    for box in (32, 64):
        out = torch.full((2, 256), -5.0, dtype=torch.bfloat16, device=G.DEV)
        err = torch.zeros(1, dtype=torch.int32, device=G.DEV)
        assert token.lost_token_copy(address(qd), address(k), address(v), address(tables), c.width, address(ctx), 2, 4, 2, 64,
                                     c.blocks, 1 << 20, address(out), ctas, box, address(err), ctypes.c_void_p(G.stream())) == 0
        torch.cuda.synchronize()
        if box == 32:
            assert err.item() == WAIT_TIMEOUT
        else:
            assert err.item() == 0
            close(G.host(out).reshape(want.shape), want, weight)
