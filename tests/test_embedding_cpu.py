"""Refusals and sizes of the embedding entry points, on the CPU."""
import ctypes

import pytest
import torch

import memoryefficientclip_b200 as m
from memoryefficientclip_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build_library()
    return _lib.load()


def test_cpu_tensors_are_refused():
    with pytest.raises(AssertionError):
        m.embed_tokens(torch.zeros(3, dtype=torch.long), torch.randn(4, 8))


def test_entry_points_refuse(lib):
    p, big = ctypes.c_void_p(0x1000), 1 << 40

    def look(tok=p, n=3, t=p, dtype=_lib.F32, v=9, d=8, ldt=8, out=p, ldo=8):
        return lib.meclip_embed(tok, n, t, dtype, v, d, ldt, 1.0, out, ldo, None)

    def grad(tok=p, n=3, g=p, dtype=_lib.F32, v=9, d=8, ldg=8, out=p, ldd=8, ws=p, nws=big):
        return lib.meclip_embed_grad(tok, n, g, dtype, v, d, ldg, 1.0, out, ldd, ws, nws, None)

    for bad in (dict(tok=None), dict(out=None), dict(dtype=7), dict(n=-1), dict(n=1 << 31), dict(v=0), dict(v=1 << 31), dict(d=0)):
        assert look(**bad) == _lib.EINVAL and grad(**bad) == _lib.EINVAL, bad
    for bad in (dict(t=None), dict(ldt=7), dict(ldo=7)):
        assert look(**bad) == _lib.EINVAL, bad
    for bad in (dict(g=None), dict(ldg=7), dict(ldd=7), dict(ws=None), dict(ws=ctypes.c_void_p(0x1010))):
        assert grad(**bad) == _lib.EINVAL, bad
    assert grad(nws=64) == _lib.ENOSPC
    assert look(n=0, tok=None, t=None) == _lib.OK            # nothing to look up: nothing is launched


def test_workspace_sizes(lib):
    size = lib.meclip_embed_grad_workspace_bytes
    assert size(0, 9, 8) > 0 and size(-1, 9, 8) == 0
    # lists of 4 words per token, two sums of the width per 32 tokens and one per 1024, counts of the sorting blocks
    n, v, d = 131072, 50000, 1152
    need = 16 * n + 4 * d * (2 * n // 32 + n // 1024)
    assert need <= size(n, v, d) <= need + 2**20
