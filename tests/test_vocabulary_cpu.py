"""Refusals of the vocabulary operators, on the CPU: checks of arguments and error codes of the C entry points."""
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
    x, y = torch.randn(4, 8), torch.randn(9, 8)
    with pytest.raises(AssertionError):
        m.token_log_probs(x, y, torch.zeros(4, dtype=torch.long))
    with pytest.raises(AssertionError):
        m.MemoryEfficientDistillLoss()(x, y, torch.zeros(4, 2, dtype=torch.long), torch.zeros(4, 2))


def test_entry_points_refuse(lib):
    p = ctypes.c_void_p(0x1000)
    odd = ctypes.c_void_p(0x1004)
    big = 1 << 30

    def score(x=p, t=p, dtype=_lib.BF16, rows=4, vocab=9, d=8, ldx=8, ldt=8, temp=1.0, tok=p, k=1, lp=p, top=0, tlp=p, tt=p,
              ws=p, nws=big):
        return lib.meclip_token_log_probs(x, t, dtype, rows, vocab, d, ldx, ldt, temp, tok, k, lp, p, top, tlp, tt, p, p, ws,
                                          nws, None, None)

    for bad in (dict(x=None), dict(t=None), dict(tok=None), dict(lp=None), dict(dtype=_lib.F32), dict(rows=0), dict(vocab=0),
                dict(rows=1 << 31), dict(d=12, ldx=16, ldt=16), dict(ldx=4), dict(ldt=12), dict(x=odd), dict(temp=0.0),
                dict(temp=-1.0), dict(temp=float("nan")), dict(temp=float("inf")), dict(k=257), dict(k=-1), dict(top=33),
                dict(top=10), dict(top=-1), dict(top=2, tlp=None), dict(top=2, tt=None)):
        assert score(**bad) == _lib.EINVAL, bad

    def teach(per_row=2, logits=p, dtype=_lib.F32, temp=1.0, loss=p, inv=p, probs=p):
        return lib.meclip_distill(p, p, _lib.BF16, 4, 9, 8, 8, 8, 1.0, p, logits, dtype, per_row, temp, 1, p, p, loss, inv, p,
                                  p, probs, p, big, None, None)

    for bad in (dict(per_row=0), dict(per_row=257), dict(logits=None), dict(dtype=9), dict(temp=0.0), dict(loss=None),
                dict(inv=None), dict(probs=None)):
        assert teach(**bad) == _lib.EINVAL, bad

    def grad(rows=4, dtype=_lib.BF16, lse=p, scores=p, h=p, ent=p, ws=p, nws=big):
        return lib.meclip_token_log_probs_grad(p, p, dtype, rows, 9, 8, 8, 8, 1.0, p, 1, lse, ent, scores, p, h, p,
                                               _lib.STORE_BF16, 8, p, _lib.STORE_BF16, 8, ws, nws, None, None)

    for bad in (dict(rows=0), dict(dtype=_lib.F32), dict(lse=None), dict(scores=None), dict(ent=None), dict(ws=None),
                dict(ws=ctypes.c_void_p(0x1010))):
        assert grad(**bad) == _lib.EINVAL, bad
    assert grad(nws=16) == _lib.ENOSPC
    assert lib.meclip_distill_grad(p, p, _lib.BF16, 4, 9, 8, 8, 8, 1.0, p, 2, p, p, p, p, None, 0, p, p, 0, 8, p, 0, 8, p, big,
                                   None, None) == _lib.EINVAL                  # no grad_out


def test_workspace_sizes(lib):
    # 16 bytes per row and half tile, 8 more per 32 columns with alternatives; rows beyond a block cost nothing
    plain, top = lib.meclip_vocab_workspace_bytes(4096, 32768, 0), lib.meclip_vocab_workspace_bytes(4096, 32768, 8)
    assert plain == 4096 * 32768 // 128 * 16 and top == plain + 4096 * 1024 * 8
    assert lib.meclip_vocab_workspace_bytes(1 << 20, 32768, 0) == lib.meclip_vocab_workspace_bytes(16384, 32768, 0)
    assert lib.meclip_vocab_workspace_bytes(0, 8, 0) == 0 and lib.meclip_vocab_grad_workspace_bytes(0, 4, 0, 8) == 0
    assert lib.meclip_vocab_grad_workspace_bytes(0, 128, 4096, 512) >= 2 * 128 * 4096 * 2


def test_module_defaults_follow_the_package():
    mod = m.MemoryEfficientDistillLoss()
    assert (mod.temperature, mod.normalized_inputs, mod.teacher_temperature, mod.reduction) == (0.07, False, 1.0, "mean")
    assert not list(mod.parameters())


def test_rows_that_the_kernels_can_address():
    """Broadcast and overlapping rows are copied, whatever else stays as it is."""
    from memoryefficientclip_b200 import ops
    m = torch.zeros(40, 64, dtype=torch.bfloat16)
    for view, plain in ((m, True), (m[::2], True), (m[:, :32], True), (m[:1].expand(40, 64), False), (m.T, False),
                        (m.reshape(-1).as_strided((30, 64), (8, 1)), False), (m[:1].as_strided((1, 64), (0, 1)), True)):
        assert (ops.row_major(view) is view) == plain
        assert view.shape[0] == 1 or ops._is_operand(view) == plain
