"""The vocabulary operators where they could go wrong unseen: what was in a workspace before, switches, derivatives that
nothing carries, near ties, rows of very different weights."""
import math
import os
import subprocess
import sys

import pytest
import torch

from oracle import vocabulary as oracle
from test_vocabulary_gpu import _inside, _pair, _teacher

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,v,d,temperature", [
    (1, 32768, 64, 1.0), (2, 32768, 64, 1e-9), (1, 10000, 64, 1e-9), (2, 10000, 16392, 1.0), (1, 9473, 16392, 1.0),
    (2, 40000, 264, 1e-9)])
def test_one_and_two_rows_in_a_used_workspace(n, v, d, temperature):
    """Whatever a workspace held before takes no part: behind the FP32 pass (the first case) and behind the tile pass, which
    wide features and very small temperatures take with one or two rows, too."""
    from memoryefficientclip_b200 import _lib, ops
    x, table, tokens, g = _pair(n, v, d, torch.bfloat16, v + n)
    x = (x.double() * temperature).bfloat16()           # scores of ordinary size
    want = oracle.token_log_probs(x, table, tokens[:, None], temperature, 3)
    xg, yg, tg = x.cuda(), table.cuda(), tokens.cuda()
    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
    size = lib.meclip_vocab_workspace_bytes(n, v, 3)
    ws = torch.full((size // 4,), 60.0, device="cuda")  # read as a partial sum: a score of 60 and a weight of 61
    assert ws.numel() * 4 == size
    lp, entropy, lse, scores = (torch.empty(n, device="cuda") for _ in range(4))
    top_lp, top = torch.empty(n, 3, device="cuda"), torch.empty(n, 3, dtype=torch.int64, device="cuda")
    _lib.check(lib.meclip_token_log_probs(
        xg.data_ptr(), yg.data_ptr(), 0, n, v, d, d, d, temperature, tg.data_ptr(), 1, lp.data_ptr(), entropy.data_ptr(), 3,
        top_lp.data_ptr(), top.data_ptr(), lse.data_ptr(), scores.data_ptr(), ws.data_ptr(), size, None, stream))
    _inside(lp, want["log_probs"][:, 0], want["err_lp"], "log_probs")
    _inside(entropy, want["entropy"], want["err_entropy"], "entropy")
    assert torch.equal(top.cpu(), want["top_tokens"])
    _inside(top_lp, want["top_log_probs"], want["err_lp"][:, None], "top_log_probs")
    logits = torch.randn(n, 2, generator=g)
    t = torch.stack([tokens, (tokens + 1) % v], 1)
    t_dev, logits_dev = t.cuda(), logits.cuda()
    size = lib.meclip_vocab_workspace_bytes(n, v, 0)
    ws = torch.full((size // 4,), 60.0, device="cuda")
    row_loss, has = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    loss, inv = torch.empty((), device="cuda"), torch.empty((), device="cuda")
    pair, probs = torch.empty(n, 2, device="cuda"), torch.empty(n, 2, device="cuda")
    _lib.check(lib.meclip_distill(
        xg.data_ptr(), yg.data_ptr(), 0, n, v, d, d, d, temperature, t_dev.data_ptr(), logits_dev.data_ptr(),
        ops._DT[torch.float32], 2, 1.0, 1, row_loss.data_ptr(), has.data_ptr(), loss.data_ptr(), inv.data_ptr(),
        lse.data_ptr(), pair.data_ptr(), probs.data_ptr(), ws.data_ptr(), size, None, stream))
    kl, there, err = oracle.distill(x, table, t, logits, temperature)
    _inside(row_loss, kl, err, "row loss")
    _inside(loss, kl.mean(), err.mean() + 2 * oracle.ULP * kl.mean(), "loss")
    assert there.all()
