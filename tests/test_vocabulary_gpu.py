"""Token log probabilities and distillation over a vocabulary against the 64-bit oracle (oracle/vocabulary.py, which
derives the bounds from the roundings of the computation)."""
import math
import os
import subprocess
import sys

import pytest
import torch

from oracle import vocabulary as oracle

pytestmark = pytest.mark.gpu


def _pair(n, v, d, dtype, seed, bump=8.0):
    """Features that lean towards one row of the table each, and that row's index."""
    g = torch.Generator().manual_seed(seed)
    table = torch.randn(v, d, generator=g) / math.sqrt(d)
    tokens = torch.randint(0, v, (n,), generator=g)
    x = 2.0 * torch.randn(n, d, generator=g) + bump * table[tokens]
    return x.to(dtype), table.to(dtype), tokens, g


def _operands(x, table):
    """What the kernels read of these inputs: fp16 pairs as they are, everything else as bf16."""
    if x.dtype == table.dtype == torch.float16:
        return x, table
    return x.bfloat16(), table.bfloat16()


def _inside(got, want, bound, what):
    got = got.detach().double().cpu()
    assert torch.isfinite(got).all(), what
    worst = ((got - want).abs() / bound).max().item()
    assert worst <= 1.0, f"{what}: {worst:.2f} of the bound"


SHAPES = [            # rows, vocabulary, features
    (1, 1, 8), (1, 33, 64), (1, 32768, 512), (3, 50, 100), (5, 257, 72), (127, 1000, 64), (128, 64, 128), (129, 4099, 512),
    (300, 2049, 96), (297, 8191, 1152), (640, 777, 1024), (2000, 333, 30)]


@pytest.mark.parametrize("n,v,d", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_scores_match_the_oracle(n, v, d, dtype):
    from memoryefficientclip_b200 import token_log_probs
    x, table, tokens, g = _pair(n, v, d, dtype, n * 7 + v)
    k = min(v, 7)
    many = torch.randint(-2, v, (n, 5), generator=g)
    many[:, 0] = tokens
    xo, yo = _operands(x, table)
    want = oracle.token_log_probs(xo, yo, many, 0.9, k)
    got = token_log_probs(x.cuda(), table.cuda(), many.cuda(), temperature=0.9, top_k=k)
    assert got.log_probs.shape == (n, 5) and got.top_tokens.dtype == torch.int64
    _inside(got.log_probs, want["log_probs"], want["err_lp"][:, None], "log_probs")
    _inside(got.entropy, want["entropy"], want["err_entropy"], "entropy")
    assert torch.equal(got.top_tokens.cpu(), want["top_tokens"])
    _inside(got.top_log_probs, want["top_log_probs"], want["err_lp"][:, None], "top_log_probs")
    one = token_log_probs(x.cuda(), table.cuda(), tokens.int().cuda(), temperature=0.9)
    assert one.log_probs.shape == (n,) and one.top_tokens is None
    assert torch.equal(one.log_probs, got.log_probs[:, 0]) and torch.equal(one.entropy, got.entropy)


@pytest.mark.parametrize("top_k", [1, 2, 8, 31, 32])
@pytest.mark.parametrize("n", [2, 400])
def test_alternatives_that_are_close_or_equal(n, top_k):
    """Best rows beside each other in one chunk of 32, repeated rows, and a row of zeros: ties go to the lower token."""
    from memoryefficientclip_b200 import token_log_probs
    v, d = 700, 64
    x, table, tokens, g = _pair(n, v, d, torch.bfloat16, 5 + top_k, bump=0.0)
    table[40:72] = (table[40] + 0.02 * torch.randn(32, d, generator=g).bfloat16())          # one direction, two chunks
    table[300:340] = table[300]                                                             # equal rows
    table[650:] = 0
    x[0] = 0                                                                                # everything ties
    x[1] = 6 * table[300]
    if n > 2:
        x[2:40] = 9 * table[40]
        x[40:60] = -4 * table[100:120]
    want = oracle.token_log_probs(x, table, tokens[:, None], 1.0, top_k)
    got = token_log_probs(x.cuda(), table.cuda(), tokens.cuda(), top_k=top_k)
    assert torch.equal(got.top_tokens.cpu(), want["top_tokens"])
    _inside(got.top_log_probs, want["top_log_probs"], want["err_lp"][:, None], "top_log_probs")


def test_all_scores_low_and_far_apart():
    """Scores of minus hundreds, and one row that holds all the probability."""
    from memoryefficientclip_b200 import token_log_probs
    g = torch.Generator().manual_seed(3)
    table = (torch.randn(517, 64, generator=g) + 3.0).bfloat16()
    x = (-3.0 + torch.randn(9, 64, generator=g)).bfloat16()
    x[4] = 20 * table[11]
    tokens = torch.full((9,), 11)
    want = oracle.token_log_probs(x, table, tokens[:, None], 1.0, 4)
    got = token_log_probs(x.cuda(), table.cuda(), tokens.cuda(), top_k=4)
    _inside(got.log_probs, want["log_probs"][:, 0], want["err_lp"], "log_probs")
    _inside(got.entropy, want["entropy"], want["err_entropy"], "entropy")
    assert torch.equal(got.top_tokens.cpu(), want["top_tokens"])


@pytest.mark.parametrize("d,bump", [(64, 24.0), (512, 16.0), (512, 40.0), (1024, 24.0)])
def test_rows_that_one_token_holds(d, bump):
    """log p = -log(1 + R), R = sum_j exp(z_j - z_t): down to 1e-11 it is as exact as the scores, which make every term of
    R off by at most the errors of its two scores."""
    from memoryefficientclip_b200 import token_log_probs
    x, table, tokens, _ = _pair(200, 3000, d, torch.bfloat16, 9, bump)
    z, err = oracle.scores(x, table, 1.0)
    rest = torch.exp(z - z.gather(1, tokens[:, None])).scatter(1, tokens[:, None], 0.0).sum(1)
    want = -torch.log1p(rest)
    best = z.argmax(1) == tokens
    assert best.sum() > 100
    got = token_log_probs(x.cuda(), table.cuda(), tokens.cuda(), top_k=2)
    bound = (2.2 * err + 16 * oracle.ULP) * want.abs()
    _inside(got.log_probs[best.cuda()], want[best], bound[best], "log_probs")
    _inside(got.top_log_probs[best.cuda(), 0], want[best], bound[best], "top_log_probs")


def test_padding_and_tokens_behind_the_table():
    from memoryefficientclip_b200 import token_log_probs
    x, table, tokens, _ = _pair(70, 300, 64, torch.bfloat16, 1)
    tokens[3], tokens[5], tokens[8] = -1, 300, -100
    x[9] = float("nan")
    got = token_log_probs(x.cuda(), table.cuda(), tokens.cuda(), top_k=3)
    lp = got.log_probs.cpu()
    assert lp[3] == 0 and lp[8] == 0 and lp[5].isnan() and lp[9].isnan() and got.entropy[9].isnan()
    keep = torch.tensor([i for i in range(70) if i not in (3, 5, 8, 9)])
    want = oracle.token_log_probs(x[keep], table, tokens[keep][:, None], 1.0, 3)
    _inside(lp[keep], want["log_probs"][:, 0], want["err_lp"], "the other rows")
    assert torch.equal(got.top_tokens.cpu()[keep], want["top_tokens"])


@pytest.mark.parametrize("n,v,d", [(1, 40, 64), (5, 1000, 64), (130, 257, 100), (300, 4099, 512), (1100, 2051, 264),
                                   (64, 9000, 96), (1500, 700, 1152)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_score_gradients(n, v, d, dtype):
    from memoryefficientclip_b200 import token_log_probs
    x, table, tokens, g = _pair(n, v, d, dtype, n + v, bump=6.0)
    many = torch.stack([tokens, torch.randint(-1, v, (n,), generator=g), tokens, torch.randint(-1, v, (n,), generator=g)], 1)
    g_lp = torch.randn(n, 4, generator=g)
    g_h = torch.randn(n, generator=g) * 0.3
    xg, yg = x.cuda().requires_grad_(True), table.cuda().requires_grad_(True)
    got = token_log_probs(xg, yg, many.cuda(), temperature=1.3)
    dx, dy = torch.autograd.grad([got.log_probs, got.entropy], [xg, yg], [g_lp.cuda(), g_h.cuda()])
    assert dx.dtype == dtype and dy.dtype == dtype
    xo, yo = _operands(x, table)
    rounding = 2.0 ** -8 if dtype == torch.float16 else 0.0      # the contractions read bf16 operands
    wx, wy, bx, by = oracle.token_log_probs_grad(xo, yo, many, 1.3, g_lp, g_h, (dtype, dtype), rounding)
    _inside(dx, wx, bx, "dx")
    _inside(dy, wy, by, "dtable")


def test_score_gradient_parts():
    """Only log probabilities, only entropy, only one input, a frozen table; differences of the loss agree."""
    from memoryefficientclip_b200 import token_log_probs
    n, v, d = 40, 500, 64
    x, table, tokens, g = _pair(n, v, d, torch.bfloat16, 11)
    g_lp, g_h, zero = torch.randn(n, generator=g), torch.randn(n, generator=g), torch.zeros(n)
    for a, b in ((g_lp, None), (None, g_h)):
        xg, yg = x.cuda().requires_grad_(True), table.cuda()
        out = token_log_probs(xg, yg, tokens.cuda())
        out = out.log_probs if b is None else out.entropy
        out.backward((a if b is None else b).cuda())
        wx, _wy, bx, _by = oracle.token_log_probs_grad(x, table, tokens[:, None], 1.0, (zero if a is None else a)[:, None],
                                                       zero if b is None else b, (torch.bfloat16, torch.bfloat16))
        _inside(xg.grad, wx, bx, "dx")
    yg = table.cuda().requires_grad_(True)
    token_log_probs(x.cuda(), yg, tokens.cuda()).log_probs.backward(g_lp.cuda())
    _wx, wy, _bx, by = oracle.token_log_probs_grad(x, table, tokens[:, None], 1.0, g_lp[:, None], zero,
                                                   (torch.bfloat16, torch.bfloat16))
    _inside(yg.grad, wy, by, "dtable")
    # differences of the 64-bit sum along a direction against the oracle's gradient (which the kernels matched above)
    def f(e):
        r = oracle.token_log_probs(x.double() + e, table, tokens[:, None], 1.0)
        return (r["log_probs"][:, 0] * g_lp.double()).sum() + (r["entropy"] * g_h.double()).sum()
    wx, _, _, _ = oracle.token_log_probs_grad(x, table, tokens[:, None], 1.0, g_lp[:, None], g_h, (torch.float64,) * 2)
    way = torch.randn(n, d, generator=g).double()
    slope = (f(1e-5 * way) - f(-1e-5 * way)) / 2e-5
    assert abs(slope - (wx * way).sum()) <= 1e-6 * wx.norm() * way.norm()


def _teacher(n, v, k, g, dtype=torch.float32):
    t = torch.stack([torch.randperm(v, generator=g)[:k] if k <= v else torch.randint(0, v, (k,), generator=g)
                     for _ in range(n)])
    logits = (3 * torch.randn(n, k, generator=g)).to(dtype)
    return t, logits


@pytest.mark.parametrize("n,v,d,k", [(1, 9, 64, 1), (7, 300, 72, 5), (129, 4099, 512, 8), (310, 1000, 1152, 64),
                                     (1200, 600, 128, 33), (33, 2000, 64, 256)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_distillation(n, v, d, k, dtype, reduction):
    from memoryefficientclip_b200 import MemoryEfficientDistillLoss
    x, table, _tokens, g = _pair(n, v, d, dtype, n + k)
    t, logits = _teacher(n, v, k, g, torch.float32 if reduction == "mean" else dtype)
    if n > 6:
        t[1, k // 2:] = -1                       # short rows, with anything in the absent places
        logits[1, k // 2:] = float("nan")
        t[2] = -1                                # nothing left
        logits[2] = float("inf")
        logits[3] = float("-inf")                # named, but impossible: nothing left either
        logits[4, :-1] = float("-inf")           # one entry left
        logits[5, 0] = torch.finfo(logits.dtype).min
    if k > 4:
        t[0, 3] = t[0, 1]                        # the same token twice
    xg, yg = x.cuda().requires_grad_(True), table.cuda().requires_grad_(True)
    mod = MemoryEfficientDistillLoss(0.8, normalized_inputs=True, teacher_temperature=1.7, reduction=reduction)
    loss = mod(xg, yg, t.cuda(), logits.cuda())
    xo, yo = _operands(x, table)
    kl, has, err = oracle.distill(xo, yo, t, logits, 0.8, 1.7)
    if reduction == "none":
        go = torch.randn(n, generator=g)
        weight = go
        assert loss.shape == (n,)
        _inside(loss, kl, err + 1e-30, "loss")
    else:
        go = torch.tensor(0.7)
        count = has.sum().double() if reduction == "mean" else 1.0
        weight = go.double() / count * torch.ones(n)
        assert loss.shape == ()
        _inside(loss, kl.sum() / count, err.sum() / count + 2 * oracle.ULP * kl.sum() / count, "loss")
    dx, dy = torch.autograd.grad(loss, [xg, yg], go.cuda())
    assert dx.dtype == dtype and dy.dtype == dtype
    rounding = 2.0 ** -8 if dtype == torch.float16 else 0.0
    wx, wy, bx, by = oracle.distill_grad(xo, yo, t, logits, 0.8, weight, (dtype, dtype), 1.7, rounding)
    _inside(dx, wx, bx, "dx")
    _inside(dy, wy, by, "dtable")
    if n > 6:
        assert not dx[2:4].any()


def test_distillation_without_any_teacher_entry():
    from memoryefficientclip_b200 import MemoryEfficientDistillLoss
    x, table, _t, _g = _pair(20, 100, 64, torch.bfloat16, 2)
    xg = x.cuda().requires_grad_(True)
    loss = MemoryEfficientDistillLoss(1.0, True)(xg, table.cuda(), torch.full((20, 3), -1).cuda(), torch.zeros(20, 3).cuda())
    loss.backward()
    assert loss.item() == 0.0 and not xg.grad.any()
    # a token behind the table is a mistake and shows
    bad = MemoryEfficientDistillLoss(1.0, True)(xg, table.cuda(), torch.full((20, 3), 100).cuda(), torch.zeros(20, 3).cuda())
    assert bad.isnan()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_distillation_of_two_towers(dtype):
    """normalized_inputs=False: both sides are normalised inside; the gradients carry the Jacobian."""
    from memoryefficientclip_b200 import MemoryEfficientDistillLoss
    n, d = 260, 96
    g = torch.Generator().manual_seed(8)
    img = torch.randn(n, d, generator=g).to(dtype)
    txt = (img.float() + torch.randn(n, d, generator=g)).to(dtype)
    t, logits = _teacher(n, n, 6, g)
    t[:, 0] = torch.arange(n)
    xg, yg = img.cuda().requires_grad_(True), txt.cuda().requires_grad_(True)
    loss = MemoryEfficientDistillLoss(0.07)(xg, yg, t.cuda(), logits.cuda())
    loss.backward()
    a, b = img.double().requires_grad_(True), txt.double().requires_grad_(True)
    z = torch.nn.functional.normalize(a, dim=1) @ torch.nn.functional.normalize(b, dim=1).T / 0.07
    q = torch.softmax(logits.double(), 1)
    ref = (torch.xlogy(q, q) - q * torch.log_softmax(z, 1).gather(1, t)).sum(1).mean()
    ref.backward()
    # the normalised operands are rounded to bf16 (2^-8 of each component; a cosine of 96 random roundings moves by
    # 2^-8 sqrt(2 / 96 / 3) or so, over T): the package's usual bars for that
    assert abs(loss.item() - ref.item()) <= 1e-3 * abs(ref.item())
    for got, want in ((xg.grad, a.grad), (yg.grad, b.grad)):
        got = got.double().cpu()
        assert (got - want).norm() <= 1e-2 * want.norm()


@pytest.mark.parametrize("make", ["strided", "offset", "transposed"])
def test_layouts(make):
    """Pitches, offsets and orders other than the plain ones."""
    from memoryefficientclip_b200 import token_log_probs
    n, v, d = 50, 333, 64
    x, table, tokens, g = _pair(n, v, d, torch.bfloat16, 4)
    if make == "strided":
        xs = torch.zeros(n, d + 24, dtype=x.dtype).cuda()[:, :d].copy_(x)
        ys = torch.zeros(2 * v, d, dtype=x.dtype).cuda()[::2].copy_(table)
    elif make == "offset":
        xs = torch.zeros(n * d + 3, dtype=x.dtype).cuda()[3:].view(n, d).copy_(x)
        ys = torch.zeros(v, d + 5, dtype=x.dtype).cuda()[:, 5:].copy_(table)
    else:
        xs, ys = x.T.contiguous().cuda().T, table.T.contiguous().cuda().T
    tk = torch.stack([tokens, tokens], 1).cuda()[:, 0]
    plain = token_log_probs(x.cuda(), table.cuda(), tokens.cuda(), top_k=3)
    got = token_log_probs(xs, ys, tk, top_k=3)
    for a, b in zip(plain, got):
        assert torch.equal(a, b)


def test_many_row_blocks_and_panels():
    """Rows over several coefficient blocks: the blocked backward puts every entry into its own panel."""
    from memoryefficientclip_b200 import _lib, MemoryEfficientDistillLoss
    n, v, d, k = 1300, 1500, 64, 9
    x, table, _t, g = _pair(n, v, d, torch.bfloat16, 21)
    t, logits = _teacher(n, v, k, g)
    _lib.check(_lib.load().meclip_debug_set_blocking(256, 256 * 2 * 512))
    try:
        xg, yg = x.cuda().requires_grad_(True), table.cuda().requires_grad_(True)
        loss = MemoryEfficientDistillLoss(1.0, True)(xg, yg, t.cuda(), logits.cuda())
        loss.backward()
        torch.cuda.synchronize()
    finally:
        _lib.check(_lib.load().meclip_debug_set_blocking(0, 0))
    wx, wy, bx, by = oracle.distill_grad(x, table, t, logits, 1.0, torch.full((n,), 1.0 / n), (torch.bfloat16,) * 2)
    _inside(xg.grad, wx, bx, "dx")
    _inside(yg.grad, wy, by, "dtable")


def test_capture_streams_and_repeats():
    """A captured step replays on new data; a side stream and repeats give the same bits."""
    from memoryefficientclip_b200 import MemoryEfficientDistillLoss, token_log_probs
    n, v, d, k = 1030, 2000, 256, 4
    x, table, tokens, g = _pair(n, v, d, torch.bfloat16, 31)
    t, logits = _teacher(n, v, k, g)
    xg, yg, t, logits, tok = x.cuda().requires_grad_(True), table.cuda().requires_grad_(True), t.cuda(), logits.cuda(), tokens.cuda()
    mod = MemoryEfficientDistillLoss(1.0, True)

    def step():
        loss = mod(xg, yg, t, logits)
        s = token_log_probs(xg, yg, tok, top_k=2)
        dx, dy = torch.autograd.grad([loss, s.log_probs.sum(), s.entropy.sum()], [xg, yg])
        return loss, s.log_probs, s.top_tokens, dx, dy

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            first = [o.detach().clone() for o in step()]
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, step()):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    x2, _, _, _ = _pair(n, v, d, torch.bfloat16, 32)
    with torch.no_grad():
        xg.copy_(x2)
    graph.replay()
    torch.cuda.synchronize()
    replayed = [o.detach().clone() for o in out]
    for a, b in zip(replayed, step()):
        assert torch.equal(a, b)


def test_entry_points_stay_inside_their_outputs():
    """Rows behind the last one keep what was in them."""
    from memoryefficientclip_b200 import ops
    n, v, d = 37, 515, 64
    x, table, tokens, _ = _pair(n, v, d, torch.bfloat16, 6)
    guard = torch.full((n + 8, d), 7.0, dtype=torch.bfloat16, device="cuda")
    guard[:n] = x.cuda()
    with torch.no_grad():
        a = ops.token_log_probs(guard[:n], table.cuda(), tokens.cuda(), 1.0, 2)
        guard[n:] = float("nan")
        b = ops.token_log_probs(guard[:n], table.cuda(), tokens.cuda(), 1.0, 2)
    for p, q in zip(a[:4], b[:4]):
        assert torch.equal(p, q)
    ops.check_status()


def test_more_rows_than_a_block_of_them():
    """Rows beyond 16384 go through the passes in blocks: scores, loss over all of them, gradients."""
    from memoryefficientclip_b200 import MemoryEfficientDistillLoss, token_log_probs
    n, v, d = 16384 + 77, 90, 24
    x, table, tokens, g = _pair(n, v, d, torch.bfloat16, 3, 4.0)
    t, logits = torch.randint(-1, v, (n, 3), generator=g), torch.randn(n, 3, generator=g)
    xg, yg = x.cuda().requires_grad_(True), table.cuda().requires_grad_(True)
    got = token_log_probs(xg, yg, tokens.cuda(), top_k=2)
    want = oracle.token_log_probs(x, table, tokens[:, None], 1.0, 2)
    _inside(got.log_probs, want["log_probs"][:, 0], want["err_lp"], "log_probs")
    assert torch.equal(got.top_tokens.cpu(), want["top_tokens"])
    loss = MemoryEfficientDistillLoss(1.0, True)(xg, yg, t.cuda(), logits.cuda())
    kl, has, err = oracle.distill(x, table, t, logits, 1.0)
    count = has.sum().double()
    _inside(loss, kl.sum() / count, err.sum() / count + 2 * oracle.ULP * kl.sum() / count, "loss")
    dx, dy = torch.autograd.grad(loss, [xg, yg])
    wx, wy, bx, by = oracle.distill_grad(x, table, t, logits, 1.0, torch.ones(n) / count, (torch.bfloat16,) * 2)
    _inside(dx, wx, bx, "dx")
    _inside(dy, wy, by, "dtable")


@pytest.mark.parametrize("n", [40, 300, 1100])
@pytest.mark.parametrize("k", [1, 2, 3])
def test_few_entries_and_the_same_one_twice(n, k):
    """One or two entries are added by the tile pass, three by the row kernel; each with repeats and padding."""
    from memoryefficientclip_b200 import MemoryEfficientDistillLoss
    v, d = 777, 264
    x, table, tokens, g = _pair(n, v, d, torch.bfloat16, n + k)
    t = torch.stack([tokens] * k, 1)
    t[n // 2:, -1] = (t[n // 2:, -1] + 1) % v
    t[::7, 0] = -1
    t[1] = -1
    logits = torch.randn(n, k, generator=g)
    xg, yg = x.cuda().requires_grad_(True), table.cuda().requires_grad_(True)
    loss = MemoryEfficientDistillLoss(0.9, True, reduction="sum")(xg, yg, t.cuda(), logits.cuda())
    dx, dy = torch.autograd.grad(loss, [xg, yg])
    wx, wy, bx, by = oracle.distill_grad(x, table, t, logits, 0.9, torch.ones(n), (torch.bfloat16,) * 2)
    _inside(dx, wx, bx, "dx")
    _inside(dy, wy, by, "dtable")


def test_two_calls_on_two_streams():
    """Calls that overlap have workspaces of their own."""
    from memoryefficientclip_b200 import token_log_probs
    a = _pair(700, 3000, 256, torch.bfloat16, 41)
    b = _pair(900, 2000, 512, torch.bfloat16, 42)
    want = [token_log_probs(x.cuda(), t.cuda(), k.cuda(), top_k=4) for x, t, k, _ in (a, b)]
    data = [(x.cuda(), t.cuda(), k.cuda()) for x, t, k, _ in (a, b)]
    streams = [torch.cuda.Stream() for _ in data]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, d in zip(streams, data):
            with torch.cuda.stream(s):
                got.append(token_log_probs(*d, top_k=4))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        for p, q in zip(g, want[i % 2]):
            assert torch.equal(p, q)


def test_large_and_small_magnitudes():
    """Features and tables far from 1: the fp16 operands of the gradient are scaled, nothing over- or underflows."""
    from memoryefficientclip_b200 import MemoryEfficientDistillLoss
    n, v, d, k = 400, 600, 264, 4
    for size_x, size_y, weight in ((1e5, 1e-5, 1.0), (1e-6, 1e6, 1e-6), (1e4, 1e4, 1e8)):
        x, table, _tokens, g = _pair(n, v, d, torch.bfloat16, 51)
        x, table = (x.float() * size_x).bfloat16(), (table.float() * size_y).bfloat16()
        t, logits = _teacher(n, v, k, g)
        temp = size_x * size_y
        xg, yg = x.cuda().requires_grad_(True), table.cuda().requires_grad_(True)
        loss = MemoryEfficientDistillLoss(temp, True, reduction="sum")(xg, yg, t.cuda(), logits.cuda())
        dx, dy = torch.autograd.grad(loss, [xg, yg], torch.tensor(weight).cuda())
        wx, wy, bx, by = oracle.distill_grad(x, table, t, logits, temp, torch.full((n,), weight), (torch.bfloat16,) * 2)
        _inside(dx, wx, bx, "dx")
        _inside(dy, wy, by, "dtable")


@pytest.mark.parametrize("switch", ["MECLIP_NO_TRANSPOSE=1", "MECLIP_DUAL=0", "MECLIP_PAIR=0", "MECLIP_SERIAL=1"])
def test_gradients_under_every_switch(switch):
    """The library's switches are read once per process: the gradient tests again, in a child."""
    name, value = switch.split("=")
    out = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-m", "gpu", "-p", "no:cacheprovider", __file__,
                          "-k", "test_score_gradients or test_distillation_of_two_towers"],
                         env=dict(os.environ, **{name: value}), capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout[-2000:]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_broadcast_and_overlapping_rows(dtype):
    """One row expanded to many, rows that overlap, and a single row of whatever pitch, against contiguous copies."""
    from memoryefficientclip_b200 import token_log_probs, MemoryEfficientDistillLoss
    n, v, d = 70, 333, 64
    x, table, tokens, g = _pair(n, v, d, dtype, 8)
    x, table, tokens = x.cuda(), table.cuda(), tokens.cuda()
    flat = table.reshape(-1)
    cases = [(x[:1].expand(n, d), table, tokens), (x, table[:1].expand(v, d), tokens),
             (x, flat.as_strided((v, d), (8, 1)), tokens), (x[:1].as_strided((1, d), (0, 1)), table, tokens[:1]),
             (x, table[:1].as_strided((1, d), (8, 1)), tokens.clamp(max=0))]
    for a, b, t in cases:
        for got, want in zip(token_log_probs(a, b, t, top_k=1), token_log_probs(a.contiguous().clone(), b.contiguous().clone(), t, top_k=1)):
            assert torch.equal(got, want)
        logits = torch.zeros(t.shape[0], 1, device="cuda")
        for normalized in (True, False):
            loss = MemoryEfficientDistillLoss(1.0, normalized)
            assert torch.equal(loss(a, b, t[:, None], logits), loss(a.contiguous().clone(), b.contiguous().clone(), t[:, None], logits))
    one = x[:1].clone().requires_grad_(True)            # the gradient of a broadcast input is the sum over its copies
    token_log_probs(one.expand(n, d), table, tokens).log_probs.sum().backward()
    many = x[:1].expand(n, d).clone().requires_grad_(True)
    token_log_probs(many, table, tokens).log_probs.sum().backward()
    assert torch.equal(one.grad, many.grad.sum(0, keepdim=True))


def test_second_derivatives_are_refused():
    from memoryefficientclip_b200 import token_log_probs, MemoryEfficientDistillLoss
    x, table, tokens, _g = _pair(20, 50, 64, torch.float32, 8)
    x, table, tokens = x.cuda().requires_grad_(True), table.cuda(), tokens.cuda()
    w = torch.ones((), device="cuda", requires_grad=True)
    for out in (token_log_probs(x, table, tokens).log_probs.sum() * w,
                MemoryEfficientDistillLoss(1.0)(x, table, tokens[:, None], torch.zeros(20, 1, device="cuda")) * w):
        (dx,) = torch.autograd.grad(out, x, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            dx.sum().backward()


@pytest.mark.parametrize("n", [3, 260])
def test_offsets_past_32_bits(n):
    """A table of 2^31 elements and more than 2^32 bytes.  All rows but a few are zero, so that the oracle needs only
    those: V - R scores of exactly 0."""
    from memoryefficientclip_b200 import embed_tokens, token_log_probs
    v, d, r = 2_100_000, 1024, 400
    g = torch.Generator().manual_seed(n)
    where = torch.cat([torch.tensor([0, v - 1, v - 2, 2 ** 31 // d, 2 ** 31 // d - 1]), torch.randint(0, v, (r,), generator=g)]).unique()
    rows = (torch.randn(len(where), d, generator=g) / math.sqrt(d)).bfloat16()
    pick = torch.randint(0, len(where), (n,), generator=g)
    pick[0] = len(where) - 1
    x = (2.0 * torch.randn(n, d, generator=g) + 20.0 * rows.float()[pick]).bfloat16()
    table = torch.zeros(v, d, dtype=torch.bfloat16, device="cuda")
    table[where.cuda()] = rows.cuda()
    table.requires_grad_(True)
    xg, tokens = x.cuda().requires_grad_(True), where[pick].cuda()
    got = token_log_probs(xg, table, tokens, top_k=1)
    z, err = oracle.scores(x, rows, 1.0)
    zeros = float(v - len(where))
    lse = torch.logsumexp(torch.cat([z, torch.full((n, 1), math.log(zeros))], 1), 1)
    lp = z.gather(1, pick[:, None])[:, 0] - lse
    _inside(got.log_probs, lp, 2 * err, "log_probs")
    assert torch.equal(got.top_tokens[:, 0].cpu(), where[z.argmax(1)])
    dx, dt = torch.autograd.grad(got.log_probs.sum(), [xg, table])
    p = (z - lse[:, None]).exp()
    one = torch.zeros_like(p).scatter_(1, pick[:, None], 1.0)
    wx, wy, bx, by = oracle._gradients(x, rows, 1.0, -p, one, p, (torch.bfloat16,) * 2, 0.0)
    # the zero rows' part of dX is zero; the panel's scaled fp16 form cuts coefficients below 2^-24 of the largest bound
    cut = 2.0 ** -24 * 2.0
    _inside(dx, wx, bx + cut * rows.double().abs().sum(0), "dx")
    _inside(dt[where.cuda()], wy, by + cut * x.double().abs().sum(0), "dtable")
    others = torch.randint(0, v, (2000,), generator=g)
    others = others[~torch.isin(others, where)]
    w0 = -(torch.exp(-lse)[:, None] * x.double()).sum(0)
    b0 = (torch.exp(-lse)[:, None] * (2.0 ** -8 + 2 * err[:, None] + 16 * oracle.ULP) * x.double().abs()).sum(0)
    b0 = b0 + 2.0 ** -8 * (w0.abs() + b0) + cut * x.double().abs().sum(0)
    worst = ((dt[others.cuda()].double().cpu() - w0).abs() / b0).max().item()
    assert worst <= 1.0, worst
    del dx, dt
    out = embed_tokens(tokens, table, 2.0)
    assert torch.equal(out.detach().float().cpu(), 2.0 * rows.float()[pick])
    go = torch.randn(n, d, generator=g).bfloat16()
    (dt,) = torch.autograd.grad(out, table, go.cuda())
    want = torch.zeros(len(where), d, dtype=torch.float64).index_add_(0, pick, 2.0 * go.double())
    size = torch.zeros(len(where), d, dtype=torch.float64).index_add_(0, pick, 2.0 * go.double().abs())
    assert ((dt[where.cuda()].double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + (n + 2) * 2.0 ** -23 * size).all()
    assert dt[others.cuda()].abs().max().item() == 0 and int(torch.count_nonzero(dt.abs().amax(1))) == len(pick.unique())


@pytest.mark.parametrize("n,v,d", [(1, 1, 8), (2, 31, 8), (1, 33, 264), (2, 95, 250), (1, 14209, 256), (2, 50001, 768),
                                   (1, 300, 16384), (2, 300, 16392), (1, 120000, 72)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_one_and_two_rows(n, v, d, dtype):
    """A token at a time: tables that end inside a chunk, of fewer chunks than blocks and more, widths up to the kernel's
    limit and behind it; rows around the operands hold what would show."""
    from memoryefficientclip_b200 import token_log_probs
    x, table, tokens, g = _pair(n, v, d, dtype, n + v)
    xg = torch.full((n + 2, d), float("nan"), dtype=dtype, device="cuda")
    xg[1:n + 1] = x.cuda()
    yg = torch.full((v + 33, d), float("nan"), dtype=dtype, device="cuda")
    yg[:v] = table.cuda()
    top_k = min(5, v)
    got = token_log_probs(xg[1:n + 1], yg[:v], tokens.cuda(), top_k=top_k)
    want = oracle.token_log_probs(*_operands(x, table), tokens[:, None], 1.0, top_k)
    _inside(got.log_probs, want["log_probs"][:, 0], want["err_lp"], "log_probs")
    _inside(got.entropy, want["entropy"], want["err_entropy"], "entropy")
    assert torch.equal(got.top_tokens.cpu(), want["top_tokens"])
    _inside(got.top_log_probs, want["top_log_probs"], want["err_lp"][:, None], "top_log_probs")
    bad = x.clone()
    bad[0, d // 2] = float("nan")
    out = token_log_probs(bad.cuda(), table.cuda(), tokens.cuda())
    assert out.log_probs[0].isnan() and out.entropy[0].isnan() and (n == 1 or torch.isfinite(out.log_probs[1]))


@pytest.mark.parametrize("n,v,top_k", [(1, 256, 8), (3, 1000, 32), (1, 1000, 31), (200, 257, 9), (400, 600, 32), (2, 33, 32),
                                       (1, 2047, 32), (300, 64, 32)])
def test_alternatives_of_small_tables(n, v, top_k):
    """So few chunks that most columns are candidates, some of them equal."""
    from memoryefficientclip_b200 import token_log_probs
    x, table, tokens, g = _pair(n, v, 72, torch.bfloat16, v)
    table[v // 2:v // 2 + 7] = table[3]
    got = token_log_probs(x.cuda(), table.cuda(), tokens.cuda(), top_k=top_k)
    want = oracle.token_log_probs(x, table, tokens[:, None], 1.0, top_k)
    assert torch.equal(got.top_tokens.cpu(), want["top_tokens"])
    _inside(got.top_log_probs, want["top_log_probs"], want["err_lp"][:, None], "top_log_probs")


def _c_grad(n, v, d, operands, tokens, per_row, saved, entropy, g, h, dx, dt, mode):
    """meclip_token_log_probs_grad as a C caller makes the call."""
    from memoryefficientclip_b200 import _lib, ops
    x, table = operands
    lib = _lib.load()
    size = lib.meclip_vocab_grad_workspace_bytes(0, n, v, d)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    lse = saved.data_ptr()
    _lib.check(lib.meclip_token_log_probs_grad(
        x.data_ptr(), table.data_ptr(), 0, n, v, d, x.stride(0), table.stride(0), 1.0, ops._ptr(tokens), per_row, lse,
        ops._ptr(entropy), lse + 4 * n, ops._ptr(g), ops._ptr(h), ops._ptr(dx), mode, d, ops._ptr(dt), mode, d,
        ws.data_ptr(), size, ops.status_word(x.device).data_ptr(), torch.cuda.current_stream().cuda_stream))


@pytest.mark.parametrize("n,v,d", [(1, 700, 64), (40, 4099, 264), (300, 2051, 264), (1100, 999, 72), (1100, 2051, 512)])
def test_c_calls_without_tokens_and_with_accumulation(n, v, d):
    """No token per row (entropy and alternatives only), gradients that are added to what is there, none at all."""
    from memoryefficientclip_b200 import _lib, ops
    x, table, tokens, gen = _pair(n, v, d, torch.bfloat16, n)
    xg, yg, tg = x.cuda(), table.cuda(), tokens.cuda()
    lib = _lib.load()
    size = lib.meclip_vocab_workspace_bytes(n, v, 2)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    entropy, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    top_lp, top = torch.empty(n, 2, device="cuda"), torch.empty(n, 2, dtype=torch.int64, device="cuda")
    _lib.check(lib.meclip_token_log_probs(
        xg.data_ptr(), yg.data_ptr(), 0, n, v, d, d, d, 1.0, None, 0, None, entropy.data_ptr(), 2, top_lp.data_ptr(),
        top.data_ptr(), lse.data_ptr(), None, ws.data_ptr(), size, None, torch.cuda.current_stream().cuda_stream))
    want = oracle.token_log_probs(x, table, tokens[:, None], 1.0, 2)
    _inside(entropy, want["entropy"], want["err_entropy"], "entropy")
    assert torch.equal(top.cpu(), want["top_tokens"])
    h = torch.randn(n, generator=gen)
    dx, dt = torch.empty(n, d, device="cuda"), torch.empty(v, d, device="cuda")
    _c_grad(n, v, d, (xg, yg), None, 0, lse, entropy, None, h.cuda(), dx, dt, ops._MODE[torch.float32])
    wx, wy, bx, by = oracle.token_log_probs_grad(x, table, tokens[:, None], 1.0, torch.zeros(n, 1), h, (torch.float32,) * 2)
    _inside(dx, wx, bx, "dx")
    _inside(dt, wy, by, "dtable")
    _c_grad(n, v, d, (xg, yg), None, 0, lse, entropy, None, None, dx, dt, ops._MODE[torch.float32])
    assert dx.abs().max().item() == 0 and dt.abs().max().item() == 0
    # accumulation: the same gradient twice onto a start value
    lp, ent, _a, _b, saved = ops.token_log_probs(xg, yg, tg, 1.0, 0, True, ops.status_word(xg.device))
    g = torch.randn(n, 1, generator=gen)
    ax, at = torch.full((n, d), 0.5, device="cuda"), torch.full((v, d), -0.25, device="cuda")
    for _ in range(2):
        _c_grad(n, v, d, (xg, yg), tg, 1, saved, ent, g.cuda(), h.cuda(), ax, at, 2)
    wx, wy, bx, by = oracle.token_log_probs_grad(x, table, tokens[:, None], 1.0, g, h, (torch.float32,) * 2)
    _inside(ax, 0.5 + 2 * wx, 2 * bx + oracle.ULP * (1 + 2 * wx.abs()), "dx")
    _inside(at, -0.25 + 2 * wy, 2 * by + oracle.ULP * (1 + 2 * wy.abs()), "dtable")
    ops.check_status()


def test_two_threads_at_once():
    """Forward and backward from two threads, each on a stream of its own."""
    import threading
    from memoryefficientclip_b200 import embed_tokens, token_log_probs
    x, table, tokens, _g = _pair(1300, 3001, 264, torch.bfloat16, 2)
    x, table, tokens = x.cuda(), table.cuda(), tokens.cuda()

    def step():
        xl, tl = x.clone().requires_grad_(True), table.clone().requires_grad_(True)
        out = token_log_probs(xl + embed_tokens(tokens, tl, 0.1), tl, tokens, top_k=3)
        return [out.log_probs.detach(), out.top_tokens, *torch.autograd.grad(out.log_probs.sum() - out.entropy.sum(), [xl, tl])]

    want = step()
    torch.cuda.synchronize()
    found, failed = {}, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    found[i] = step()
                torch.cuda.current_stream().synchronize()
        except Exception as e:          # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for i in range(2):
        for a, b in zip(found[i], want):
            assert torch.equal(a, b)


def test_two_threads_with_different_sizes():
    """Calls that want different amounts of shared memory from the same kernels."""
    import threading
    from memoryefficientclip_b200 import embed_tokens, token_log_probs
    x, table, tokens, _g = _pair(400, 40000, 72, torch.bfloat16, 5)
    x, table, tokens = x.cuda(), table.cuda(), tokens.cuda()
    many = torch.stack([tokens] * 256, 1)
    calls = [lambda: token_log_probs(x, table[:600], tokens, top_k=32), lambda: token_log_probs(x, table, many, top_k=1),
             lambda: token_log_probs(x[:1], table, many[:1], top_k=32), lambda: token_log_probs(x[:1, :64], table[:, :64], tokens[:1])]
    tables = [table.clone().requires_grad_(True), table[:100].clone().requires_grad_(True)]
    calls += [lambda t=t: torch.autograd.grad(embed_tokens(tokens % t.shape[0], t).float().sum(), t) for t in tables]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    failed = []

    def work(which):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    for a, b in zip(calls[which](), want[which]):
                        # (tokens behind the smaller table are NaN on both sides)
                        assert a is b or torch.allclose(a, b, rtol=0, atol=0, equal_nan=True)
        except BaseException as e:      # noqa: BLE001
            failed.append((which, e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
