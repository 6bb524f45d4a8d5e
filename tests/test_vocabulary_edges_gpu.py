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


@pytest.mark.parametrize("switch", ["MECLIP_WIDE=1", "MECLIP_WIDE=1 MECLIP_SERIAL=1", "MECLIP_WIDE=1 MECLIP_NO_TRANSPOSE=1",
                                    "MECLIP_PAIR=1", "MECLIP_STATIC_SCHED=1"])
def test_gradients_under_the_other_switches(switch):
    """Switches are read once per process: the widths below in a child, with tiles of more than 256 columns among them."""
    out = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-m", "gpu", "-p", "no:cacheprovider", __file__,
                          "-k", "test_gradients_of_wide_features"],
                         env=dict(os.environ, **dict(s.split("=") for s in switch.split())), capture_output=True, text=True,
                         timeout=300)
    assert out.returncode == 0, out.stdout[-2000:]


@pytest.mark.parametrize("n,v,d", [(300, 2100, 512), (257, 5000, 1152), (1100, 3000, 520), (60, 4099, 768)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sides", ["both", "features", "table"])
def test_gradients_of_wide_features(n, v, d, dtype, sides):
    from memoryefficientclip_b200 import token_log_probs
    x, table, tokens, g = _pair(n, v, d, dtype, n + v, bump=6.0)
    g_lp, g_h = torch.randn(n, generator=g), torch.randn(n, generator=g) * 0.3
    xg, yg = x.cuda().requires_grad_(sides != "table"), table.cuda().requires_grad_(sides != "features")
    got = token_log_probs(xg, yg, tokens.cuda(), temperature=1.3)
    (got.log_probs * g_lp.cuda() + got.entropy * g_h.cuda()).sum().backward()
    wx, wy, bx, by = oracle.token_log_probs_grad(x, table, tokens[:, None], 1.3, g_lp[:, None], g_h, (dtype, dtype))
    if sides != "table":
        _inside(xg.grad, wx, bx, "dx")
    if sides != "features":
        _inside(yg.grad, wy, by, "dtable")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_forward_mode_derivatives_are_refused(dtype):
    """There is none of these operators; a tangent is never dropped, with or without grad mode."""
    import torch.autograd.forward_ad as fwd
    from memoryefficientclip_b200 import MemoryEfficientDistillLoss, embed_tokens, token_log_probs
    x, table, tokens, _g = _pair(20, 50, 64, dtype, 8)
    x, table, tokens = x.cuda(), table.cuda(), tokens.cuda()
    want = token_log_probs(x, table, tokens, top_k=2), embed_tokens(tokens, table)
    distill = MemoryEfficientDistillLoss(1.0)
    logits = torch.zeros(20, 1, device="cuda")
    with fwd.dual_level():
        dual_x, dual_t = fwd.make_dual(x, torch.ones_like(x)), fwd.make_dual(table, torch.ones_like(table))
        for grad_mode in (True, False):
            with torch.set_grad_enabled(grad_mode):
                for call in (lambda: token_log_probs(dual_x, table, tokens), lambda: token_log_probs(x, dual_t, tokens, top_k=1),
                             lambda: embed_tokens(tokens, dual_t), lambda: distill(dual_x, table, tokens[:, None], logits),
                             lambda: distill(x, dual_t, tokens[:, None], logits)):
                    with pytest.raises((RuntimeError, NotImplementedError)):
                        call()
                # plain inputs are answered as ever while such a level is open
                for a, b in zip(token_log_probs(x, table, tokens, top_k=2), want[0]):
                    assert torch.equal(a, b)
                assert torch.equal(embed_tokens(tokens, table), want[1])


def _near_ties(n, v, members, seed):
    """Features and a table of whole numbers (every product and sum is exact in 64 bits): the rows of `members` score the same
    but for steps of 2^-26, far below what an fp32 sum of this size holds, in a random order; all others score far less."""
    g = torch.Generator().manual_seed(seed)
    d = 64
    table = torch.zeros(v, d)
    x = torch.zeros(n, d)
    x[:, :40] = torch.randint(4, 12, (n, 40), generator=g).float()
    place = torch.randperm(len(members), generator=g)
    table[members, :40] = 8.0
    table[members, 40], table[members, 41] = (place // 64).float(), (place % 64).float()
    x[:, 40], x[:, 41] = 2.0 ** -20, 2.0 ** -26
    return x.bfloat16(), table.bfloat16()


@pytest.mark.parametrize("top_k", [1, 2, 8, 32])
@pytest.mark.parametrize("n", [1, 2, 40, 400])
@pytest.mark.parametrize("which", ["all", "two of a chunk in few chunks", "two of a chunk in all chunks", "the last chunks"])
def test_near_ties_in_many_chunks(n, top_k, which):
    """The order is that of exact scores, however many columns are closer than the tile pass can tell apart."""
    from memoryefficientclip_b200 import token_log_probs
    v = 4001
    every = torch.arange(v)
    members = {"all": every, "two of a chunk in few chunks": every[(every % 32 < 2) & (every // 32 % 16 == 5)],
               "two of a chunk in all chunks": every[every % 32 < 2], "the last chunks": every[v - 100:]}[which]
    x, table = _near_ties(n, v, members, top_k + n)
    if len(members) < top_k:
        pytest.skip("fewer of them than alternatives")
    z = x.double() @ table.double().T
    want = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :top_k]
    got = token_log_probs(x.cuda(), table.cuda(), want[:, 0].contiguous().cuda(), top_k=top_k)
    assert torch.equal(got.top_tokens.cpu(), want)
    lp = torch.log_softmax(z, 1).gather(1, want)
    _z, err = oracle.scores(x, table, 1.0)
    _inside(got.top_log_probs, lp, 2 * err[:, None], "top_log_probs")


def test_crowds_of_equal_scores_stay_cheap():
    """Rows of zeros tie everywhere: the first tokens win, and the row does not look at every column to find that out."""
    from memoryefficientclip_b200 import token_log_probs
    x, table, tokens, _g = _pair(700, 20000, 128, torch.bfloat16, 4)
    x[::3] = 0
    got = token_log_probs(x.cuda(), table.cuda(), tokens.cuda(), top_k=9)
    assert torch.equal(got.top_tokens[::3].cpu(), torch.arange(9).expand(234, 9))
    _inside(got.top_log_probs[::3], torch.full((234, 9), -math.log(20000), dtype=torch.float64),
            torch.full((), 8 * oracle.ULP * math.log(20000), dtype=torch.float64), "top_log_probs")


@pytest.mark.parametrize("n,v,d", [(40, 999, 64), (300, 2051, 264), (1100, 2051, 264), (1100, 999, 72)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("frozen", [True, False])
def test_rows_that_are_not_finite_leave_the_others_alone(n, v, d, dtype, frozen):
    """An infinite incoming gradient, eight neighbouring rows of NaN: they show in their own rows (and in the table's
    gradient), the other rows are as exact as without them."""
    from memoryefficientclip_b200 import token_log_probs
    x, table, tokens, g = _pair(n, v, d, dtype, n + d, bump=5.0)
    g_lp, g_h = 1e-4 * torch.randn(n, generator=g), 1e-5 * torch.randn(n, generator=g)
    bad = torch.zeros(n, dtype=torch.bool)
    g_lp[3], bad[3] = float("inf"), True
    g_h[17], bad[17] = float("-inf"), True
    g_lp[24:32], bad[24:32] = float("nan"), True
    xg, yg = x.cuda().requires_grad_(True), table.cuda().requires_grad_(not frozen)
    got = token_log_probs(xg, yg, tokens.cuda())
    torch.autograd.backward([got.log_probs, got.entropy], [g_lp.cuda(), g_h.cuda()])
    xo, yo = (x, table) if dtype == torch.float16 else (x.bfloat16(), table.bfloat16())
    wx, _wy, bx, _by = oracle.token_log_probs_grad(xo[~bad], yo, tokens[~bad][:, None], 1.0, g_lp[~bad][:, None], g_h[~bad],
                                                   (dtype, dtype))
    _inside(xg.grad[~bad.cuda()], wx, bx, "dx")
    assert not torch.isfinite(xg.grad[bad.cuda()]).any(1).any()
    assert frozen or not torch.isfinite(yg.grad).any()


@pytest.mark.parametrize("n,v,d", [(40, 999, 64), (300, 2051, 264), (1100, 2051, 264), (1100, 999, 72), (700, 40, 8)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("per_row", [1, 4])
def test_rows_of_very_different_weights(n, v, d, dtype, per_row):
    """A row's gradient is as exact as if it were alone, whatever the other rows weigh: 2^0 to 2^-80 and none at all."""
    from memoryefficientclip_b200 import ops
    x, table, tokens, g = _pair(n, v, d, dtype, n + v, bump=4.0)
    many = torch.stack([tokens] + [torch.randint(-1, v, (n,), generator=g) for _ in range(per_row - 1)], 1)
    weight = 2.0 ** -torch.randint(0, 81, (n,), generator=g).double()
    weight[::11] = 0
    weight[5] = 1.0
    g_lp, g_h = torch.randn(n, per_row, generator=g), torch.randn(n, generator=g) * 0.3
    xg, yg, tk = x.cuda(), table.cuda(), many.cuda()
    status = ops.status_word(xg.device)
    _lp, entropy, _a, _b, saved = ops.token_log_probs(xg, yg, tk, 1.0, 0, True, status)
    f32 = torch.float32
    wg, wh = (g_lp.double() * weight[:, None]).float(), (g_h.double() * weight).float()
    for sides in ((True, True), (True, False), (False, True)):
        dx, dt = ops.token_log_probs_grad(xg, yg, tk, 1.0, saved, entropy, wg.cuda(), wh.cuda(), f32, f32, *sides, status)
        wx, _wy, bx, _by = oracle.token_log_probs_grad(x, table, many, 1.0, g_lp, g_h, (f32, f32))
        if dx is not None:
            _inside(dx, weight[:, None] * wx, weight[:, None] * bx + torch.finfo(f32).tiny, "dx")
            assert not dx[::11].any()
        _wx, wy, _bx, by = oracle.token_log_probs_grad(x, table, many, 1.0, wg, wh, (f32, f32))
        if dt is not None:
            _inside(dt, wy, by, "dtable")


@pytest.mark.parametrize("n,v,d", [(300, 700, 264), (1100, 700, 264)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_distillation_rows_of_very_different_weights(n, v, d, dtype):
    """The same with a weight for each row's loss, and features whose lengths differ as much the other way round, so that
    every row has a say in the table's gradient."""
    from memoryefficientclip_b200 import ops
    x, table, _tokens, g = _pair(n, v, d, dtype, 3)
    shift = torch.randint(0, 11, (n,), generator=g)
    x = (x.double() * 2.0 ** -shift[:, None].double()).to(dtype)
    t, logits = _teacher(n, v, 5, g)
    weight = (2.0 ** shift.double()).float()
    xg, yg, tg = x.cuda(), table.cuda(), t.cuda()
    status = ops.status_word(xg.device)
    _loss, saved = ops.distill_forward(xg, yg, tg, logits.cuda(), 1.0, 1.0, "none", status)
    dx, dt = ops.distill_backward(xg, yg, tg, 1.0, saved, weight.cuda(), torch.float32, torch.float32, status=status)
    wx, wy, bx, by = oracle.distill_grad(x, table, t, logits, 1.0, weight, (torch.float32,) * 2)
    _inside(dx, wx, bx, "dx")
    _inside(dt, wy, by, "dtable")


@pytest.mark.parametrize("size_x,size_g", [(2.0 ** 60, 2.0 ** -50), (2.0 ** -60, 2.0 ** 50), (2.0 ** -110, 1.0),
                                           (1.0, 2.0 ** -100), (1.0, 2.0 ** 100), (2.0 ** 50, 2.0 ** 50),
                                           (2.0 ** -50, 2.0 ** -60)])
@pytest.mark.parametrize("n", [300, 1100])
def test_magnitudes_at_the_ends_of_the_range(n, size_x, size_g):
    """Powers of two on the features and the incoming gradients come out again as powers of two."""
    from memoryefficientclip_b200 import ops
    v, d, f32 = 500, 264, torch.float32
    x, table, tokens, g = _pair(n, v, d, torch.bfloat16, 7)
    g_lp = torch.randn(n, generator=g)
    grads = []
    for sx, sg in ((1.0, 1.0), (size_x, size_g)):
        xg, yg, tk = (x.double() * sx).bfloat16().cuda(), (table.double() / sx).bfloat16().cuda(), tokens.cuda()
        assert torch.isfinite(yg).all() and (yg.double() * sx).cpu().equal(table.double())
        _lp, entropy, _a, _b, saved = ops.token_log_probs(xg, yg, tk, 1.0, 0, True, None)
        dx, dt = ops.token_log_probs_grad(xg, yg, tk, 1.0, saved, entropy, (g_lp.double() * sg).float().cuda(), None, f32, f32)
        grads.append((dx.double() * sx / sg, dt.double() / sx / sg))
    for got, want in zip(grads[1], grads[0]):
        # (the smallest results are fp32's subnormal numbers: half of 2^-149 over 2^-110 for every part of a sum and its scale)
        assert ((got - want).abs() <= 4 * oracle.ULP * want.abs() + 40 * 2.0 ** -150 / 2.0 ** -110).all()


@pytest.mark.parametrize("n,v,d", [(1, 40, 64), (5, 1000, 64), (130, 257, 104), (300, 4099, 512), (1100, 2051, 264),
                                   (64, 9000, 96), (1500, 700, 1152), (2000, 333, 30)])
def test_fp16_gradients_keep_their_bits(n, v, d):
    """Two fp16 inputs are contracted as they are: no operand is rounded, and an fp16 coefficient keeps 11 bits."""
    from memoryefficientclip_b200 import MemoryEfficientDistillLoss, token_log_probs
    half = torch.float16
    x, table, tokens, g = _pair(n, v, d, half, n + v, bump=6.0)
    many = torch.stack([tokens, torch.randint(-1, v, (n,), generator=g), tokens], 1)
    g_lp, g_h = torch.randn(n, 3, generator=g), torch.randn(n, generator=g) * 0.3
    xg, yg = x.cuda().requires_grad_(True), table.cuda().requires_grad_(True)
    got = token_log_probs(xg, yg, many.cuda(), temperature=1.3)
    dx, dy = torch.autograd.grad([got.log_probs, got.entropy], [xg, yg], [g_lp.cuda(), g_h.cuda()])
    wx, wy, bx, by = oracle.token_log_probs_grad(x, table, many, 1.3, g_lp, g_h, (half, half))
    _inside(dx, wx, bx, "dx")
    _inside(dy, wy, by, "dtable")
    t, logits = _teacher(n, v, 6, g)
    loss = MemoryEfficientDistillLoss(0.8, normalized_inputs=True, reduction="none")(xg, yg, t.cuda(), logits.cuda())
    weight = torch.randn(n, generator=g)
    dx, dy = torch.autograd.grad(loss, [xg, yg], weight.cuda())
    wx, wy, bx, by = oracle.distill_grad(x, table, t, logits, 0.8, weight, (half, half))
    _inside(dx, wx, bx, "dx")
    _inside(dy, wy, by, "dtable")


@pytest.mark.parametrize("n", [3, 260])
def test_gradient_of_rows_past_32_bits(n):
    """A table of 2^31 elements, all but a few rows of which are zero: the gradient of those rows is far above what the
    comparison allows, so that none at all would be noticed."""
    from memoryefficientclip_b200 import token_log_probs
    v, d = 2_100_000, 1024
    g = torch.Generator().manual_seed(n)
    where = torch.cat([torch.tensor([0, v - 1, v - 2, 2 ** 31 // d, 2 ** 31 // d - 1]), torch.randint(0, v, (40,), generator=g)]).unique()
    rows = (torch.randn(len(where), d, generator=g) / math.sqrt(d)).bfloat16()
    pick = torch.randint(0, len(where), (n,), generator=g)
    # features that agree on a direction, so that the zero rows' sums do not cancel
    x = (torch.randn(d, generator=g) + 0.5 * torch.randn(n, d, generator=g)).bfloat16()
    table = torch.zeros(v, d, dtype=torch.bfloat16, device="cuda")
    table[where.cuda()] = rows.cuda()
    xg, table = x.cuda().requires_grad_(True), table.requires_grad_(True)
    got = token_log_probs(xg, table, where[pick].cuda())
    z, err = oracle.scores(x, rows, 1.0)
    zeros = torch.full((n, 1), math.log(float(v - len(where))), dtype=torch.float64)
    lse = torch.logsumexp(torch.cat([z, zeros], 1), 1)
    _dx, dt = torch.autograd.grad(got.log_probs.sum(), [xg, table])
    p0 = torch.exp(-lse)[:, None]
    want = -(p0 * x.double()).sum(0)
    # a coefficient's 2^-11 (two bf16 panels: less) and its floor, 2^-39 of the bound 2; the score's error; the contraction's
    # cuts, 2^-23 of a partial sum every 16 of n terms; the output's rounding
    off = p0 * (2.0 ** -11 + 2 * err[:, None] + 16 * oracle.ULP) + 2.0 ** -39 * 2
    bound = ((off + oracle.ULP * (n / 16 + 4) * (p0 + off)) * x.double().abs()).sum(0)
    bound = bound + 2.0 ** -8 * (want.abs() + bound)
    assert (want.abs() > 8 * bound).double().mean() > 0.9
    others = torch.cat([torch.tensor([1, v - 3, 2 ** 31 // d + 1, 2 ** 32 // d // 2 + 1, 2 ** 32 // d // 2 - 2]),
                        torch.randint(0, v, (2000,), generator=g)])
    others = others[~torch.isin(others, where)]
    worst = ((dt[others.cuda()].double().cpu() - want).abs() / bound).max().item()
    assert worst <= 1.0, worst
    same = dt[others[0].cuda()]
    alike = (dt == same).all(1)
    alike[where.cuda()] = True
    assert alike.all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("teacher_temperature", [0.25, 1.0, 3.0])
@pytest.mark.parametrize("n", [10, 400])
def test_teacher_logits_at_the_ends_of_their_type(n, dtype, teacher_temperature):
    """The lowest value of a type is a logit like any other, whatever it is divided by: a row of nothing else is spread over its
    entries, and only -inf says that an entry is not there."""
    from memoryefficientclip_b200 import MemoryEfficientDistillLoss
    v, d, k = 200, 64, 5
    x, table, _tokens, g = _pair(n, v, d, torch.bfloat16, n)
    t, logits = _teacher(n, v, k, g, dtype)
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    logits[0], logits[1, 1:], logits[2, :3] = low, low, high
    logits[3, 0], logits[3, 1], logits[4, 2:] = high, low, float("-inf")
    logits[4, :2], logits[5, 0], logits[6] = low, float("-inf"), float("-inf")
    xg, yg = x.cuda().requires_grad_(True), table.cuda().requires_grad_(True)
    loss = MemoryEfficientDistillLoss(1.0, True, teacher_temperature, "none")(xg, yg, t.cuda(), logits.cuda())
    kl, has, err = oracle.distill(x, table, t, logits, 1.0, teacher_temperature)
    assert has[:6].all() and not has[6]
    # where the logits are the type's ends their differences are 0 or beyond any exponential's range, so that q has no error
    ends = torch.zeros(n, dtype=torch.bool)
    ends[[0, 2, 3, 4]] = True
    _z, score_err = oracle.scores(x, table, 1.0)
    err = torch.where(ends, 2 * score_err + 16 * oracle.ULP * (kl.abs() + 10), err)
    _inside(loss, kl, err + 1e-30, "loss")
    weight = torch.randn(n, generator=g)
    dx, dy = torch.autograd.grad(loss, [xg, yg], weight.cuda())
    q, has = oracle.teacher(t, logits, teacher_temperature)
    w = (weight.double() * has)[:, None]
    dense = torch.softmax(x.double() @ table.double().T, 1) * w
    entries = torch.zeros_like(dense).scatter_add_(1, t, -q * w)
    u = torch.where((q > 0) & ~ends[:, None], logits.double().abs() / teacher_temperature, torch.zeros_like(q)).max()
    wx, wy, bx, by = oracle._gradients(x, table, 1.0, dense, entries, dense.abs() + entries.abs() * (1 + u),
                                       (torch.bfloat16,) * 2, 0.0)
    _inside(dx, wx, bx, "dx")
    _inside(dy, wy, by, "dtable")


def test_temperatures_without_a_finite_inverse_are_refused():
    from memoryefficientclip_b200 import MemoryEfficientDistillLoss, _lib, token_log_probs
    x, table, tokens, _g = _pair(4, 9, 8, torch.bfloat16, 1)
    x, table, tokens = x.cuda(), table.cuda(), tokens.cuda()
    logits = torch.zeros(4, 1, device="cuda")
    for call in (lambda: token_log_probs(x, table, tokens, temperature=1e-39),
                 lambda: MemoryEfficientDistillLoss(1e-39, True)(x, table, tokens[:, None], logits),
                 lambda: MemoryEfficientDistillLoss(1.0, True, 1e-39)(x, table, tokens[:, None], logits)):
        with pytest.raises(_lib.MeclipError):
            call()


@pytest.mark.parametrize("n,v,d", [(700, 1500, 64), (1300, 1500, 264), (200, 1500, 264)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("per_row", [1, 3])
def test_weights_over_several_blocks(n, v, d, dtype, per_row):
    """Row factors, entries and scaled features of every block of rows and panel of columns are that block's own."""
    from memoryefficientclip_b200 import _lib, ops
    x, table, tokens, g = _pair(n, v, d, dtype, n + per_row, bump=4.0)
    many = torch.stack([tokens] + [torch.randint(-1, v, (n,), generator=g) for _ in range(per_row - 1)], 1)
    weight = 2.0 ** -torch.randint(0, 31, (n,), generator=g).double()
    weight[::13] = 0
    g_lp, g_h = torch.randn(n, per_row, generator=g), torch.randn(n, generator=g) * 0.3
    wg, wh = (g_lp.double() * weight[:, None]).float(), (g_h.double() * weight).float()
    xg, yg, tk = x.cuda(), table.cuda(), many.cuda()
    f32, status = torch.float32, ops.status_word(xg.device)
    _lp, entropy, _a, _b, saved = ops.token_log_probs(xg, yg, tk, 1.0, 0, True, status)
    _lib.check(_lib.load().meclip_debug_set_blocking(128, 128 * 2 * 512))
    try:
        dx, dt = ops.token_log_probs_grad(xg, yg, tk, 1.0, saved, entropy, wg.cuda(), wh.cuda(), f32, f32, status=status)
        torch.cuda.synchronize()
    finally:
        _lib.check(_lib.load().meclip_debug_set_blocking(0, 0))
    wx, _wy, bx, _by = oracle.token_log_probs_grad(x, table, many, 1.0, g_lp, g_h, (f32, f32))
    # (three panels and eleven blocks of rows: their sums are fewer roundings than the bounds count for the cut contractions)
    _inside(dx, weight[:, None] * wx, weight[:, None] * bx + torch.finfo(f32).tiny, "dx")
    _wx, wy, _bx, by = oracle.token_log_probs_grad(x, table, many, 1.0, wg, wh, (f32, f32))
    _inside(dt, wy, by, "dtable")
