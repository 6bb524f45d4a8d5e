"""Embedding lookup and its gradient against 64 bits.

The lookup rounds a product once to fp32 and once to the output's type.  A row of the gradient is a sum of c terms in
fp32, in some order: its error is at most c 2^-24 of the sum of magnitudes, then the scale and the output's rounding."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _reference(tokens, table, scale, grad):
    v = table.shape[0]
    inside = (tokens >= 0) & (tokens < v)
    at = tokens.clamp(0, v - 1)
    out = torch.where(inside[:, None], table.double()[at] * scale, torch.zeros(()).double())
    g = torch.where(inside[:, None], grad.double(), torch.zeros(()).double())
    zero = torch.zeros(v, table.shape[1], dtype=torch.float64)
    dt, size = zero.clone().index_add_(0, at, g), zero.index_add_(0, at, g.abs())
    count = torch.bincount(at[inside], minlength=v).double()[:, None]
    half = torch.finfo(table.dtype).eps / 2
    bound = abs(scale) * ((count + 2) * 2.0 ** -24 * size)
    bound = bound + half * (dt.abs() * abs(scale) + bound) + torch.finfo(table.dtype).tiny
    err_out = (half + 2.0 ** -24 * (1 + half)) * out.abs() + torch.finfo(table.dtype).tiny
    return out, dt * scale, err_out, bound


def _check(tokens, table, grad, scale):
    from memoryefficientclip_b200 import embed_tokens
    tg = table.cuda().requires_grad_(True)
    out = embed_tokens(tokens.cuda(), tg, scale)
    assert out.shape == (*tokens.shape, table.shape[1]) and out.dtype == table.dtype
    (dt,) = torch.autograd.grad(out, tg, grad.cuda())
    wo, wt, eo, et = _reference(tokens.reshape(-1).long(), table, scale, grad.reshape(-1, grad.shape[-1]))
    assert ((out.detach().double().cpu().reshape(wo.shape) - wo).abs() <= eo).all()
    worst = ((dt.double().cpu() - wt).abs() / et).max().item()
    assert worst <= 1.0, worst
    return dt


@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (1, 70000, 8), (5, 3, 7), (33, 1000, 64), (511, 40, 100), (512, 1024, 1032),
                                   (4096, 1023, 72), (4097, 257, 65), (9000, 5000, 520), (40000, 3, 16), (20000, 66000, 24)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_lookup_and_gradient(n, v, d, dtype):
    g = torch.Generator().manual_seed(n + v)
    tokens = torch.randint(0, v, (n,), generator=g)
    tokens[torch.rand(n, generator=g) < 0.15] = -1
    table = torch.randn(v, d, generator=g).to(dtype)
    grad = torch.randn(n, d, generator=g).to(dtype)
    _check(tokens, table, grad, math.sqrt(d))


@pytest.mark.parametrize("n", [1000, 4096, 70001])
def test_common_tokens(n):
    """Runs that fill whole chunks, end inside one, start on an edge; all positions one token; nothing but padding."""
    g = torch.Generator().manual_seed(n)
    v, d = 90, 40
    table, grad = torch.randn(v, d, generator=g), torch.randn(n, d, generator=g)
    u = torch.rand(n, generator=g)
    for tokens in ((torch.exp(u * math.log(v + 1.0)) - 1).long().clamp(0, v - 1), torch.full((n,), 7),
                   torch.arange(n) * 3 // n, torch.full((n,), -1), torch.arange(n) // 32 % v, torch.arange(n) // 1024 % v):
        _check(tokens, table, grad, 1.0)


@pytest.mark.parametrize("n,v,d", [(5000, 1200000, 8), (3000, 1100000, 4), (70000, 1023, 260), (6000, 1024, 257)])
def test_wide_keys_and_several_column_blocks(n, v, d):
    """Three sorting passes, keys that fill their bits, rows of more than one warp's columns."""
    g = torch.Generator().manual_seed(v)
    tokens = torch.randint(-1, v, (n,), generator=g)
    _check(tokens, torch.randn(v, d, generator=g), torch.randn(n, d, generator=g), 1.5)


def test_shapes_layouts_and_repeats():
    from memoryefficientclip_b200 import embed_tokens
    g = torch.Generator().manual_seed(1)
    table = torch.randn(50, 24, generator=g).bfloat16()
    tokens = torch.randint(-1, 50, (4, 3, 5), generator=g)
    grad = torch.randn(4, 3, 5, 24, generator=g).bfloat16()
    first = _check(tokens, table, grad, 0.5)
    assert torch.equal(first, _check(tokens.int(), table, grad, 0.5))
    wide = torch.zeros(50, 40, dtype=torch.bfloat16).cuda()
    wide[:, 3:27] = table.cuda()
    a = embed_tokens(tokens.cuda().transpose(0, 1), wide[:, 3:27], 0.5)
    assert torch.equal(a, embed_tokens(tokens.cuda(), table.cuda(), 0.5).transpose(0, 1))
    turned = table.T.contiguous().cuda().T
    assert torch.equal(embed_tokens(tokens.cuda(), turned, 0.5), embed_tokens(tokens.cuda(), table.cuda(), 0.5))
    # gradients that are not laid out row by row: an expanded one and a transposed one
    tg = table.cuda().requires_grad_(True)
    flat = tokens.reshape(-1).cuda()
    for go in (torch.ones(1, 24, dtype=torch.bfloat16, device="cuda").expand(60, 24),
               torch.randn(24, 60, device="cuda").bfloat16().T):
        (x,) = torch.autograd.grad(embed_tokens(flat, tg), tg, go)
        (y,) = torch.autograd.grad(embed_tokens(flat, tg), tg, go.contiguous())
        assert torch.equal(x, y)


def test_empty_and_outside():
    from memoryefficientclip_b200 import embed_tokens
    tg = torch.randn(6, 16, device="cuda", requires_grad=True)
    out = embed_tokens(torch.zeros(0, 3, dtype=torch.long, device="cuda"), tg)
    assert out.shape == (0, 3, 16)
    (dt,) = torch.autograd.grad(out, tg, torch.zeros_like(out))
    assert not dt.any()
    out = embed_tokens(torch.tensor([6, 2, -3], device="cuda"), tg)
    assert out[0].isnan().all() and torch.equal(out[1], tg[2]) and not out[2].any()
    (dt,) = torch.autograd.grad(out, tg, torch.ones_like(out))
    want = torch.zeros(6, 16, device="cuda")
    want[2] = 1
    assert torch.equal(dt, want)


def test_a_tied_table_as_it_is_used():
    """One table looked up, scored against and distilled into: the sum of its gradients, eager and captured."""
    from memoryefficientclip_b200 import MemoryEfficientDistillLoss, embed_tokens, token_log_probs
    n, v, d, k = 300, 800, 64, 4
    g = torch.Generator().manual_seed(5)
    table = (torch.randn(v, d, generator=g) / 8).bfloat16()
    tokens = torch.randint(0, v, (n,), generator=g)
    teacher = torch.randint(0, v, (n, k), generator=g)
    logits = torch.randn(n, k, generator=g)
    tg, tok, te, lo = table.cuda().requires_grad_(True), tokens.cuda(), teacher.cuda(), logits.cuda()
    distil = MemoryEfficientDistillLoss(1.0, normalized_inputs=True)

    def step():
        x = embed_tokens(tok, tg, 8.0)
        loss = distil(x, tg, te, lo) - 0.5 * token_log_probs(x, tg, tok.roll(-1)).log_probs.mean()
        return loss, torch.autograd.grad(loss, tg)[0]

    # detached: a living eager graph of the same leaf would tie the capture below to the stream it was made on
    loss, dt = (o.detach() for o in step())
    ref = table.double().requires_grad_(True)
    x = 8.0 * ref[tokens]
    lp = torch.log_softmax(x @ ref.T, 1)
    q = torch.softmax(logits.double(), 1)
    want = (torch.xlogy(q, q) - q * lp.gather(1, teacher)).sum(1).mean() - 0.5 * lp.gather(1, tokens.roll(-1)[:, None]).mean()
    want.backward()
    assert abs(loss.item() - want.item()) <= 1e-5 * abs(want.item())
    # three bf16 gradients of about this size are added in bf16, and each went through bf16 coefficients: at most
    # five half steps of 2^-8 of the parts' norms, which are at most a few times the sum's
    assert (dt.double().cpu() - ref.grad).norm() <= 5 * 2.0 ** -8 * ref.grad.norm()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], loss) and torch.equal(out[1], dt)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_broadcast_and_overlapping_tables(dtype):
    """One row expanded to many, rows that overlap, and a single row of whatever pitch."""
    from memoryefficientclip_b200 import embed_tokens
    table = torch.randn(300, 64, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    tokens = (torch.arange(90) * 7 % 300).cuda()
    for t, at in ((table[:1].expand(300, 64), tokens), (table.reshape(-1).as_strided((300, 64), (8, 1)), tokens),
                  (table[:1].as_strided((1, 64), (0, 1)), tokens.clamp(max=0))):
        assert torch.equal(embed_tokens(at, t, 0.5), (t.float()[at] * 0.5).to(dtype))
    one = table[:1].clone().requires_grad_(True)
    embed_tokens(tokens, one.expand(300, 64)).float().sum().backward()
    assert torch.equal(one.grad.float(), torch.full((1, 64), 90.0, device="cuda"))


def test_second_derivatives_are_refused():
    from memoryefficientclip_b200 import embed_tokens
    table = torch.randn(30, 8, device="cuda", requires_grad=True)
    w = torch.ones((), device="cuda", requires_grad=True)
    (dt,) = torch.autograd.grad(embed_tokens(torch.arange(9, device="cuda"), table).sum() * w, table, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dt.sum().backward()
