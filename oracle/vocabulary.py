"""Softmax over a vocabulary in 64 bits on the CPU: what the vocabulary operators are tested against, with bounds on
how far correctly rounded kernels may be off.

Bounds count the roundings of the computation, for operands that are exact:
  scores     the products are exact in fp32; a dot product adds D / 16 groups, each dropping up to one fp32 ulp (2^-23)
             of a partial sum that stays below |x_i| |y_j|; scale and exponent add a few ulps of the score itself
  p, log p   the error of the scores, plus that of summing V exponentials (a few ulps: the partial sums are positive)
  entropy    sum_j p_j |log p_j + H| <= 2 ln V times the error of the scores
  gradients  every coefficient is rounded once to fp16, its row scaled so that a bound on its coefficients comes to 2^14
             (half a step, 2^-11 relative, or half of fp16's smallest, 2^-25, over the scale: 2^-39 of that bound, for
             which the largest of all rows' bounds stands here) or to two bf16 numbers (less); it carries the error of its p, and the contraction drops up to 2^-23 of a partial sum
             every 16 terms; then one rounding to the output's type
"""
import torch

ULP = 2.0 ** -23


def scores(x, table, temperature):
    """(z [N, V] in fp64, bound on the error of a computed score per row [N])."""
    x, y = x.double(), table.double()
    z = x @ y.T / temperature
    norms = x.norm(dim=1) * y.norm(dim=1).max() / temperature
    err = ULP * ((x.shape[1] / 16 + 4) * norms + 8 * z.abs().amax(dim=1) + 8)
    return z, err


def token_log_probs(x, table, tokens, temperature, top_k=0):
    """Dict of log_probs [N, k], entropy, top_log_probs, top_tokens and the bounds err_lp, err_entropy, all fp64."""
    z, err = scores(x, table, temperature)
    v = z.shape[1]
    lse = torch.logsumexp(z, dim=1)
    log_p = z - lse[:, None]
    p = log_p.exp()
    entropy = -(p * log_p).sum(1)
    at = tokens.clamp(0, v - 1)
    lp = log_p.gather(1, at)
    lp = torch.where(tokens < 0, torch.zeros_like(lp), lp)
    lp = torch.where(tokens >= v, torch.full_like(lp, float("nan")), lp)
    out = {"log_probs": lp, "entropy": entropy, "p": p, "log_p": log_p,
           "err_lp": 2 * err, "err_entropy": err * 2 * max(1.0, float(torch.log(torch.tensor(float(v)))))}
    if top_k:
        top, idx = torch.sort(z, dim=1, descending=True, stable=True)
        out["top_log_probs"] = (top - lse[:, None])[:, :top_k]
        out["top_tokens"] = idx[:, :top_k]
    return out


def _gradients(x, table, temperature, dense, entries, dense_size, out_dtypes, operand_rounding):
    """(dx, dtable, bound dx, bound dtable) of dz = dense + entries; dense_size bounds |dense| before cancellation."""
    x, y = x.double(), table.double()
    _z, err = scores(x, table, temperature)
    dz = (dense + entries) / temperature
    size = (dense_size + entries.abs()) / temperature
    # a coefficient: half an fp16 step of itself or of the smallest number, and the score's error on every part of it
    off = 2.0 ** -11 * dz.abs() + 2.0 ** -39 * size.sum(1).max() + (2 * err[:, None] + 16 * ULP) * size
    out = []
    for dim, (g, o, sz, other, dtype) in enumerate(((dz, off, size, y, out_dtypes[0]),
                                                    (dz.T, off.T, size.T, x, out_dtypes[1]))):
        k = g.shape[1]
        value = g @ other
        bound = (o + (operand_rounding + ULP * (k / 16 + 4)) * (g.abs() + o)) @ other.abs()
        bound = bound + torch.finfo(dtype).eps / 2 * (value.abs() + bound) + torch.finfo(dtype).tiny
        out.append((value, bound))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def token_log_probs_grad(x, table, tokens, temperature, grad_log_probs, grad_entropy, out_dtypes, operand_rounding=0.0):
    r = token_log_probs(x, table, tokens, temperature)
    p, log_p, h = r["p"], r["log_p"], r["entropy"]
    v = p.shape[1]
    inside = (tokens >= 0) & (tokens < v)
    a = torch.where(inside, grad_log_probs.double(), torch.zeros(()).double())
    b = grad_entropy.double()[:, None]
    dense = -p * (a.sum(1, keepdim=True) + b * (log_p + h[:, None]))
    size = p * (a.abs().sum(1, keepdim=True) + b.abs() * (log_p.abs() + h[:, None] + 1))
    entries = torch.zeros_like(p).scatter_add_(1, tokens.clamp(0, v - 1), a)
    return _gradients(x, table, temperature, dense, entries, size, out_dtypes, operand_rounding)


def teacher(teacher_tokens, teacher_logits, teacher_temperature=1.0):
    """(q [N, k], rows that have an entry [N])."""
    logits = teacher_logits.double() / teacher_temperature
    there = (teacher_tokens >= 0) & ~(teacher_logits == float("-inf"))
    logits = torch.where(there, logits, torch.full_like(logits, float("-inf")))
    has = there.any(1)
    q = torch.where(has[:, None], torch.softmax(torch.where(has[:, None], logits, torch.zeros_like(logits)), dim=1),
                    torch.zeros_like(logits))
    return q, has


def distill(x, table, teacher_tokens, teacher_logits, temperature, teacher_temperature=1.0):
    """(KL per row [N], rows with an entry [N], bound on the error of a row's loss [N])."""
    z, err = scores(x, table, temperature)
    log_p = torch.log_softmax(z, dim=1)
    q, has = teacher(teacher_tokens, teacher_logits, teacher_temperature)
    at = teacher_tokens.clamp(0, z.shape[1] - 1)
    kl = (torch.xlogy(q, q) - q * log_p.gather(1, at)).sum(1)
    # q itself: a few ulps of an exponential of a rounded difference, weighed with the logarithms it multiplies
    spread = torch.where(q > 0, log_p.gather(1, at).abs() + torch.xlogy(torch.ones_like(q), q.clamp(min=1e-300)).abs(),
                         torch.zeros_like(q))
    u = torch.where(q > 0, teacher_logits.double().abs() / teacher_temperature, torch.zeros_like(q)).amax(1, keepdim=True)
    return kl, has, 2 * err + (q * spread * ULP * (8 + 4 * u)).sum(1) + ULP * kl.abs()


def distill_grad(x, table, teacher_tokens, teacher_logits, temperature, weight, out_dtypes, teacher_temperature=1.0,
                 operand_rounding=0.0):
    """weight [N]: the incoming gradient of each row's loss."""
    z, _err = scores(x, table, temperature)
    p = torch.softmax(z, dim=1)
    q, has = teacher(teacher_tokens, teacher_logits, teacher_temperature)
    w = (weight.double() * has)[:, None]
    entries = torch.zeros_like(p).scatter_add_(1, teacher_tokens.clamp(0, z.shape[1] - 1), -q * w)
    # a few ulps of q on top (its exponent's rounding grows with the logits)
    u = torch.where(q > 0, teacher_logits.double().abs() / teacher_temperature, torch.zeros_like(q)).max().item()
    dense = p * w
    return _gradients(x, table, temperature, dense, entries, dense.abs() + entries.abs() * (1 + u), out_dtypes,
                      operand_rounding)
