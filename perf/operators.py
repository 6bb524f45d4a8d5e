"""What is measured of the vocabulary operators: a table of V rows that tokens are looked up in and features are
scored against.

  score    log probabilities of given tokens under softmax(x table^T / T), with the entropy of each row and its top
           alternatives; with train=True also the gradients of the log probabilities and the entropy
  distill  KL divergence from a teacher's top logits to softmax(x table^T / T), a training step: loss and gradients
  embed    rows of a table scaled, and with train=True the gradient of the table

Sizes: features of 512, 768, 1024 and 1152 columns and batches up to 8192 rows as in this repository's benchmark and
tests, vocabularies of generic sizes.
"""
import math

import torch

own = False

IGNORE = -1


def listed():
    return [
        # one token of one sequence is being generated: which tokens come next
        {"name": "score_1_token", "op": "score", "rows": 1, "vocab": 32768, "dim": 1024, "top": 8, "dtype": "bfloat16",
         "temperature": 0.8, "train": False},
        # a serving batch, a vocabulary that fills no tile, half precision
        {"name": "score_61_tokens", "op": "score", "rows": 61, "vocab": 50001, "dim": 768, "top": 5, "dtype": "float16",
         "temperature": 1.0, "train": False},
        # a prompt or a set of answers is scored
        {"name": "score_prompt", "op": "score", "rows": 4096, "vocab": 32768, "dim": 1024, "top": 8, "dtype": "bfloat16",
         "temperature": 1.0, "train": False},
        # a policy update on a short batch: gradients of log probabilities and entropy, odd sizes
        {"name": "score_train_2047", "op": "score", "rows": 2047, "vocab": 32001, "dim": 512, "top": 0,
         "dtype": "bfloat16", "temperature": 1.0, "train": True},
        # a captioner's head on a full batch
        {"name": "score_train_8192", "op": "score", "rows": 8192, "vocab": 49999, "dim": 1152, "top": 0,
         "dtype": "bfloat16", "temperature": 1.0, "train": True},
        # a small step: few rows, a table of a few thousand classes
        {"name": "distill_128", "op": "distill", "rows": 128, "vocab": 4099, "dim": 512, "teacher": 8,
         "dtype": "bfloat16", "temperature": 1.0, "unit": False},
        # two towers distilled: unit features, the teacher's best 32 of the batch's texts
        {"name": "distill_towers_4096", "op": "distill", "rows": 4096, "vocab": 32768, "dim": 768, "teacher": 32,
         "dtype": "bfloat16", "temperature": 0.07, "unit": True},
        # a language model's head distilled on a full batch
        {"name": "distill_8192", "op": "distill", "rows": 8192, "vocab": 65536, "dim": 1152, "teacher": 64,
         "dtype": "bfloat16", "temperature": 1.0, "unit": False},
        # the lookup in front of one generated token's pass for a serving batch
        {"name": "embed_61_tokens", "op": "embed", "rows": 61, "vocab": 50001, "dim": 768, "dtype": "float16",
         "train": False},
        # the lookup of a prompt
        {"name": "embed_32768", "op": "embed", "rows": 32768, "vocab": 32768, "dim": 1024, "dtype": "bfloat16",
         "train": False},
        # a small training step
        {"name": "embed_train_2047", "op": "embed", "rows": 2047, "vocab": 32001, "dim": 512, "dtype": "float32",
         "train": True},
        # a full training step: common tokens are thousands of times as frequent as rare ones, a fifth is padding
        {"name": "embed_train_131072", "op": "embed", "rows": 131072, "vocab": 49999, "dim": 1152, "dtype": "bfloat16",
         "train": True},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["score", "score", "distill", "embed"])
    dim = rng.choice([_spread(rng, 64, 1152), 8 * _spread(rng, 8, 144), 512, 768, 1024, 1152])
    if op == "score":
        train = rng.random() < 0.5
        return {"op": op, "rows": _spread(rng, 1, 8192), "vocab": _spread(rng, 1000, 65536), "dim": dim,
                "top": 0 if train else rng.randint(0, 16), "dtype": "bfloat16" if train else rng.choice(["bfloat16", "float16"]),
                "temperature": round(rng.uniform(0.6, 1.5), 2), "train": train}
    if op == "distill":
        unit = rng.random() < 0.5
        return {"op": op, "rows": _spread(rng, 16, 8192), "vocab": _spread(rng, 1000, 65536), "dim": dim,
                "teacher": _spread(rng, 1, 64), "dtype": "bfloat16",
                "temperature": 0.07 if unit else round(rng.uniform(0.8, 2.0), 2), "unit": unit}
    return {"op": op, "rows": _spread(rng, 1, 131072), "vocab": _spread(rng, 1000, 65536), "dim": dim,
            "dtype": rng.choice(["bfloat16", "float16", "float32"]), "train": rng.random() < 0.6}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n, v, d = case["rows"], case["vocab"], case["dim"]
    dtype = getattr(torch, case["dtype"])
    state = {"case": case}

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    # tokens as text has them: the frequency of a token falls with its rank
    u = torch.rand(n, generator=g, device="cuda")
    tokens = (torch.exp(u * math.log(v + 1.0)) - 1.0).long().clamp_(0, v - 1)
    if case["op"] == "embed":
        if case["train"]:
            tokens = torch.where(torch.rand(n, generator=g, device="cuda") < 0.2, torch.full_like(tokens, IGNORE), tokens)
            state["grad"] = randn(n, d).to(dtype)
        state |= {"tokens": tokens, "table": (0.02 * randn(v, d)).to(dtype), "scale": math.sqrt(d)}
        if case["train"]:
            state["table"].requires_grad_(True)
        return state
    table = randn(v, d) / math.sqrt(d)
    if case.get("unit"):
        table = torch.nn.functional.normalize(table, dim=1)
        x = torch.nn.functional.normalize(0.5 * table[tokens] + randn(n, d) / math.sqrt(d), dim=1)
    else:
        x = 2.0 * randn(n, d) + 10.0 * table[tokens]
    x, table = x.to(dtype), table.to(dtype)
    state |= {"x": x, "table": table}
    if case["op"] == "score":
        drop = 0.05 if case["train"] else 0.0
        tokens = torch.where(torch.rand(n, generator=g, device="cuda") < drop, torch.full_like(tokens, IGNORE), tokens)
        state["tokens"] = tokens
        if case["train"]:
            state["grad_log_probs"] = -torch.rand(n, generator=g, device="cuda") / n
            state["grad_entropy"] = randn(n) * (0.01 / n)
            x.requires_grad_(True)
            table.requires_grad_(True)
        return state
    k = case["teacher"]
    # the teacher's best entries: the target first, then distinct others; logits fall off. Some rows have fewer than
    # k entries, some none; what stands in an absent entry's place means nothing
    step = torch.randint(1, max(2, (v - 1) // max(k, 1)), (n, 1), generator=g, device="cuda")
    teacher_tokens = (tokens[:, None] + step * torch.arange(k, device="cuda")) % v
    teacher_logits = 12.0 - 3.0 * torch.log1p(torch.arange(k, device="cuda").float()) + randn(n, k)
    present = torch.randint(1, k + 1, (n, 1), generator=g, device="cuda")
    present = torch.where(torch.rand(n, 1, generator=g, device="cuda") < 0.5, torch.full_like(present, k), present)
    present = torch.where(torch.rand(n, 1, generator=g, device="cuda") < 0.05, torch.zeros_like(present), present)
    present[0] = k
    absent = torch.arange(k, device="cuda") >= present
    state["teacher_tokens"] = torch.where(absent, torch.full_like(teacher_tokens, IGNORE), teacher_tokens)
    state["teacher_logits"] = torch.where(absent, torch.full_like(teacher_logits, math.nan), teacher_logits)
    x.requires_grad_(True)
    table.requires_grad_(True)
    return state


def run(state):
    case = state["case"]
    return {"score": _score, "distill": _distill, "embed": _embed}[case["op"]](case, state)


def _score(case, s):
    t, k = case["temperature"], case["top"]
    if own:
        import memoryefficientclip_b200 as m
        got = m.token_log_probs(s["x"], s["table"], s["tokens"], temperature=t, top_k=k)
        if case["train"]:
            dx, dtable = torch.autograd.grad([got.log_probs, got.entropy], [s["x"], s["table"]],
                                             [s["grad_log_probs"], s["grad_entropy"]])
            return {"log_probs": got.log_probs, "entropy": got.entropy, "dx": dx, "dtable": dtable}
        out = {"log_probs": got.log_probs, "entropy": got.entropy}
        if k:
            out |= {"top_log_probs": got.top_log_probs, "top_tokens": got.top_tokens}
        return out
    with torch.no_grad():
        x, y, tokens = s["x"].float(), s["table"].float(), s["tokens"]
        z = x @ y.T / t
        peak = z.max(1, keepdim=True).values
        lse = peak + torch.log(torch.exp(z - peak).sum(1, keepdim=True))
        log_p = z - lse
        p = torch.exp(log_p)
        entropy = -(p * log_p).sum(1)
        valid = tokens >= 0
        at = tokens.clamp(min=0)[:, None]
        out = {"log_probs": torch.where(valid, log_p.gather(1, at)[:, 0], 0.0), "entropy": entropy}
        if case["train"]:
            a = torch.where(valid, s["grad_log_probs"], 0.0)
            dz = -p * (a[:, None] + s["grad_entropy"][:, None] * (log_p + entropy[:, None]))
            dz.scatter_add_(1, at, a[:, None])
            dz /= t
            return out | {"dx": (dz @ y).to(s["x"].dtype), "dtable": (dz.T @ x).to(s["table"].dtype)}
        if k:
            # the order of the best ones is decided in 64 bits: 32 may swap neighbours
            near = torch.topk(z, min(k + 8, case["vocab"]), dim=1).indices.sort(1).values
            score = torch.matmul(s["table"][near].double(), s["x"].double()[:, :, None])[:, :, 0] / t
            score, order = torch.sort(score, dim=1, descending=True, stable=True)
            out |= {"top_log_probs": (score[:, :k] - lse.double()).float(), "top_tokens": near.gather(1, order[:, :k])}
        return out


def _distill(case, s):
    t = case["temperature"]
    if own:
        import memoryefficientclip_b200 as m
        loss = m.MemoryEfficientDistillLoss(temperature=t, normalized_inputs=True)(s["x"], s["table"], s["teacher_tokens"],
                                                                                   s["teacher_logits"])
        dx, dtable = torch.autograd.grad(loss, [s["x"], s["table"]])
        return {"loss": loss, "dx": dx, "dtable": dtable}
    with torch.no_grad():
        x, y = s["x"].float(), s["table"].float()
        there = s["teacher_tokens"] >= 0
        at = s["teacher_tokens"].clamp(min=0)
        u = torch.where(there, s["teacher_logits"], -1e30)
        q = torch.where(there, torch.exp(u - u.max(1, keepdim=True).values), 0.0)
        counts = there.any(1)
        q = q / torch.where(counts, q.sum(1), 1.0)[:, None]
        z = x @ y.T / t
        peak = z.max(1, keepdim=True).values
        log_p = z - (peak + torch.log(torch.exp(z - peak).sum(1, keepdim=True)))
        terms = torch.where(q > 0, q * (torch.log(torch.where(q > 0, q, 1.0)) - log_p.gather(1, at)), 0.0)
        rows = counts.sum()
        loss = terms.sum(1).sum() / rows
        dz = torch.exp(log_p)
        dz.scatter_add_(1, at, -q)
        dz *= (counts / (rows * t))[:, None]
        return {"loss": loss, "dx": (dz @ y).to(s["x"].dtype), "dtable": (dz.T @ x).to(s["table"].dtype)}


def _embed(case, s):
    if own:
        import memoryefficientclip_b200 as m
        out = m.embed_tokens(s["tokens"], s["table"], scale=s["scale"])
        if not case["train"]:
            return {"out": out}
        return {"out": out, "dtable": torch.autograd.grad(out, s["table"], s["grad"])[0]}
    with torch.no_grad():
        tokens, table = s["tokens"], s["table"]
        valid = (tokens >= 0)[:, None]
        at = tokens.clamp(min=0)
        out = torch.where(valid, table[at].float() * s["scale"], 0.0).to(table.dtype)
        if not case["train"]:
            return {"out": out}
        g = torch.where(valid, s["grad"].float() * s["scale"], 0.0)
        dtable = torch.zeros(table.shape, device="cuda").index_add_(0, at, g)
        return {"out": out, "dtable": dtable.to(table.dtype)}


def work(case):
    n, v, d = case["rows"], case["vocab"], case["dim"]
    e = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "embed":
        # the tokens, the rows looked up and written; the gradient's rows read and the table's gradient written
        return {"bytes": 8.0 * n + 2.0 * n * d * e + (n * d * e + v * d * e if case["train"] else 0.0),
                "flops": float(n * d) * (2 if case["train"] else 1)}
    train = case["op"] == "distill" or case["train"]
    k = case.get("teacher", 1)
    read = (n + v) * d * e + n * k * 12.0
    written = n * (8.0 + 12.0 * case.get("top", 0)) + ((n + v) * d * e if train else 0.0)
    return {"bytes": read + written, "flops": (6.0 if train else 2.0) * n * v * d}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "embed":
            pad = torch.cat([s["table"].detach().double(), torch.zeros(1, case["dim"], dtype=torch.float64, device="cuda")])
            slot = torch.where(s["tokens"] < 0, case["vocab"], s["tokens"])
            out = {"out": pad[slot] * s["scale"]}
            if case["train"]:
                total = torch.zeros_like(pad)
                for first in range(0, case["rows"], 16384):
                    part = slice(first, first + 16384)
                    total.index_put_((slot[part],), s["grad"][part].double() * s["scale"], accumulate=True)
                out["dtable"] = total[:-1]
            return out
        x, y, t = s["x"].detach().double(), s["table"].detach().double(), case["temperature"]
        train = case["op"] == "distill" or case["train"]
        block = 1024
        parts = []
        dtable = torch.zeros_like(y) if train else None
        rows = (s["teacher_tokens"] >= 0).any(1).sum().double() if case["op"] == "distill" else None
        for first in range(0, case["rows"], block):
            part = slice(first, first + block)
            log_p = torch.log_softmax(torch.einsum("nd,vd->nv", x[part], y) / t, dim=1)
            p = log_p.exp()
            index = torch.arange(log_p.shape[0], device="cuda")
            if case["op"] == "score":
                tokens = s["tokens"][part]
                keep = (tokens >= 0).double()
                h = -torch.einsum("nv,nv->n", p, log_p)
                got = {"log_probs": torch.where(tokens >= 0, log_p[index, tokens.clamp(min=0)], 0.0), "entropy": h}
                if train:
                    # d log p_t = onehot - p, d H = -p (log p + H), against the incoming gradients
                    a, b = s["grad_log_probs"][part].double() * keep, s["grad_entropy"][part].double()
                    dz = -a[:, None] * p - b[:, None] * p * (log_p + h[:, None])
                    dz[index, tokens.clamp(min=0)] += a
                elif case["top"]:
                    best, where = torch.sort(log_p, dim=1, descending=True, stable=True)
                    got |= {"top_log_probs": best[:, :case["top"]].clone(), "top_tokens": where[:, :case["top"]].clone()}
            else:
                there = s["teacher_tokens"][part] >= 0
                logits = s["teacher_logits"][part].double().masked_fill(~there, -math.inf)
                q = torch.softmax(logits, dim=1).nan_to_num(0.0)
                at = s["teacher_tokens"][part].clamp(min=0)
                kl = (torch.xlogy(q, q) - q * log_p.gather(1, at)).sum(1)
                got = {"loss": kl}
                dz = p * there.any(1).double()[:, None] / rows
                dz.scatter_add_(1, at, -q / rows)
            if train:
                got["dx"] = dz @ y / t
                dtable += dz.T @ x[part] / t
            parts.append(got)
        out = {name: torch.cat([q[name] for q in parts]) for name in parts[0]}
        if case["op"] == "distill":
            out["loss"] = out["loss"].sum() / rows
        if train:
            out["dtable"] = dtable
        return out
