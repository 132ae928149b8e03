"""Cases that measure the operators over wide rows of logits: log-probabilities of given tokens (with entropy, normaliser and the top
alternatives) and distillation from a teacher's top log-probabilities, forward and backward.

``own`` False: ``run`` computes the operators in elementary torch operations in fp32 (64 bits where a difference from 1 is taken).
``own`` True: ``run`` calls ``autognothi_amd.ops`` / ``autognothi_amd.models.distill``.
"""
import math

import torch

own = False

MAX_TOP = 128             # alternatives of a row that are asked for, at most
MAX_BYTES = 1 << 31       # of the logits of the largest case


def _case(name, op, rows, vocab, dtype, k, tau=1.0, pad=0, masked=False, tail=False, ragged=False):
    """``k``: alternatives asked for / the teacher's list length; ``pad``: unused columns behind every row (a head padded to a round width);
    ``masked``: some of the vocabulary is ruled out with -inf; ``tail``: the teacher's remaining mass is a class of its own; ``ragged``:
    teacher lists of different lengths and rows of weight 0 (padding tokens)."""
    return dict(name=name, op=op, rows=rows, vocab=vocab, dtype=dtype, k=k, tau=tau, pad=pad, masked=masked, tail=tail, ragged=ragged)


def listed():
    return [
        # the [MASK] position of one sentence: which words would fit there (BERT's vocabulary); latency
        _case("alternatives_1x30522_f32_k5", "logprobs", 1, 30522, "f32", 5),
        # every position of one 128-token sequence
        _case("alternatives_128x30522_bf16_k20", "logprobs", 128, 30522, "bf16", 20),
        # the class logits of 32 masked forwards of 2000 images
        _case("classes_64000x10_f32_k3", "logprobs", 64000, 10, "f32", 3),
        # scoring a batch of text, an odd vocabulary (no row is 16-byte aligned), part of it ruled out
        _case("scores_4096x50001_bf16_k64", "logprobs", 4096, 50001, "bf16", 64, masked=True),
        # recording a teacher: its top 100 at the distillation temperature, a large vocabulary
        _case("record_8192x131072_bf16_k100_t2", "logprobs", 8192, 131072, "bf16", 100, tau=2.0),
        # a policy-gradient / entropy-regularised step: the log-probabilities and their gradients
        _case("train_logp_2000x32000_f32", "logprobs_train", 2000, 32000, "f32", 0, pad=64),
        _case("train_logp_16384x30522_bf16", "logprobs_train", 16384, 30522, "bf16", 0),
        # distillation of a few positions; latency
        _case("distill_16x30522_f32_k16_tail", "distill", 16, 30522, "f32", 16, tail=True),
        # an image classifier's 1000 classes, 25 kept, softened
        _case("distill_24576x1000_f32_k25_t4", "distill", 24576, 1000, "f32", 25, tau=4.0),
        # sequence distillation from a record with lists of different lengths and padding tokens, odd vocabulary
        _case("distill_4097x50001_bf16_k64_ragged", "distill", 4097, 50001, "bf16", 64, ragged=True),
        # the same with a large vocabulary and the teacher's remaining mass, the largest case
        _case("distill_8192x131072_bf16_k100_tail", "distill", 8192, 131072, "bf16", 100, tail=True),
        # the loss as a module of an autograd graph: forward and backward apart
        _case("distill_graph_2048x65537_bf16_k50", "distill_graph", 2048, 65537, "bf16", 50, tau=2.0, tail=True, ragged=True),
    ]


def draw(rng):
    vocab = int(round(math.exp(rng.uniform(math.log(2), math.log(262144)))))
    dtype = rng.choice(["f32", "bf16"])
    most = min(16384 if vocab > 512 else 65536, MAX_BYTES // (vocab * (4 if dtype == "f32" else 2)))
    rows = int(round(math.exp(rng.uniform(0.0, math.log(most)))))
    op = rng.choice(["logprobs", "logprobs", "logprobs_train", "distill", "distill", "distill_graph"])
    k = min(vocab, int(round(math.exp(rng.uniform(0.0, math.log(MAX_TOP))))))
    if op == "logprobs_train":
        k = 0
    c = _case("", op, rows, vocab, dtype, k, tau=rng.choice([1.0, 1.0, 2.0, rng.uniform(0.7, 5.0)]),
              pad=rng.choice([0, 0, rng.randrange(1, 100)]), masked=op.startswith("logprobs") and rng.random() < 0.4,
              tail=op.startswith("distill") and k < vocab and rng.random() < 0.5, ragged=op.startswith("distill") and rng.random() < 0.4)
    del c["name"]
    return c


def _randint(g, high, size, dev):
    return torch.randint(0, high, size, generator=g, device=dev)


def prepare(case, seed):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev)
    g.manual_seed(seed * 7919 + 17)
    n, v, k, tau = case["rows"], case["vocab"], case["k"], case["tau"]
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    # logits as a trained head gives them: a broad bell and, in every row, some tokens that stand out (less so among few classes)
    z = torch.randn((n, v + case["pad"]), generator=g, device=dev, dtype=dtype).mul_(1.5)
    z = z[:, :v]
    s = min(v, max(k, 8))
    width = v // s
    spikes = torch.arange(s, device=dev) * width + _randint(g, width, (n, s), dev)        # distinct tokens
    spikes = spikes.gather(1, torch.rand((n, s), generator=g, device=dev).argsort(dim=1))
    heights = torch.rand((n, s), generator=g, device=dev).pow_(2).mul_(12.0 * min(1.0, math.log(v) / 10.0))
    z.scatter_(1, spikes, heights.to(dtype))
    state = {"case": case, "logits": z}
    if case["op"].startswith("logprobs"):
        tokens = torch.where(torch.rand(n, generator=g, device=dev) < 0.5, spikes[:, 0], _randint(g, v, (n,), dev))
        if case["masked"]:    # a band of the vocabulary is ruled out (special and unused ids), never the given tokens
            z[:, v // 3: v // 3 + max(0, v // 20)] = float("-inf")
            inside = (tokens >= v // 3) & (tokens < v // 3 + max(0, v // 20))
            tokens = torch.where(inside, torch.full_like(tokens, v // 3 + max(0, v // 20)), tokens)
        if n > 4:
            tokens = torch.where(torch.rand(n, generator=g, device=dev) < 0.1, torch.full_like(tokens, -100), tokens)
        state["tokens"] = tokens
        if case["op"] == "logprobs_train":
            state["d_logp"] = -torch.randn(n, generator=g, device=dev) / n
            state["d_entropy"] = -0.01 * torch.rand(n, generator=g, device=dev) / n
        return state
    # the teacher's list: its own idea of the same tokens, in descending order, with 1 % to 40 % of its mass elsewhere
    t = (heights[:, :k] + torch.randn((n, k), generator=g, device=dev)) / tau
    order = t.argsort(dim=1, descending=True)
    kept = torch.rand((n, 1), generator=g, device=dev).mul_(0.39).add_(0.6).log_()
    state["teacher_ids"] = spikes[:, :k].gather(1, order)
    state["teacher_logp"] = torch.log_softmax(t.gather(1, order), dim=1) + kept
    state["weights"] = torch.full((n,), 1.0 / n, device=dev)
    if case["ragged"]:
        lengths = 1 + _randint(g, k, (n, 1), dev)
        state["teacher_ids"] = torch.where(torch.arange(k, device=dev) < lengths, state["teacher_ids"], torch.full_like(state["teacher_ids"], -1))
        real = torch.rand(n, generator=g, device=dev) < 0.85
        state["weights"] = real.float() / n
    if case["op"] == "distill_graph":
        state["logits"].requires_grad_(True)
    return state


# ----------------------------------------------------------------------------- plain forms
def _softmax_parts(z, tau):
    """-> (x - max, exp of it, its sum, max) in fp32, x = z / tau"""
    x = z.float() / tau
    m = x.amax(dim=1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    return d, e, e.sum(dim=1, keepdim=True), m


def _top(z, k):
    """the k largest of every row, ties by the lowest index -> indices: one 64-bit key per element (the value's order, then the index's)"""
    v = z.shape[1]
    bits = (z.float() + 0.0).view(torch.int32)
    keys = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).to(torch.int64)
    keys = keys * (1 << 32) + (v - 1 - torch.arange(v, device=z.device))
    best = torch.topk(keys, k, dim=1, largest=True, sorted=True).values
    return v - 1 - (best & 0xFFFFFFFF)


def _logprobs_plain(z, tokens, k, tau):
    d, e, s, m = _softmax_parts(z, tau)
    log_s = torch.log(s)
    logp = d - log_s
    entropy = -(e / s * torch.where(e > 0, logp, torch.zeros_like(logp))).sum(dim=1)
    given = logp.gather(1, tokens.clamp(min=0)[:, None])[:, 0]
    out = {"logp": torch.where(tokens >= 0, given, torch.zeros_like(given)), "entropy": entropy, "lse": (m + log_s)[:, 0]}
    if k:
        out["top_ids"] = _top(z, k)
        out["top_logp"] = logp.gather(1, out["top_ids"])
    return out


def _logprobs_train_plain(st, tau):
    z, tokens, g, ge = st["logits"], st["tokens"], st["d_logp"], st["d_entropy"]
    d, e, s, m = _softmax_parts(z, tau)
    log_s = torch.log(s)
    logp, p = d - log_s, e / s
    plogp = torch.where(e > 0, logp, torch.zeros_like(logp))
    entropy = -(p * plogp).sum(dim=1)
    valid = tokens >= 0
    at = tokens.clamp(min=0)[:, None]
    given = logp.gather(1, at)[:, 0]
    g = torch.where(valid, g, torch.zeros_like(g))
    grad = p * (-g[:, None] - ge[:, None] * (plogp + entropy[:, None]))
    grad = grad.scatter_add(1, at, g[:, None]) / tau
    return {"logp": torch.where(valid, given, torch.zeros_like(given)), "entropy": entropy, "lse": (m + log_s)[:, 0], "dlogits": grad.to(z.dtype)}


def _distill_plain(st, tau, tail):
    z, ids, weights = st["logits"].detach(), st["teacher_ids"], st["weights"]
    d, e, s, _ = _softmax_parts(z, tau)
    log_s = torch.log(s)
    p = e / s
    there = ids >= 0
    at = ids.clamp(min=0)
    t = torch.where(there, st["teacher_logp"].double(), torch.full_like(ids, -math.inf, dtype=torch.float64))
    if not tail:
        t = torch.log_softmax(t, dim=1)
    q = torch.exp(t)
    logq = torch.where(there, t, torch.zeros_like(t))
    logp = (d.gather(1, at) - log_s).double()
    row = torch.where(there, q * (logq - logp), torch.zeros_like(q)).sum(dim=1)
    if tail:
        rest = (1.0 - q.sum(dim=1)).clamp(min=0.0)
        # (an empty slot names its row's first token once more: every list has at least one)
        inside = torch.zeros_like(z, dtype=torch.bool).scatter_(1, torch.where(there, at, at[:, :1]), True)
        outside = torch.where(inside, torch.zeros_like(e), e).sum(dim=1) / s[:, 0]
        row = row + rest * (rest.log() - outside.log().double())
        coef = (q.sum(dim=1) + rest).float()
        grad = p * torch.where(inside, coef[:, None], (coef - rest.float() / outside)[:, None])
    else:
        grad = p * q.sum(dim=1).float()[:, None]
    grad = grad.scatter_add(1, at, -torch.where(there, q, torch.zeros_like(q)).float())
    row = torch.where(weights != 0, row * (tau * tau), torch.zeros_like(row))     # a row of weight 0 takes no part
    grad = grad * (weights * tau)[:, None]
    return {"loss": (row * weights).sum().float(), "row_loss": row.float(), "dlogits": grad.to(z.dtype)}


def run(state):
    case = state["case"]
    op, k, tau, tail = case["op"], case["k"], case["tau"], case["tail"]
    if not own:
        if op == "logprobs":
            return _logprobs_plain(state["logits"], state["tokens"], k, tau)
        return _logprobs_train_plain(state, tau) if op == "logprobs_train" else _distill_plain(state, tau, tail)
    from autognothi_amd import ops
    from autognothi_amd.models import distill
    z = state["logits"]
    if op == "logprobs":
        r = ops.token_logprobs(z, state["tokens"], top_k=k, temperature=tau)
        return {"logp": r.logp, "entropy": r.entropy, "lse": r.lse, "top_ids": r.top_ids, "top_logp": r.top_logp}
    if op == "logprobs_train":
        r = ops.token_logprobs(z, state["tokens"], temperature=tau)
        dz = ops.token_logprobs_bwd(z, r, state["tokens"], d_logp=state["d_logp"], d_entropy=state["d_entropy"])
        return {"logp": r.logp, "entropy": r.entropy, "lse": r.lse, "dlogits": dz}
    if op == "distill":
        r = ops.topk_distill(z, state["teacher_ids"], state["teacher_logp"], weights=state["weights"], temperature=tau, tail=tail)
        return {"loss": r.loss.reshape(()), "row_loss": r.row_loss, "dlogits": r.dlogits}
    loss, row = distill.loss_topk_distillation(z, state["teacher_ids"], state["teacher_logp"], weights=state["weights"], temperature=tau,
                                               tail=tail)
    (dz,) = torch.autograd.grad(loss, z)
    return {"loss": loss.detach(), "row_loss": row, "dlogits": dz}


def work(case):
    n, v, k = case["rows"], case["vocab"], case["k"]
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "logprobs":    # logits and tokens in; three numbers and k (id, log-probability) pairs out; exp, max, two sums
        return {"bytes": n * v * size + n * (8 + 12 + 12 * k), "flops": 6.0 * n * v}
    if case["op"] == "logprobs_train":    # logits in, their gradient out
        return {"bytes": 2 * n * v * size + n * (8 + 8 + 12), "flops": 12.0 * n * v}
    return {"bytes": 2 * n * v * size + n * (12 * k + 8), "flops": 9.0 * n * v}


def exact(case, seed):
    """the definitions in 64 bits: softmax cross terms through torch.logsumexp, gradients through the formula of a softmax's Jacobian"""
    st = prepare(case, seed)
    tau, k = case["tau"], case["k"]
    x = st["logits"].detach().double().div_(tau)
    lse = torch.logsumexp(x, dim=1)
    if case["op"].startswith("logprobs"):
        tokens = st["tokens"]
        valid = (tokens >= 0).double()
        at = tokens.clamp(min=0)
        picked = (x[torch.arange(case["rows"], device=x.device), at] - lse) * valid
        prob = torch.exp(x - lse[:, None])
        cross = (prob * x.clamp(min=-1e6)).sum(dim=1)          # E[x]; a ruled-out token has probability 0
        entropy = lse - cross
        out = {"logp": picked, "entropy": entropy, "lse": lse}
        if case["op"] == "logprobs":
            out["top_ids"] = None
            out["top_logp"] = torch.topk(x, k, dim=1).values - lse[:, None]
            return out
        g, ge = st["d_logp"].double() * valid, st["d_entropy"].double()
        # d logp_t / dx = 1[t] - p;  d H / dx = -p (x - E[x])
        grad = -prob * (g[:, None] + ge[:, None] * (x.clamp(min=-1e6) - cross[:, None]))
        grad[torch.arange(case["rows"], device=x.device), at] += g
        out["dlogits"] = grad / tau
        return out
    ids, w = st["teacher_ids"], st["weights"].double()
    keep = (ids >= 0)
    t = st["teacher_logp"].double().masked_fill(~keep, -math.inf)
    if not case["tail"]:
        t = t - torch.logsumexp(t, dim=1, keepdim=True)
    q = t.exp()
    student = x.gather(1, ids.clamp(min=0)) - lse[:, None]
    row = (q * (t - student).masked_fill(~keep, 0.0)).sum(dim=1)
    grad = torch.exp(x - lse[:, None])                          # p
    if case["tail"]:
        # the student's mass off the list, summed over those tokens alone
        off = x.clone()
        off[torch.arange(case["rows"], device=x.device)[:, None].expand_as(ids)[keep], ids[keep]] = -math.inf
        log_r = torch.logsumexp(off, dim=1) - lse
        rest = (1.0 - q.sum(dim=1)).clamp(min=0.0)
        row = row + torch.where(rest > 0, rest * (rest.log() - log_r), torch.zeros_like(rest))
        # d(-rest log r)/dx = rest p - rest softmax(x off the list)
        listed_mass = q.sum(dim=1)
        grad = grad * (listed_mass + rest)[:, None] - rest[:, None] * torch.exp(off - lse[:, None] - log_r[:, None])
    grad.scatter_add_(1, ids.clamp(min=0), -q)
    row = row * tau ** 2 * (w != 0)
    return {"loss": (row * w).sum(), "row_loss": row, "dlogits": grad * (w * tau)[:, None]}
