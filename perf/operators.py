"""Workloads of the vocabulary-head operators: log-probabilities of given tokens, the largest log-probabilities of a teacher and
distillation from them, each straight from hidden states (or logits) over the whole vocabulary.

`own` chooses what `run` does: the plain form in elementary torch operations, or the framework's operators.  Sizes are the heads of the
two Qwen2.5-VL configurations (2048 x 151936 and 3584 x 152064) and generic smaller ones."""
import math

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def listed():
    return [
        # scoring of given tokens (no gradient): the old / reference policy's log-probabilities of a response
        dict(name="score-1x2048", kind="score", rows=1, hidden=2048, vocab=151936, temperature=1.0),           # one token of one sequence
        dict(name="score-203x3584", kind="score", rows=203, hidden=3584, vocab=152064, temperature=0.7),       # one short response
        dict(name="score-4096x3584", kind="score", rows=4096, hidden=3584, vocab=152064, temperature=1.0),     # a pass of the old policy
        # the same with the gradients of hidden states and head: the policy update
        dict(name="train-77x1024", kind="train", rows=77, hidden=1024, vocab=50257, temperature=1.0),          # a small model, odd vocabulary
        dict(name="train-1000x2048", kind="train", rows=1000, hidden=2048, vocab=151936, temperature=1.0),     # a micro-batch of the 2048-wide head
        dict(name="train-8192x3584", kind="train", rows=8192, hidden=3584, vocab=152064, temperature=1.0),     # an update pass
        # a teacher's largest log-probabilities, from its logits
        dict(name="top-1x20", kind="top", rows=1, vocab=152064, k=20, temperature=1.0),                        # one token being sampled
        dict(name="top-2048x64", kind="top", rows=2048, vocab=152064, k=64, temperature=1.0),                  # a teacher pass
        # distillation from them
        dict(name="distill-150x2048", kind="distill", rows=150, hidden=2048, vocab=151936, k=8, temperature=2.0, renormalize=True),
        dict(name="distill-1501x3584", kind="distill", rows=1501, hidden=3584, vocab=152064, k=33, temperature=1.0, renormalize=True),
        dict(name="distill-4096x3584", kind="distill", rows=4096, hidden=3584, vocab=152064, k=64, temperature=1.0, renormalize=False),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["score", "train", "top", "distill"])
    hidden, vocab = rng.choice([(2048, 151936), (3584, 152064), (64 * rng.randint(2, 56), _log_uniform(rng, 500, 152064))])
    temperature = rng.choice([1.0, round(rng.uniform(0.5, 2.0), 2)])
    if kind == "top":
        return dict(kind=kind, rows=_log_uniform(rng, 1, 2048), vocab=vocab, k=_log_uniform(rng, 1, 128), temperature=temperature)
    if kind == "distill":
        return dict(kind=kind, rows=_log_uniform(rng, 1, 4096), hidden=hidden, vocab=vocab, k=_log_uniform(rng, 1, 128), temperature=temperature,
                    renormalize=rng.random() < 0.5)
    return dict(kind=kind, rows=_log_uniform(rng, 1, 8192), hidden=hidden, vocab=vocab, temperature=temperature)


def _head(case, seed):
    """Hidden states behind a final norm, the head, and tokens that the model gives anything from 1 / vocab to nearly 1."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, hidden, vocab = case["rows"], case["hidden"], case["vocab"]
    weight = torch.empty(vocab, hidden, device="cuda", dtype=BF16).normal_(0.0, 1.4 / math.sqrt(hidden), generator=g)
    token = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    toward = weight[token].float()
    h = torch.randn(rows, hidden, device="cuda", generator=g)
    h += (20.0 * torch.rand(rows, 1, device="cuda", generator=g)) * toward / toward.square().sum(1, keepdim=True)
    return g, h, weight, token


def prepare(case, seed):
    if case["kind"] == "top":
        g = torch.Generator(device="cuda").manual_seed(seed)
        hidden = 256
        weight = torch.empty(case["vocab"], hidden, device="cuda", dtype=BF16).normal_(0.0, 1.0, generator=g)
        h = torch.randn(case["rows"], hidden, device="cuda", generator=g) * (0.06 + 0.2 * torch.rand(case["rows"], 1, device="cuda", generator=g))
        return dict(case=case, logits=h.to(BF16) @ weight.t())
    g, h, weight, token = _head(case, seed)
    state = dict(case=case, hidden=h.to(BF16), weight=weight)
    rows = case["rows"]
    if case["kind"] == "distill":
        k, vocab = min(case["k"], case["vocab"]), case["vocab"]
        teacher = (h + torch.randn(h.shape, device="cuda", generator=g)).to(BF16)
        logits = (teacher @ weight.t()).float().div_(case["temperature"])
        lse = torch.logsumexp(logits, 1, keepdim=True)
        top, ids = torch.topk(logits, k, dim=1)
        absent = torch.rand(rows, k, device="cuda", generator=g) < 0.03                 # ragged teachers: some slots hold nothing
        absent[torch.rand(rows, device="cuda", generator=g) < 0.02] = True             # rows that are masked as a whole
        state["ids"] = ids.masked_fill(absent, -1).to(torch.int32)
        state["teacher"] = top - lse
    else:
        state["labels"] = token.masked_fill(torch.rand(rows, device="cuda", generator=g) < 0.05, -100)     # prompt and padding rows
    if case["kind"] != "score":
        state["grad"] = torch.randn(rows, device="cuda", generator=g) * (2.0 / rows)
        state["hidden"].requires_grad_(True)
        state["weight"].requires_grad_(True)
    return state


# ---------------------------------------------------------------- the framework's operators
def _run_own(s):
    from verl.utils import torch_functional as F
    case = s["case"]
    if case["kind"] == "top":
        ids, logp, lse = F.top_log_probs(s["logits"], case["k"], temperature=case["temperature"])
        return dict(ids=ids, logp=logp, lse=lse)
    if case["kind"] == "score":
        with torch.no_grad():
            return dict(logp=F.linear_log_probs(s["hidden"], s["weight"], s["labels"], temperature=case["temperature"]))
    if case["kind"] == "train":
        out = F.linear_log_probs(s["hidden"], s["weight"], s["labels"], temperature=case["temperature"])
        name = "logp"
    else:
        out = F.linear_topk_kl(s["hidden"], s["weight"], s["ids"], s["teacher"], temperature=case["temperature"], renormalize=case["renormalize"])
        name = "kl"
    dhidden, dweight = torch.autograd.grad(out, (s["hidden"], s["weight"]), s["grad"])
    return {name: out.detach(), "dhidden": dhidden, "dweight": dweight}


# ---------------------------------------------------------------- the plain form
def _log_softmax32(s):
    z = s["hidden"].float() @ s["weight"].float().t() / s["case"]["temperature"]
    m = z.amax(1, keepdim=True)
    return z - (m + (z - m).exp().sum(1, keepdim=True).log())


def _grads32(s, dz):
    dz = dz / s["case"]["temperature"]
    return (dz @ s["weight"].float()).to(BF16), (dz.t() @ s["hidden"].float()).to(BF16)


def _run_plain(s):
    case = s["case"]
    if case["kind"] == "top":
        z = s["logits"].float()
        vocab = z.shape[1]
        # ties go to the lowest id: order by (value, -id) in one whole number, exact for 16-bit values
        bits = s["logits"].view(torch.int16).long() & 0xffff
        up = torch.where(bits >= 0x8000, 0x8000 - (bits & 0x7fff), 0x8000 + bits)
        key = (up << 32) + (vocab - 1 - torch.arange(vocab, device=z.device))
        ids = vocab - 1 - (torch.topk(key, min(case["k"], vocab), dim=1).values & 0xffffffff)
        z = z / case["temperature"]
        m = z.amax(1, keepdim=True)
        lse = m + (z - m).exp().sum(1, keepdim=True).log()
        return dict(ids=ids.to(torch.int32), logp=z.gather(1, ids) - lse, lse=lse[:, 0])
    if case["kind"] == "distill":
        ids, have = s["ids"].long().clamp(min=0), s["ids"] >= 0
        a = s["teacher"].masked_fill(~have, -math.inf)
        if case["renormalize"]:
            m = a.amax(1, keepdim=True).clamp(min=-1e30)
            a = a - (m + (a - m).exp().sum(1, keepdim=True).log())
        p = torch.where(have, a.exp(), 0.0)
        logq = _log_softmax32(s)
        kl = torch.where(have, p * (a.masked_fill(~have, 0.0) - logq.gather(1, ids)), 0.0).sum(1)
        dz = logq.exp() * (s["grad"] * p.sum(1))[:, None]
        dz.scatter_add_(1, ids, -s["grad"][:, None] * p)
        dhidden, dweight = _grads32(s, dz)
        return dict(kl=kl, dhidden=dhidden, dweight=dweight)
    live = s["labels"] >= 0
    label = s["labels"].clamp(min=0)[:, None]
    logq = _log_softmax32(s)
    logp = torch.where(live, logq.gather(1, label)[:, 0], 0.0)
    if case["kind"] == "score":
        return dict(logp=logp)
    g = torch.where(live, s["grad"], 0.0)[:, None]
    dz = -g * logq.exp()
    dz.scatter_add_(1, label, g)
    dhidden, dweight = _grads32(s, dz)
    return dict(logp=logp, dhidden=dhidden, dweight=dweight)


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _run_plain(state)


def work(case):
    rows, vocab = case["rows"], case["vocab"]
    if case["kind"] == "top":
        return dict(bytes=2.0 * rows * vocab + 8.0 * rows * case["k"] + 4.0 * rows, flops=0.0)
    operands = 2.0 * rows * case["hidden"] + 2.0 * vocab * case["hidden"]
    product = 2.0 * rows * vocab * case["hidden"]
    if case["kind"] == "score":
        return dict(bytes=operands + 12.0 * rows, flops=product)
    targets = 8.0 * rows * case["k"] if case["kind"] == "distill" else 8.0 * rows
    return dict(bytes=2.0 * operands + targets + 8.0 * rows, flops=3.0 * product)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "top":
        z = s["logits"].to(F64)
        order = torch.sort(z, dim=1, descending=True, stable=True)
        ids = order.indices[:, :case["k"]]
        logq = torch.log_softmax(z / case["temperature"], 1)
        return dict(ids=ids.to(torch.int32), logp=logq.gather(1, ids), lse=torch.logsumexp(z / case["temperature"], 1))
    h, w = (s[n].detach().to(F64).requires_grad_(case["kind"] != "score") for n in ("hidden", "weight"))
    logq = torch.log_softmax((h @ w.t()) / case["temperature"], dim=1)
    if case["kind"] == "distill":
        have = s["ids"] >= 0
        a = s["teacher"].to(F64)
        p = torch.where(have, a.exp(), 0.0)
        if case["renormalize"]:
            total = p.sum(1, keepdim=True)
            a = a - torch.where(total > 0, total, 1.0).log()
            p = torch.where(have, a.exp(), 0.0)
        out = (p * (a - logq.gather(1, s["ids"].long().clamp(min=0)))).sum(1)
        name = "kl"
    else:
        live = s["labels"] >= 0
        out = logq.gather(1, s["labels"].clamp(min=0)[:, None])[:, 0].masked_fill(~live, 0.0)
        name = "logp"
    if case["kind"] == "score":
        return {name: out}
    dhidden, dweight = torch.autograd.grad(out, (h, w), s["grad"].to(F64))
    return {name: out.detach(), "dhidden": dhidden, "dweight": dweight}
