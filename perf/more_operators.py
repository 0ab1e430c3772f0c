"""What stands between a model's logits and its gradients, as cases that can be timed and compared: the scores of given tokens, and
distillation from a teacher of which only the top tokens are kept.

A case is a dict of plain values.  `op` names the call:

  token_logprobs       log probability of each row's token, with the row's entropy and its top alternatives
  token_logprobs_grad  the logits' gradient from those of the log probabilities and of the entropies
  distill_top          divergence from a teacher's top tokens, renormalised or with all others as one more class
  distill_top_grad     the logits' gradient of that

Where `own` is false the operators run in elementary torch operations in 32 bits, the teacher's few tokens in 64: what it and the
student leave to the rest are ones minus small sums, and the loss is the difference of the two.
"""
import math

import torch

own = False  # set by whoever measures: False for the plain forms, True for the framework's kernels

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _case(op, **given):
    """Every case says all choices of its operator."""
    choices = {"token_logprobs": dict(rows=1, vocab=1, dtype="bf16", temperature=1.0, masked=0.0, entropy=False, top=0),
               "token_logprobs_grad": dict(rows=1, vocab=1, dtype="bf16", temperature=1.0, masked=0.0, entropy=False, ignored=0.0, out="bf16"),
               "distill_top": dict(rows=1, vocab=1, dtype="bf16", temperature=1.0, masked=0.0, k=1, teacher="f32", rest=False),
               "distill_top_grad": dict(rows=1, vocab=1, dtype="bf16", temperature=1.0, masked=0.0, k=1, teacher="f32", rest=False, ignored=0.0, out="bf16")}[op]
    return dict(choices, op=op, **given)


def listed():
    return [
        # one new token while serving, with alternatives: latency counts
        _case("token_logprobs", name="score_one_token", rows=1, vocab=128000, top=20),
        # the tokens of many requests at once, sampled at a temperature under a grammar that forbids most of the vocabulary
        _case("token_logprobs", name="score_requests", rows=64, vocab=128000, dtype="f32", temperature=0.7, masked=0.75, top=5, entropy=True),
        # a document's perplexity, odd sizes
        _case("token_logprobs", name="score_document", rows=4095, vocab=10007, dtype="f32"),
        # policy training: log probabilities and entropies of a batch of answers
        _case("token_logprobs", name="score_answers", rows=16384, vocab=32000, entropy=True),
        # running the teacher: its top tokens are kept for later
        _case("token_logprobs", name="score_teacher", rows=8192, vocab=128000, temperature=2.0, top=64),
        # fine-tuning on prompts of which only the answers count
        _case("token_logprobs_grad", name="grad_answers", rows=616, vocab=49408, ignored=0.5),
        # odd sizes in 32 bits
        _case("token_logprobs_grad", name="grad_odd_f32", rows=1025, vocab=10007, dtype="f32", temperature=0.7, entropy=True, out="f32"),
        # the backward pass of policy training, with its bonus for entropy
        _case("token_logprobs_grad", name="grad_batch", rows=8192, vocab=128000, entropy=True),
        # a short sequence's loss
        _case("distill_top", name="distill_sequence", rows=77, vocab=49408, k=20, temperature=2.0),
        # a training batch; the teacher's rest is one more class
        _case("distill_top", name="distill_batch", rows=8192, vocab=128000, k=64, temperature=2.0, rest=True),
        # odd sizes in 32 bits, a teacher stored in 16
        _case("distill_top_grad", name="distill_grad_odd_f32", rows=1025, vocab=10007, dtype="f32", k=17, teacher="bf16", rest=True, out="f32"),
        # the backward pass of the training batch
        _case("distill_top_grad", name="distill_grad_batch", rows=8192, vocab=128000, k=64, temperature=2.0, rest=True, ignored=0.1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _vocab(rng):
    """A vocabulary's size: of the usual multiples, or any."""
    to = rng.choice([1, 1, 8, 64, 128])
    return max(128, _log_int(rng, 128, 262144) // to * to)


def draw(rng):
    """One more case of the same ranges."""
    op = rng.choice(["token_logprobs", "token_logprobs_grad", "distill_top", "distill_top_grad"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    out = rng.choice([dtype, dtype, "f32"])
    vocab = _vocab(rng)
    rows = min(_log_int(rng, 1, 16384), max(1, (1000000000 if dtype == "bf16" and out == "bf16" else 500000000) // vocab))
    case = dict(rows=rows, vocab=vocab, dtype=dtype, temperature=rng.choice([1.0, 1.0, round(rng.uniform(0.5, 4.0), 2)]),
                masked=rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.9), 2)]))
    if op.startswith("distill"):
        case.update(k=rng.choice([1, 5, 8, 20, 50, 64, rng.randint(1, 64)]), teacher=rng.choice(["f32", "bf16"]), rest=rng.random() < 0.5)
    else:
        case["entropy"] = rng.random() < 0.5
    if op == "token_logprobs":
        case["top"] = rng.choice([0, 0, 1, 5, 20, 64, rng.randint(1, 64)])
    if op.endswith("grad"):
        case.update(out=out, ignored=rng.choice([0.0, round(rng.uniform(0.01, 0.8), 2)]))
    return _case(op, **case)


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------

IGNORED = -100


def _spread(rows, cols, g, masked):
    """Logits as a trained model's: most of them within a few units, a few far above; and which columns hold the latter.

    `masked` is the share of the other columns that stand at minus infinity."""
    x = torch.randn(rows, cols, generator=g, device="cuda").mul_(2.0)
    if masked:
        x.masked_fill_(torch.rand(rows, cols, generator=g, device="cuda") < masked, -math.inf)
    peaks = torch.randint(0, cols, (rows, 8), generator=g, device="cuda")
    x.scatter_(1, peaks, torch.rand(rows, 8, generator=g, device="cuda") * 10 + 6)
    return x, peaks


def _tops(x, k):
    """The k largest of each row with their columns; of equal ones the lowest columns first."""
    bits = (x + 0.0).view(torch.int32).long()  # minus zero is zero
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)  # as the values are ordered
    last = x.shape[1] - 1
    keys = order.mul_(x.shape[1]).add_(last - torch.arange(x.shape[1], device=x.device))
    ids = last - torch.topk(keys, k, 1).values % x.shape[1]
    return x.gather(1, ids), ids


def _stats(x, t):
    """The largest of each row and the log of the sum of exp((x - largest) / t), in 32 bits."""
    most = x.amax(1, keepdim=True)
    return torch.cat((most, ((x - most) / t).exp().sum(1, keepdim=True).log()), 1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, vocab, t = case["rows"], case["vocab"], case["temperature"]
    x, peaks = _spread(rows, vocab, g, case["masked"])
    s = dict(case=case, logits=x.to(DTYPES[case["dtype"]]))

    def row_values(scale, mean=0.0):
        return torch.randn(rows, generator=g, device="cuda").mul_(scale).add_(mean)

    def some_rows():
        return torch.rand(rows, generator=g, device="cuda") < case["ignored"]

    if case["op"].startswith("token"):
        s["ids"] = peaks[:, 0].clone()
        if not case["masked"]:  # and now and then a token that nobody would have expected
            odd = torch.rand(rows, generator=g, device="cuda") < 0.2
            s["ids"] = torch.where(odd, torch.randint(0, vocab, (rows,), generator=g, device="cuda"), s["ids"])
        if case["op"] == "token_logprobs_grad":  # what the forward pass left, and the gradients that arrive
            s["ids"][some_rows()] = IGNORED
            s["stats"] = _stats(s["logits"].float(), t)
            s["grad"] = row_values(1.0 / rows)
            s["grad_entropy"] = s["entropy"] = None
            if case["entropy"]:
                s["grad_entropy"] = row_values(1e-3 / rows, -1e-2 / rows).masked_fill_(s["ids"] == IGNORED, 0.0)
                s["entropy"] = _plain_entropy(s["logits"].float(), s["stats"], t)
        return s
    # a teacher that agrees with the student on some of its favourites: log probabilities at the loss's temperature
    teacher, _ = _spread(rows, vocab, g, 0.0)
    teacher[:, :] = torch.where(x.isinf(), x, teacher)
    teacher.scatter_(1, peaks[:, :4], torch.rand(rows, 4, generator=g, device="cuda") * 10 + 6)
    teacher.div_(t)
    most = teacher.amax(1, keepdim=True)
    norm = (teacher - most).exp().sum(1, keepdim=True).log() + most
    values, ids = torch.topk(teacher, case["k"], 1)
    s.update(ids=ids, teacher=(values - norm).to(DTYPES[case["teacher"]]))
    if case["op"] == "distill_top_grad":
        s["stats"] = _plain_distill_top(s, case)["stats"]
        s["grad"] = row_values(0.2 / rows, 1.0 / rows).masked_fill_(some_rows(), 0.0)
    return s


# ---------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------

def _plain_entropy(x, stats, t):
    d = (x - stats[:, :1]) / t
    e = d.exp()
    return stats[:, 1] - torch.where(e > 0, e * d, 0.0).sum(1) / e.sum(1)


def _plain_token_logprobs(s, case):
    x, t = s["logits"].float(), case["temperature"]
    stats = _stats(x, t)
    out = {"stats": stats, "logprob": (x.gather(1, s["ids"][:, None]).squeeze(1) - stats[:, 0]) / t - stats[:, 1]}
    if case["entropy"]:
        out["entropy"] = _plain_entropy(x, stats, t)
    if case["top"]:
        values, out["top_ids"] = _tops(x, case["top"])
        out["top"] = (values - stats[:, :1]) / t - stats[:, 1:]
    return out


def _plain_token_logprobs_grad(s, case):
    x, t, ids = s["logits"].float(), case["temperature"], s["ids"]
    logp = (x - s["stats"][:, :1]) / t - s["stats"][:, 1:]
    p = logp.exp()
    real = ids != IGNORED
    g = torch.where(real, s["grad"], 0.0)[:, None]
    dx = -g * p
    if case["entropy"]:
        dx -= s["grad_entropy"][:, None] * torch.where(p > 0, p * (logp + s["entropy"][:, None]), 0.0)
    dx.scatter_add_(1, torch.where(real, ids, 0)[:, None], g)
    return {"logits": (dx / t).to(DTYPES[case["out"]])}


def _shares(teacher, apart):
    """The teacher's probabilities, the log of what they are divided by, and their sum, in 64 bits.

    In rows where the rest is no class of its own the probabilities are renormalised."""
    teacher = teacher.double()
    most = teacher.amax(1, keepdim=True)
    norm = (teacher - most).exp().sum(1, keepdim=True).log() + most
    norm = torch.where(apart[:, None], norm.clamp(min=0.0), norm)
    q = (teacher - norm).exp()
    return q, norm, q.sum(1)


def _plain_distill_top(s, case):
    """stats: largest logit and log of the sum of exp, the same over the tokens that the teacher does not name where they are a
    class, the log of the teacher's divisor, and by how much the student's share for the rest is over the teacher's (1 where it is
    no class).  It is none where the student leaves it nothing."""
    x, ids, t = s["logits"].float(), s["ids"], case["temperature"]
    others = all_ = _stats(x, t)
    apart = torch.zeros_like(x[:, 0], dtype=torch.bool)
    if case["rest"]:
        outside = x.scatter(1, ids, -math.inf)
        apart = outside.amax(1) > -math.inf
        others = torch.where(apart[:, None], _stats(outside, t), all_)
    q, norm, named = _shares(s["teacher"], apart)
    logp = (x.gather(1, ids).double() - all_[:, :1]) / t - ((x - all_[:, :1]) / t).exp().sum(1, keepdim=True).double().log()
    loss = torch.where(q > 0, q * (s["teacher"].double() - norm - logp), 0.0).sum(1)
    named_p, log_rest = logp.exp().sum(1), (others[:, 0].double() - all_[:, 0]) / t + others[:, 1] - all_[:, 1]
    # the log of what is left: from what is not, where that is the smaller part
    log_rest = torch.where(named_p < 0.5, torch.log1p(-named_p.clamp(max=0.5)), log_rest)
    rest = (1 - named).clamp(min=0.0)
    loss = loss + torch.where(apart & (rest > 0), rest * (torch.log1p(-named.clamp(max=1 - 1e-16)) - log_rest), 0.0)
    over = torch.where(apart, torch.where(named_p < 0.5, named - named_p, log_rest.exp() - rest), 1.0)
    return {"loss": loss.float(), "stats": torch.cat((all_, others, norm.float(), over.float()[:, None]), 1)}


def _plain_distill_top_grad(s, case):
    x, ids, t, stats = s["logits"].float(), s["ids"], case["temperature"], s["stats"]
    q = (s["teacher"].float() - stats[:, 4:5]).exp()
    share = ((x - stats[:, 2:3]) / t - stats[:, 3:4]).exp() * stats[:, 5:]  # of each token among the others
    p = ((x.gather(1, ids) - stats[:, :1]) / t - stats[:, 1:2]).exp()
    dx = share.scatter(1, ids, p - q)
    return {"logits": (dx * (s["grad"] / t)[:, None]).to(DTYPES[case["out"]])}


PLAIN = {"token_logprobs": _plain_token_logprobs, "token_logprobs_grad": _plain_token_logprobs_grad,
         "distill_top": _plain_distill_top, "distill_top_grad": _plain_distill_top_grad}


# ---------------------------------------------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------------------------------------------

def _own_token_logprobs(losses, s, case):
    r = losses.token_logprobs(s["logits"], s["ids"], temperature=case["temperature"], entropy=case["entropy"], top=case["top"])
    out = {"stats": r.stats, "logprob": r.logprob}
    if case["entropy"]:
        out["entropy"] = r.entropy
    return dict(out, top=r.top, top_ids=r.top_ids) if case["top"] else out


def _own_token_logprobs_grad(losses, s, case):
    return {"logits": losses.token_logprobs_grad(s["logits"], s["ids"], s["stats"], s["grad"], grad_entropy=s["grad_entropy"], entropy=s["entropy"],
                                                 temperature=case["temperature"], dtype=DTYPES[case["out"]])}


def _own_distill_top(losses, s, case):
    r = losses.distill_top(s["logits"], s["ids"], s["teacher"], temperature=case["temperature"], rest=case["rest"])
    return {"loss": r.loss, "stats": r.stats}


def _own_distill_top_grad(losses, s, case):
    return {"logits": losses.distill_top_grad(s["logits"], s["ids"], s["teacher"], s["stats"], s["grad"], temperature=case["temperature"],
                                              dtype=DTYPES[case["out"]])}


OWN = {"token_logprobs": _own_token_logprobs, "token_logprobs_grad": _own_token_logprobs_grad,
       "distill_top": _own_distill_top, "distill_top_grad": _own_distill_top_grad}


def run(state):
    case = state["case"]
    if own:
        from eridiffusion_amd import losses
        return OWN[case["op"]](losses, state, case)
    return PLAIN[case["op"]](state, case)


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without, and the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------

def work(case):
    size = {"bf16": 2, "f32": 4}
    rows, n = case["rows"], case["rows"] * case["vocab"]
    read = n * size[case["dtype"]] * (1 - case.get("ignored", 0.0))
    small = rows * case["k"] * (8 + size[case["teacher"]]) if "k" in case else rows * 8
    if case["op"] == "token_logprobs":
        small += rows * (12 + 4 * case["entropy"] + 12 * case["top"])
        return {"bytes": read + small, "flops": n * (4 + 2 * case["entropy"])}
    if case["op"] == "token_logprobs_grad":
        small += rows * (12 + 8 * case["entropy"])
        return {"bytes": read + small + n * size[case["out"]], "flops": n * (1 - case["ignored"]) * (5 + 3 * case["entropy"])}
    if case["op"] == "distill_top":
        return {"bytes": read + small + rows * 28, "flops": n * 4}
    return {"bytes": read + small + rows * 28 + n * size[case["out"]], "flops": n * (1 - case["ignored"]) * 5}


def _by_rows(case, s, one):
    """`one` over parts of the rows, so that 64 bits fit, joined."""
    step = max(1, (1 << 27) // case["vocab"])
    parts = [one({k: v[at:at + step] if isinstance(v, torch.Tensor) else v for k, v in s.items()}) for at in range(0, case["rows"], step)]
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}


def _exact_token_logprobs(s, case):
    z = s["logits"].double() / case["temperature"]
    most = z.max(1).values
    logsum = torch.logsumexp(z - most[:, None], 1)
    p = torch.softmax(z, 1)
    out = {"stats": torch.stack((most * case["temperature"], logsum), 1), "logprob": torch.log_softmax(z, 1)[torch.arange(z.shape[0], device=z.device), s["ids"]]}
    if case["entropy"]:
        out["entropy"] = -torch.special.xlogy(p, p).sum(1)
    if case["top"]:
        values, ids = torch.sort(s["logits"].double(), dim=1, descending=True, stable=True)
        out["top_ids"] = ids[:, :case["top"]].clone()
        out["top"] = values[:, :case["top"]] / case["temperature"] - (most + logsum)[:, None]
    return out


def _exact_token_logprobs_grad(s, case):
    z = s["logits"].double() / case["temperature"]
    logp = z - torch.logsumexp(z, 1, keepdim=True)
    p = logp.exp()
    one = s["ids"][:, None] == torch.arange(case["vocab"], device=z.device)
    real = (s["ids"] >= 0).double()[:, None]
    dz = s["grad"].double()[:, None] * (one.double() - p * real)
    if case["entropy"]:
        plogp = torch.special.xlogy(p, p)
        dz -= s["grad_entropy"].double()[:, None] * (plogp - p * plogp.sum(1, keepdim=True))
    return {"logits": dz / case["temperature"]}


def _exact_distill(s, case):
    """Loss, gradient and stats over the classes: the teacher's tokens, and the others as one where they count."""
    t = case["temperature"]
    z = s["logits"].double() / t
    log_all = torch.logsumexp(z, 1, keepdim=True)
    outside = torch.where(torch.zeros_like(z).scatter_(1, s["ids"], 1.0) > 0, -math.inf, z)
    log_others = torch.logsumexp(outside, 1, keepdim=True)
    apart = (log_others > -math.inf) if case["rest"] else torch.zeros_like(log_all, dtype=torch.bool)
    outside, log_others = torch.where(apart, outside, z), torch.where(apart, log_others, log_all)
    weight = s["teacher"].double().exp()
    total = weight.sum(1, keepdim=True)
    total = torch.where(apart & (total < 1), 1.0, total)
    q = weight / total
    rest = torch.where(apart, 1 - q.sum(1, keepdim=True), 0.0).clamp(min=0.0)
    logp = (z - log_all).gather(1, s["ids"])
    loss = torch.special.xlogy(q, q) - torch.where(q > 0, q * logp, 0.0)
    loss_rest = torch.special.xlogy(rest, rest) - rest * (log_others - log_all)
    most, most_others = s["logits"].double().max(1, keepdim=True).values, outside.max(1, keepdim=True).values * t
    over = torch.where(apart, q.sum(1, keepdim=True) - torch.where(torch.zeros_like(z).scatter_(1, s["ids"], 1.0) > 0, (z - log_all).exp(), 0.0).sum(1, keepdim=True), 1.0)
    stats = (most, log_all - most / t, most_others, log_others - most_others / t, total.log(), over)
    dz = (z - log_all).exp() - rest * torch.where(apart, (outside - log_others).exp(), 0.0)
    dz.scatter_add_(1, s["ids"], -q)
    return {"loss": loss.sum(1) + loss_rest.squeeze(1), "dx": dz / t, "stats": torch.cat(stats, 1)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "token_logprobs":
        return _by_rows(case, s, lambda r: _exact_token_logprobs(r, case))
    if case["op"] == "token_logprobs_grad":
        return _by_rows(case, s, lambda r: _exact_token_logprobs_grad(r, case))

    def part(r):
        got = _exact_distill(r, case)
        if case["op"] == "distill_top":
            return {"loss": got["loss"], "stats": got["stats"]}
        return {"logits": got["dx"] * r["grad"].double()[:, None]}
    return _by_rows(case, s, part)
